// Sampling of the next token for gfx950: temperature, top-k, top-p, min-p and
// the draw, from a uniform number per row.
//
// With m the row's largest logit, w_i = exp((l_i - m) / temperature), and the
// words ordered by (logit descending, index ascending): kept are the first k; of
// these those whose weight before them is below top_p of the k's total (the first
// always); of these those with w_i >= min_p. The token is the first kept word, by
// index, whose running sum of kept weights exceeds uniform times their total.
//
// Which word that is turns on where sums cross a border, so that weights are
// computed in 64 bits and summed as integers, w 2^S rounded (S 45, less above
// 2^17 words): sums that no order of additions changes, off by less than 2^-S of the
// likeliest word's weight per word.
//
// The first kernel has a block per row. It reads the words for the maximum, each thread's own
// being kept; the k-th largest of the threads' maxima bounds the k-th largest logit from
// below (min-p bounds the kept words in the same way), and a second reading collects the few
// words from there on in LDS. Up to 1024 words are all taken. What is asked of such a list
// (the k-th word, the one at top-p's border, by index the one that is drawn) is each the first, in
// an order, at which a running sum reaches a number: a descent over the order's bits, six at a
// time, with the digits' sums in LDS.
// The rows whose settings keep more words are left to further kernels: the weights by bins
// of their logarithm (1/16 of a factor of 2), by part of 8192 words and by row, a block per part;
// the words of the bin in which top-p's border falls, collected; and, by a block per row, their
// cut, the part in which the draw falls (from the bins), and the word.
// What no list holds (very many words of one weight, k above 1024 of many words) is found by
// a search over the bits of the logits' keys, a reading each.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kMassBins = 1024;   // of 2^-1/16, down to 2^-64
constexpr int kAllWords = 1024;   // up to this many words the first kernel takes all
constexpr int kPart = 8192;       // words of a part
constexpr int kFirstList = 2048;  // words of the first kernel's list
constexpr int kRowList = 4096;    // of a row's list behind it

struct SampleArgs {
  const void* logits;        // (rows, vocab), rows ld apart
  long long ld;
  const float* uniform;      // (rows)
  const float *temperature, *top_p, *min_p;   // (rows), or null: the values below
  const void* top_k;
  int k64;
  float temperature_v, top_p_v, min_p_v;
  long long top_k_v;
  long long* tokens;         // (rows)
  float* logprobs;           // (rows) or null
  int vocab, scale;          // weights are counted in 2^-scale
  // what the first kernel leaves
  struct SampleRow* state;   // (rows)
  unsigned long long* bins;  // (rows, parts, kMassBins)
  int parts;
};
// What is left of a row: nothing; to look at all words; to cut and draw from list; to
// search for the border.
constexpr int kRowDone = 0, kRowAll = 1, kRowCut = 2, kRowSearch = 3;
struct SampleRow {
  float m;
  int left;
  unsigned count;    // of list
  int unused;
  unsigned long long total[kMassBins], list[kRowList];
};

// Bits of an fp32 that a T's value never sets.
template <class T> constexpr int kLowBits = 0;
template <> constexpr int kLowBits<Bf16> = 16;
template <> constexpr int kLowBits<Fp16> = 13;

// A logit as it counts: NaN as -inf, -0 as 0.
__device__ __forceinline__ float as_logit(float v) { return v == v ? v + 0.f : -INFINITY; }
template <class T>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  return as_logit(ld_p<T>(row, i));
}
// Keys order as their floats do.
template <class T>
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned u = __float_as_uint(v);
  return (u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u)) >> kLowBits<T>;
}
template <class T>
__device__ __forceinline__ float value_of(unsigned key) {
  unsigned u = key << kLowBits<T>;
  if (u >> 31) u ^= 0x80000000u;
  else u = ~(u | ((1u << kLowBits<T>) - 1));
  return __uint_as_float(u);
}

typedef unsigned long long u64;

// A word's place in the order, the first the largest: by key, then by index.
__device__ __forceinline__ u64 place_of(unsigned key, int i) {
  return (u64)key << 32 | (0xFFFFFFFFu - (unsigned)i);
}
__device__ __forceinline__ int index_at(u64 place) { return (int)(0xFFFFFFFFu - (unsigned)place); }

template <int NTH_, int LIST>
struct SampleShared {
  static constexpr int NTH = NTH_, kWaves = NTH / 64, kList = LIST, E = LIST / NTH;
  union {
    u64 bins[kMassBins];
    u64 list[LIST];
  };
  u64 digits[3][64];
  u64 wave[kWaves];
  float wave_f[kWaves];
  u64 above;
  unsigned bin, count;
};

// v of the lane that CTRL names in the rows of ROWS, 0 where there is none.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xF,
                                                  false);
  return (u64)hi << 32 | lo;
}
// Inclusive sum of v over the lanes up to this one: within the rows of 16 lanes by shifts, then
// the last lane of a row to the next one (row_bcast:15) and of the first half to the second
// (row_bcast:31).
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v += dpp_u64<0x111>(v);
  v += dpp_u64<0x112>(v);
  v += dpp_u64<0x114>(v);
  v += dpp_u64<0x118>(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane);
}
__device__ __forceinline__ u64 wave_total(u64 v) { return lane_u64(wave_scan(v), 63); }
// The block's sum of v, in every thread.
template <class Sh>
__device__ __forceinline__ u64 block_total(Sh& sh, u64 v) {
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int w = 0; w < Sh::kWaves; ++w) s += sh.wave[w];
  __syncthreads();
  return s;
}
// The sum of v over the threads before this one.
template <class Sh>
__device__ __forceinline__ u64 block_before(Sh& sh, u64 v, u64* total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const u64 run = wave_scan(v);
  __syncthreads();
  if (lane == 63) sh.wave[wave] = run;
  __syncthreads();
  u64 before = run - v, all = 0;
#pragma unroll
  for (int w = 0; w < Sh::kWaves; ++w) {
    if (w < wave) before += sh.wave[w];
    all += sh.wave[w];
  }
  __syncthreads();
  *total = all;
  return before;
}

// f(i, word i, group) for the words lo .. lo + n - 1, each once, by `threads` threads (this one
// is number t): 16 bytes at a time but for the ends, four such loads in flight. The group
// (0 .. 3) names one of four about equal shares of the thread's words.
template <class T, class F>
__device__ __forceinline__ void for_groups(const char* row, int lo, int n, int t, int threads,
                                           F&& f) {
  constexpr int E = kElem<T>, W = 16 / E;
  const char* p = row + (size_t)lo * E;
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / E);
  for (int i = t; i < head; i += threads) f(lo + i, ld_p<T>(row, lo + i), 0);
  const int vecs = (n - head) / W;
  const uint4* q = reinterpret_cast<const uint4*>(p + (size_t)head * E);
  const int b = lo + head;
  const auto word = [&](const uint4& r, int v, int group) {
    const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < W; ++e) {
      float x;
      if constexpr (E == 4) x = __uint_as_float(u[e]);
      else x = T::to((unsigned short)(u[e / 2] >> (16 * (e & 1))));
      f(b + v * W + e, x, group);
    }
  };
  int v = t;
  for (; v + 3 * threads < vecs; v += 4 * threads) {
    const uint4 r0 = q[v], r1 = q[v + threads], r2 = q[v + 2 * threads], r3 = q[v + 3 * threads];
    word(r0, v, 0);
    word(r1, v + threads, 1);
    word(r2, v + 2 * threads, 2);
    word(r3, v + 3 * threads, 3);
  }
  if (v < vecs) word(q[v], v, 0);
  if (v + threads < vecs) word(q[v + threads], v + threads, 1);
  if (v + 2 * threads < vecs) word(q[v + 2 * threads], v + 2 * threads, 2);
  const int tail = head + vecs * W;
  for (int i = tail + t; i < n; i += threads) f(lo + i, ld_p<T>(row, lo + i), 3);
}
template <class T, class F>
__device__ __forceinline__ void for_words(const char* row, int lo, int n, int t, int threads,
                                          F&& f) {
  for_groups<T>(row, lo, n, t, threads, [&](int i, float v, int) { f(i, v); });
}

// The first index i of [from, from + n) with f(from) + .. + f(i) > target(total), total the
// sum of all; from + n if there is none. *total_out is that total. All threads of the block
// call it.
template <class T, class Sh, class F, class G>
__device__ __forceinline__ int locate(Sh& sh, const char* row, int from, int n,
                                      F&& f, G&& target_of, u64* total_out) {
  constexpr int NTH = Sh::NTH, WAVES = Sh::kWaves;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int lo = from, len = n;
  u64 base = 0, target = 0;
  bool first = true;
  for (;;) {
    const int seg = (len + NTH - 1) / NTH * 64;   // a wave's share
    const int b = min(len, wave * seg), e = min(len, b + seg);
    u64 s = 0;
    for_words<T>(row, lo + b, e - b, lane, 64, [&](int i, float v) { s += f(i, v); });
    s = wave_total(s);
    __syncthreads();
    if (lane == 0) sh.wave[wave] = s;
    __syncthreads();
    u64 run = base;
    if (first) {
      u64 total = 0;
      for (int w = 0; w < WAVES; ++w) total += sh.wave[w];
      *total_out = total;
      target = target_of(total);
      first = false;
    }
    int w = 0;
    while (w < WAVES && run + sh.wave[w] <= target) run += sh.wave[w++];
    if (w == WAVES) return from + n;
    base = run;
    lo += w * seg;
    len = min(seg, len - w * seg);
    if (len <= 64) break;
  }
  // every wave alike
  const u64 mine = lane < len ? f(lo + lane, ld_p<T>(row, lo + lane)) : 0;
  const u64 run = base + wave_scan(mine);
  const u64 hit = __ballot(lane < len && run > target);
  return hit ? lo + __ffsll((long long)hit) - 1 : from + n;
}

// Of the entries order[e] (below 2^bits, those with w[e] > 0), from the largest on,
// the first at which the sum of w reaches `want` (1 .. their total). All threads of the block
// call it; one barrier a digit of six bits, whose sums lie in one of three buffers: the one in
// use, the next one's being cleared, the last one's still being read. (A bitonic sort
// of 1024 entries took 28 us through LDS, 41 with its strides below 64 in registers; this
// about 0.3 us a digit.)
template <class Sh, int E>
__device__ __forceinline__ u64 select(Sh& sh, const u64 (&order)[E], const u64 (&w)[E], int bits,
                                      u64 want) {
  const int tid = threadIdx.x, lane = tid & 63;
  u64 prefix = 0, above = 0;
  __syncthreads();
  if (tid < 64) sh.digits[0][tid] = 0;
  __syncthreads();
  int at = 0;
  for (int shift = bits; shift > 0;) {
    const int up = shift;
    shift = max(0, shift - 6);
    u64* now = sh.digits[at];
    at = at == 2 ? 0 : at + 1;
    if (tid < 64) sh.digits[at][tid] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (w[e] && order[e] >> up == prefix)
        atomicAdd(&now[(order[e] >> shift) & ((1u << (up - shift)) - 1)], w[e]);
    __syncthreads();
    const u64 v = now[63 - lane], run = above + wave_scan(v);
    const u64 hit = __ballot(run >= want);
    const int l = hit ? __ffsll((long long)hit) - 1 : 63;
    above = lane_u64(run - v, l);
    prefix = prefix << (up - shift) | (63 - l);
  }
  return prefix;
}
__device__ __forceinline__ int bits_of(u64 v) { return v ? 64 - __clzll((long long)v) : 0; }

// The places of the words that take(v) names go to list (of `most` entries, in LDS or not);
// *count, 0 before, is how many there are.
template <class T, class F>
__device__ __forceinline__ void collect(u64* list, int most, unsigned* count, const char* row,
                                        int lo, int n, int t, int threads, F&& take) {
  for_words<T>(row, lo, n, t, threads, [&](int i, float v) {
    if (!take(v)) return;
    const unsigned at = atomicAdd(count, 1u);
    if (at < (unsigned)most) list[at] = place_of(key_of<T>(as_logit(v)), i);
  });
}
// The same of a whole row by its block, to the list in LDS (or another).
template <class T, class Sh, class F>
__device__ __forceinline__ int collect_row(Sh& sh, const char* row, int n, F&& take,
                                           u64* list = nullptr, int most = 0) {
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  collect<T>(list ? list : sh.list, list ? most : Sh::kList, &sh.count, row, 0, n, threadIdx.x,
             Sh::NTH, take);
  __syncthreads();
  return (int)sh.count;
}

// 2^y for y <= 0 (0 below -64): e^(f ln 2) for the fraction |f| <= 1/2 by its series to the
// 12th power (what is left out is below 2^-52), scaled by the integer part.
__device__ __forceinline__ double exp2_64(double y) {
  if (!(y > -64.0)) return 0.0;
  const double n = rint(y), f = y - n;
  double p = 2.5678435993488196e-11;   // ln2^k / k!, k = 12 .. 0
  p = fma(p, f, 4.44553827187081e-10);
  p = fma(p, f, 7.054911620801121e-09);
  p = fma(p, f, 1.0178086009239696e-07);
  p = fma(p, f, 1.3215486790144305e-06);
  p = fma(p, f, 1.5252733804059838e-05);
  p = fma(p, f, 0.00015403530393381606);
  p = fma(p, f, 0.0013333558146428441);
  p = fma(p, f, 0.009618129107628477);
  p = fma(p, f, 0.055504108664821576);
  p = fma(p, f, 0.2402265069591007);
  p = fma(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}

// A row: its words, settings and largest logit, and what follows from them.
template <class T>
struct RowOf {
  const SampleArgs& a;
  int r, V;
  const char* row;
  float temp, top_p, min_p, uniform, m, low_v;
  long long k;
  bool peak;   // the largest logits alone (temperature 0, or a row that has +inf)
  double md, rate, low, one;
  __device__ __forceinline__ RowOf(const SampleArgs& args, int row_)
      : a(args), r(row_), V(args.vocab),
        row(static_cast<const char*>(args.logits) + (size_t)row_ * args.ld * kElem<T>) {
    temp = a.temperature ? a.temperature[r] : a.temperature_v;
    top_p = a.top_p ? a.top_p[r] : a.top_p_v;
    min_p = a.min_p ? a.min_p[r] : a.min_p_v;
    uniform = a.uniform[r];
    k = !a.top_k ? a.top_k_v
        : a.k64 ? static_cast<const long long*>(a.top_k)[r]
                : (long long)static_cast<const int*>(a.top_k)[r];
    one = (double)(1ULL << a.scale);
  }
  __device__ __forceinline__ void set_max(float m_) {
    m = m_;
    peak = temp == 0.f || m == INFINITY;
    md = m;
    rate = 1.4426950408889634 / (double)temp;
    low = min_p;
    // (a logit that min-p leaves out by more than the rounding of this is not looked at)
    low_v = min_p > 0.f && !peak
                ? (float)(md + temp * log(low) - 1e-6 * (fabs(md) + temp * 100.0))
                : -INFINITY;
  }
  __device__ __forceinline__ bool valid() const {
    return temp >= 0.f && temp < INFINITY && min_p <= 1.f && top_p == top_p && m > -INFINITY;
  }
  __device__ __forceinline__ double power(float v) const {   // log2 of the weight
    return v == m ? 0.0 : peak ? -INFINITY : ((double)v - md) * rate;
  }
  __device__ __forceinline__ u64 fixed(double w) const {   // w 2^scale, below 2^52, rounded
    return (u64)__double_as_longlong(w * one + 4503599627370496.0) & 0xFFFFFFFFFFFFFULL;
  }
  __device__ __forceinline__ u64 weight(float v) const { return fixed(exp2_64(power(v))); }
  // with min-p
  __device__ __forceinline__ u64 counted(float v) const {
    if (!(v >= low_v)) return 0;
    const double w = exp2_64(power(v));
    return w >= low ? fixed(w) : 0;
  }
  // kept by the place `least` (0: all) and min-p
  __device__ __forceinline__ u64 counted_from(u64 least, float from, int i, float v) const {
    if (least && (!(v >= from) || place_of(key_of<T>(as_logit(v)), i) < least)) return 0;
    return counted(v);
  }
  // whether a logit may have its weight's logarithm in the bin (a test in fp32, a little wide)
  __device__ __forceinline__ void bin_range(int bin, float* lo, float* hi) const {
    const double slack = 1e-6 * (fabs(md) + temp * 100.0);
    *hi = (float)(md - bin * 0.0625 / rate + slack);
    *lo = (float)(md - (bin + 1) * 0.0625 / rate - slack);
  }
  // the bin of a weight's logarithm above -64
  static __device__ __forceinline__ int bin_of(double y) {
    return min(kMassBins - 1, (int)(y * -16.0));
  }
  __device__ __forceinline__ u64 target_of(u64 all) const {
    const double t = (double)uniform * (double)all;
    // x > t <=> x > floor(t); below 0 and NaN: the first; at or past the total: the last
    return !(t > 0.0) ? 0 : t >= (double)all ? all - 1 : (u64)t;
  }
  // weights before a word that are below top_p of `all`: below this integer
  __device__ __forceinline__ u64 border_of(u64 all) const {
    const double t = (double)top_p * (double)all;
    return t > 0.0 ? (u64)ceil(t) : 0;
  }
  __device__ __forceinline__ void answer(int token, float v, u64 total) const {
    a.tokens[r] = token;
    if (a.logprobs)
      a.logprobs[r] = (float)(power(v) * 0.6931471805599453 - log((double)total / one));
  }
};

// The list's entries in the threads' registers: their places (0: none) and weights.
template <class T, class Sh>
struct ListOf {
  static constexpr int E = Sh::E;
  Sh& sh;
  const RowOf<T>& R;
  u64 place[E], w[E];
  int ib;           // bits of an index
  unsigned base;    // the smallest key
  int bits;         // of an order
  __device__ __forceinline__ ListOf(Sh& shared, const RowOf<T>& row, int n, float from)
      : sh(shared), R(row), ib(max(1, bits_of((u64)row.V - 1))), base(key_of<T>(from)) {
    bits = bits_of(key_of<T>(R.m) - base) + ib;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = e * Sh::NTH + threadIdx.x;
      place[e] = i < n ? sh.list[i] : 0;
    }
  }
  static __device__ __forceinline__ float value(u64 p) { return value_of<T>((unsigned)(p >> 32)); }
  // by key, then index, within `bits`
  __device__ __forceinline__ u64 order(u64 p) const {
    return (u64)((unsigned)(p >> 32) - base) << ib | ((1u << ib) - 1 - (unsigned)index_at(p));
  }
  __device__ __forceinline__ u64 place_at(u64 o) const {
    return place_of((unsigned)(o >> ib) + base, (int)((1u << ib) - 1 - ((unsigned)o & ((1u << ib) - 1))));
  }
  // The place of the k-th entry.
  __device__ __forceinline__ u64 kth(int k) {
    u64 o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] = place[e] ? order(place[e]) : 0;
      w[e] = place[e] != 0;
    }
    return place_at(select(sh, o, w, bits, (u64)k));
  }
  // The place of the last entry, of those from `least` on, that has less than top_p of
  // `all` (0: of their own weight) before it, `above` being the weight before them.
  __device__ __forceinline__ u64 cut(u64 least, u64 above, u64 all) {
    u64 o[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] = place[e] ? order(place[e]) : 0;
      w[e] = place[e] && place[e] >= least ? R.weight(value(place[e])) : 0;
      sum += w[e];
    }
    if (all == 0) all = block_total(sh, sum);
    return place_at(select(sh, o, w, bits, max((u64)1, R.border_of(all)) - above));
  }
  // The draw from the entries from `least` on, with min-p: they are all that is kept.
  __device__ __forceinline__ void draw(u64 least) {
    u64 o[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] = (1u << ib) - 1 - (unsigned)index_at(place[e] ? place[e] : ~0ULL);
      w[e] = place[e] && place[e] >= least ? R.counted(value(place[e])) : 0;
      sum += w[e];
    }
    const u64 total = block_total(sh, sum);
    const u64 at = select(sh, o, w, ib, R.target_of(total) + 1);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (w[e] && o[e] == at) R.answer(index_at(place[e]), value(place[e]), total);
  }
};

// From the weights by bin: the bin in which the border `want` falls, the weight before it.
template <class T, class Sh, class F>
__device__ __forceinline__ int border_bin(Sh& sh, const RowOf<T>& R, F&& bin_at, u64 before_all,
                                          u64* above, u64* all, u64 want) {
  constexpr int PER = kMassBins / Sh::NTH;
  const int tid = threadIdx.x;
  u64 w[PER], sum = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    w[e] = bin_at(tid * PER + e);
    sum += w[e];
  }
  if (tid == 0) {
    sh.bin = 0;      // (border 0: only the first word, in the first bin)
    sh.above = 0;
  }
  u64 run = before_all + block_before(sh, sum, all);
  if (want == ~0ULL) want = R.border_of(*all);
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (w[e] && run < want && run + w[e] >= want) {
      sh.bin = tid * PER + e;
      sh.above = run;
    }
    run += w[e];
  }
  __syncthreads();
  *above = sh.above;
  const int b = (int)sh.bin;
  __syncthreads();
  return b;
}

// The weights of the words with bin(y) >= 0, y a weight's logarithm, added to the bins in LDS.
template <class T, class Sh, class F>
__device__ __forceinline__ void fill_bins(Sh& sh, const RowOf<T>& R, int lo, int n, F&& bin) {
  __syncthreads();
  for (int i = threadIdx.x; i < kMassBins; i += Sh::NTH) sh.bins[i] = 0;
  __syncthreads();
  for_words<T>(R.row, lo, n, threadIdx.x, Sh::NTH, [&](int, float v) {
    const double y = R.power(v);
    const int b = y > -64.0 ? bin(y) : -1;
    if (b < 0) return;
    const u64 w = R.fixed(exp2_64(y));
    if (w) atomicAdd(&sh.bins[b], w);
  });
  __syncthreads();
}

// The first kernel. PARTS: rows may be left.
template <class T, class Sh, bool PARTS>
__global__ void __launch_bounds__(Sh::NTH)
sample_kernel(SampleArgs a) {
  constexpr int NTH = Sh::NTH;
  __shared__ Sh sh;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  RowOf<T> R(a, blockIdx.x);
  const int V = a.vocab;
  const char* row = R.row;
  // ---- the largest logit
  float mine[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  for_groups<T>(row, 0, V, tid, NTH,
                [&](int, float v, int group) { mine[group] = fmaxf(mine[group], v); });
#pragma unroll
  for (int g = 0; g < 4; ++g) mine[g] = as_logit(mine[g]);
  float m = fmaxf(fmaxf(mine[0], mine[1]), fmaxf(mine[2], mine[3]));
  const float thread_max = m;
#pragma unroll
  for (int s = 32; s; s /= 2) m = fmaxf(m, __shfl_xor(m, s));
  if (lane == 0) sh.wave_f[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < Sh::kWaves; ++w) m = fmaxf(m, sh.wave_f[w]);
  R.set_max(m);
  SampleRow* const st = PARTS ? a.state + R.r : nullptr;
  if (PARTS && tid == 0) {
    st->m = m;
    st->left = kRowDone;
    st->count = 0;
  }
  if (!R.valid()) {
    if (tid == 0) {
      a.tokens[R.r] = -1;
      if (a.logprobs) a.logprobs[R.r] = __builtin_nanf("");
    }
    return;
  }
  if (R.temp == 0.f) {
    u64 total;
    const int token = locate<T>(sh, row, 0, V, [&](int, float v) { return (u64)(v == m); },
                                [&](u64) -> u64 { return 0; }, &total);
    if (tid == 0) R.answer(token, m, (u64)R.one);
    return;
  }
  const int k = R.k > 0 && R.k < V ? (int)R.k : 0;
  float from = -INFINITY;
  if constexpr (PARTS) {
    if (k > 2 * NTH || (k == 0 && (R.top_p < 1.f || !(R.low_v > -INFINITY)))) {
      if (tid == 0) st->left = k ? kRowSearch : kRowAll;
      for (int i = tid; i < kMassBins; i += NTH) st->total[i] = 0;
      return;
    }
    if (k) {
      // The k-th largest of the threads' own maxima, to 18 bits, rounded down; from
      // k 129 on of four a thread (1024 maxima of which 1000 are wanted would let in a tenth of
      // 131072 words, 4096 let in 1150).
      constexpr int kBits = 32 - kLowBits<T>, kDrop = kBits > 18 ? kBits - 18 : 0;
      unsigned at;
      if (k <= NTH / 8) {
        const u64 x[1] = {key_of<T>(thread_max) >> kDrop}, one[1] = {1};
        at = (unsigned)select(sh, x, one, kBits - kDrop, (u64)k);
      } else {
        u64 x[4];
        const u64 one[4] = {1, 1, 1, 1};
#pragma unroll
        for (int g = 0; g < 4; ++g) x[g] = key_of<T>(mine[g]) >> kDrop;
        at = (unsigned)select(sh, x, one, kBits - kDrop, (u64)k);
      }
      if (at > key_of<T>(-INFINITY) >> kDrop) from = value_of<T>(at << kDrop);
    } else {
      from = R.low_v;
    }
  }
  // (!PARTS: all words; NaN too, as -inf)
  const int n = collect_row<T>(sh, row, V, [&](float v) { return !PARTS || v >= from; });
  if (PARTS && (n > Sh::kList || n < k)) {
    // too many for this list: to the row's (the search where that is too short, or NaNs count)
    if (n >= k && n <= kRowList) {
      collect_row<T>(sh, row, V, [&](float v) { return v >= from; }, st->list, kRowList);
      if (tid == 0) {
        st->count = n;
        st->left = kRowCut;
      }
    } else {
      for (int i = tid; i < kMassBins; i += NTH) st->total[i] = 0;
      if (tid == 0) st->left = k ? kRowSearch : kRowAll;
    }
    return;
  }
  ListOf<T, Sh> list(sh, R, n, from);
  u64 least = 0;
  if (k) least = list.kth(k);
  if (R.top_p < 1.f) least = list.cut(least, 0, 0);
  list.draw(least);
}

// Part blockIdx.x of row blockIdx.y: its weights by bin, to the part's and to the row's.
template <class T>
__global__ void __launch_bounds__(256)
sample_bins_kernel(SampleArgs a) {
  __shared__ SampleShared<256, 1024> sh;
  SampleRow& st = a.state[blockIdx.y];
  if (st.left != kRowAll) return;
  RowOf<T> R(a, blockIdx.y);
  R.set_max(st.m);
  if (R.peak) return;
  const int lo = blockIdx.x * kPart;
  fill_bins(sh, R, lo, min(kPart, R.V - lo), [&](double y) { return R.bin_of(y); });
  u64* out = a.bins + ((size_t)blockIdx.y * a.parts + blockIdx.x) * kMassBins;
  for (int i = threadIdx.x; i < kMassBins; i += 256) {
    const u64 w = sh.bins[i];
    out[i] = w;
    if (w) atomicAdd(&st.total[i], w);
  }
}

// The words of the border's bin, of a part, to the row's list.
template <class T>
__global__ void __launch_bounds__(256)
sample_border_kernel(SampleArgs a) {
  __shared__ SampleShared<256, 1024> sh;
  SampleRow& st = a.state[blockIdx.y];
  if (st.left != kRowAll) return;
  RowOf<T> R(a, blockIdx.y);
  R.set_max(st.m);
  if (R.peak || !(R.top_p < 1.f)) return;
  u64 above, all;
  const int bin = border_bin(sh, R, [&](int i) { return st.total[i]; }, 0, &above, &all, ~0ULL);
  const int lo = blockIdx.x * kPart;
  float least, most;
  R.bin_range(bin, &least, &most);
  collect<T>(st.list, kRowList, &st.count, R.row, lo, min(kPart, R.V - lo), threadIdx.x, 256,
             [&](float v) {
               if (!(v >= least && v <= most)) return false;
               const double y = R.power(v);
               return y > -64.0 && R.bin_of(y) == bin;
             });
}

// The last kept place by a search over the bits of the keys: of the words, a reading a bit.
template <class T, class Sh>
__device__ __forceinline__ u64 search_border(Sh& sh, const RowOf<T>& R) {
  const int tid = threadIdx.x, V = R.V;
  const u64 k = R.k > 0 && R.k < V ? (u64)R.k : 0;
  // what the words of at least a key come to: their number, or their weight (of those above
  // kkey, and `ties` of it)
  unsigned kkey = 0;
  u64 ties = ~0ULL;
  const auto sum_from = [&](unsigned key, bool by_count) {
    u64 s = 0;
    for_words<T>(R.row, 0, V, tid, Sh::NTH, [&](int, float v) {
      v = as_logit(v);
      const unsigned own = key_of<T>(v);
      if (own < key || own < kkey) return;
      if (by_count) ++s;
      else if (own > kkey || ties == ~0ULL) s += R.weight(v);
    });
    s = block_total(sh, s);
    if (!by_count && ties != ~0ULL && key <= kkey) s += ties * R.weight(value_of<T>(kkey));
    return s;
  };
  // the largest key that has words worth `want` from it on
  const auto search = [&](u64 want, bool by_count) {
    unsigned key = 0;
    for (int bit = 31 - kLowBits<T>; bit >= 0; --bit)
      if (sum_from(key | 1u << bit, by_count) >= want) key |= 1u << bit;
    return key;
  };
  const auto own_of = [&](unsigned key) {   // words of the key
    u64 s = 0;
    for_words<T>(R.row, 0, V, tid, Sh::NTH,
                 [&](int, float v) { s += key_of<T>(as_logit(v)) == key; });
    return block_total(sh, s);
  };
  unsigned edge = 0;
  u64 keep = ~0ULL, own = 0;   // words of the edge's key that are kept
  if (k) {
    edge = search(k, true);
    own = own_of(edge);
    keep = k - (edge == 0xFFFFFFFFu >> kLowBits<T> ? 0 : sum_from(edge + 1, true));
    kkey = edge;
    ties = keep;
  }
  if (R.top_p < 1.f) {
    const u64 want = R.border_of(sum_from(0, false));
    if (want == 0) {
      edge = key_of<T>(R.m);
      keep = 1;
      own = ~0ULL;
    } else {
      const unsigned pkey = search(want, false);
      // the words of pkey in turn: the i-th has above + i w before it
      const u64 w = R.weight(value_of<T>(pkey)), above = sum_from(pkey + 1, false);
      u64 most = ties;
      if (!k || pkey != kkey) most = own = own_of(pkey);
      const u64 n = w ? (want - above + w - 1) / w : most;
      keep = n < most ? n : most;
      edge = pkey;
    }
  }
  if (keep >= own) return (u64)edge << 32;
  u64 total;
  __syncthreads();
  const int last = locate<T>(
      sh, R.row, 0, V, [&](int, float v) { return (u64)(key_of<T>(as_logit(v)) == edge); },
      [&](u64) { return keep - 1; }, &total);
  return place_of(edge, last);
}

// The rows left.
template <class T>
__global__ void __launch_bounds__(1024)
sample_finish_kernel(SampleArgs a) {
  constexpr int NTH = 1024;
  typedef SampleShared<NTH, kRowList> Sh;
  __shared__ Sh sh;
  __shared__ u64 part_sum[256];
  SampleRow& st = a.state[blockIdx.x];
  if (st.left == kRowDone) return;
  RowOf<T> R(a, blockIdx.x);
  R.set_max(st.m);
  const int tid = threadIdx.x, V = R.V, left = st.left;
  const int k = R.k > 0 && R.k < V ? (int)R.k : 0;
  u64 least = 0, total;
  int bin = kMassBins;   // the bins before it are kept whole
  int n = 0;             // words of it
  const bool binned = left == kRowAll && a.parts > 1 && !R.peak;   // (by the kernels before)
  bool search = left == kRowSearch || (R.peak && R.top_p < 1.f), by_parts = binned && a.parts <= 256;
  if (left == kRowCut) {
    n = (int)st.count;
    for (int i = tid; i < n; i += NTH) sh.list[i] = st.list[i];
    ListOf<T, Sh> list(sh, R, n, -INFINITY);
    if (k) least = list.kth(k);
    if (R.top_p < 1.f) least = list.cut(least, 0, 0);
    list.draw(least);
    return;
  }
  if (!search && R.top_p < 1.f) {
    u64 above, all;
    if (binned) {
      bin = border_bin(sh, R, [&](int i) { return st.total[i]; }, 0, &above, &all, ~0ULL);
      n = (int)st.count;
      for (int i = tid; i < min(n, kRowList); i += NTH) sh.list[i] = st.list[i];
    } else {
      fill_bins(sh, R, 0, V, [&](double y) { return R.bin_of(y); });
      bin = border_bin(sh, R, [&](int i) { return sh.bins[i]; }, 0, &above, &all, ~0ULL);
      n = collect_row<T>(sh, R.row, V, [&](float v) {
        const double y = R.power(v);
        return y > -64.0 && R.bin_of(y) == bin;
      });
    }
    if (n > kRowList) {
      // a bin of many words (a flat distribution): 1024 bins of it
      by_parts = false;
      const auto sub = [&](double y) {
        return R.bin_of(y) == bin ? max(0, min(kMassBins - 1, (int)((y * -16.0 - bin) * kMassBins)))
                                  : -1;
      };
      fill_bins(sh, R, 0, V, sub);
      u64 none;
      const int at = border_bin(sh, R, [&](int i) { return sh.bins[i]; }, above, &above, &none,
                                max((u64)1, R.border_of(all)));
      n = collect_row<T>(sh, R.row, V, [&](float v) {
        const double y = R.power(v);
        return y > -64.0 && sub(y) == at;
      });
    }
    search = n > kRowList;
    if (!search) {
      ListOf<T, Sh> list(sh, R, n, -INFINITY);
      least = list.cut(0, above, all);
      __syncthreads();
    }
  }
  if (search) {
    by_parts = false;
    least = search_border(sh, R);
    __syncthreads();
  }
  const float from = value_of<T>((unsigned)(least >> 32));
  const auto kept = [&](int i, float v) { return R.counted_from(least, from, i, v); };
  if (R.min_p > 0.f) {
    // (min-p may leave fewer)
    const float lo = least ? fmaxf(from, R.low_v) : R.low_v;
    n = collect_row<T>(sh, R.row, V, [&](float v) { return v >= lo; });
    if (n <= kRowList) {
      ListOf<T, Sh>(sh, R, n, lo).draw(least);
      return;
    }
    by_parts = false;
  }
  int lo = 0, words = V;
  u64 before = 0, want = 0;
  if (by_parts) {
    // the parts' kept weights: their bins before the border's, and its words that are kept
    for (int p = tid; p < 256; p += NTH) part_sum[p] = 0;
    __syncthreads();
    const u64* bins = a.bins + (size_t)R.r * a.parts * kMassBins;
    for (int p = tid >> 6; p < a.parts; p += NTH / 64) {
      u64 s = 0;
      for (int b = tid & 63; b < bin; b += 64) s += bins[(size_t)p * kMassBins + b];
      s = wave_total(s);
      if ((tid & 63) == 0) atomicAdd(&part_sum[p], s);
    }
    for (int i = tid; i < n; i += NTH) {
      const u64 x = sh.list[i];
      if (x >= least)
        atomicAdd(&part_sum[index_at(x) / kPart], R.weight(value_of<T>((unsigned)(x >> 32))));
    }
    __syncthreads();
    total = 0;
    for (int p = 0; p < a.parts; ++p) total += part_sum[p];
    want = R.target_of(total);
    int p = 0;
    while (p < a.parts - 1 && before + part_sum[p] <= want) before += part_sum[p++];
    lo = p * kPart;
    words = min(kPart, V - lo);
    __syncthreads();
  }
  u64 own;
  const int token = locate<T>(sh, R.row, lo, words, kept, [&](u64 all) {
    if (by_parts) return want - before;
    total = all;
    return R.target_of(all);
  }, &own);
  if (tid == 0) R.answer(token, logit_at<T>(R.row, token), total);
}

}  // namespace mhs
