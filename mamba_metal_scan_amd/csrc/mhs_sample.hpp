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
// The first kernel has a block per row. It reads the words for the maximum, each thread
// keeping those of its vectors (or, of a large vocabulary, of 16 groups of them). The k-th
// largest of the threads' maxima bounds the k-th largest logit from below (min-p bounds
// the kept words in the same way), and the few vectors that reach it are read again, their
// words from there on collected in LDS. A list of up to 256 words is put in order by counting,
// for each word, those before it by place and by index, and one wave then goes through its
// running sums. What is asked of a longer list (the k-th word, the one at top-p's border,
// by index the one that is drawn) is each the first, in an order, at which a running sum
// reaches a number: a descent over the order's bits, six at a time, with the digits' sums
// in LDS.
// Rows whose settings keep more words (top-p alone, or no setting) are left to two further
// kernels: the weights by bins of their logarithm (1/16 of a factor of 2), by part of 8192
// words and by row, a block per part; and, a block per row, the words of the bin in which
// top-p's border falls, their cut, the part in which the draw falls (from the bins), and the
// word.
// What no list holds is found by a search over the bits of the logits' keys, a reading each and, with
// top-p, as many again: very many words of one weight; k above 2048 of many words; and k above
// the number of the threads' maxima, which in a short row is that of its vectors (k 1000 of
// 4097 to 7999 words in 16 bits, k 2000 of up to about 8000 in fp32). (us, without and with top-p
// 0.9, 256 rows: of 131072 words at k 5000 in fp32 699 and 1944, in bf16 327 and 975; of 6000 in
// bf16 at k 1000 54 and 107, of 9000 by the list 25 and 29.)
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kMassBins = 1024;   // of 2^-1/16, down to 2^-64
constexpr int kPart = 8192;       // words of a part
constexpr int kSlots = 16;        // maxima that a thread keeps
constexpr int kFlight = 8;        // loads in flight

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
  unsigned long long* bins;  // (rows, parts, kMassBins); of a row that has no top-p a part's sum
  int parts;
};
struct SampleRow {
  float m;
  int left;                  // whether the row is left to the further kernels
  unsigned long long total[kMassBins];
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

// kList: words of a block's list; kShort: of one put in order by counting (the square of
// that many comparisons, shared by the threads, 64 each).
template <int NTH_>
struct ListShared {
  static constexpr int NTH = NTH_, kWaves = NTH / 64, kList = 4 * NTH,
                       kShort = NTH == 1024 ? 256 : 128;
  u64 list[kList];
  u64 sorted[kShort], by_index[kShort];   // weights by place; places by index
  unsigned order[kShort], ranks[kShort];  // by index the place's number; both of the list's
  u64 digits[3][64];
  u64 wave[kWaves];
  float wave_f[2][kWaves];
  unsigned count;
};
// Of the last kernel.
struct RowShared : ListShared<1024> {
  u64 bins[kMassBins];
  u64 part[256];
  u64 above;
  unsigned bin;
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

// f(i, word i) for the words of vector r, whose first is word b.
template <class T, class F>
__device__ __forceinline__ void vector_words(const uint4& r, int b, F&& f) {
  constexpr int E = kElem<T>, W = 16 / E;
  const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int e = 0; e < W; ++e) {
    float x;
    if constexpr (E == 4) x = __uint_as_float(u[e]);
    else x = T::to((unsigned short)(u[e / 2] >> (16 * (e & 1))));
    f(b + e, x);
  }
}

// f(i, word i) for the words lo .. lo + n - 1, each once, by `threads` threads (this one is
// number t): 16 bytes at a time but for the ends, four such loads in flight.
template <class T, class F>
__device__ __forceinline__ void for_words(const char* row, int lo, int n, int t, int threads,
                                          F&& f) {
  constexpr int E = kElem<T>, W = 16 / E;
  const char* p = row + (size_t)lo * E;
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / E);
  for (int i = t; i < head; i += threads) f(lo + i, ld_p<T>(row, lo + i));
  const int vecs = (n - head) / W, b = lo + head;
  const uint4* q = reinterpret_cast<const uint4*>(p + (size_t)head * E);
  int v = t;
  for (; v + 3 * threads < vecs; v += 4 * threads) {
    const uint4 r0 = q[v], r1 = q[v + threads], r2 = q[v + 2 * threads], r3 = q[v + 3 * threads];
    vector_words<T>(r0, b + v * W, f);
    vector_words<T>(r1, b + (v + threads) * W, f);
    vector_words<T>(r2, b + (v + 2 * threads) * W, f);
    vector_words<T>(r3, b + (v + 3 * threads) * W, f);
  }
  for (; v < vecs; v += threads) vector_words<T>(q[v], b + v * W, f);
  const int tail = head + vecs * W;
  for (int i = tail + t; i < n; i += threads) f(lo + i, ld_p<T>(row, lo + i));
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

// Of the n entries order[e] (below 2^bits, those with w[e] > 0), from the largest on,
// the first at which the sum of w reaches `want` (1 .. their total). All threads of the block
// call it; one barrier a digit of six bits, whose sums lie in one of three buffers: the one in
// use, the next one's being cleared, the last one's still being read. (A bitonic sort
// of 1024 entries took 28 us through LDS, 41 with its strides below 64 in registers; this
// about 0.3 us a digit.)
template <class Sh, int E>
__device__ __forceinline__ u64 select(Sh& sh, const u64 (&order)[E], const u64 (&w)[E], int n,
                                      int bits, u64 want, u64* found = nullptr) {
  const int tid = threadIdx.x, lane = tid & 63;
  u64 prefix = 0, above = 0, reached = 0;
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
      if (e * Sh::NTH < n && w[e] && order[e] >> up == prefix)
        atomicAdd(&now[(order[e] >> shift) & ((1u << (up - shift)) - 1)], w[e]);
    __syncthreads();
    const u64 v = now[63 - lane], run = above + wave_scan(v);
    const u64 hit = __ballot(run >= want);
    const int l = hit ? __ffsll((long long)hit) - 1 : 63;
    reached = lane_u64(run, l);
    above = lane_u64(run - v, l);
    prefix = prefix << (up - shift) | (63 - l);
  }
  if (found) *found = reached;
  return prefix;
}
__device__ __forceinline__ int bits_of(u64 v) { return v ? 64 - __clzll((long long)v) : 0; }

// A row as its `head` words before the first whole vector, `vecs` vectors and `tail` words.
template <class T>
struct Vectors {
  static constexpr int E = kElem<T>, W = 16 / E;
  const char* row;
  const uint4* q;
  int V, head, vecs, tail;
  __device__ __forceinline__ Vectors(const char* row_, int V_) : row(row_), V(V_) {
    head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / E);
    vecs = (V - head) / W;
    tail = V - head - vecs * W;
    q = reinterpret_cast<const uint4*>(row + (size_t)head * E);
  }
  template <class F>
  __device__ __forceinline__ void in_head(F&& f) const {
    if ((int)threadIdx.x < head) f((int)threadIdx.x, ld_p<T>(row, threadIdx.x));
  }
  template <class F>
  __device__ __forceinline__ void in_tail(F&& f) const {
    const int i = V - tail + threadIdx.x;
    if (i < V) f(i, ld_p<T>(row, i));
  }
};

// A row's words, a thread's largest ones kept: those of vectors t, t + kSlots, .. of the thread
// in slot t (of NaN and where there is none -inf).
template <class T, int NTH>
struct SlotMaxima : Vectors<T> {
  using Vectors<T>::q;
  using Vectors<T>::vecs;
  using Vectors<T>::head;
  static constexpr int W = Vectors<T>::W;
  float slot[kSlots], most;   // most: of the words before and behind the vectors too
  __device__ __forceinline__ SlotMaxima(const char* row, int V) : Vectors<T>(row, V) {
    const GBuf g(reinterpret_cast<const float*>(q), 16u * (unsigned)vecs);
#pragma unroll
    for (int t = 0; t < kSlots; ++t) slot[t] = -INFINITY;
    for (int v0 = 0; v0 < vecs; v0 += kSlots * NTH) {
#pragma unroll
      for (int h = 0; h < kSlots; h += kFlight) {
        if (v0 + h * NTH >= vecs) break;
        uint4 r[kFlight];
#pragma unroll
        for (int t = 0; t < kFlight; ++t) {
          const auto l = __builtin_amdgcn_raw_buffer_load_b128(
              g.r, 16u * (unsigned)(v0 + (h + t) * NTH + (int)threadIdx.x), 0, 0);
          r[t] = uint4{l[0], l[1], l[2], l[3]};
        }
#pragma unroll
        for (int t = 0; t < kFlight; ++t) {
          float w = -INFINITY;
          vector_words<T>(r[t], 0, [&](int, float v) { w = fmaxf(w, v); });
          if (v0 + (h + t) * NTH + (int)threadIdx.x >= vecs) w = -INFINITY;
          slot[h + t] = fmaxf(slot[h + t], w);
        }
      }
    }
    most = -INFINITY;
    const auto end = [&](int, float v) { most = fmaxf(most, v); };
    this->in_head(end);
    this->in_tail(end);
    most += 0.f;   // (-0 as 0: its key is the words' in the list)
#pragma unroll
    for (int t = 0; t < kSlots; ++t) {
      slot[t] += 0.f;
      most = fmaxf(most, slot[t]);
    }
  }
  // the largest of every fourth slot, from g on
  __device__ __forceinline__ float group(int g) const {
    return fmaxf(fmaxf(slot[g], slot[g + 4]), fmaxf(slot[g + 8], slot[g + 12]));
  }
  // f(vector, its first word) of the vectors in whose slot a word is >= from
  template <class F>
  __device__ __forceinline__ void vectors_from(float from, F&& f) const {
    unsigned mask = 0;
#pragma unroll
    for (int t = 0; t < kSlots; ++t) mask |= slot[t] >= from ? 1u << t : 0u;
    const auto next = [&] {   // (a thread's few loads: the next under way before one is used)
      const int t = __ffs((int)mask) - 1;
      mask &= mask - 1;
      return t * NTH + (int)threadIdx.x;
    };
    if (!mask) return;
    int v = next();
    uint4 r = q[v];   // (a slot that has such a word has a vector)
    for (;;) {
      const int own = v;
      const uint4 mine = r;
      v += kSlots * NTH;
      const bool more = v < vecs || mask;
      if (v >= vecs && mask) v = next();
      if (more) r = q[v];
      f(mine, head + own * W);
      if (!more) break;
    }
  }
  // The first word that is m, the largest, of the thread's; V if there is none.
  __device__ __forceinline__ int first(float m) const {
    int at = this->V;
    const auto look = [&](int i, float v) { at = v == m ? min(at, i) : at; };
    vectors_from(m, [&](const uint4& r, int b) { vector_words<T>(r, b, look); });
    this->in_head(look);
    this->in_tail(look);
    return at;
  }
  // The places of the words >= from (a finite number) to the list in LDS; how many there are.
  template <class Sh>
  __device__ __forceinline__ int collect(Sh& sh, float from) const {
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    const auto put = [&](unsigned at, int i, float v) {
      if (at < (unsigned)Sh::kList) sh.list[at] = place_of(key_of<T>(v + 0.f), i);
    };
    vectors_from(from, [&](const uint4& r, int b) {
      int n = 0;
      vector_words<T>(r, b, [&](int, float v) { n += v >= from; });
      unsigned at = n ? atomicAdd(&sh.count, (unsigned)n) : 0;
      vector_words<T>(r, b, [&](int i, float v) {
        if (v >= from) put(at++, i, v);
      });
    });
    const auto end = [&](int i, float v) {
      if (v >= from) put(atomicAdd(&sh.count, 1u), i, v);
    };
    this->in_head(end);
    this->in_tail(end);
    __syncthreads();
    return (int)sh.count;
  }
};

// The places of the row's words v in [lo, hi] that take(v) names, to the list in LDS; how many
// there are. Of 16 vectors a thread notes which words are in the range, then looks at those
// few again. (us of 465 words among 131072, looked at as they come: 16; this way 6.)
template <class T, class Sh, class F>
__device__ __forceinline__ int collect(Sh& sh, const char* row, int n, float lo, float hi,
                                       F&& take) {
  constexpr int W = Vectors<T>::W, NTH = Sh::NTH;
  const Vectors<T> words(row, n);
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  const auto word = [&](int i, float v) {
    if (!(v >= lo && v <= hi && take(v))) return;
    const unsigned at = atomicAdd(&sh.count, 1u);
    if (at < (unsigned)Sh::kList) sh.list[at] = place_of(key_of<T>(as_logit(v)), i);
  };
  const GBuf g(reinterpret_cast<const float*>(words.q), 16u * (unsigned)words.vecs);
  for (int v0 = 0; v0 < words.vecs; v0 += 16 * NTH) {
    unsigned in[4] = {0, 0, 0, 0};   // a byte for a vector
#pragma unroll
    for (int h = 0; h < 16; h += kFlight) {
      if (v0 + h * NTH >= words.vecs) break;
      uint4 r[kFlight];
#pragma unroll
      for (int t = 0; t < kFlight; ++t) {
        const auto l = __builtin_amdgcn_raw_buffer_load_b128(
            g.r, 16u * (unsigned)(v0 + (h + t) * NTH + (int)threadIdx.x), 0, 0);
        r[t] = uint4{l[0], l[1], l[2], l[3]};
      }
#pragma unroll
      for (int t = 0; t < kFlight; ++t) {
        unsigned bits = 0;
        vector_words<T>(r[t], 0, [&](int e, float v) {
          bits |= v >= lo && v <= hi ? 1u << e : 0u;
        });
        if (v0 + (h + t) * NTH + (int)threadIdx.x >= words.vecs) bits = 0;
        in[(h + t) / 4] |= bits << (h + t) % 4 * 8;
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      while (in[w]) {
        const int b = __ffs((int)in[w]) - 1, v = v0 + (4 * w + b / 8) * NTH + (int)threadIdx.x;
        in[w] &= in[w] - 1;
        const int i = words.head + v * W + b % 8;
        word(i, ld_p<T>(row, i));
      }
    }
  }
  words.in_head(word);
  words.in_tail(word);
  __syncthreads();
  return (int)sh.count;
}

// 2^y for y <= 0 (0 below -64): e^(f ln 2) for the fraction |f| <= 1/2 by its series to the
// 12th power (what is left out is below 2^-52), scaled by the integer part, which an addition
// of 1.5 2^52 rounds to and leaves in the sum's low bits.
__device__ __forceinline__ double exp2_64(double y) {
  if (!(y > -64.0)) return 0.0;
  const double t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);
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
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
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
    if (peak) return v == m ? 0.0 : -INFINITY;
    return ((double)v - md) * rate;
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
  static constexpr int E = Sh::kList / Sh::NTH;
  Sh& sh;
  const RowOf<T>& R;
  u64 place[E], w[E];
  int n;
  int ib;           // bits of an index
  unsigned base;    // the smallest key
  int bits;         // of an order
  __device__ __forceinline__ ListOf(Sh& shared, const RowOf<T>& row, int count, float from)
      : sh(shared), R(row), n(count), ib(max(1, bits_of((u64)row.V - 1))), base(key_of<T>(from)) {
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
    const unsigned low = (1u << ib) - 1;
    return place_of((unsigned)(o >> ib) + base, (int)(low - ((unsigned)o & low)));
  }
  // The place of the k-th entry.
  __device__ __forceinline__ u64 kth(int k) {
    u64 o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] = place[e] ? order(place[e]) : 0;
      w[e] = place[e] != 0;
    }
    return place_at(select(sh, o, w, n, bits, (u64)k));
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
    return place_at(select(sh, o, w, n, bits, max((u64)1, R.border_of(all)) - above));
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
    const u64 at = select(sh, o, w, n, ib, R.target_of(total) + 1);
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

// The weights of a part's words with bin(y) >= 0, y a weight's logarithm, added to the bins:
// `copies` of them in LDS, a lane's own by its number, whose adds to one bin wait for
// each other.
template <class T, int NTH, int COPIES, class F>
__device__ __forceinline__ void fill_bins(u64* bins, const RowOf<T>& R, int lo, int n, F&& bin) {
  __syncthreads();
  for (int i = threadIdx.x; i < COPIES * kMassBins; i += NTH) bins[i] = 0;
  __syncthreads();
  u64* const own = bins + threadIdx.x % COPIES * kMassBins;
  for_words<T>(R.row, lo, n, threadIdx.x, NTH, [&](int, float v) {
    const double y = R.power(v);
    const int b = y > -64.0 ? bin(y) : -1;
    if (b < 0) return;
    const u64 w = R.fixed(exp2_64(y));
    if (w) atomicAdd(&own[b], w);
  });
  __syncthreads();
}

// A list of up to kShort words in order: sh.sorted, by_index, order. Every word is compared with
// every other, a share of them by each thread. This thread's word (of tid < n) and its number.
template <class T, class Sh>
__device__ __forceinline__ u64 short_order(Sh& sh, const RowOf<T>& R, int n, unsigned* number) {
  const int tid = threadIdx.x;
  if (tid < Sh::kShort) sh.ranks[tid] = 0;
  __syncthreads();
  int bits = 6;
  while (1 << bits < n) ++bits;
  const int e = tid & ((1 << bits) - 1), share = (1 << 2 * bits) / Sh::NTH;
  const int j0 = (tid >> bits) * share, j1 = min(n, j0 + share);
  const u64 p = e < n ? sh.list[e] : 0;
  unsigned before = 0;   // by place and, in the upper half, by index
  for (int j = j0; j < j1; ++j) {
    const u64 o = sh.list[j];
    before += (o > p) + ((unsigned)o > (unsigned)p ? 1u << 16 : 0u);
  }
  if (e < n && before) atomicAdd(&sh.ranks[e], before);
  const u64 own = tid < n ? R.weight(value_of<T>((unsigned)(p >> 32))) : 0;
  __syncthreads();
  *number = ~0u;
  if (tid < n) {
    const unsigned r = sh.ranks[tid];
    *number = r & 0xFFFF;
    sh.sorted[r & 0xFFFF] = own;
    sh.by_index[r >> 16] = p;
    sh.order[r >> 16] = r & 0xFFFF;
  }
  __syncthreads();
  return p;
}
// Of the first `kept` words in order, how many top-p keeps, `above` being the weight before
// them and `all` (0: their own) the total. By one wave, four words a lane.
template <class T, class Sh>
__device__ __forceinline__ int short_kept(Sh& sh, const RowOf<T>& R, int kept, u64 above, u64 all) {
  const int lane = threadIdx.x & 63;
  u64 w[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * lane + i;
    w[i] = at < kept ? sh.sorted[at] : 0;
    sum += w[i];
  }
  u64 run = wave_scan(sum);
  const u64 border = R.border_of(all ? all : lane_u64(run, 63));
  run += above - sum;
  int count = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * lane + i;
    count += __popcll(__ballot(at < kept && (at == 0 || run < border)));
    run += w[i];
  }
  return count;
}
// The place of the last word that top-p keeps of a list of up to kShort words.
template <class T, class Sh>
__device__ __forceinline__ u64 short_cut(Sh& sh, const RowOf<T>& R, int n, u64 above, u64 all) {
  unsigned number;
  const u64 p = short_order(sh, R, n, &number);
  const int kept = short_kept(sh, R, n, above, all);   // (every wave alike)
  if ((int)number == kept - 1) sh.wave[0] = p;
  __syncthreads();
  return sh.wave[0];
}
// The draw from a list of up to kShort words, with k (0: all), top-p and min-p.
template <class T, class Sh>
__device__ __forceinline__ void short_draw(Sh& sh, const RowOf<T>& R, int n, int k) {
  const int lane = threadIdx.x & 63;
  const auto value = [](u64 p) { return value_of<T>((unsigned)(p >> 32)); };
  unsigned number;
  short_order(sh, R, n, &number);
  if (threadIdx.x >= 64) return;
  int kept = k && k < n ? k : n;
  if (R.top_p < 1.f) kept = short_kept(sh, R, kept, 0, 0);
  // four words by index
  u64 w[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * lane + i;
    const unsigned r = at < n ? sh.order[at] : ~0u;
    w[i] = r >= (unsigned)kept ? 0
           : R.min_p > 0.f ? R.counted(value(sh.by_index[at])) : sh.sorted[r];
    sum += w[i];
  }
  u64 run = wave_scan(sum);
  const u64 total = lane_u64(run, 63), target = R.target_of(total);
  run -= sum;
  int hit = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    run += w[i];
    if (hit < 0 && run > target) hit = 4 * lane + i;
  }
  const u64 hits = __ballot(hit >= 0);
  if (hits && lane == __ffsll((long long)hits) - 1) {
    const u64 at = sh.by_index[hit];
    R.answer(index_at(at), value(at), total);
  }
}

// The same as locate of up to kPart words, each thread having 8 neighbouring ones: its
// answer goes out at once.
template <class T, class Sh, class F>
__device__ __forceinline__ void locate_part(Sh& sh, const RowOf<T>& R, int from, int n, F&& f,
                                            u64 before, u64 target, u64 total) {
  constexpr int PER = kPart / Sh::NTH;
  float v[PER];
  u64 w[PER], sum = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = PER * threadIdx.x + e;
    v[e] = i < n ? logit_at<T>(R.row, from + i) : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    w[e] = f(from + PER * (int)threadIdx.x + e, v[e]);
    sum += w[e];
  }
  u64 all;
  u64 run = before + block_before(sh, sum, &all);
  if (!(run <= target && run + sum > target)) return;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (run <= target && run + w[e] > target)
      R.answer(from + PER * (int)threadIdx.x + e, v[e], total);
    run += w[e];
  }
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

// The first kernel: rows of up to kList words, and those whose kept words fit the list. us: 4 x
// 32768 in fp32, top-k 50 and top-p 0.9, 11, of which the maxima 1.8, the bound 2.6, the list
// 1.8, its draw 2.1, the rest the launch and the settings; 256 x 131072 in bf16 the same 18 (the
// maxima 9 to 12: the words at 6 to 7 TB/s), and with k up to 1000 in some rows 39 (their
// bound 6, list 10, descents 13). Loads: eight in flight; all 16 with the words kept in
// registers for the second pass took 14 us for the maxima, and spilled.
template <class T, int NTH>
__global__ void __launch_bounds__(NTH)
sample_kernel(SampleArgs a) {
  typedef ListShared<NTH> Sh;
  __shared__ Sh sh;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  RowOf<T> R(a, blockIdx.x);
  const int V = a.vocab;
  const SlotMaxima<T, NTH> words(R.row, V);
  float m = words.most;
  // (the least of the threads' finite maxima)
  float least_most = words.most > -INFINITY ? words.most : INFINITY;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (words.group(g) > -INFINITY) least_most = fminf(least_most, words.group(g));
#pragma unroll
  for (int s = 32; s; s /= 2) {
    m = fmaxf(m, __shfl_xor(m, s));
    least_most = fminf(least_most, __shfl_xor(least_most, s));
  }
  if (lane == 0) {
    sh.wave_f[0][wave] = m;
    sh.wave_f[1][wave] = least_most;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < Sh::kWaves; ++w) {
    m = fmaxf(m, sh.wave_f[0][w]);
    least_most = fminf(least_most, sh.wave_f[1][w]);
  }
  R.set_max(m);
  SampleRow* const st = V > Sh::kList ? a.state + R.r : nullptr;
  if (st && tid == 0) {
    st->m = m;
    st->left = 0;
  }
  if (!R.valid()) {
    if (tid == 0) {
      a.tokens[R.r] = -1;
      if (a.logprobs) a.logprobs[R.r] = __builtin_nanf("");
    }
    return;
  }
  if (R.temp == 0.f) {
    int first = words.most == m ? words.first(m) : V;
#pragma unroll
    for (int s = 32; s; s /= 2) first = min(first, __shfl_xor(first, s));
    if (lane == 0) sh.wave[wave] = (u64)first;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Sh::kWaves; ++w) first = min(first, (int)sh.wave[w]);
    if (tid == 0) R.answer(first, m, (u64)R.one);
    return;
  }
  // ---- a list of all words that can be kept. (Words of -inf, and NaN, weigh nothing.)
  int k = R.k > 0 && R.k < V ? (int)R.k : 0;
  const bool nucleus = R.top_p < 1.f;
  bool few = V <= Sh::kList;
  float from = -__FLT_MAX__;
  if (k && k <= 2 * NTH) {
    // The k-th largest of the threads' own maxima, in 4096 steps between the least and the
    // largest of them, rounded down; from k 129 on of four a thread (1024 maxima of which 1000
    // are wanted would let in a tenth of 131072 words, 4096 let in 1150).
    const unsigned base = key_of<T>(least_most), range = key_of<T>(m) - base;
    const int drop = max(0, bits_of(range) - 12), bits = max(1, bits_of(range) - drop);
    const auto step = [&](float v) -> u64 { return (key_of<T>(v) - base) >> drop; };
    const auto counts = [](float v) -> u64 { return v > -INFINITY; };
    u64 steps, found;
    if (k <= NTH / 8) {
      const u64 x[1] = {step(words.most)}, one[1] = {counts(words.most)};
      steps = select(sh, x, one, NTH, bits, (u64)k, &found);
    } else {
      u64 x[4], one[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        x[g] = step(words.group(g));
        one[g] = counts(words.group(g));
      }
      steps = select(sh, x, one, 4 * NTH, bits, (u64)k, &found);
    }
    if (found >= (u64)k) from = value_of<T>(base + ((unsigned)steps << drop));
    few = true;
  } else if (!k && !nucleus && R.low_v > -INFINITY) {
    from = fmaxf(from, R.low_v);
    few = true;
  }
  const int n = few ? words.collect(sh, from) : 0;
  if (!few || n > Sh::kList) {
    if (tid == 0) st->left = 1;
    for (int i = tid; i < kMassBins; i += NTH) st->total[i] = 0;
    return;
  }
  if (n <= k) k = 0;
  if (n <= Sh::kShort) {
    short_draw(sh, R, n, k);
    return;
  }
  ListOf<T, Sh> list(sh, R, n, from);
  u64 least = 0;
  if (k) least = list.kth(k);
  if (nucleus) least = list.cut(least, 0, 0);
  list.draw(least);
}

// Bound by the weights' arithmetic, some 50 instructions a word, most in 64 bits, and by the
// adds to LDS: 256 x 131072 words 58 us, a third of those rows 18 us.
// Of the rows left those that neither k nor +inf with top-p leaves to the search: part blockIdx.x
// of row blockIdx.y, its weights by bin, to the part's and to the row's; without top-p their sum.
template <class T>
__global__ void __launch_bounds__(256)
sample_bins_kernel(SampleArgs a) {
  constexpr int kCopies = 4;
  __shared__ u64 bins[kCopies][kMassBins];
  SampleRow& st = a.state[blockIdx.y];
  if (!st.left) return;
  RowOf<T> R(a, blockIdx.y);
  if (R.k > 0 && R.k < R.V) return;
  R.set_max(st.m);
  const int lo = blockIdx.x * kPart, n = min(kPart, R.V - lo);
  u64* out = a.bins + ((size_t)blockIdx.y * a.parts + blockIdx.x) * kMassBins;
  if (!(R.top_p < 1.f)) {
    u64 s = 0;
    for_words<T>(R.row, lo, n, threadIdx.x, 256, [&](int, float v) { s += R.counted(v); });
    s = wave_total(s);
    if ((threadIdx.x & 63) == 0) bins[0][threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) out[0] = (bins[0][0] + bins[0][1]) + (bins[0][2] + bins[0][3]);
    return;
  }
  if (R.peak) return;
  fill_bins<T, 256, kCopies>(bins[0], R, lo, n, [&](double y) { return R.bin_of(y); });
  for (int i = threadIdx.x; i < kMassBins; i += 256) {
    u64 w = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) w += bins[c][i];
    out[i] = w;
    if (w) atomicAdd(&st.total[i], w);
  }
}

// The rows left. Bound by its steps' latencies (us, 4 x 131072 words: the border's bin 2.3, its
// words 8 to 9, their cut 2.3 or, of more than 256 words, 5.8, the parts' sums 3.3, the word 6.5).
template <class T>
__global__ void __launch_bounds__(1024)
sample_rest_kernel(SampleArgs a) {
  typedef RowShared Sh;
  constexpr int NTH = Sh::NTH;
  __shared__ Sh sh;
  const SampleRow& st = a.state[blockIdx.x];
  if (!st.left) return;
  const int tid = threadIdx.x;
  RowOf<T> R(a, blockIdx.x);
  R.set_max(st.m);
  const int V = R.V;
  const bool nucleus = R.top_p < 1.f, k = R.k > 0 && R.k < V;
  // ---- the place of the last word that k and top-p keep
  u64 least = 0;
  bool search = k || (R.peak && nucleus);
  bool by_parts = a.parts > 1 && a.parts <= 256 && !search;
  int bin = 0, n = 0;   // the bins before it are kept whole; words of it
  if (nucleus && !search) {
    u64 above, all;
    if (a.parts > 1) {
      bin = border_bin(sh, R, [&](int i) { return st.total[i]; }, 0, &above, &all, ~0ULL);
    } else {
      fill_bins<T, NTH, 1>(sh.bins, R, 0, V, [&](double y) { return R.bin_of(y); });
      bin = border_bin(sh, R, [&](int i) { return sh.bins[i]; }, 0, &above, &all, ~0ULL);
    }
    // (where min-p's border is in a bin before it, that is the border; too near to a bin's end to
    // tell, the words are gone through)
    bool cut = true;
    if (R.min_p > 0.f) {
      const double y = log2(R.low);
      if (R.bin_of(y + 1e-9) != R.bin_of(y - 1e-9)) {
        by_parts = false;
      } else if (R.bin_of(y) < bin) {
        bin = R.bin_of(y);
        cut = false;
      }
    }
    float lo, hi;
    R.bin_range(bin, &lo, &hi);
    n = collect<T>(sh, R.row, V, lo, hi, [&](float v) {
      const double y = R.power(v);
      return y > -64.0 && R.bin_of(y) == bin;
    });
    if (n > Sh::kList && cut) {
      // a bin of many words (a flat distribution): 1024 bins of it
      by_parts = false;
      const auto sub = [&](double y) {
        return R.bin_of(y) == bin ? max(0, min(kMassBins - 1, (int)((y * -16.0 - bin) * kMassBins)))
                                  : -1;
      };
      fill_bins<T, NTH, 1>(sh.bins, R, 0, V, sub);
      u64 none;
      const int at = border_bin(sh, R, [&](int i) { return sh.bins[i]; }, above, &above, &none,
                                max((u64)1, R.border_of(all)));
      n = collect<T>(sh, R.row, V, lo, hi, [&](float v) {
        const double y = R.power(v);
        return y > -64.0 && sub(y) == at;
      });
    }
    if (!cut) {
      by_parts = by_parts && n <= Sh::kList;
    } else if (n > Sh::kList) {
      search = true;
    } else if (n <= Sh::kShort) {
      least = short_cut(sh, R, n, above, all);
    } else {
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
  const float low = value_of<T>((unsigned)(least >> 32));
  const auto kept = [&](int i, float v) { return R.counted_from(least, low, i, v); };
  // ---- the draw, from the part in which it falls
  u64 total = 0;
  if (by_parts) {
    // the parts' kept weights: their bins before the border's, and its words that are kept
    const u64* bins = a.bins + (size_t)R.r * a.parts * kMassBins;
    for (int p = tid >> 6; p < a.parts; p += Sh::kWaves) {
      u64 s = 0;
      if (nucleus) {
#pragma unroll 4
        for (int b = tid & 63; b < bin; b += 64) s += bins[(size_t)p * kMassBins + b];
        s = wave_total(s);
      } else {
        s = bins[(size_t)p * kMassBins];
      }
      if ((tid & 63) == 0) sh.part[p] = s;
    }
    __syncthreads();
    if (nucleus) {
      for (int i = tid; i < n; i += NTH) {
        const u64 x = sh.list[i];
        if (x >= least)
          atomicAdd(&sh.part[index_at(x) / kPart], R.counted(value_of<T>((unsigned)(x >> 32))));
      }
      __syncthreads();
    }
    for (int p = 0; p < a.parts; ++p) total += sh.part[p];
    const u64 want = R.target_of(total);
    u64 before = 0;
    int p = 0;
    while (p < a.parts - 1 && before + sh.part[p] <= want) before += sh.part[p++];
    locate_part(sh, R, p * kPart, min(kPart, V - p * kPart), kept, before, want, total);
    return;
  }
  const int token = locate<T>(sh, R.row, 0, V, kept, [&](u64 all) { return R.target_of(all); },
                              &total);
  if (tid == 0) R.answer(token, logit_at<T>(R.row, token), total);
}

}  // namespace mhs
