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
// A block has a row. Its words are read as often as the settings need:
//   - once for the maximum, each thread's own being kept;
//   - top-k (up to a word per thread): the k-th largest of the threads' maxima bounds
//     the k-th largest logit from below, so that a second reading collects the few words
//     from there on in LDS, where they are sorted, cut, put in the order of
//     their indices and drawn from. min-p bounds the kept words in the same way;
//   - top-p of all words: the weights by bins of their logarithm (1/16 of a factor
//     of 2), the words of the bin in which the border falls, sorted, and a
//     reading that sums the kept weights by wave, the wave in which the draw falls being
//     divided further.
// Lists that are too long (many equal words) and large k take a radix descent over the
// logits' keys instead, a reading per 11 bits.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kDigitBits = 11;
constexpr int kBins = 1 << kDigitBits;
constexpr int kMassBins = 1024;   // of 2^-1/16, down to 2^-64

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

template <int NTH>
struct SampleShared {
  static constexpr int kWaves = NTH / 64, kList = 4 * NTH;
  union {
    struct {
      u64 mass[kBins];
      unsigned count[kBins];
    } radix;
    u64 bins[kMassBins];
    u64 list[kList];
  };
  u64 wave[kWaves];
  float wave_f[kWaves];
  u64 above;
  unsigned bin, count;
};

// Inclusive sum of v over the lanes up to this one.
__device__ __forceinline__ u64 wave_scan(u64 v, int lane) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) {
    const u64 o = __shfl_up(v, s);
    if (lane >= s) v += o;
  }
  return v;
}
__device__ __forceinline__ u64 wave_total(u64 v) {
#pragma unroll
  for (int s = 32; s; s /= 2) v += __shfl_xor(v, s);
  return v;
}
// The block's sum of v, in every thread.
template <int NTH>
__device__ __forceinline__ u64 block_total(SampleShared<NTH>& sh, u64 v) {
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int w = 0; w < SampleShared<NTH>::kWaves; ++w) s += sh.wave[w];
  __syncthreads();
  return s;
}
// The sum of v over the threads before this one.
template <int NTH>
__device__ __forceinline__ u64 block_before(SampleShared<NTH>& sh, u64 v, u64* total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const u64 run = wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) sh.wave[wave] = run;
  __syncthreads();
  u64 before = run - v, all = 0;
#pragma unroll
  for (int w = 0; w < SampleShared<NTH>::kWaves; ++w) {
    if (w < wave) before += sh.wave[w];
    all += sh.wave[w];
  }
  __syncthreads();
  *total = all;
  return before;
}

// f(i, word i) for the words lo .. lo + n - 1, each once, by `threads` threads (this one
// is number t): 16 bytes at a time but for the ends, four such loads in flight.
template <class T, class F>
__device__ __forceinline__ void for_words(const char* row, int lo, int n, int t, int threads,
                                          F&& f) {
  constexpr int E = kElem<T>, W = 16 / E;
  const char* p = row + (size_t)lo * E;
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / E);
  for (int i = t; i < head; i += threads) f(lo + i, ld_p<T>(row, lo + i));
  const int vecs = (n - head) / W;
  const uint4* q = reinterpret_cast<const uint4*>(p + (size_t)head * E);
  const int b = lo + head;
  const auto word = [&](const uint4& r, int v) {
    const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < W; ++e) {
      float x;
      if constexpr (E == 4) x = __uint_as_float(u[e]);
      else x = T::to((unsigned short)(u[e / 2] >> (16 * (e & 1))));
      f(b + v * W + e, x);
    }
  };
  int v = t;
  for (; v + 3 * threads < vecs; v += 4 * threads) {
    const uint4 r0 = q[v], r1 = q[v + threads], r2 = q[v + 2 * threads], r3 = q[v + 3 * threads];
    word(r0, v);
    word(r1, v + threads);
    word(r2, v + 2 * threads);
    word(r3, v + 3 * threads);
  }
  for (; v < vecs; v += threads) word(q[v], v);
  const int tail = head + vecs * W;
  for (int i = tail + t; i < n; i += threads) f(lo + i, ld_p<T>(row, lo + i));
}

// The first index i of [0, n) with f(0) + .. + f(i) > target(total), total the sum
// of all; n if there is none. *total_out is that total. All threads of the block call it.
template <class T, int NTH, class F, class G>
__device__ __forceinline__ int locate(SampleShared<NTH>& sh, const char* row, int n, F&& f, G&& target_of,
                      u64* total_out) {
  constexpr int WAVES = NTH / 64;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int lo = 0, len = n;
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
    if (w == WAVES) return n;
    base = run;
    lo += w * seg;
    len = min(seg, len - w * seg);
    if (len <= 64) break;
  }
  // every wave alike
  const u64 mine = lane < len ? f(lo + lane, ld_p<T>(row, lo + lane)) : 0;
  const u64 run = base + wave_scan(mine, lane);
  const u64 hit = __ballot(lane < len && run > target);
  return hit ? lo + __ffsll((long long)hit) - 1 : n;
}

// list[0 .. n) sorted, largest first; the next power of two of them are touched (n at
// most kList). A bitonic network; strides up to 64 stay within a wave's 128 entries.
template <int NTH>
__device__ __forceinline__ void sort_list(SampleShared<NTH>& sh, int n) {
  int n2 = 2;
  while (n2 < n) n2 *= 2;
  for (int i = n + threadIdx.x; i < n2; i += NTH) sh.list[i] = 0;
  __syncthreads();
  for (int size = 2; size <= n2; size *= 2) {
    for (int stride = size / 2; stride; stride /= 2) {
      for (int t = threadIdx.x; t < n2 / 2; t += NTH) {
        const int i = 2 * t - (t & (stride - 1)), j = i + stride;
        const u64 x = sh.list[i], y = sh.list[j];
        if ((x < y) == ((i & size) == 0)) {
          sh.list[i] = y;
          sh.list[j] = x;
        }
      }
      if (stride > 64 || (stride == 1 && size >= 128)) __syncthreads();
      else wave_lds_sync();
    }
  }
  __syncthreads();
}

// The words with take(i, v), their places in the list; returns how many there are
// (more than kList: the list is not whole).
template <class T, int NTH, class F>
__device__ __forceinline__ int collect(SampleShared<NTH>& sh, const char* row, int n, F&& take) {
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  for_words<T>(row, 0, n, threadIdx.x, NTH, [&](int i, float v) {
    if (!take(v)) return;
    const unsigned at = atomicAdd(&sh.count, 1u);
    if (at < SampleShared<NTH>::kList) sh.list[at] = place_of(key_of<T>(as_logit(v)), i);
  });
  __syncthreads();
  return (int)sh.count;
}

// Radix descent to a key. Each level counts, per digit, the words whose higher digits
// are those found and that take(key, v, &weight) names, and goes on in a digit: with
// BY_COUNT the first from the top at which the words reach `want`, else the lowest that has
// words and less than `want` weight above it. Returns the key; *above is the count (weight)
// of the keys above it, *own its own words.
template <class T, int NTH, bool BY_COUNT, class F>
__device__ __forceinline__ unsigned descend(SampleShared<NTH>& sh, const char* row, int n, F&& take, u64 want,
                            u64* above_out, unsigned* own) {
  constexpr int PER = kBins / NTH;   // bins of a thread, from the top
  const int tid = threadIdx.x;
  unsigned prefix = 0;
  u64 above = 0;
  int shift = 32 - kLowBits<T>;
  while (shift > 0) {
    const int bits = min(kDigitBits, shift);
    const bool top = shift == 32 - kLowBits<T>;
    const int up = shift;
    shift -= bits;
    __syncthreads();
    for (int i = tid; i < kBins; i += NTH) {
      sh.radix.mass[i] = 0;
      sh.radix.count[i] = 0;
    }
    __syncthreads();
    for_words<T>(row, 0, n, tid, NTH, [&](int, float v) {
      v = as_logit(v);
      const unsigned key = key_of<T>(v);
      u64 m = 0;
      if (!(top || key >> up == prefix) || !take(key, v, &m)) return;
      const unsigned bin = (key >> shift) & ((1u << bits) - 1);
      atomicAdd(&sh.radix.count[bin], 1u);
      if (!BY_COUNT && m) atomicAdd(&sh.radix.mass[bin], m);
    });
    __syncthreads();
    u64 own_sum = 0;
    const int b0 = kBins - 1 - PER * tid;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      own_sum += BY_COUNT ? sh.radix.count[b0 - i] : sh.radix.mass[b0 - i];
    if (tid == 0) sh.bin = 0;
    u64 all;
    u64 before = above + block_before(sh, own_sum, &all);
    // (of the bins that qualify the lowest: bins are numbered from the top, plus one)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const u64 v = BY_COUNT ? sh.radix.count[b0 - i] : sh.radix.mass[b0 - i];
      if (BY_COUNT ? before < want && before + v >= want
                   : sh.radix.count[b0 - i] && before < want)
        atomicMax(&sh.bin, (unsigned)(PER * tid + i + 1));
      before += v;
    }
    __syncthreads();
    const int from_top = (int)sh.bin - 1;
    before -= own_sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (PER * tid + i == from_top) sh.above = before;
      before += BY_COUNT ? sh.radix.count[b0 - i] : sh.radix.mass[b0 - i];
    }
    __syncthreads();
    if (from_top < 0) break;   // (nothing to find: not reached by the calls below)
    const unsigned bin = kBins - 1 - from_top;
    above = sh.above;
    *own = sh.radix.count[bin];
    prefix = (prefix << bits) | bin;
  }
  __syncthreads();
  *above_out = above;
  return prefix;
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

template <class T, int NTH>
__global__ void __launch_bounds__(NTH)
sample_kernel(SampleArgs a) {
  typedef SampleShared<NTH> Sh;
  __shared__ Sh sh;
  const int r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int V = a.vocab;
  const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.ld * kElem<T>;
  const float temp = a.temperature ? a.temperature[r] : a.temperature_v;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p_v;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p_v;
  const float uf = a.uniform[r];
  const long long kk = !a.top_k ? a.top_k_v
                       : a.k64 ? static_cast<const long long*>(a.top_k)[r]
                               : (long long)static_cast<const int*>(a.top_k)[r];
  // ---- the largest logit
  float mine = -INFINITY;
  for_words<T>(row, 0, V, tid, NTH, [&](int, float v) { mine = fmaxf(mine, v); });
  mine = as_logit(mine);
  float m = mine;
#pragma unroll
  for (int s = 32; s; s /= 2) m = fmaxf(m, __shfl_xor(m, s));
  if (lane == 0) sh.wave_f[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < Sh::kWaves; ++w) m = fmaxf(m, sh.wave_f[w]);
  if (!(temp >= 0.f && temp < INFINITY && min_p <= 1.f && top_p == top_p) || m == -INFINITY) {
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = __builtin_nanf("");
    }
    return;
  }
  // (temperature 0, or a row that has +inf: the largest logits alone)
  const bool peak = temp == 0.f || m == INFINITY;
  const double md = m, rate = 1.4426950408889634 / (double)temp, low = min_p;
  const auto power = [&](float v) {   // log2 of the weight
    return v == m ? 0.0 : peak ? -INFINITY : ((double)v - md) * rate;
  };
  const double one = (double)(1ULL << a.scale);
  const auto fixed = [&](double w) {   // w 2^scale, an integer below 2^52, rounded
    return (u64)__double_as_longlong(w * one + 4503599627370496.0) & 0xFFFFFFFFFFFFFULL;
  };
  // (a logit that min-p leaves out by more than the rounding of this is not looked at)
  const float low_v = min_p > 0.f && !peak
                          ? (float)(md + temp * log(low) - 1e-6 * (fabs(md) + temp * 100.0))
                          : -INFINITY;
  const auto counted = [&](float v) -> u64 {
    if (!(v >= low_v)) return 0;
    const double w = exp2_64(power(v));
    return w >= low ? fixed(w) : 0;
  };
  const auto target_of = [&](u64 all) -> u64 {
    const double t = (double)uf * (double)all;
    // x > t <=> x > floor(t); below 0 and NaN: the first; at or past the total: the last
    return !(t > 0.0) ? 0 : t >= (double)all ? all - 1 : (u64)t;
  };
  // weights before a word that are below top_p of `all`: below this integer
  const auto border_of = [&](u64 all) -> u64 {
    const double t = (double)top_p * (double)all;
    return t > 0.0 ? (u64)ceil(t) : 0;
  };
  const auto answer = [&](int token, float v, u64 total) {
    a.tokens[r] = token;
    if (a.logprobs)
      a.logprobs[r] = (float)(power(v) * 0.6931471805599453 - log((double)total / one));
  };
  const bool has_k = kk > 0 && kk < V;
  const bool has_p = top_p < 1.f;
  u64 least = 0;   // the place of the last kept word (before min-p)
  u64 total;

  // ---- the draw from list[0 .. n), which holds every word that is kept by the place
  // `least` and min-p (and may hold others)
  const auto draw_list = [&](int n) {
    constexpr int PER = Sh::kList / NTH;
    // by index: a word's index in the high half, its key in the low
    for (int i = tid; i < n; i += NTH) {
      const u64 x = sh.list[i];
      sh.list[i] = x >= least ? x << 32 | x >> 32 : 0;
    }
    sort_list(sh, n);
    u64 w[PER], sum = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = tid * PER + e;
      const u64 x = i < n ? sh.list[i] : 0;
      w[e] = x ? counted(value_of<T>((unsigned)x)) : 0;
      sum += w[e];
    }
    u64 run = block_before(sh, sum, &total);
    const u64 target = target_of(total);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (run <= target && run + w[e] > target) {
        const u64 x = sh.list[tid * PER + e];
        answer((int)(0xFFFFFFFFu - (unsigned)(x >> 32)), value_of<T>((unsigned)x), total);
      }
      run += w[e];
    }
  };
  // The place in the sorted list[0 .. n), of which the first `most` may be kept, of the last
  // word that has less than top_p of `all` (0: of their own total) before it, `above` being
  // the weight before the list.
  const auto cut_list = [&](int n, int most, u64 above, u64 all) -> u64 {
    constexpr int PER = Sh::kList / NTH;
    u64 w[PER], sum = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = tid * PER + e;
      w[e] = i < most ? fixed(exp2_64(power(value_of<T>((unsigned)(sh.list[i] >> 32))))) : 0;
      sum += w[e];
    }
    u64 own;
    u64 run = above + block_before(sh, sum, &own);
    const u64 want = border_of(all ? all : own);
    int keep = 0;   // this thread's words that are kept
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (tid * PER + e < most && run < want) ++keep;
      run += w[e];
    }
    const int kept = max(1, (int)block_total(sh, (u64)keep));
    return sh.list[kept - 1];
  };

  if (temp == 0.f) {
    const int token = locate<T>(sh, row, V, [&](int, float v) { return (u64)(v == m); },
                                [&](u64) -> u64 { return 0; }, &total);
    if (tid == 0) answer(token, m, (u64)one);
    return;
  }
  if (has_k && kk <= NTH) {
    // the k-th largest of the threads' own maxima
    sh.list[tid] = (u64)key_of<T>(mine) + 1;
    sort_list(sh, NTH);
    const float from = value_of<T>((unsigned)(sh.list[kk - 1] - 1));
    const int n = collect<T>(sh, row, V, [&](float v) { return v >= from; });
    if (n <= Sh::kList && n >= kk) {
      sort_list(sh, n);
      least = sh.list[kk - 1];
      if (has_p) least = cut_list(n, (int)kk, 0, 0);
      __syncthreads();
      draw_list((int)kk);
      return;
    }
  }
  u64 all = 0;   // the weight of all words, where they are looked at for top-p
  if (!has_k && has_p && !peak) {
    // weights by bins of their logarithm
    __syncthreads();
    for (int i = tid; i < kMassBins; i += NTH) sh.bins[i] = 0;
    __syncthreads();
    for_words<T>(row, 0, V, tid, NTH, [&](int, float v) {
      const double y = power(v);
      const u64 w = fixed(exp2_64(y));
      if (w) atomicAdd(&sh.bins[min(kMassBins - 1, (int)(y * -16.0))], w);
    });
    __syncthreads();
    constexpr int PER = kMassBins / NTH;
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum += sh.bins[tid * PER + e];
    u64 run = block_before(sh, sum, &all);
    const u64 want = border_of(all);
    if (tid == 0) sh.bin = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const u64 w = sh.bins[tid * PER + e];
      if (w && run < want && run + w >= want) {
        sh.bin = tid * PER + e;
        sh.above = run;
      } else if (want == 0 && tid == 0 && e == 0) {
        sh.above = 0;   // (only the first word: in the first bin)
      }
      run += w;
    }
    __syncthreads();
    const int bin = (int)sh.bin;
    const u64 above = sh.above;
    const int n = collect<T>(sh, row, V, [&](float v) {
      const double y = power(v);
      return y > -64.0 && min(kMassBins - 1, (int)(y * -16.0)) == bin;
    });
    if (n <= Sh::kList) {
      sort_list(sh, n);
      least = cut_list(n, n, above, all);
    } else {
      all = 0;   // (the descent below)
    }
  }
  if (has_k || (has_p && all == 0)) {
    // ---- top-k: the key of the k-th word, and how many of that key are kept
    unsigned kkey = 0;
    u64 ties = ~0ULL;    // of kkey, by index
    bool cut = false;    // whether some word of kkey is left out
    unsigned own = 0;
    u64 above;
    if (has_k) {
      kkey = descend<T, NTH, true>(sh, row, V, [&](unsigned, float, u64*) { return true; },
                                   (u64)kk, &above, &own);
      ties = (u64)kk - above;
      cut = ties < own;
    }
    // ---- top-p among those
    if (has_p) {
      u64 s = 0;   // the total: words above kkey, and `ties` of it
      for_words<T>(row, 0, V, tid, NTH, [&](int, float v) {
        v = as_logit(v);
        const unsigned key = key_of<T>(v);
        if (key > kkey || (key == kkey && !cut)) s += fixed(exp2_64(power(v)));
      });
      u64 sum = block_total(sh, s);
      if (cut) sum += ties * fixed(exp2_64(power(value_of<T>(kkey))));
      const u64 want = border_of(sum);
      if (want == 0) {
        kkey = key_of<T>(m);
        ties = 1;
        cut = true;
      } else {
        const unsigned pkey = descend<T, NTH, false>(
            sh, row, V, [&](unsigned key, float v, u64* w) {
              if (key < kkey) return false;
              *w = fixed(exp2_64(power(v)));
              return true;
            }, want, &above, &own);
        // the words of pkey in turn: the i-th has above + i w before it
        const u64 w = fixed(exp2_64(power(value_of<T>(pkey))));
        u64 most = pkey == kkey && cut ? ties : own;
        const u64 n = w ? (want - above + w - 1) / w : most;
        if (n < most) most = n;
        cut = most < own;
        ties = most;
        kkey = pkey;
      }
    }
    least = (u64)kkey << 32;
    if (cut) {
      __syncthreads();
      const int last = locate<T>(
          sh, row, V, [&](int, float v) { return (u64)(key_of<T>(as_logit(v)) == kkey); },
          [&](u64) { return ties - 1; }, &total);
      least = place_of(kkey, last);
    }
  }
  // ---- the draw
  __syncthreads();
  const float from = value_of<T>((unsigned)(least >> 32));
  const int token = locate<T>(sh, row, V, [&](int i, float v) -> u64 {
    if (least) {
      if (!(v >= from)) return 0;
      if (place_of(key_of<T>(as_logit(v)), i) < least) return 0;
    }
    return counted(v);
  }, target_of, &total);
  if (tid == 0) answer(token, logit_at<T>(row, token), total);
}

}  // namespace mhs
