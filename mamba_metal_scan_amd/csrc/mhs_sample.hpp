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
// computed in 64 bits and summed as integers, w 2^S rounded down (S 45, less
// above 2^17 words): sums that no order of additions changes, off by less than
// 2^-S of the likeliest word per word.
//
// A block of 1024 threads has a row: a pass for its maximum, a radix descent
// over the keys of the logits (an order-preserving integer) where a border is wanted, with
// the words' count or weight per digit in LDS, and a pass for the kept weights' sums by
// wave, the wave in which the draw falls being divided further. Weights are formed only
// for words that can still be kept.
#pragma once

#include "mhs_packed.hpp"

namespace mhs {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kDigitBits = 11;
constexpr int kBins = 1 << kDigitBits;

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
template <class T>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  const float v = ld_p<T>(row, i);
  return v == v ? v + 0.f : -INFINITY;
}
// Keys order as their floats do.
template <class T>
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned u = __float_as_uint(v);
  return (u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u)) >> kLowBits<T>;
}

typedef unsigned long long u64;

struct SampleShared {
  u64 mass[kBins];
  unsigned count[kBins];
  u64 wave[kSampleWaves];
  float wave_f[kSampleWaves];
  u64 found_above, found_mass;
  unsigned found_bin, found_count;
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

// The first index i of [0, n) with f(0) + .. + f(i) > target(total), total the sum
// of all; n if there is none. *total_out is that total. All threads of the block call it.
template <class F, class G>
__device__ int locate(SampleShared& sh, int n, F&& f, G&& target_of, u64* total_out) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int lo = 0, len = n;
  u64 base = 0, target = 0;
  bool first = true;
  for (;;) {
    const int seg = (len + kSampleThreads - 1) / kSampleThreads * 64;   // a wave's share
    const int b = min(len, wave * seg), e = min(len, b + seg);
    u64 s = 0;
    for (int i = b + lane; i < e; i += 64) s += f(lo + i);
    s = wave_total(s);
    __syncthreads();
    if (lane == 0) sh.wave[wave] = s;
    __syncthreads();
    u64 run = base;
    if (first) {
      u64 total = 0;
      for (int w = 0; w < kSampleWaves; ++w) total += sh.wave[w];
      *total_out = total;
      target = target_of(total);
      first = false;
    }
    int w = 0;
    while (w < kSampleWaves && run + sh.wave[w] <= target) run += sh.wave[w++];
    if (w == kSampleWaves) return n;
    base = run;
    lo += w * seg;
    len = min(seg, len - w * seg);
    if (len <= 64) break;
  }
  // every wave alike
  const u64 mine = lane < len ? f(lo + lane) : 0;
  const u64 run = base + wave_scan(mine, lane);
  const u64 hit = __ballot(lane < len && run > target);
  return hit ? lo + __ffsll((long long)hit) - 1 : n;
}

// Radix descent to a key. Each level counts, per digit, the words whose higher digits
// are those found (take(i, v, key): false leaves a word out; *m its weight), and goes on
// in the digit that choose(above, count, mass, bin's own) names: with BY_COUNT the
// first from the top at which the words reach `want`, else the last (lowest) that has
// words and less than `want` weight above it. Returns the key; *above is the count (weight)
// of the keys above it, *own its own words.
template <class T, bool BY_COUNT, class F>
__device__ unsigned descend(SampleShared& sh, int n, F&& take, u64 want, u64* above_out,
                            unsigned* own) {
  constexpr int kBits = 32 - kLowBits<T>;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  unsigned prefix = 0;
  u64 above = 0;
  int shift = kBits;
  while (shift > 0) {
    const int bits = min(kDigitBits, shift);
    shift -= bits;
    for (int i = tid; i < kBins; i += kSampleThreads) {
      sh.mass[i] = 0;
      sh.count[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
      unsigned key;
      u64 m = 0;
      if (!take(i, shift + bits, prefix, &key, &m)) continue;
      const unsigned bin = (key >> shift) & ((1u << bits) - 1);
      atomicAdd(&sh.count[bin], 1u);
      if (!BY_COUNT && m) atomicAdd(&sh.mass[bin], m);
    }
    __syncthreads();
    // Bins from the top: thread t has bins kBins - 1 - 2 t and the one below.
    const int b0 = kBins - 1 - 2 * tid, b1 = b0 - 1;
    const u64 v0 = BY_COUNT ? sh.count[b0] : sh.mass[b0];
    const u64 v1 = BY_COUNT ? sh.count[b1] : sh.mass[b1];
    const u64 mine = v0 + v1;
    u64 run = wave_scan(mine, lane);
    if (lane == 63) sh.wave[wave] = run;
    if (tid == 0) sh.found_bin = 0xFFFFFFFFu;
    __syncthreads();
    u64 before = above + run - mine;
    for (int w = 0; w < wave; ++w) before += sh.wave[w];
    // the bins' weight above: before, before + v0
    if (BY_COUNT) {
      if (before < want && before + v0 >= want) {
        sh.found_bin = b0;
        sh.found_above = before;
      } else if (before + v0 < want && before + v0 + v1 >= want) {
        sh.found_bin = b1;
        sh.found_above = before + v0;
      }
    } else {
      // the lowest: the smallest bin number wins
      const unsigned c0 = sh.count[b0], c1 = sh.count[b1];
      if (c1 && before + v0 < want) atomicMin(&sh.found_bin, (unsigned)b1);
      else if (c0 && before < want) atomicMin(&sh.found_bin, (unsigned)b0);
    }
    __syncthreads();
    const unsigned bin = sh.found_bin;
    if (!BY_COUNT) {
      if (bin == (unsigned)b0) sh.found_above = before;
      if (bin == (unsigned)b1) sh.found_above = before + v0;
      __syncthreads();
    }
    if (bin == 0xFFFFFFFFu) break;   // (nothing to find: not reached by the calls below)
    above = sh.found_above;
    *own = sh.count[bin];
    prefix = (prefix << bits) | bin;
    __syncthreads();
  }
  *above_out = above;
  return prefix;
}

template <class T>
__global__ void __launch_bounds__(kSampleThreads)
sample_kernel(SampleArgs a) {
  __shared__ SampleShared sh;
  const int r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int V = a.vocab;
  const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.ld * kElem<T>;
  const float temp = a.temperature ? a.temperature[r] : a.temperature_v;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p_v;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p_v;
  const long long kk = !a.top_k ? a.top_k_v
                       : a.k64 ? static_cast<const long long*>(a.top_k)[r]
                               : (long long)static_cast<const int*>(a.top_k)[r];
  // ---- the largest logit
  float m = -INFINITY;
  for (int i = tid; i < V; i += kSampleThreads) m = fmaxf(m, logit_at<T>(row, i));
#pragma unroll
  for (int s = 32; s; s /= 2) m = fmaxf(m, __shfl_xor(m, s));
  if (lane == 0) sh.wave_f[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) m = fmaxf(m, sh.wave_f[w]);
  if (!(temp >= 0.f && temp < INFINITY && min_p <= 1.f && top_p == top_p) || m == -INFINITY) {
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = __builtin_nanf("");
    }
    return;
  }
  const double md = m, td = temp;
  const double one = (double)(1ULL << a.scale);
  // (temperature 0, or a row that has +inf: the largest logits alone)
  const bool peak = temp == 0.f || m == INFINITY;
  const auto weight = [&](float v) { return peak ? (v == m ? 1.0 : 0.0) : exp(((double)v - md) / td); };
  const auto fixed = [&](double w) { return (u64)(w * one); };

  // ---- top-k: the key of the k-th word, and how many of that key are kept
  unsigned kkey = 0;
  u64 ties = ~0ULL;    // of kkey, by index
  bool cut = false;    // whether some word of kkey is left out
  if (temp == 0.f) {
    kkey = key_of<T>(m);
    ties = 1;
    cut = true;
  } else if (kk > 0 && kk < V) {
    u64 above;
    unsigned own = 0;
    kkey = descend<T, true>(sh, V, [&](int i, int sh_, unsigned pre, unsigned* key, u64*) {
      *key = key_of<T>(logit_at<T>(row, i));
      return (sh_ == 32 - kLowBits<T> ? 0 : *key >> sh_) == pre;
    }, (u64)kk, &above, &own);
    ties = (u64)kk - above;
    cut = ties < own;
  }
  // ---- top-p among those
  if (temp > 0.f && top_p < 1.f) {
    // the total: words above kkey, and `ties` of it
    u64 s = 0;
    unsigned own = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float v = logit_at<T>(row, i);
      const unsigned key = key_of<T>(v);
      if (key > kkey || (key == kkey && !cut)) s += fixed(weight(v));
    }
    s = wave_total(s);
    __syncthreads();
    if (lane == 0) sh.wave[wave] = s;
    __syncthreads();
    u64 total = 0;
    for (int w = 0; w < kSampleWaves; ++w) total += sh.wave[w];
    __syncthreads();
    // a key's float, for the weight of the words that share it
    const auto value = [&](unsigned key) {
      unsigned u = key << kLowBits<T>;
      if (u >> 31) u ^= 0x80000000u;
      else u = ~(u | ((1u << kLowBits<T>) - 1));
      return __uint_as_float(u);
    };
    if (cut) total += ties * fixed(weight(value(kkey)));
    const double border = (double)top_p * (double)total;
    // weights below it, as integers: x < border <=> x < ceil(border)
    const u64 want = border > 0.0 ? (u64)ceil(border) : 0;
    if (want == 0) {
      kkey = key_of<T>(m);
      ties = 1;
      cut = true;
    } else {
      u64 above;
      const unsigned pkey = descend<T, false>(
          sh, V, [&](int i, int sh_, unsigned pre, unsigned* key, u64* w) {
            const float v = logit_at<T>(row, i);
            *key = key_of<T>(v);
            if (*key < kkey || (sh_ == 32 - kLowBits<T> ? 0 : *key >> sh_) != pre) return false;
            *w = fixed(weight(v));
            return true;
          }, want, &above, &own);
      // the words of pkey in turn: the i-th has above + i w before it
      const u64 w = fixed(weight(value(pkey)));
      u64 most = pkey == kkey && cut ? ties : own;
      u64 n = w ? (want - above + w - 1) / w : most;
      if (n < most) most = n;
      cut = most < own;
      ties = most;
      kkey = pkey;
    }
  }
  // ---- the draw
  int last_tie = V;   // words of kkey from here on are left out
  u64 total;
  if (cut) {
    __syncthreads();
    last_tie = locate(sh, V, [&](int i) { return (u64)(key_of<T>(logit_at<T>(row, i)) == kkey); },
                      [&](u64) { return ties - 1; }, &total) + 1;
  }
  const auto kept = [&](int i, float* v) {
    *v = logit_at<T>(row, i);
    const unsigned key = key_of<T>(*v);
    return key > kkey || (key == kkey && i < last_tie);
  };
  const double low = min_p;
  const auto counted = [&](int i) -> u64 {
    float v;
    if (!kept(i, &v)) return 0;
    const double w = weight(v);
    return w >= low ? fixed(w) : 0;
  };
  __syncthreads();
  const float uf = a.uniform[r];
  const int token = locate(sh, V, counted, [&](u64 all) -> u64 {
    const double t = (double)uf * (double)all;
    // x > t <=> x > floor(t); below 0 and NaN: the first; at or past the total: the last
    return !(t > 0.0) ? 0 : t >= (double)all ? all - 1 : (u64)t;
  }, &total);
  if (tid == 0) {
    a.tokens[r] = token;
    if (a.logprobs)
      a.logprobs[r] = (float)log(weight(logit_at<T>(row, token)) * one / (double)total);
  }
}

}  // namespace mhs
