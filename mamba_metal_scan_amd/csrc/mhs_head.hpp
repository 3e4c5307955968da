// Losses of a language model's head from its hidden states, for gfx950: the
// logits z = h W^T (h (rows, dim), W (vocab, dim)) are formed tile by tile. With
// c = log2(e) / temperature and everything in base 2,
//   lse2_r = log2 sum_v 2^(c z_rv),       p_rv = 2^(c z_rv - lse2_r)
// and a row's targets (ids id_k with weights q_k; one of weight 1 for the
// cross entropy, the teacher's words for distillation) give
//   cross entropy   loss_r = ln(2) lse2_r - z_r,id             (temperature 1)
//   distillation    loss_r = t^2 sum_k q_k (ln q_k - z_r,k / t + ln(2) lse2_r)
//   dz_rv = coef_r (p_rv - sum_{k: id_k = v} q_k)
//   dh = dz W,  dW = dz^T h
// with coef_r the gradient that reaches the row's loss, times t for
// distillation.
//
// Forward: the product W h^T, whose epilogue reduces each tile to a maximum and
// a sum per row (head_lse); a pass over the rows joins the tiles, forms the
// logits of the row's ids again as dot products, and the loss.
// Backward, a piece of the vocabulary at a time: the product again, or the logits
// that the forward kept in fp32, and from them dz (16 bits, or fp32 for fp32
// operands) to the workspace, then the products with W and h. dW's rows are
// complete with their piece, dh sums over the pieces in fp32.
#pragma once

#include "mhs_common.hpp"
#include "mhs_gemm.hpp"
#include "mhs_mm16.hpp"
#include "mhs_xent.hpp"

namespace mhs {

// ---------------------------------------------------------------- elements

// fp32 beside Bf16 and Fp16: an element's storage and conversions.
struct Fp32 {
  typedef float type;
  static __device__ __forceinline__ float from(float v) { return v; }
  static __device__ __forceinline__ float to(float v) { return v; }
};
template <class T>
struct ElemOf {
  typedef unsigned short type;
};
template <>
struct ElemOf<Fp32> {
  typedef float type;
};
template <class T>
using elem_t = typename ElemOf<T>::type;
template <class T>
constexpr int kVec = 16 / sizeof(elem_t<T>);   // elements of a 16-byte access

template <class T>
struct alignas(16) Vec {
  elem_t<T> v[kVec<T>];
};

// ------------------------------------------------------- sums of exponentials

// The log-sum-exp of a lane's part of a column of an accumulated tile (N values,
// value i at row row(i) of the vocabulary), in base 2 of y = c z over rows below
// `left`. A NaN logit makes the sum NaN.
template <int N, class Z, class R>
__device__ __forceinline__ void column_lse2(const Z& z, const R& row, float c, int left, float& m,
                                            float& s) {
  m = -INFINITY;
  s = 0.f;
  if (row(N - 1) < left) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, z(i));
    m *= c;
    const float sh = lse2_shift(m);
#pragma unroll
    for (int i = 0; i < N; ++i) s += exp2_hw(__builtin_fmaf(z(i), c, -sh));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, row(i) < left ? z(i) : -INFINITY);
    m *= c;
    const float sh = lse2_shift(m);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = exp2_hw(__builtin_fmaf(z(i), c, -sh));
      s += row(i) < left ? e : 0.f;
    }
  }
}

// Joins the (m, s) of a tile's WM waves per column (cols columns, red: 2 WM cols
// floats of LDS) and writes the tile's row of the partials.
template <int WM>
__device__ __forceinline__ void store_partials(float* red, float2* part, int n0, int rows,
                                               int cols, long long at) {
  for (int n = threadIdx.x; n < cols; n += blockDim.x) {
    float m = red[n], s = red[cols + n];
#pragma unroll
    for (int w = 1; w < WM; ++w)
      lse2_combine(m, s, red[2 * w * cols + n], red[(2 * w + 1) * cols + n]);
    if (n0 + n < rows) part[at * rows + n0 + n] = make_float2(m, s);
  }
}

// Logits that a forward keeps for its backward, fp32: (rows, ld) of 16-bit
// operands, (words, ld) of fp32 ones, as dz; ld a multiple of 4. Null: none.
struct KeptLogits {
  float* z;
  long long ld;
};

// part[tile of the vocabulary][row] = (m, s) of the tile's logits, and, KEEP, the
// logits. A = W (M = vocab), B = h (N = rows). Bound by the matrix cores: the tiles
// run as one stream (mm_stream), so that a tile's exponentials overlap the next one's
// loads. bf16 8192 x 640 x 32768 348 us (987 TFLOP/s; a block per tile 377), 8192 x
// 4096 x 131072 6206 us (1417).
template <class T, class S, bool KEEP>
__global__ void __launch_bounds__(S::kThreads, 2)
head_lse_kernel(MmArgs g, float c, float2* __restrict__ part, KeptLogits kept) {
  extern __shared__ float lds_f[];
  float* const red = lds_f + S::kLds / 4;   // [WM][max, sum][BN]
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = S::wave_m(wave), wn = S::wave_n(wave);
  const auto none = [](int, int) {};
  mm_stream<T, S>(g, reinterpret_cast<char*>(lds_f), none, [&](auto& acc, int m0, int n0, int) {
    const int lane = mm_opaque(threadIdx.x & 63);
    const int left = g.M - m0 - wm * (S::FM * 16) - 32 * (lane >> 5) - 4 * ((lane >> 4) & 1);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      float m, s;
      column_lse2<S::FM * 4>([&](int i) { return acc[i / 4][j][i % 4]; },
                             [](int i) { return 64 * (i / 16) + 8 * (i / 4 % 4) + i % 4; }, c,
                             left, m, s);
#pragma unroll
      for (int o = 16; o < 64; o *= 2)
        lse2_combine(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
      const int n = (wn * S::FN + j) * 16 + lane;
      if (lane < 16) {
        red[2 * wm * S::BN + n] = m;
        red[(2 * wm + 1) * S::BN + n] = s;
      }
      if (!KEEP) continue;
      // 16 bytes a lane, 32 of 16 rows at a time; four stores fill a row's 128.
      const int r = n0 + (wn * S::FN + j) * 16 + (lane & 15);
      float* const row = kept.z + (long long)r * kept.ld + g.M - left;
      if (r < g.N)
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
          if (64 * (i / 4) + 8 * (i % 4) < left)
            *reinterpret_cast<f32x4*>(row + 64 * (i / 4) + 8 * (i % 4)) =
                f32x4{acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
    }
    mm_lds_barrier();
    store_partials<S::WM>(red, part, n0, g.N, S::BN, m0 / S::BM);
  });
}

// The same for fp32 operands, on the products of three bf16 parts, whose rate
// bounds it: 8192 x 640 x 32768 1820 us (189 TFLOP/s), 1985 with the logits kept.
template <int TILE>
__global__ void __launch_bounds__(kGemmThreads, TILE == kGemmTile ? 3 : 4)
head_lse3_kernel(GemmArgs g, float c, float2* __restrict__ part, KeptLogits kept) {
  extern __shared__ float lds_f[];
  constexpr int F = TILE / 64;
  int m0, n0;
  gemm3_place<TILE>(g, m0, n0);
  f32x16 acc[F][F];
  gemm3_products<true, true, TILE>(acc, g, m0, n0, 0, g.K);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < F; ++j) {
    float m, s;
    column_lse2<F * 16>([&](int i) { return acc[i / 16][j][i % 16]; },
                        [](int i) { return i / 16 * 32 + 8 * (i % 16 / 4) + i % 4; }, c,
                        g.M - m0 - wm * (TILE / 2) - 4 * (lane >> 5), m, s);
    lse2_combine(m, s, __shfl_xor(m, 32, 64), __shfl_xor(s, 32, 64));
    const int n = wn * (TILE / 2) + j * 32 + lane;
    if (lane < 32) {
      lds_f[2 * wm * TILE + n] = m;
      lds_f[(2 * wm + 1) * TILE + n] = s;
    }
    const int r = n0 + wn * (TILE / 2) + j * 32 + (lane & 31);
    if (kept.z && r < g.N)
#pragma unroll
      for (int i = 0; i < F * 16; ++i) {
        const int v = m0 + wm * (TILE / 2) + i / 16 * 32 + 8 * (i % 16 / 4) + 4 * (lane >> 5) +
                      i % 4;
        if (v < g.M) kept.z[v * kept.ld + r] = acc[i / 16][j][i % 16];
      }
  }
  __syncthreads();
  store_partials<2>(lds_f, part, n0, g.N, TILE, m0 / TILE);
}

// The same from logits in memory, for products whose tiles are too few to fill the
// CUs and which are cut up in k: bound by their latency, a few us. fp32, (words,
// ld): 64 words by 64 rows a block, a wave 16 words of each.
constexpr int kLogitWords = 64;
template <int UNUSED = 0>
__global__ void __launch_bounds__(256)
head_lse_of_logits_kernel(KeptLogits logits, int words, int rows, float c,
                          float2* __restrict__ part) {
  __shared__ float red[2 * 4 * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = blockIdx.y * 64, v0 = blockIdx.x * kLogitWords + wave * 16;
  const int left = words - v0, r = min(n0 + lane, rows - 1);
  float z[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    z[i] = i < left ? logits.z[(long long)(v0 + i) * logits.ld + r] : 0.f;
  float m, s;
  column_lse2<16>([&](int i) { return z[i]; }, [](int i) { return i; }, c, left, m, s);
  red[2 * wave * 64 + lane] = m;
  red[(2 * wave + 1) * 64 + lane] = s;
  __syncthreads();
  store_partials<4>(red, part, n0, rows, 64, blockIdx.x);
}

// 16 bits, the sums (splits, rows, ld) of the splits: a wave takes 256 words of a
// row, sums the splits in order and, kept given, leaves the logits there.
constexpr int kSplitWords = 256;
template <int UNUSED = 0>
__global__ void __launch_bounds__(256)
head_lse_of_splits_kernel(const float* __restrict__ sums, long long ld, int splits, int words,
                          int rows, float c, float2* __restrict__ part, KeptLogits kept) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;   // (whole waves; no barrier below)
  const int v = blockIdx.x * kSplitWords + 4 * lane;
  float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
  if (v < words) {
    for (int k = 0; k < splits; ++k)
      z = add(z, *reinterpret_cast<const float4*>(sums + ((long long)k * rows + r) * ld + v));
    if (kept.z) *reinterpret_cast<float4*>(kept.z + r * kept.ld + v) = z;
  }
  const float y[4] = {z.x, z.y, z.z, z.w};
  float m, s;
  column_lse2<4>([&](int i) { return y[i]; }, [](int i) { return i; }, c, words - v, m, s);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1)
    lse2_combine(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
  if (lane == 0) part[(long long)blockIdx.x * rows + r] = make_float2(m, s);
}

// --------------------------------------------------------------- few rows
//
// Up to 16 NF rows: bound by reading W once. A block takes 64 words straight from
// memory as operands of 16 x 16 MFMAs (lane: word lane % 16, 16 bytes at lane / 16
// of each 64), the rows' operands beside them (in L1 and L2), so nothing is
// staged. The waves share the block's words and cut up k, 128 bytes of each row in
// turn, so that a row's operand serves four of the words'; their sums meet in LDS.
// (With 16 words and all of k to a wave the rows' operands are read as often as
// the words': 16 rows of 4096 x 131072 words took 584 us in fp32 and 294 in bf16,
// against 476 and 254, which is 4.5 TB/s and 4.2; one row 447 and 222 against 436
// and 218. 640 x 32768, 16 rows, with the loss: 29 us and 19.)

constexpr int kSmallWords = 64;   // per block of 4 waves

template <class T>
struct SmallMma {   // 64 bytes of k per step
  static constexpr int kDepth = 32;
  typedef s16x8 frag;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 acc) {
    if constexpr (__is_same(T, Bf16))
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                     __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                    __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
};
template <>
struct SmallMma<Fp32> {   // element e of every lane: one MFMA, its k's 4 (lane / 16) + e
  static constexpr int kDepth = 16;
  typedef f32x4 frag;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 acc) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
    return acc;
  }
};

struct SmallArgs {
  const void* h;
  const void* w;
  long long ldh, ldw;   // rows 16-byte aligned
  int rows, vocab, dim; // dim a multiple of a 16-byte access
};

// One operand's 16 bytes for k step `k` of a row (zeros past the row's end).
template <class T>
__device__ __forceinline__ typename SmallMma<T>::frag small_load(const elem_t<T>* p, int k,
                                                                 int dim, bool ok) {
  typedef typename SmallMma<T>::frag frag;
  frag f = {};
  if (ok && k < dim) f = *reinterpret_cast<const frag*>(p + k);
  return f;
}

template <class T, int NF>
__global__ void __launch_bounds__(256)
head_small_kernel(SmallArgs g, float c, float2* __restrict__ part, KeptLogits kept) {
  typedef SmallMma<T> M;
  constexpr int FW = kSmallWords / 16;   // fragments of words; one for each wave at the end
  __shared__ f32x4 sums[FW][4][NF][64];
  __shared__ float red[2][4][16 * NF];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int word = blockIdx.x * kSmallWords + (lane & 15);
  const int k0 = kVec<T> * (lane >> 4);
  const elem_t<T>* w[FW];
  const elem_t<T>* h[NF];
  bool okw[FW], ok[NF];
#pragma unroll
  for (int i = 0; i < FW; ++i) {
    okw[i] = word + 16 * i < g.vocab;
    w[i] = static_cast<const elem_t<T>*>(g.w) + (long long)(okw[i] ? word + 16 * i : 0) * g.ldw;
  }
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int r = 16 * j + (lane & 15);
    ok[j] = r < g.rows;
    h[j] = static_cast<const elem_t<T>*>(g.h) + (long long)(ok[j] ? r : 0) * g.ldh;
  }
  f32x4 acc[FW][NF] = {};
  constexpr int U = 2;   // k steps whose loads are in flight together, 128 bytes of each row
                         // (503 us with 4, 520 with 8 where 2 take 476: 16 x 4096 x 131072, fp32)
  for (int k = 2 * wave * M::kDepth; k < g.dim; k += 4 * U * M::kDepth) {
    typename M::frag a[U][FW], b[U][NF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + u * M::kDepth + k0;
#pragma unroll
      for (int i = 0; i < FW; ++i) a[u][i] = small_load<T>(w[i], at, g.dim, okw[i]);
#pragma unroll
      for (int j = 0; j < NF; ++j) b[u][j] = small_load<T>(h[j], at, g.dim, ok[j]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < FW; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = M::mma(a[u][i], b[u][j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < FW; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) sums[i][wave][j][lane] = acc[i][j];
  __syncthreads();
  // The wave joins fragment `wave`. Element e of a lane: word 4 (lane / 16) + e,
  // row lane % 16.
  const int left = g.vocab - (blockIdx.x * kSmallWords + wave * 16 + 4 * (lane >> 4));
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    f32x4 z = sums[wave][0][j][lane];
#pragma unroll
    for (int v = 1; v < 4; ++v) z += sums[wave][v][j][lane];
    if (kept.z && ok[j] && left > 0) {
      const long long v = g.vocab - left, r = 16 * j + (lane & 15);
      if constexpr (__is_same(T, Fp32)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) kept.z[(v + e) * kept.ld + r] = z[e];
      } else {
        *reinterpret_cast<f32x4*>(kept.z + r * kept.ld + v) = z;
      }
    }
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, e < left ? z[e] * c : -INFINITY);
    const float sh = lse2_shift(m);
#pragma unroll
    for (int e = 0; e < 4; ++e) s += e < left ? exp2_hw(__builtin_fmaf(z[e], c, -sh)) : 0.f;
#pragma unroll
    for (int o = 16; o <= 32; o *= 2)
      lse2_combine(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
    if (lane < 16) {
      red[0][wave][16 * j + lane] = m;
      red[1][wave][16 * j + lane] = s;
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < min(g.rows, 16 * NF)) {
    const int r = threadIdx.x;
    float m = red[0][0][r], s = red[1][0][r];
#pragma unroll
    for (int v = 1; v < 4; ++v) lse2_combine(m, s, red[0][v][r], red[1][v][r]);
    part[(long long)blockIdx.x * g.rows + r] = make_float2(m, s);
  }
}

// ---------------------------------------------------------------- the rows

// The dot products of row a with U rows b[u] of dim elements (16-byte aligned,
// whole accesses) over the wave's lanes, their loads in flight together; every
// lane returns them. Of W waves, each a part of every row.
template <class T, int U, int W = 1>
__device__ __forceinline__ void wave_dots(const elem_t<T>* a, const elem_t<T>* const (&b)[U],
                                          int dim, float (&s)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u) s[u] = 0.f;
  for (int i = (threadIdx.x & (64 * W - 1)) * kVec<T>; i < dim; i += 64 * W * kVec<T>) {
    const Vec<T> x = *reinterpret_cast<const Vec<T>*>(a + i);
    Vec<T> y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = *reinterpret_cast<const Vec<T>*>(b[u] + i);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e)
        s[u] = __builtin_fmaf(T::to(x.v[e]), T::to(y[u].v[e]), s[u]);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] += __shfl_xor(s[u], o, 64);
}

struct HeadRows {
  const void* h;          // (rows, dim)
  const void* w;          // (vocab, dim)
  long long ldh, ldw;
  const float2* part;     // (tiles, rows)
  const long long* ids;   // (rows) targets, or (rows, k) the teacher's words
  const float* teacher;   // (rows, k) the teacher's logits
  float* lse2;            // (rows)
  float* picked;          // (rows, k) logits of the ids
  float* q;               // (rows, k) the words' weights, see teacher_row
  float* loss;            // (rows)
  float* keep;            // (rows) 1: the row counts, 0: ignored or empty
  KeptLogits kept;        // the forward's logits, or null
  int rows, vocab, dim, k, tiles;
  long long ignore;
  float temperature;
};

// The logit of row r and word id: one of the sums that lse2 is of. Where logits are kept
// the ids' come from there, not from dot products of their own: their errors would not
// cancel against lse2's in a row that is sure of its word (of 595 x 64 x 2832 fp32,
// distillation, gradients off by 2.0e-6 of their norm for 1.0e-6 so).
template <class T>
__device__ __forceinline__ float kept_logit(const KeptLogits& kept, long long r, long long id) {
  return kept.z[__is_same(T, Fp32) ? id * kept.ld + r : r * kept.ld + id];
}

// Cross entropy: W waves (1 or 4) per row. Bound by latency: 12 us at 8192 rows of
// 640 and 128 tiles, 50 at 4096 and 512.
template <class T, int W>
__global__ void __launch_bounds__(256)
head_xent_rows_kernel(HeadRows g) {
  __shared__ float red[W];
  const int lane = threadIdx.x & (64 * W - 1);
  const int r = blockIdx.x * (4 / W) + threadIdx.x / (64 * W);
  if (r >= g.rows) return;   // (whole waves; with four, no block is past the rows)
  float m = -INFINITY, s = 0.f;
  for (int t = lane; t < g.tiles; t += 64 * W) {
    const float2 p = g.part[(long long)t * g.rows + r];
    lse2_combine(m, s, p.x, p.y);
  }
  if constexpr (W == 4) {
    block_lse2(m, s);
  } else {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
      lse2_combine(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64));
  }
  const float lse2 = m + log2f(s);
  const long long t = g.ids[r];
  const bool in = t >= 0 && t < g.vocab;
  float dot[1];
  if (g.kept.z) {
    dot[0] = kept_logit<T>(g.kept, r, in ? t : 0);
  } else {
    const elem_t<T>* const word[1] = {static_cast<const elem_t<T>*>(g.w) + (in ? t : 0) * g.ldw};
    wave_dots<T, 1, W>(static_cast<const elem_t<T>*>(g.h) + (long long)r * g.ldh, word, g.dim, dot);
    if constexpr (W == 4) {
      if ((lane & 63) == 0) red[lane >> 6] = dot[0];
      __syncthreads();
      dot[0] = red[0] + red[1] + red[2] + red[3];
    }
  }
  const float z = in ? dot[0] : 0.f;
  if (lane == 0) {
    const bool keep = t != g.ignore;
    g.lse2[r] = lse2;
    g.picked[r] = z;
    g.loss[r] = !keep ? 0.f : in ? lse2 * kLn2 - z : __builtin_nanf("");
    g.keep[r] = keep ? 1.f : 0.f;
  }
}

// The block's sum of v, the same in every thread (256 threads, fixed order).
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The teacher's probabilities of row r over its kept words (id >= 0), and the
// row's loss from the student's logits zk at the ids (LDS, k floats, then room
// for k more) and lse2; offset(lse2) may take one away from both, and returns the
// lse2 that the backward gets. To q goes each word's whole weight in the row: a word
// that the row names twice has both entries' sum at each. A row that keeps no
// word, or whose kept logits are all -inf, is empty: loss 0, probabilities 0. An
// id at or past the vocabulary: NaN.
template <class Offset>
__device__ __forceinline__ void teacher_row(const HeadRows& g, int r, float lse2, float* zk,
                                            float* red, const Offset& offset) {
  const long long at = (long long)r * g.k;
  const float c = kLog2e / g.temperature;
  float m = -INFINITY, bad = 0.f;
  for (int k = threadIdx.x; k < g.k; k += 256) {
    const long long id = g.ids[at + k];
    if (id >= 0) m = fmaxf(m, g.teacher[at + k]);
    if (id >= g.vocab) bad = 1.f;
  }
  m = block_max(m, red);
  bad = block_max(bad, red);
  float any = 0.f, s = 0.f;
  const float sh = lse2_shift(m);   // (the difference first: no loss to a common offset)
  for (int k = threadIdx.x; k < g.k; k += 256)
    if (g.ids[at + k] >= 0) {
      const float e = exp2_hw((g.teacher[at + k] - sh) * c);
      s += e;
      if (e != 0.f) any = 1.f;   // (NaN counts: the row's loss is NaN)
    }
  s = block_sum(s, red);
  any = block_max(any, red);
  const float stored = offset(lse2);
  const float log2s = log2f(s), inv = any != 0.f ? 1.f / s : 0.f;
  float loss = 0.f;
  for (int k = threadIdx.x; k < g.k; k += 256) {
    float q = 0.f;
    if (any != 0.f && g.ids[at + k] >= 0) {
      const float y = (g.teacher[at + k] - sh) * c;
      q = exp2_hw(y) * inv;
      if (q != 0.f)
        loss += q * ((y - log2s + lse2) * kLn2 - zk[k] / g.temperature);
    }
    zk[g.k + k] = q;
  }
  loss = block_sum(loss, red);   // (its barriers publish the q's)
  // (constant memory: scalar loads, which the compiler gives up behind offset's branch;
  // vector ones take 10 us of distill_fwd_kernel's 236 at 64 words)
  typedef const __attribute__((address_space(4))) long long* ConstIds;
  const ConstIds ids = (ConstIds)(unsigned long long)(g.ids + at);
  for (int k = threadIdx.x; k < g.k; k += 256) {
    const long long id = g.ids[at + k];
    float q = 0.f;
    for (int j = 0; j < g.k; ++j) q += ids[j] == id ? zk[g.k + j] : 0.f;
    g.q[at + k] = q;
  }
  if (threadIdx.x == 0) {
    g.lse2[r] = stored;
    g.keep[r] = any;
    g.loss[r] = any == 0.f ? 0.f
                // (t^2 by itself is 0 or infinite where the loss is neither)
                : bad != 0.f ? __builtin_nanf("") : g.temperature * (g.temperature * loss);
  }
}

// Distillation: a block per row. Bound by the gathered rows of W, from the caches:
// 8192 rows of 64 words of 640, 671 MB in 16 bits, 105 us (6.4 TB/s).
template <class T>
__global__ void __launch_bounds__(256)
head_distill_rows_kernel(HeadRows g) {
  extern __shared__ float zk[];   // 2 k floats
  __shared__ float red[4];
  const int r = blockIdx.x, wave = threadIdx.x >> 6;
  const elem_t<T>* h = static_cast<const elem_t<T>*>(g.h) + (long long)r * g.ldh;
  if (g.kept.z) {
    for (int k = threadIdx.x; k < g.k; k += 256) {
      const long long id = g.ids[(long long)r * g.k + k];
      const bool in = id >= 0 && id < g.vocab;
      zk[k] = in ? kept_logit<T>(g.kept, r, id) : 0.f;
      g.picked[(long long)r * g.k + k] = zk[k];
    }
  }
  constexpr int U = 4;   // words at a time (8192 x 640, 64 words: one 138 us, four 105)
  for (int k = U * wave; !g.kept.z && k < g.k; k += 4 * U) {
    const elem_t<T>* word[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long id = k + u < g.k ? g.ids[(long long)r * g.k + k + u] : -1;
      in[u] = id >= 0 && id < g.vocab;
      word[u] = static_cast<const elem_t<T>*>(g.w) + (in[u] ? id : 0) * g.ldw;
    }
    float z[U];
    wave_dots<T, U>(h, word, g.dim, z);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if ((int)(threadIdx.x & 63) == u && k + u < g.k) {
        zk[k + u] = in[u] ? z[u] : 0.f;
        g.picked[(long long)r * g.k + k + u] = in[u] ? z[u] : 0.f;
      }
  }
  float m = -INFINITY, s = 0.f;
  for (int t = threadIdx.x; t < g.tiles; t += 256) {
    const float2 p = g.part[(long long)t * g.rows + r];
    lse2_combine(m, s, p.x, p.y);
  }
  block_lse2(m, s);   // (its barrier publishes zk)
  teacher_row(g, r, m + log2f(s), zk, red, [](float& lse2) { return lse2; });
}

// loss[0] = the sum of the rows' losses, over the count of rows kept for the
// mean (0 / 0 = NaN where none is); count[0] = that count. Blocks of 4096 rows
// leave their sums in `sums` (2 doubles each) for a last block of the same
// kernel; one block's rows need none. Sums in 64 bits, in a fixed order.
constexpr int kLossThreads = 1024, kLossRows = 4096;
template <int UNUSED = 0>
__global__ void __launch_bounds__(kLossThreads)
head_loss_kernel(const float* __restrict__ rows_loss, const float* __restrict__ keep,
                 const double2* __restrict__ in, double2* __restrict__ out,
                 float* __restrict__ loss, float* __restrict__ count, long long n, int mean) {
  __shared__ double sums[2][kLossThreads / 64];
  double s = 0.0, k = 0.0;
  const long long first = (long long)blockIdx.x * kLossRows;
  const long long end = out ? min(n, first + kLossRows) : n;
  for (long long i = first + threadIdx.x; i < end; i += kLossThreads) {
    const double2 v = in ? in[i] : make_double2((double)rows_loss[i], (double)keep[i]);
    s += v.x;
    k += v.y;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    k += __shfl_xor(k, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[0][threadIdx.x >> 6] = s;
    sums[1][threadIdx.x >> 6] = k;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kLossThreads / 64; ++w) {
    s += sums[0][w];
    k += sums[1][w];
  }
  if (out) {
    out[blockIdx.x] = make_double2(s, k);
  } else {
    loss[0] = (float)(mean ? s / k : s);
    count[0] = (float)k;
  }
}

// ---------------------------------------------------------------- backward

// The gradient that reaches each row's loss: upstream[0] (over count[0] for the
// mean), or upstream[r] where the rows' losses are the output; 0 for rows that
// do not count.
struct RowScale {
  const float* upstream;
  const float* count;   // null: no mean
  const float* keep;
  int per_row;
  float factor;         // distillation: the temperature
  __device__ __forceinline__ float reaching(long long r) const {
    const float u = upstream[per_row ? r : 0] * factor;
    return count ? u / count[0] : u;
  }
  __device__ __forceinline__ float at(long long r) const {
    return keep[r] == 0.f ? 0.f : reaching(r);
  }
};

// largest[0] = the largest |gradient| that reaches a row (per-row upstreams). One
// block.
template <int UNUSED = 0>
__global__ void __launch_bounds__(1024)
head_largest_kernel(RowScale rs, float* __restrict__ largest, long long rows) {
  __shared__ float red[16];
  float m = 0.f;
  for (long long r = threadIdx.x; r < rows; r += 1024) m = fmaxf(m, fabsf(rs.at(r)));
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) m = fmaxf(m, red[i]);
  largest[0] = m;
}

// The power of two by which dz is stored larger, such that the largest |coef| lies
// in [2^(to-1), 2^to); 1 where that is 0 or not finite. fp16: to 2^15, |dz| stays
// below 2^16, and probabilities below 2^-24 of it keep their bits. fp32: to 2^32
// (and never smaller: a row whose gradient is far below the largest keeps it), which
// takes the smallest probabilities (2^-126) to 2^-95, below which the fp32 product goes
// by fp32 MFMAs at half its rate (gemm3; 1024 x 4096 x 131072 of
// logits of std 64 without it: 41.2 ms for loss and gradients, 22.5 with std 1).
// bf16 products have no such bounds.
__device__ __forceinline__ float lift_of(float largest, int to) {
  if (!(largest > 0.f && largest < INFINITY)) return 1.f;
  int e = 0;
  (void)frexpf(largest, &e);   // largest in [2^(e-1), 2^e)
  return ldexpf(1.f, min(max(to - e, to == 32 ? 0 : -126), 126));
}

constexpr int kCopyRows = 8;   // rows per block

// What dz is stored with and what the products' sums are multiplied by. s is dz's
// power of two (lift_of to `lift`, scale[2] the largest per-row gradient; lift 0:
// 1). Where all rows share their coef = 2^e f, f in [1, 2), dz is stored with its
// 2^e alone and the sums take f: stored with coef, the id's element, about -coef,
// would be off by the same rounding in every row (errors relative to the gradients'
// norm: fp16 1001 x 384 x 50257 0.00030 to 0.00032, so 0.00025, of which 0.00021 is
// the results' own rounding; bf16 8192 x 4096 x 131072 0.0025, so 0.0019, and 0.0017).
// rows2[r] = (2^e s, or the row's coef s, lse2); scale[0] = f / s; and, `out` given, out
// (out_rows, per) = in (rows, per) in 16-byte words, rows ldi apart, with zeros in the
// rows past `rows` and those whose coef is 0: what a padded row holds, NaN too, does not
// reach dW.
template <int UNUSED = 0>
__global__ void __launch_bounds__(256)
head_rows_in_kernel(const uint4* __restrict__ in, long long ldi, RowScale rs,
                    const float* __restrict__ lse2, float2* __restrict__ rows2,
                    float* __restrict__ scale, uint4* __restrict__ out, long long rows,
                    long long out_rows, int per, int lift) {
  __shared__ float cf[kCopyRows];
  const long long r0 = (long long)blockIdx.x * kCopyRows;
  if (threadIdx.x < kCopyRows) {
    // (without per-row gradients the largest is the one that every kept row has)
    const float all = rs.per_row ? 1.f : fabsf(rs.reaching(0));
    const float s = !lift ? 1.f : lift_of(rs.per_row ? scale[2] : all, lift);
    int e = 0;
    const float f = all > 0.f && all < INFINITY ? 2.f * frexpf(all, &e) : 1.f;
    const long long r = r0 + threadIdx.x;
    const float c = r < rows ? rs.at(r) : 0.f;
    cf[threadIdx.x] = c;
    // (c / f: a power of two, exactly)
    if (r < ((rows + 1) & ~1LL)) rows2[r] = make_float2(c / f * s, r < rows ? lse2[r] : 0.f);
    if (r == 0) scale[0] = f / s;
  }
  if (!out) return;
  __syncthreads();
  const int n = (int)min((long long)kCopyRows, out_rows - r0) * per;   // (dim <= 2^20)
  for (int i = threadIdx.x; i < n; i += 256) {
    const int row = i / per;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (cf[row] != 0.f) v = in[(r0 + row) * ldi + i - row * per];
    out[r0 * per + i] = v;
  }
}

template <int UNUSED = 0>
__global__ void __launch_bounds__(256)
head_zero_kernel(unsigned* __restrict__ out, long long n) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (long long)gridDim.x * 256)
    out[i] = 0u;
}

// out's rows (rows, 4 per) whose coef is 0 are zeros: of an fp32 product their zeros
// times an infinity or NaN of the weight are not (the 16-bit ones' reduction sees to
// it). A wave a row: 3 us at 8 rows, 4 at 8192, of which none is zeroed.
template <int UNUSED = 0>
__global__ void __launch_bounds__(256)
head_zero_rows_kernel(const float2* __restrict__ rows2, float4* __restrict__ out, long long rows,
                      int per) {
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows || rows2[r].x != 0.f) return;
  for (int i = threadIdx.x & 63; i < per; i += 64)
    out[r * per + i] = make_float4(0.f, 0.f, 0.f, 0.f);
}

struct HeadGrad {
  const float2* rows2;     // (rows, to an even number) (coef s, lse2)
  const float* scale;      // what the sums are multiplied by
  const long long* ids;    // (rows, k)
  const float* q;          // (rows, k) the words' whole weights, or null: 1
  const float* picked;     // (rows, k)
  int k;
  int v0;                  // the piece's first word; M words in it
  float c;
  void* dz;                // (rows, ldz), or for fp32 (words, ldz)
  long long ldz;
};

// Exchanges 4 registers' groups of 16 lanes: v[q] then holds in group g what
// v[g] held in group q.
__device__ __forceinline__ void exchange4(unsigned (&v)[4]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const auto r = __builtin_amdgcn_permlane32_swap(v[q], v[q + 2], false, false);
    v[q] = r[0];
    v[q + 2] = r[1];
  }
#pragma unroll
  for (int q = 0; q < 4; q += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(v[q], v[q + 1], false, false);
    v[q] = r[0];
    v[q + 1] = r[1];
  }
}

// p's part of dz of a piece, 16 bits, (rows, ldz). Bound as head_lse_kernel, and by
// writing dz: 8192 x 640 x 32768 381 us in two pieces (902 TFLOP/s), 8192 x 4096 x
// 131072 6731 us in eight (1307). The tile has the words in m, dz
// the rows: a lane's 4 words of 4 fragments become 16 of one row (exchange4), in
// two stores of 16 bytes, each 64 bytes of 16 rows at a time; no LDS.
constexpr int kPairBytes = 2048;   // of LDS per slot: 256 rows' (coef, lse2)
template <class T, class S>
__global__ void __launch_bounds__(S::kThreads, 2)
head_dz_kernel(MmArgs g, HeadGrad a) {
  extern __shared__ float lds_f[];
  // The rows' (coef, lse2) of the stream's slots.
  static_assert(S::BN * 8 == kPairBytes, "two direct loads hold a tile's rows");
  char* const pairs = reinterpret_cast<char*>(lds_f) + S::kLds;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = S::wave_m(wave), wn = S::wave_n(wave);
  const auto load_pairs = [&](int n0, int slot) {
    if (wave >= 2) return;
    const int at = 128 * wave + 2 * (int)(threadIdx.x & 63);   // 2 rows a lane
    mm_load_lds(mm_resource(a.rows2 + n0), at < g.N - n0 ? 8u * (unsigned)at : kOOB,
                (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)pairs +
                    kPairBytes * slot + 1024 * wave);
  };
  mm_stream<T, S>(g, reinterpret_cast<char*>(lds_f), load_pairs, [&](auto& acc, int m0, int n0,
                                                                    int slot) {
    const int lane = mm_opaque(threadIdx.x & 63);
    m0 += wm * (S::FM * 16);
    const int left = g.M - m0 - 32 * (lane >> 5) - 4 * ((lane >> 4) & 1);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int in = (wn * S::FN + j) * 16 + (lane & 15), n = n0 + in;
      const float2 row2 = *reinterpret_cast<const float2*>(pairs + kPairBytes * slot + 8 * in);
      const float f = row2.x, l2 = row2.y;
      unsigned short* const row = static_cast<unsigned short*>(a.dz) + (long long)n * a.ldz + m0 +
                                  8 * (lane >> 4);
#pragma unroll
      for (int h = 0; h < S::FM / 4; ++h) {
        unsigned lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unsigned short v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = exp2_hw(__builtin_fmaf(acc[4 * h + i][j][e], a.c, -l2)) * f;
            // (an ignored row's zeros whatever its logits are)
            v[e] = T::from(f == 0.f || 64 * h + 8 * i + e >= left ? 0.f : p);
          }
          lo[i] = v[0] | (unsigned)v[1] << 16;
          hi[i] = v[2] | (unsigned)v[3] << 16;
        }
        exchange4(lo);
        exchange4(hi);
        if (n < g.N) {
          *reinterpret_cast<uint4*>(row + 64 * h) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
          *reinterpret_cast<uint4*>(row + 64 * h + 32) = make_uint4(lo[2], hi[2], lo[3], hi[3]);
        }
      }
    }
  });
}

// The same in fp32, transposed: (words, ldz), its rows contiguous. Bound by the
// product: 8192 x 640 x 32768 1870 us (184 TFLOP/s).
template <int TILE>
__global__ void __launch_bounds__(kGemmThreads, TILE == kGemmTile ? 3 : 4)
head_dz3_kernel(GemmArgs g, HeadGrad a) {
  constexpr int F = TILE / 64;
  int m0, n0;
  gemm3_place<TILE>(g, m0, n0);
  f32x16 acc[F][F];
  gemm3_products<true, true, TILE>(acc, g, m0, n0, 0, g.K);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  float* const dz = static_cast<float*>(a.dz);
#pragma unroll
  for (int j = 0; j < F; ++j) {
    const int r = n0 + wn * (TILE / 2) + j * 32 + (lane & 31);
    const int rc = min(r, g.N - 1);
    const float cf = a.rows2[rc].x, l2 = a.rows2[rc].y;
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + wm * (TILE / 2) + i * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        const float p = exp2_hw(__builtin_fmaf(acc[i][j][e], a.c, -l2)) * cf;
        // (columns past the rows, up to ldz: zeros for the next product)
        if (m < g.M && r < a.ldz) dz[m * a.ldz + r] = cf == 0.f || r >= g.N ? 0.f : p;
      }
  }
}

// p's part of dz of a piece from the logits that the forward kept: bound by
// reading them and writing dz (fp32, 8192 x 32768: 348 us, 2.1 GB at 6.2 TB/s with
// dz's pieces in the caches). 8 words of a row to a thread, or, fp32, 4 rows of a
// word, as they lie. `blocks` of 16 bytes to a row of dz, n in all.
template <class T>
__global__ void __launch_bounds__(256)
head_dz_kept_kernel(KeptLogits kept, HeadGrad a, int rows, int words, unsigned blocks,
                    long long n) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= n) return;
  const long long row = n < 0xFFFFFFFF ? (unsigned)id / blocks : id / blocks;
  const int at = kVec<T> * (int)(id - row * blocks);
  Vec<T> out;
  if constexpr (__is_same(T, Fp32)) {
    const float4 z = *reinterpret_cast<const float4*>(kept.z + (a.v0 + row) * kept.ld + at);
    const float v[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 row2 = a.rows2[min(at + e, rows - 1)];
      const float p = exp2_hw(__builtin_fmaf(v[e], a.c, -row2.y)) * row2.x;
      out.v[e] = row2.x == 0.f || at + e >= rows ? 0.f : p;
    }
  } else {
    const float2 row2 = a.rows2[row];
    const float* const z = kept.z + row * kept.ld + a.v0 + at;
    const float4 lo = *reinterpret_cast<const float4*>(z);
    float4 hi = make_float4(0.f, 0.f, 0.f, 0.f);
    if (at + 4 < words) hi = *reinterpret_cast<const float4*>(z + 4);
    const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = exp2_hw(__builtin_fmaf(v[e], a.c, -row2.y)) * row2.x;
      out.v[e] = T::from(row2.x == 0.f || at + e >= words ? 0.f : p);
    }
  }
  *reinterpret_cast<Vec<T>*>(static_cast<elem_t<T>*>(a.dz) + row * a.ldz + at) = out;
}

// dz at the rows' ids within a piece of `words` words, over what head_dz wrote:
// coef (p - q) from the logit kept in fp32, rounded once (a word that a row names
// twice: the same value twice). A wave per row. (Within head_dz, where every tile
// looks through its rows' ids, 64 ids a row cost 2400 us more at 8192 x 640 x
// 32768; this takes 20.)
template <class T>
__global__ void __launch_bounds__(256)
head_ids_kernel(HeadGrad a, long long rows, int words) {
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const float f = a.rows2[r].x, l2 = a.rows2[r].y;
  if (f == 0.f) return;
  const long long at = r * a.k;
  for (int k = threadIdx.x & 63; k < a.k; k += 64) {
    const long long word = a.ids[at + k] - a.v0;
    if (word < 0 || word >= words) continue;
    const float q = a.q ? a.q[at + k] : 1.f;
    const float v = f * (exp2_hw(__builtin_fmaf(a.picked[at + k], a.c, -l2)) - q);
    elem_t<T>* const dz = static_cast<elem_t<T>*>(a.dz);
    dz[__is_same(T, Fp32) ? word * a.ldz + r : r * a.ldz + word] = T::from(v);
  }
}

// What becomes of a 16-bit product: fp32 sums of split blockIdx.y (overwritten,
// or added to for later pieces), or the rounded result times scale[0]; transposed,
// so that a lane's neighbouring rows are neighbours in memory.
struct MmOut {
  float* part;          // (splits, N, ldo), or null
  int accumulate;
  unsigned short* out;  // (N, ldo)
  long long ldo;        // M to a multiple of 4; of out, of 8, as M is
  const float* scale;
};

// (16 bytes a lane where fragments stored as they lie, 2 bytes a lane, took 3 to 10%
// more of a whole backward.) Bound by the matrix cores: 8192 x 640 x 32768 dh 417 us
// and dW 394 (824 and 872 TFLOP/s; 640 columns are two and a half tiles), 8192 x 4096
// x 131072 6545 and 6348 (1344 and 1386).
template <class T, class S, bool AK, bool BK>
__global__ void __launch_bounds__(S::kThreads, 2)
head_mm_kernel(MmArgs g, MmOut o) {
  extern __shared__ float lds_f[];
  int tm, tn;
  mm_tile(g, blockIdx.x, tm, tn);
  const int k_first = blockIdx.y * g.kt_per_split * kMmK;
  f32x4 acc[S::FM][S::FN];
  mm_products<T, S, AK, BK>(acc, g, tm * S::BM, tn * S::BN, k_first,
                            min(g.K - k_first, g.kt_per_split * kMmK),
                            reinterpret_cast<char*>(lds_f));
  static_assert(S::FM % 4 == 0, "a lane's 4 rows of 4 fragments");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int mb = tm * S::BM + S::wave_m(wave) * (S::FM * 16);
  const int nb = tn * S::BN + S::wave_n(wave) * (S::FN * 16) + (lane & 15);
  const float scale = o.part ? 1.f : o.scale[0];
#pragma unroll
  for (int j = 0; j < S::FN; ++j) {
    const int n = nb + 16 * j;
    if (o.part) {   // 16 bytes a lane, 64 of 16 rows at a time
      float* const row = o.part + ((long long)blockIdx.y * g.N + n) * o.ldo;
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        const int m = mb + 16 * i + 4 * (lane >> 4);
        if (m >= g.M || n >= g.N) continue;
        f32x4* const p = reinterpret_cast<f32x4*>(row + m);
        const f32x4 v = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        *p = o.accumulate ? *p + v : v;
      }
    } else {        // a lane's 4 rows of 4 fragments become one fragment's 16
#pragma unroll
      for (int h = 0; h < S::FM / 4; ++h) {
        unsigned lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          unsigned short v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = T::from(acc[4 * h + i][j][e] * scale);
          lo[i] = v[0] | (unsigned)v[1] << 16;
          hi[i] = v[2] | (unsigned)v[3] << 16;
        }
        exchange4(lo);
        exchange4(hi);
        const int m = mb + 64 * h + 16 * (lane >> 4);
        unsigned short* const row = o.out + (long long)n * o.ldo + m;
        if (n < g.N && m < g.M)
          *reinterpret_cast<uint4*>(row) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
        if (n < g.N && m + 8 < g.M)
          *reinterpret_cast<uint4*>(row + 8) = make_uint4(lo[2], hi[2], lo[3], hi[3]);
      }
    }
  }
}

// out (M, 4 N4) = scale[0] times the sum of the splits' sums, in order, rounded;
// rows2 given, rows whose coef is 0 are zeros.
template <class T>
__global__ void __launch_bounds__(256)
head_mm_reduce_kernel(const float4* __restrict__ part, ushort4* __restrict__ out,
                      const float* __restrict__ scale, const float2* __restrict__ rows2,
                      int splits, long long M, int N4) {
  const long long n = M * N4;
  const float f = scale[0];
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (long long)gridDim.x * 256) {
    float4 s = part[i];
    for (int k = 1; k < splits; ++k) s = add(s, part[k * n + i]);
    const bool zero = rows2 && rows2[i / N4].x == 0.f;
    out[i] = zero ? make_ushort4(0, 0, 0, 0)
                  : make_ushort4(T::from(s.x * f), T::from(s.y * f), T::from(s.z * f),
                                 T::from(s.w * f));
  }
}

}  // namespace mhs
