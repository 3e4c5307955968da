// C ABI of the head's losses (declared in include/mamba_hip_scan.h): cross
// entropy and distillation from hidden states, distillation of given logits.
//
// Host-side responsibilities as in mhs_capi.hip: argument checks, grids, the
// workspace's layout, the pieces of the vocabulary. No allocation.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mamba_hip_scan.h"
#include "mhs_distill.hpp"
#include "mhs_head.hpp"
#include "mhs_host.hpp"

namespace {

using mhs::aligned16;
using mhs::Bf16;
using mhs::check_launch;
using mhs::device_cus;
using mhs::fail;
using mhs::Fp16;
using mhs::Fp32;
using mhs::round_up;

typedef mhs::MmShape<256, 256, 2, 4> Shape;

// Rows that the kernel for few rows takes, by bytes of an element. us of it and of
// the tiles, with the loss's kernel: fp32, 32 rows, 640 x 32768 36 and 46, 4096 x
// 131072 654 and 702 (its registers hold no more rows); 16 bits, 16 rows, 19 and 25,
// 254 and 236, and one row 17 and 24, 218 and 239; at 32 rows it took 20 and 25, but
// 62 and 54 with 2048 x 50257 and 282 and 239 with 4096 x 131072.
constexpr int64_t small_rows(int elem) { return elem == 4 ? 32 : 16; }
// Bytes of dz that the backward holds at a time (at least 256 words' worth). us
// with 64, 128, 256 and 512 MB: 8192 x 640 x 32768 bf16 1620, 1488, 1446, 1467, fp32
// 7226, 6400, 6126, 6014; 8192 x 4096 x 131072 27300, 26300, 26100, 25970.
constexpr int64_t kPieceBytes = 256LL << 20;
// Rows that one block sums. (us with one block and with blocks of 4096 rows and a
// last one, behind a kernel of one block per row: 4096 rows 32.7 and 34.9, 8192 56.6
// and 57.8, 16384 101.9 and 100.5, 65536 384 and 367.)
constexpr int64_t kLossOneBlock = 8192;

// Blocks of 256 threads that a launch may have: it counts its threads in 32 bits.
constexpr int64_t kMostBlocks = 1LL << 24;

int elem_bytes(int dtype) { return dtype == MHS_F32 ? 4 : 2; }

int check_dtype(int dtype) {
  if (dtype != MHS_F32 && dtype != MHS_BF16 && dtype != MHS_F16)
    return fail(MHS_EINVAL, "dtype must be MHS_F32, MHS_BF16 or MHS_F16; got %d", dtype);
  return MHS_OK;
}

int check_reduction(int reduction) {
  if (reduction != MHS_REDUCE_NONE && reduction != MHS_REDUCE_MEAN && reduction != MHS_REDUCE_SUM)
    return fail(MHS_EINVAL, "reduction must be MHS_REDUCE_NONE, _MEAN or _SUM; got %d", reduction);
  return MHS_OK;
}

// The head's sizes. Rows of hidden and weight are read 16 bytes at a time.
struct Head {
  int dtype;
  int64_t rows, vocab, dim;
  const void* hidden = nullptr;
  const void* weight = nullptr;
  int64_t ldh = 0, ldw = 0;
};

bool few_rows(const Head& p) { return p.rows <= small_rows(elem_bytes(p.dtype)); }

// Tile of the forward's fp32 product. (us with 64 and 128, 64 rows: 640 x 32768 40
// and 48, 4096 x 131072 689 and 748; 96 rows: 54 and 48, 1050 and 797.)
int gemm3_tile(int64_t rows) { return rows <= 64 ? mhs::kGemmSmallTile : mhs::kGemmTile; }

int check_sizes(const Head& p) {
  int rc = check_dtype(p.dtype);
  if (rc) return rc;
  if (p.rows < 0 || p.vocab < 1 || p.dim < 1 || p.rows > (1LL << 30) || p.vocab > (1LL << 30))
    return fail(MHS_EINVAL, "rows must be in [0, 2^30], vocab in [1, 2^30], dim >= 1; got %lld, "
                "%lld, %lld", (long long)p.rows, (long long)p.vocab, (long long)p.dim);
  const int v = 16 / elem_bytes(p.dtype);
  if (p.dim % v || p.dim > (1LL << 20))
    return fail(MHS_EINVAL, "dim must be a multiple of %d up to 2^20; got %lld", v,
                (long long)p.dim);
  // The forward's product, a block per tile (16 bits: tiles counted in an int), and
  // the rows' kernels, a wave per row.
  const int t = few_rows(p) ? mhs::kSmallWords : gemm3_tile(p.rows);
  const int64_t tiles = ((p.vocab + t - 1) / t) * (few_rows(p) ? 1 : (p.rows + t - 1) / t);
  const bool streamed = p.dtype != MHS_F32 && !few_rows(p);
  const bool fits = streamed ? ((p.vocab + 63) / 64) * ((p.rows + 63) / 64) <= 0x7FFFFFFF
                             : tiles < kMostBlocks;
  if (!fits || (p.rows + 3) / 4 >= kMostBlocks)
    return fail(MHS_EINVAL, "%lld rows x %lld words is too large", (long long)p.rows,
                (long long)p.vocab);
  return MHS_OK;
}

// Distillation takes a block per row.
int check_block_rows(int64_t rows) {
  if (rows < 0 || rows >= kMostBlocks)
    return fail(MHS_EINVAL, "distillation takes rows in [0, 2^24); got %lld", (long long)rows);
  return MHS_OK;
}

int check_head(const Head& p) {
  int rc = check_sizes(p);
  if (rc) return rc;
  if (!p.weight || (p.rows > 0 && !p.hidden)) return fail(MHS_EINVAL, "null pointer argument");
  const int v = 16 / elem_bytes(p.dtype);
  for (const int64_t ld : {p.ldh, p.ldw})
    if (ld < p.dim || ld % v || ld >= (1LL << 21))
      return fail(MHS_EINVAL, "row strides must be multiples of %d, at least dim and below 2^21; "
                  "got %lld", v, (long long)ld);
  if (!aligned16(p.hidden) || !aligned16(p.weight))
    return fail(MHS_EINVAL, "hidden and weight must be 16-byte aligned");
  return MHS_OK;
}

int check_top(int64_t top, float temperature) {
  if (top < 1 || top > mhs::kMaxTop)
    return fail(MHS_EINVAL, "the teacher's words per row must be in [1, %d]; got %lld",
                mhs::kMaxTop, (long long)top);
  if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(1.f / temperature))
    return fail(MHS_EINVAL, "temperature must be positive and finite; got %g", temperature);
  return MHS_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return fail(MHS_EINVAL, "workspace too small: %zu < %zu bytes", have, need);
  if (need && (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(MHS_EINVAL, "workspace must be 256-byte aligned");
  return MHS_OK;
}

// ----------------------------------------------------------------- forward

// Splits of a 16-bit forward's product in k: 1 where the tiles' own kernel takes
// it whole. A k tile takes 1.07 us of a block (the direct kernel's blocks wait for
// each: it has one per CU), the sums' kernel 5 us, and a split's sums are written
// and read at 7.5 TB/s, from the caches. With tiles for more than a quarter of the
// CUs W's bytes count instead. (us, whole and split: 33 x 1024 x 1360 30 and 17,
// 64 x 4096 x 16384 81 and 39, 256 x 2048 x 8192 48 and 37; not split, 256 x 512 x
// 16384 21 and 33, 512 x 1024 x 16384 33 and 45, 512 x 4096 x 24576 93 and 117.)
struct KSplit {
  int splits, kt_per_split;
};
KSplit lse_splits(const Head& p) {
  const int64_t tiles = (p.vocab + Shape::BM - 1) / Shape::BM *
                        ((p.rows + Shape::BN - 1) / Shape::BN);
  const int kt = (int)((p.dim + mhs::kMmK - 1) / mhs::kMmK);
  KSplit best{1, kt};
  if (4 * tiles > device_cus()) return best;
  double least = 1.07 * kt;
  for (int n = 2; n <= std::min<int64_t>(device_cus() / std::max<int64_t>(tiles, 1), kt / 4); ++n) {
    const int per = (kt + n - 1) / n;
    const double us = 1.07 * per + 5 + n * (double)p.rows * p.vocab * 8 / 7.5e6;
    if (us >= least) continue;
    least = us;
    best.kt_per_split = per;
    best.splits = (kt + per - 1) / per;
  }
  return best;
}

// Whether a forward's tiles are so few, and its k's so many, that its product is
// taken by itself, cut up in k, and the sums of exponentials from the logits in
// memory. fp32 (us, tiles' own kernel and so): 33 x 640 x 1360, 22 tiles, 26 and 21,
// 128 x 640 x 8192, 64 tiles, 37 and 36, 256 x 640 x 8192, 128, 39 and 43; with 2896
// columns 89 and 30, 161 and 67, 160 and 104, and 256 x 16384, 256 tiles, 170 and
// 178; with 256 columns 15 and 22, 20 and 24, 21 and 29.
bool few_tiles(const Head& p) {
  if (few_rows(p) || p.rows == 0) return false;
  if (p.dtype != MHS_F32) return lse_splits(p).splits > 1;
  const int t = gemm3_tile(p.rows);
  const int64_t tiles = ((p.vocab + t - 1) / t) * ((p.rows + t - 1) / t);
  return p.dim >= 512 && tiles <= std::min<int64_t>(p.dim / 10, device_cus() / 2);
}

// Tiles of the vocabulary in the forward's partials.
int64_t lse_tiles(const Head& p) {
  static_assert(mhs::kSmallWords == mhs::kLogitWords, "one size of partials");
  static_assert(mhs::kSplitWords == Shape::BM, "and of 16 bits");
  if (few_rows(p) || (p.dtype == MHS_F32 && few_tiles(p)))
    return (p.vocab + mhs::kSmallWords - 1) / mhs::kSmallWords;
  const int bm = p.dtype == MHS_F32 ? gemm3_tile(p.rows) : Shape::BM;
  return (p.vocab + bm - 1) / bm;
}

size_t loss_ws(int64_t rows) {
  return rows <= kLossOneBlock
             ? 0
             : round_up((size_t)((rows + mhs::kLossRows - 1) / mhs::kLossRows) * 16, 256);
}

// The forward's workspace: partials, the loss's sums and, of few tiles, the logits
// and the product's own.
size_t logits_at(const Head& p) {
  return round_up((size_t)lse_tiles(p) * p.rows * 8, 256) + loss_ws(p.rows);
}

size_t gemm_ws(int64_t m, int64_t n, int64_t k) {
  return (size_t)std::max<int64_t>(mhs_gemm_workspace_bytes(m, n, k), 0);
}

size_t logits_bytes(const Head& p) {
  return round_up(p.dtype == MHS_F32 ? (size_t)p.vocab * round_up(p.rows, 4) * 4
                                     : (size_t)p.rows * round_up(p.vocab, 4) * 4, 256);
}

size_t fwd_ws(const Head& p) {
  if (!few_tiles(p)) return logits_at(p);
  if (p.dtype != MHS_F32) return logits_at(p) + lse_splits(p).splits * logits_bytes(p);
  return logits_at(p) + logits_bytes(p) +
         gemm_ws(p.vocab, p.rows, p.dim);
}

template <class F>
void allow_lds(F* fn, int bytes) {
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(fn),
                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// Tiles in m per group of the block order (mm_tile). (us of the loss and its
// gradients with 1, 2, 4, 8 and 16, bf16: 8192 x 640 x 32768 1633, 1485, 1473, 1506,
// 1539; 8192 x 4096 x 131072 28090, 26580, 26120, 26520, 27210.)
constexpr int kGroupM = 4;

template <class S>
mhs::MmArgs mm_args(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t N,
                    int64_t K) {
  mhs::MmArgs g;
  g.A = a;
  g.B = b;
  g.lda = lda;
  g.ldb = ldb;
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.kt_per_split = (int)((K + mhs::kMmK - 1) / mhs::kMmK);
  g.grid_m = (int)((M + S::BM - 1) / S::BM);
  g.grid_n = (int)((N + S::BN - 1) / S::BN);
  g.group_m = kGroupM;
  return g;
}

// Blocks of a streamed product: as many as run at once (one per CU).
unsigned stream_blocks(const mhs::MmArgs& g) {
  return (unsigned)std::min<int64_t>((int64_t)g.grid_m * g.grid_n, device_cus());
}

// The logits' product for fp32: W (v0 .. v0 + words) h^T.
mhs::GemmArgs gemm3_args(const Head& p, int64_t v0, int64_t words, int tile) {
  mhs::GemmArgs g{};
  g.A = static_cast<const float*>(p.weight) + v0 * p.ldw;
  g.B = static_cast<const float*>(p.hidden);
  g.lda = p.ldw;
  g.ldb = p.ldh;
  g.M = (int)words;
  g.N = (int)p.rows;
  g.K = (int)p.dim;
  g.grid_m = (int)((words + tile - 1) / tile);
  g.grid_n = (int)((p.rows + tile - 1) / tile);
  return g;
}

// The kept logits' rows: of words of 16-bit operands, of rows of fp32 ones.
mhs::KeptLogits kept_logits(const Head& p, float* z) {
  return {z, (long long)round_up(p.dtype == MHS_F32 ? p.rows : p.vocab, 4)};
}

template <class T>
int launch_lse16(const Head& p, float c, float2* part, const mhs::KeptLogits& kept,
                 hipStream_t s) {
  const mhs::MmArgs g = mm_args<Shape>(p.weight, p.ldw, p.hidden, p.ldh, p.vocab, p.rows, p.dim);
  const auto fn = kept.z ? &mhs::head_lse_kernel<T, Shape, true>
                         : &mhs::head_lse_kernel<T, Shape, false>;
  constexpr int lds = Shape::kLds + 2 * Shape::WM * Shape::BN * 4;
  allow_lds(fn, lds);
  hipLaunchKernelGGL(fn, dim3(stream_blocks(g)), dim3(Shape::kThreads), lds, s, g, c, part,
                     kept);
  return check_launch("head log-sum-exp kernel");
}

template <class T>
int launch_small(const Head& p, float c, float2* part, const mhs::KeptLogits& kept,
                 hipStream_t s) {
  const mhs::SmallArgs g{p.hidden, p.weight, p.ldh, p.ldw, (int)p.rows, (int)p.vocab, (int)p.dim};
  auto fn = &mhs::head_small_kernel<T, 1>;
  if constexpr (small_rows(sizeof(mhs::elem_t<T>)) > 16)
    if (p.rows > 16) fn = &mhs::head_small_kernel<T, 2>;
  hipLaunchKernelGGL(fn, dim3((unsigned)lse_tiles(p)), dim3(256), 0, s, g, c, part, kept);
  return check_launch("head log-sum-exp kernel of few rows");
}

// Of few tiles: the logits (to kept, or the workspace) and their sums.
int launch_lse_of_logits(const Head& p, float c, mhs::KeptLogits kept, char* ws, hipStream_t s) {
  float2* part = reinterpret_cast<float2*>(ws);
  if (!kept.z) kept.z = reinterpret_cast<float*>(ws + logits_at(p));
  const size_t at = logits_at(p) + logits_bytes(p);
  int rc = mhs::gemm_f32(MHS_GEMM_NT, static_cast<const float*>(p.weight), p.ldw,
                         static_cast<const float*>(p.hidden), p.ldh, kept.z, kept.ld, p.vocab,
                         p.rows, p.dim, 0, nullptr, ws + at, fwd_ws(p) - at, s);
  if (rc) return rc;
  hipLaunchKernelGGL(mhs::head_lse_of_logits_kernel<>,
                     dim3((unsigned)lse_tiles(p), (unsigned)((p.rows + 63) / 64)), dim3(256), 0, s,
                     kept, (int)p.vocab, (int)p.rows, c, part);
  return check_launch("log-sum-exp of logits kernel");
}

template <class T>
int launch_lse_of_splits(const Head& p, float c, const mhs::KeptLogits& kept, char* ws,
                         hipStream_t s) {
  mhs::MmArgs g = mm_args<Shape>(p.weight, p.ldw, p.hidden, p.ldh, p.vocab, p.rows, p.dim);
  const KSplit k = lse_splits(p);
  g.kt_per_split = k.kt_per_split;
  mhs::MmOut o{};
  o.part = reinterpret_cast<float*>(ws + logits_at(p));
  o.ldo = (long long)round_up(p.vocab, 4);
  const auto fn = &mhs::head_mm_kernel<T, Shape, true, true>;
  allow_lds(fn, Shape::kLds);
  hipLaunchKernelGGL(fn, dim3((unsigned)(g.grid_m * g.grid_n), (unsigned)k.splits),
                     dim3(Shape::kThreads), Shape::kLds, s, g, o);
  int rc = check_launch("logits kernel");
  if (rc) return rc;
  hipLaunchKernelGGL(mhs::head_lse_of_splits_kernel<>,
                     dim3((unsigned)lse_tiles(p), (unsigned)((p.rows + 3) / 4)), dim3(256), 0, s,
                     o.part, o.ldo, k.splits, (int)p.vocab, (int)p.rows, c,
                     reinterpret_cast<float2*>(ws), kept);
  return check_launch("log-sum-exp of logits kernel");
}

int launch_lse(const Head& p, float c, char* ws, const mhs::KeptLogits& kept, hipStream_t s) {
  float2* part = reinterpret_cast<float2*>(ws);
  if (few_tiles(p))
    return p.dtype == MHS_F32    ? launch_lse_of_logits(p, c, kept, ws, s)
           : p.dtype == MHS_BF16 ? launch_lse_of_splits<Bf16>(p, c, kept, ws, s)
                                 : launch_lse_of_splits<Fp16>(p, c, kept, ws, s);
  if (few_rows(p))
    return p.dtype == MHS_F32    ? launch_small<Fp32>(p, c, part, kept, s)
           : p.dtype == MHS_BF16 ? launch_small<Bf16>(p, c, part, kept, s)
                                 : launch_small<Fp16>(p, c, part, kept, s);
  if (p.dtype == MHS_BF16) return launch_lse16<Bf16>(p, c, part, kept, s);
  if (p.dtype == MHS_F16) return launch_lse16<Fp16>(p, c, part, kept, s);
  const int tile = gemm3_tile(p.rows);
  const mhs::GemmArgs g = gemm3_args(p, 0, p.vocab, tile);
  hipLaunchKernelGGL((tile == mhs::kGemmTile ? &mhs::head_lse3_kernel<mhs::kGemmTile>
                                             : &mhs::head_lse3_kernel<mhs::kGemmSmallTile>),
                     dim3((unsigned)g.grid_m * (unsigned)g.grid_n), dim3(mhs::kGemmThreads),
                     mhs::gemm_lds_bytes(tile, tile), s, g, c, part, kept);
  return check_launch("head log-sum-exp kernel");
}

// loss[0] and count[0] from the rows' losses.
int launch_loss(const float* rows_loss, const float* keep, float* loss, float* count, int64_t rows,
                int reduction, void* ws, hipStream_t s) {
  const int mean = reduction == MHS_REDUCE_MEAN;
  if (rows <= kLossOneBlock) {
    hipLaunchKernelGGL(mhs::head_loss_kernel<>, dim3(1), dim3(mhs::kLossThreads), 0, s, rows_loss,
                       keep, static_cast<const double2*>(nullptr), static_cast<double2*>(nullptr),
                       loss, count, (long long)rows, mean);
    return check_launch("loss kernel");
  }
  const int64_t blocks = (rows + mhs::kLossRows - 1) / mhs::kLossRows;
  double2* sums = static_cast<double2*>(ws);
  hipLaunchKernelGGL(mhs::head_loss_kernel<>, dim3((unsigned)blocks), dim3(mhs::kLossThreads), 0, s,
                     rows_loss, keep, static_cast<const double2*>(nullptr), sums, loss, count,
                     (long long)rows, mean);
  int rc = check_launch("loss kernel");
  if (rc) return rc;
  hipLaunchKernelGGL(mhs::head_loss_kernel<>, dim3(1), dim3(mhs::kLossThreads), 0, s, rows_loss,
                     keep, static_cast<const double2*>(sums), static_cast<double2*>(nullptr), loss,
                     count, (long long)blocks, mean);
  return check_launch("loss kernel");
}

// Rows up to which each takes a block of the rows' kernel, then a wave. (us of the
// forward with a block and with a wave, 640 x 32768 bf16: 16 rows 16.5 and 18.9,
// 512 28.3 and 28.4, 1024 48.1 and 46.8, 8192 320 and 312; 4 rows of 4096 x 131072
// 213 and 227.)
constexpr int64_t kBlockRows = 512;

template <class T>
int launch_rows(const mhs::HeadRows& g, hipStream_t s) {
  if (g.teacher)
    hipLaunchKernelGGL(mhs::head_distill_rows_kernel<T>, dim3((unsigned)g.rows), dim3(256),
                       2 * g.k * sizeof(float), s, g);
  else if (g.rows <= kBlockRows)
    hipLaunchKernelGGL((mhs::head_xent_rows_kernel<T, 4>), dim3((unsigned)g.rows), dim3(256), 0, s,
                       g);
  else
    hipLaunchKernelGGL((mhs::head_xent_rows_kernel<T, 1>), dim3((unsigned)((g.rows + 3) / 4)),
                       dim3(256), 0, s, g);
  return check_launch("head rows kernel");
}

// The forward from the hidden states: g's ids, teacher and outputs are set.
int head_fwd(const Head& p, mhs::HeadRows g, float* logits, float* loss, float* count,
             int reduction, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_workspace(workspace, workspace_bytes, fwd_ws(p));
  if (rc) return rc;
  if (reduction != MHS_REDUCE_NONE && (!loss || !count))
    return fail(MHS_EINVAL, "null pointer argument");
  if (!aligned16(logits)) return fail(MHS_EINVAL, "logits must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  float2* part = static_cast<float2*>(workspace);
  if (p.rows > 0) {
    if (!g.ids || !g.lse2 || !g.picked || !g.loss || !g.keep)
      return fail(MHS_EINVAL, "null pointer argument");
    rc = launch_lse(p, mhs::kLog2e / g.temperature, static_cast<char*>(workspace),
                    kept_logits(p, logits), s);
    if (rc) return rc;
    g.h = p.hidden;
    g.w = p.weight;
    g.ldh = p.ldh;
    g.ldw = p.ldw;
    g.part = part;
    g.kept = kept_logits(p, logits);
    g.rows = (int)p.rows;
    g.vocab = (int)p.vocab;
    g.dim = (int)p.dim;
    g.tiles = (int)lse_tiles(p);
    rc = p.dtype == MHS_F32    ? launch_rows<Fp32>(g, s)
         : p.dtype == MHS_BF16 ? launch_rows<Bf16>(g, s)
                               : launch_rows<Fp16>(g, s);
    if (rc) return rc;
  }
  if (reduction == MHS_REDUCE_NONE) return MHS_OK;
  return launch_loss(g.loss, g.keep, loss, count, p.rows, reduction,
                     static_cast<char*>(workspace) +
                         round_up((size_t)lse_tiles(p) * p.rows * 8, 256),
                     s);
}

// ---------------------------------------------------------------- backward

// Where things lie in the backward's workspace, and how it is cut up.
struct BwdPlan {
  int64_t piece, ldz;      // words per piece; dz's row stride
  int64_t rows4;           // fp32: the rows, to a multiple of 4
  KSplit dh, dw;           // 16 bits: of dh's sums over a piece's words, dW's over the rows
  size_t rows2, hidden, dz, part, part_w, bytes;
};

int64_t piece_words(int64_t rows, int64_t vocab, int es) {
  const int64_t fit = kPieceBytes / (std::max<int64_t>(rows, 1) * es) / 256 * 256;
  return std::min(round_up(vocab, 256), (size_t)std::max<int64_t>(fit, 256));
}

// Splits of a product (M, N) over K in its k's, such that its tiles fill the CUs:
// a k tile takes 1.5 us of a CU, a block's start and end about 4 more, and the sums
// of a split are written and read at about 4 TB/s; whole: 1 if one split's sums go
// through memory too. (dh, 1001 x 384 x 16384, us: 4 splits 80, 16 35, 32 32; 8192 x
// 640 x 16384: 2 splits 182, 5 206. dW split and whole, the loss and its gradients:
// 8192 x 64 x 1009 84 and 172, 8192 x 640 x 8192 400 and 413, 8192 x 64 x 32768 519
// and 680, 4096 x 640 x 16384 372 and 366; whole by this, 8192 x 1024 x 32768.)
KSplit bwd_splits(int64_t M, int64_t N, int64_t K, int whole) {
  const int64_t tiles = (M + Shape::BM - 1) / Shape::BM * ((N + Shape::BN - 1) / Shape::BN);
  const int64_t kt = (K + mhs::kMmK - 1) / mhs::kMmK;
  const int cus = device_cus();
  KSplit b{};
  double best = 0;
  for (int64_t n = 1; n <= std::min<int64_t>(64, kt); ++n) {
    const double t = std::ceil((double)tiles * n / cus) * 1.5 * ((double)((kt + n - 1) / n) + 4) +
                     (n > 1 || whole ? n * (double)M * N * 8 / 4e6 : 0) + (n > 1 && !whole ? 5 : 0);
    if (n > 1 && t >= best) continue;
    best = t;
    b.kt_per_split = (int)((kt + n - 1) / n);
  }
  b.splits = (int)((kt + b.kt_per_split - 1) / b.kt_per_split);
  return b;
}

BwdPlan bwd_plan(const Head& p) {
  BwdPlan b;
  const int es = elem_bytes(p.dtype);
  b.piece = std::min<int64_t>(piece_words(p.rows, p.vocab, es), 1 << 20);
  b.rows4 = p.dtype == MHS_F32 ? (int64_t)round_up(p.rows, 4) : p.rows;
  b.ldz = p.dtype == MHS_F32 ? b.rows4 : b.piece;
  b.rows2 = 256;
  b.hidden = b.rows2 + round_up((size_t)(p.rows + 1) * 8, 256);
  b.dz = b.hidden + round_up((size_t)b.rows4 * p.dim * es, 256);
  b.part = b.dz + round_up((size_t)(p.dtype == MHS_F32 ? b.piece * b.rows4 : p.rows * b.piece) * es,
                           256);
  size_t part, part_w = 0;
  if (p.dtype == MHS_F32) {
    const int64_t words = std::min(b.piece, p.vocab);
    // (the last piece may be shorter, and its products' splits other ones)
    const int64_t last = p.vocab % b.piece ? p.vocab % b.piece : words;
    part = 0;
    for (const int64_t w : {words, last})
      part = std::max({part, gemm_ws(p.rows, p.dim, w), gemm_ws(w, p.dim, b.rows4)});
  } else {
    const int64_t words = std::min(b.piece, p.vocab);
    b.dh = bwd_splits(p.dim, p.rows, words, 1);
    b.dw = bwd_splits(p.dim, words, p.rows, 0);
    part = (size_t)b.dh.splits * p.rows * p.dim * 4;
    if (b.dw.splits > 1) part_w = (size_t)b.dw.splits * words * p.dim * 4;
  }
  b.part_w = b.part + round_up(part, 256);
  b.bytes = b.part_w + round_up(part_w, 256);
  return b;
}

size_t bwd_ws(const Head& p) { return p.rows == 0 ? 0 : bwd_plan(p).bytes; }

struct BwdOut {
  void* dhidden;   // (rows, dim), or null
  void* dweight;   // (vocab, dim), or null
};

template <class T>
int launch_ids(const Head& p, const mhs::HeadGrad& a, int64_t words, hipStream_t s) {
  hipLaunchKernelGGL(mhs::head_ids_kernel<T>, dim3((unsigned)((p.rows + 3) / 4)), dim3(256), 0, s,
                     a, (long long)p.rows, (int)words);
  return check_launch("gradient of the ids kernel");
}

// p's part of dz of a piece from the kept logits.
template <class T>
int launch_dz_kept(const Head& p, const mhs::KeptLogits& kept, const mhs::HeadGrad& a,
                   int64_t words, hipStream_t s) {
  const bool f32 = p.dtype == MHS_F32;
  const int64_t v = 16 / elem_bytes(p.dtype);
  const int64_t blocks = ((f32 ? p.rows : words) + v - 1) / v;
  const int64_t n = blocks * (f32 ? words : p.rows);
  hipLaunchKernelGGL(mhs::head_dz_kept_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0,
                     s, kept, a, (int)p.rows, (int)words, (unsigned)blocks, (long long)n);
  return check_launch("gradient of kept logits kernel");
}

// out (rows, cols) of the splits' sums (head_mm_reduce_kernel).
template <class T>
int launch_reduce(const float* part, void* out, const float* scale, const float2* rows2,
                  int splits, int64_t rows, int64_t cols, hipStream_t s) {
  const int64_t n = rows * cols / 4;
  hipLaunchKernelGGL(mhs::head_mm_reduce_kernel<T>,
                     dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096)), dim3(256), 0, s,
                     reinterpret_cast<const float4*>(part), static_cast<ushort4*>(out), scale,
                     rows2, splits, (long long)rows, (int)(cols / 4));
  return check_launch("gradient reduction kernel");
}

template <class T>
int bwd16(const Head& p, const BwdPlan& b, mhs::HeadGrad a, const mhs::KeptLogits& kept,
          const BwdOut& out, char* ws, hipStream_t s) {
  const auto fz = &mhs::head_dz_kernel<T, Shape>;
  const auto fh = &mhs::head_mm_kernel<T, Shape, false, true>;
  const auto fw = &mhs::head_mm_kernel<T, Shape, false, false>;
  constexpr int lds_z = Shape::kLds + mhs::kMmSlots * mhs::kPairBytes;
  allow_lds(fz, lds_z);
  allow_lds(fh, Shape::kLds);
  allow_lds(fw, Shape::kLds);
  typedef unsigned short u16;
  const u16* w = static_cast<const u16*>(p.weight);
  u16* hz = reinterpret_cast<u16*>(ws + b.hidden);
  float* part = reinterpret_cast<float*>(ws + b.part);
  int rc;
  for (int64_t v0 = 0; v0 < p.vocab; v0 += b.piece) {
    const int64_t words = std::min(b.piece, p.vocab - v0);
    mhs::MmArgs g = mm_args<Shape>(w + v0 * p.ldw, p.ldw, p.hidden, p.ldh, words, p.rows, p.dim);
    a.v0 = (int)v0;
    if (kept.z) {
      rc = launch_dz_kept<T>(p, kept, a, words, s);
    } else {
      hipLaunchKernelGGL(fz, dim3(stream_blocks(g)), dim3(Shape::kThreads), lds_z, s, g, a);
      rc = check_launch("head gradient kernel");
    }
    if (rc) return rc;
    if ((rc = launch_ids<T>(p, a, words, s)) != 0) return rc;
    mhs::MmOut o{};
    o.scale = a.scale;
    if (out.dhidden) {
      g = mm_args<Shape>(w + v0 * p.ldw, p.ldw, a.dz, b.ldz, p.dim, p.rows, words);
      g.kt_per_split = b.dh.kt_per_split;
      o.part = part;
      o.ldo = p.dim;
      o.accumulate = v0 > 0;
      hipLaunchKernelGGL(fh, dim3((unsigned)(g.grid_m * g.grid_n), (unsigned)b.dh.splits),
                         dim3(Shape::kThreads), Shape::kLds, s, g, o);
      if ((rc = check_launch("hidden gradient kernel")) != 0) return rc;
    }
    if (out.dweight) {
      g = mm_args<Shape>(hz, p.dim, a.dz, b.ldz, p.dim, words, p.rows);
      g.kt_per_split = b.dw.kt_per_split;
      o.part = b.dw.splits > 1 ? reinterpret_cast<float*>(ws + b.part_w) : nullptr;
      o.accumulate = 0;
      o.out = static_cast<u16*>(out.dweight) + v0 * p.dim;
      o.ldo = p.dim;
      hipLaunchKernelGGL(fw, dim3((unsigned)(g.grid_m * g.grid_n), (unsigned)b.dw.splits),
                         dim3(Shape::kThreads), Shape::kLds, s, g, o);
      if ((rc = check_launch("weight gradient kernel")) != 0) return rc;
      if (o.part && (rc = launch_reduce<T>(o.part, o.out, a.scale, nullptr, b.dw.splits, words,
                                           p.dim, s)) != 0)
        return rc;
    }
  }
  if (out.dhidden)
    return launch_reduce<T>(part, out.dhidden, a.scale, a.rows2, b.dh.splits, p.rows, p.dim, s);
  return MHS_OK;
}

int bwd32(const Head& p, const BwdPlan& b, mhs::HeadGrad a, const mhs::KeptLogits& kept,
          const BwdOut& out, char* ws, hipStream_t s) {
  const float* w = static_cast<const float*>(p.weight);
  const float* hz = reinterpret_cast<const float*>(ws + b.hidden);
  float* dz = static_cast<float*>(a.dz);
  void* part = ws + b.part;
  const size_t part_bytes = b.bytes - b.part;
  int rc;
  for (int64_t v0 = 0; v0 < p.vocab; v0 += b.piece) {
    const int64_t words = std::min(b.piece, p.vocab - v0);
    const mhs::GemmArgs g = gemm3_args(p, v0, words, mhs::kGemmTile);
    a.v0 = (int)v0;
    if (kept.z) {
      rc = launch_dz_kept<Fp32>(p, kept, a, words, s);
    } else {
      hipLaunchKernelGGL(mhs::head_dz3_kernel<mhs::kGemmTile>,
                         dim3((unsigned)g.grid_m * (unsigned)g.grid_n), dim3(mhs::kGemmThreads),
                         mhs::gemm_lds_bytes(mhs::kGemmTile, mhs::kGemmTile), s, g, a);
      rc = check_launch("head gradient kernel");
    }
    if (rc) return rc;
    if ((rc = launch_ids<Fp32>(p, a, words, s)) != 0) return rc;
    if (out.dhidden &&
        (rc = mhs::gemm_f32(MHS_GEMM_TN, dz, b.ldz, w + v0 * p.ldw, p.ldw,
                            static_cast<float*>(out.dhidden), p.dim, p.rows, p.dim, words, v0 > 0,
                            a.scale, part, part_bytes, s)) != 0)
      return rc;
    if (out.dweight &&
        (rc = mhs::gemm_f32(MHS_GEMM_NN, dz, b.ldz, hz, p.dim,
                            static_cast<float*>(out.dweight) + v0 * p.dim, p.dim, words, p.dim,
                            b.rows4, 0, a.scale, part, part_bytes, s)) != 0)
      return rc;
  }
  if (!out.dhidden) return MHS_OK;
  hipLaunchKernelGGL(mhs::head_zero_rows_kernel<>, dim3((unsigned)((p.rows + 3) / 4)), dim3(256), 0,
                     s, a.rows2, static_cast<float4*>(out.dhidden), (long long)p.rows,
                     (int)(p.dim / 4));
  return check_launch("zero rows kernel");
}

// See lift_of.
int lift(int dtype) { return dtype == MHS_F16 ? 15 : dtype == MHS_F32 ? 32 : 0; }

// The rows' coefficients, the scale and (hidden given) the copy of the rows.
int launch_rows_in(const Head& p, const BwdPlan& b, const mhs::RowScale& rs, const float* lse2,
                   float2* rows2, float* scale, void* hidden, hipStream_t s) {
  const int64_t es = elem_bytes(p.dtype);
  // (rows2 has an even number of rows, hidden rows4)
  const int64_t out_rows = std::max<int64_t>(b.rows4, (int64_t)round_up(p.rows, 2));
  const int64_t blocks = (out_rows + mhs::kCopyRows - 1) / mhs::kCopyRows;
  hipLaunchKernelGGL(mhs::head_rows_in_kernel<>, dim3((unsigned)blocks), dim3(256), 0, s,
                     static_cast<const uint4*>(p.hidden), (long long)(p.ldh * es / 16), rs, lse2,
                     rows2, scale, static_cast<uint4*>(hidden), (long long)p.rows,
                     (long long)b.rows4, (int)(p.dim * es / 16), lift(p.dtype));
  return check_launch("rows kernel");
}

// zeros: a gradient that no row reaches.
int launch_zero(void* p, int64_t n, int es, hipStream_t s) {
  const int64_t words = n * es / 4;   // (dim is a multiple of 16 bytes)
  hipLaunchKernelGGL(mhs::head_zero_kernel<>,
                     dim3((unsigned)std::min<int64_t>((words + 255) / 256, 4096)), dim3(256), 0, s,
                     static_cast<unsigned*>(p), (long long)words);
  return check_launch("zero fill kernel");
}

int head_bwd(const Head& p, mhs::HeadGrad a, mhs::RowScale rs, const float* lse2,
             const float* logits, const BwdOut& out, void* workspace, size_t workspace_bytes,
             void* stream) {
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int es = elem_bytes(p.dtype);
  if (out.dhidden == nullptr && out.dweight == nullptr) return MHS_OK;
  if (p.rows == 0) return out.dweight ? launch_zero(out.dweight, p.vocab * p.dim, es, s) : MHS_OK;
  if (!a.ids || !lse2 || !a.picked || !rs.keep || !rs.upstream)
    return fail(MHS_EINVAL, "null pointer argument");
  if (!aligned16(out.dhidden) || !aligned16(out.dweight) || !aligned16(logits))
    return fail(MHS_EINVAL, "dhidden, dweight and logits must be 16-byte aligned");
  if (p.dtype == MHS_F32 && p.rows > (1LL << 22) - 4)   // (dz's row stride)
    return fail(MHS_EINVAL, "the fp32 backward takes rows below 2^22; got %lld", (long long)p.rows);
  int rc = check_workspace(workspace, workspace_bytes, bwd_ws(p));
  if (rc) return rc;
  const BwdPlan b = bwd_plan(p);
  char* ws = static_cast<char*>(workspace);
  float* scale = reinterpret_cast<float*>(ws);
  float2* rows2 = reinterpret_cast<float2*>(ws + b.rows2);
  if (lift(p.dtype) && rs.per_row) {
    hipLaunchKernelGGL(mhs::head_largest_kernel<>, dim3(1), dim3(1024), 0, s, rs, scale + 2,
                       (long long)p.rows);
    if ((rc = check_launch("largest gradient kernel")) != 0) return rc;
  }
  rc = launch_rows_in(p, b, rs, lse2, rows2, scale, out.dweight ? ws + b.hidden : nullptr, s);
  if (rc) return rc;
  a.rows2 = rows2;
  a.scale = scale;
  a.dz = ws + b.dz;
  a.ldz = b.ldz;
  const mhs::KeptLogits kept = kept_logits(p, const_cast<float*>(logits));   // (only read)
  return p.dtype == MHS_F32    ? bwd32(p, b, a, kept, out, ws, s)
         : p.dtype == MHS_BF16 ? bwd16<Bf16>(p, b, a, kept, out, ws, s)
                               : bwd16<Fp16>(p, b, a, kept, out, ws, s);
}

mhs::RowScale row_scale(const float* upstream, const float* count, const float* keep, int reduction,
                        float factor) {
  mhs::RowScale rs;
  rs.upstream = upstream;
  rs.count = reduction == MHS_REDUCE_MEAN ? count : nullptr;
  rs.keep = keep;
  rs.per_row = reduction == MHS_REDUCE_NONE;
  rs.factor = factor;
  return rs;
}

Head head_of(int dtype, const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
             int64_t rows, int64_t vocab, int64_t dim) {
  Head p;
  p.dtype = dtype;
  p.rows = rows;
  p.vocab = vocab;
  p.dim = dim;
  p.hidden = hidden;
  p.weight = weight;
  p.ldh = ldh;
  p.ldw = ldw;
  return p;
}

const long long* ll(const int64_t* p) { return reinterpret_cast<const long long*>(p); }

template <class T>
int launch_distill_bwd(const void* logits, int64_t ld, const int64_t* ids, const float* q,
                       const float* lse2, const mhs::RowScale& rs, void* dlogits, int64_t rows,
                       int64_t vocab, int64_t top, float c, hipStream_t s) {
  hipLaunchKernelGGL(mhs::distill_bwd_kernel<T>, dim3((unsigned)rows), dim3(mhs::kXentThreads), 0,
                     s, static_cast<const mhs::elem_t<T>*>(logits), (long long)ld, ll(ids), q,
                     lse2, rs, static_cast<mhs::elem_t<T>*>(dlogits), (long long)vocab, (int)top,
                     c);
  return check_launch("distillation backward kernel");
}

int check_logits(int dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab,
                 int64_t top, float temperature, int reduction) {
  int rc = check_dtype(dtype);
  if (rc || (rc = check_reduction(reduction)) || (rc = check_top(top, temperature)) ||
      (rc = check_block_rows(rows)))
    return rc;
  if (vocab < 1 || vocab > 0x7FFFFFFF || ld < vocab)
    return fail(MHS_EINVAL, "vocab must be in [1, 2^31) and the row stride at least vocab; got "
                "%lld, %lld", (long long)vocab, (long long)ld);
  if (rows > 0 && !logits) return fail(MHS_EINVAL, "null pointer argument");
  if (reinterpret_cast<uintptr_t>(logits) % elem_bytes(dtype))
    return fail(MHS_EINVAL, "logits must be aligned to their elements");
  return MHS_OK;
}

}  // namespace

extern "C" {

size_t mhs_linear_xent_fwd_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int64_t dim) {
  mhs::clear_error();
  const Head p = head_of(dtype, nullptr, dim, nullptr, dim, rows, vocab, dim);
  return check_sizes(p) ? 0 : std::max(fwd_ws(p), (size_t)256);
}

int mhs_linear_xent_fwd(int dtype, const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                        const int64_t* targets, float* lse2, float* picked, float* keep,
                        float* logits, float* loss_rows, float* loss, float* count, int64_t rows,
                        int64_t vocab, int64_t dim, int64_t ignore_index, int reduction,
                        void* workspace, size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  const Head p = head_of(dtype, hidden, ldh, weight, ldw, rows, vocab, dim);
  int rc = check_head(p);
  if (rc || (rc = check_reduction(reduction))) return rc;
  mhs::HeadRows g{};
  g.ids = ll(targets);
  g.lse2 = lse2;
  g.picked = picked;
  g.loss = loss_rows;
  g.keep = keep;
  g.k = 1;
  g.ignore = ignore_index;
  g.temperature = 1.f;
  return head_fwd(p, g, logits, loss, count, reduction, workspace, workspace_bytes, stream);
}

size_t mhs_linear_xent_bwd_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int64_t dim) {
  mhs::clear_error();
  const Head p = head_of(dtype, nullptr, dim, nullptr, dim, rows, vocab, dim);
  return check_sizes(p) ? 0 : std::max(bwd_ws(p), (size_t)256);
}

int mhs_linear_xent_bwd(int dtype, const void* hidden, int64_t ldh, const void* weight, int64_t ldw,
                        const int64_t* targets, const float* lse2, const float* picked,
                        const float* keep, const float* logits, const float* upstream,
                        const float* count, void* dhidden, void* dweight, int64_t rows,
                        int64_t vocab, int64_t dim, int reduction, void* workspace,
                        size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  const Head p = head_of(dtype, hidden, ldh, weight, ldw, rows, vocab, dim);
  int rc = check_head(p);
  if (rc || (rc = check_reduction(reduction))) return rc;
  if (reduction == MHS_REDUCE_MEAN && rows > 0 && !count)
    return fail(MHS_EINVAL, "null pointer argument");
  mhs::HeadGrad a{};
  a.ids = ll(targets);
  a.picked = picked;
  a.k = 1;
  a.c = mhs::kLog2e;
  return head_bwd(p, a, row_scale(upstream, count, keep, reduction, 1.f), lse2, logits,
                  BwdOut{dhidden, dweight}, workspace, workspace_bytes, stream);
}

int mhs_linear_distill_fwd(int dtype, const void* hidden, int64_t ldh, const void* weight,
                           int64_t ldw, const float* teacher, const int64_t* ids, float* lse2,
                           float* picked, float* q, float* keep, float* logits, float* loss_rows,
                           float* loss, float* count, int64_t rows, int64_t vocab, int64_t dim,
                           int64_t top, float temperature, int reduction, void* workspace,
                           size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  const Head p = head_of(dtype, hidden, ldh, weight, ldw, rows, vocab, dim);
  int rc = check_head(p);
  if (rc || (rc = check_reduction(reduction)) || (rc = check_top(top, temperature)) ||
      (rc = check_block_rows(rows)))
    return rc;
  if (rows > 0 && (!teacher || !q)) return fail(MHS_EINVAL, "null pointer argument");
  mhs::HeadRows g{};
  g.ids = ll(ids);
  g.teacher = teacher;
  g.lse2 = lse2;
  g.picked = picked;
  g.q = q;
  g.loss = loss_rows;
  g.keep = keep;
  g.k = (int)top;
  g.temperature = temperature;
  return head_fwd(p, g, logits, loss, count, reduction, workspace, workspace_bytes, stream);
}

int mhs_linear_distill_bwd(int dtype, const void* hidden, int64_t ldh, const void* weight,
                           int64_t ldw, const int64_t* ids, const float* lse2, const float* picked,
                           const float* q, const float* keep, const float* logits,
                           const float* upstream, const float* count, void* dhidden,
                           void* dweight, int64_t rows, int64_t vocab, int64_t dim, int64_t top,
                           float temperature, int reduction, void* workspace,
                           size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  const Head p = head_of(dtype, hidden, ldh, weight, ldw, rows, vocab, dim);
  int rc = check_head(p);
  if (rc || (rc = check_reduction(reduction)) || (rc = check_top(top, temperature)) ||
      (rc = check_block_rows(rows)))
    return rc;
  if (rows > 0 && (!q || (reduction == MHS_REDUCE_MEAN && !count)))
    return fail(MHS_EINVAL, "null pointer argument");
  mhs::HeadGrad a{};
  a.ids = ll(ids);
  a.q = q;
  a.picked = picked;
  a.k = (int)top;
  a.c = mhs::kLog2e / temperature;
  return head_bwd(p, a, row_scale(upstream, count, keep, reduction, temperature), lse2, logits,
                  BwdOut{dhidden, dweight}, workspace, workspace_bytes, stream);
}

size_t mhs_distill_workspace_bytes(int64_t rows) {
  mhs::clear_error();
  return check_block_rows(rows) ? 0 : std::max(loss_ws(rows), (size_t)256);
}

int mhs_distill_fwd(int dtype, const void* logits, int64_t ld, const float* teacher,
                    const int64_t* ids, float* lse2, float* q, float* keep, float* loss_rows,
                    float* loss, float* count, int64_t rows, int64_t vocab, int64_t top,
                    float temperature, int reduction, void* workspace, size_t workspace_bytes,
                    void* stream) {
  mhs::clear_error();
  int rc = check_logits(dtype, logits, ld, rows, vocab, top, temperature, reduction);
  if (rc) return rc;
  if ((rows > 0 && (!teacher || !ids || !lse2 || !q || !keep || !loss_rows)) ||
      (reduction != MHS_REDUCE_NONE && (!loss || !count)))
    return fail(MHS_EINVAL, "null pointer argument");
  rc = check_workspace(workspace, workspace_bytes,
                       reduction == MHS_REDUCE_NONE ? 0 : loss_ws(rows));
  if (rc) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    mhs::HeadRows g{};
    g.h = logits;
    g.ldh = ld;
    g.ids = ll(ids);
    g.teacher = teacher;
    g.lse2 = lse2;
    g.q = q;
    g.loss = loss_rows;
    g.keep = keep;
    g.rows = (int)rows;
    g.vocab = (int)vocab;
    g.k = (int)top;
    g.temperature = temperature;
    const auto fn = dtype == MHS_F32    ? &mhs::distill_fwd_kernel<Fp32>
                    : dtype == MHS_BF16 ? &mhs::distill_fwd_kernel<Bf16>
                                        : &mhs::distill_fwd_kernel<Fp16>;
    hipLaunchKernelGGL(fn, dim3((unsigned)rows), dim3(mhs::kXentThreads),
                       2 * (size_t)top * sizeof(float), s, g);
    if ((rc = check_launch("distillation forward kernel")) != 0) return rc;
  }
  if (reduction == MHS_REDUCE_NONE) return MHS_OK;
  return launch_loss(loss_rows, keep, loss, count, rows, reduction, workspace, s);
}

int mhs_distill_bwd(int dtype, const void* logits, int64_t ld, const int64_t* ids,
                    const float* lse2, const float* q, const float* keep, const float* upstream,
                    const float* count, void* dlogits, int64_t rows, int64_t vocab, int64_t top,
                    float temperature, int reduction, void* stream) {
  mhs::clear_error();
  int rc = check_logits(dtype, logits, ld, rows, vocab, top, temperature, reduction);
  if (rc) return rc;
  if (rows == 0) return MHS_OK;
  if (!ids || !lse2 || !q || !keep || !upstream || !dlogits ||
      (reduction == MHS_REDUCE_MEAN && !count))
    return fail(MHS_EINVAL, "null pointer argument");
  if (dlogits == logits) return fail(MHS_EINVAL, "dlogits may not alias logits");
  if (!aligned16(dlogits)) return fail(MHS_EINVAL, "dlogits must be 16-byte aligned");
  const mhs::RowScale rs = row_scale(upstream, count, keep, reduction, temperature);
  const float c = mhs::kLog2e / temperature;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const auto fn = dtype == MHS_F32    ? &launch_distill_bwd<Fp32>
                  : dtype == MHS_BF16 ? &launch_distill_bwd<Bf16>
                                      : &launch_distill_bwd<Fp16>;
  return fn(logits, ld, ids, q, lse2, rs, dlogits, rows, vocab, top, c, s);
}

}  // extern "C"
