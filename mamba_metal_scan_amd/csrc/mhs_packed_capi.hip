// C ABI of the operators over packed sequences and of the tokens by slot (declared in
// include/mamba_hip_scan.h): argument checks, the pieces' length, grids, the
// workspaces' layout. No allocation.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mamba_hip_scan.h"
#include "mhs_host.hpp"
#include "mhs_packed_conv.hpp"
#include "mhs_packed_launch.hpp"
#include "mhs_packed_sum.hpp"

namespace {

using mhs::aligned16;
using mhs::check_launch;
using mhs::device_cus;
using mhs::fail;
using mhs::round_up;

// Channels, row strides and rows that the kernels' 32-bit offsets within a piece (and their
// grids) hold.
constexpr int64_t kMaxDim = 1LL << 17;
constexpr int64_t kMaxStride = 1LL << 18;
constexpr int64_t kMaxSeqs = 1LL << 22;
constexpr int64_t kMaxRows = (1LL << 31) - 1;
constexpr int64_t kMaxStepRows = 1LL << 22;

int elem(int dtype) { return dtype == MHS_F32 ? 4 : 2; }

int check_dtype(int dtype) {
  if (dtype != MHS_F32 && dtype != MHS_BF16 && dtype != MHS_F16)
    return fail(MHS_EINVAL, "dtype must be MHS_F32, MHS_BF16 or MHS_F16; got %d", dtype);
  return MHS_OK;
}

int check_packed(const void* cu, int64_t nseq, int64_t total, int64_t dim) {
  if (total < 0 || total > kMaxRows || nseq < 0 || nseq > kMaxSeqs || dim < 1 || dim > kMaxDim)
    return fail(MHS_EINVAL, "rows must be in [0, 2^31), sequences in [0, 2^22], channels in "
                "[1, 2^17]; got %lld, %lld, %lld", (long long)total, (long long)nseq,
                (long long)dim);
  if (!cu) return fail(MHS_EINVAL, "null pointer argument");
  return MHS_OK;
}

int check_ld(const char* what, int64_t ld, int64_t width) {
  if (ld < width || ld >= kMaxStride)
    return fail(MHS_EINVAL, "the rows of %s must be at least %lld elements apart and less than "
                "2^18; got %lld", what, (long long)width, (long long)ld);
  return MHS_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return fail(MHS_EINVAL, "workspace too small: %zu < %zu bytes", have, need);
  if (need && (reinterpret_cast<uintptr_t>(ws) & 255u))
    return fail(MHS_EINVAL, "workspace must be 256-byte aligned");
  return MHS_OK;
}

// f(a value of the type that dtype names).
template <class F>
auto by_type(int dtype, F&& f) {
  if (dtype == MHS_F32) return f(mhs::F32{});
  if (dtype == MHS_BF16) return f(mhs::Bf16{});
  return f(mhs::Fp16{});
}

mhs::Seqs seqs(const void* cu, int cu64, int64_t nseq, int64_t total) {
  return {cu, cu64, (int)nseq, (int)total};
}
int64_t piece_count(int64_t total, int64_t nseq, int tc) { return total / tc + nseq + 1; }

// ---------------------------------------------------------------- the scan

// Rows of a piece: as many pieces as give each SIMD twelve waves, eight in the backward, which
// holds two at a time (their latencies then hide each other's, and pieces of unlike
// length even out), rounded down to whole sub-chunks. The launches of a captured call, us, in
// pieces of 16 rows | 32 | 48 | 64 | 80 | 96 | 128 | 160 | 256:
//   8192 x 1536 x 16 in fp32, 24 sequences,
//     forward (this gives 32)   153 | 122 | 117 | 115 | 118 | 121 | 137 | 141 | 150
//     backward (48)             247 | 208 | 197 | 193 | 204 | 218 | 221 | 228 | 262
//   32768 x 2048 x 16 in bf16, 9 sequences,
//     forward (160)             616 | 495 | 477 | 456 | 444 | 449 | 444 | 438 | 449
//     backward (256)           1079 | 893 | 827 | 798 | 791 | 786 | 780 | 791 | 804
//   4096 x 4096 x 16 in bf16, 12 prompts to states (32)
//                               141 | 122 | 114 | 113 | 119 | 124 | 137 | 153 | 162
//   one prompt of 509 x 640 x 16 in fp32 (16)
//                                18 |  20 |  24 |  28 |  32 |  36 |  45 |  53 |  77
// It counts the waves alone and not the states that a piece more has carried, written and
// read, and loses up to 7% to the best of these: 64 rows in the first case and the third.
// Few rows are one piece, without carries: of 640 x 16 in fp32 at 32 | 64 | 96 rows one launch
// takes 8.2 | 12.8 | 17.4 us and the three 13.1 | 13.3 | 13.4 (captured; a call 14.4 | 14.3 | 17.5
// and 20), the backward in one piece 18.9 | 30.0 | 40.8, in several 20.8 | 21.1 | 21.3.
int scan_piece(int64_t total, int64_t dim, int64_t n, bool back) {
  if (total <= (back ? 32 : 64)) return back ? 32 : 64;
  const int64_t waves = (dim + 31) / 32 * mhs::scan_state_waves(n);
  const int64_t pieces = std::max<int64_t>(1, (back ? 32 : 48) * device_cus() / waves);
  const int64_t tc = total / pieces / mhs::kSub * mhs::kSub;
  return (int)std::min<int64_t>(1024, std::max<int64_t>(16, tc));
}

using mhs::ScanPlan;
ScanPlan scan_plan(int64_t total, int64_t nseq, int64_t dim, int64_t n, bool back) {
  ScanPlan p;
  p.tc = scan_piece(total, dim, n, back);
  p.pieces = piece_count(total, nseq, p.tc);
  p.blocks = (dim + mhs::scan_block_chans(n) - 1) / mhs::scan_block_chans(n);
  p.carried = total > p.tc;
  return p;
}

// A direction's launches are counted by its own plan: of 33 to 64 rows the backward has the shorter
// pieces, of more the forward.
int check_scan(int dtype, const void* cu, int64_t nseq, int64_t total, int64_t dim, int64_t n,
               bool back) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  if ((rc = check_packed(cu, nseq, total, dim))) return rc;
  if (n < 1 || n > MHS_MAX_DSTATE)
    return fail(MHS_EINVAL, "d_state must be in [1, %d]; got %lld", MHS_MAX_DSTATE, (long long)n);
  const ScanPlan p = scan_plan(total, nseq, dim, n, back);
  // (a launch counts its threads in 32 bits: the pass, the fold, the sums)
  if (p.pieces * p.blocks >= 1LL << 24 || nseq * ((dim * n + 255) / 256) >= 1LL << 24 ||
      (total * 2 * n + 255) / 256 >= 1LL << 24)
    return fail(MHS_EINVAL, "%lld rows x %lld channels are too many", (long long)total,
                (long long)dim);
  return MHS_OK;
}

struct Parts {
  char* p;
  size_t used = 0;
  float* take(size_t floats) {
    char* at = p ? p + used : nullptr;
    used += round_up(floats * 4, 256);
    return reinterpret_cast<float*>(at);
  }
};

// Workspace of either direction from `ws` (null: its size alone).
size_t scan_parts(void* ws, const ScanPlan& p, int64_t total, int64_t dim, int64_t n, bool back,
                  mhs::PackedScanArgs* a) {
  Parts w{static_cast<char*>(ws)};
  mhs::PackedScanArgs none;
  if (!a) a = &none;
  const size_t slice = (size_t)dim * n;
  if (p.carried) {
    a->carry = w.take(p.pieces * slice);
    a->start = w.take(p.pieces * slice);
    a->sdt = w.take((size_t)p.pieces * dim);
  }
  if (back) {
    a->part_bc = w.take((size_t)p.blocks * total * 2 * n);
    a->part_a = w.take(p.pieces * slice);
  }
  return w.used;
}

int run_scan_t(int dtype, bool back, const mhs::PackedScanArgs& a, const ScanPlan& p,
               hipStream_t s) {
  return by_type(dtype, [&](auto t) { return mhs::run_packed_scan<decltype(t)>(back, a, p, s); });
}

// --------------------------------------------------------- the convolution

// Whether a thread may have several channels: width, strides and addresses allow it.
bool conv_wide(int dtype, bool back, int64_t dim, std::initializer_list<const void*> ps,
               std::initializer_list<int64_t> lds) {
  const int v = back ? mhs::kConvBackVec : 8 / elem(dtype);
  bool ok = dim % v == 0;
  for (const void* p : ps) ok = ok && aligned16(p);
  for (const int64_t ld : lds) ok = ok && ld % v == 0;
  return ok;
}
using mhs::kConvBackPiece;
using mhs::kConvPiece;

int check_conv(int dtype, const void* cu, int64_t nseq, int64_t total, int64_t dim, int64_t taps) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  if ((rc = check_packed(cu, nseq, total, dim))) return rc;
  if (taps < 1 || taps > mhs::kPackedMaxTaps)
    return fail(MHS_EINVAL, "taps must be in [1, %d]; got %lld", mhs::kPackedMaxTaps,
                (long long)taps);
  if (((piece_count(total, nseq, kConvPiece) + 3) / 4) * ((dim + 63) / 64) >= 1LL << 24)
    return fail(MHS_EINVAL, "%lld rows x %lld channels are too many", (long long)total,
                (long long)dim);
  return MHS_OK;
}

template <class T, int K, int V>
int run_conv(bool back, const mhs::PackedConvArgs& a, hipStream_t s) {
  const int64_t pieces = piece_count(a.q.total, a.q.nseq, back ? kConvBackPiece : kConvPiece);
  const dim3 grid((unsigned)((pieces + 3) / 4), (unsigned)((a.D + 64 * V - 1) / (64 * V)));
  if (back) mhs::packed_conv_bwd_kernel<T, K, V><<<grid, 256, 0, s>>>(a, (int)pieces);
  else mhs::packed_conv_fwd_kernel<T, K, V><<<grid, 256, 0, s>>>(a, (int)pieces);
  return check_launch("packed conv kernel");
}
template <class T, int K>
int run_conv_v(bool wide, bool back, const mhs::PackedConvArgs& a, hipStream_t s) {
  if (!wide) return run_conv<T, K, 1>(back, a, s);
  return back ? run_conv<T, K, mhs::kConvBackVec>(true, a, s)
              : run_conv<T, K, mhs::kConvVec<T>>(false, a, s);
}
template <class T>
int run_conv_k(int64_t taps, bool wide, bool back, const mhs::PackedConvArgs& a, hipStream_t s) {
  switch (taps) {
    case 1: return run_conv_v<T, 1>(wide, back, a, s);
    case 2: return run_conv_v<T, 2>(wide, back, a, s);
    case 3: return run_conv_v<T, 3>(wide, back, a, s);
    case 4: return run_conv_v<T, 4>(wide, back, a, s);
    case 5: return run_conv_v<T, 5>(wide, back, a, s);
    case 6: return run_conv_v<T, 6>(wide, back, a, s);
    case 7: return run_conv_v<T, 7>(wide, back, a, s);
    default: return run_conv_v<T, 8>(wide, back, a, s);
  }
}
int run_conv_t(int dtype, int64_t taps, bool wide, bool back, const mhs::PackedConvArgs& a,
               hipStream_t s) {
  return by_type(dtype, [&](auto t) { return run_conv_k<decltype(t)>(taps, wide, back, a, s); });
}

// ------------------------------------------------------------------ tokens

int check_step(int dtype, const void* slots, int64_t rows, int64_t pool, int64_t dim) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  if (rows < 0 || rows > kMaxStepRows || pool < 0 || pool > kMaxRows || dim < 1 || dim > kMaxDim)
    return fail(MHS_EINVAL, "rows must be in [0, 2^22], the pool's entries in [0, 2^31), channels "
                "in [1, 2^17]; got %lld, %lld, %lld", (long long)rows, (long long)pool,
                (long long)dim);
  if (!slots && rows > pool)
    return fail(MHS_EINVAL, "%lld rows without slots need as many entries; got %lld",
                (long long)rows, (long long)pool);
  if (rows * ((dim + 31) / 32) >= 1LL << 24)
    return fail(MHS_EINVAL, "%lld rows x %lld channels are too many", (long long)rows,
                (long long)dim);
  return MHS_OK;
}

template <class T>
void launch_conv_step(int64_t taps, const mhs::ConvStepArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.rows, (unsigned)((a.D + 255) / 256));
  switch (taps) {
    case 1: mhs::conv_step_kernel<T, 1><<<grid, 256, 0, s>>>(a); break;
    case 2: mhs::conv_step_kernel<T, 2><<<grid, 256, 0, s>>>(a); break;
    case 3: mhs::conv_step_kernel<T, 3><<<grid, 256, 0, s>>>(a); break;
    case 4: mhs::conv_step_kernel<T, 4><<<grid, 256, 0, s>>>(a); break;
    case 5: mhs::conv_step_kernel<T, 5><<<grid, 256, 0, s>>>(a); break;
    case 6: mhs::conv_step_kernel<T, 6><<<grid, 256, 0, s>>>(a); break;
    case 7: mhs::conv_step_kernel<T, 7><<<grid, 256, 0, s>>>(a); break;
    default: mhs::conv_step_kernel<T, 8><<<grid, 256, 0, s>>>(a); break;
  }
}

template <class T, int V, int LPC>
void launch_state_step(const mhs::StateStepArgs& a, hipStream_t s) {
  constexpr int ch = 256 / LPC;
  const dim3 grid((unsigned)a.rows, (unsigned)((a.D + ch - 1) / ch));
  mhs::state_step_kernel<T, V, LPC><<<grid, 256, 0, s>>>(a);
}
// Lanes of a channel: as many as hold its states in float4s (or singly).
template <class T>
void run_state_step(const mhs::StateStepArgs& a, hipStream_t s) {
  if (a.N % 4) launch_state_step<T, 1, 4>(a, s);
  else if (a.N <= 4) launch_state_step<T, 4, 1>(a, s);
  else if (a.N <= 8) launch_state_step<T, 4, 2>(a, s);
  else if (a.N <= 16) launch_state_step<T, 4, 4>(a, s);
  else launch_state_step<T, 4, 8>(a, s);
}

}  // namespace

extern "C" {

int64_t mhs_packed_ckpt_floats(int64_t total, int64_t dim, int64_t d_state) {
  return total / mhs::kCkpt * dim * d_state;
}

size_t mhs_packed_scan_workspace_bytes(int64_t nseq, int64_t total, int64_t dim, int64_t d_state,
                                       int backward) {
  mhs::clear_error();
  if (check_scan(MHS_F32, &nseq, nseq, total, dim, d_state, backward != 0)) return 0;
  return scan_parts(nullptr, scan_plan(total, nseq, dim, d_state, backward != 0), total, dim,
                    d_state, backward != 0, nullptr);
}

int mhs_packed_scan_fwd(int dtype, const void* x, int64_t ld_x, const void* dt, int64_t ld_dt,
                        const float* aneg, const void* B, int64_t ld_b, const void* C,
                        int64_t ld_c, const void* cu_seqlens, int cu64, const float* h0, void* y,
                        float* h_last, float* ckpt, int64_t nseq, int64_t total, int64_t dim,
                        int64_t d_state, void* workspace, size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  int rc = check_scan(dtype, cu_seqlens, nseq, total, dim, d_state, false);
  if (rc) return rc;
  if (ckpt && (rc = check_scan(dtype, cu_seqlens, nseq, total, dim, d_state, true))) return rc;
  if (!aneg || (total > 0 && (!x || !dt || !B || !C || !y)))
    return fail(MHS_EINVAL, "null pointer argument");
  if ((rc = check_ld("x", ld_x, dim)) || (rc = check_ld("dt", ld_dt, dim)) ||
      (rc = check_ld("B", ld_b, d_state)) || (rc = check_ld("C", ld_c, d_state)))
    return rc;
  for (const float* p : {aneg, h0, (const float*)h_last, (const float*)ckpt})
    if (!aligned16(p)) return fail(MHS_EINVAL, "fp32 tensors must be 16-byte aligned");
  mhs::PackedScanArgs a{};
  const ScanPlan p = scan_plan(total, nseq, dim, d_state, false);
  if ((rc = check_workspace(workspace, workspace_bytes,
                            scan_parts(workspace, p, total, dim, d_state, false, &a))))
    return rc;
  a.q = seqs(cu_seqlens, cu64, nseq, total);
  a.x = x; a.dt = dt; a.B = B; a.C = C;
  a.ld_x = (int)ld_x; a.ld_dt = (int)ld_dt; a.ld_b = (int)ld_b; a.ld_c = (int)ld_c;
  a.aneg = aneg; a.h0 = h0; a.y = y; a.h_last = h_last; a.ckpt = ckpt;
  a.D = (int)dim; a.N = (int)d_state; a.tc = p.tc;
  return run_scan_t(dtype, false, a, p, static_cast<hipStream_t>(stream));
}

int mhs_packed_scan_bwd(int dtype, const void* x, int64_t ld_x, const void* dt, int64_t ld_dt,
                        const float* aneg, const void* B, int64_t ld_b, const void* C,
                        int64_t ld_c, const void* cu_seqlens, int cu64, const float* h0,
                        const float* ckpt, const void* dy, int64_t ld_dy, const float* dh_last,
                        void* dx, void* ddt, float* daneg, void* dB, void* dC, float* dh0,
                        int64_t nseq, int64_t total, int64_t dim, int64_t d_state,
                        void* workspace, size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  int rc = check_scan(dtype, cu_seqlens, nseq, total, dim, d_state, true);
  if (rc) return rc;
  if (!aneg || !daneg ||
      (total > 0 && (!x || !dt || !B || !C || !dy || !dx || !ddt || !dB || !dC)) ||
      (total >= mhs::kCkpt && !ckpt))
    return fail(MHS_EINVAL, "null pointer argument");
  if ((rc = check_ld("x", ld_x, dim)) || (rc = check_ld("dt", ld_dt, dim)) ||
      (rc = check_ld("B", ld_b, d_state)) || (rc = check_ld("C", ld_c, d_state)) ||
      (rc = check_ld("dy", ld_dy, dim)))
    return rc;
  for (const float* p : {aneg, h0, ckpt, dh_last, (const float*)daneg, (const float*)dh0})
    if (!aligned16(p)) return fail(MHS_EINVAL, "fp32 tensors must be 16-byte aligned");
  mhs::PackedScanArgs a{};
  const ScanPlan p = scan_plan(total, nseq, dim, d_state, true);
  if ((rc = check_workspace(workspace, workspace_bytes,
                            scan_parts(workspace, p, total, dim, d_state, true, &a))))
    return rc;
  a.q = seqs(cu_seqlens, cu64, nseq, total);
  a.x = x; a.dt = dt; a.B = B; a.C = C;
  a.ld_x = (int)ld_x; a.ld_dt = (int)ld_dt; a.ld_b = (int)ld_b; a.ld_c = (int)ld_c;
  a.aneg = aneg; a.h0 = h0; a.ckpt = const_cast<float*>(ckpt);
  a.dy = dy; a.ld_dy = (int)ld_dy; a.dh_last = dh_last;
  a.dx = dx; a.ddt = ddt; a.dh0 = dh0;
  a.D = (int)dim; a.N = (int)d_state; a.tc = p.tc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = run_scan_t(dtype, true, a, p, s))) return rc;
  const int64_t sums = total * 2 * d_state;
  if (sums) {
    const unsigned grid = (unsigned)((sums + 255) / 256);
    const int nblk = (int)p.blocks;
    by_type(dtype, [&](auto t) {
      mhs::packed_sum_bc_kernel<decltype(t)><<<grid, 256, 0, s>>>(a.part_bc, dB, dC, nblk, total,
                                                                  a.N);
    });
    if ((rc = check_launch("packed scan dB / dC sums"))) return rc;
  }
  const int slice = a.D * a.N;
  mhs::packed_sum_a_kernel<<<(slice + 63) / 64, 1024, 0, s>>>(a.part_a, daneg, (int)p.pieces,
                                                              slice);
  return check_launch("packed scan dAneg sum");
}

size_t mhs_packed_conv_bwd_workspace_bytes(int64_t nseq, int64_t total, int64_t dim,
                                           int64_t taps) {
  mhs::clear_error();
  if (check_conv(MHS_F32, &nseq, nseq, total, dim, taps)) return 0;
  return round_up((size_t)((piece_count(total, nseq, kConvBackPiece) + 3) / 4) * (taps + 1) * dim *
                      4, 256);
}

int mhs_packed_conv_fwd(int dtype, const void* x, int64_t ld_x, const void* weight,
                        const void* bias, int weight_f32, const void* cu_seqlens, int cu64,
                        const void* window, void* out, void* window_out, int64_t nseq,
                        int64_t total, int64_t dim, int64_t taps, void* stream) {
  mhs::clear_error();
  int rc = check_conv(dtype, cu_seqlens, nseq, total, dim, taps);
  if (rc) return rc;
  if (!weight || !bias || (total > 0 && (!x || !out)))
    return fail(MHS_EINVAL, "null pointer argument");
  if ((rc = check_ld("x", ld_x, dim))) return rc;
  mhs::PackedConvArgs a{};
  a.q = seqs(cu_seqlens, cu64, nseq, total);
  a.x = x; a.ld_x = ld_x; a.w = weight; a.bias = bias; a.wf32 = weight_f32;
  a.window = window; a.out = out; a.window_out = window_out;
  a.D = (int)dim;
  const bool wide = conv_wide(dtype, false, dim, {x, out, weight, bias}, {ld_x});
  return run_conv_t(dtype, taps, wide, false, a, static_cast<hipStream_t>(stream));
}

int mhs_packed_conv_bwd(int dtype, const void* x, int64_t ld_x, const void* weight,
                        const void* bias, int weight_f32, const void* cu_seqlens, int cu64,
                        const void* window, const void* dout, int64_t ld_dout,
                        const void* dwindow_out, void* dx, void* dweight, void* dbias,
                        void* dwindow, int64_t nseq, int64_t total, int64_t dim, int64_t taps,
                        void* workspace, size_t workspace_bytes, void* stream) {
  mhs::clear_error();
  int rc = check_conv(dtype, cu_seqlens, nseq, total, dim, taps);
  if (rc) return rc;
  if (!weight || !bias || !dweight || !dbias || (total > 0 && (!x || !dout || !dx)))
    return fail(MHS_EINVAL, "null pointer argument");
  if ((rc = check_ld("x", ld_x, dim)) || (rc = check_ld("dout", ld_dout, dim))) return rc;
  if ((rc = check_workspace(workspace, workspace_bytes,
                            mhs_packed_conv_bwd_workspace_bytes(nseq, total, dim, taps))))
    return rc;
  mhs::PackedConvArgs a{};
  a.q = seqs(cu_seqlens, cu64, nseq, total);
  a.x = x; a.ld_x = ld_x; a.w = weight; a.bias = bias; a.wf32 = weight_f32;
  a.window = window; a.dout = dout; a.ld_g = ld_dout; a.dwindow_out = dwindow_out;
  a.dx = dx; a.dwindow = dwindow; a.part = static_cast<float*>(workspace);
  a.D = (int)dim;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = conv_wide(dtype, true, dim, {x, dout, dx, weight, bias}, {ld_x, ld_dout});
  rc = run_conv_t(dtype, taps, wide, true, a, s);
  if (rc) return rc;
  const int n = (int)((piece_count(total, nseq, kConvBackPiece) + 3) / 4);
  const dim3 grid((unsigned)((dim + 63) / 64), (unsigned)(taps + 1));
  const int k = (int)taps;
  by_type(dtype, [&](auto t) {
    mhs::packed_conv_sum_kernel<decltype(t)><<<grid, 1024, 0, s>>>(a.part, dweight, dbias,
                                                                   weight_f32, n, k, a.D);
  });
  return check_launch("packed conv weight gradient sum");
}

int mhs_conv_step(int dtype, const void* x, int64_t ld_x, const void* weight, const void* bias,
                  int weight_f32, void* window, const void* slots, int slots64, void* out,
                  int64_t rows, int64_t pool, int64_t dim, int64_t taps, void* stream) {
  mhs::clear_error();
  int rc = check_step(dtype, slots, rows, pool, dim);
  if (rc) return rc;
  if (taps < 1 || taps > mhs::kPackedMaxTaps)
    return fail(MHS_EINVAL, "taps must be in [1, %d]; got %lld", mhs::kPackedMaxTaps,
                (long long)taps);
  if (rows == 0) return MHS_OK;
  if (!x || !weight || !bias || !out || (pool > 0 && taps > 1 && !window))
    return fail(MHS_EINVAL, "null pointer argument");
  if ((rc = check_ld("x", ld_x, dim))) return rc;
  mhs::ConvStepArgs a{x, ld_x, weight, bias, weight_f32, window, slots, slots64, out, (int)rows,
                      (int)pool, (int)dim};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MHS_F32) launch_conv_step<mhs::F32>(taps, a, s);
  else if (dtype == MHS_BF16) launch_conv_step<mhs::Bf16>(taps, a, s);
  else launch_conv_step<mhs::Fp16>(taps, a, s);
  return check_launch("conv step kernel");
}

int mhs_state_step(int dtype, float* h, const void* x, int64_t ld_x, const void* dt, int64_t ld_dt,
                   const float* aneg, const void* B, int64_t ld_b, const void* C, int64_t ld_c,
                   const void* slots, int slots64, void* y, int64_t rows, int64_t pool,
                   int64_t dim, int64_t d_state, void* stream) {
  mhs::clear_error();
  int rc = check_step(dtype, slots, rows, pool, dim);
  if (rc) return rc;
  if (d_state < 1 || d_state > MHS_MAX_DSTATE)
    return fail(MHS_EINVAL, "d_state must be in [1, %d]; got %lld", MHS_MAX_DSTATE,
                (long long)d_state);
  if (rows == 0) return MHS_OK;
  if (!x || !dt || !aneg || !B || !C || !y || (pool > 0 && !h))
    return fail(MHS_EINVAL, "null pointer argument");
  if ((rc = check_ld("x", ld_x, dim)) || (rc = check_ld("dt", ld_dt, dim)) ||
      (rc = check_ld("B", ld_b, d_state)) || (rc = check_ld("C", ld_c, d_state)))
    return rc;
  if (!aligned16(h) || !aligned16(aneg))
    return fail(MHS_EINVAL, "fp32 tensors must be 16-byte aligned");
  mhs::StateStepArgs a{h, x, dt, B, C, ld_x, ld_dt, ld_b, ld_c, aneg, slots, slots64, y, (int)rows,
                       (int)pool, (int)dim, (int)d_state};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MHS_F32) run_state_step<mhs::F32>(a, s);
  else if (dtype == MHS_BF16) run_state_step<mhs::Bf16>(a, s);
  else run_state_step<mhs::Fp16>(a, s);
  return check_launch("state step kernel");
}

}  // extern "C"
