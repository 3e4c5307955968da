// The launches of mhs_packed_launch.hpp, to be instantiated.
#pragma once

#include "mhs_packed_launch.hpp"

namespace mhs {

template <class T, int NPL, int WS, bool VEC>
int run_scan(bool back, const PackedScanArgs& a, const ScanPlan& p, hipStream_t s) {
  const dim3 all((unsigned)p.pieces, (unsigned)p.blocks);
  if (p.carried && a.q.nseq > 0) {
    if (back) packed_scan_back_carry_kernel<T, NPL, WS, VEC><<<all, 256, 0, s>>>(a);
    else packed_scan_fwd_kernel<T, NPL, WS, VEC, true, false><<<all, 256, 0, s>>>(a);
    int rc = check_launch("packed scan carry kernel");
    if (rc) return rc;
    const dim3 grid((unsigned)a.q.nseq, (unsigned)(((int64_t)a.D * a.N + 255) / 256));
    if (back) packed_fold_kernel<true><<<grid, 256, 0, s>>>(a);
    else packed_fold_kernel<false><<<grid, 256, 0, s>>>(a);
    if ((rc = check_launch("packed scan fold kernel"))) return rc;
  }
  if (back) packed_scan_bwd_kernel<T, NPL, WS, VEC><<<all, 256, 0, s>>>(a);
  else if (a.ckpt) packed_scan_fwd_kernel<T, NPL, WS, VEC, false, true><<<all, 256, 0, s>>>(a);
  else packed_scan_fwd_kernel<T, NPL, WS, VEC, false, false><<<all, 256, 0, s>>>(a);
  return check_launch("packed scan kernel");
}
// Whether two channels (and NPL states) can be moved in one access of whole words.
template <class T, int NPL>
bool scan_vec(bool back, const PackedScanArgs& a) {
  if (a.D % 2 || a.N % NPL) return false;
  if (kElem<T> == 4) return true;
  const auto even = [](const void* p, int ld) {
    return ld % 2 == 0 && (reinterpret_cast<uintptr_t>(p) & 3u) == 0;
  };
  return even(a.x, a.ld_x) && even(a.dt, a.ld_dt) && even(a.B, a.ld_b) && even(a.C, a.ld_c) &&
         (!back || even(a.dy, a.ld_dy));
}
template <class T, int NPL, int WS>
int run_scan_v(bool back, const PackedScanArgs& a, const ScanPlan& p, hipStream_t s) {
  return scan_vec<T, NPL>(back, a) ? run_scan<T, NPL, WS, true>(back, a, p, s)
                                   : run_scan<T, NPL, WS, false>(back, a, p, s);
}
template <class T>
int run_packed_scan(bool back, const PackedScanArgs& a, const ScanPlan& p, hipStream_t s) {
  switch (scan_lane_states(a.N) * 8 + scan_state_waves(a.N)) {
    case 1 * 8 + 1: return run_scan_v<T, 1, 1>(back, a, p, s);
    case 2 * 8 + 1: return run_scan_v<T, 2, 1>(back, a, p, s);
    case 4 * 8 + 1: return run_scan_v<T, 4, 1>(back, a, p, s);
    case 4 * 8 + 2: return run_scan_v<T, 4, 2>(back, a, p, s);
    default: return run_scan_v<T, 4, 4>(back, a, p, s);
  }
}
}  // namespace mhs
