// Launches of the packed scan's kernels, by type in a unit each.
#pragma once

#include "mamba_hip_scan.h"
#include "mhs_host.hpp"
#include "mhs_packed_scan.hpp"

namespace mhs {

// State groups (waves) of a block and states of a lane, by d_state.
inline int scan_lane_states(int64_t n) { return n <= 4 ? 1 : n <= 8 ? 2 : 4; }
inline int scan_state_waves(int64_t n) { return n <= 16 ? 1 : n <= 32 ? 2 : 4; }
inline int scan_block_chans(int64_t n) { return 32 * (4 / scan_state_waves(n)); }

struct ScanPlan {
  int tc;
  int64_t pieces, blocks;
  bool carried;   // whether a sequence can be longer than a piece
};
template <class T>
int run_packed_scan(bool back, const PackedScanArgs& a, const ScanPlan& p, hipStream_t s);

}  // namespace mhs
