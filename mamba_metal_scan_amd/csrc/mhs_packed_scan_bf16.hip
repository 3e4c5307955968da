// Packed scan, bf16: the instantiations of mhs_packed_instances.hpp.
#include "mhs_packed_instances.hpp"

namespace mhs {
template int run_packed_scan<Bf16>(bool, const PackedScanArgs&, const ScanPlan&, hipStream_t);
}
