// The kernels of the selective scan for fp32 rows.
#include "ring_scan.hpp"

hipError_t ring_launch_scan_f32(const RingScanArgs& p, int mode, hipStream_t st) { return ring_scan::launch<float>(p, mode, st); }
