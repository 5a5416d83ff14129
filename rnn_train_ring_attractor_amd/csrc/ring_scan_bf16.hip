// The kernels of the selective scan for bf16 rows.
#include "ring_scan.hpp"

hipError_t ring_launch_scan_bf16(const RingScanArgs& p, int mode, hipStream_t st) { return ring_scan::launch<__bf16>(p, mode, st); }
