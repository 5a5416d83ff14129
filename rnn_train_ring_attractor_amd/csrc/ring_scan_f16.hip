// The kernels of the selective scan for fp16 rows.
#include "ring_scan.hpp"

hipError_t ring_launch_scan_f16(const RingScanArgs& p, int mode, hipStream_t st) { return ring_scan::launch<_Float16>(p, mode, st); }
