// Kernels of the selective scan for __half rows.
#include "selscan_impl.cuh"

namespace fdwt {
FDWT_SCAN_TYPE(__half)
}  // namespace fdwt
