// Kernels of the selective scan for double rows.
#include "selscan_impl.cuh"

namespace fdwt {
FDWT_SCAN_TYPE(double)
}  // namespace fdwt
