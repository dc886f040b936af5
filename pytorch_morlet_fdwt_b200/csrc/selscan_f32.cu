// Kernels of the selective scan for float rows.
#include "selscan_impl.cuh"

namespace fdwt {
FDWT_SCAN_TYPE(float)
}  // namespace fdwt
