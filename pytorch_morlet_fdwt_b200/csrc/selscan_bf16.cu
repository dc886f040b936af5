// Kernels of the selective scan for __nv_bfloat16 rows.
#include "selscan_impl.cuh"

namespace fdwt {
FDWT_SCAN_TYPE(__nv_bfloat16)
}  // namespace fdwt
