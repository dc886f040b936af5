#include "linattn.cuh"
namespace fdwt { namespace linattn {
bool tc_supports(int, const Call&) { return false; }
int tc_launch(int, const Call&, bool, cudaStream_t) { return FDWT_ERR_UNSUPPORTED; }
} }
