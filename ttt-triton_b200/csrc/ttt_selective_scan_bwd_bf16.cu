// Backward of the selective scan for bf16 activations.
#include "selective_scan_bwd.cuh"

namespace ttt {
namespace scan {
template int launch_bwd<__nv_bfloat16>(Params, void*, void*, float*, cudaStream_t, const char*);
}  // namespace scan
}  // namespace ttt
