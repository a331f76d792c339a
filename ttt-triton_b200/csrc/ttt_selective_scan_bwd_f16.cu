// Backward of the selective scan for fp16 activations.
#include "selective_scan_bwd.cuh"

namespace ttt {
namespace scan {
template int launch_bwd<__half>(Params, void*, void*, float*, cudaStream_t, const char*);
}  // namespace scan
}  // namespace ttt
