// Backward of the selective scan for fp32 activations.
#include "selective_scan_bwd.cuh"

namespace ttt {
namespace scan {
template int launch_bwd<float>(Params, void*, void*, float*, cudaStream_t, const char*);
}  // namespace scan
}  // namespace ttt
