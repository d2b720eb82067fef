// Gated delta rule: the kernels for bf16 activations.
#include "delta_instances.cuh"

namespace slx {
namespace delta {
template int launch_fwd_as<__nv_bfloat16>(const Args &, int, int, cudaStream_t);
template int launch_bwd_as<__nv_bfloat16>(const Args &, int, void *, void *, int, cudaStream_t);
}  // namespace delta
}  // namespace slx
