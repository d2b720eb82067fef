// Launches of the gated delta rule's kernels, by activation dtype and by the width N is padded to (64 or 128).
#pragma once

#include "delta.cuh"

namespace slx {
namespace delta {

template <typename TI>
int launch_fwd_as(const Args &a, int NT, int warps, cudaStream_t st);
template <typename TI>
int launch_bwd_as(const Args &a, int NT, void *dq, void *dk, int warps, cudaStream_t st);

}  // namespace delta
}  // namespace slx
