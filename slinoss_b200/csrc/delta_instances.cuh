// Instances of the gated delta rule's kernels for one activation dtype: included by a source file each.
#pragma once

#include "delta_chunk.cuh"
#include "delta_grad.cuh"
#include "delta_launch.cuh"
#include "delta_scan.cuh"
#include "delta_team.cuh"

namespace slx {
namespace delta {

template <int NT, int SI, int SC, typename TI>
static int launch_chunk(const Args &a, cudaStream_t st) {
  constexpr int bytes = chunk_smem<NT, SI>();
  auto kernel = delta_chunk_kernel<NT, SI, TI>;
  if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
  kernel<<<dim3(a.NC, a.batch * a.key_heads), kThreads, bytes, st>>>(a);
  return check_launch("delta_chunk_kernel");
}
// warps == 0: teams on 16 value channels (where their tiles fit an SM: not fp32 of more than 64 columns)
template <int NT, int SI>
constexpr bool has_team = SI == 1 || NT == 64;

template <int NT, int SI, int SC, typename TI>
static int launch_fwd(const Args &a, int warps, cudaStream_t st) {
  if (const int rc = launch_chunk<NT, SI, SC, TI>(a, st)) return rc;
  if constexpr (has_team<NT, SI>) {
    if (warps == 0) {
      constexpr int bytes = sizeof(TeamShared<NT, SI, SC, TI>);
      auto kernel = delta_fwd_team_kernel<NT, SI, SC, TI>;
      if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
      kernel<<<dim3(a.P16 / 16, a.batch * a.heads), kTeamThreads, bytes, st>>>(a);
      return check_launch("delta_fwd_team_kernel");
    }
  }
  if (warps == 0) warps = a.P16 < 64 ? a.P16 / 16 : 4;
  constexpr int bytes = scan_smem<NT, SI, SC, TI>(false);
  auto kernel = delta_fwd_kernel<NT, SI, SC, TI>;
  if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
  kernel<<<dim3((a.P16 / 16 + warps - 1) / warps, a.batch * a.heads), kThreads, bytes, st>>>(a, warps);
  return check_launch("delta_fwd_kernel");
}
template <int NT, int SI, int SC, typename TI>
static int launch_bwd(const Args &a, void *dq, void *dk, int warps, cudaStream_t st) {
  bool done = false;
  if constexpr (has_team<NT, SI>) {
    if (warps == 0) {
      constexpr int bytes = sizeof(TeamShared<NT, SI, 2, TI>);
      auto kernel = delta_bwd_team_kernel<NT, SI, SC, TI>;
      if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
      kernel<<<dim3(a.P16 / 16, a.batch * a.heads), kTeamThreads, bytes, st>>>(a);
      if (const int rc = check_launch("delta_bwd_team_kernel")) return rc;
      done = true;
    }
  }
  if (warps == 0) warps = a.P16 < 64 ? a.P16 / 16 : 4;
  if (!done) {
    constexpr int bytes = scan_smem<NT, SI, SC, TI>(true);
    auto kernel = delta_bwd_kernel<NT, SI, SC, TI>;
    if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
    kernel<<<dim3((a.P16 / 16 + warps - 1) / warps, a.batch * a.heads), kThreads, bytes, st>>>(a, warps);
    if (const int rc = check_launch("delta_bwd_kernel")) return rc;
  }
  {
    constexpr int bytes = grad_smem<NT, SI, SC>();
    auto kernel = delta_grad_kernel<NT, SI, SC, TI>;
    if (const int rc = ensure_dyn_smem(kernel, bytes)) return rc;
    kernel<<<dim3(a.NC, a.batch * a.heads), kThreads, bytes, st>>>(a);
    if (const int rc = check_launch("delta_grad_kernel")) return rc;
  }
  if (a.heads != a.key_heads) {
    const int64_t per = (int64_t)a.T * a.N;
    const bool wide = per % 4 == 0 && ((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk)) & 15) == 0;
    const int64_t want = (per + (wide ? 1023 : 255)) / (wide ? 1024 : 256), fill = 16 * kB200Sms / (a.batch * a.key_heads) + 1;
    auto kernel = wide ? delta_share_kernel<4, TI> : delta_share_kernel<1, TI>;
    kernel<<<dim3((unsigned)(want < fill ? want : fill), a.batch * a.key_heads, 2), 256, 0, st>>>(
        static_cast<const float *>(a.dq), static_cast<const float *>(a.dk), static_cast<TI *>(dq), static_cast<TI *>(dk),
        a.heads / a.key_heads, per);
    return check_launch("delta_share_kernel");
  }
  return SLX_OK;
}

// planes of the inputs and of computed operands
template <typename TI>
constexpr int input_planes = sizeof(TI) == 4 ? 2 : 1;
template <typename TI>
constexpr int computed_planes = std::is_same<TI, __nv_bfloat16>::value ? 1 : 2;

template <typename TI>
int launch_fwd_as(const Args &a, int NT, int warps, cudaStream_t st) {
  constexpr int SI = input_planes<TI>, SC = computed_planes<TI>;
  return NT == 64 ? launch_fwd<64, SI, SC, TI>(a, warps, st) : launch_fwd<128, SI, SC, TI>(a, warps, st);
}
template <typename TI>
int launch_bwd_as(const Args &a, int NT, void *dq, void *dk, int warps, cudaStream_t st) {
  constexpr int SI = input_planes<TI>, SC = computed_planes<TI>;
  return NT == 64 ? launch_bwd<64, SI, SC, TI>(a, dq, dk, warps, st) : launch_bwd<128, SI, SC, TI>(a, dq, dk, warps, st);
}

}  // namespace delta
}  // namespace slx
