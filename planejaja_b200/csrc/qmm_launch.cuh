// qmm_launch.cuh -- launches qmm_kernel; included by the per-format files.
#pragma once

#include "qmm.cuh"

namespace nsq {

template <int TYPE, int LAYOUT, int TC, int MODE>
int launch_qmm_t(const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st) {
  auto kern = qmm_kernel<TYPE, LAYOUT, TC, MODE>;
  // the opt-in limit is set once per device; the launches ask for what they need
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return NSQ_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kQmmSmemMax) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) !=
            cudaSuccess)
      return NSQ_ERR_CUDA;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kQmmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, kern, p, maps[0], maps[1]) == cudaSuccess ? NSQ_OK : NSQ_ERR_CUDA;
}

template <int TYPE, int LAYOUT, int TC>
int launch_qmm_mode(const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st) {
  if (p.mode == kQmmLinear) return launch_qmm_t<TYPE, LAYOUT, TC, kQmmLinear>(p, maps, grid, smem, st);
  if (p.mode == kQmmUp) return launch_qmm_t<TYPE, LAYOUT, TC, kQmmUp>(p, maps, grid, smem, st);
  return launch_qmm_t<TYPE, LAYOUT, TC, kQmmDown>(p, maps, grid, smem, st);
}

template <int TYPE, int LAYOUT>
int launch_qmm_layout(const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st) {
  if (p.TS <= 2) return launch_qmm_mode<TYPE, LAYOUT, 2>(p, maps, grid, smem, st);
  if (p.TS <= 4) return launch_qmm_mode<TYPE, LAYOUT, 4>(p, maps, grid, smem, st);
  if (p.TS <= 8) return launch_qmm_mode<TYPE, LAYOUT, 8>(p, maps, grid, smem, st);
  return launch_qmm_mode<TYPE, LAYOUT, 16>(p, maps, grid, smem, st);
}

template <int TYPE>
int launch_qmm_type(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st) {
  if constexpr (TYPE == NSQ_TYPE_Q5_K || TYPE == NSQ_TYPE_Q6_K) {
    if (layout == NSQ_Q6K_NODESTOR) return launch_qmm_layout<TYPE, NSQ_Q6K_NODESTOR>(p, maps, grid, smem, st);
  }
  return launch_qmm_layout<TYPE, NSQ_Q6K_GGML>(p, maps, grid, smem, st);
}

}  // namespace nsq
