// The products of qmm.cuh over this format's weights.
#include "qmm_launch.cuh"

namespace nsq {
int launch_qmm_q80(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st) {
  return launch_qmm_type<NSQ_TYPE_Q8_0>(layout, p, maps, grid, smem, st);
}
}  // namespace nsq
