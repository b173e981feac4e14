// The products of qmm.cuh over this format's weights.
#include "qmm_launch.cuh"

namespace nsq {
int launch_qmm_q6k(int layout, const QmmParams& p, const CUtensorMap* maps, int grid, size_t smem, cudaStream_t st) {
  return launch_qmm_type<NSQ_TYPE_Q6_K>(layout, p, maps, grid, smem, st);
}
}  // namespace nsq
