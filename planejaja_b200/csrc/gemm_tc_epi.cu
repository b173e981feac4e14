// gemm_tc_epi.cu -- the prefill GEMM of nsq_linear, y = act(x . W^T + bias) +
// residual: the kernel of gemm_tc.cuh with its epilogue.
#include "gemm_tc.cuh"

namespace nsq {

int run_gemm_epi(const uint8_t* w, int type, int layout, const void* x, const float* bias, int act, const void* residual,
                 void* y, int64_t M, int64_t N, int64_t K, cudaStream_t st, int num_sms) {
  GemmParams p{};
  p.w = w;
  p.y = static_cast<__nv_bfloat16*>(y);
  p.M = M;
  p.N = N;
  p.K = K;
  p.act = act;
  p.bias = bias;
  p.residual = static_cast<const __nv_bfloat16*>(residual);
  return run_gemm<true>(p, type, layout, x, st, num_sms);
}

}  // namespace nsq
