// gemm_tc.cu -- the plain prefill GEMM, y = x . W^T (see gemm_tc.cuh).
#include "gemm_tc.cuh"

namespace nsq {

int run_gemm_bf16(const uint8_t* w, int type, int layout, const void* x, void* y, int64_t M, int64_t N, int64_t K,
                  cudaStream_t st, int num_sms) {
  GemmParams p{};
  p.w = w;
  p.y = static_cast<__nv_bfloat16*>(y);
  p.M = M;
  p.N = N;
  p.K = K;
  return run_gemm<false>(p, type, layout, x, st, num_sms);
}

}  // namespace nsq
