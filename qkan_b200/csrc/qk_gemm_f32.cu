// The float32 products, three bfloat16 parts per operand (qk_gemm.cuh).
#include "qk_gemm.cuh"

namespace qk {

cudaError_t launch_gemm_f32(const GemmArgs& a, int bn, cudaStream_t st) {
    return bn == 128 ? launch_tile<128, 3>(a, st) : launch_tile<64, 3>(a, st);
}
cudaError_t gave_up_f32(unsigned* total, cudaStream_t st) { return take_gave_up(total, st); }

}  // namespace qk
