// The bfloat16 products (qk_gemm.cuh).
#include "qk_gemm.cuh"

namespace qk {

cudaError_t launch_gemm_bf16(const GemmArgs& a, int bn, cudaStream_t st) {
    if (bn == 256) return launch_tile<256, 1>(a, st);
    return bn == 128 ? launch_tile<128, 1>(a, st) : launch_tile<64, 1>(a, st);
}
cudaError_t gave_up_bf16(unsigned* total, cudaStream_t st) { return take_gave_up(total, st); }

}  // namespace qk
