// Host side of the products (qk_gemm.cuh): their tensor maps, and the launch for each type.
#include "qk_linear.cuh"

namespace qk {

cudaError_t launch_gemm_bf16(const GemmArgs& a, int bn, cudaStream_t st);
cudaError_t launch_gemm_f32(const GemmArgs& a, int bn, cudaStream_t st);
cudaError_t gave_up_bf16(unsigned* total, cudaStream_t st);
cudaError_t gave_up_f32(unsigned* total, cudaStream_t st);

namespace {

constexpr int kDepth = 64;     // of a stage
constexpr int kTileRows = 128;

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult got = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &got) != cudaSuccess ||
            got != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// `inner` contiguous elements of `el` bytes per row, `outer` rows `ld` elements apart, `planes` of them
bool make_map(CUtensorMap* map, const void* base, int el, long inner, long outer, long ld, int planes, int box_inner,
              int box_outer, CUtensorMapSwizzle swizzle) {
    const EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * el, (cuuint64_t)ld * outer * el};
    const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1}, step[3] = {1, 1, 1};
    return fn(map, el == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// boxes that a stage takes of an operand whose tile has `tile` rows, of which `rows` exist at most: no more than there is
// (what is left of the tile in shared memory is whatever was there; it reaches only rows of C that do not exist)
bool bind_operand(CUtensorMap* map, const Operand& o, int planes, int tile, int rows, int* boxes, int* box_bytes) {
    const int need = rows < tile ? (rows + 7) / 8 * 8 : tile;
    *boxes = o.mn_major ? (need + 63) / 64 : 1;
    const int outer = o.mn_major ? kDepth : need;
    *box_bytes = outer * 128;
    return make_map(map, o.base, 2, o.inner, o.outer, o.ld, planes, 64, outer, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

bool gemm_bind(GemmProblem& g, const Operand& p, const Operand& q, int planes, int bn) {
    g.p_mn = p.mn_major;
    g.q_mn = q.mn_major;
    if (!bind_operand(&g.p_map, p, planes == 1 && g.wrap < g.kblocks ? 2 : planes, kTileRows, g.rows, &g.p_boxes,
                      &g.p_box_bytes) ||
        !bind_operand(&g.q_map, q, planes, bn, g.cols, &g.q_boxes, &g.q_box_bytes))
        return false;
    const int el = planes == 3 ? 4 : 2, out_el = g.part ? 4 : el;
    auto words = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    g.vec = (long)g.cols * el % 16 == 0 && words(g.bias) && words(g.residual);
    void* out = g.part ? static_cast<void*>(g.part) : g.out;
    const bool tape = g.tape && !g.part;  // partial sums leave the tape to the reduction
    g.tma_out = (long)g.cols * out_el % 16 == 0 && words(out) && (!tape || words(g.tape));
    if (!g.tma_out) return true;
    if (!make_map(&g.out_map, out, out_el, g.cols, g.rows, g.cols, g.part ? g.splits : 1, 64 / out_el, 32,
                  CU_TENSOR_MAP_SWIZZLE_64B))
        return false;
    return !tape || make_map(&g.tape_map, g.tape, el, g.cols, g.rows, g.cols, 1, 64 / el, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

cudaError_t launch_gemm(const GemmArgs& a, int planes, int bn, cudaStream_t st) {
    return planes == 3 ? launch_gemm_f32(a, bn, st) : launch_gemm_bf16(a, bn, st);
}

cudaError_t gemm_gave_up(unsigned* count, cudaStream_t st) {
    *count = 0;
    const cudaError_t e = gave_up_bf16(count, st), e2 = gave_up_f32(count, st);
    return e != cudaSuccess ? e : e2;
}

}  // namespace qk
