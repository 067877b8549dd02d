// Argument blocks of the linear map's kernels.
#pragma once

#include <cuda.h>

#include "qk_dense.cuh"

namespace qk {

// ---- tensor-core products (qk_gemm.cu) -----------------------------------------
// C[r,c] = sum_k P[r,k] Q[c,k], C row-major (rows, cols).

// A matrix of bfloat16 as it lies in memory, rows 16-byte aligned; for float32 the three parts follow one another.
struct Operand {
    const void* base;
    long inner, outer, ld;  // contiguous elements, rows, elements from row to row
    bool mn_major;          // the contiguous axis is the product's row (column), not the summed one
};

struct alignas(64) GemmProblem {
    CUtensorMap p_map, q_map, out_map, tape_map;  // out_map: of `part` where there is one
    int rows, cols;
    int kblocks, kper, splits;  // 64-deep blocks in all, per slice of the depth, slices
    int wrap;                   // blocks of one part of P where P has two (Q again for the second); kblocks otherwise
    int tiles_r, tiles_c, units;
    bool p_mn, q_mn;
    int p_boxes, q_boxes, p_box_bytes, q_box_bytes;  // what one stage takes of each operand (and part)
    bool vec;      // bias and residual can be read in 16-byte words
    bool tma_out;  // out (part) and tape can be written by TMA
    float* part;  // splits > 1: [splits][rows][cols] sums, no epilogue; nullptr otherwise
    float* row_sums;  // [splits][rows] sums of P's rows over the depth; nullptr: not wanted (bfloat16, no activation)
    // The epilogue, as in Epilogue. What it lacks points to `out`, so that a load of either is good whether or not it is
    // wanted: where a null pointer stood behind a test, hoisting the load over the test made it a fault.
    bool has_bias, has_residual;
    const void* bias;
    const void* residual;
    void* out;
    void* tape;
    int act;
};

// One launch: one problem, or two that share the SMs, the first `first` CTAs with g[0].
struct GemmArgs {
    GemmProblem g[2];
    int first, ctas;
};

// fills in the tensor maps and what goes with them; false: the driver refused one
bool gemm_bind(GemmProblem& g, const Operand& p, const Operand& q, int planes, int bn);
cudaError_t launch_gemm(const GemmArgs& a, int planes, int bn, cudaStream_t st);
// waits that ran out on the current device since the last call; synchronises the stream
cudaError_t gemm_gave_up(unsigned* count, cudaStream_t st);

// ---- few rows (qk_gemv.cu) -------------------------------------------------------
// Rows up to which it is taken. bfloat16: 2 (at 4096 x 4096, 4 rows took 14 us here and 9 us as a tensor-core product);
// float32, whose products split W first: 16 (8 rows 20 us, as a product 64).
inline bool few_rows(int rows, int io_dtype) { return rows <= (io_dtype == QK_BF16 ? 2 : 16); }
struct GemvArgs {
    int rows, cols, depth;
    const void* x;
    const void* w;
    Epilogue epi;
    int cuts, per;  // filled by the launcher: warps that share the depth, elements of it for each
};
cudaError_t launch_gemv(const GemvArgs& a, cudaStream_t st);

// The backward of a few rows, all gradients in one pass over W.
inline bool few_rows_backward(int rows, int io_dtype) { return rows <= (io_dtype == QK_BF16 ? 4 : 16); }
struct FewArgs {
    int rows, in, out, act, io_dtype;
    const void* x;
    const void* w;
    const void* gy;
    const void* tape;
    float* gx_part;  // [slabs][rows][in] sums; nullptr: grad_x not wanted
    void* gw;
    void* gb;
    int blocks, slab;  // CTAs side by side, rows of W for each
};
struct FewPlan {
    int blocks, slab, slabs;
};
FewPlan few_plan(int in, int out);
cudaError_t launch_few_backward(const FewArgs& a, cudaStream_t st);

// ---- few outputs, or few of everything, in float32 (qk_narrow.cu) ------------------
// Few of them: up to 32 (48: 8192 x 768 39 us here, 20 on the tensor cores). And small products, where the launch that
// prepares the operands counts: up to 2^24 multiplications (us here and there: 64 x 64 -> 64 4.6 and 7.5, 256 x 256 -> 256
// 7.9 and 11.3, 333 x 517 -> 333 18.3 and 16.6) for up to 2^18 results (344 x 18 -> 3416 15.4 and 13.7).
inline bool is_narrow(long rows, long cols, long depth, int io_dtype) {
    if (io_dtype != QK_F32) return false;
    return cols <= 32 || (rows * cols <= 1 << 18 && rows * cols * depth <= 1 << 24);
}
struct NarrowPlan {
    int tm;                   // rows of a thread
    int chunks, per, splits;  // chunks of the depth in all, per slice, slices
};
NarrowPlan narrow_plan(int rows, int cols, int depth);
struct NarrowArgs : NarrowPlan {
    int rows, cols, depth;
    const void* x;
    const void* w;
    float* part;  // splits > 1: [splits][rows][cols] sums, no epilogue; nullptr otherwise
    Epilogue epi;
};
cudaError_t launch_narrow(const NarrowArgs& a, cudaStream_t st);

// ---- the map (qk_linear.cu) ----------------------------------------------------
struct LinearArgs {
    int rows, in, out, act, io_dtype;
    uint32_t flags;
    const void* x;
    const void* w;
    const void* bias;
    const void* residual;
    void* y;
    void* tape;
    const void* gy;
    void* gx;
    void* gw;
    void* gb;
    void* scratch;
};

// of product 0 (forward), 1 (grad_weight), 2 (grad_x)
QkLinearPlan linear_plan(const QkLinearDesc& d, int product);
// bytes of scratch
size_t linear_forward_scratch(const QkLinearDesc& d);
size_t linear_backward_scratch(const QkLinearDesc& d);
// whether the products read rows of `width` elements in place, which then have to start on a 16-byte boundary
inline bool reads_in_place(int width, int io_dtype) { return io_dtype == QK_BF16 && width % 8 == 0; }
cudaError_t launch_linear_forward(const LinearArgs& a, cudaStream_t st);
cudaError_t launch_linear_backward(const LinearArgs& a, cudaStream_t st);

}  // namespace qk
