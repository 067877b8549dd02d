// Argument blocks of the linear map's kernels.
#pragma once

#include "qk_dense.cuh"

namespace qk {

// One matrix product: C[r,c] = sum_k P[r,k] Q[c,k], C row-major (rows, cols). P is stored (rows, depth) when p_kmajor
// and (depth, rows) otherwise; Q likewise with cols.
struct Product {
    int rows, cols, depth;
    const void* p;
    const void* q;
    bool p_kmajor, q_kmajor;
    Epilogue epi;
};

struct LinearArgs {
    int rows, in, out, act, io_dtype;
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

// bytes of scratch (0: a product too large for the launch grid)
size_t linear_forward_scratch(const QkLinearDesc& d);
size_t linear_backward_scratch(const QkLinearDesc& d);
cudaError_t launch_linear_forward(const LinearArgs& a, cudaStream_t st);
cudaError_t launch_linear_backward(const LinearArgs& a, cudaStream_t st);

}  // namespace qk
