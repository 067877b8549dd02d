// The linear map y = act(x W^T + b) + r and its backward pass: C entry points' launch sequence and the plain kernels.
#include "qk_linear.cuh"

namespace qk {
namespace {

constexpr int kTile = 64, kStep = 16, kThreads = 256;

// C[r,c] = sum_k P[r,k] Q[c,k], any strides: one 64 x 64 tile per CTA, 4 x 4 sums per thread.
template <typename IO>
__global__ void __launch_bounds__(kThreads) product_kernel(const Product g) {
    __shared__ float ps[kStep][kTile + 1], qs[kStep][kTile + 1];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const long r0 = (long)blockIdx.y * kTile, c0 = (long)blockIdx.x * kTile;
    const IO* p = static_cast<const IO*>(g.p);
    const IO* q = static_cast<const IO*>(g.q);
    float acc[4][4] = {};
    for (int k0 = 0; k0 < g.depth; k0 += kStep) {
        for (int t = threadIdx.x; t < kTile * kStep; t += kThreads) {
            // neighbouring threads along the contiguous axis of each operand
            const int pr = g.p_kmajor ? t / kStep : t % kTile, pk = g.p_kmajor ? t % kStep : t / kTile;
            const int qc = g.q_kmajor ? t / kStep : t % kTile, qk_ = g.q_kmajor ? t % kStep : t / kTile;
            const bool pin = r0 + pr < g.rows && k0 + pk < g.depth, qin = c0 + qc < g.cols && k0 + qk_ < g.depth;
            const size_t pat = g.p_kmajor ? (size_t)(r0 + pr) * g.depth + k0 + pk : (size_t)(k0 + pk) * g.rows + r0 + pr;
            const size_t qat = g.q_kmajor ? (size_t)(c0 + qc) * g.depth + k0 + qk_ : (size_t)(k0 + qk_) * g.cols + c0 + qc;
            ps[pk][pr] = pin ? as_float(p[pat]) : 0.f;
            qs[qk_][qc] = qin ? as_float(q[qat]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            float pv[4], qv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = ps[k][ty * 4 + i], qv[i] = qs[k][tx + 16 * i];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(pv[i], qv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long r = r0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long c = c0 + tx + 16 * j;
            if (r < g.rows && c < g.cols) finish_element(g.epi, (size_t)r * g.cols + c, (int)c, acc[i][j]);
        }
    }
}

// gz = gy * act'(tape)
__global__ void slope_kernel(const void* gy, const void* tape, void* gz, size_t n, int act, int io_dtype) {
    for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        store_dt(gz, i, io_dtype, load_dt(gy, i, io_dtype) * act_slope(load_tape(tape, i, io_dtype), act));
}

// grad_bias[n] = sum_m gy[m,n] * act'(tape[m,n]): 32 columns per CTA, 32 row slices
__global__ void __launch_bounds__(1024) column_sum_kernel(const void* gy, const void* tape, void* gb, int rows, int cols,
                                                          int act, int io_dtype) {
    __shared__ float tile[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (c < cols)
        for (long r = threadIdx.y; r < rows; r += 32) {
            const size_t at = (size_t)r * cols + c;
            const float g = load_dt(gy, at, io_dtype);
            s += tape ? g * act_slope(load_tape(tape, at, io_dtype), act) : g;
        }
    tile[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < cols) {
        for (int k = 1; k < 32; ++k) s += tile[k][threadIdx.x];
        store_dt(gb, c, io_dtype, s);
    }
}

cudaError_t launch_product(const Product& g, cudaStream_t st) {
    if (g.rows == 0 || g.cols == 0) return cudaSuccess;
    const dim3 grid((g.cols + kTile - 1) / kTile, (g.rows + kTile - 1) / kTile);
    if (grid.y > 65535) return cudaErrorInvalidConfiguration;
    if (g.epi.io_dtype == QK_BF16) product_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(g);
    else product_kernel<float><<<grid, kThreads, 0, st>>>(g);
    return cudaPeekAtLastError();
}

}  // namespace

size_t linear_forward_scratch(const QkLinearDesc&) { return 256; }

size_t linear_backward_scratch(const QkLinearDesc& d) {
    if (d.activation == QK_ACT_NONE) return 256;
    return align256((size_t)d.rows * d.out_features * dtype_bytes(d.io_dtype));
}

cudaError_t launch_linear_forward(const LinearArgs& a, cudaStream_t st) {
    Product g{};
    g.rows = a.rows, g.cols = a.out, g.depth = a.in;
    g.p = a.x, g.q = a.w;
    g.p_kmajor = g.q_kmajor = true;
    g.epi = {a.bias, a.residual, a.y, a.tape, a.act, a.io_dtype};
    return launch_product(g, st);
}

cudaError_t launch_linear_backward(const LinearArgs& a, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    const void* gz = a.gy;
    if (a.act != QK_ACT_NONE && (a.gx || a.gw)) {
        slope_kernel<<<4 * kSms, 256, 0, st>>>(a.gy, a.tape, a.scratch, (size_t)a.rows * a.out, a.act, a.io_dtype);
        e = cudaPeekAtLastError();
        gz = a.scratch;
    }
    if (e == cudaSuccess && a.gx) {
        Product g{};
        g.rows = a.rows, g.cols = a.in, g.depth = a.out;
        g.p = gz, g.q = a.w;
        g.p_kmajor = true, g.q_kmajor = false;
        g.epi = {nullptr, nullptr, a.gx, nullptr, QK_ACT_NONE, a.io_dtype};
        e = launch_product(g, st);
    }
    if (e == cudaSuccess && a.gw) {
        Product g{};
        g.rows = a.out, g.cols = a.in, g.depth = a.rows;
        g.p = gz, g.q = a.x;
        g.epi = {nullptr, nullptr, a.gw, nullptr, QK_ACT_NONE, a.io_dtype};
        e = launch_product(g, st);
    }
    if (e == cudaSuccess && a.gb && a.out) {
        column_sum_kernel<<<(a.out + 31) / 32, dim3(32, 32), 0, st>>>(
            a.gy, a.act == QK_ACT_NONE ? nullptr : a.tape, a.gb, a.rows, a.out, a.act, a.io_dtype);
        e = cudaPeekAtLastError();
    }
    return e;
}

}  // namespace qk
