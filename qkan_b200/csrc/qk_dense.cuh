// Shared pieces of the dense operators (layer norm, linear map with epilogue): typed loads, activations, argument
// blocks and launchers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qk_kernels.cuh"

namespace qk {

constexpr int kSms = 148;

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The kernels of these operators follow one another closely, and each may be set up while the one before it drains
// (programmatic dependent launch). So each calls after_previous() before it touches anything in global memory, and
// lets its own successor come as soon as its CTAs are all placed.
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... K, typename... A>
cudaError_t launch_after(void (*kernel)(K...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cfg.attrs = &at, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// one element of a tensor whose QkDtype is known at run time only
__device__ __forceinline__ float load_dt(const void* p, size_t i, int dtype) {
    return dtype == QK_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                            : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_dt(void* p, size_t i, int dtype, float v) {
    if (dtype == QK_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<float*>(p)[i] = v;
}
inline size_t dtype_bytes(int dtype) { return dtype == QK_BF16 ? 2 : 4; }

struct NormArgs {
    int rows, dim, io_dtype, param_dtype;
    float eps;
    const void* x;
    const void* w;  // nullptr: ones
    const void* b;  // nullptr: zeros
    void* y;
    float2* stats_out;     // (mean, rstd) of each row; nullptr: not wanted
    const float2* stats;
    const void* gy;
    void* gx;              // nullptr: not wanted
    void* gw;
    void* gb;
    float* part;           // [2][slices][dim] partial sums of gw, gb
};
// slices of the backward's partial sums for this problem
int norm_slices(int rows, int dim, int io_dtype, int param_dtype);
cudaError_t launch_norm_forward(const NormArgs& a, cudaStream_t st);
cudaError_t launch_norm_backward(const NormArgs& a, cudaStream_t st);

// ---- linear map --------------------------------------------------------------
// act(z) and its derivative in float32, by CUDA's own functions. FAST, for values that are rounded to bfloat16 next: exp
// and the reciprocal by the special-function unit (off by some 2^-20 where bfloat16 is off by 2^-9). tanh and erf are the
// full ones throughout: near zero theirs is a relative error.
template <bool FAST>
__device__ __forceinline__ float exp_of(float z) {
    if constexpr (FAST) {  // without the steps that keep results below float32's normal numbers
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(z * 1.44269504088896341f));
        return r;
    } else {
        return expf(z);
    }
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_of(float z) {
    if constexpr (FAST) {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + exp_of<FAST>(-z)));
        return r;
    } else {
        return __fdividef(1.f, 1.f + expf(-z));  // off by 2 steps at most; the exact quotient took twice as long
    }
}
template <bool FAST>
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case QK_ACT_SILU: return FAST ? z * sigmoid_of<FAST>(z) : __fdividef(z, 1.f + expf(-z));
        case QK_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
        case QK_ACT_GELU_TANH: return 0.5f * z * (1.f + tanhf(0.79788456080286536f * fmaf(0.044715f * z * z, z, z)));
        case QK_ACT_RELU: return z < 0.f ? 0.f : z;  // a NaN stays one
        case QK_ACT_TANH: return tanhf(z);
        case QK_ACT_SIGMOID: return sigmoid_of<FAST>(z);
        default: return z;
    }
}
// Beyond +-10^4 every derivative has reached its limit, which is what an infinite z (and one that the tape holds as such)
// gets; a NaN passes, but for relu, whose derivative is 1 above 0 and 0 elsewhere (torch's lets the gradient through at NaN).
template <bool FAST>
__device__ __forceinline__ float act_slope(float z, int act) {
    asm("{max.NaN.f32 %0, %0, %1;\n min.NaN.f32 %0, %0, %2;}" : "+f"(z) : "f"(-1e4f), "f"(1e4f));
    switch (act) {
        case QK_ACT_SILU: {
            const float s = sigmoid_of<FAST>(z);
            return s * fmaf(z, 1.f - s, 1.f);
        }
        case QK_ACT_GELU: {
            const float e = exp_of<FAST>(-0.5f * z * z);
            return fmaf(z * 0.39894228040143268f, e, 0.5f * (1.f + erff(z * 0.70710678118654752f)));
        }
        case QK_ACT_GELU_TANH: {
            const float t = tanhf(0.79788456080286536f * fmaf(0.044715f * z * z, z, z));
            return 0.5f * (1.f + t) +
                   0.5f * z * (1.f - t * t) * 0.79788456080286536f * fmaf(3.f * 0.044715f * z, z, 1.f);
        }
        case QK_ACT_RELU: return z > 0.f ? 1.f : 0.f;
        case QK_ACT_TANH: {
            const float t = tanhf(z);
            return 1.f - t * t;
        }
        case QK_ACT_SIGMOID: {
            const float s = sigmoid_of<FAST>(z);
            return s * (1.f - s);
        }
        default: return 1.f;
    }
}
// the same for N values at once, one test of `act` for all
template <bool FAST, int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
    switch (act) {
#define QK_CASE(code)                                                                 \
    case code:                                                                        \
        _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] = activate<FAST>(v[i], code); \
        break;
        QK_CASE(QK_ACT_SILU)
        QK_CASE(QK_ACT_GELU)
        QK_CASE(QK_ACT_GELU_TANH)
        QK_CASE(QK_ACT_RELU)
        QK_CASE(QK_ACT_TANH)
        QK_CASE(QK_ACT_SIGMOID)
        default: break;
    }
}
template <bool FAST, int N>
__device__ __forceinline__ void times_slope(float (&v)[N], const float (&z)[N], int act) {
    switch (act) {
#undef QK_CASE
#define QK_CASE(code)                                                                      \
    case code:                                                                             \
        _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] *= act_slope<FAST>(z[i], code); \
        break;
        QK_CASE(QK_ACT_SILU)
        QK_CASE(QK_ACT_GELU)
        QK_CASE(QK_ACT_GELU_TANH)
        QK_CASE(QK_ACT_RELU)
        QK_CASE(QK_ACT_TANH)
        QK_CASE(QK_ACT_SIGMOID)
#undef QK_CASE
        default: break;
    }
}

// The tape: float32, or half for bfloat16 activations. Rounding an argument of the activation to half moves it by at
// most 2^-12 of itself (2^-9 in bfloat16). What is beyond half's range becomes infinite, where the derivatives have their
// limits; what is below it becomes zero, which matters to relu alone: its tape keeps the sign as half's smallest number.
__device__ __forceinline__ __half tape_half(float z, int act) {
    const __half h = __float2half_rn(z);
    if (act == QK_ACT_RELU && z != 0.f && __half2float(h) == 0.f) return __ushort_as_half(z < 0.f ? 0x8001 : 0x0001);
    return h;
}
__device__ __forceinline__ void store_tape(void* tape, size_t i, int io_dtype, float z, int act) {
    if (io_dtype == QK_BF16) static_cast<__half*>(tape)[i] = tape_half(z, act);
    else static_cast<float*>(tape)[i] = z;
}
__device__ __forceinline__ float load_tape(const void* tape, size_t i, int io_dtype) {
    return io_dtype == QK_BF16 ? __half2float(static_cast<const __half*>(tape)[i]) : static_cast<const float*>(tape)[i];
}

// What becomes of the sums acc[r,c]: z = acc + bias[c]; tape = z; out = act(z) + residual[r,c]
struct Epilogue {
    const void* bias;      // nullptr: none
    const void* residual;  // nullptr: none; row-major, `cols` wide, like out and tape
    void* out;
    void* tape;            // nullptr: not wanted
    int act, io_dtype;
};
__device__ __forceinline__ void finish_element(const Epilogue& e, size_t at, int c, float acc) {
    float z = acc;
    if (e.bias) z += load_dt(e.bias, c, e.io_dtype);
    if (e.tape) store_tape(e.tape, at, e.io_dtype, z, e.act);
    float y = e.io_dtype == QK_BF16 ? activate<true>(z, e.act) : activate<false>(z, e.act);
    if (e.residual) y += load_dt(e.residual, at, e.io_dtype);
    store_dt(e.out, at, e.io_dtype, y);
}

}  // namespace qk
