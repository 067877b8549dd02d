// Layer norm, forward and backward.
//
//   xh = (x - mean) * rstd          y = xh * w + b
//   gx = rstd * (gw - mean(gw) - xh * mean(gw * xh)),  gw = gy * w
//   grad_w = sum over rows of gy * xh                  grad_b = sum over rows of gy
//
// Bound by memory: 2 M D elements forward, 3 M D backward. So each row is read once: T threads hold it in registers
// (16 elements each), take the mean, then the squares about the mean (no cancellation, whatever the row's offset), and
// write. The backward walks rows with a fixed set of CTAs, so that the threads' own columns of grad_w and grad_b stay in
// registers over all their rows; one partial row per CTA goes to scratch, and a second launch adds those in order (no
// atomics: the same bits every run). The next row's x and gy are fetched before the current one is worked on.
#include <type_traits>

#include "qk_dense.cuh"

namespace qk {
namespace {

constexpr int kElems = 16;      // of a row, per thread
constexpr int kMaxT = 512;      // threads of a row: rows up to 8192 stay in registers, wider ones are read again
constexpr int kWideThreads = 256;
constexpr int kFinishSlices = 32;

__host__ __device__ constexpr int block_of(int t) { return t < 256 ? 256 : t; }

// The part of one row that a thread holds: NV vectors of VEC elements, vector j at column (j * T + lane) * VEC.
template <typename IO, int VEC, int T>
struct Piece {
    static constexpr int NV = kElems / VEC;
    using Raw = std::conditional_t<VEC == 1, IO, uint4>;
    Raw v[NV];
    __device__ __forceinline__ void load(const IO* row, int dim, int lane) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * T + lane) * VEC;
            v[j] = Raw{};
            if (c < dim) v[j] = *reinterpret_cast<const Raw*>(row + c);
        }
    }
    __device__ __forceinline__ void unpack(float (&f)[kElems]) const {
        if constexpr (VEC == 1) {
#pragma unroll
            for (int j = 0; j < NV; ++j) f[j] = as_float(v[j]);
        } else if constexpr (VEC == 4) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                f[4 * j] = __uint_as_float(v[j].x);
                f[4 * j + 1] = __uint_as_float(v[j].y);
                f[4 * j + 2] = __uint_as_float(v[j].z);
                f[4 * j + 3] = __uint_as_float(v[j].w);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const unsigned u[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    f[8 * j + 2 * k] = __uint_as_float(u[k] << 16);
                    f[8 * j + 2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
                }
            }
        }
    }
};

template <typename IO, int VEC>
__device__ __forceinline__ void store_vec(IO* at, const float* f) {
    if constexpr (VEC == 1) {
        *at = from_float<IO>(f[0]);
    } else if constexpr (VEC == 4) {
        *reinterpret_cast<float4*>(at) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        unsigned u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
            u[k] = *reinterpret_cast<const unsigned*>(&h);
        }
        *reinterpret_cast<uint4*>(at) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// VEC parameters from column c on; `p` null gives `other`
template <int VEC>
__device__ __forceinline__ void load_params(const void* p, int dtype, int c, float other, float* f) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = other;
    } else if constexpr (VEC == 1) {
        f[0] = load_dt(p, c, dtype);
    } else if (dtype == QK_F32) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + i);
            f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + c + i);
            f[i] = __uint_as_float(v.x << 16), f[i + 1] = __uint_as_float(v.x & 0xffff0000u);
            f[i + 2] = __uint_as_float(v.y << 16), f[i + 3] = __uint_as_float(v.y & 0xffff0000u);
        }
    }
}

// Sums over the T threads of a group. Two buffers used in turn make one barrier per sum enough: who writes a buffer
// again has passed the barrier of the sum between, behind which nobody reads it any more.
template <int T>
struct GroupSum {
    float2* buf;  // [2][T / 32]
    int group, flip;
    __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            v.x += __shfl_xor_sync(~0u, v.x, o);
            v.y += __shfl_xor_sync(~0u, v.y, o);
        }
        if constexpr (T > 32) {
            float2* b = buf + flip * (T / 32);
            flip ^= 1;
            if (threadIdx.x % 32 == 0) b[threadIdx.x % T / 32] = v;
            asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(T) : "memory");
            v = b[0];
#pragma unroll
            for (int k = 1; k < T / 32; ++k) {
                v.x += b[k].x;
                v.y += b[k].y;
            }
        }
        return v;
    }
};

template <typename IO, int VEC, int T>
__global__ void __launch_bounds__(block_of(T)) norm_forward_kernel(const NormArgs a) {
    after_previous();
    constexpr int G = block_of(T) / T;
    __shared__ float2 buf[G][2][T / 32];
    const int group = threadIdx.x / T, lane = threadIdx.x % T;
    const long row = (long)blockIdx.x * G + group;
    if (row >= a.rows) return;  // a whole group leaves together: its barrier counts its own threads only
    GroupSum<T> sum{&buf[group][0][0], group, 0};
    Piece<IO, VEC, T> p;
    p.load(static_cast<const IO*>(a.x) + row * a.dim, a.dim, lane);
    float x[kElems];
    p.unpack(x);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kElems; ++e) s += x[e];  // columns past the end hold zeros
    const float mean = sum(make_float2(s, 0.f)).x / a.dim;
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
        const int c = (e / VEC * T + lane) * VEC;
        x[e] -= mean;
        if (c < a.dim) q = fmaf(x[e], x[e], q);
    }
    const float rstd = 1.f / sqrtf(sum(make_float2(q, 0.f)).x / a.dim + a.eps);
    if (lane == 0 && a.stats_out) a.stats_out[row] = make_float2(mean, rstd);
    IO* y = static_cast<IO*>(a.y) + row * a.dim;
#pragma unroll
    for (int j = 0; j < kElems / VEC; ++j) {
        const int c = (j * T + lane) * VEC;
        if (c >= a.dim) continue;
        float w[VEC], b[VEC], o[VEC];
        load_params<VEC>(a.w, a.param_dtype, c, 1.f, w);
        load_params<VEC>(a.b, a.param_dtype, c, 0.f, b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = fmaf(x[j * VEC + i] * rstd, w[i], b[i]);
        store_vec<IO, VEC>(y + c, o);
    }
}

template <typename IO, int VEC, int T>
__global__ void __launch_bounds__(block_of(T)) norm_backward_kernel(const NormArgs a) {
    after_previous();
    constexpr int G = block_of(T) / T;
    __shared__ float2 buf[G][2][T / 32];
    __shared__ float cols[G > 1 ? G * T * kElems : 1];
    const int group = threadIdx.x / T, lane = threadIdx.x % T;
    GroupSum<T> sum{&buf[group][0][0], group, 0};
    float dw[kElems], db[kElems];
#pragma unroll
    for (int e = 0; e < kElems; ++e) dw[e] = db[e] = 0.f;
    const IO* xs = static_cast<const IO*>(a.x);
    const IO* gys = static_cast<const IO*>(a.gy);
    const long step = (long)gridDim.x * G;
    long row = (long)blockIdx.x * G + group;
    Piece<IO, VEC, T> px, pg;
    float2 st{};
    if (row < a.rows) {
        px.load(xs + row * a.dim, a.dim, lane);
        pg.load(gys + row * a.dim, a.dim, lane);
        st = a.stats[row];
    }
    for (; row < a.rows; row += step) {
        float xh[kElems], g[kElems];
        px.unpack(xh);
        pg.unpack(g);
        const float mean = st.x, rstd = st.y;
        if (row + step < a.rows) {
            px.load(xs + (row + step) * a.dim, a.dim, lane);
            pg.load(gys + (row + step) * a.dim, a.dim, lane);
            st = a.stats[row + step];
        }
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < kElems / VEC; ++j) {
            const int c = (j * T + lane) * VEC;
            if (c >= a.dim) continue;
            float w[VEC];
            load_params<VEC>(a.w, a.param_dtype, c, 1.f, w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int e = j * VEC + i;
                xh[e] = (xh[e] - mean) * rstd;
                dw[e] = fmaf(g[e], xh[e], dw[e]);
                db[e] += g[e];
                g[e] *= w[i];
                s.x += g[e];
                s.y = fmaf(g[e], xh[e], s.y);
            }
        }
        if (!a.gx) continue;
        s = sum(s);
        const float m1 = s.x / a.dim, m2 = s.y / a.dim;
        IO* gx = static_cast<IO*>(a.gx) + row * a.dim;
#pragma unroll
        for (int j = 0; j < kElems / VEC; ++j) {
            const int c = (j * T + lane) * VEC;
            if (c >= a.dim) continue;
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int e = j * VEC + i;
                o[i] = (g[e] - m1 - xh[e] * m2) * rstd;
            }
            store_vec<IO, VEC>(gx + c, o);
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = a.part + ((size_t)which * gridDim.x + blockIdx.x) * a.dim;
        if constexpr (G == 1) {
#pragma unroll
            for (int e = 0; e < kElems; ++e) {
                const int c = (e / VEC * T + lane) * VEC + e % VEC;
                if (c < a.dim) out[c] = which ? db[e] : dw[e];
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kElems; ++e)
                cols[group * T * kElems + (e / VEC * T + lane) * VEC + e % VEC] = which ? db[e] : dw[e];
            __syncthreads();
            for (int c = threadIdx.x; c < a.dim; c += block_of(T)) {
                float s = cols[c];
#pragma unroll
                for (int k = 1; k < G; ++k) s += cols[k * T * kElems + c];
                out[c] = s;
            }
        }
    }
}

// Rows wider than the registers of a group hold: one CTA per row, which reads the row once per pass (from L2 after the
// first).
template <typename IO>
__global__ void __launch_bounds__(kWideThreads) norm_wide_forward_kernel(const NormArgs a) {
    after_previous();
    __shared__ float2 buf[2][kWideThreads / 32];
    GroupSum<kWideThreads> sum{&buf[0][0], 0, 0};
    const size_t at = (size_t)blockIdx.x * a.dim;
    const IO* x = static_cast<const IO*>(a.x) + at;
    float s = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += kWideThreads) s += as_float(x[c]);
    const float mean = sum(make_float2(s, 0.f)).x / a.dim;
    float q = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += kWideThreads) {
        const float d = as_float(x[c]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(sum(make_float2(q, 0.f)).x / a.dim + a.eps);
    if (threadIdx.x == 0 && a.stats_out) a.stats_out[blockIdx.x] = make_float2(mean, rstd);
    IO* y = static_cast<IO*>(a.y) + at;
    for (int c = threadIdx.x; c < a.dim; c += kWideThreads) {
        const float w = a.w ? load_dt(a.w, c, a.param_dtype) : 1.f, b = a.b ? load_dt(a.b, c, a.param_dtype) : 0.f;
        y[c] = from_float<IO>(fmaf((as_float(x[c]) - mean) * rstd, w, b));
    }
}

template <typename IO>
__global__ void __launch_bounds__(kWideThreads) norm_wide_gx_kernel(const NormArgs a) {
    after_previous();
    __shared__ float2 buf[2][kWideThreads / 32];
    GroupSum<kWideThreads> sum{&buf[0][0], 0, 0};
    const size_t at = (size_t)blockIdx.x * a.dim;
    const IO* x = static_cast<const IO*>(a.x) + at;
    const IO* gy = static_cast<const IO*>(a.gy) + at;
    IO* gx = static_cast<IO*>(a.gx) + at;
    const float2 st = a.stats[blockIdx.x];
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < a.dim; c += kWideThreads) {
        const float g = as_float(gy[c]) * (a.w ? load_dt(a.w, c, a.param_dtype) : 1.f);
        s.x += g;
        s.y = fmaf(g, (as_float(x[c]) - st.x) * st.y, s.y);
    }
    s = sum(s);
    const float m1 = s.x / a.dim, m2 = s.y / a.dim;
    for (int c = threadIdx.x; c < a.dim; c += kWideThreads) {
        const float g = as_float(gy[c]) * (a.w ? load_dt(a.w, c, a.param_dtype) : 1.f);
        gx[c] = from_float<IO>((g - m1 - (as_float(x[c]) - st.x) * st.y * m2) * st.y);
    }
}

// partial sums of grad_w and grad_b: one thread per column, one slice of rows per blockIdx.y
template <typename IO>
__global__ void __launch_bounds__(kWideThreads) norm_wide_param_kernel(const NormArgs a) {
    after_previous();
    const int c = blockIdx.x * kWideThreads + threadIdx.x;
    if (c >= a.dim) return;
    const IO* x = static_cast<const IO*>(a.x) + c;
    const IO* gy = static_cast<const IO*>(a.gy) + c;
    float dw = 0.f, db = 0.f;
    for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float2 st = a.stats[r];
        const float g = as_float(gy[r * a.dim]);
        dw = fmaf(g, (as_float(x[r * a.dim]) - st.x) * st.y, dw);
        db += g;
    }
    a.part[(size_t)blockIdx.y * a.dim + c] = dw;
    a.part[((size_t)gridDim.y + blockIdx.y) * a.dim + c] = db;
}

// grad_w (blockIdx.y 0) and grad_b (1): adds the slices of 32 columns, each in a fixed order
__global__ void __launch_bounds__(32 * kFinishSlices) norm_finish_kernel(const NormArgs a, int slices) {
    after_previous();
    __shared__ float tile[kFinishSlices][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    void* out = blockIdx.y ? a.gb : a.gw;
    if (!out) return;
    const float* part = a.part + (size_t)blockIdx.y * slices * a.dim;
    float s = 0.f;
    if (c < a.dim)
        for (int k = threadIdx.y; k < slices; k += kFinishSlices) s += part[(size_t)k * a.dim + c];
    tile[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < a.dim) {
#pragma unroll
        for (int k = 1; k < kFinishSlices; ++k) s += tile[k][threadIdx.x];
        store_dt(out, c, a.param_dtype, s);
    }
}

bool is_wide(int dim) { return dim > kMaxT * kElems; }

// threads of a row: the smallest power of two whose registers hold it
int threads_of(int dim) {
    int t = 32;
    while (t < kMaxT && t * kElems < dim) t *= 2;
    return t;
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

template <typename IO, int VEC, int T>
cudaError_t run_t(const NormArgs& a, bool backward, cudaStream_t st) {
    constexpr int G = block_of(T) / T;
    if (backward) return launch_after(norm_backward_kernel<IO, VEC, T>, norm_slices(a.rows, a.dim), block_of(T), 0, st, a);
    return launch_after(norm_forward_kernel<IO, VEC, T>, (unsigned)((a.rows + G - 1L) / G), block_of(T), 0, st, a);
}

template <typename IO, int VEC>
cudaError_t run_vec(const NormArgs& a, bool backward, cudaStream_t st) {
    switch (threads_of(a.dim)) {
        case 32: return run_t<IO, VEC, 32>(a, backward, st);
        case 64: return run_t<IO, VEC, 64>(a, backward, st);
        case 128: return run_t<IO, VEC, 128>(a, backward, st);
        case 256: return run_t<IO, VEC, 256>(a, backward, st);
        default: return run_t<IO, VEC, 512>(a, backward, st);
    }
}

template <typename IO>
cudaError_t run_rows(const NormArgs& a, bool backward, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(IO);
    // 16-byte accesses where every row of every tensor starts on such a boundary
    const bool vec = a.dim % VEC == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.gy) && aligned16(a.gx) &&
                     aligned16(a.w) && aligned16(a.b);
    return vec ? run_vec<IO, VEC>(a, backward, st) : run_vec<IO, 1>(a, backward, st);
}

template <typename IO>
cudaError_t run_wide(const NormArgs& a, bool backward, cudaStream_t st) {
    if (!backward) return launch_after(norm_wide_forward_kernel<IO>, a.rows, kWideThreads, 0, st, a);
    cudaError_t e = cudaSuccess;
    if (a.gx) e = launch_after(norm_wide_gx_kernel<IO>, a.rows, kWideThreads, 0, st, a);
    if (e == cudaSuccess && a.part)
        e = launch_after(norm_wide_param_kernel<IO>,
                         dim3((a.dim + kWideThreads - 1) / kWideThreads, norm_slices(a.rows, a.dim)), kWideThreads, 0, st, a);
    return e;
}

cudaError_t run(const NormArgs& a, bool backward, cudaStream_t st) {
    const bool half = a.io_dtype == QK_BF16;
    if (is_wide(a.dim)) return half ? run_wide<__nv_bfloat16>(a, backward, st) : run_wide<float>(a, backward, st);
    return half ? run_rows<__nv_bfloat16>(a, backward, st) : run_rows<float>(a, backward, st);
}

}  // namespace

int norm_slices(int rows, int dim) {
    if (is_wide(dim)) return rows < 64 ? rows : 64;
    const int t = threads_of(dim), g = block_of(t) / t;
    const int most = kSms * (block_of(t) == 256 ? 2 : 1);
    const int need = (int)((rows + (long)g - 1) / g);
    return need < most ? need : most;
}

cudaError_t launch_norm_forward(const NormArgs& a, cudaStream_t st) { return run(a, false, st); }

cudaError_t launch_norm_backward(const NormArgs& a, cudaStream_t st) {
    const cudaError_t e = run(a, true, st);
    if (e != cudaSuccess || !a.part) return e;
    return launch_after(norm_finish_kernel, dim3((a.dim + 31) / 32, 2), dim3(32, kFinishSlices), 0, st, a,
                        norm_slices(a.rows, a.dim));
}

}  // namespace qk
