// Layer norm, forward and backward.
//
//   xh = (x - mean) * rstd          y = xh * w + b
//   gx = rstd * (gw - mean(gw) - xh * mean(gw * xh)),  gw = gy * w
//   grad_w = sum over rows of gy * xh                  grad_b = sum over rows of gy
//
// Bound by memory: 2 M D elements forward, 3 M D backward. So each row is read once: T threads hold it in registers, E
// elements each, take the mean, then the squares about the mean, and write. Both directions take x - mean first, which for
// values near the mean is exact (x * rstd - mean * rstd would round mean * rstd, an error that grows with the row's offset).
// A fixed set of CTAs walks the rows, so that weight and bias, and in the backward the threads' own columns of grad_w and
// grad_b, stay in registers; one partial row per CTA goes to scratch, and a second launch adds those in order (no
// atomics: the same bits every run). The next row is fetched before the current one is worked on.
//
// A warp takes a whole row where it can: then the sums need no barrier, and their cost is spread over up to 24
// elements per thread. (With 16 elements per thread and weight and bias read again for every row, bfloat16 rows were bound by
// instructions, at half of float32's bandwidth.)
//
// Measured: 16384 x 4096 float32 forward 87 us (6.2 TB/s), backward 139 us (5.8 TB/s); 65536 x 768 bfloat16 36.9 us (5.5 TB/s)
// and 64.1 us (4.7 TB/s); 8192 x 768 bfloat16 5.2 us and 12.8 us, of which the second launch is 4; one row 1.7 us.
#include <type_traits>

#include "qk_dense.cuh"
#include "qk_packed.cuh"

namespace qk {
namespace {

constexpr int kMaxT = 512;       // threads of a row, 16 elements each at least: rows up to 8192 stay in registers,
constexpr int kMaxDim = 8192;    // wider ones are read again
constexpr int kWideThreads = 256;
constexpr int kFinishSlices = 32;

__host__ __device__ constexpr int block_of(int t) { return t < 256 ? 256 : t; }

// The part of one row that a thread holds: NV vectors of VEC elements, vector j at column (j * T + lane) * VEC.
template <typename IO, int VEC, int T, int E>
struct Piece {
    static constexpr int NV = E / VEC;
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
    __device__ __forceinline__ void unpack(f2 (&f)[E / 2]) const {
        if constexpr (VEC == 1) {
#pragma unroll
            for (int j = 0; j < NV; j += 2) f[j / 2] = make_float2(as_float(v[j]), as_float(v[j + 1]));
        } else if constexpr (VEC == 4) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                f[2 * j] = make_float2(__uint_as_float(v[j].x), __uint_as_float(v[j].y));
                f[2 * j + 1] = make_float2(__uint_as_float(v[j].z), __uint_as_float(v[j].w));
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const unsigned u[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    f[4 * j + k] = make_float2(__uint_as_float(u[k] << 16), __uint_as_float(u[k] & 0xffff0000u));
            }
        }
    }
};

// element e of a thread's values
template <int N>
__device__ __forceinline__ float at(const f2 (&f)[N], int e) {
    return e % 2 ? f[e / 2].y : f[e / 2].x;
}

// the thread's values to its columns of a row
template <typename IO, int VEC, int T, int E>
__device__ __forceinline__ void store_row(IO* row, int dim, int lane, const f2 (&f)[E / 2]) {
#pragma unroll
    for (int j = 0; j < E / VEC; ++j) {
        const int c = (j * T + lane) * VEC;
        if (c >= dim) continue;
        if constexpr (VEC == 1) {
            row[c] = from_float<IO>(at(f, j));
        } else if constexpr (VEC == 4) {
            *reinterpret_cast<float4*>(row + c) = make_float4(f[2 * j].x, f[2 * j].y, f[2 * j + 1].x, f[2 * j + 1].y);
        } else {
            unsigned u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[4 * j + k].x, f[4 * j + k].y);
                u[k] = *reinterpret_cast<const unsigned*>(&h);
            }
            *reinterpret_cast<uint4*>(row + c) = make_uint4(u[0], u[1], u[2], u[3]);
        }
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

// sum / dim, correctly rounded but for rare last bits, so that the mean of a constant row is that constant; `inv` is 1 / dim
__device__ __forceinline__ float mean_of(float sum, float dim, float inv) {
    const float m = sum * inv;
    return fmaf(fmaf(-m, dim, sum), inv, m);
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

// the thread's parameters, columns behind the row's end as `other`
template <int VEC, int T, int E>
__device__ __forceinline__ void own_params(const void* p, int dtype, int dim, int lane, float other, f2 (&f)[E / 2]) {
    float v[E];
#pragma unroll
    for (int j = 0; j < E / VEC; ++j) {
        const int c = (j * T + lane) * VEC;
        load_params<VEC>(c < dim ? p : nullptr, dtype, c, other, v + j * VEC);
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) f[i] = make_float2(v[2 * i], v[2 * i + 1]);
}

// CTAs of 256 threads: two on an SM at least, so 128 registers at most. Arithmetic on pairs: one issue slot for both.
template <typename IO, int VEC, int T, int E>
__global__ void __launch_bounds__(block_of(T), 512 / block_of(T)) norm_forward_kernel(const NormArgs a) {
    constexpr int G = block_of(T) / T;
    __shared__ float2 buf[G][2][T / 32];
    after_previous();
    const int group = threadIdx.x / T, lane = threadIdx.x % T;
    GroupSum<T> sum{&buf[group][0][0], group, 0};
    const IO* xs = static_cast<const IO*>(a.x);
    const long step = (long)gridDim.x * G;
    long row = (long)blockIdx.x * G + group;  // a whole group leaves together: its barrier counts its own threads only
    Piece<IO, VEC, T, E> p;
    if (row < a.rows) p.load(xs + row * a.dim, a.dim, lane);
    f2 w[E / 2], b[E / 2];
    own_params<VEC, T, E>(a.w, a.param_dtype, a.dim, lane, 1.f, w);
    own_params<VEC, T, E>(a.b, a.param_dtype, a.dim, lane, 0.f, b);
    const float inv = 1.f / a.dim;
    for (; row < a.rows; row += step) {
        f2 x[E / 2], s = pk(0.f);
        p.unpack(x);
        if (row + step < a.rows) p.load(xs + (row + step) * a.dim, a.dim, lane);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) s = add2(s, x[i]);  // columns past the end hold zeros
        const float mean = mean_of(sum(make_float2(s.x + s.y, 0.f)).x, (float)a.dim, inv);
        f2 q = pk(0.f);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            x[i] = add2(x[i], pk(-mean));
            // and stay zero there: an end falls between the pairs of a vector, but within one of single elements
            if ((2 * i / VEC * T + lane) * VEC >= a.dim) x[i].x = 0.f;
            if (((2 * i + 1) / VEC * T + lane) * VEC >= a.dim) x[i].y = 0.f;
            q = fma2(x[i], x[i], q);
        }
        const float rstd = rsqrtf(sum(make_float2(q.x + q.y, 0.f)).x * inv + a.eps);
        if (lane == 0 && a.stats_out) a.stats_out[row] = make_float2(mean, rstd);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) x[i] = fma2(mul2(x[i], pk(rstd)), w[i], b[i]);
        store_row<IO, VEC, T, E>(static_cast<IO*>(a.y) + row * a.dim, a.dim, lane, x);
    }
}

template <typename IO, int VEC, int T, int E>
__global__ void __launch_bounds__(block_of(T), 512 / block_of(T)) norm_backward_kernel(const NormArgs a) {
    constexpr int G = block_of(T) / T;
    constexpr bool kKeepW = sizeof(IO) == 2;  // float32 rows leave no registers for the weight: from L1 for every row
    __shared__ float2 buf[G][2][T / 32];
    __shared__ __align__(16) float cols[2][G > 1 ? G * T * E : 1];
    after_previous();
    const int group = threadIdx.x / T, lane = threadIdx.x % T;
    GroupSum<T> sum{&buf[group][0][0], group, 0};
    f2 dw[E / 2], db[E / 2], w[kKeepW ? E / 2 : 1];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) dw[i] = db[i] = pk(0.f);
    const IO* xs = static_cast<const IO*>(a.x);
    const IO* gys = static_cast<const IO*>(a.gy);
    const float inv = 1.f / a.dim;
    const long step = (long)gridDim.x * G;
    long row = (long)blockIdx.x * G + group;
    Piece<IO, VEC, T, E> px, pg;
    float2 st{};
    if (row < a.rows) {
        px.load(xs + row * a.dim, a.dim, lane);
        pg.load(gys + row * a.dim, a.dim, lane);
        st = a.stats[row];
    }
    if constexpr (kKeepW) own_params<VEC, T, E>(a.w, a.param_dtype, a.dim, lane, 1.f, w);
    for (; row < a.rows; row += step) {
        f2 xh[E / 2], g[E / 2], s1 = pk(0.f), s2 = pk(0.f);
        px.unpack(xh);
        pg.unpack(g);
        const f2 rstd = pk(st.y);
        const float mean = st.x;
        if (row + step < a.rows) {
            px.load(xs + (row + step) * a.dim, a.dim, lane);
            pg.load(gys + (row + step) * a.dim, a.dim, lane);
            st = a.stats[row + step];
        }
        // past the end gy is zero, and so is all that it is a factor of, as long as xh there is finite: so x stays zero there
        auto shift_of = [&](int e) { return (e / VEC * T + lane) * VEC < a.dim ? -mean : 0.f; };
        auto pair = [&](int i, f2 weight) {
            xh[i] = mul2(add2(xh[i], make_float2(shift_of(2 * i), shift_of(2 * i + 1))), rstd);
            dw[i] = fma2(g[i], xh[i], dw[i]);
            db[i] = add2(db[i], g[i]);
            g[i] = mul2(g[i], weight);
            s1 = add2(s1, g[i]);
            s2 = fma2(g[i], xh[i], s2);
        };
        if constexpr (kKeepW) {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) pair(i, w[i]);
        } else {
            constexpr int W = VEC == 1 ? 2 : VEC;  // elements at a time
#pragma unroll
            for (int j = 0; j < E / W; ++j) {
                float v[W];
#pragma unroll
                for (int k = 0; k < W / VEC; ++k) {
                    const int c = ((j * (W / VEC) + k) * T + lane) * VEC;
                    load_params<VEC>(c < a.dim ? a.w : nullptr, a.param_dtype, c, 1.f, v + k * VEC);
                }
#pragma unroll
                for (int k = 0; k < W / 2; ++k) pair(j * (W / 2) + k, make_float2(v[2 * k], v[2 * k + 1]));
            }
        }
        if (!a.gx) continue;
        const float2 s = sum(make_float2(s1.x + s1.y, s2.x + s2.y));
        const f2 m1 = pk(-s.x * inv * rstd.x), m2 = pk(-s.y * inv * rstd.x);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) g[i] = fma2(g[i], rstd, fma2(xh[i], m2, m1));
        store_row<IO, VEC, T, E>(static_cast<IO*>(a.gx) + row * a.dim, a.dim, lane, g);
    }
    if (!a.part) return;
    // this CTA's sums: straight to scratch, or over its groups first
    auto put = [&](float* out, const f2(&v)[E / 2], int end) {
#pragma unroll
        for (int j = 0; j < E / VEC; ++j) {
            const int c = (j * T + lane) * VEC;
            if (c >= end) continue;
            if constexpr (VEC == 1) {
                out[c] = at(v, j);
            } else {
#pragma unroll
                for (int i = j * VEC / 2; i < (j + 1) * VEC / 2; i += 2)
                    *reinterpret_cast<float4*>(out + c + 2 * i - j * VEC) = make_float4(v[i].x, v[i].y, v[i + 1].x, v[i + 1].y);
            }
        }
    };
    float* out = a.part + (size_t)blockIdx.x * a.dim;
    const size_t bias = (size_t)gridDim.x * a.dim;
    if constexpr (G == 1) {
        put(out, dw, a.dim);
        put(out + bias, db, a.dim);
    } else {
        put(cols[0] + group * T * E, dw, T * E);
        put(cols[1] + group * T * E, db, T * E);
        __syncthreads();
        for (int c = threadIdx.x; c < a.dim; c += block_of(T)) {
            double u = cols[0][c], v = cols[1][c];
#pragma unroll
            for (int k = 1; k < G; ++k) u += cols[0][k * T * E + c], v += cols[1][k * T * E + c];
            out[c] = (float)u;
            out[bias + c] = (float)v;
        }
    }
}

// Rows wider than the registers of a group hold: one CTA per row, which reads the row once per pass (from L2 after the
// first), an element at a time, and is bound by those loads: 8192 x 16384 float32 forward 291 us (3.7 TB/s), backward 698
// (2.3 TB/s), bfloat16 184 and 476. Kept simple: no model of the framework has such rows.
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

// partial sums of grad_w and grad_b: one thread per column, one slice of rows per blockIdx.y; in double, since a thread adds rows
// / 64 of them in order (in float32 8192 x 10000 came out 2.1e-7 off, torch's sums 1.3e-7)
template <typename IO>
__global__ void __launch_bounds__(kWideThreads) norm_wide_param_kernel(const NormArgs a) {
    after_previous();
    const int c = blockIdx.x * kWideThreads + threadIdx.x;
    if (c >= a.dim) return;
    const IO* x = static_cast<const IO*>(a.x) + c;
    const IO* gy = static_cast<const IO*>(a.gy) + c;
    double dw = 0., db = 0.;
    for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float2 st = a.stats[r];
        const float g = as_float(gy[r * a.dim]);
        dw = fma((double)g, (double)((as_float(x[r * a.dim]) - st.x) * st.y), dw);
        db += g;
    }
    a.part[(size_t)blockIdx.y * a.dim + c] = (float)dw;
    a.part[((size_t)gridDim.y + blockIdx.y) * a.dim + c] = (float)db;
}

// grad_w (blockIdx.y 0) and grad_b (1): adds the slices of 32 columns in a fixed order, 32 slices at a time, each warp one
// column in the end. In double: some 300 slices added in float32 were as large an error as all sums before them, 1.3 times that
// of torch's elementary sums at 16384 x 4096; in double it is 1.0 times. (256 threads of four columns each took 0.7 us longer
// over 296 slices.)
__global__ void __launch_bounds__(32 * kFinishSlices) norm_finish_kernel(const NormArgs a, int slices) {
    static_assert(kFinishSlices == 32, "a warp per column");
    after_previous();
    __shared__ double tile[kFinishSlices][33];
    const int first = blockIdx.x * 32, c = first + threadIdx.x;
    void* out = blockIdx.y ? a.gb : a.gw;
    if (!out) return;
    const float* part = a.part + (size_t)blockIdx.y * slices * a.dim;
    double s = 0.;
    if (c < a.dim) {
#pragma unroll 10
        for (int k = threadIdx.y; k < slices; k += kFinishSlices) s += part[(size_t)k * a.dim + c];
    }
    tile[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = tile[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (threadIdx.x == 0 && first + threadIdx.y < a.dim) store_dt(out, first + threadIdx.y, a.param_dtype, (float)s);
}

bool is_wide(int dim) { return dim > kMaxDim; }

// Elements of a row that a thread can hold without spilling its 128 registers (bfloat16 at 24 spills 45 of them in the
// backward: 12.6 against 8.4 us at 8192 x 768; single elements at 16 spill up to 127)
int most_of(int io_dtype, int dim, bool backward) {
    const bool vec = dim % (io_dtype == QK_BF16 ? 8 : 4) == 0;
    if (backward) return vec ? 16 : 8;
    return vec && io_dtype == QK_BF16 ? 24 : 16;
}
// Threads of a row: a warp while they hold it, doubled until they do. Few rows get more threads each, down to eight
// elements per thread, until there are some 512 threads per SM: a row then takes less time.
int threads_of(int rows, int dim, int io_dtype, bool backward) {
    const int most = most_of(io_dtype, dim, backward);
    int t = 32;
    while (t < kMaxT && (t * most < dim || (t * 8 < dim && (long)rows * t < 512l * kSms))) t *= 2;
    return t;
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// CTAs for groups of `each` rows at least; as many as the SMs hold, or that many times over so that no group has more than
// `most_rows` (0: any number)
int ctas_of(int rows, int t, int each, int most_rows) {
    const long groups = block_of(t) / t, held = kSms * (512 / block_of(t));
    const long need = (rows + groups * each - 1) / (groups * each);
    if (need <= held) return (int)need;
    const long turns = most_rows ? (rows + held * groups * most_rows - 1) / (held * groups * most_rows) : 1;
    return (int)(held * turns);
}
// A CTA of the backward leaves a row of partial sums, which the second launch reads again: not for a single row each. For
// float32 gradients no group has more than 64 rows, which are added in order: K of them are sqrt(K / 6) steps off. (65536 x 8192,
// 443 rows each: grad_weight 3.8e-7 off where torch's sums are 1.9e-7, 1154 us; 64 rows: 1.6e-7, 1199 us.) Gradients that are
// rounded to bfloat16 would not show it.
constexpr int kBackwardEach = 2, kBackwardMost = 64;
int most_rows(int param_dtype) { return param_dtype == QK_F32 ? kBackwardMost : 0; }

template <typename IO, int VEC, int T, int E>
cudaError_t run_e(const NormArgs& a, bool backward, cudaStream_t st) {
    const dim3 grid(backward ? ctas_of(a.rows, T, kBackwardEach, most_rows(a.param_dtype)) : ctas_of(a.rows, T, 1, 0)), block(block_of(T));
    if constexpr (E <= 16)
        if (backward) return launch_after(norm_backward_kernel<IO, VEC, T, E>, grid, block, 0, st, a);
    return launch_after(norm_forward_kernel<IO, VEC, T, E>, grid, block, 0, st, a);
}

template <typename IO, int VEC, int T>
cudaError_t run_t(const NormArgs& a, bool backward, cudaStream_t st) {
    const int need = (a.dim + T - 1) / T;  // elements per thread
    if (need <= 8) return run_e<IO, VEC, T, 8>(a, backward, st);
    if constexpr (sizeof(IO) == 2 && T * 16 < kMaxDim)  // rows of whole 16-byte words that do not start on one: by element, as many of them
        if (need > 16 && !backward) return run_e<IO, VEC, T, 24>(a, backward, st);
    return run_e<IO, VEC, T, 16>(a, backward, st);
}

template <typename IO, int VEC>
cudaError_t run_vec(const NormArgs& a, bool backward, cudaStream_t st) {
    switch (threads_of(a.rows, a.dim, a.io_dtype, backward)) {
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
                         dim3((a.dim + kWideThreads - 1) / kWideThreads, norm_slices(a.rows, a.dim, a.io_dtype, a.param_dtype)), kWideThreads, 0, st, a);
    return e;
}

cudaError_t run(const NormArgs& a, bool backward, cudaStream_t st) {
    const bool half = a.io_dtype == QK_BF16;
    if (is_wide(a.dim)) return half ? run_wide<__nv_bfloat16>(a, backward, st) : run_wide<float>(a, backward, st);
    return half ? run_rows<__nv_bfloat16>(a, backward, st) : run_rows<float>(a, backward, st);
}

}  // namespace

int norm_slices(int rows, int dim, int io_dtype, int param_dtype) {
    if (is_wide(dim)) return rows < 64 ? rows : 64;
    return ctas_of(rows, threads_of(rows, dim, io_dtype, true), kBackwardEach, most_rows(param_dtype));
}

cudaError_t launch_norm_forward(const NormArgs& a, cudaStream_t st) { return run(a, false, st); }

cudaError_t launch_norm_backward(const NormArgs& a, cudaStream_t st) {
    const cudaError_t e = run(a, true, st);
    if (e != cudaSuccess || !a.part) return e;
    const dim3 grid((a.dim + 31) / 32, 2);
    const int slices = norm_slices(a.rows, a.dim, a.io_dtype, a.param_dtype);
    return launch_after(norm_finish_kernel, grid, dim3(32, kFinishSlices), 0, st, a, slices);
}

}  // namespace qk
