// The linear map for a few rows (single tokens): y[m,n] = act(sum_k x[m,k] W[n,k] + b[n]) + r[m,n], a few rows only.
//
// Bound by reading W once. A warp takes C rows of W at a time, 16 bytes per lane and row, the next kAhead such loads
// under way, and keeps C x R sums; x comes from L1, each piece of it used for C rows of W. Where there are too few rows of W to
// occupy the GPU, the warps of a CTA share them and cut the depth. float32 is multiplied as it is: the three-part form of
// the tensor-core products would write W out again, six bytes for four.
// Measured: 1 x 4096 -> 4096 in bfloat16 6.3 us with W in L2, 8.8 from memory (5.1 at the copy's rate); float32 12.5 (10.2).
// The backward of a few rows is below: 4 x 4096 -> 4096 float32, all gradients, 27 us, 5 TB/s.
#include <type_traits>

#include "qk_linear.cuh"

namespace qk {
namespace {

constexpr int kWarps = 8;
constexpr int kAhead = 2;

template <typename IO, int VEC>
__device__ __forceinline__ void widen(const uint4& u, float (&f)[VEC]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(IO) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

// VEC elements per lane and load: 16 bytes, or one element where rows are not whole 16-byte words
template <typename IO, int R, int C, int VEC>
__global__ void __launch_bounds__(kWarps * 32) gemv_kernel(const GemvArgs a) {
    using Raw = std::conditional_t<VEC == 1, IO, uint4>;
    __shared__ float sums[kWarps][R * C];
    after_previous();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int part = warp % a.cuts, group = warp / a.cuts, groups = kWarps / a.cuts;
    const long n0 = ((long)blockIdx.x * groups + group) * C;
    const IO* x = static_cast<const IO*>(a.x);
    // rows past the last are the last one again: loaded, never stored
    const IO* w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) w[c] = static_cast<const IO*>(a.w) + (size_t)min(n0 + c, a.cols - 1L) * a.depth;
    const long begin = (long)part * a.per, end = min((long)a.depth, begin + a.per);
    float acc[C][R] = {};
    auto load = [&](long k, Raw(&v)[C]) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            v[c] = Raw{};
            if (k < end) v[c] = *reinterpret_cast<const Raw*>(w[c] + k);
        }
    };
    constexpr int kStep = 32 * VEC;
    const int row0 = blockIdx.y * R;
    Raw ahead[kAhead][C];
    long k = begin + lane * VEC;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(k + i * kStep, ahead[i]);
    for (; k < end; k += kAhead * kStep) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const long at = k + i * kStep;
            float wf[C][VEC];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if constexpr (VEC == 1) wf[c][0] = as_float(ahead[i][c]);
                else widen<IO, VEC>(ahead[i][c], wf[c]);
            }
            load(at + kAhead * kStep, ahead[i]);
            if (at >= end) continue;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const IO* row = x + (size_t)min(row0 + r, a.rows - 1) * a.depth + at;
                float xf[VEC];
                if constexpr (VEC == 1) xf[0] = as_float(*row);
                else widen<IO, VEC>(*reinterpret_cast<const uint4*>(row), xf);
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) acc[c][r] = fmaf(xf[e], wf[c][e], acc[c][r]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s = acc[c][r];
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
            if (lane == 0) sums[warp][c * R + r] = s;
        }
    __syncthreads();
    // the sums of this CTA's groups, their parts in order
    for (int t = threadIdx.x; t < groups * R * C; t += kWarps * 32) {
        const int g = t / (R * C), e = t % (R * C), r = row0 + e % R;
        const long n = ((long)blockIdx.x * groups + g) * C + e / R;
        if (r >= a.rows || n >= a.cols) continue;
        float s = sums[g * a.cuts][e];
        for (int p = 1; p < a.cuts; ++p) s += sums[g * a.cuts + p][e];
        finish_element(a.epi, (size_t)r * a.cols + n, (int)n, s);
    }
}

template <typename IO, int R, int C>
cudaError_t launch_rows(GemvArgs& a, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(IO);
    const long groups = (a.cols + C - 1L) / C;
    // cut the depth until there are some 8 warps per SM, while each has a load or more per lane
    const bool vec = a.depth % VEC == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.w % 16 == 0;
    const int step = 32 * (vec ? VEC : 1);
    a.cuts = 1;
    while (a.cuts < kWarps && groups * a.cuts < 8 * kSms && a.depth > (long)a.cuts * step) a.cuts *= 2;
    a.per = (int)(((long)a.depth + a.cuts * step - 1) / (a.cuts * step) * step);
    const long grid = (groups + kWarps / a.cuts - 1) / (kWarps / a.cuts);
    return launch_after(vec ? gemv_kernel<IO, R, C, VEC> : gemv_kernel<IO, R, C, 1>,
                        dim3((unsigned)grid, (a.rows + R - 1) / R), kWarps * 32, 0, st, a);
}

template <typename IO>
cudaError_t launch_typed(GemvArgs& a, cudaStream_t st) {
    if (a.rows == 1) return launch_rows<IO, 1, 4>(a, st);
    if (a.rows == 2) return launch_rows<IO, 2, 4>(a, st);
    if constexpr (sizeof(IO) == 4) {
        if (a.rows <= 4) return launch_rows<IO, 4, 4>(a, st);
        return launch_rows<IO, 8, 4>(a, st);  // groups of eight, the later ones with W from L2
    }
    return cudaErrorInvalidValue;  // few_rows() lets none through
}

// ---- backward ------------------------------------------------------------------
constexpr int kFewThreads = 128, kFewCols = 4, kFewSlab = 128;

// A thread has four columns of W, x, grad_x and grad_weight, and walks a slab of W's rows: each is read once for grad_x
// (sums over the slab in registers), and the row of grad_weight beside it is written. gz = gy * act'(tape), in float32, is
// made once per CTA in shared memory, a row of W's R values together. Bound by reading W and writing grad_weight.
// VEC 4: the four columns are neighbours, moved at once; 1: they lie kFewThreads apart.
template <typename IO, int R, int VEC>
__global__ void __launch_bounds__(kFewThreads) few_backward_kernel(const FewArgs a) {
    __shared__ __align__(16) float gz[kFewSlab][R];
    after_previous();
    const int block = blockIdx.x % a.blocks, slab = blockIdx.x / a.blocks;
    const long n0 = (long)slab * a.slab;
    const int count = (int)min((long)a.slab, a.out - n0);
    for (int t = threadIdx.x; t < a.slab * R; t += kFewThreads) {
        const int r = t / a.slab, n = t % a.slab;  // along the rows of gy
        float v = 0.f;
        if (r < a.rows && n < count) {
            const size_t at = (size_t)r * a.out + n0 + n;
            v = load_dt(a.gy, at, a.io_dtype);
            if (a.tape) v *= act_slope<false>(load_tape(a.tape, at, a.io_dtype), a.act);
        }
        gz[n][r] = v;
    }
    __syncthreads();
    if (a.gb && block == 0)
        for (int n = threadIdx.x; n < count; n += kFewThreads) {
            double s = 0.;
#pragma unroll
            for (int r = 0; r < R; ++r) s += gz[n][r];
            store_dt(a.gb, n0 + n, a.io_dtype, (float)s);
        }
    const long first = (long)block * kFewThreads * kFewCols + threadIdx.x * VEC;
    long col[kFewCols];
#pragma unroll
    for (int i = 0; i < kFewCols; ++i) col[i] = VEC == 4 ? first + i : first + (long)i * kFewThreads;
    // columns behind the edge hold zeros and are not stored
    auto load = [&](const void* p, size_t row, float(&v)[kFewCols]) {
        const IO* q = static_cast<const IO*>(p) + row * a.in;
        if constexpr (VEC == 4 && sizeof(IO) == 4) {
            float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
            if (col[0] < a.in) u = *reinterpret_cast<const float4*>(q + col[0]);
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else if constexpr (VEC == 4) {
            uint2 u = make_uint2(0, 0);
            if (col[0] < a.in) u = *reinterpret_cast<const uint2*>(q + col[0]);
            v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
            v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < kFewCols; ++i) {
                v[i] = 0.f;
                if (col[i] < a.in) v[i] = as_float(q[col[i]]);
            }
        }
    };
    float x[R][kFewCols], acc[R][kFewCols] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < kFewCols; ++i) x[r][i] = 0.f;
        if (a.gw && r < a.rows) load(a.x, r, x[r]);
    }
    if (!a.gx_part && !a.gw) return;
    // U rows of W are fetched together: one after the other, each behind the store of the row before, they took four times
    // as long
    constexpr int U = R <= 8 ? 8 : 4;
    for (int n = 0; n < count; n += U) {
        float w[U][kFewCols];
#pragma unroll
        for (int j = 0; j < U; ++j) {
#pragma unroll
            for (int i = 0; i < kFewCols; ++i) w[j][i] = 0.f;
            if (a.gx_part && n + j < count) load(a.w, n0 + n + j, w[j]);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (n + j >= count) break;
            float out[kFewCols] = {};
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float g = gz[n + j][r];
#pragma unroll
                for (int i = 0; i < kFewCols; ++i) {
                    acc[r][i] = fmaf(g, w[j][i], acc[r][i]);
                    out[i] = fmaf(g, x[r][i], out[i]);
                }
            }
            if (!a.gw) continue;
            IO* to = static_cast<IO*>(a.gw) + (size_t)(n0 + n + j) * a.in;
            if constexpr (VEC == 4) {
                if (col[0] >= a.in) continue;
                if constexpr (sizeof(IO) == 4) {
                    *reinterpret_cast<float4*>(to + col[0]) = make_float4(out[0], out[1], out[2], out[3]);
                } else {
                    uint2 u;
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u.x) : "f"(out[1]), "f"(out[0]));
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u.y) : "f"(out[3]), "f"(out[2]));
                    *reinterpret_cast<uint2*>(to + col[0]) = u;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kFewCols; ++i)
                    if (col[i] < a.in) to[col[i]] = from_float<IO>(out[i]);
            }
        }
    }
    if (!a.gx_part) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= a.rows) continue;
        float* to = a.gx_part + ((size_t)slab * a.rows + r) * a.in;
#pragma unroll
        for (int i = 0; i < kFewCols; ++i)
            if (col[i] < a.in) to[col[i]] = acc[r][i];
    }
}

template <typename IO, int R>
cudaError_t launch_few_rows(const FewArgs& a, cudaStream_t st) {
    auto words = [](const void* p) { return (uintptr_t)p % (4 * sizeof(IO)) == 0; };
    const bool vec = a.in % 4 == 0 && words(a.x) && words(a.w) && words(a.gw);
    const long grid = (long)a.blocks * ((a.out + (long)a.slab - 1) / a.slab);
    if (grid > 0x7fffffffl) return cudaErrorInvalidConfiguration;
    return launch_after(vec ? few_backward_kernel<IO, R, 4> : few_backward_kernel<IO, R, 1>, (unsigned)grid, kFewThreads, 0, st, a);
}

template <typename IO>
cudaError_t launch_few_typed(const FewArgs& a, cudaStream_t st) {
    if (a.rows <= 2) return launch_few_rows<IO, 2>(a, st);
    if (a.rows <= 4) return launch_few_rows<IO, 4>(a, st);
    if constexpr (sizeof(IO) == 4) return a.rows <= 8 ? launch_few_rows<IO, 8>(a, st) : launch_few_rows<IO, 16>(a, st);
    return cudaErrorInvalidValue;  // few_rows_backward() lets none through
}

}  // namespace

// some six CTAs per SM, of eight rows of W at least
FewPlan few_plan(int in, int out) {
    FewPlan p;
    p.blocks = (int)((in + kFewThreads * kFewCols - 1L) / (kFewThreads * kFewCols));
    if (p.blocks == 0) p.blocks = 1;  // grad_bias alone
    const long slabs = (6l * kSms + p.blocks - 1) / p.blocks;
    long slab = (out + slabs - 1) / slabs;
    if (slab < 8) slab = 8;
    if (slab > kFewSlab) slab = kFewSlab;
    p.slab = (int)slab;
    p.slabs = (int)((out + slab - 1) / slab);
    return p;
}

cudaError_t launch_few_backward(const FewArgs& a, cudaStream_t st) {
    return a.io_dtype == QK_BF16 ? launch_few_typed<__nv_bfloat16>(a, st) : launch_few_typed<float>(a, st);
}

cudaError_t launch_gemv(const GemvArgs& args, cudaStream_t st) {
    GemvArgs a = args;
    return a.epi.io_dtype == QK_BF16 ? launch_typed<__nv_bfloat16>(a, st) : launch_typed<float>(a, st);
}

}  // namespace qk
