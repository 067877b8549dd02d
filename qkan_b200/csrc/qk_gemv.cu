// The linear map for a few rows (single tokens): y[m,n] = act(sum_k x[m,k] W[n,k] + b[n]) + r[m,n], a few rows only.
//
// Bound by reading W once. A warp takes C rows of W at a time, 16 bytes per lane and row, the next kAhead such loads
// under way, and keeps C x R sums; x comes from L1, each piece of it used for C rows of W. Where there are too few rows of W to
// occupy the GPU, the warps of a CTA share them and cut the depth. float32 is multiplied as it is: the three-part form of
// the tensor-core products would write W out again, six bytes for four.
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

}  // namespace

cudaError_t launch_gemv(const GemvArgs& args, cudaStream_t st) {
    GemvArgs a = args;
    return a.epi.io_dtype == QK_BF16 ? launch_typed<__nv_bfloat16>(a, st) : launch_typed<float>(a, st);
}

}  // namespace qk
