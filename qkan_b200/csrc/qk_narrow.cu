// The linear map in float32 for few outputs (the hybrid block's down projection), or little of everything:
// y[m,n] = act(sum_k x[m,k] W[n,k] + b[n]) + r[m,n], 16 or 32 columns n at a time.
//
// Bound by reading x once, from some 16 columns on by the float32 units. On the tensor cores x would be split into its three
// parts first, 6 bytes written and read again for each 4: with so few columns that costs more than the products. Measured,
// in us, against the tensor cores: 55447 x 1032 -> 16 69 (3.3 TB/s) and 201, -> 32 114 and 203; 8192 x 768 -> 10 12.7 and 19.6;
// 24 x 100 -> 10 3.4 and 7.5, there for want of a second launch.
//
// A CTA has a tile of rows by 16 or 32 columns, and walks the depth in chunks of 32 through a ring in shared memory
// (cp.async). A warp's lanes are 8 rows by 4 columns, TM x TN sums each, rows (columns) 8 (4) apart: with 36 floats from row
// to row the lanes meet no bank twice. Two neighbouring products of the depth go through one packed operation, which needs
// no value twice in a pair. Where there are too few tiles, the depth is cut and the slices added by the reduction.
#include "qk_linear.cuh"
#include "qk_packed.cuh"

namespace qk {
namespace {

constexpr int kThreads = 128;
constexpr int kDepth = 32;
constexpr int kPitch = kDepth + 4;
constexpr int kStages = 3;

template <int NP, int M>
struct Tile {
    static constexpr int TN = NP / 4, TM = M;
    static constexpr int kRows = kThreads / 32 * 8 * TM;
    static constexpr int kStage = (kRows + NP) * kPitch;  // floats
    static constexpr int kSmem = kStages * kStage * 4;
};

// BYTES from global to shared memory, zeros unless `there`
template <int BYTES>
__device__ __forceinline__ void copy_async(float* to, const float* from, bool there) {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(to);
    const int n = there ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(from), "r"(n) : "memory");
}

template <int NP, int TM, bool VEC>
__global__ void __launch_bounds__(kThreads, 3) narrow_kernel(const NarrowArgs a) {
    using T = Tile<NP, TM>;
    extern __shared__ __align__(16) float ring[];
    after_previous();
    const int tile = blockIdx.x / a.splits, split = blockIdx.x - tile * a.splits;
    const long r0 = (long)tile * T::kRows;
    const int c0 = blockIdx.y * NP, width = min(NP, a.cols - c0);
    const int chunk0 = split * a.per, chunks = min(a.per, a.chunks - chunk0);
    const float* x = static_cast<const float*>(a.x);
    const float* w = static_cast<const float*>(a.w);
    // This thread's pieces of a chunk: four of the depth, rows kThreads / 8 apart. Rows past the last are the last one again,
    // never stored.
    constexpr int kApart = kThreads / (kDepth / 4), kPieces = (T::kRows + NP) / kApart;
    const int row0 = threadIdx.x / (kDepth / 4), part0 = threadIdx.x % (kDepth / 4) * 4;
    const float* from[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int row = row0 + i * kApart;
        from[i] = (row < T::kRows ? x + (size_t)min(r0 + row, a.rows - 1L) * a.depth
                                  : w + (size_t)(c0 + min(row - T::kRows, width - 1)) * a.depth) + part0;
    }
    auto fetch = [&](int c) {
        if (c < chunks) {
            float* to = ring + c % kStages * T::kStage + row0 * kPitch + part0;
            const long k = (long)(chunk0 + c) * kDepth, left = a.depth - part0 - k;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                if constexpr (VEC) {
                    copy_async<16>(to + i * kApart * kPitch, left > 0 ? from[i] + k : x, left > 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        copy_async<4>(to + i * kApart * kPitch + e, e < left ? from[i] + k + e : x, e < left);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int lane = threadIdx.x % 32, m = threadIdx.x / 32 * 8 * T::TM + lane / 4, n = lane % 4;
    f2 acc[T::TM][T::TN];
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) acc[i][j] = pk(0.f);
    for (int c = 0; c < kStages - 1; ++c) fetch(c);
    for (int c = 0; c < chunks; ++c) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // chunk c is there for all, and chunk c - 1 is done with: its stage is the next one's
        fetch(c + kStages - 1);
        const float* xs = ring + c % kStages * T::kStage + m * kPitch;
        const float* ws = ring + c % kStages * T::kStage + (T::kRows + n) * kPitch;
#pragma unroll
        for (int k = 0; k < kDepth; k += 4) {
            float4 xv[T::TM];
#pragma unroll
            for (int i = 0; i < T::TM; ++i) xv[i] = *reinterpret_cast<const float4*>(xs + i * 8 * kPitch + k);
#pragma unroll
            for (int j = 0; j < T::TN; ++j) {
                const float4 wv = *reinterpret_cast<const float4*>(ws + j * 4 * kPitch + k);
#pragma unroll
                for (int i = 0; i < T::TM; ++i) {
                    acc[i][j] = fma2(make_float2(xv[i].x, xv[i].y), make_float2(wv.x, wv.y), acc[i][j]);
                    acc[i][j] = fma2(make_float2(xv[i].z, xv[i].w), make_float2(wv.z, wv.w), acc[i][j]);
                }
            }
        }
    }
    // The sums by way of shared memory, where the tile lies as it does in y: whole lines stored, and one copy of the
    // epilogue's code (unrolled over a thread's sums it was most of the time of a short depth).
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int j = 0; j < T::TN; ++j)
            if (n + 4 * j < width) ring[(m + 8 * i) * width + n + 4 * j] = acc[i][j].x + acc[i][j].y;
    __syncthreads();
    const int count = (int)min((long)T::kRows, a.rows - r0) * width;
    float* part = a.part ? a.part + (size_t)split * a.rows * a.cols : nullptr;
#pragma unroll 1
    for (int t = threadIdx.x; t < count; t += kThreads) {
        const int row = t / width, col = c0 + t - row * width;
        const size_t at = (size_t)(r0 + row) * a.cols + col;
        if (part) part[at] = ring[t];
        else finish_element(a.epi, at, col, ring[t]);
    }
}

template <int NP, int TM, bool VEC>
cudaError_t run(const NarrowArgs& a, cudaStream_t st) {
    using T = Tile<NP, TM>;
    static unsigned long long opted = 0;
    const cudaError_t e = opt_in_smem(narrow_kernel<NP, TM, VEC>, &opted, T::kSmem);
    if (e != cudaSuccess) return e;
    const long tiles = ((long)a.rows + T::kRows - 1) / T::kRows;
    if (tiles * a.splits > 0x7fffffffl) return cudaErrorInvalidConfiguration;
    return launch_after(narrow_kernel<NP, TM, VEC>, dim3((unsigned)(tiles * a.splits), (a.cols + NP - 1) / NP), kThreads, T::kSmem, st, a);
}

template <int NP, int TM>
cudaError_t run_tile(const NarrowArgs& a, cudaStream_t st) {
    const bool vec = a.depth % 4 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.w % 16 == 0;
    return vec ? run<NP, TM, true>(a, st) : run<NP, TM, false>(a, st);
}

template <int NP>
cudaError_t run_np(const NarrowArgs& a, cudaStream_t st) {
    if (a.tm == 1) return run_tile<NP, 1>(a, st);
    return a.tm == 2 ? run_tile<NP, 2>(a, st) : run_tile<NP, 4>(a, st);
}

}  // namespace

// One row per thread while there are few of them or little to do, since a chunk then takes least time: four where there is
// much, since W is read from shared memory for all of them. (us with 1, 2, 4: 100 x 768 -> 10 5.5, 5.8, 6.7; 8192 x 100 -> 10
// 8.8, 5.9, 6.2; 2000 x 4096 -> 10 27, 17, 15; 55447 x 1032 -> 32 238, 136, 114.) The depth is cut until there are four CTAs per
// SM, of four chunks at least (2000 x 4096 -> 10: two per SM 17, one 23).
NarrowPlan narrow_plan(int rows, int cols, int depth) {
    NarrowPlan p;
    const long across = (cols + 31L) / 32;
    auto tiles_of = [&](int tm) { return ((long)rows + kThreads / 4 * tm - 1) / (kThreads / 4 * tm) * across; };
    p.tm = 1;
    while (p.tm < 4 && (tiles_of(p.tm) > kSms || (rows >= 256 * p.tm && across * rows * depth >= 1 << 20))) p.tm *= 2;
    p.chunks = (int)((depth + kDepth - 1L) / kDepth);
    const long tiles = tiles_of(p.tm), want = (4 * kSms + tiles - 1) / tiles, most = p.chunks < 4 ? 1 : p.chunks / 4;
    const int splits = (int)(want < most ? want : most);
    p.per = (p.chunks + splits - 1) / splits;
    p.splits = (p.chunks + p.per - 1) / p.per;
    return p;
}

cudaError_t launch_narrow(const NarrowArgs& a, cudaStream_t st) {
    return a.cols > 16 ? run_np<32>(a, st) : run_np<16>(a, st);
}

}  // namespace qk
