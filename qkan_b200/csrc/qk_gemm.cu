// Matrix products of the linear map on the tensor cores (tcgen05): C[r,c] = sum_k P[r,k] Q[c,k] with the epilogue
// act(C + bias[c]) + residual[r,c].
//
// The MMA's M side (the 128 lanes of tensor memory) is Q's side, so a thread of the epilogue owns one column c and its
// warp 32 neighbouring ones: bias sits in a register, and residual, output and tape are read and written along rows
// without a detour through shared memory, whatever the width or alignment of a row.
//
// One CTA per SM walks units of work (tile, slice of the depth). Warp 0 copies 64-deep blocks of both operands into a
// ring of stages (TMA, 128-byte swizzle), warp 1 issues the MMAs, eight warps drain the sums from one of two
// accumulators while the other one is filled. An operand is read as it lies in memory: "K-major" when the summed axis is
// contiguous (forward: x and W), "MN-major" when it is the other axis (W in grad_x, x and gz in grad_weight).
//
// float32 (PLANES == 3): x = h + m + l exactly, each part a bfloat16 (8 significant bits, float32's exponents). Six of
// the nine products are kept: hh | hm mh hl lh mm; what is dropped is below 2^-22 of |x||w|. hh goes to one accumulator
// and the five small ones to another. The tensor core truncates where it adds to its accumulator, which over a long
// sum would drift by more than float32 rounding does: so hh is drained every kChunk blocks and added in registers, with
// rounding. Where hh's sum is not finite the small products are left out: float32's own infinities come out.
#include <cuda.h>

#include "qk_linear.cuh"

namespace qk {
namespace {

constexpr int kBK = 64;             // depth of a stage: 128 bytes of bfloat16, one swizzle row
constexpr int kTileC = 128;         // the MMA's M
constexpr int kChunk = 2;           // stages between two drains of hh (float32)
constexpr int kGemmThreads = 320;   // producer, MMA issuer, 8 epilogue warps
constexpr int kDrainWarps = 8;
constexpr unsigned long long kGiveUpNs = 10ull * 1000 * 1000 * 1000;  // the longest that a wait may take

template <int BN, int PLANES>
struct Shape {
    static constexpr int kABytes = kTileC * 128;
    static constexpr int kBBytes = (BN < 64 ? 64 : BN) * 128;  // an MN-major box is 64 wide at least
    static constexpr int kStageBytes = PLANES * (kABytes + kBBytes);
    static constexpr int kStagesFit = (196 * 1024) / kStageBytes;
    static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
    static constexpr int kAccCols = 2 * BN;
    static constexpr int kColsWanted = PLANES == 3 ? 2 * kAccCols : kAccCols;
    static constexpr int kTmemCols = kColsWanted < 32 ? 32 : kColsWanted;
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + 1024 + 256;
    static_assert(kStages >= 2 && kTmemCols <= 512 && kSmem <= kSmemCap, "does not fit an SM");
};

struct Barriers {
    unsigned long long full[8], empty[8];
    unsigned long long acc_full[2], acc_empty[2];    // the accumulator (of hh)
    unsigned long long corr_full[2], corr_empty[2];  // the accumulator of the small products
    unsigned long long drain;
    unsigned tmem;
    int abort;
};

__device__ unsigned g_gave_up;  // waits that ran out

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(unsigned long long* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(unsigned long long* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(unsigned long long* b, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(unsigned long long* b, unsigned parity) {
    unsigned done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase of `parity` to end. Every wait ends: after kGiveUpNs, or once another warp has given up, the
// answer is false, and the caller leaves its loop.
__device__ __noinline__ bool bar_wait_long(unsigned long long* b, unsigned parity, volatile int* abort) {
    const unsigned long long start = now_ns();
    while (now_ns() - start < kGiveUpNs) {
        for (int i = 0; i < 64; ++i)
            if (bar_try(b, parity)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    atomicAdd(&g_gave_up, 1u);
    return false;
}
__device__ __forceinline__ bool bar_wait(unsigned long long* b, unsigned parity, volatile int* abort) {
    for (int i = 0; i < 16; ++i)
        if (bar_try(b, parity)) return true;
    return bar_wait_long(b, parity, abort);
}
__device__ __forceinline__ void tma_load(const CUtensorMap* map, unsigned dst, unsigned long long* bar, int x, int y,
                                         int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_load16(unsigned addr, float (&v)[16]) {
    unsigned u[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(u[i]);
}

template <int N>
__device__ __forceinline__ void tmem_load(unsigned addr, float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; j += 16) {
        float u[16];
        tmem_load16(addr + j, u);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[j + i] = u[i];
    }
}

// Shared-memory matrix descriptor, 128-byte swizzle. K-major: rows of 128 bytes, 8-row groups 1024 bytes apart, a
// 16-deep step is 32 bytes on. MN-major: 64-wide boxes (8 KB each) of 64 rows of the depth, 8-row groups 1024 bytes
// apart, a 16-deep step is 16 rows on.
__device__ __forceinline__ unsigned long long smem_desc(unsigned addr, bool mn) {
    const unsigned long long lead = mn ? 8192 >> 4 : 1, stride = 1024 >> 4;
    return (unsigned long long)((addr & 0x3ffff) >> 4) | lead << 16 | stride << 32 | 1ull << 46 | 2ull << 61;
}

// One unit of work: a tile of C and a slice of the depth.
struct Unit {
    int r0, c0, kb0, kbs, split;  // first row in tiles, first column, first block and number of blocks of the slice
};
__device__ __forceinline__ Unit unit_at(const GemmProblem& g, int u) {
    Unit t;
    const int tiles = g.tiles_r * g.tiles_c;
    t.split = u / tiles;
    u -= t.split * tiles;
    t.r0 = u / g.tiles_c;  // columns run fastest, so that neighbouring CTAs share P
    t.c0 = (u - t.r0 * g.tiles_c) * kTileC;
    t.kb0 = t.split * g.kper;
    t.kbs = min(g.kper, g.kblocks - t.kb0);
    return t;
}

// The residual of column c, rows r .. r + N - 1, fetched before the sums are waited for. Row and column are held inside
// the matrix, so that every load is good by itself; what lies behind its edge is never stored.
template <typename IO, int N>
__device__ __forceinline__ void load_residual(const GemmProblem& g, long r, int c, float (&q)[N]) {
    const long first = min(r, g.rows - 1L);
    const int last = (int)min(N - 1L, g.rows - 1 - first);
    const IO* res = static_cast<const IO*>(g.residual) + (size_t)first * g.cols + min(c, g.cols - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = as_float(res[(size_t)min(i, last) * g.cols]);
}

// N sums of column c, rows r .. r + N - 1, of which n exist (none for a lane behind the last column: the warp stays
// together, since it has to be whole when it reads tensor memory again).
template <typename IO, int N>
__device__ __forceinline__ void write_out(const GemmProblem& g, int split, long r, int c, int n, float bias,
                                          const float (&q)[N], float (&v)[N]) {
    const size_t cols = g.cols, at = (size_t)r * cols + c;
    if (g.part) {
        float* out = g.part + (size_t)split * g.rows * cols + at;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) out[i * cols] = v[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += bias;
    if (g.tape) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) store_tape(g.tape, at + i * cols, sizeof(IO) == 2 ? QK_BF16 : QK_F32, v[i]);
    }
    activate_all<sizeof(IO) == 2>(v, g.act);
    IO* out = static_cast<IO*>(g.out) + at;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) out[i * cols] = from_float<IO>(v[i] + q[i]);
}

template <int BN, int PLANES>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmProblem g) {
    using S = Shape<BN, PLANES>;
    using IO = std::conditional_t<PLANES == 3, float, __nv_bfloat16>;
    extern __shared__ char raw[];
    char* stages = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    Barriers& bars = *reinterpret_cast<Barriers*>(stages + (size_t)S::kStages * S::kStageBytes);
    static_assert(sizeof(Barriers) <= 256, "barriers");
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    volatile int* abort = &bars.abort;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) bar_init(&bars.full[i], 1), bar_init(&bars.empty[i], 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(&bars.acc_full[i], 1), bar_init(&bars.acc_empty[i], kDrainWarps);
            bar_init(&bars.corr_full[i], 1), bar_init(&bars.corr_empty[i], kDrainWarps);
        }
        bar_init(&bars.drain, 1);
        bars.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)),
                     "n"(S::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = bars.tmem, corr_base = tmem + S::kAccCols;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            unsigned phase = 0, issued = 0;
            bool ok = true;
            for (int u = blockIdx.x; ok && u < g.units; u += gridDim.x) {
                const Unit t = unit_at(g, u);
                const int r0 = t.r0 * BN;
                const unsigned bytes = PLANES * (S::kABytes + (g.p_mn ? S::kBBytes : BN * 128));
                for (int kb = t.kb0; kb < t.kb0 + t.kbs; ++kb) {
                    ok = bar_wait(&bars.empty[stage], phase ^ 1, abort);
                    if (!ok) break;
                    unsigned long long* bar = &bars.full[stage];
                    bar_expect(bar, bytes);
                    unsigned dst = smem_u32(stages) + stage * S::kStageBytes;
                    for (int p = 0; p < PLANES; ++p, dst += S::kABytes) {
                        if (g.q_mn) {
                            tma_load(&g.q_map, dst, bar, t.c0, kb * kBK, p);
                            tma_load(&g.q_map, dst + 8192, bar, t.c0 + 64, kb * kBK, p);
                        } else {
                            tma_load(&g.q_map, dst, bar, kb * kBK, t.c0, p);
                        }
                    }
                    for (int p = 0; p < PLANES; ++p, dst += S::kBBytes) {
                        if (g.p_mn) {
                            for (int b = 0; b < S::kBBytes / 8192; ++b)
                                tma_load(&g.p_map, dst + b * 8192, bar, r0 + b * 64, kb * kBK, p);
                        } else {
                            tma_load(&g.p_map, dst, bar, kb * kBK, r0, p);
                        }
                    }
                    ++issued;
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
            }
            if (!ok) {  // the copies still in flight write to this CTA's shared memory: see them land before it is given up
                for (unsigned n = 0; n < S::kStages && n < issued; ++n) {
                    if (--stage < 0) stage = S::kStages - 1, phase ^= 1;
                    for (int i = 0; i < (1 << 20) && !bar_try(&bars.full[stage], phase); ++i) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, acc = 0, corr = 0;
            unsigned phase = 0, acc_phase = 0, corr_phase = 0;
            bool ok = true;
            for (int u = blockIdx.x; ok && u < g.units; u += gridDim.x) {
                const Unit t = unit_at(g, u);
                const unsigned idesc = 1u << 4 | 1u << 7 | 1u << 10 | (unsigned)g.q_mn << 15 | (unsigned)g.p_mn << 16 |
                                       (BN / 8) << 17 | (kTileC / 16) << 24;
                const unsigned a_step = g.q_mn ? 2048 >> 4 : 32 >> 4, b_step = g.p_mn ? 2048 >> 4 : 32 >> 4;
                if (PLANES == 3) {
                    ok = bar_wait(&bars.corr_empty[corr], corr_phase ^ 1, abort);
                    if (!ok) break;
                }
                for (int kb = 0; kb < t.kbs; ++kb) {
                    const bool opens = PLANES == 3 ? kb % kChunk == 0 : kb == 0;
                    if (opens) {
                        ok = bar_wait(&bars.acc_empty[acc], acc_phase ^ 1, abort);
                        if (!ok) break;
                    }
                    ok = bar_wait(&bars.full[stage], phase, abort);
                    if (!ok) break;
                    fence_after();
                    const unsigned base = smem_u32(stages) + stage * S::kStageBytes;
                    const unsigned long long da = smem_desc(base, g.q_mn);
                    const unsigned long long db = smem_desc(base + PLANES * S::kABytes, g.p_mn);
                    const unsigned d = tmem + acc * BN;
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma(d, da + k * a_step, db + k * b_step, idesc, !(opens && k == 0));
                    if constexpr (PLANES == 3) {
                        const unsigned dc = corr_base + corr * BN;
                        constexpr int kA = S::kABytes >> 4, kB = S::kBBytes >> 4;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const unsigned long long ak = da + k * a_step, bk = db + k * b_step;
                            mma(dc, ak + 2 * kA, bk, idesc, !(kb == 0 && k == 0));
                            mma(dc, ak, bk + 2 * kB, idesc, true);
                            mma(dc, ak + kA, bk + kB, idesc, true);
                            mma(dc, ak + kA, bk, idesc, true);
                            mma(dc, ak, bk + kB, idesc, true);
                        }
                    }
                    mma_commit(&bars.empty[stage]);
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                    if (PLANES == 3 ? (kb % kChunk == kChunk - 1 || kb == t.kbs - 1) : kb == t.kbs - 1) {
                        mma_commit(&bars.acc_full[acc]);
                        if (++acc == 2) acc = 0, acc_phase ^= 1;
                    }
                }
                if (ok && PLANES == 3) {
                    mma_commit(&bars.corr_full[corr]);
                    if (++corr == 2) corr = 0, corr_phase ^= 1;
                }
            }
            if (!ok) {  // products still running write to the tensor memory that is freed below
                mma_commit(&bars.drain);
                for (int i = 0; i < (1 << 20) && !bar_try(&bars.drain, 0); ++i) {
                }
            }
        }
    } else {
        const int quad = warp % 4, half = (warp - 2) / 4;
        const unsigned lanes = (unsigned)(quad * 32) << 16;
        int acc = 0, corr = 0;
        unsigned acc_phase = 0, corr_phase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < g.units; u += gridDim.x) {
            const Unit t = unit_at(g, u);
            const int c = t.c0 + quad * 32 + lane;
            const long r0 = (long)t.r0 * BN + half * (BN / 2);
            const bool live = c < g.cols;
            float bias = as_float(static_cast<const IO*>(g.bias)[min(c, g.cols - 1)]);
            if (!g.has_bias) bias = 0.f;
            if constexpr (PLANES == 1) {
                constexpr int N = BN / 2 < 32 ? BN / 2 : 32;
#pragma unroll 1
                for (int j = 0; j < BN / 2; j += N) {
                    const int n = live ? (int)max(0L, min((long)N, g.rows - r0 - j)) : 0;
                    float q[N], v[N];
                    if (g.has_residual) {
                        load_residual<IO, N>(g, r0 + j, c, q);
                    } else {
#pragma unroll
                        for (int i = 0; i < N; ++i) q[i] = 0.f;
                    }
                    if (j == 0) {
                        ok = bar_wait(&bars.acc_full[acc], acc_phase, abort);
                        ok = __all_sync(~0u, ok);
                        if (!ok) break;
                        fence_after();
                    }
                    __syncwarp();
                    tmem_load<N>(tmem + lanes + acc * BN + half * (BN / 2) + j, v);
                    if (j + N == BN / 2) {
                        fence_before();
                        if (lane == 0) bar_arrive(&bars.acc_empty[acc]);
                    }
                    write_out<IO, N>(g, t.split, r0 + j, c, n, bias, q, v);
                }
                if (!ok) break;
                if (++acc == 2) acc = 0, acc_phase ^= 1;
            } else {
                float sum[BN / 2];
#pragma unroll
                for (int j = 0; j < BN / 2; ++j) sum[j] = 0.f;
                for (int kb = 0; kb < t.kbs; kb += kChunk) {
                    ok = bar_wait(&bars.acc_full[acc], acc_phase, abort);
                    ok = __all_sync(~0u, ok);
                    if (!ok) break;
                    fence_after();
#pragma unroll
                    for (int j = 0; j < BN / 2; j += 16) {
                        float v[16];
                        tmem_load<16>(tmem + lanes + acc * BN + half * (BN / 2) + j, v);
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[j + i] += v[i];
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&bars.acc_empty[acc]);
                    if (++acc == 2) acc = 0, acc_phase ^= 1;
                }
                if (!ok) break;
                ok = bar_wait(&bars.corr_full[corr], corr_phase, abort);
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int j = 0; j < BN / 2; j += 16) {
                    const int n = live ? (int)max(0L, min(16L, g.rows - r0 - j)) : 0;
                    float q[16], v[16];
                    if (g.has_residual) {
                        load_residual<IO, 16>(g, r0 + j, c, q);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) q[i] = 0.f;
                    }
                    __syncwarp();
                    tmem_load<16>(corr_base + lanes + corr * BN + half * (BN / 2) + j, v);
                    if (j + 16 == BN / 2) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(&bars.corr_empty[corr]);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = isfinite(sum[j + i]) ? sum[j + i] + v[i] : sum[j + i];
                    write_out<IO, 16>(g, t.split, r0 + j, c, n, bias, q, v);
                }
                if (++corr == 2) corr = 0, corr_phase ^= 1;
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols) : "memory");
    }
}

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

// `inner` contiguous elements per row, `outer` rows `ld` elements apart, `planes` of them; boxes of 64 x box_outer
bool make_map(CUtensorMap* map, const void* base, long inner, long outer, long ld, int planes, int box_outer) {
    const EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * outer * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_outer, 1}, step[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, int PLANES>
cudaError_t launch_shape(const GemmProblem& g, cudaStream_t st) {
    static unsigned long long opted = 0;
    cudaError_t e = opt_in_smem(gemm_kernel<BN, PLANES>, &opted);
    if (e != cudaSuccess) return e;
    const int grid = g.units < kSms ? g.units : kSms;
    gemm_kernel<BN, PLANES><<<grid, kGemmThreads, Shape<BN, PLANES>::kSmem, st>>>(g);
    return cudaPeekAtLastError();
}

}  // namespace

bool gemm_bind(GemmProblem& g, const Operand& p, const Operand& q, int planes, int bn) {
    g.p_mn = p.mn_major;
    g.q_mn = q.mn_major;
    return make_map(&g.p_map, p.base, p.inner, p.outer, p.ld, planes, p.mn_major ? kBK : bn) &&
           make_map(&g.q_map, q.base, q.inner, q.outer, q.ld, planes, q.mn_major ? kBK : kTileC);
}

cudaError_t launch_gemm(const GemmProblem& a, int planes, int bn, cudaStream_t st) {
    if (planes == 3) {
        if (bn == 128) return launch_shape<128, 3>(a, st);
        if (bn == 64) return launch_shape<64, 3>(a, st);
        return launch_shape<32, 3>(a, st);
    }
    if (bn == 256) return launch_shape<256, 1>(a, st);
    if (bn == 128) return launch_shape<128, 1>(a, st);
    if (bn == 64) return launch_shape<64, 1>(a, st);
    return launch_shape<32, 1>(a, st);
}

cudaError_t gemm_gave_up(unsigned* count, cudaStream_t st) {
    const unsigned zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(count, g_gave_up, sizeof(unsigned), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && *count) e = cudaMemcpyToSymbolAsync(g_gave_up, &zero, sizeof(unsigned), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    return e;
}

}  // namespace qk
