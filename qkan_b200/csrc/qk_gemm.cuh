// Matrix products of the linear map on the tensor cores (tcgen05): C[r,c] = sum_k P[r,k] Q[c,k] with the epilogue
// act(C + bias[c]) + residual[r,c].
//
// One CTA per SM walks units of work (a tile of 128 rows and BN columns, a slice of the depth). Two warps copy 64-deep
// blocks of the operands, one each, into a ring of stages (TMA, 128-byte swizzle; one thread for both, at 140 clocks a
// copy, was slower than the MMAs of narrow tiles), warp 1 issues the MMAs, eight warps drain the sums from one of two
// accumulators in tensor memory while the other one is filled. An operand is read as it lies in
// memory: "K-major" when the summed axis is contiguous (forward: x and W), "MN-major" when it is the other axis (W in
// grad_x, x and gz in grad_weight).
//
// A lane of tensor memory is a row of C, so a thread of the epilogue has one row. Results go through 64-byte rows in
// shared memory, from where TMA stores them (rows of whole 16-byte words) or the warp does, row by row. Lanes along the
// columns, two bytes stored by each straight from its registers, made the epilogue the whole time of a product with a short
// depth.
//
// Measured (bfloat16): 8192 x 4096 -> 4096 forward 185 us, 1.48 PFLOP/s, bound by the tensor core; 8192 x 768 -> 768 11.6 us;
// 8192 x 64 -> 768 5.4 us, bound by the epilogue; 64 x 64 -> 64 2.4 us, the latency of one tile. float32: 8192 x 4096 -> 4096
// 1.26 ms, 218 TFLOP/s of 280 that six bfloat16 products leave, bound by shared memory (the MMAs read 192 KB per block of
// 1536 clocks, the copies write 96 KB).
//
// A product of bfloat16 operands can take P in two parts, h + m, with 16 significant bits: gz of a backward, where
// rounding it to eight would show beside the rounding of the result. The depth is walked twice, Q being read again.
//
// The sums of P's rows (grad_bias, where P is gz transposed) come from the tensor core as well: one more column group,
// against a tile of ones.
//
// float32 (PLANES == 3): x = h + m + l exactly, each part a bfloat16 (8 significant bits, float32's exponents). Six of
// the nine products are kept: hh | hm mh hl lh mm; what is dropped is below 2^-22 of |x||w|. hh goes to one accumulator
// and the five small ones to another. The tensor core truncates where it adds to its accumulator, which over a long
// sum would drift by more than float32 rounding does: so hh is drained every kChunk blocks and added in registers, with
// rounding. Where hh's sum is not finite the small products are left out: float32's own infinities come out.
#pragma once

#include <atomic>

#include "qk_linear.cuh"

namespace qk {
namespace {

constexpr int kBK = 64;             // depth of a stage: 128 bytes of bfloat16, one swizzle row
constexpr int kTileR = 128;         // the MMA's M
constexpr int kChunk = 2;           // stages between two drains of hh (float32)
constexpr int kGemmThreads = 352;   // copies of P, MMAs, 8 epilogue warps, copies of Q
constexpr int kDrainWarps = 8;
constexpr int kQWarp = 10;
// The longest that a wait may take: this time, and this many rounds of 64 tries (a try that fails takes 1.36 us, so 1.4 s).
// The clock runs on while another process has the GPU, the tries do not.
constexpr unsigned long long kGiveUpNs = 10ull * 1000 * 1000 * 1000;
constexpr int kGiveUpRounds = 1 << 14;

constexpr int kStoreBytes = 2048;   // 32 rows of 64 bytes: what a warp stages for one store; two of them per warp

// Three kernels of each shape: without and with activation and tape, and one that sums P's rows as well (bfloat16, where
// tensor memory has the room; float32 sums them where it splits them, with rounding). The sums are a few instructions in
// the MMA loop, but products that do not want them took up to a quarter longer with those inside.
enum Kind { kPlain, kFull, kSumRows };
constexpr int kOnesBytes = 512;  // 16 rows of 16, without swizzle: four 8 x 16-byte pieces; every 16 of the depth reads them again

template <int BN, int PLANES, Kind KIND>
struct Shape {
    static constexpr int kABytes = kTileR * 128;
    static constexpr int kBBytes = BN * 128;
    static constexpr int kStageBytes = PLANES * (kABytes + kBBytes);
    static constexpr int kStagingBytes = kDrainWarps * 2 * kStoreBytes;
    static constexpr bool kSums = KIND == kSumRows;
    static constexpr int kExtraBytes = kStagingBytes + (kSums ? kOnesBytes : 0);
    static constexpr int kStagesFit = (225 * 1024 - kExtraBytes) / kStageBytes;
    static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
    static constexpr int kAccCols = 2 * BN;
    static constexpr int kTmemCols = PLANES == 3 || kSums ? 2 * kAccCols : kAccCols;  // a power of two
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kExtraBytes + 1024 + 256;
    static_assert(kStages >= 2 && kTmemCols <= 512 && kSmem <= 227 * 1024, "does not fit an SM");
};

struct Barriers {
    unsigned long long full[8], empty[8];
    unsigned long long acc_full[2], acc_empty[2];    // the accumulator (of hh)
    unsigned long long corr_full[2], corr_empty[2];  // the accumulator of the small products
    unsigned long long drain;
    unsigned tmem;
    int abort;
};

__device__ unsigned g_gave_up;  // waits that ran out; one count for each translation unit, gemm_gave_up() adds them

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
// One lane of a whole warp. The compiler knows what this instruction chooses: what stands behind it is issued once, its
// operands in uniform registers. Behind "lane == 0" a copy took 150 clocks to issue and an MMA 72.
__device__ __forceinline__ bool elect_one() {
    unsigned chosen;
    asm volatile(
        "{\n.reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(chosen));
    return chosen != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase of `parity` to end. Every wait ends: after kGiveUpNs and kGiveUpRounds, or once another warp has given up, the
// answer is false, and the caller leaves its loop.
__device__ __noinline__ bool bar_wait_long(unsigned long long* b, unsigned parity, volatile int* abort) {
    const unsigned long long start = now_ns();
    for (int round = 0; round < kGiveUpRounds || now_ns() - start < kGiveUpNs; ++round) {
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
__device__ __forceinline__ void tma_store(const CUtensorMap* map, unsigned src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src),
                 "r"(x), "r"(y), "r"(z)
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

// The fields of the problem that the loops use, in registers. Read from the parameter itself they are fetched again after
// every asm statement, since its address is taken for the tensor maps.
struct Fields {
    int rows, cols, tiles, tiles_c, kper, kblocks, units, act;
    bool has_bias, has_residual, vec, tma_out;
    const void* bias;
    const void* residual;
    void* out;
    void* tape;
    float* part;
    float* row_sums;
    __device__ __forceinline__ explicit Fields(const GemmProblem& g)
        : rows(g.rows), cols(g.cols), tiles(g.tiles_r * g.tiles_c), tiles_c(g.tiles_c), kper(g.kper), kblocks(g.kblocks),
          units(g.units), act(g.act), has_bias(g.has_bias), has_residual(g.has_residual), vec(g.vec), tma_out(g.tma_out),
          bias(g.bias), residual(g.residual), out(g.out), tape(g.tape), part(g.part),
          row_sums(g.row_sums) {}
};

// One unit of work: a tile of C and a slice of the depth.
struct Unit {
    int r0, c0, kb0, kbs, split;  // first row and column, first block and number of blocks of the slice
};
template <int BN>
__device__ __forceinline__ Unit unit_at(const Fields& f, int u) {
    Unit t;
    t.split = u / f.tiles;
    u -= t.split * f.tiles;
    t.r0 = u / f.tiles_c;  // columns run fastest, so that neighbouring CTAs share P
    t.c0 = (u - t.r0 * f.tiles_c) * BN;
    t.r0 *= kTileR;
    t.kb0 = t.split * f.kper;
    t.kbs = min(f.kper, f.kblocks - t.kb0);
    return t;
}

// What aligned matrices do not need, out of the way of the code that they run: a tile's rows between global memory and a
// staged piece, element by element, a row of N at a time by N lanes. (Staged rows: 64 bytes, their 16-byte words swizzled
// by the row as in the 64-byte swizzle of a tensor map, so that lanes meet no bank twice.)
template <typename T>
__device__ __forceinline__ T* staged(char* piece, int row, int j) {
    return reinterpret_cast<T*>(piece + row * 64 + ((j * (int)sizeof(T) / 16) ^ (row >> 1 & 3)) * 16 + j * (int)sizeof(T) % 16);
}
template <typename T>
__device__ __noinline__ void copy_in(char* piece, const T* from, long r, int c, int rows, int cols) {
    constexpr int N = 64 / sizeof(T);
    const int lane = threadIdx.x % 32, j = lane % N;
#pragma unroll 8
    for (int i = lane / N; i < 32; i += 32 / N)
        if (r + i < rows && c + j < cols) *staged<T>(piece, i, j) = from[(size_t)(r + i) * cols + c + j];
}
template <typename T>
__device__ __noinline__ void copy_out(char* piece, T* to, long r, int c, int rows, int cols) {
    constexpr int N = 64 / sizeof(T);
    const int lane = threadIdx.x % 32, j = lane % N;
#pragma unroll 8
    for (int i = lane / N; i < 32; i += 32 / N)
        if (r + i < rows && c + j < cols) to[(size_t)(r + i) * cols + c + j] = *staged<T>(piece, i, j);
}

// 64 bytes of this lane's row as words; T: float, __nv_bfloat16, or __half for the tape
template <typename T, int N>
__device__ __forceinline__ void pack_row(const float (&v)[N], unsigned (&u)[16]) {
    static_assert(N * sizeof(T) == 64, "a staged row");
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if constexpr (sizeof(T) == 4) {
            u[i] = __float_as_uint(v[i]);
        } else if constexpr (std::is_same_v<T, __half>) {
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
        } else {
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
        }
    }
}

// A warp's way between its registers and 32 rows of a matrix in global memory: two 2 KB pieces of shared memory in turn.
struct Stage {
    char* buf;
    unsigned flip;
    bool leader;  // the lane that issues the copies and waits for them
    __device__ __forceinline__ char* next() {
        // all but the latest store have been read out of shared memory: the piece of the one before that is free
        if (leader) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        __syncwarp();
        char* b = buf + flip * kStoreBytes;
        flip ^= 1;
        return b;
    }
    // N elements per lane, by way of piece b, to rows r .. r + 31, columns c .. c + N - 1, of slice z
    template <typename T, int N>
    __device__ __forceinline__ void store(char* b, const CUtensorMap* map, void* out, const Fields& f, const float (&v)[N],
                                          long r, int c, int z) {
        unsigned u[16];
        pack_row<T>(v, u);
        store_words<T>(b, map, out, f, u, r, c, z);
    }
    template <typename T>
    __device__ __forceinline__ void store_words(char* b, const CUtensorMap* map, void* out, const Fields& f,
                                                const unsigned (&u)[16], long r, int c, int z) {
        const int lane = threadIdx.x % 32;
        uint4* row = reinterpret_cast<uint4*>(b + lane * 64);
        const int x = lane >> 1 & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) row[i ^ x] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
        if (f.tma_out) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (leader) {
                if (r < f.rows && c < f.cols) tma_store(map, smem_u32(b), c, (int)r, z);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            __syncwarp();
            copy_out<T>(b, static_cast<T*>(out) + (size_t)z * f.rows * f.cols, r, c, f.rows, f.cols);
            __syncwarp();
        }
    }
};

// 32 rows of 64 bytes of the residual on their way: four lanes to a row, so that a load meets 8 lines and not 32 (with a
// row per lane the loads of a 128 x 128 tile took 2000 clocks). Rows are held inside the matrix, whole pieces only: what
// a ragged edge cuts is fetched when it is needed.
struct Ahead {
    uint4 w[4];
    template <typename T>
    __device__ __forceinline__ void fetch(const Fields& f, long r, int c) {
        const int lane = threadIdx.x % 32;
        if (!f.vec || c + 64 / (int)sizeof(T) > f.cols) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long row = min(r + 8 * i + lane / 4, f.rows - 1L);
            w[i] = reinterpret_cast<const uint4*>(static_cast<const T*>(f.residual) + (size_t)row * f.cols + c)[lane % 4];
        }
    }
    // adds them to v, lane by lane a row, by way of piece b
    template <typename T, int N>
    __device__ __forceinline__ void add(char* b, const Fields& f, long r, int c, float (&v)[N]) {
        const int lane = threadIdx.x % 32;
        if (!f.vec || c + N > f.cols) {
            copy_in<T>(b, static_cast<const T*>(f.residual), r, c, f.rows, f.cols);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 8 * i + lane / 4;
                reinterpret_cast<uint4*>(b + row * 64)[lane % 4 ^ (row >> 1 & 3)] = w[i];
            }
        }
        __syncwarp();
        const uint4* own = reinterpret_cast<const uint4*>(b + lane * 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 q = own[i ^ (lane >> 1 & 3)];
            const unsigned u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    v[4 * i + k] += __uint_as_float(u[k]);
                } else {
                    v[8 * i + 2 * k] += __uint_as_float(u[k] << 16);
                    v[8 * i + 2 * k + 1] += __uint_as_float(u[k] & 0xffff0000u);
                }
            }
        }
        // a lane writes its own row of the piece next, and no other one's: no barrier
    }
};

// The epilogue of one piece: N sums per lane, which has row r + lane, from column c on. bias: lane i has that of column
// c + i; q: the residual. FULL: with activation and tape.
template <typename IO, bool FULL, int N>
__device__ __forceinline__ void write_out(const GemmProblem& g, const Fields& f, Stage& stage, long r, int c, float bias,
                                          Ahead& q, float (&v)[N]) {
    if (f.has_bias) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_sync(~0u, bias, i);
    }
    if constexpr (FULL) {
        if (f.tape) {
            char* b = stage.next();
            if (sizeof(IO) == 2 && f.act == QK_ACT_RELU) {
                unsigned u[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    u[i] = (unsigned)__half_as_ushort(tape_half(v[2 * i % N], f.act)) |
                           (unsigned)__half_as_ushort(tape_half(v[(2 * i + 1) % N], f.act)) << 16;
                stage.store_words<__half>(b, &g.tape_map, f.tape, f, u, r, c, 0);
            } else {
                stage.store<std::conditional_t<sizeof(IO) == 2, __half, float>>(b, &g.tape_map, f.tape, f, v, r, c, 0);
            }
        }
        activate_all<sizeof(IO) == 2>(v, f.act);
    }
    char* b = stage.next();
    if (f.has_residual) q.add<IO>(b, f, r, c, v);
    stage.store<IO>(b, &g.out_map, f.out, f, v, r, c, 0);
}

// Where a warp of the epilogue stands: the next accumulator of each kind and its phase.
struct Drain {
    int acc = 0, corr = 0;
    unsigned acc_phase = 0, corr_phase = 0;

    // One unit: rows r0 .. r0 + 31, W columns of the tile from `offset` on. main, small: the accumulators of BN columns;
    // lanes: the warp's part of tensor memory. False: a wait was given up.
    template <typename IO, Kind KIND, int PLANES, int BN, int W>
    __device__ __forceinline__ bool unit(const GemmProblem& g, const Fields& f, Stage& out, Barriers& bars, const Unit& t,
                                         long r0, int offset, unsigned main, unsigned small, unsigned lanes) {
        constexpr int N = 64 / sizeof(IO);  // columns of a piece
        constexpr bool FULL = KIND == kFull;
        volatile int* abort = &bars.abort;
        const int lane = threadIdx.x % 32, c0 = t.c0 + offset;
        auto bias_of = [&](int c) { return f.has_bias ? as_float(static_cast<const IO*>(f.bias)[min(c + lane, f.cols - 1)]) : 0.f; };
        bool ok;
        Ahead q[PLANES == 1 ? 2 : 1];  // residual of this piece and of the next (float32 has no registers for two)
        float bias = bias_of(c0), next_bias = 0.f;
        if (f.has_residual) q[0].template fetch<IO>(f, r0, c0);
        if constexpr (PLANES == 1) {
            ok = bar_wait(&bars.acc_full[acc], acc_phase, abort);
            if (!__all_sync(~0u, ok)) return false;
            fence_after();
            const unsigned from = main + lanes + acc * BN + offset;
            if constexpr (KIND == kSumRows) {
                if (f.row_sums && t.c0 == 0 && offset == 0) {
                    unsigned sum;
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\ntcgen05.wait::ld.sync.aligned;"
                                 : "=r"(sum)
                                 : "r"(main + 2 * BN + lanes + acc * 16)
                                 : "memory");
                    if (r0 + lane < f.rows) f.row_sums[(size_t)t.split * f.rows + r0 + lane] = __uint_as_float(sum);
                    __syncwarp();
                }
            }
            if (f.part) {
#pragma unroll 1
                for (int j = 0; j < W; j += 16) {
                    float v[16];
                    __syncwarp();
                    tmem_load<16>(from + j, v);
                    if (j + 16 == W) {
                        fence_before();
                        if (lane == 0) bar_arrive(&bars.acc_empty[acc]);
                    }
                    out.store<float>(out.next(), &g.out_map, f.part, f, v, r0, c0 + j, t.split);
                }
            } else {
                // two pieces a turn, so that the residuals change places without being moved
                constexpr int kTurn = W < 2 * N ? 1 : 2;
#pragma unroll 1
                for (int j = 0; j < W; j += kTurn * N) {
#pragma unroll
                    for (int h = 0; h < kTurn; ++h) {
                        const int at = j + h * N;
                        float v[N];
                        __syncwarp();
                        tmem_load<N>(from + at, v);
                        if (at + N == W) {
                            fence_before();
                            if (lane == 0) bar_arrive(&bars.acc_empty[acc]);
                        } else {
                            next_bias = bias_of(c0 + at + N);
                            if (f.has_residual) q[(h + 1) % 2].template fetch<IO>(f, r0, c0 + at + N);
                        }
                        write_out<IO, FULL, N>(g, f, out, r0, c0 + at, bias, q[h], v);
                        bias = next_bias;
                    }
                }
            }
            if (++acc == 2) acc = 0, acc_phase ^= 1;
        } else {
            float sum[W];
#pragma unroll
            for (int j = 0; j < W; ++j) sum[j] = 0.f;
            for (int kb = 0; kb < t.kbs; kb += kChunk) {
                ok = bar_wait(&bars.acc_full[acc], acc_phase, abort);
                if (!__all_sync(~0u, ok)) return false;
                fence_after();
#pragma unroll
                for (int j = 0; j < W; j += 16) {
                    float v[16];
                    tmem_load<16>(main + lanes + acc * BN + offset + j, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[j + i] += v[i];
                }
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&bars.acc_empty[acc]);
                if (++acc == 2) acc = 0, acc_phase ^= 1;
            }
            ok = bar_wait(&bars.corr_full[corr], corr_phase, abort);
            if (!__all_sync(~0u, ok)) return false;
            fence_after();
#pragma unroll
            for (int j = 0; j < W; j += 16) {
                float v[16];
                __syncwarp();
                tmem_load<16>(small + lanes + corr * BN + offset + j, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[j + i] = isfinite(sum[j + i]) ? sum[j + i] + v[i] : sum[j + i];
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars.corr_empty[corr]);
            if (++corr == 2) corr = 0, corr_phase ^= 1;
            // the sums leave sixteen at a time, the others moving up: one copy of the epilogue's code
#pragma unroll 1
            for (int j = 0; j < W; j += 32) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = j + h * 16;
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = sum[h * 16 + i];
                    if (f.part) {
                        out.store<float>(out.next(), &g.out_map, f.part, f, v, r0, c0 + at, t.split);
                        continue;
                    }
                    if (at + N < W) next_bias = bias_of(c0 + at + N);
                    write_out<IO, FULL, 16>(g, f, out, r0, c0 + at, bias, q[0], v);
                    bias = next_bias;
                    if (f.has_residual && at + N < W) q[0].template fetch<IO>(f, r0, c0 + at + N);
                }
#pragma unroll
                for (int i = 0; i + 32 < W; ++i) sum[i] = sum[i + 32];
            }
        }
        return true;
    }
};

template <int BN, int PLANES, Kind KIND>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmArgs a) {
    const bool second = (int)blockIdx.x >= a.first;
    const GemmProblem& g = second ? a.g[1] : a.g[0];
    const int cta = blockIdx.x - (second ? a.first : 0), ctas = second ? a.ctas - a.first : a.first;
    using S = Shape<BN, PLANES, KIND>;
    using IO = std::conditional_t<PLANES == 3, float, __nv_bfloat16>;
    extern __shared__ char raw[];
    char* stages = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    char* staging = stages + (size_t)S::kStages * S::kStageBytes;
    char* ones = staging + S::kStagingBytes;
    Barriers& bars = *reinterpret_cast<Barriers*>(staging + S::kExtraBytes);
    static_assert(sizeof(Barriers) <= 256, "barriers");
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    volatile int* abort = &bars.abort;
    const Fields f(g);
    if (threadIdx.x == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&g.p_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&g.q_map) : "memory");
        if (f.tma_out) asm volatile("prefetch.tensormap [%0];" ::"l"(&g.out_map) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) bar_init(&bars.full[i], 2), bar_init(&bars.empty[i], 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(&bars.acc_full[i], 1), bar_init(&bars.acc_empty[i], kDrainWarps);
            bar_init(&bars.corr_full[i], 1), bar_init(&bars.corr_empty[i], kDrainWarps);
        }
        bar_init(&bars.drain, 1);
        bars.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (S::kSums) {
        if (threadIdx.x < kOnesBytes / 16)
            reinterpret_cast<uint4*>(ones)[threadIdx.x] = make_uint4(0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
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
    after_previous();

    if (warp == 0 || warp == kQWarp) {
        if (elect_one()) {
            // an operand's copies: K-major, one box of a tile's rows; MN-major, boxes 64 wide, 8 KB each
            const bool is_p = warp == 0;
            const CUtensorMap* map = is_p ? &g.p_map : &g.q_map;
            const int boxes = is_p ? g.p_boxes : g.q_boxes;
            const bool mn = is_p ? g.p_mn : g.q_mn;
            const unsigned bytes = PLANES * boxes * (is_p ? g.p_box_bytes : g.q_box_bytes);
            const unsigned base = smem_u32(stages) + (is_p ? 0 : PLANES * S::kABytes);
            const unsigned plane = is_p ? S::kABytes : S::kBBytes;
            const int wrap = g.wrap;
            int stage = 0;
            unsigned phase = 0, issued = 0;
            bool ok = true;
            for (int u = cta; ok && u < f.units; u += ctas) {
                const Unit t = unit_at<BN>(f, u);
                const int row = is_p ? t.r0 : t.c0;
                for (int kb = t.kb0; kb < t.kb0 + t.kbs; ++kb) {
                    const bool again = kb >= wrap;  // P's second part, Q once more
                    const int k = (again ? kb - wrap : kb) * kBK, z = again && is_p ? 1 : 0;
                    ok = bar_wait(&bars.empty[stage], phase ^ 1, abort);
                    if (!ok) break;
                    unsigned long long* bar = &bars.full[stage];
                    bar_expect(bar, bytes);
                    unsigned dst = base + stage * S::kStageBytes;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p, dst += plane) {
                        if (mn) {
                            for (int b = 0; b < boxes; ++b) tma_load(map, dst + b * 8192, bar, row + b * 64, k, z + p);
                        } else {
                            tma_load(map, dst, bar, k, row, z + p);
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
        if (elect_one()) {
            int stage = 0, acc = 0, corr = 0;
            unsigned phase = 0, acc_phase = 0, corr_phase = 0;
            bool ok = true;
            const bool p_mn = g.p_mn, q_mn = g.q_mn;
            // D float32, A and B bfloat16, which of them MN-major, N / 8, M / 16
            const unsigned idesc = 1u << 4 | 1u << 7 | 1u << 10 | (unsigned)p_mn << 15 | (unsigned)q_mn << 16 |
                                   (BN / 8) << 17 | (kTileR / 16) << 24;
            const unsigned a_step = p_mn ? 2048 >> 4 : 32 >> 4, b_step = q_mn ? 2048 >> 4 : 32 >> 4;
            const unsigned long long a_desc = smem_desc(smem_u32(stages), p_mn);
            const unsigned long long b_desc = smem_desc(smem_u32(stages) + PLANES * S::kABytes, q_mn);
            const unsigned long long ones_desc = (unsigned long long)((smem_u32(ones) & 0x3ffff) >> 4) | (128ull >> 4) << 16 |
                                                 (256ull >> 4) << 32 | 1ull << 46;
            const unsigned ones_idesc = (idesc & ~(1u << 16 | 0x3fu << 17)) | (16 / 8) << 17;  // K-major, 16 columns
            for (int u = cta; ok && u < f.units; u += ctas) {
                const Unit t = unit_at<BN>(f, u);
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
                    const unsigned long long da = a_desc + stage * (S::kStageBytes >> 4);
                    const unsigned long long db = b_desc + stage * (S::kStageBytes >> 4);
                    const unsigned d = tmem + acc * BN;
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma(d, da + k * a_step, db + k * b_step, idesc, !(opens && k == 0));
                    if constexpr (S::kSums) {
                        if (f.row_sums && t.c0 == 0) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma(tmem + S::kAccCols + acc * 16, da + k * a_step, ones_desc, ones_idesc, !(opens && k == 0));
                        }
                    }
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
        // a warp reads the 32 lanes of its number mod 4; two warps share them, half of the columns each
        const int quad = warp % 4, half = (warp - 2) / 4;
        const unsigned lanes = (unsigned)(quad * 32) << 16;
        Stage out{staging + (warp - 2) * 2 * kStoreBytes, 0, elect_one()};
        Drain d;
        bool ok = true;
        for (int u = cta; ok && u < f.units; u += ctas) {
            const Unit t = unit_at<BN>(f, u);
            ok = d.unit<IO, KIND, PLANES, BN, BN / 2>(g, f, out, bars, t, t.r0 + quad * 32, half * (BN / 2), tmem, corr_base,
                                                      lanes);
        }
        // shared memory is given up once every store has read its piece
        if (out.leader) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols) : "memory");
    }
}

template <int BN, int PLANES, Kind KIND>
cudaError_t launch_shape(const GemmArgs& a, cudaStream_t st) {
    using S = Shape<BN, PLANES, KIND>;
    static unsigned long long opted = 0;
    cudaError_t e = opt_in_smem(gemm_kernel<BN, PLANES, KIND>, &opted, (int)S::kSmem);
    if (e != cudaSuccess) return e;
    return launch_after(gemm_kernel<BN, PLANES, KIND>, a.ctas, kGemmThreads, S::kSmem, st, a);
}

template <int BN, int PLANES>
cudaError_t launch_tile(const GemmArgs& a, cudaStream_t st) {
    const GemmProblem& g = a.g[0];  // two problems: gradients, neither has an activation
    if (!g.part && (g.tape || g.act != QK_ACT_NONE)) return launch_shape<BN, PLANES, kFull>(a, st);
    if constexpr (PLANES == 1 && BN <= 128)
        if (g.row_sums) return launch_shape<BN, PLANES, kSumRows>(a, st);
    return g.row_sums ? cudaErrorInvalidValue : launch_shape<BN, PLANES, kPlain>(a, st);
}

// Adds this unit's waits that ran out since the last call; synchronises the stream. The count on the device only grows, and
// what was reported of it is kept here: clearing it would lose a wait of another stream between the read and the write.
inline cudaError_t take_gave_up(unsigned* total, cudaStream_t st) {
    static std::atomic<unsigned> reported[64];
    int dev = 0;
    unsigned n = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&n, g_gave_up, sizeof n, 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return e;
    unsigned before = reported[dev & 63].load();
    while (n > before && !reported[dev & 63].compare_exchange_weak(before, n)) {
    }
    if (n > before) *total += n - before;
    return e;
}

}  // namespace
}  // namespace qk
