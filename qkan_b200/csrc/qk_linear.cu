// The linear map y = act(x W^T + b) + r and its backward pass: choice of tiles, scratch, launch sequence, and the small
// kernels around the products of qk_gemm.cu.
//
//   prepare   operands that the products cannot read where they lie: float32 is split into three bfloat16 parts, rows
//             that are no multiple of 16 bytes are padded, and in the backward gz = gy * act'(tape) is formed, with
//             its column sums for grad_bias on the way
//   products  forward: one; backward: grad_weight and grad_x, in one launch where both fit the GPU side by side. A few rows
//             take the kernels of qk_gemv.cu in both directions, few outputs or little of everything in float32 the one of
//             qk_narrow.cu forward; neither needs anything prepared.
//   reduce    adds the slices of a depth that was cut for want of tiles, then the epilogue; adds grad_bias' slabs
#include "qk_linear.cuh"

namespace qk {
namespace {

constexpr int kThreads = 256;

struct PrepJob {
    const void* src;
    const void* tape;      // nullptr: the source as it is
    __nv_bfloat16* dst;    // [parts][rows][ld]; nullptr: column sums only
    bool two;              // bfloat16: two parts, h + m (float32 has three)
    float* colpart;        // [slabs][cols]; nullptr: not wanted
    int rows, cols, ld, act;
    int slab_rows, cblocks, tx_log2, blocks;
    bool vec;              // whole 8-column groups, 16-byte aligned
};
struct PrepArgsL {
    PrepJob job[3];
    int count;
};

// x = h + m + l, two values at a time. h is x cut off after eight bits (rounding could reach infinity), m and l round
// what is left, which is exact in float32 until l has it all. For an infinity or a NaN h is that, and m and l are NaN:
// the products leave theirs out where h's are not finite.
__device__ __forceinline__ void split3(float x, float y, unsigned& h, unsigned& m, unsigned& l) {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(y), "f"(x));
    x -= __uint_as_float(h << 16), y -= __uint_as_float(h & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(m) : "f"(y), "f"(x));
    x -= __uint_as_float(m << 16), y -= __uint_as_float(m & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(l) : "f"(y), "f"(x));
}

// x = h + m to within 2^-16 of x, for products that add both parts' to one sum. An infinity in the other operand has to give
// an infinity there and not inf - inf or 0 * inf: so h is cut off, which leaves m the sign of x, and m is not zero beside an h
// that is not (2^-24 of it, for |h| from 2^-109 on). Beside an infinite h m is infinite too.
__device__ __forceinline__ void split2(float x, float y, unsigned& h, unsigned& m) {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(y), "f"(x));
    auto rest = [](float v, float cut) { return copysignf(fmaxf(fabsf(v - cut), fabsf(cut) * 0x1p-24f), v); };
    x = rest(x, __uint_as_float(h << 16)), y = rest(y, __uint_as_float(h & 0xffff0000u));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(m) : "f"(y), "f"(x));
}

template <typename IO>
__device__ __forceinline__ void load8(const void* p, size_t at, bool vec, int n, float (&v)[8]) {
    const IO* s = static_cast<const IO*>(p) + at;
    if (vec) {
        if constexpr (sizeof(IO) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(s), b = reinterpret_cast<const float4*>(s)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(s);
            const unsigned u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const IO* q = reinterpret_cast<const IO*>(&u[i]);
                v[2 * i] = as_float(q[0]), v[2 * i + 1] = as_float(q[1]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? as_float(s[i]) : 0.f;
    }
}

// Bound by memory: reads the source once, writes 2 (bfloat16; gz in two parts 4) or 6 (float32) bytes per element. A thread owns eight
// columns and walks the rows of a slab, so that column sums stay in its registers. Measured, x and gy of 65536 x 256 and a
// small W in float32: 54 us for 336 MB, 6.2 TB/s; gz in two parts and its sums, 16384 x 2048 in bfloat16 with SiLU: 59 us for
// 268 MB (in one part 50 for 201), bound by the slope's instructions.
template <typename IO>
__global__ void __launch_bounds__(kThreads) prepare_kernel(const PrepArgsL a) {
    __shared__ float sums[kThreads * 8];
    after_previous();
    int b = blockIdx.x;
    PrepJob j = a.job[0];  // in registers: a reference would be read again behind every store
    if (a.count > 1 && b >= a.job[0].blocks) {
        b -= a.job[0].blocks;
        j = a.job[1];
        if (a.count > 2 && b >= a.job[1].blocks) {
            b -= a.job[1].blocks;
            j = a.job[2];
        }
    }
    const int tx = threadIdx.x & ((1 << j.tx_log2) - 1), ty = threadIdx.x >> j.tx_log2, ny = kThreads >> j.tx_log2;
    const int slab = b / j.cblocks, c = ((b - slab * j.cblocks) << j.tx_log2 | tx) * 8;
    const long end = min((long)j.rows, (long)(slab + 1) * j.slab_rows);
    const size_t plane = (size_t)j.rows * j.ld;
    float sum[8] = {};
    if (c < j.ld) {
        const int n = min(8, j.cols - c);  // none in the padding
        const bool vec = j.vec && n > 0;
#pragma unroll 4
        for (long r = (long)slab * j.slab_rows + ty; r < end; r += ny) {
            const size_t at = (size_t)r * j.cols + c;
            float v[8];
            load8<IO>(j.src, at, vec, n, v);
            if (j.tape) {
                float z[8];
                if constexpr (sizeof(IO) == 4) load8<float>(j.tape, at, vec, n, z);
                else load8<__half>(j.tape, at, vec, n, z);
                times_slope<sizeof(IO) == 2>(v, z, j.act);  // columns past the end: 0 times a slope at 0
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[i];
            if (!j.dst) continue;
            uint4* out = reinterpret_cast<uint4*>(j.dst + (size_t)r * j.ld + c);
            unsigned h[4];
            if constexpr (sizeof(IO) == 4) {
                unsigned m[4], l[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) split3(v[2 * i], v[2 * i + 1], h[i], m[i], l[i]);
                out[plane / 8] = make_uint4(m[0], m[1], m[2], m[3]);
                out[plane / 4] = make_uint4(l[0], l[1], l[2], l[3]);
            } else {
                if (j.two) {
                    unsigned m[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) split2(v[2 * i], v[2 * i + 1], h[i], m[i]);
                    out[plane / 8] = make_uint4(m[0], m[1], m[2], m[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
                }
            }
            out[0] = make_uint4(h[0], h[1], h[2], h[3]);
        }
    }
    if (!j.colpart) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[(ty << j.tx_log2 | tx) * 8 + i] = sum[i];
    __syncthreads();
    const int width = 8 << j.tx_log2;
    for (int t = threadIdx.x; t < width; t += kThreads) {
        const int col = (b - slab * j.cblocks) * width + t;
        if (col >= j.cols) break;
        double s = 0.;  // up to 256 of them in order
        for (int y = 0; y < ny; ++y) s += sums[y * width + t];
        j.colpart[(size_t)slab * j.cols + col] = (float)s;
    }
}

struct ReduceJob {
    const float* part;  // [splits][rows][cols]; splits 0: sums of nothing
    int splits, cols, blocks;
    bool tall;          // many slices of few sums: eight threads share a sum
    size_t n;
    Epilogue epi;
};
struct ReduceArgs {
    ReduceJob job[2];
    int count;
    const float* colpart;  // [slabs][cols]
    void* gb;
    int slabs, cols, io_dtype;
};

// The sum over `count` slices, n apart, of 32 neighbouring elements, by 256 threads; valid in the first 32 of them. In double:
// some hundred float32 additions in order were most of grad_bias' error (1000 x 4096 -> 16 1.8e-7, torch's sums 8e-8).
__device__ __forceinline__ float tall_sum(const float* part, size_t n, size_t at, int count, double (&tile)[8][33]) {
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    double s = 0.;
    if (at < n) {
#pragma unroll 8
        for (int k = y; k < count; k += 8) s += part[(size_t)k * n + at];
    }
    tile[y][x] = s;
    __syncthreads();
    if (y == 0) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += tile[k][x];
    }
    return (float)s;
}

// The slices of each sum in a fixed order, then the epilogue: an element per thread, or (tall) 32 per CTA. The blocks
// behind those add grad_bias' slabs, 32 columns each.
__global__ void __launch_bounds__(kThreads) reduce_kernel(const ReduceArgs a) {
    after_previous();
    __shared__ double tile[8][33];
    int b = blockIdx.x;
    ReduceJob j = a.job[0];
    bool sums = a.count > 0 && b < j.blocks;
    if (a.count > 0 && !sums) {
        b -= j.blocks;
        j = a.job[1];
        sums = a.count > 1 && b < j.blocks;
        if (a.count > 1 && !sums) b -= j.blocks;
    }
    if (sums && !j.tall) {
        const size_t i = (size_t)b * kThreads + threadIdx.x;
        if (i >= j.n) return;
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < j.splits; ++k) s += j.part[(size_t)k * j.n + i];
        finish_element(j.epi, i, (int)(i % j.cols), s);
    } else if (sums) {
        const size_t i = (size_t)b * 32 + threadIdx.x % 32;
        const float s = tall_sum(j.part, j.n, i, j.splits, tile);
        if (threadIdx.x < 32 && i < j.n) finish_element(j.epi, i, (int)(i % j.cols), s);
    } else {
        const size_t c = (size_t)b * 32 + threadIdx.x % 32;
        const float s = tall_sum(a.colpart, a.cols, c, a.slabs, tile);
        if (threadIdx.x < 32 && c < a.cols) store_dt(a.gb, c, a.io_dtype, s);
    }
}

// ---- choice of tiles -----------------------------------------------------------
// Clocks of one SM, from the rates of its parts: the tensor core takes 2 BN clocks for a 128 x BN x 64 block, six times
// that in float32; L2 feeds some 56 bytes per clock; the epilogue takes about 12 clocks per column.
struct Cut {
    int splits, kper;
};

struct Size {
    long rows, cols;
    int kblocks;
    long tiles(int bn) const { return (rows + 127) / 128 * ((cols + bn - 1) / bn); }
};

double block_clocks(const Size& s, int bn, int planes) {
    const double mma = 2.0 * bn * (planes == 3 ? 6 : 1);
    const double rows = (s.rows < 128 ? s.rows : 128) + (s.cols < bn ? s.cols : bn), load = planes * rows * 128 / 56 + 100;
    return mma > load ? mma : load;
}
double drain_clocks(int bn) { return 12.0 * bn + 500; }

Cut cut_into(int kblocks, int splits) {
    Cut c;
    c.kper = (kblocks + splits - 1) / splits;
    c.splits = (kblocks + c.kper - 1) / c.kper;
    return c;
}

constexpr int kCuts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 148};
constexpr long kMostPart = 64l << 20;  // floats of partial sums: 256 MB

struct Plan {
    int bn;
    Cut cut;
};

double cost_of(const Size& s, int bn, int planes, const Cut& c) {
    const long units = s.tiles(bn) * c.splits;
    const double mainloop = c.kper * block_clocks(s, bn, planes), drain = drain_clocks(bn);
    double t = (double)((units + kSms - 1) / kSms) * (mainloop > drain ? mainloop : drain) + drain + 2500;
    if (c.splits > 1) t += 4800 + 2.0 * c.splits * s.rows * s.cols * 4 / (kSms * 24.0);
    return t;
}

// the cheapest plan, of at most `most_units` units where that is not 0, with tiles of `only_bn` columns where that is not
Plan plan_for(const Size& s, int planes, double* cost = nullptr, long most_units = 0, int only_bn = 0, int most_bn = 256) {
    Plan best{};
    double least = 1e300;
    for (int bn = planes == 3 ? 128 : 256; bn >= 64; bn /= 2) {
        if ((only_bn && bn != only_bn) || bn > most_bn) continue;
        for (int k : kCuts) {
            if (k > 1 && (k > s.kblocks || s.tiles(bn) * k > 4l * kSms || (double)k * s.rows * s.cols > kMostPart)) break;
            const Cut c = cut_into(s.kblocks, k);
            if (most_units && s.tiles(bn) * c.splits > most_units) break;
            const double t = cost_of(s, bn, planes, c);
            if (t < least) least = t, best = {bn, c};
        }
    }
    if (cost) *cost = least;
    return best;
}

// Two products in one launch: where both fit the SMs side by side, that costs the longer of the two, not the sum.
// False: one after the other is cheaper. Tiles have at most `most_bn` columns.
bool plan_pair(const Size& a, const Size& b, int planes, Plan* pa, Plan* pb, double* cost, int most_bn = 256) {
    double ca, cb;
    *pa = plan_for(a, planes, &ca, 0, 0, most_bn);
    *pb = plan_for(b, planes, &cb, 0, 0, most_bn);
    double least = ca + cb;
    bool together = false;
    for (int bn = planes == 3 || most_bn < 256 ? 128 : 256; bn >= 64; bn /= 2)
        for (int first = kSms / 8; first < kSms; first += kSms / 8) {
            double ta, tb;
            const Plan qa = plan_for(a, planes, &ta, first, bn), qb = plan_for(b, planes, &tb, kSms - first, bn);
            const double t = ta > tb ? ta : tb;
            if (t < least) least = t, *pa = qa, *pb = qb, together = true;
        }
    *cost = least;
    return together;
}

// ---- scratch -------------------------------------------------------------------
int planes_of(int io_dtype) { return io_dtype == QK_F32 ? 3 : 1; }
// Packed rows: whole 16-byte words, and 128 bytes at least, which is what a copy takes of them (rows of 32 bytes came
// 1 to 2 us later)
long padded(long n) { return n < 64 ? 64 : (n + 7) / 8 * 8; }
size_t packed_bytes(long rows, long cols, int planes) { return align256((size_t)planes * rows * padded(cols) * 2); }
int blocks_of(long depth) { return (int)((depth + 63) / 64); }

struct Slabs {
    int rows, count, cblocks, tx_log2;
};
// 256 threads as 2^tx_log2 groups of eight columns by the rest in rows; enough slabs of rows for four CTAs per SM, each
// of four rows per thread at least
Slabs slabs_of(long rows, long cols) {
    const long groups = padded(cols) / 8;
    Slabs s{};
    while (s.tx_log2 < 5 && (1 << s.tx_log2) < groups) ++s.tx_log2;
    s.cblocks = (int)((groups + (1 << s.tx_log2) - 1) >> s.tx_log2);
    const long ny = kThreads >> s.tx_log2;
    long want = (4l * kSms + s.cblocks - 1) / s.cblocks;
    const long most = (rows + 4 * ny - 1) / (4 * ny);
    if (want > most) want = most;
    if (want < 1) want = 1;
    s.rows = (int)((rows + want - 1) / want);
    s.count = (int)((rows + s.rows - 1) / s.rows);
    return s;
}

struct ForwardScratch {
    Plan plan;
    NarrowPlan narrow;  // few outputs or little of everything in float32
    size_t x, w, part, total;
};
ForwardScratch plan_forward(const QkLinearDesc& d) {
    ForwardScratch s{};
    if (is_narrow(d.rows, d.out_features, d.in_features, d.io_dtype)) {
        s.narrow = narrow_plan(d.rows, d.out_features, d.in_features);
        if (s.narrow.splits > 1) s.total = align256((size_t)s.narrow.splits * d.rows * d.out_features * 4);
        return s;
    }
    const int planes = planes_of(d.io_dtype);
    const bool pack = !reads_in_place(d.in_features, d.io_dtype);
    s.plan = plan_for({d.rows, d.out_features, blocks_of(d.in_features)}, planes);
    s.x = 0;
    s.w = pack ? packed_bytes(d.rows, d.in_features, planes) : 0;
    s.part = s.w + (pack ? packed_bytes(d.out_features, d.in_features, planes) : 0);
    s.total = s.part;
    if (s.plan.cut.splits > 1) s.total += align256((size_t)s.plan.cut.splits * d.rows * d.out_features * 4);
    return s;
}

// The layout is that of all gradients, whatever is asked for. grad_bias: the sums of gz's columns come from the products
// (the tensor core sums gz as it makes grad_weight) where nothing else needs to go over gz, else from prepare.
//
// gz in bfloat16: where it is not gy itself it is taken in two parts, products of twice the depth, so that the gradients
// carry the rounding of their own type alone. Rounded to bfloat16 once, as a framework that stores gz has it, its error is as
// large as that of rounding the gradients, whatever the depth: theirs is 1.41 times as large then (measured at 800 x 72 ->
// 400 and 8192 x 4096 -> 4096), or up to twice where one term makes the sum. The caller can ask for that
// (QK_LINEAR_ROUND_GRADS); all gradients with SiLU then take, in us, 500 for 856 at 8192 x 4096 -> 4096, 68 for 85 at
// 65536 x 256 -> 256, 16.6 for 18.7 at 1501 x 517 -> 333. Few rows have gz in float32.
struct BackwardScratch {
    Plan plan_w, plan_x;
    bool two;       // gz in two parts
    FewPlan few;    // slab 0: not a matter of few rows
    bool together;  // both products in one launch
    bool sums;      // grad_weight's product can sum gz's columns
    Slabs slabs;
    size_t gz, x, w, colpart, part_w, part_x, total;
};
BackwardScratch plan_backward(const QkLinearDesc& d) {
    BackwardScratch s{};
    const int planes = planes_of(d.io_dtype);
    const long M = d.rows, K = d.in_features, N = d.out_features;
    const bool pack_gz = d.activation != QK_ACT_NONE || !reads_in_place(N, d.io_dtype);
    const bool pack = !reads_in_place(K, d.io_dtype);
    if (few_rows_backward(d.rows, d.io_dtype)) {
        s.few = few_plan((int)K, (int)N);
        s.total = align256((size_t)s.few.slabs * M * K * 4);  // partial sums of grad_x
        return s;
    }
    s.two = d.activation != QK_ACT_NONE && planes == 1 && !(d.flags & QK_LINEAR_ROUND_GRADS);
    const int times = s.two ? 2 : 1;
    const Size size_w{N, K, times * blocks_of(M)}, size_x{M, K, times * blocks_of(N)};
    double least = 0;
    s.together = K > 0 && plan_pair(size_w, size_x, planes, &s.plan_w, &s.plan_x, &least);
    if (!pack_gz && s.plan_w.bn > 128) {
        // Narrower tiles, whose product can sum gz, save the pass over gz: both products in one launch with such tiles, or
        // grad_weight's alone with them and grad_x's as is best for it.
        least += 5000 + 2.0 * M * N / (kSms * 16);
        Plan w, x;
        double cost, cost_x;
        if (plan_pair(size_w, size_x, planes, &w, &x, &cost, 128) && cost < least) least = cost, s.plan_w = w, s.plan_x = x, s.together = true;
        w = plan_for(size_w, planes, &cost, 0, 0, 128), x = plan_for(size_x, planes, &cost_x);
        if (cost + cost_x < least) s.plan_w = w, s.plan_x = x, s.together = false;
    }
    s.slabs = slabs_of(M, N);
    s.sums = K > 0 && !pack_gz && s.plan_w.bn <= 128;
    s.gz = 0;
    s.x = pack_gz ? packed_bytes(M, N, s.two ? 2 : planes) : 0;
    s.w = s.x + (pack ? packed_bytes(M, K, planes) : 0);
    s.colpart = s.w + (pack ? packed_bytes(N, K, planes) : 0);
    const int parts = s.sums && s.plan_w.cut.splits > s.slabs.count ? s.plan_w.cut.splits : s.slabs.count;
    s.part_w = s.colpart + align256((size_t)parts * N * 4);
    s.part_x = s.part_w + (s.plan_w.cut.splits > 1 ? align256((size_t)s.plan_w.cut.splits * N * K * 4) : 0);
    s.total = s.part_x + (s.plan_x.cut.splits > 1 ? align256((size_t)s.plan_x.cut.splits * M * K * 4) : 0);
    return s;
}

// The size query and the call that follows it plan the same problem: each thread keeps its last few plans, which
// depend on the descriptor alone.
template <typename S, S (*plan)(const QkLinearDesc&)>
const S& remembered(const QkLinearDesc& d) {
    constexpr int kKept = 8;
    static thread_local struct {
        bool set;
        QkLinearDesc desc;
        S s;
    } kept[kKept];
    static thread_local int next = 0;
    for (auto& k : kept)
        if (k.set && k.desc.rows == d.rows && k.desc.in_features == d.in_features &&
            k.desc.out_features == d.out_features && k.desc.io_dtype == d.io_dtype && k.desc.activation == d.activation &&
            k.desc.flags == d.flags)
            return k.s;
    auto& k = kept[next];
    next = (next + 1) % kKept;
    k.s = plan(d);
    k.desc = d;
    k.set = true;
    return k.s;
}
const ForwardScratch& forward_scratch(const QkLinearDesc& d) { return remembered<ForwardScratch, plan_forward>(d); }
const BackwardScratch& backward_scratch(const QkLinearDesc& d) { return remembered<BackwardScratch, plan_backward>(d); }

// ---- launches ------------------------------------------------------------------
PrepJob prep_job(const void* src, const void* tape, void* dst, float* colpart, int rows, int cols, int act, int io_dtype) {
    PrepJob j{};
    const Slabs s = slabs_of(rows, cols);
    j.src = src, j.tape = tape, j.dst = static_cast<__nv_bfloat16*>(dst), j.colpart = colpart;
    j.rows = rows, j.cols = cols, j.ld = (int)padded(cols), j.act = act;
    j.slab_rows = s.rows, j.cblocks = s.cblocks, j.tx_log2 = s.tx_log2, j.blocks = s.cblocks * s.count;
    j.vec = cols % 8 == 0 && (uintptr_t)src % 16 == 0 && (uintptr_t)tape % 16 == 0;
    return j;
}

cudaError_t launch_prepare(const PrepArgsL& p, int io_dtype, cudaStream_t st) {
    long blocks = 0;
    for (int i = 0; i < p.count; ++i) blocks += p.job[i].blocks;
    if (blocks == 0) return cudaSuccess;
    return launch_after(io_dtype == QK_BF16 ? prepare_kernel<__nv_bfloat16> : prepare_kernel<float>, (unsigned)blocks,
                        kThreads, 0, st, p);
}

cudaError_t launch_reduce(const ReduceArgs& r, cudaStream_t st) {
    long blocks = 0;
    for (int i = 0; i < r.count; ++i) blocks += r.job[i].blocks;
    if (r.gb) blocks += (r.cols + 31) / 32;
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7fffffffl) return cudaErrorInvalidConfiguration;
    return launch_after(reduce_kernel, (unsigned)blocks, kThreads, 0, st, r);
}

void add_reduce(ReduceArgs& r, const float* part, int splits, int rows, int cols, const Epilogue& epi) {
    ReduceJob& j = r.job[r.count++];
    j.part = part, j.splits = splits, j.cols = cols, j.epi = epi;
    j.n = (size_t)rows * cols;
    j.tall = splits > 8 && j.n < 64l * kThreads * kSms;
    j.blocks = (int)(j.tall ? (j.n + 31) / 32 : (j.n + kThreads - 1) / kThreads);
}

// an operand of `rows` x `cols`, packed or as it is
Operand operand(const void* base, int rows, int cols, bool packed, bool mn_major) {
    return {base, cols, rows, packed ? padded(cols) : (long)cols, mn_major};
}

// C (rows, cols) = P Q^T over `depth`, with its epilogue; where the depth is cut, the sums wait in `part` for `red`
cudaError_t set_product(GemmProblem& g, int rows, int cols, int depth, bool two, const Plan& plan, const Operand& p, const Operand& q,
                        float* part, const Epilogue& epi, ReduceArgs& red) {
    g.rows = rows, g.cols = cols;
    g.wrap = blocks_of(depth), g.kblocks = (two ? 2 : 1) * g.wrap, g.kper = plan.cut.kper, g.splits = plan.cut.splits;
    g.tiles_r = (rows + 127) / 128, g.tiles_c = (cols + plan.bn - 1) / plan.bn;
    const long units = (long)g.tiles_r * g.tiles_c * g.splits;
    if (units > 0x3fffffff) return cudaErrorInvalidConfiguration;
    g.units = (int)units;
    g.part = g.splits > 1 ? part : nullptr;
    g.has_bias = epi.bias && !g.part, g.has_residual = epi.residual && !g.part;
    g.bias = g.has_bias ? epi.bias : epi.out, g.residual = g.has_residual ? epi.residual : epi.out;
    g.out = epi.out, g.tape = epi.tape, g.act = epi.act;
    if (!gemm_bind(g, p, q, planes_of(epi.io_dtype), plan.bn)) return cudaErrorInvalidValue;
    if (g.splits > 1) add_reduce(red, part, g.splits, rows, cols, epi);
    return cudaSuccess;
}

// one of the problems of `a` by itself
cudaError_t run_alone(GemmArgs& a, int which, int planes, int bn, cudaStream_t st) {
    if (which) a.g[0] = a.g[1];
    a.first = a.ctas = a.g[0].units < kSms ? a.g[0].units : kSms;
    return launch_gemm(a, planes, bn, st);
}

}  // namespace

QkLinearPlan linear_plan(const QkLinearDesc& d, int product) {
    QkLinearPlan p{};
    const long M = d.rows, K = d.in_features, N = d.out_features;
    p.gz_parts = planes_of(d.io_dtype);
    if (M == 0 || K == 0 || N == 0) return p;
    if (product == 0 ? few_rows(d.rows, d.io_dtype) : few_rows_backward(d.rows, d.io_dtype)) {
        p.path = QK_LINEAR_FEW_ROWS;
        return p;
    }
    if (product == 0 && is_narrow(M, N, K, d.io_dtype)) {
        p.path = QK_LINEAR_SMALL;
        return p;
    }
    p.path = QK_LINEAR_TENSOR;
    Plan plan = {};
    long rows = M;
    if (product == 0) {
        plan = forward_scratch(d).plan;
    } else {
        const BackwardScratch& s = backward_scratch(d);
        plan = product == 1 ? s.plan_w : s.plan_x;
        if (product == 1) rows = N;
        p.paired = s.together, p.sums_bias = s.sums;
        if (s.two) p.gz_parts = 2;
    }
    p.tile_cols = plan.bn, p.slices = plan.cut.splits, p.blocks = plan.cut.kper;
    const long units = Size{rows, product == 0 ? N : K, 0}.tiles(plan.bn) * plan.cut.splits;
    p.units = units < INT32_MAX ? (int)units : INT32_MAX;
    return p;
}

size_t linear_forward_scratch(const QkLinearDesc& d) {
    if (few_rows(d.rows, d.io_dtype) || d.out_features == 0 || d.in_features == 0) return 0;
    return forward_scratch(d).total;
}

size_t linear_backward_scratch(const QkLinearDesc& d) {
    if (d.rows == 0 || d.out_features == 0) return 0;
    return backward_scratch(d).total;
}

cudaError_t launch_linear_forward(const LinearArgs& a, cudaStream_t st) {
    const int M = a.rows, K = a.in, N = a.out;
    const Epilogue epi{a.bias, a.residual, a.y, a.tape, a.act, a.io_dtype};
    ReduceArgs red{};
    if (K == 0) {
        add_reduce(red, nullptr, 0, M, N, epi);
        return launch_reduce(red, st);
    }
    if (few_rows(M, a.io_dtype)) return launch_gemv({M, N, K, a.x, a.w, epi, 0, 0}, st);
    const QkLinearDesc d{M, K, N, a.io_dtype, a.act, 0};
    const ForwardScratch& s = forward_scratch(d);
    char* ws = static_cast<char*>(a.scratch);
    if (is_narrow(M, N, K, a.io_dtype)) {
        float* part = s.narrow.splits > 1 ? reinterpret_cast<float*>(ws) : nullptr;
        const cudaError_t e = launch_narrow({s.narrow, M, N, K, a.x, a.w, part, epi}, st);
        if (e != cudaSuccess || !part) return e;
        add_reduce(red, part, s.narrow.splits, M, N, epi);
        return launch_reduce(red, st);
    }
    const bool pack = !reads_in_place(K, a.io_dtype);
    const void *x = a.x, *w = a.w;
    cudaError_t e = cudaSuccess;
    if (pack) {
        PrepArgsL p{};
        p.job[p.count++] = prep_job(a.x, nullptr, ws + s.x, nullptr, M, K, 0, a.io_dtype);
        p.job[p.count++] = prep_job(a.w, nullptr, ws + s.w, nullptr, N, K, 0, a.io_dtype);
        e = launch_prepare(p, a.io_dtype, st);
        if (e != cudaSuccess) return e;
        x = ws + s.x, w = ws + s.w;
    }
    GemmArgs g{};
    e = set_product(g.g[0], M, N, K, false, s.plan, operand(x, M, K, pack, false), operand(w, N, K, pack, false),
                    reinterpret_cast<float*>(ws + s.part), epi, red);
    if (e == cudaSuccess) e = run_alone(g, 0, planes_of(a.io_dtype), s.plan.bn, st);
    return e == cudaSuccess ? launch_reduce(red, st) : e;
}

cudaError_t launch_linear_backward(const LinearArgs& a, cudaStream_t st) {
    const int M = a.rows, K = a.in, N = a.out;
    const QkLinearDesc d{M, K, N, a.io_dtype, a.act, a.flags};
    const BackwardScratch& s = backward_scratch(d);
    char* ws = static_cast<char*>(a.scratch);
    ReduceArgs red{};
    if (s.few.slab) {
        float* part = a.gx ? reinterpret_cast<float*>(ws) : nullptr;
        cudaError_t e = launch_few_backward({M, K, N, a.act, a.io_dtype, a.x, a.w, a.gy, a.act == QK_ACT_NONE ? nullptr : a.tape,
                                             part, a.gw, a.gb, s.few.blocks, s.few.slab}, st);
        if (e != cudaSuccess) return e;
        if (a.gx) add_reduce(red, part, s.few.slabs, M, K, {nullptr, nullptr, a.gx, nullptr, QK_ACT_NONE, a.io_dtype});
        return launch_reduce(red, st);
    }
    const bool pack = !reads_in_place(K, a.io_dtype);
    const bool pack_gz = (a.gx || a.gw) && (a.act != QK_ACT_NONE || !reads_in_place(N, a.io_dtype));
    float* colpart = a.gb ? reinterpret_cast<float*>(ws + s.colpart) : nullptr;
    const bool sums = a.gb && a.gw && s.sums;
    PrepArgsL p{};
    if (pack_gz || (a.gb && !sums))
        p.job[p.count++] = prep_job(a.gy, a.act == QK_ACT_NONE ? nullptr : a.tape, pack_gz ? ws + s.gz : nullptr, colpart, M,
                                    N, a.act, a.io_dtype);
    if (p.count) p.job[0].two = s.two;
    if (pack && a.gw) p.job[p.count++] = prep_job(a.x, nullptr, ws + s.x, nullptr, M, K, 0, a.io_dtype);
    if (pack && a.gx) p.job[p.count++] = prep_job(a.w, nullptr, ws + s.w, nullptr, N, K, 0, a.io_dtype);
    cudaError_t e = launch_prepare(p, a.io_dtype, st);
    if (e != cudaSuccess) return e;
    const void* gz = pack_gz ? ws + s.gz : a.gy;
    GemmArgs g{};
    const int planes = planes_of(a.io_dtype);
    if (a.gw)
        e = set_product(g.g[0], N, K, M, s.two, s.plan_w, operand(gz, M, N, pack_gz, true), operand(pack ? ws + s.x : a.x, M, K, pack, true),
                        reinterpret_cast<float*>(ws + s.part_w), {nullptr, nullptr, a.gw, nullptr, QK_ACT_NONE, a.io_dtype}, red);
    if (sums) g.g[0].row_sums = colpart;
    if (e == cudaSuccess && a.gx)
        e = set_product(g.g[1], M, K, N, s.two, s.plan_x, operand(gz, M, N, pack_gz, false), operand(pack ? ws + s.w : a.w, N, K, pack, true),
                        reinterpret_cast<float*>(ws + s.part_x), {nullptr, nullptr, a.gx, nullptr, QK_ACT_NONE, a.io_dtype}, red);
    if (e == cudaSuccess && a.gw && a.gx && s.together) {
        g.first = g.g[0].units, g.ctas = g.first + g.g[1].units;
        e = launch_gemm(g, planes, s.plan_w.bn, st);
    } else {
        if (e == cudaSuccess && a.gw) e = run_alone(g, 0, planes, s.plan_w.bn, st);
        if (e == cudaSuccess && a.gx) e = run_alone(g, 1, planes, s.plan_x.bn, st);
    }
    if (e != cudaSuccess) return e;
    red.colpart = colpart, red.gb = a.gb, red.slabs = sums ? s.plan_w.cut.splits : s.slabs.count, red.cols = N, red.io_dtype = a.io_dtype;
    return launch_reduce(red, st);
}

}  // namespace qk
