// Grouped and block-scaled products (grouped.cuh) on the tensor cores: tcgen05.mma kind::f16 / kind::f8f6f4 fed by TMA.
//
// Orientation.  Weights stand on the M side of the MMA (128 of their rows per CTA), the rows of a group on the N side, 16 to kTN of them:
// a group pads its last tile to 16 rows instead of 128, its weights are read once for as many rows as fit (few rows: bound by the
// weights' bytes; many: by the tensor pipe), and 128 weight rows share one scale per block of K.
//
// Tiles of 256 rows run on CTA pairs (cta_group::2, 256 weight rows, each CTA loads 128 of them and half of the group's rows): a CTA
// alone would need 48 KiB per block of K, a pair needs 32, and 148 SMs that take 48 KiB every 512 cycles are more than L2 delivers.
//
// Roles: warp 0 loads (TMA), warp 1 issues MMAs, warp 2 fetches the scales, warps 4-11 (4-7 for short tiles) take the accumulators: a warp
// owns 32 TMEM lanes (weight rows) and, where there are eight, every other chunk of columns (rows of the group).  CTAs are persistent; a
// work item = (group, rows tile, weight rows) is found by a search in the groups' running item counts, which every CTA builds from the
// offsets.
//
// Scales.  The accumulator of a block of 128 k leaves tensor memory by itself (two to four buffers take turns) and is added to fp32
// registers with the product of its scales.  Tensor memory is read as 16 lanes x 128 bits, so that a thread holds every fourth column and
// needs a fourth of the scales: one 16-byte read of shared memory serves 16 FMAs.  Measured alone, cycles per 128 x 256 accumulator,
// loads and FMAs of 8 warps: 16 x 128 bits 494, 16 x 256 bits 659 (its loads alone 377, against 269), 32 x 32 bits with every column's
// scale read by every thread 589; the MMAs of a block take 512.
//
// Scaled products of tall tiles stand the other way round: rows on the M side, 256 weight rows on the N side.  A lane then holds a row
// and a warp the columns of one scale, so that an accumulator element costs one FMA with a scalar of the thread (327 cycles per 128 x 256)
// and rows are stored straight from registers; a group's last tile is padded to 256 rows instead of 32.  Measured in the kernel, cycles
// per block of K: weights on the M side 1170, of which the sums 760; rows on the M side 860, of which the MMAs 512.
//
// What bounds tall scaled tiles (4096 x 11008 x 4096, 171 us in short runs; each part taken out in turn): copies alone 84 us, with the MMAs
// and the exchange of buffers 121, with the loads from tensor memory 134, with the FMAs 148; the rest is a tile's results, in which the
// MMAs stand still but for the two blocks that tensor memory holds.  In runs of seconds the board's power cap takes the clock to 1.4 GHz.
//
// Few items: clusters of two or four CTAs cut K, exchange their partial sums through distributed shared memory and add them in rank order.
#pragma once

#include "grouped.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace kb {

namespace grp {

constexpr int kControlThreads = 128;
constexpr int kTileN = 128;             // weight rows per CTA
constexpr int kWeightBytes = kTileN * 128;
constexpr int kMaxStages = 12;
constexpr int kMaxBuffers = 4;
constexpr int kScaleSlots = 8;
constexpr int kUnitPitch = 40;          // floats between the columns of a staged unit of 16 columns x 32 rows: conflict-free both ways
constexpr int kUnitBytes = 16 * kUnitPitch * 4;
constexpr int kSmemLimit = 232448;      // of one CTA
constexpr int kSmemPerSm = 233472;
// registers per thread where a warp's sums take 128 of them: 4 control warps and 8 that sum share what the launch has, 168 each
constexpr int kControlRegs = 88, kSumRegs = 208;
static_assert(128 * kControlRegs + 256 * kSumRegs <= 384 * 168, "register split");
constexpr int kBarrierBytes = (2 * kMaxStages + 2 * kMaxBuffers + 2 * kScaleSlots) * 8 + 16;

// How the blocks of K add up: in tensor memory; in fp32 registers with their scales (e4m3); or there without, p.drain blocks at a time, for
// fp32 results of 16-bit operands.  The tensor cores cut every addition, always towards zero: 3000 x 1024 x 8192 is 1.0e-5 off in the
// norm when all of it stays in tensor memory, and 16-bit results do not see that, but fp32 ones do.
constexpr int kPlain = 0, kWithScales = 1, kDrained = 2;

// kRows: the rows of the group on the M side (see above)
template <int kMode, int kTN, bool kRows>
struct Shape {
    static constexpr bool kScaled = kMode == kWithScales, kSums = kMode != kPlain;
    static_assert(!kRows || (kScaled && kTN == 256), "rows on the M side: scaled products of tall tiles");
    static constexpr bool kPair = kTN == 256;
    // Short tiles are bound by the weights' bytes: small CTAs, of which two or three share an SM, keep many copies in flight and even out
    // the SMs' shares.
    static constexpr int kCtas = kTN == 32 ? 3 : kTN == 64 ? 2 : 1;
    static constexpr int kSumWarps = kTN <= 64 ? 4 : 8;
    static constexpr int kWays = kSumWarps / 4;               // warps that share a quarter of the lanes: they take chunks in turn
    static constexpr int kThreads = kControlThreads + 32 * kSumWarps;
    static constexpr int kBuffers = kSums && kTN != 256 ? 4 : 2;
    static constexpr int kTmemCols = kBuffers * kTN;
    static constexpr int kChunk = kTN >= 64 ? 32 : 16;        // columns a warp takes at a time
    static constexpr int kChunks = kTN / kChunk / kWays;      // per warp
    static constexpr int kRound = kPair ? 32 : 16;            // N of an MMA is a multiple of this
    static constexpr int kLoadRows = kPair ? kTN / 2 : kTN;   // rows of a that one CTA loads, at most
    static constexpr int kBoxRows = kTN >= 128 ? 64 : kTN / 2;  // of them in one copy
    static constexpr int kStageBytes = kWeightBytes + kLoadRows * 128;
    // Whether launches may cut K.  Not tiles of 64 rows: where they cost less than those of 32, they are more than half of the SMs.
    static constexpr bool kSplits = kTN == 32;
    static constexpr int kUnits = kTN / 16 * 4;               // of a whole tile; partial sums lie where the ring was
    static constexpr int kLeastStages = kTN == 32 ? 2 : 3;
    static_assert(!kSplits || (kUnits + kSumWarps) * kUnitBytes <= kLeastStages * kStageBytes, "room for the partial sums");
    static constexpr int kScaleBytes = kScaled && !kRows ? kScaleSlots * kTN * 4 : 0;
    static constexpr int kBiasBytes = kSumWarps * (kRows ? 512 : 128);
    static constexpr int kFixedBytes = kSumWarps * kUnitBytes + kBiasBytes + kScaleBytes + kBarrierBytes;
};

struct TcParams {
    GroupedParams g;
    int num_kb;        // blocks of 128 bytes of K
    int kb_elems;      // elements in one
    int tiles_n;       // of 128 weight rows, 256 for pairs
    int splits, kb_per_split;
    int drain;         // kDrained: blocks of K that add up in tensor memory
    int stages;
    int band;          // row tiles that share the weight tiles of a raster band
    int vec;           // 1: rows of c are contiguous, four of their elements aligned, and finish_unit knows the activation; 2: 32-byte aligned too
    unsigned idesc;    // without N
    int load_kb;       // k-blocks from this one on are not loaded (test hook)
    DeviceStatus *status;
    long long wait_limit;
};

struct Item {
    int group, row0, count, cols, n0;  // cols: N of the MMAs; count rounded up to what they take, or 256 weight rows
};

template <int kTN, bool kRows>
__device__ __forceinline__ Item find_item(const TcParams &p, const int *begins, const int *items, int item)
{
    int lo = 0, hi = p.g.groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (items[mid] <= item) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    constexpr int kRound = kTN == 256 ? 32 : 16, kWide = kTN == 256 ? 2 * kTileN : kTileN;
    const int local = item - items[lo], begin = begins[lo], rows = begins[lo + 1] - begin;
    Item w;
    w.group = lo;
    int tall;  // rows of a tile: the group cut evenly, or what the M side holds
    if (rows <= kTN) {
        tall = rows;
        w.n0 = local * kWide;
        w.row0 = begin;
    } else {
        const int tiles = (rows + kTN - 1) / kTN;
        tall = kRows ? kTN : ((rows + tiles - 1) / tiles + kRound - 1) / kRound * kRound;
        const int per_band = p.band * p.tiles_n, band = local / per_band, in_band = local - band * per_band;
        const int first = band * p.band, wide = tiles - first < p.band ? tiles - first : p.band;
        const int column = in_band / wide;
        w.n0 = column * kWide;
        w.row0 = begin + (first + in_band - column * wide) * tall;
    }
    const int left = begin + rows - w.row0;
    w.count = left < tall ? left : tall;
    w.cols = kRows ? 256 : (w.count + kRound - 1) / kRound * kRound;
    return w;
}

template <bool kPair>
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    if (kPair) {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
            "}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
            "}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

// Tile load of one CTA of a pair into its own shared memory, counted on the leader's barrier (a cluster address).
__device__ __forceinline__ void tma_load_3d_pair(void *smem_dst, const CUtensorMap *tmap, uint32_t leader_bar, int x, int y, int z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(smem_dst)),
        "l"(tmap), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// 16 lanes x 32 columns: register 2j + h holds lane (thread / 4) + 8h, column 4j + thread % 4
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.16x128b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// the same, 16 columns
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.16x128b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8])
{
    tmem_load_wait(r);
}

__device__ __forceinline__ void load_shared_4(uint32_t at, float *v)
{
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at));
}
__device__ __forceinline__ void store_shared(uint32_t at, float v)
{
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

// Whether a phase has ended, without waiting (mbarrier.try_wait may hold the thread for microseconds)
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// A wait of a whole warp, which gets one answer.  The first look is apart from the bounded loop: an arrival that is there already, the
// usual case, costs one round trip to shared memory, and several looks that are asked for together cost one.
__device__ __forceinline__ bool warp_wait(bool there, uint64_t *bar, uint32_t parity, volatile int *abort_flag, DeviceStatus *status, int where,
                                          long long limit)
{
    if (__all_sync(0xffffffffu, there)) {
        return true;
    }
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, where, limit));
}

__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(p));
    return p != 0u;
}

__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

template <int kAct, bool kPrecise>
__device__ __forceinline__ void activate(float (&v)[4][4], float alpha)
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float &x = v[i / 4][i % 4];
        x = kAct == KUDNN_B200_ACT_GELU_TANH && !kPrecise ? gelu_tanh_sigmoid(x) : activation<kPrecise>(x, kAct, alpha);
    }
}

// A staged unit: 16 rows of c x 32 neighbouring columns, the rows kUnitPitch floats apart.  finish_unit takes it where the columns are
// inside of c, aligned and contiguous and the activation is a short one: a lane takes 4 columns of every fourth row, straight
// through.  finish_unit_any takes the rest, element by element.  The epilogues of a tile are one loop over its units with one copy of this
// code: unrolled, with the cases inside, a tile of 128 x 256 took 27 thousand cycles to finish.
__device__ __forceinline__ void finish_unit(const GroupedParams &g, int row0, int count, int n, const float (&bias)[4], float (&v)[4][4], int lane)
{
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        v[i / 4][i % 4] += bias[i % 4];
    }
    const bool precise = g.c_dtype == KUDNN_B200_F32;
    if (g.act != KUDNN_B200_ACT_NONE) {
        if (g.act == KUDNN_B200_ACT_RELU) {
            activate<KUDNN_B200_ACT_RELU, true>(v, g.act_alpha);
        } else if (g.act == KUDNN_B200_ACT_GELU_TANH) {
            activate<KUDNN_B200_ACT_GELU_TANH, false>(v, g.act_alpha);
        } else if (precise) {
            activate<KUDNN_B200_ACT_SWISH, true>(v, g.act_alpha);
        } else {
            activate<KUDNN_B200_ACT_SWISH, false>(v, g.act_alpha);
        }
    }
    const int first = lane / 8;
    char *to = static_cast<char *>(g.c) + ((row0 + first) * g.c_sm + n) * (precise ? 4 : 2);
    const long long step = 4 * g.c_sm * (precise ? 4 : 2);
    if (precise) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (first + 4 * i < count) {
                *reinterpret_cast<float4 *>(to + i * step) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
            }
        }
        return;
    }
    uint2 w[4];
    if (g.c_dtype == KUDNN_B200_F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 lo = __floats2half2_rn(v[i][0], v[i][1]), hi = __floats2half2_rn(v[i][2], v[i][3]);
            w[i] = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v[i][0], v[i][1]), hi = __floats2bfloat162_rn(v[i][2], v[i][3]);
            w[i] = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (first + 4 * i < count) {
            *reinterpret_cast<uint2 *>(to + i * step) = w[i];
        }
    }
}

// bias_at: 32 floats of shared memory.  A lane takes a column, so that the 32 of a row are stored side by side however c is aligned.
static __device__ __noinline__ void finish_unit_any(const GroupedParams &g, int row0, int count, int n0, uint32_t bias_at, uint32_t unit_at, int lane)
{
    if (n0 + lane >= g.n) {
        return;
    }
    float bias, v[4][4];
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(bias) : "r"(bias_at + static_cast<uint32_t>(lane * 4)));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[r / 4][r % 4]) : "r"(unit_at + static_cast<uint32_t>((r * kUnitPitch + lane) * 4)));
        v[r / 4][r % 4] += bias;
    }
    const bool precise = g.c_dtype == KUDNN_B200_F32;
    if (g.act == KUDNN_B200_ACT_RELU) {
        activate<KUDNN_B200_ACT_RELU, true>(v, g.act_alpha);
    } else if (g.act == KUDNN_B200_ACT_SWISH && !precise) {
        activate<KUDNN_B200_ACT_SWISH, false>(v, g.act_alpha);
    } else if (g.act == KUDNN_B200_ACT_GELU_TANH && !precise) {
        activate<KUDNN_B200_ACT_GELU_TANH, false>(v, g.act_alpha);
    } else if (g.act != KUDNN_B200_ACT_NONE) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            v[r / 4][r % 4] = activation_any(v[r / 4][r % 4], g.act, g.act_alpha, precise ? 1 : 0);
        }
    }
    const long long at = row0 * g.c_sm + (n0 + lane) * g.c_sn;
    if (precise) {
        float *to = static_cast<float *>(g.c) + at;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (r < count) {
                to[r * g.c_sm] = v[r / 4][r % 4];
            }
        }
    } else {
        unsigned short *to = static_cast<unsigned short *>(g.c) + at;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (r < count) {
                to[r * g.c_sm] = g.c_dtype == KUDNN_B200_F16 ? f32_to_f16_rne_bits(v[r / 4][r % 4]) : f32_to_bf16_rne_bits(v[r / 4][r % 4]);
            }
        }
    }
}

// ---- rows on the M side: a lane holds a row, and its 128 columns of a warp share one scale

template <int kAct, bool kPrecise>
__device__ __forceinline__ void activate_32(float *v, float alpha)
{
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        v[i] = kAct == KUDNN_B200_ACT_GELU_TANH && !kPrecise ? gelu_tanh_sigmoid(v[i]) : activation<kPrecise>(v[i], kAct, alpha);
    }
}

__device__ __forceinline__ void tmem_load_32x16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ void store_32_bytes(void *to, const uint32_t *w, int vec)
{
    if (vec == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            reinterpret_cast<uint2 *>(to)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
        }
        return;
    }
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// The scale of this lane's row times that of the warp's 128 weight rows, for one block of K; 0 where there is no such row or column.
struct ScaleSource {
    const float *row, *weights;
    bool inside;
};
__device__ __forceinline__ ScaleSource scale_source(const GroupedParams &g, const Item &w, int row_in_tile, int n)
{
    ScaleSource s;
    s.inside = row_in_tile < w.count && n < g.n;
    s.row = g.a_scale + (s.inside ? (w.row0 + row_in_tile) * g.as_sm : 0);
    s.weights = g.b_scale + w.group * g.bs_sg + (s.inside ? n / kScaleBlock * g.bs_sn : 0);
    return s;
}

__device__ __forceinline__ void sum_rows(const TcParams &p, const int *begins, const int *items, int num_items, int first_item, int stride, int rank,
                                         int warp, int lane, uint32_t tmem_base, uint64_t *tmem_full, uint64_t *tmem_empty, uint32_t units_at,
                                         uint32_t bias_at, volatile int *abort_flag)
{
    constexpr int kBuffers = Shape<kWithScales, 256, true>::kBuffers;
    const GroupedParams &g = p.g;
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int row_in_tile = rank * 128 + quarter * 32 + lane;
    const uint32_t my_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(half * 128);
    const uint32_t drained = map_to_rank(smem_u32(tmem_empty), 0u);
    const uint32_t my_unit = units_at + static_cast<uint32_t>((warp - 4) * kUnitBytes);
    const uint32_t my_bias = bias_at + static_cast<uint32_t>((warp - 4) * 512);  // 128 floats
    int buffer = 0;
    uint32_t phase = 0;
    Item w;
    ScaleSource s;
    float row_next = 0.0f, weights_next = 0.0f, row_after = 0.0f, weights_after = 0.0f;  // of the next two blocks
    auto begin_item = [&](int item) {
        w = find_item<256, true>(p, begins, items, item);
        s = scale_source(g, w, row_in_tile, w.n0 + half * 128);
        if (s.inside) {
            row_next = s.row[0];
            weights_next = s.weights[0];
            if (p.num_kb > 1) {
                row_after = s.row[g.as_sk];
                weights_after = s.weights[g.bs_sk];
            }
        } else {
            row_next = weights_next = row_after = weights_after = 0.0f;
        }
    };
    if (first_item < num_items) {
        begin_item(first_item);
    }
    for (int item = first_item; item < num_items; item += stride) {
        const Item mine = w;
        const int n_half = mine.n0 + half * 128;
        float bias[4] = {};
        if (g.has_bias != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = n_half + i * 32 + lane;
                bias[i] = n < g.n ? load_as_f32(g.bias, g.bias_dtype, mine.group * g.bias_sg + n * g.bias_sn) : 0.0f;
            }
        }
        float sum[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) {
            sum[j] = 0.0f;
        }
        bool alive = true;
#pragma unroll 1
        for (int kb = 0; kb < p.num_kb; ++kb) {
            const float scale = row_next * weights_next;
            row_next = row_after;
            weights_next = weights_after;
            if (kb + 2 < p.num_kb && s.inside) {
                row_after = s.row[(kb + 2) * g.as_sk];
                weights_after = s.weights[(kb + 2) * g.bs_sk];
            }
            alive = warp_wait(mbar_test(tmem_full + buffer, phase), tmem_full + buffer, phase, abort_flag, p.status, 4, p.wait_limit);
            if (!alive) {
                break;
            }
            tc_fence_after();
            const uint32_t from = my_tmem + static_cast<uint32_t>(buffer * 256);
            uint32_t part[2][16];  // one load ahead of the FMAs
            tmem_load_32x16(from, part[0]);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                tmem_wait(part[c & 1]);
                if (c < 7) {
                    tmem_load_32x16(from + static_cast<uint32_t>((c + 1) * 16), part[(c + 1) & 1]);
                } else {  // everything is in registers: the MMAs may have the buffer again
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_cluster(drained + static_cast<uint32_t>(buffer * 8));
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    sum[c * 16 + j] = fmaf(__uint_as_float(part[c & 1][j]), scale, sum[c * 16 + j]);
                }
            }
            if (++buffer == kBuffers) {
                buffer = 0;
                phase ^= 1u;
            }
        }
        if (!alive) {
            return;
        }
        if (item + stride < num_items) {
            begin_item(item + stride);  // the next item's first scales are on their way while this one is finished
        }
        if (g.has_bias != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                store_shared(my_bias + static_cast<uint32_t>((i * 32 + lane) * 4), bias[i]);
            }
            __syncwarp();
        }
        const int row = mine.row0 + row_in_tile;
        const bool precise = g.c_dtype == KUDNN_B200_F32;
#pragma unroll 1
        for (int c0 = 0; c0 < 128 && n_half + c0 < g.n; c0 += 32) {
            if (p.vec != 0 && n_half + c0 + 32 <= g.n) {
                if (g.has_bias != 0) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        float b[4];
                        load_shared_4(my_bias + static_cast<uint32_t>((c0 + j) * 4), b);
                        sum[j] += b[0];
                        sum[j + 1] += b[1];
                        sum[j + 2] += b[2];
                        sum[j + 3] += b[3];
                    }
                }
                if (g.act != KUDNN_B200_ACT_NONE) {
                    if (g.act == KUDNN_B200_ACT_RELU) {
                        activate_32<KUDNN_B200_ACT_RELU, true>(sum, g.act_alpha);
                    } else if (g.act == KUDNN_B200_ACT_GELU_TANH) {
                        activate_32<KUDNN_B200_ACT_GELU_TANH, false>(sum, g.act_alpha);
                    } else if (precise) {
                        activate_32<KUDNN_B200_ACT_SWISH, true>(sum, g.act_alpha);
                    } else {
                        activate_32<KUDNN_B200_ACT_SWISH, false>(sum, g.act_alpha);
                    }
                }
                if (row_in_tile < mine.count) {
                    char *to = static_cast<char *>(g.c) + (row * g.c_sm + n_half + c0) * (precise ? 4 : 2);
                    if (precise) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t v[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                v[j] = __float_as_uint(sum[i * 8 + j]);
                            }
                            store_32_bytes(to + i * 32, v, p.vec);
                        }
                    } else {
                        uint32_t v[16];
                        if (g.c_dtype == KUDNN_B200_F16) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const __half2 h = __floats2half2_rn(sum[2 * j], sum[2 * j + 1]);
                                v[j] = *reinterpret_cast<const uint32_t *>(&h);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const __nv_bfloat162 h = __floats2bfloat162_rn(sum[2 * j], sum[2 * j + 1]);
                                v[j] = *reinterpret_cast<const uint32_t *>(&h);
                            }
                        }
                        store_32_bytes(to, v, p.vec);
                        store_32_bytes(to + 32, v + 8, p.vec);
                    }
                }
            } else {
                if (g.has_bias == 0) {
                    store_shared(my_bias + static_cast<uint32_t>((c0 + lane) * 4), 0.0f);
                }
                // 16 rows at a time through shared memory
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    __syncwarp();
                    if (lane / 16 == part) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            store_shared(my_unit + static_cast<uint32_t>(((lane & 15) * kUnitPitch + j) * 4), sum[j]);
                        }
                    }
                    __syncwarp();
                    const int first = rank * 128 + quarter * 32 + part * 16;
                    finish_unit_any(g, mine.row0 + first, mine.count - first, n_half + c0, my_bias + static_cast<uint32_t>(c0 * 4), my_unit, lane);
                }
            }
#pragma unroll
            for (int j = 0; j < 96; ++j) {
                sum[j] = sum[j + 32];
            }
        }
        __syncwarp();
    }
}

template <int kMode, int kTN, bool kRows>
__global__ void __launch_bounds__(Shape<kMode, kTN, kRows>::kThreads, Shape<kMode, kTN, kRows>::kCtas)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ TcParams p)
{
    using S = Shape<kMode, kTN, kRows>;
    constexpr bool kScaled = S::kScaled, kSums = S::kSums;
    extern __shared__ __align__(1024) unsigned char smem[];
    constexpr int kThreads = S::kThreads, kSumWarps = S::kSumWarps;
    unsigned char *behind_ring = smem + p.stages * S::kStageBytes;
    unsigned char *units = S::kSplits && p.splits > 1 ? smem : behind_ring;  // staged results; partial sums lie where the ring was
    unsigned char *bias_area = behind_ring + kSumWarps * kUnitBytes;
    unsigned char *scales = bias_area + S::kBiasBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(scales + S::kScaleBytes);
    uint64_t *full_bar = bars;
    uint64_t *empty_bar = full_bar + kMaxStages;
    uint64_t *tmem_full = empty_bar + kMaxStages;
    uint64_t *tmem_empty = tmem_full + kMaxBuffers;
    uint64_t *scale_full = tmem_empty + kMaxBuffers;
    uint64_t *scale_empty = scale_full + kScaleSlots;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(scale_empty + kScaleSlots);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    int *begins = reinterpret_cast<int *>(tmem_slot + 4);  // first row of each group, then the end of the last
    int *items = begins + p.g.groups + 1;                  // work items before each group, then all

    // (from a shuffle, so that the compiler knows it to be the same in all lanes and keeps the roles' addresses in uniform registers)
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    if ((smem_u32(smem) & 1023u) != 0) {  // never: the declaration asks for the alignment
        if (threadIdx.x == 0) {
            atomicCAS(&p.status->code, kErrNone, kErrTimeout);
        }
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) {
            mbar_init(full_bar + s, 1);
            mbar_init(empty_bar + s, 1);
        }
        for (int s = 0; s < kMaxBuffers; ++s) {
            mbar_init(tmem_full + s, 1);
            mbar_init(tmem_empty + s, S::kPair ? 2 * kSumWarps : kSumWarps);  // pair: the sums of both CTAs
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            mbar_init(scale_full + s, 1);
            mbar_init(scale_empty + s, kSumWarps);
        }
        *abort_flag = 0;
        if (p.g.offsets == nullptr) {
            begins[0] = items[0] = 0;
            begins[1] = p.g.rows;
            items[1] = (p.g.rows + kTN - 1) / kTN * p.tiles_n;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if (S::kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(S::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(S::kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    if (warp == 0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_b) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (S::kPair) {
        cluster_barrier();  // the peer's barriers are initialised before anything is signalled on them
    }
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();  // only now that this CTA holds its tensor memory
    pdl_wait();

    // ---- the groups: offsets made to ascend, and the items before each group (without offsets thread 0 has written them above)
    if (p.g.offsets != nullptr) {
        for (int i = threadIdx.x; i <= p.g.groups; i += kThreads) {
            begins[i] = group_offset(p.g, i);
        }
        __syncthreads();
        if (warp == 0) {
            int most = 0;
            for (int i0 = 0; i0 <= p.g.groups; i0 += 32) {
                int v = i0 + lane <= p.g.groups ? begins[i0 + lane] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int before = __shfl_up_sync(0xffffffffu, v, o);
                    v = lane >= o && before > v ? before : v;
                }
                v = v > most ? v : most;
                if (i0 + lane <= p.g.groups) {
                    begins[i0 + lane] = v;
                }
                most = __shfl_sync(0xffffffffu, v, 31);
            }
            __syncwarp();
            int all = 0;
            for (int i0 = 0; i0 < p.g.groups; i0 += 32) {
                int v = 0;
                if (i0 + lane < p.g.groups) {
                    v = (begins[i0 + lane + 1] - begins[i0 + lane] + kTN - 1) / kTN * p.tiles_n;
                }
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int before = __shfl_up_sync(0xffffffffu, v, o);
                    v += lane >= o ? before : 0;
                }
                if (i0 + lane < p.g.groups) {
                    items[i0 + lane + 1] = all + v;
                }
                all += __shfl_sync(0xffffffffu, v, 31);
            }
            if (lane == 0) {
                items[0] = 0;
            }
        }
        __syncthreads();
    }
    const int num_items = items[p.g.groups];
    const int rank = S::kPair || p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
    // launches that cut K have a cluster for every item that there can be
    const int first_item = S::kPair ? static_cast<int>(blockIdx.x >> 1) : p.splits > 1 ? static_cast<int>(blockIdx.x) / p.splits : static_cast<int>(blockIdx.x);
    const int stride = S::kPair ? static_cast<int>(gridDim.x >> 1) : p.splits > 1 ? num_items + 1 : static_cast<int>(gridDim.x);
    const int kb_begin = S::kPair ? 0 : rank * p.kb_per_split;
    const int kb_end = kb_begin + p.kb_per_split < p.num_kb ? kb_begin + p.kb_per_split : p.num_kb;
    const int my_n = S::kPair ? rank * kTileN : 0;  // of a pair's 256 weight rows, the CTA's begin here

    // rows that no group holds
    const int outside_first = begins[0], outside = p.g.rows - (begins[p.g.groups] - begins[0]);
    if (outside > 0) {
        const long long count = static_cast<long long>(outside) * p.g.n;
        for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < count; i += static_cast<long long>(gridDim.x) * kThreads) {
            const int r = static_cast<int>(i / p.g.n), n = static_cast<int>(i % p.g.n);
            store_exact(p.g.c, p.g.c_dtype, (r < outside_first ? r : r + p.g.rows - outside) * p.g.c_sm + n * p.g.c_sn, 0.0f);
        }
    }

    if (warp < 4) {
        if (kSums && kTN == 256) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        }
        // The whole warp runs a role's loop and one lane issues: what an instruction needs then lies in uniform registers.
        if (warp == 0) {
            // ------------------------------------------------------------------ loads
            int stage = 0;
            uint32_t phase = 0;
            bool alive = true;
            for (int item = first_item; alive && item < num_items; item += stride) {
                const Item w = find_item<kTN, kRows>(p, begins, items, item);
                const int mine = S::kPair ? w.cols / 2 : w.cols, row0 = w.row0 + (S::kPair ? rank * mine : 0);
                const int boxes = (mine + S::kBoxRows - 1) / S::kBoxRows;
                const uint32_t bytes = static_cast<uint32_t>(kWeightBytes + boxes * S::kBoxRows * 128) * (S::kPair ? 2u : 1u);
                const int end = kb_end < p.load_kb ? kb_end : p.load_kb;
                for (int kb = kb_begin; kb < end; ++kb) {
                    alive = warp_wait(mbar_test(empty_bar + stage, phase ^ 1u), empty_bar + stage, phase ^ 1u, abort_flag, p.status, 1, p.wait_limit);
                    if (!alive) {
                        break;
                    }
                    unsigned char *at = smem + stage * S::kStageBytes;
                    const int x = kb * p.kb_elems;
                    if (elect_one()) {
                        if (S::kPair) {
                            // the leader's barriers count both CTAs' bytes; only the leader announces them
                            const uint32_t bar = map_to_rank(smem_u32(full_bar + stage), 0u);
                            if (rank == 0) {
                                mbar_expect_tx(full_bar + stage, bytes);
                            }
                            tma_load_3d_pair(at, &tmap_b, bar, x, w.n0 + my_n, w.group);
                            for (int i = 0; i < boxes; ++i) {
                                tma_load_3d_pair(at + kWeightBytes + i * S::kBoxRows * 128, &tmap_a, bar, x, row0 + i * S::kBoxRows, 0);
                            }
                        } else {
                            mbar_expect_tx(full_bar + stage, bytes);
                            tma_load_3d(at, &tmap_b, full_bar + stage, x, w.n0, w.group);
                            for (int i = 0; i < boxes; ++i) {
                                tma_load_3d(at + kWeightBytes + i * S::kBoxRows * 128, &tmap_a, full_bar + stage, x, row0 + i * S::kBoxRows, 0);
                            }
                        }
                    }
                    __syncwarp();
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        } else if (warp == 1 && (!S::kPair || rank == 0)) {
            // ------------------------------------------------------------------ MMAs, of a pair by its leader
            int stage = 0, buffer = 0;
            uint32_t phase = 0, buffer_phase = 0;
            bool alive = true;
            bool loaded = mbar_test(full_bar, 0);  // looked up one k-block ahead, so that the answer is there when it is needed
            for (int item = first_item; alive && item < num_items; item += stride) {
                const Item w = find_item<kTN, kRows>(p, begins, items, item);
                const uint32_t idesc = p.idesc | (kRows ? 0u : static_cast<uint32_t>(w.cols >> 3) << 17);
                int held = 0;  // blocks that the buffer has added up
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    if (held == 0) {
                        alive = warp_wait(mbar_test(tmem_empty + buffer, buffer_phase ^ 1u), tmem_empty + buffer, buffer_phase ^ 1u, abort_flag,
                                          p.status, 2, p.wait_limit);
                    }
                    alive = alive && warp_wait(loaded, full_bar + stage, phase, abort_flag, p.status, 3, p.wait_limit);
                    if (!alive) {
                        break;
                    }
                    tc_fence_after();
                    const uint32_t at = smem_u32(smem) + static_cast<uint32_t>(stage * S::kStageBytes);
                    const uint64_t first = make_smem_desc(at), second = make_smem_desc(at + kWeightBytes);
                    const uint64_t mdesc = kRows ? second : first, ndesc = kRows ? first : second;
                    const uint32_t to = tmem_base + static_cast<uint32_t>(buffer * kTN);
                    const bool whole = kScaled || kb + 1 == kb_end || (kSums && held + 1 == p.drain);  // the buffer is complete
                    const int this_stage = stage;
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    loaded = mbar_test(full_bar + stage, phase);
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const uint64_t d = static_cast<uint64_t>(2 * ks);
                            const uint32_t more = ks != 0 || held != 0 ? 1u : 0u;
                            if (kScaled) {
                                umma_f8<S::kPair>(to, mdesc + d, ndesc + d, idesc, more);
                            } else if (S::kPair) {
                                umma_pair<KUDNN_B200_F16>(to, mdesc + d, ndesc + d, idesc, more);
                            } else {
                                umma<KUDNN_B200_F16>(to, mdesc + d, ndesc + d, idesc, more);
                            }
                        }
                        if (S::kPair) {
                            if (whole) {
                                umma_commit_pair(tmem_full + buffer);
                            }
                            umma_commit_pair(empty_bar + this_stage);
                        } else {
                            if (whole) {
                                umma_commit(tmem_full + buffer);
                            }
                            umma_commit(empty_bar + this_stage);
                        }
                    }
                    __syncwarp();
                    held = whole ? 0 : held + 1;
                    if (whole && ++buffer == S::kBuffers) {
                        buffer = 0;
                        buffer_phase ^= 1u;
                    }
                }
            }
        } else if (kScaled && !kRows && warp == 2) {
            // ------------------------------------------------------------------ scales of the rows times the weights' one
            constexpr int kPer = kTN / 32, kAhead = kTN == 256 ? 2 : 8;
            int slot = 0;
            uint32_t phase = 0;
            bool alive = true;
            for (int item = first_item; alive && item < num_items; item += stride) {
                const Item w = find_item<kTN, kRows>(p, begins, items, item);
                const float *sa = p.g.a_scale + w.row0 * p.g.as_sm;
                const bool held = w.n0 + my_n < p.g.n;  // else this CTA of the pair has no weights
                const float *sb = p.g.b_scale + w.group * p.g.bs_sg + (held ? (w.n0 + my_n) / kScaleBlock : 0) * p.g.bs_sn;
                for (int kb0 = kb_begin; alive && kb0 < kb_end; kb0 += kAhead) {
                    float s[kAhead][kPer], t[kAhead];
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        const bool there = kb0 + i < kb_end;
                        t[i] = there ? sb[(kb0 + i) * p.g.bs_sk] : 0.0f;
#pragma unroll
                        for (int j = 0; j < kPer; ++j) {
                            const int c = j * 32 + lane;
                            s[i][j] = there && c < w.count ? sa[c * p.g.as_sm + (kb0 + i) * p.g.as_sk] : 0.0f;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kAhead; ++i) {
                        if (alive && kb0 + i < kb_end) {
                            alive = warp_wait(mbar_test(scale_empty + slot, phase ^ 1u), scale_empty + slot, phase ^ 1u, abort_flag, p.status, 5,
                                              p.wait_limit);
                            const uint32_t at = smem_u32(scales) + static_cast<uint32_t>(slot * kTN * 4);
#pragma unroll
                            for (int j = 0; j < kPer; ++j) {
                                // column 16u + 4j + q goes to 16u + 4q + j: the columns of a thread lie next to one another
                                const uint32_t c = static_cast<uint32_t>(j * 32 + lane);
                                const uint32_t to = (c & ~15u) | (c & 3u) << 2 | (c & 12u) >> 2;
                                store_shared(at + to * 4, s[i][j] * t[i]);
                            }
                            __syncwarp();
                            if (lane == 0) {
                                mbar_arrive(scale_full + slot);
                            }
                            if (++slot == kScaleSlots) {
                                slot = 0;
                                phase ^= 1u;
                            }
                        }
                    }
                }
            }
        }
    } else {
        if (kSums && kTN == 256) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        }
        // ---------------------------------------------------------------------- sums and results
        if constexpr (kRows) {
            sum_rows(p, begins, items, num_items, first_item, stride, rank, warp, lane, tmem_base, tmem_full, tmem_empty, smem_u32(units),
                     smem_u32(bias_area), abort_flag);
        } else {
            constexpr int kRegs = S::kChunk / 2;  // registers of 16 lanes x a chunk of columns
            const int quarter = warp & 3, half = (warp - 4) >> 2;
            const uint32_t my_bias = smem_u32(bias_area) + static_cast<uint32_t>((warp - 4) * 128);
            const uint32_t lanes_at = static_cast<uint32_t>(quarter * 32) << 16;
            const uint32_t drained = S::kPair ? map_to_rank(smem_u32(tmem_empty), 0u) : 0u;
            int buffer = 0, slot = 0;
            uint32_t buffer_phase = 0, slot_phase = 0;
            auto release = [&]() {  // the MMAs may have the buffer again
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (S::kPair) {
                        mbar_arrive_cluster(drained + static_cast<uint32_t>(buffer * 8));
                    } else {
                        mbar_arrive(tmem_empty + buffer);
                    }
                }
                if (++buffer == S::kBuffers) {
                    buffer = 0;
                    buffer_phase ^= 1u;
                }
            };
            for (int item = first_item; item < num_items; item += stride) {
                const Item w = find_item<kTN, kRows>(p, begins, items, item);
                const int n_warp = w.n0 + my_n + quarter * 32;
                float bias_lane = 0.0f;
                if (p.g.has_bias != 0 && n_warp + lane < p.g.n) {
                    bias_lane = load_as_f32(p.g.bias, p.g.bias_dtype, w.group * p.g.bias_sg + (n_warp + lane) * p.g.bias_sn);
                }
                bool alive = true;
                float sum[kSums ? S::kChunks : 1][2][kRegs];  // 16 lanes each
                if (kSums) {
#pragma unroll
                    for (int i = 0; i < S::kChunks; ++i) {
#pragma unroll
                        for (int j = 0; j < kRegs; ++j) {
                            sum[i][0][j] = 0.0f;
                            sum[i][1][j] = 0.0f;
                        }
                    }
#pragma unroll 1
                    for (int kb = kb_begin; kb < kb_end; kb += kScaled ? 1 : p.drain) {
                        const bool scales_there = !kScaled || mbar_test(scale_full + slot, slot_phase);
                        const bool sums_there = mbar_test(tmem_full + buffer, buffer_phase);
                        alive = (!kScaled || warp_wait(scales_there, scale_full + slot, slot_phase, abort_flag, p.status, 6, p.wait_limit)) &&
                                warp_wait(sums_there, tmem_full + buffer, buffer_phase, abort_flag, p.status, 4, p.wait_limit);
                        if (!alive) {
                            break;
                        }
                        tc_fence_after();
                        const uint32_t from = tmem_base + lanes_at + static_cast<uint32_t>(buffer * kTN);
                        const uint32_t scale_at = smem_u32(scales) + static_cast<uint32_t>(slot * kTN * 4 + (lane & 3) * 16);
#pragma unroll
                        for (int i = 0; i < S::kChunks; ++i) {
                            const int c0 = (S::kWays * i + half) * S::kChunk;
                            if (c0 >= w.cols) {
                                break;
                            }
                            uint32_t lo[kRegs], hi[kRegs];
                            tmem_load(from + static_cast<uint32_t>(c0), lo);
                            tmem_load(from + (16u << 16) + static_cast<uint32_t>(c0), hi);
                            float s[S::kChunk / 4];
#pragma unroll
                            for (int u = 0; kScaled && u < S::kChunk / 16; ++u) {
                                load_shared_4(scale_at + static_cast<uint32_t>((c0 + u * 16) * 4), s + 4 * u);
                            }
                            tmem_wait(lo);
                            tmem_wait(hi);
#pragma unroll
                            for (int j = 0; j < kRegs; ++j) {
                                const float scale = kScaled ? s[j / 2] : 1.0f;
                                sum[i][0][j] = fmaf(__uint_as_float(lo[j]), scale, sum[i][0][j]);
                                sum[i][1][j] = fmaf(__uint_as_float(hi[j]), scale, sum[i][1][j]);
                            }
                        }
                        release();
                        if (kScaled) {
                            if (lane == 0) {
                                mbar_arrive(scale_empty + slot);
                            }
                            if (++slot == kScaleSlots) {
                                slot = 0;
                                slot_phase ^= 1u;
                            }
                        }
                    }
                } else {
                    alive = warp_wait(mbar_test(tmem_full + buffer, buffer_phase), tmem_full + buffer, buffer_phase, abort_flag, p.status, 4, p.wait_limit);
                    tc_fence_after();
                }
                if (!alive) {
                    break;
                }
                store_shared(my_bias + static_cast<uint32_t>(lane * 4), bias_lane);
                __syncwarp();
                float bias[4];
                load_shared_4(my_bias + static_cast<uint32_t>((lane & 7) * 16), bias);
                const uint32_t from = tmem_base + lanes_at + static_cast<uint32_t>(buffer * kTN);
                constexpr int kUnitsPerChunk = S::kChunk / 16;
#pragma unroll 1
                for (int u = 0; u < S::kChunks * kUnitsPerChunk; ++u) {
                    const int c0 = (S::kWays * (u / kUnitsPerChunk) + half) * S::kChunk + u % kUnitsPerChunk * 16;
                    if (c0 >= w.cols) {
                        break;
                    }
                    const int unit = p.splits > 1 ? c0 / 16 * 4 + quarter : warp - 4;
                    const uint32_t unit_at = smem_u32(units) + static_cast<uint32_t>(unit * kUnitBytes);
                    // column 4j + lane % 4, row lane / 4 (+ 8 and 16)
                    const uint32_t put_at = unit_at + static_cast<uint32_t>(((lane & 3) * kUnitPitch + lane / 4) * 4);
                    if constexpr (kSums) {
                        __syncwarp();
                        auto put = [&](auto which) {
                            constexpr int v = decltype(which)::value;
                            if constexpr (v < S::kChunks * kUnitsPerChunk) {
#pragma unroll
                                for (int j = 0; j < 16; ++j) {  // j: lanes' half, column / 4, lanes' eight
                                    store_shared(put_at + static_cast<uint32_t>(((j >> 1 & 3) * 4 * kUnitPitch + (j >> 3) * 16 + (j & 1) * 8) * 4),
                                                 sum[v / kUnitsPerChunk][j >> 3][v % kUnitsPerChunk * 8 + (j & 7)]);
                                }
                            }
                        };
                        switch (u) {  // the registers' numbers are fixed
                            case 0: put(std::integral_constant<int, 0>()); break;
                            case 1: put(std::integral_constant<int, 1>()); break;
                            case 2: put(std::integral_constant<int, 2>()); break;
                            case 3: put(std::integral_constant<int, 3>()); break;
                            case 4: put(std::integral_constant<int, 4>()); break;
                            case 5: put(std::integral_constant<int, 5>()); break;
                            case 6: put(std::integral_constant<int, 6>()); break;
                            default: put(std::integral_constant<int, 7>()); break;
                        }
                    } else {
                        uint32_t lo[8], hi[8];
                        tmem_load(from + static_cast<uint32_t>(c0), lo);
                        tmem_load(from + (16u << 16) + static_cast<uint32_t>(c0), hi);
                        tmem_wait(lo);
                        tmem_wait(hi);
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t to = put_at + static_cast<uint32_t>(((j >> 1) * 4 * kUnitPitch + (j & 1) * 8) * 4);
                            store_shared(to, __uint_as_float(lo[j]));
                            store_shared(to + 64, __uint_as_float(hi[j]));
                        }
                    }
                    __syncwarp();
                    if (p.splits == 1) {
                        if (p.vec != 0 && n_warp + 32 <= p.g.n) {
                            float v[4][4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                load_shared_4(unit_at + static_cast<uint32_t>(((lane / 8 + 4 * i) * kUnitPitch + (lane & 7) * 4) * 4), v[i]);
                            }
                            finish_unit(p.g, w.row0 + c0, w.count - c0, n_warp + (lane & 7) * 4, bias, v, lane);
                        } else {
                            finish_unit_any(p.g, w.row0 + c0, w.count - c0, n_warp, my_bias, unit_at, lane);
                        }
                    }
                }
                if (!kSums) {
                    release();
                }
            }
        }
    }

    // ---------------------------------------------------------------------- teardown
    // Tensor memory goes back before a CTA waits for others of its cluster: launches on two streams that share SMs could each hold what
    // the other's CTAs, and with them its own, wait for.
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort_flag != 0) {
        // give copies and MMAs that were already issued time to land before the memory is handed back
        const long long t0 = clock64();
        while (clock64() - t0 < 400000ll) {
            __nanosleep(1000);
        }
        __syncthreads();
    }
    if (S::kPair) {
        cluster_barrier();  // neither CTA leaves while the other's MMAs or arrivals may still reach it
    }
    if (warp == 1 && S::kPair) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
    } else if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
    }

    if (S::kSplits && p.splits > 1) {
        // ---------------------------------------------------------------------- partial sums of the cluster, in rank order
        __syncwarp();
        cluster_barrier();
        if (warp >= 4 && first_item < num_items && *abort_flag == 0) {
            unsigned char *whole = smem + S::kUnits * kUnitBytes;
            const Item w = find_item<kTN, kRows>(p, begins, items, first_item);
            for (int unit = rank + (warp - 4) * p.splits; unit < w.cols / 16 * 4; unit += kSumWarps * p.splits) {
                const int c0 = unit / 4 * 16, quarter = unit & 3, n0 = w.n0 + quarter * 32;
                const uint32_t unit_at = smem_u32(units) + static_cast<uint32_t>(unit * kUnitBytes);
                float v[4][4] = {};
                for (int r = 0; r < p.splits; ++r) {
                    const uint32_t from = map_to_rank(unit_at + static_cast<uint32_t>((lane / 8 * kUnitPitch + (lane & 7) * 4) * 4), static_cast<uint32_t>(r));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x[4];
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                                     : "r"(from + static_cast<uint32_t>(4 * i * kUnitPitch * 4)));
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            v[i][j] += x[j];
                        }
                    }
                }
                const uint32_t bias_at = smem_u32(bias_area) + static_cast<uint32_t>(quarter * 128);  // of the first warp that owns the quarter
                if (p.vec != 0 && n0 + 32 <= p.g.n) {
                    float bias[4];
                    load_shared_4(bias_at + static_cast<uint32_t>((lane & 7) * 16), bias);
                    finish_unit(p.g, w.row0 + c0, w.count - c0, n0 + (lane & 7) * 4, bias, v, lane);
                } else {
                    // not over the partial sums, which other CTAs may still have to read
                    const uint32_t whole_at = smem_u32(whole) + static_cast<uint32_t>((warp - 4) * kUnitBytes);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                                         whole_at + static_cast<uint32_t>(((lane / 8 + 4 * i) * kUnitPitch + (lane & 7) * 4) * 4)),
                                     "f"(v[i][0]), "f"(v[i][1]), "f"(v[i][2]), "f"(v[i][3])
                                     : "memory");
                    }
                    __syncwarp();
                    finish_unit_any(p.g, w.row0 + c0, w.count - c0, n0, bias_at, whole_at, lane);
                }
            }
        }
        __syncwarp();
        cluster_barrier();  // no CTA leaves while another still reads its shared memory
    }
}

}  // namespace grp

}  // namespace kb
