// Grouped and block-scaled products (grouped.cuh) on the tensor cores: tcgen05.mma kind::f16 / kind::f8f6f4 fed by TMA.
//
// Orientation.  Weights stand on the M side of the MMA (128 of their rows per CTA), the rows of a group on the N side, 16 to kTN of them:
// a group pads its last tile to 16 rows instead of 128, its weights are read once for as many rows as fit (few rows: bound by the
// weights' bytes; many: by the tensor pipe), and 128 weight rows share one scale per block of K.
//
// Roles (384 threads): warp 0 loads (TMA), warp 1 issues MMAs, warp 2 fetches the scales, warps 4-11 take the accumulators: a warp
// owns 32 TMEM lanes (weight rows) and every other chunk of columns (rows of the group).  CTAs are persistent; work item = (group, rows
// tile, 128 weight rows), found by a search in the groups' running item counts, which every CTA builds from the offsets.
//
// Scales.  The accumulator of a block of 128 k leaves tensor memory by itself (two to four buffers take turns) and is added to fp32
// registers with the product of its scales, two elements per fma.rn.f32x2.  Tensor memory is read as 16 lanes x 256 bits, so that a thread
// holds few columns (2 of 8) of many rows and needs few scales: two columns' scales serve 4 rows, one 16-byte read of shared memory 16 FMAs.
//
// Few items: clusters of up to 8 CTAs cut K, exchange their partial sums through distributed shared memory and add them in rank order.
#pragma once

#include "grouped.cuh"
#include "sm100_ptx.cuh"

namespace kb {

namespace grp {

constexpr int kThreads = 384;
constexpr int kSumWarps = 8;
constexpr int kTileN = 128;             // weight rows per CTA
constexpr int kWeightBytes = kTileN * 128;
constexpr int kBoxRows = 32;            // rows of a per copy
constexpr int kMaxStages = 12;
constexpr int kMaxBuffers = 4;
constexpr int kScaleSlots = 8;
constexpr int kUnitPitch = 36;          // floats between the columns of a staged unit of 16 columns x 32 rows: conflict-free both ways
constexpr int kUnitBytes = 16 * kUnitPitch * 4;
constexpr int kSmemLimit = 232448;
// registers per thread where a warp's sums take 128 of them: 4 control warps and 8 that sum share what the launch has, 168 each
constexpr int kControlRegs = 88, kSumRegs = 208;
static_assert(128 * kControlRegs + 256 * kSumRegs <= kThreads * 168, "register split");
constexpr int kBarrierBytes = (2 * kMaxStages + 2 * kMaxBuffers + 2 * kScaleSlots) * 8 + 16;

template <bool kScaled, int kTN>
struct Shape {
    static constexpr int kBuffers = kScaled ? (kTN == 256 ? 2 : 4) : 2;
    static constexpr int kTmemCols = kBuffers * kTN;
    static constexpr int kChunk = kTN >= 128 ? 32 : 16;       // columns a warp takes at a time; the two warps of a lane quarter take turns
    static constexpr int kChunks = kTN / kChunk / 2;          // per warp
    static constexpr int kStageBytes = kWeightBytes + kTN * 128;
    static constexpr bool kSplits = kTN <= 64;                // whether launches may cut K (the partial sums have to fit)
    static constexpr int kUnits = kSplits && kTN / 16 * 4 > kSumWarps ? kTN / 16 * 4 : kSumWarps;
    static constexpr int kScaleBytes = kScaled ? kScaleSlots * kTN * 4 : 0;
    static constexpr int kFixedBytes = kUnits * kUnitBytes + kSumWarps * 128 + kScaleBytes + kBarrierBytes;
};

struct TcParams {
    GroupedParams g;
    int num_kb;        // blocks of 128 bytes of K
    int kb_elems;      // elements in one
    int tiles_n;
    int splits, kb_per_split;
    int stages;
    int band;          // row tiles that share the weight tiles of a raster band
    int vec;           // rows of c begin on 16-byte boundaries and are contiguous
    unsigned idesc;    // without N
    int load_kb;       // k-blocks from this one on are not loaded (test hook)
    DeviceStatus *status;
    long long wait_limit;
};

struct Item {
    int group, row0, count, cols, n0;  // cols: count rounded up to 16
};

template <int kTN>
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
    const int local = item - items[lo], begin = begins[lo], rows = begins[lo + 1] - begin;
    const int tiles = (rows + kTN - 1) / kTN;
    const int tall = ((rows + tiles - 1) / tiles + 15) & ~15;  // rows of a tile: the group cut evenly
    const int per_band = p.band * p.tiles_n;
    const int first = local / per_band * p.band;
    const int wide = tiles - first < p.band ? tiles - first : p.band;
    const int in_band = local % per_band;
    Item w;
    w.group = lo;
    w.n0 = in_band / wide * kTileN;
    w.row0 = begin + (first + in_band % wide) * tall;
    const int left = begin + rows - w.row0;
    w.count = left < tall ? left : tall;
    w.cols = (w.count + 15) & ~15;
    return w;
}

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 16 lanes x 32 columns: registers 4g + 2h + e hold lane (thread / 4) + 8h, column 8g + 2 (thread % 4) + e
__device__ __forceinline__ void tmem_load_16x32(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// the same, 16 columns
__device__ __forceinline__ void tmem_load_16x16(uint32_t taddr, uint32_t (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
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
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16])
{
    tmem_load_16x32(taddr, r);
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[8])
{
    tmem_load_16x16(taddr, r);
}

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void load_shared_2x64(uint32_t at, uint64_t &a, uint64_t &b)
{
    asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(at));
}
__device__ __forceinline__ void load_shared_4(uint32_t at, float *v)
{
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at));
}
__device__ __forceinline__ void store_shared(uint32_t at, float v)
{
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
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

template <bool kPrecise>
__device__ __forceinline__ void activate(float (&v)[8], int act, float alpha)
{
    switch (act) {
        case KUDNN_B200_ACT_NONE:
            break;
        case KUDNN_B200_ACT_RELU:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = activation<kPrecise>(v[i], KUDNN_B200_ACT_RELU, alpha);
            }
            break;
        case KUDNN_B200_ACT_SWISH:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = activation<kPrecise>(v[i], KUDNN_B200_ACT_SWISH, alpha);
            }
            break;
        case KUDNN_B200_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = kPrecise ? activation<true>(v[i], KUDNN_B200_ACT_GELU_TANH, alpha) : gelu_tanh_sigmoid(v[i]);
            }
            break;
        default:
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                const float x = i < 4 ? (i < 2 ? (i == 0 ? v[0] : v[1]) : (i == 2 ? v[2] : v[3])) : (i < 6 ? (i == 4 ? v[4] : v[5]) : (i == 6 ? v[6] : v[7]));
                const float y = activation_any(x, act, alpha, kPrecise ? 1 : 0);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = i == j ? y : v[j];
                }
            }
            break;
    }
}

// Eight neighbouring results of one row of c: bias, activation, rounding, store.
__device__ __forceinline__ void finish_8(const TcParams &p, int row, int n, float (&v)[8], uint32_t bias_at)
{
    const GroupedParams &g = p.g;
    if (g.has_bias != 0) {
        float b[8];
        load_shared_4(bias_at, b);
        load_shared_4(bias_at + 16, b + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] += b[i];
        }
    }
    if (g.c_dtype == KUDNN_B200_F32) {
        activate<true>(v, g.act, g.act_alpha);
    } else {
        activate<false>(v, g.act, g.act_alpha);
    }
    const long long at = row * g.c_sm + n * g.c_sn;
    if (p.vec != 0 && n + 8 <= g.n) {
        if (g.c_dtype == KUDNN_B200_F32) {
            float4 *to = reinterpret_cast<float4 *>(static_cast<float *>(g.c) + at);
            to[0] = make_float4(v[0], v[1], v[2], v[3]);
            to[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (g.c_dtype == KUDNN_B200_F16) {
                    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            *reinterpret_cast<uint4 *>(static_cast<unsigned short *>(g.c) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (n + i < g.n) {
                store_exact(g.c, g.c_dtype, at + i * g.c_sn, round_rne(v[i], g.c_dtype));
            }
        }
    }
}

template <bool kScaled, int kTN>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ TcParams p)
{
    using S = Shape<kScaled, kTN>;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *units = smem + p.stages * S::kStageBytes;
    unsigned char *bias_area = units + S::kUnits * kUnitBytes;
    unsigned char *scales = bias_area + kSumWarps * 128;
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

    const int warp = threadIdx.x >> 5;
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
            mbar_init(tmem_empty + s, kSumWarps);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            mbar_init(scale_full + s, 1);
            mbar_init(scale_empty + s, kSumWarps);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(S::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_b) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();  // only now that this CTA holds its tensor memory
    pdl_wait();

    // ---- the groups: offsets made to ascend, and the items before each group
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
    const int num_items = items[p.g.groups];
    const int first_item = p.splits > 1 ? static_cast<int>(blockIdx.x) / p.splits : static_cast<int>(blockIdx.x);
    // launches that cut K have a cluster for every item that there can be
    const int stride = p.splits > 1 ? num_items + 1 : static_cast<int>(gridDim.x);
    const int rank = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int kb_begin = rank * p.kb_per_split;
    const int kb_end = kb_begin + p.kb_per_split < p.num_kb ? kb_begin + p.kb_per_split : p.num_kb;

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
        if (kScaled && kTN == 256) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kControlRegs));
        }
        if (warp == 0 && lane == 0) {
            // ------------------------------------------------------------------ loads
            int stage = 0;
            uint32_t phase = 0;
            bool alive = true;
            for (int item = first_item; alive && item < num_items; item += stride) {
                const Item w = find_item<kTN>(p, begins, items, item);
                const int boxes = (w.cols + kBoxRows - 1) / kBoxRows;
                const uint32_t bytes = static_cast<uint32_t>(kWeightBytes + boxes * kBoxRows * 128);
                const int end = kb_end < p.load_kb ? kb_end : p.load_kb;
                for (int kb = kb_begin; kb < end; ++kb) {
                    if (!mbar_wait(empty_bar + stage, phase ^ 1u, abort_flag, p.status, 1, p.wait_limit)) {
                        alive = false;
                        break;
                    }
                    unsigned char *at = smem + stage * S::kStageBytes;
                    const int x = kb * p.kb_elems;
                    mbar_expect_tx(full_bar + stage, bytes);
                    tma_load_3d(at, &tmap_b, full_bar + stage, x, w.n0, w.group);
                    for (int i = 0; i < boxes; ++i) {
                        tma_load_3d(at + kWeightBytes + i * kBoxRows * 128, &tmap_a, full_bar + stage, x, w.row0 + i * kBoxRows, 0);
                    }
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        } else if (warp == 1 && lane == 0) {
            // ------------------------------------------------------------------ MMAs
            int stage = 0, buffer = 0;
            uint32_t phase = 0, buffer_phase = 0;
            bool alive = true;
            for (int item = first_item; alive && item < num_items; item += stride) {
                const Item w = find_item<kTN>(p, begins, items, item);
                const uint32_t idesc = p.idesc | static_cast<uint32_t>(w.cols >> 3) << 17;
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    if (kScaled || kb == kb_begin) {
                        alive = mbar_wait(tmem_empty + buffer, buffer_phase ^ 1u, abort_flag, p.status, 2, p.wait_limit);
                        tc_fence_after();
                    }
                    alive = alive && mbar_wait(full_bar + stage, phase, abort_flag, p.status, 3, p.wait_limit);
                    if (!alive) {
                        break;
                    }
                    tc_fence_after();
                    const uint32_t at = smem_u32(smem) + static_cast<uint32_t>(stage * S::kStageBytes);
                    const uint64_t wdesc = make_smem_desc(at), xdesc = make_smem_desc(at + kWeightBytes);
                    const uint32_t to = tmem_base + static_cast<uint32_t>(buffer * kTN);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint64_t d = static_cast<uint64_t>(2 * ks);
                        if (kScaled) {
                            umma_f8(to, wdesc + d, xdesc + d, idesc, ks != 0 ? 1u : 0u);
                        } else {
                            umma<KUDNN_B200_F16>(to, wdesc + d, xdesc + d, idesc, kb != kb_begin || ks != 0 ? 1u : 0u);
                        }
                    }
                    umma_commit(empty_bar + stage);
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (kScaled || kb + 1 == kb_end) {
                        umma_commit(tmem_full + buffer);
                        if (++buffer == S::kBuffers) {
                            buffer = 0;
                            buffer_phase ^= 1u;
                        }
                    }
                }
            }
        } else if (kScaled && warp == 2) {
            // ------------------------------------------------------------------ scales of the rows times the weights' one
            constexpr int kPer = kTN / 32, kAhead = kTN == 256 ? 2 : 8;
            int slot = 0;
            uint32_t phase = 0;
            bool alive = true;
            for (int item = first_item; alive && item < num_items; item += stride) {
                const Item w = find_item<kTN>(p, begins, items, item);
                const float *sa = p.g.a_scale + w.row0 * p.g.as_sm;
                const float *sb = p.g.b_scale + w.group * p.g.bs_sg + w.n0 / kScaleBlock * p.g.bs_sn;
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
                            alive = __all_sync(0xffffffffu, mbar_wait(scale_empty + slot, phase ^ 1u, abort_flag, p.status, 5, p.wait_limit));
                            const uint32_t at = smem_u32(scales) + static_cast<uint32_t>(slot * kTN * 4);
#pragma unroll
                            for (int j = 0; j < kPer; ++j) {
                                // column 16u + 8g + 2q + e goes to 16u + 4q + 2g + e, so that a thread's two pairs of a unit are 16 bytes
                                const uint32_t c = static_cast<uint32_t>(j * 32 + lane);
                                const uint32_t to = (c & ~15u) | (c & 6u) << 1 | (c & 8u) >> 2 | (c & 1u);
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
        if (kScaled && kTN == 256) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        }
        // ---------------------------------------------------------------------- sums and results
        constexpr int kRegs = S::kChunk / 2;  // 32-bit registers of 16 lanes x a chunk of columns
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t my_bias = smem_u32(bias_area) + static_cast<uint32_t>((warp - 4) * 128);
        const uint32_t lanes_at = static_cast<uint32_t>(quarter * 32) << 16;
        int buffer = 0, slot = 0;
        uint32_t buffer_phase = 0, slot_phase = 0;
        for (int item = first_item; item < num_items; item += stride) {
            const Item w = find_item<kTN>(p, begins, items, item);
            const int n_warp = w.n0 + quarter * 32;
            float bias = 0.0f;
            if (p.g.has_bias != 0 && n_warp + lane < p.g.n) {
                bias = load_as_f32(p.g.bias, p.g.bias_dtype, w.group * p.g.bias_sg + (n_warp + lane) * p.g.bias_sn);
            }
            bool alive = true;
            uint64_t sum[S::kChunks][2][kRegs / 2];  // 16 lanes at a time; in pairs of neighbouring columns
            if (kScaled) {
#pragma unroll
                for (int i = 0; i < S::kChunks; ++i) {
#pragma unroll
                    for (int j = 0; j < kRegs / 2; ++j) {
                        sum[i][0][j] = 0;
                        sum[i][1][j] = 0;
                    }
                }
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    alive = mbar_wait(scale_full + slot, slot_phase, abort_flag, p.status, 6, p.wait_limit) &&
                            mbar_wait(tmem_full + buffer, buffer_phase, abort_flag, p.status, 4, p.wait_limit);
                    alive = __all_sync(0xffffffffu, alive);
                    if (!alive) {
                        break;
                    }
                    tc_fence_after();
                    const uint32_t from = tmem_base + lanes_at + static_cast<uint32_t>(buffer * kTN);
                    const uint32_t scale_at = smem_u32(scales) + static_cast<uint32_t>(slot * kTN * 4 + (lane & 3) * 16);
#pragma unroll
                    for (int i = 0; i < S::kChunks; ++i) {
                        const int c0 = (2 * i + half) * S::kChunk;
                        if (c0 < w.cols) {
                            uint32_t lo[kRegs], hi[kRegs];
                            tmem_load(from + static_cast<uint32_t>(c0), lo);
                            tmem_load(from + (16u << 16) + static_cast<uint32_t>(c0), hi);
                            uint64_t s[S::kChunk / 8];
#pragma unroll
                            for (int u = 0; u < S::kChunk / 16; ++u) {
                                load_shared_2x64(scale_at + static_cast<uint32_t>((c0 + u * 16) * 4), s[2 * u], s[2 * u + 1]);
                            }
                            tmem_wait(lo);
                            tmem_wait(hi);
#pragma unroll
                            for (int j = 0; j < kRegs / 2; ++j) {  // pair j: group of 8 columns j / 2, lane half j % 2
                                sum[i][0][j] = fma2(pack2(lo[2 * j], lo[2 * j + 1]), s[j / 2], sum[i][0][j]);
                                sum[i][1][j] = fma2(pack2(hi[2 * j], hi[2 * j + 1]), s[j / 2], sum[i][1][j]);
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(tmem_empty + buffer);
                        mbar_arrive(scale_empty + slot);
                    }
                    if (++buffer == S::kBuffers) {
                        buffer = 0;
                        buffer_phase ^= 1u;
                    }
                    if (++slot == kScaleSlots) {
                        slot = 0;
                        slot_phase ^= 1u;
                    }
                }
            } else {
                alive = __all_sync(0xffffffffu, mbar_wait(tmem_full + buffer, buffer_phase, abort_flag, p.status, 4, p.wait_limit));
                tc_fence_after();
            }
            if (!alive) {
                break;
            }
            store_shared(my_bias + static_cast<uint32_t>(lane * 4), bias);
            const uint32_t from = tmem_base + lanes_at + static_cast<uint32_t>(buffer * kTN);
#pragma unroll
            for (int i = 0; i < S::kChunks; ++i) {
                const int c0 = (2 * i + half) * S::kChunk;
                if (c0 < w.cols) {
                    if (!kScaled) {
                        uint32_t lo[kRegs], hi[kRegs];
                        tmem_load(from + static_cast<uint32_t>(c0), lo);
                        tmem_load(from + (16u << 16) + static_cast<uint32_t>(c0), hi);
                        tmem_wait(lo);
                        tmem_wait(hi);
#pragma unroll
                        for (int j = 0; j < kRegs / 2; ++j) {
                            sum[i][0][j] = pack2(lo[2 * j], lo[2 * j + 1]);
                            sum[i][1][j] = pack2(hi[2 * j], hi[2 * j + 1]);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < S::kChunk / 16; ++u) {
                        const int unit = p.splits > 1 ? (c0 / 16 + u) * 4 + quarter : warp - 4;
                        const uint32_t unit_at = smem_u32(units) + static_cast<uint32_t>(unit * kUnitBytes);
                        __syncwarp();
#pragma unroll
                        for (int hl = 0; hl < 2; ++hl) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                float x, y;
                                unpack2(sum[i][hl][4 * u + j], x, y);
                                const int col = (j / 2) * 8 + 2 * (lane & 3), row = hl * 16 + (j & 1) * 8 + lane / 4;
                                store_shared(unit_at + static_cast<uint32_t>((col * kUnitPitch + row) * 4), x);
                                store_shared(unit_at + static_cast<uint32_t>(((col + 1) * kUnitPitch + row) * 4), y);
                            }
                        }
                        __syncwarp();
                        if (p.splits == 1) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const int col = j * 8 + lane / 4, n8 = (lane & 3) * 8;
                                float v[8];
                                load_shared_4(unit_at + static_cast<uint32_t>((col * kUnitPitch + n8) * 4), v);
                                load_shared_4(unit_at + static_cast<uint32_t>((col * kUnitPitch + n8 + 4) * 4), v + 4);
                                if (c0 + u * 16 + col < w.count && n_warp + n8 < p.g.n) {
                                    finish_8(p, w.row0 + c0 + u * 16 + col, n_warp + n8, v, my_bias + static_cast<uint32_t>(n8 * 4));
                                }
                            }
                        }
                    }
                }
            }
            if (!kScaled) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(tmem_empty + buffer);
                }
                if (++buffer == S::kBuffers) {
                    buffer = 0;
                    buffer_phase ^= 1u;
                }
            }
        }
    }

    if (S::kSplits && p.splits > 1) {
        // ---------------------------------------------------------------------- partial sums of the cluster, in rank order
        __syncwarp();
        cluster_barrier();
        if (warp >= 4 && first_item < num_items && *abort_flag == 0) {
            const Item w = find_item<kTN>(p, begins, items, first_item);
            for (int unit = rank + (warp - 4) * p.splits; unit < w.cols / 16 * 4; unit += kSumWarps * p.splits) {
                const int c0 = unit / 4 * 16, quarter = unit & 3;
                const uint32_t unit_at = smem_u32(units) + static_cast<uint32_t>(unit * kUnitBytes);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int col = j * 8 + lane / 4, n8 = (lane & 3) * 8, n = w.n0 + quarter * 32 + n8;
                    if (c0 + col < w.count && n < p.g.n) {
                        float v[8] = {};
                        for (int r = 0; r < p.splits; ++r) {
                            const uint32_t at = map_to_rank(unit_at + static_cast<uint32_t>((col * kUnitPitch + n8) * 4), static_cast<uint32_t>(r));
                            float x[8];
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                                         : "r"(at));
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                                         : "r"(at + 16));
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                v[i] += x[i];
                            }
                        }
                        // the bias of this warp's own quarter lies in its area; another quarter's in the area of that quarter's warp
                        finish_8(p, w.row0 + c0 + col, n, v, smem_u32(bias_area) + static_cast<uint32_t>(quarter * 128 + n8 * 4));
                    }
                }
            }
        }
        __syncwarp();
        cluster_barrier();  // no CTA leaves while another still reads its shared memory
    }

    // ---------------------------------------------------------------------- teardown
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
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::kTmemCols) : "memory");
    }
}

}  // namespace grp

}  // namespace kb
