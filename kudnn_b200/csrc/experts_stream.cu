// The block of experts for few tokens in two kernels that stream the weights once (experts.cuh).
//
// What bounds it is reading the chosen experts' weights; everything here serves to keep as many bytes in flight as HBM wants, without pauses:
//   * Both products are cut by weight rows alone: the rows (gate and up rows in pairs) of all chosen experts are dealt out evenly, one CTA per SM,
//     so that every SM streams the same number of bytes; nothing is added up across CTAs, no atomics, and the same call gives the same bits.
//   * The 8 warps of a CTA stream on their own, without barriers.  First kernel: as many groups of warps as the CTA has tiles of rows, up to 8;
//     a group's warps split K and add up at the end of a tile (with a tile per warp, what large batches have, nothing is added up).  Second
//     kernel: each warp an eighth of all steps of all experts at the CTA's rows, with sums of y of its own, added up at the end.
//   * A step of a warp is 128 bytes of up to 32 rows: up to four TMA boxes of eight rows, into a ring of the warp's own, some steps ahead.  Rows and
//     columns beyond the matrix come as zeros, rows beyond the tile are another warp's (their products are dropped).  (Copies by every lane,
//     cp.async or straight into registers, took three to five times the instructions of the products, and their latency bound the whole.)
//   * 16 bytes per lane, as they lie in the ring, are operand fragments of mma.m16n8k16 with a permuted k: weights on the side of 16 rows, tokens on
//     that of 8.  The tokens' fragments are read from L1 and L2 in the same permutation, one step ahead.
//   * The second kernel starts its copies of `down` while the first one ends (its CTAs take the place of the first one's as those leave) and
//     waits only before it reads h.
// h is kept as the tensor cores take it without loss: two bf16 halves (of bf16 and e4m3 weights), or fp32 that the second kernel splits into two
// tf32 halves (of fp16 weights: halves of fp16 would overflow beyond 65504 and lose small values).
#include "experts.cuh"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace kb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMostPairs = kMostExpertTokens * kMostExpertTop;

enum Weights { kBf16, kF16, kE4m3 };

// Waits that gave up, on this device since the last look.
__device__ DeviceStatus experts_status;

struct Waits {
    long long limit;  // in cycles
    int skip_step;    // test hook: from which step of K on nothing is copied, -1 off
};
std::atomic<long long> wait_limit{0};
std::atomic<int> wait_skip{-1};


// Which tokens the experts have: pairs in order of experts and tokens.
struct Lists {
    unsigned long long tokens[kMostExperts];  // bit t: token t is the expert's
    short start[kMostExperts];                // of its pairs
    short expert[kMostExperts];               // the active experts; what follows is by their rank
    short first[kMostExperts];
    short count[kMostExperts];
    unsigned char token[kMostPairs];
    float p[kMostPairs];
    int ids[kMostPairs];  // as given, and the weights
    float given[kMostPairs];
    int active;
    // first kernel: how many warps share a tile, how many tiles an expert's rows are cut into
    // of at least tile_pairs pairs of rows, the first `longer` of one more
    int group_warps, tiles, tile_pairs, longer;
    int abort;  // some wait of the CTA gave up
    unsigned long long full[kWarps][8];
};

template <bool kBf>
__device__ __forceinline__ void mma_16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (kBf) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], float a0, float a1, float a2, float a3, float b0, float b1)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)),
                   "r"(__float_as_uint(b1)));
}

__device__ __forceinline__ uint32_t word(const uint4 &q, int i)
{
    return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w;
}

// Two e4m3 values as fp16 or bf16, exactly, NaN as NaN.  There is no instruction to bf16: by way of fp16 and fp32.
template <bool kBf>
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t w, bool upper)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(upper ? w >> 16 : w)));
    if (!kBf) {
        return h;
    }
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&b);
}

// The first `left` of 8 values of 16 bits (a loop: it is seldom run, and must not become instructions of the path beside it)
__device__ __forceinline__ uint4 load_some(const unsigned short *at, int left)
{
    unsigned long long lo = 0ull, hi = 0ull;
#pragma unroll 1
    for (int i = min(left, 8) - 1; i >= 0; --i) {
        hi = hi << 16 | lo >> 48;
        lo = lo << 16 | at[i];
    }
    return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32));
}
// The first `left` of 4 values of fp32
__device__ __forceinline__ uint4 load_some(const float *at, int left)
{
    unsigned long long lo = 0ull, hi = 0ull;
#pragma unroll 1
    for (int i = min(left, 4) - 1; i >= 0; --i) {
        hi = hi << 32 | lo >> 32;
        lo = lo << 32 | __float_as_uint(at[i]);
    }
    return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32));
}

// The value's upper tf32 half and what is left; a value that is not finite has no rest.
__device__ __forceinline__ float2 split_tf32(float v)
{
    const float hi = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
    return isfinite(v) ? make_float2(hi, v - hi) : make_float2(v, 0.0f);
}

// h in the workspace, a row per pair in the lists' order: bf16 upper halves, then lower ones, or fp32.
__device__ __forceinline__ long long h_pitch(const ExpertsParams &p)
{
    return (p.ffn + 63) / 64 * 64;
}

// A tile has 32 rows of weights, a step 128 bytes of each.
constexpr int kRows = 32;
constexpr int kMostTilePairs = kRows / 2;  // of a gate's and an up's row
constexpr int kBoxRows = 8;
constexpr int kBoxBytes = kBoxRows * 128;
constexpr int kStageBytes = kRows * 128;

// The kernels for experts of up to 8 kTokens tokens: the ring, and behind it the warps' sums.
template <bool kDown, int kTokens>
struct Layout {
    static constexpr int kStages = kTokens == 8 && kDown ? 4 : 5;
    static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
    // up: the sums of 8 tokens of every warp, in two buffers; down: each warp's sums of y
    static constexpr int kSumBytes = kDown ? kWarps * 8 * kTokens * kRows * 4 : 2 * kWarps * 1024;
    static constexpr size_t kBytes = kRingBytes + kSumBytes + sizeof(Lists) + 1024;  // the ring begins on a multiple of 1024
};

// A warp's way through the weights, piece by piece: steps of K of a tile of one expert's rows.  32 bits hold every count (see the launcher).
template <bool kDown>
struct Cursor {
    int rank, row, rows;       // the expert, its first row (of the gate, or of down), how many
    int step, steps, stride;   // of K
    int depth;                 // steps of an expert
    int at, end;               // up: tiles of all active experts, one after the other; down: rows of y
    int offset;                // of the warp in its group
    int begin, until, begin_rank, position;  // down: the group's steps of all experts, one after the other
    __device__ __forceinline__ void start_up(const Lists &l, int warp, int depth_steps)
    {
        // consecutive tiles go to different SMs; next_up() adds a whole round
        at = (warp / l.group_warps - kWarps / l.group_warps) * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);
        end = l.active * l.tiles;
        stride = l.group_warps;
        offset = warp & (stride - 1);
        depth = depth_steps;
        step = offset;
        steps = depth > offset ? (depth - offset + stride - 1) / stride : 0;
    }
    __device__ __forceinline__ bool next_up(const Lists &l)
    {
        at += kWarps / stride * static_cast<int>(gridDim.x);
        if (at >= end) {
            return false;
        }
        rank = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(l.tiles));
        const int tile = at - rank * l.tiles;
        row = tile * l.tile_pairs + min(tile, l.longer);
        rows = l.tile_pairs + (tile < l.longer ? 1 : 0);
        return true;
    }
    // Down: the steps of all experts at the same rows go to groups of warps, as many to each, and a group's warps take turns, so that they read
    // what lies side by side; groups of as many warps as leave each eight steps of an expert.
    __device__ __forceinline__ void start_down(const ExpertsParams &p, const Lists &l, int warp, int depth_steps)
    {
        at = static_cast<int>(static_cast<unsigned>(p.hidden) * blockIdx.x / gridDim.x);
        end = static_cast<int>(static_cast<unsigned>(p.hidden) * (blockIdx.x + 1) / gridDim.x);
        depth = depth_steps;
        stride = depth >= 64 ? 8 : depth >= 32 ? 4 : depth >= 16 ? 2 : 1;
        const int groups = kWarps / stride, group = warp / stride, all = l.active * depth;
        begin = all * group / groups;
        until = all * (group + 1) / groups;
        begin_rank = begin / depth;
        offset = warp & (stride - 1);
        rows = 0;
        position = until;
    }
    // true while the group has steps at the present rows
    __device__ __forceinline__ bool next_down()
    {
        if (position >= until) {
            return false;
        }
        ++rank;
        const int from = position - rank * depth, to = min(depth, until - rank * depth);
        step = from + offset;
        steps = to > step ? (to - step + stride - 1) / stride : 0;
        position += to - from;
        return true;
    }
    __device__ __forceinline__ bool next_rows()
    {
        at += rows;
        if (at >= end) {
            return false;
        }
        row = at;
        const int tiles = (end - at + kRows - 1) / kRows;  // equal ones
        rows = (end - at + tiles - 1) / tiles;
        rank = begin_rank - 1;
        position = begin;
        return true;
    }
};

// How the first kernel's tiles are cut, by one warp: with kWarps / w groups of w warps per SM and r rounds of tiles, an expert's rows are cut into
// as many tiles as that has room for.  What a round costs: the bytes of the SM's tiles at its share of HBM's rate (24 a cycle; a tenth more
// where no warps read side by side), or the steps of a warp at what one takes in latency where HBM waits (800 cycles), and the sums of a group.
__device__ __forceinline__ void plan_tiles(Lists &l, int active, int ffn, int depth_steps, int lane)
{
    const int w = 1 << (lane & 3), extra = lane >> 2, some = max(active, 1);
    const unsigned groups = kWarps / w * gridDim.x;
    const unsigned least = (ffn + kMostTilePairs - 1) / kMostTilePairs;
    const unsigned rounds = (some * least + groups - 1) / groups + extra;
    const int tiles = static_cast<int>(min(static_cast<unsigned>(ffn), max(rounds * groups / some, least)));
    const int pairs = (ffn + tiles - 1) / tiles;
    const float steps = static_cast<float>((depth_steps + w - 1) / w);
    const float bytes = static_cast<float>(kWarps / w * pairs) * 256.0f * static_cast<float>(depth_steps);
    float cost = static_cast<float>(rounds) * (fmaxf(bytes / (w > 2 ? 24.0f : w > 1 ? 23.0f : 21.5f), 800.0f * steps) + (w > 1 ? 600.0f : 300.0f));
    int best = lane;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, cost, o);
        const int other_best = __shfl_xor_sync(0xffffffffu, best, o);
        if (other < cost || (other == cost && other_best < best)) {
            cost = other;
            best = other_best;
        }
    }
    if (best == lane) {
        l.group_warps = w;
        l.tiles = tiles;
        l.tile_pairs = ffn / tiles;
        l.longer = ffn % tiles;
    }
}

// All threads of the CTA; l.tokens is zero.  An id that a token names twice counts once, with both weights.
template <bool kPlan>
__device__ __forceinline__ void make_lists(Lists &l, const ExpertsParams &p, int depth_steps)
{
    const int pairs = p.tokens * p.top, tid = static_cast<int>(threadIdx.x);
    for (int i = tid; i < pairs; i += kThreads) {
        const int e = p.ids[i];
        l.ids[i] = e;
        l.given[i] = p.p[i];
        if (e >= 0 && e < p.experts) {
            atomicOr(&l.tokens[e], 1ull << (i / p.top));  // whatever the order
        }
    }
    __syncthreads();
    if (tid < 32) {
        int active = 0, first = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + tid, count = e < p.experts ? __popcll(l.tokens[e]) : 0;
            const unsigned some = __ballot_sync(0xffffffffu, count > 0);
            int sum = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, sum, o);
                sum += tid >= o ? other : 0;
            }
            if (count > 0) {
                const int at = active + __popc(some & ((1u << tid) - 1u)), start = first + sum - count;
                l.start[e] = static_cast<short>(start);
                l.expert[at] = static_cast<short>(e);
                l.first[at] = static_cast<short>(start);
                l.count[at] = static_cast<short>(count);
            }
            active += __popc(some);
            first += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (tid == 0) {
            l.active = active;
        }
        if (kPlan) {
            plan_tiles(l, active, p.ffn, depth_steps, tid);
        }
    }
    __syncthreads();
    for (int i = tid; i < pairs; i += kThreads) {
        const int e = l.ids[i], t = i / p.top;
        if (e >= 0 && e < p.experts) {
            bool again = false;
            float sum = 0.0f;
            for (int j = t * p.top; j < (t + 1) * p.top; ++j) {
                const bool same = l.ids[j] == e;
                again |= same && j < i;
                sum += same ? l.given[j] : 0.0f;
            }
            if (!again) {
                const int at = l.start[e] + __popcll(l.tokens[e] & ((1ull << t) - 1ull));
                l.token[at] = static_cast<unsigned char>(t);
                l.p[at] = sum;
            }
        }
    }
    __syncthreads();
}

// kTokens: an expert's most, in eights.
template <Weights kW, bool kBf, bool kDown, int kTokens>
__global__ void __launch_bounds__(kThreads, 1) experts_stream_kernel(const __grid_constant__ ExpertsParams p, const __grid_constant__ CUtensorMap map,
                                                                     const __grid_constant__ Waits waits)
{
    using L = Layout<kDown, kTokens>;
    constexpr int kStages = L::kStages;
    constexpr int kElem = kW == kE4m3 ? 1 : 2;
    constexpr int kStep = 128 / kElem;                // of K
    constexpr int kPiece = 16 / kElem;                // of a lane, twice in a step
    constexpr bool kTf32 = kDown && kW == kF16;       // h in fp32, products of tf32
    constexpr bool kBfMma = kW == kBf16 || (kW == kE4m3 && (kBf || kDown));
    constexpr int kPlanes = kDown ? 2 : 1, kLoads = kPiece / 8;
    extern __shared__ unsigned char raw[];
    unsigned char *shared = raw + (1024u - (smem_u32(raw) & 1023u)) % 1024u;
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char *ring = shared + warp * kStages * kStageBytes;
    float4 *sums = reinterpret_cast<float4 *>(shared + L::kRingBytes);  // up: [2][kWarps][2][32]
    float *y_sums = reinterpret_cast<float *>(shared + L::kRingBytes);  // down: [kWarps][tokens][kRows]
    Lists &lists = *reinterpret_cast<Lists *>(shared + L::kRingBytes + L::kSumBytes);
    const int depth = kDown ? p.ffn : p.hidden;  // K
    uint64_t *full = reinterpret_cast<uint64_t *>(lists.full[warp]);  // a barrier per stage of the warp's ring
    volatile int *abort_flag = &lists.abort;
    if (tid == 0) {
        lists.abort = 0;
    }
    if (lane < kStages) {
        mbar_init(full + lane, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");

    if (warp == 0 && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
    }
    for (int e = tid; e < p.experts; e += kThreads) {
        lists.tokens[e] = 0ull;
    }
    __syncthreads();
    const int depth_steps = (depth + kStep - 1) / kStep;
    if (!kDown) {
        pdl_wait();
        pdl_launch_dependents();  // behind the wait: what the second kernel reads ahead of its own is older than this one
    }
    make_lists<!kDown>(lists, p, depth_steps);
    using Place = Cursor<kDown>;
    auto start = [&](Place &c) {
        if (kDown) {
            c.start_down(p, lists, warp, depth_steps);
        } else {
            c.start_up(lists, warp, depth_steps);
        }
    };
    // the next piece with steps of its own; false: none is left
    auto advance = [&](Place &c) {
        do {
            if (kDown) {
                while (!c.next_down()) {
                    if (!c.next_rows() || c.begin == c.until) {
                        return false;
                    }
                }
            } else if (!c.next_up(lists)) {
                return false;
            }
        } while (c.steps == 0);
        return true;
    };

    // ---- the stream: lane i < 4 brings eight rows (up: of the gate, of the up, and the next eight of both)
    int box_row = 0, boxes = 0;
    int ahead_k = 0, ahead_left = 0, ahead_stage = 0, ahead_expert = 0;
    Place ahead;
    start(ahead);
    auto aim = [&]() {
        ahead_left = 0;
        if (advance(ahead)) {
            ahead_left = ahead.steps;
            ahead_k = ahead.step * kStep;
            ahead_expert = lists.expert[ahead.rank];
            boxes = kDown ? (ahead.rows + 7) / 8 : ahead.rows > 8 ? 4 : 2;
            box_row = ahead.row + (kDown ? lane * 8 : (lane >> 1) * 8 + (lane & 1) * p.ffn);
        }
    };
    aim();
    bool gave_up = false;
    auto issue = [&]() {
        if (ahead_left > 0) {
            if (lane < boxes && !gave_up) {
                if (lane == 0) {
                    mbar_expect_tx(full + ahead_stage, boxes * kBoxBytes);
                }
                if (waits.skip_step < 0 || ahead_k / kStep < waits.skip_step) {
                    tma_load_3d(ring + ahead_stage * kStageBytes + lane * kBoxBytes, &map, full + ahead_stage, ahead_k, box_row, ahead_expert);
                }
            }
            ahead_k += ahead.stride * kStep;
            if (--ahead_left == 0) {
                aim();
            }
            ahead_stage = ahead_stage + 1 == kStages ? 0 : ahead_stage + 1;
        }
    };
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) {
        issue();
    }
    if (kDown) {
        for (int i = tid; i < kWarps * p.tokens * kRows; i += kThreads) {
            y_sums[i] = 0.0f;
        }
        pdl_wait();
        pdl_launch_dependents();
        __syncthreads();
    }

    // ---- the tokens' fragments of a step, and its scales: the first eight tokens' are fetched one step ahead
    const long long pitch = h_pitch(p);
    const long long plane_step = static_cast<long long>(p.tokens) * p.top * pitch;
    const bool vector = kDown || ((reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && p.x_ld % 8 == 0);
    const float *scale = kDown ? p.down_scale : p.gate_up_scale;
    const long long ss_e = kDown ? p.ds_se : p.gus_se, ss_n = kDown ? p.ds_sn : p.gus_sn, ss_k = kDown ? p.ds_sk : p.gus_sk;
    struct Tokens {
        uint4 q[2][kPlanes][kLoads];  // [which 64 bytes of weights]; kTf32: [..][which four][0]
    };
    // at: the row of x or h of this lane's token (of lanes without one: of any, their sums are dropped); from element k on; whole: all of the
    // step's elements exist, on 16-byte boundaries
    auto load_tokens = [&](Tokens &b, const void *at, int k, bool whole) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int from_k = k + u * 4 * kPiece, some = depth - from_k;
#pragma unroll
            for (int plane = 0; plane < kPlanes; ++plane) {
                if (kTf32) {
                    const float *from = static_cast<const float *>(at) + from_k + plane * 4;
                    if (whole) {
                        b.q[u][plane][0] = *reinterpret_cast<const uint4 *>(from);
                    } else {
                        b.q[u][plane][0] = load_some(from, some - plane * 4);
                    }
                } else {
                    const unsigned short *from = static_cast<const unsigned short *>(at) + plane * plane_step + from_k;
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        if (whole) {
                            b.q[u][plane][i] = reinterpret_cast<const uint4 *>(from)[i];
                        } else {
                            b.q[u][plane][i] = load_some(from + i * 8, some - i * 8);
                        }
                    }
                }
            }
        }
    };
    auto token_row = [&](int pair) -> const void * {
        if (kTf32) {
            return static_cast<const float *>(p.h) + pair * pitch;
        }
        return kDown ? static_cast<const unsigned short *>(p.h) + pair * pitch
                     : static_cast<const unsigned short *>(p.x) + lists.token[pair] * p.x_ld;
    };
    Tokens next;
    float next_scale[4];
    Place soon;
    start(soon);
    int soon_left = 0, soon_step = 0;
    const void *soon_row = nullptr;
    const float *soon_scale[4];
    auto fetch = [&]() {
        if (soon_left == 0) {
            if (!advance(soon)) {
                return;
            }
            soon_left = soon.steps;
            soon_step = soon.step;
            const int first = lists.first[soon.rank];
            soon_row = token_row(first + min(g, lists.count[soon.rank] - 1));
            if (kW == kE4m3) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // rows g + 8 i, or g and g of the up, then 8 on
                    const int r = min(kDown ? i * 8 + g : (i >> 1) * 8 + g, soon.rows - 1);
                    soon_scale[i] = scale + lists.expert[soon.rank] * ss_e + (soon.row + r + (!kDown && (i & 1) != 0 ? p.ffn : 0)) / 128 * ss_n;
                }
            }
        }
        load_tokens(next, soon_row, soon_step * kStep + t * kPiece, vector && (soon_step + 1) * kStep <= depth);
        if (kW == kE4m3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                next_scale[i] = soon_scale[i][soon_step * ss_k];
            }
        }
        soon_step += soon.stride;
        --soon_left;
    };
    fetch();

    // ---- the products
    // where this lane's fragments of row g lie: chunks t and t + 4, which the copies put in place t ^ g and so on
    const unsigned char *fragment = ring + g * 128 + (t ^ g) * 16;
    const int other = (g & 4) != 0 ? -64 : 64;
    int stage = 0, turn = 0;
    uint32_t parity = 0;

    // a piece for experts of up to 8 kN tokens: sums in c
    auto multiply = [&](const Place &now, auto &c) {
        constexpr int kN = sizeof(c) / 32;
        constexpr bool kAhead = kW == kE4m3 && kN > 1;  // widened once for all tokens
        const int first = lists.first[now.rank], count = lists.count[now.rank];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                c[n][m][0] = c[n][m][1] = c[n][m][2] = c[n][m][3] = 0.0f;
            }
        }
        int step = now.step;
#pragma unroll 1
        for (int s = 0; s < now.steps; ++s, step += now.stride) {
            gave_up = gave_up || !mbar_wait(full + stage, parity, abort_flag, &experts_status, kDown ? 2 : 1, waits.limit);
            uint4 a[2][4];  // [which 64 bytes][row g + 8 i of the tile's 32]
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned char *at = fragment + stage * kStageBytes + r * 1024;
                a[0][r] = *reinterpret_cast<const uint4 *>(at);
                a[1][r] = *reinterpret_cast<const uint4 *>(at + other);
            }
            __syncwarp();
            issue();  // into the stage that has just been read
            if (++stage == kStages) {
                stage = 0;
                parity ^= 1u;
            }
            uint32_t wide[kAhead ? 2 : 1][kAhead ? 4 : 1][kAhead ? 8 : 1];
            if (kAhead) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            wide[kAhead ? u : 0][kAhead ? r : 0][kAhead ? j : 0] = widen_e4m3<kBfMma>(word(a[u][r], j / 2), j % 2 != 0);
                        }
                    }
                }
            }
            float of_block[4];
            if (kW == kE4m3) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    of_block[i] = next_scale[i];
                }
            }
            // sums of the tokens `b`, in two chains in turn: the matrix instructions of one wait for one another
            auto add = [&](float(&sum)[2][4], const Tokens &b) {
                float part[2][4];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    part[m][0] = part[m][1] = part[m][2] = part[m][3] = 0.0f;
                }
                float(&to)[2][4] = kW == kE4m3 ? part : sum;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (kTf32) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint4 &q = b.q[u][kPlanes * (j / 2) / 2][0];
                            const float2 b0 = split_tf32(__uint_as_float(word(q, j % 2 * 2)));
                            const float2 b1 = split_tf32(__uint_as_float(word(q, j % 2 * 2 + 1)));
                            float2 f[4];
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const uint32_t w = word(a[u][r], j);
                                f[r] = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                            }
                            mma_tf32(to[0], f[0].x, f[1].x, f[0].y, f[1].y, b0.y, b1.y);
                            mma_tf32(to[1], f[2].x, f[3].x, f[2].y, f[3].y, b0.y, b1.y);
                            mma_tf32(to[0], f[0].x, f[1].x, f[0].y, f[1].y, b0.x, b1.x);
                            mma_tf32(to[1], f[2].x, f[3].x, f[2].y, f[3].y, b0.x, b1.x);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 2 * kLoads; ++j) {
                            uint32_t w[2][4];
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                if (kAhead) {
                                    w[r / 2][r % 2] = wide[kAhead ? u : 0][kAhead ? r : 0][kAhead ? 2 * j : 0];
                                    w[r / 2][2 + r % 2] = wide[kAhead ? u : 0][kAhead ? r : 0][kAhead ? 2 * j + 1 : 0];
                                } else if (kW == kE4m3) {
                                    w[r / 2][r % 2] = widen_e4m3<kBfMma>(word(a[u][r], j), false);
                                    w[r / 2][2 + r % 2] = widen_e4m3<kBfMma>(word(a[u][r], j), true);
                                } else {
                                    w[r / 2][r % 2] = word(a[u][r], 2 * j);
                                    w[r / 2][2 + r % 2] = word(a[u][r], 2 * j + 1);
                                }
                            }
#pragma unroll
                            for (int plane = kPlanes - 1; plane >= 0; --plane) {
                                const uint4 &q = b.q[u][plane][j / 2];
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    mma_16<kBfMma>(to[m], w[m][0], w[m][1], w[m][2], w[m][3], word(q, j % 2 * 2), word(q, j % 2 * 2 + 1));
                                }
                            }
                        }
                    }
                }
                if (kW == kE4m3) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            sum[m][i] = fmaf(part[m][i], of_block[2 * m + i / 2], sum[m][i]);
                        }
                    }
                }
            };
            add(c[0], next);
            fetch();
            if (kN > 1) {
                const bool whole = vector && (step + 1) * kStep <= depth;
#pragma unroll
                for (int n = 1; n < kN; ++n) {
                    Tokens b;
                    load_tokens(b, token_row(first + min(n * 8 + g, count - 1)), step * kStep + t * kPiece, whole);
                    add(c[n], b);
                }
            }
        }
    };
    // piece by the number of its expert's tokens: every width has code of its own, so that none runs through what is left out
    auto by_width = [&](const Place &now, auto &&piece) {
        const int count = lists.count[now.rank];
        if (kTokens == 1 || count <= 8) {
            float c[1][2][4];
            piece(c, count);
        } else if (kTokens == 2 || count <= 16) {
            float c[kTokens < 2 ? kTokens : 2][2][4];
            piece(c, count);
        } else if (kTokens == 4 || count <= 32) {
            float c[kTokens < 4 ? kTokens : 4][2][4];
            piece(c, count);
        } else {
            float c[kTokens][2][4];
            piece(c, count);
        }
    };

    Place now;
    start(now);
    if (!kDown) {
        auto store_h = [&](long long to, float gate, float up) {
            const float v = expert_gate(gate, up);
            if (kW == kF16) {
                static_cast<float *>(p.h)[to] = v;
            } else {
                const float hi = __bfloat162float(__float2bfloat16_rn(v));
                unsigned short *planes = static_cast<unsigned short *>(p.h);
                planes[to] = f32_to_bf16_rne_bits(v);
                planes[plane_step + to] = f32_to_bf16_rne_bits(isfinite(hi) ? v - hi : 0.0f);
            }
        };
        const int group_warps = lists.group_warps;
        while (now.next_up(lists)) {
            const int first = lists.first[now.rank];
            by_width(now, [&](auto &c, int count) {
                constexpr int kN = sizeof(c) / 32;
                multiply(now, c);
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    if (group_warps == 1) {
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const int r = m * 8 + g, column = n * 8 + 2 * t + j;
                                if (r < now.rows && column < count) {
                                    store_h((first + column) * pitch + now.row + r, c[n][m][j], c[n][m][2 + j]);
                                }
                            }
                        }
                    } else {
                        // the group's sums, eight tokens at a time; two buffers take turns, so that one barrier does
                        float4 *buffer = sums + turn * kWarps * 64;
                        turn ^= 1;
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            buffer[warp * 64 + m * 32 + lane] = make_float4(c[n][m][0], c[n][m][1], c[n][m][2], c[n][m][3]);
                        }
                        const int group = warp / group_warps, threads = group_warps * 32;
                        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads) : "memory");
                        const float *from = reinterpret_cast<const float *>(buffer + group * group_warps * 64);
                        for (int i = tid & (threads - 1); i < 128; i += threads) {
                            const int m = i >> 6, of = i >> 1 & 31, j = i & 1;  // element j of lane `of`, and the one of the up's row
                            float gate = 0.0f, up = 0.0f;
                            for (int w = 0; w < group_warps; ++w) {
                                const float *at = from + (w * 64 + m * 32 + of) * 4 + j;
                                gate += at[0];
                                up += at[2];
                            }
                            const int r = m * 8 + (of >> 2), column = n * 8 + (of & 3) * 2 + j;
                            if (r < now.rows && column < count) {
                                store_h((first + column) * pitch + now.row + r, gate, up);
                            }
                        }
                    }
                }
            });
        }
    } else {
        float *mine = y_sums + warp * p.tokens * kRows;
        while (now.next_rows()) {
            while (now.next_down()) {
                const int first = lists.first[now.rank];
                by_width(now, [&](auto &c, int count) {
                    constexpr int kN = sizeof(c) / 32;
                    multiply(now, c);
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int column = n * 8 + 2 * t + j;
                            if (column < count) {
                                float *to = mine + lists.token[first + column] * kRows + g;
                                const float weight = lists.p[first + column];
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    to[m * 16] = fmaf(weight, c[n][m][j], to[m * 16]);
                                    to[m * 16 + 8] = fmaf(weight, c[n][m][2 + j], to[m * 16 + 8]);
                                }
                            }
                        }
                    }
                });
                __syncwarp();  // the next expert's columns may be other lanes' tokens
            }
            __syncthreads();
            for (int i = tid; i < p.tokens * kRows; i += kThreads) {
                float y = 0.0f;
                for (int w = 0; w < kWarps; ++w) {
                    y += y_sums[w * p.tokens * kRows + i];
                    y_sums[w * p.tokens * kRows + i] = 0.0f;
                }
                const int token = i / kRows, r = i % kRows;
                if (r < now.rows) {
                    store_exact(p.y, p.x_dtype, token * p.y_ld + now.row + r, round_rne(y, p.x_dtype));
                }
            }
            __syncthreads();
        }
    }
    if (gave_up) {
        // the copies that are still on their way, each for a moment
        for (int i = 0; i < kStages; ++i) {
            for (int spin = 0; spin < 100000 && !mbar_try_wait(full + i, parity ^ (i < stage ? 1u : 0u)); ++spin) {
            }
        }
    }
}

template <Weights kW, bool kBf, bool kDown, int kTokens>
cudaError_t launch_one(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    constexpr size_t kShared = Layout<kDown, kTokens>::kBytes;
    static_assert(kShared <= 227 * 1024, "shared memory");
    alignas(64) CUtensorMap map;
    cudaError_t e = tc_encode_groups(&map, kDown ? p.down : p.gate_up, p.w_dtype, p.experts, kDown ? p.hidden : 2ll * p.ffn, kDown ? p.ffn : p.hidden,
                                     std::max(kDown ? p.d_se : p.gu_se, 16ll), kDown ? p.d_sn : p.gu_sn, kBoxRows);
    if (e == cudaSuccess) {
        e = cudaFuncSetAttribute(experts_stream_kernel<kW, kBf, kDown, kTokens>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kShared));
    }
    const long long limit = wait_limit.load();
    const Waits waits = {limit > 0 ? limit : kDefaultWaitLimitCycles, wait_skip.load()};
    return e != cudaSuccess
               ? e
               : launch_chained(experts_stream_kernel<kW, kBf, kDown, kTokens>, dim3(sm_count), dim3(kThreads), kShared, stream, 1u, p, map, waits);
}

template <Weights kW, bool kBf, int kTokens>
cudaError_t launch_both(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    const cudaError_t e = launch_one<kW, kBf, false, kTokens>(p, sm_count, stream);
    return e != cudaSuccess ? e : launch_one<kW, kBf, true, kTokens>(p, sm_count, stream);
}

template <Weights kW, bool kBf>
cudaError_t launch_tokens(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    return p.tokens <= 8    ? launch_both<kW, kBf, 1>(p, sm_count, stream)
           : p.tokens <= 16 ? launch_both<kW, kBf, 2>(p, sm_count, stream)
           : p.tokens <= 32 ? launch_both<kW, kBf, 4>(p, sm_count, stream)
                            : launch_both<kW, kBf, 8>(p, sm_count, stream);
}

}  // namespace

// K-contiguous rows on 16-byte boundaries; the tokens may begin anywhere.  Sizes whose counts of rows, tiles and steps 32 bits hold: 148 x 2^22
// rows, 1024 experts x 2^22 / 16 tiles (and a round or eight more).
bool experts_stream_takes(const ExpertsParams &p)
{
    if (p.hidden > 1 << 22 || p.ffn > 1 << 22) {
        return false;
    }
    const long long elem = p.w_dtype == KUDNN_B200_E4M3 ? 1 : 2;
    auto rows = [&](const void *w, long long se, long long sn, long long sk, long long depth) {
        return (sk == 1 || depth == 1) && (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && se * elem % 16 == 0 && sn * elem % 16 == 0 && sn > 0 &&
               (se > 0 || p.experts == 1) && se < 1ll << 38 && sn < 1ll << 38;
    };
    return rows(p.gate_up, p.gu_se, p.gu_sn, p.gu_sk, p.hidden) && rows(p.down, p.d_se, p.d_sn, p.d_sk, p.ffn);
}

void experts_set_wait(long long limit_cycles, int skip_step)
{
    wait_limit.store(limit_cycles);
    wait_skip.store(skip_step);
}

cudaError_t experts_take_status(DeviceStatus *status)
{
    cudaError_t e = cudaMemcpyFromSymbol(status, experts_status, sizeof(DeviceStatus));
    if (e == cudaSuccess && status->code != kErrNone) {
        const DeviceStatus none = {};
        e = cudaMemcpyToSymbol(experts_status, &none, sizeof(DeviceStatus));
    }
    return e;
}

cudaError_t launch_experts_stream(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    const bool bf = p.x_dtype == KUDNN_B200_BF16;
    if (p.w_dtype == KUDNN_B200_E4M3) {
        return bf ? launch_tokens<kE4m3, true>(p, sm_count, stream) : launch_tokens<kE4m3, false>(p, sm_count, stream);
    }
    return bf ? launch_tokens<kBf16, true>(p, sm_count, stream) : launch_tokens<kF16, false>(p, sm_count, stream);
}

}  // namespace kb
