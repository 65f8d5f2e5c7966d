// The block of experts for few tokens in two kernels that stream the weights once (experts.cuh).
//
// What bounds it is reading the chosen experts' weights; everything here serves to keep as many bytes in flight as HBM wants, without pauses:
//   * Both products are cut by weight rows: the rows (gate and up rows in pairs) of all chosen experts are dealt out evenly, one CTA of 8 to 16
//     warps per SM or two of 8.  No atomics; sums are added in a fixed order, so that the same call gives the same bits.
//   * The warps stream on their own.  First kernel: tiles of up to 16 pairs of rows go to warps, or to groups of warps that take turns along K
//     and add up at the end of a tile (plan_tiles).  Second kernel: the CTA's rows times all experts' steps along K are dealt out to the
//     warps; each keeps sums of y of its own, added up once at the end.  Where a CTA would have 16 rows or fewer, two CTAs of a cluster
//     share twice as many, half of the steps each.
//   * A step of a warp is 128 bytes of up to 32 rows, up to four TMA boxes of eight rows, and as much of the first eight tokens' rows, into a ring
//     of the warp's own, of as many steps as shared memory has room for (launch_one).  Rows and columns beyond the matrix come as zeros, rows
//     beyond the tile are another warp's (their products are dropped).  Copies by every lane (cp.async) or loads into registers took three to
//     five times the instructions of the products and were bound by their latency; tokens loaded one step ahead were bound by L2's latency.
//   * 16 bytes per lane, as they lie in the ring, are operand fragments of mma.m16n8k16 with a permuted k: weights on the side of 16 rows, tokens on
//     that of 8, read in the same permutation.
//   * The second kernel's CTAs take the place of the first one's as those leave, or stand beside them where two fit an SM: they make their lists, fill
//     their rings with weights, and wait only before they read h.
// 1 token, 8 experts 4096 x 2048 of bf16: 74 to 78 us, 5.2 to 5.5 TB/s; 64 tokens, 120 experts 2048 x 768: 261 to 270 us, 4.2 to 4.4 TB/s; 14 tokens, 50
// experts 4096 x 2048 of e4m3: 307 to 320 us, 4 TB/s.  What is left is latency: of the instructions of a step (1 of 4 issue slots busy with 8 warps), of
// the next step's copies where a ring has one step only, and 5 us of start.
// h is kept as the tensor cores take it without loss: two bf16 halves (of bf16 and e4m3 weights), or fp32 that the second kernel splits into two
// tf32 halves (of fp16 weights: halves of fp16 would overflow beyond 65504 and lose small values).
#include "experts.cuh"
#include "sm100_ptx.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

namespace kb {

namespace {

namespace cg = cooperative_groups;

constexpr int kRows = 32;                  // of a tile of weights; a step has 128 bytes of each
constexpr int kMostTilePairs = kRows / 2;  // of a gate's and an up's row
constexpr int kBoxRows = 8;
constexpr int kBoxBytes = kBoxRows * 128;
constexpr int kStageBytes = kRows * 128;
constexpr int kMostStages = 8;
constexpr int kPad = 128;  // h's rows are multiples of this many elements, zeros behind the last one

enum Weights { kBf16, kF16, kE4m3 };

// Warps of a CTA for experts of up to 8 kTokens tokens.  e4m3 weights take four instructions for every two to become bf16: with two warps per
// scheduler their latency is the bound (16 tokens, 50 experts 4096 x 2048: 375 us), so as many as their registers leave room for.
template <Weights kW, int kTokens>
constexpr int kWarpsOf = kW != kE4m3 || kTokens > 2 ? 8 : kTokens == 2 ? 12 : 16;

// Waits that gave up, on this device: how many lanes had one, ever, and which was the last.  Nothing takes it back, so that no look at it takes
// another's report away (see experts_api.cu).
__device__ DeviceStatus experts_status;
__device__ unsigned experts_gave_up;

struct Waits {
    long long limit;  // in cycles
    int skip_step;    // test hook: from which step of K on no weights are copied, -1 off
};
std::atomic<long long> wait_limit{0};
std::atomic<int> wait_skip{-1};

// Shared memory of a launch: [ring of weights][ring of tokens][sums][lists]
struct Shape {
    int stages;
    int token_rows;   // of a stage: as many as an expert has, at most eight
    int token_bytes;  // of a stage
    int cluster;      // CTAs that share rows of y
};

// Which tokens the experts have: pairs in order of experts and tokens.
struct Lists {
    unsigned long long *tokens;  // of each expert; bit t: token t is the expert's
    short *start;                // of its pairs
    short *expert;               // the active experts; what follows is by their rank
    short *first;
    short *count;
    unsigned char *token;        // of each pair
    float *p;
    int *ids;                    // as given, and the weights
    float *given;
    // first kernel: how many warps share a tile, how many tiles an expert's rows are cut into, of at least tile_pairs pairs of rows, the first
    // `longer` of one more
    int &active, &group_warps, &tiles, &tile_pairs, &longer;
    static constexpr int kCounts = 32;
    static constexpr __host__ __device__ __forceinline__ int bytes(int experts, int pairs)
    {
        return kCounts + experts * 16 + (pairs * 13 + 15) / 16 * 16;
    }
    __device__ __forceinline__ Lists(unsigned char *at, int experts, int pairs)
        : tokens(reinterpret_cast<unsigned long long *>(at + kCounts)),
          start(reinterpret_cast<short *>(at + kCounts + experts * 8)),
          expert(start + experts),
          first(expert + experts),
          count(first + experts),
          token(at + kCounts + experts * 16 + pairs * 12),
          p(reinterpret_cast<float *>(at + kCounts + experts * 16)),
          ids(reinterpret_cast<int *>(p + pairs)),
          given(p + 2 * pairs),
          active(reinterpret_cast<int *>(at)[0]),
          group_warps(reinterpret_cast<int *>(at)[1]),
          tiles(reinterpret_cast<int *>(at)[2]),
          tile_pairs(reinterpret_cast<int *>(at)[3]),
          longer(reinterpret_cast<int *>(at)[4])
    {
    }
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

// 16 bytes multiples from global to shared memory, on 16-byte boundaries both
__device__ __forceinline__ void bulk_copy(void *to, const void *from, int bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
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

// The value's upper tf32 half and what is left; a value that is not finite has no rest.
__device__ __forceinline__ float2 split_tf32(float v)
{
    const float hi = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
    return isfinite(v) ? make_float2(hi, v - hi) : make_float2(v, 0.0f);
}

// h in the workspace, a row per pair in the lists' order: bf16 upper halves, then lower ones, or fp32.
__host__ __device__ __forceinline__ long long h_pitch(int ffn)
{
    return static_cast<long long>((ffn + kPad - 1) / kPad) * kPad;
}

// A warp's way through the weights, piece by piece: steps of K of a tile of one expert's rows.  32 bits hold every count (see the launcher).
template <bool kDown, int kWarps>
struct Cursor {
    int rank, row, rows;       // the expert, its first row (of the gate, or of down), how many
    int step, steps, stride;   // of K
    int depth;                 // steps of an expert
    int at, end;               // up: tiles of all active experts, one after the other; down: rows of y
    int offset;                // up: of the warp in its group
    int begin, until, begin_rank, position;  // down: the warp's steps of all experts, one after the other
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
    // Down: the steps of all experts at the same rows are dealt out to the warps, as many to each.
    __device__ __forceinline__ void start_down(const ExpertsParams &p, const Lists &l, int warp, int depth_steps, int cluster)
    {
        const unsigned shares = gridDim.x / cluster, share = blockIdx.x / cluster;
        at = static_cast<int>(static_cast<unsigned>(p.hidden) * share / shares);
        end = static_cast<int>(static_cast<unsigned>(p.hidden) * (share + 1) / shares);
        depth = depth_steps;
        stride = 1;
        const int warps = kWarps * cluster, number = blockIdx.x % cluster * kWarps + warp, all = l.active * depth;
        begin = all / warps * number + min(number, all % warps);
        until = begin + all / warps + (number < all % warps ? 1 : 0);
        begin_rank = begin / depth;
        rows = 0;
        position = until;
    }
    // true while the warp has steps at the present rows
    __device__ __forceinline__ bool next_down()
    {
        if (position >= until) {
            return false;
        }
        ++rank;
        step = position - rank * depth;
        steps = min(depth - step, until - position);
        position += steps;
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
// as many tiles as that has room for.  What a round costs: the bytes of the SM's tiles at its share of HBM's rate (23 a cycle), or the steps of a
// warp at what one takes in latency where HBM waits (800 cycles), and the sums of a group, which its stream does not outlast (64 tokens, 120
// experts 2048 x 768, first kernel: 134 us with tiles per warp, 144, 197 and 178 for groups of 2, 4 and 8).  The rate is that of one CTA per SM:
// where two share an SM the bytes count for half of what they take.
template <int kWarps>
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
    float cost = static_cast<float>(rounds) * (fmaxf(bytes / 23.0f, 800.0f * steps) + (w > 1 ? 3000.0f : 500.0f));
    if (kWarps % w != 0) {
        cost = 3e38f;
    }
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
template <bool kPlan, int kWarps>
__device__ __forceinline__ void make_lists(Lists &l, const ExpertsParams &p, int depth_steps)
{
    constexpr int kThreads = kWarps * 32;
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
            plan_tiles<kWarps>(l, active, p.ffn, depth_steps, tid);
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
__global__ void __launch_bounds__(kWarpsOf<kW, kTokens> * 32, kTokens == 1 && kW != kE4m3 ? 2 : 1)
    experts_stream_kernel(const __grid_constant__ ExpertsParams p, const __grid_constant__ CUtensorMap map, const __grid_constant__ Shape shape,
                          const __grid_constant__ Waits waits)
{
    constexpr int kWarps = kWarpsOf<kW, kTokens>, kThreads = kWarps * 32;
    constexpr int kElem = kW == kE4m3 ? 1 : 2;
    constexpr int kStep = 128 / kElem;                // of K
    constexpr int kPiece = 16 / kElem;                // of a lane, twice in a step
    constexpr bool kTf32 = kDown && kW == kF16;       // h in fp32, products of tf32
    constexpr bool kBfMma = kW == kBf16 || (kW == kE4m3 && (kBf || kDown));
    constexpr int kPlanes = kDown && !kTf32 ? 2 : 1;  // of the tokens' rows
    constexpr int kTokenElem = kTf32 ? 4 : 2;
    constexpr int kTokenRow = kStep * kTokenElem;     // bytes of a token's row in a step
    constexpr int kTokenPitch = kTokenRow + 64;       // two rows of 128 bytes lie in different banks then, of 256 bytes in the same
    constexpr int kLoads = kPiece * kTokenElem / 16;  // 16-byte pieces of a lane's fragment
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t barriers[kWarps][kMostStages];
    __shared__ int abort_word;
    unsigned char *shared = raw + (1024u - (smem_u32(raw) & 1023u)) % 1024u;
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int stages = shape.stages;
    unsigned char *ring = shared + warp * stages * kStageBytes;
    unsigned char *token_ring = shared + kWarps * stages * kStageBytes + warp * stages * shape.token_bytes;
    unsigned char *behind = shared + kWarps * stages * (kStageBytes + shape.token_bytes);
    float4 *sums = reinterpret_cast<float4 *>(behind);  // up: [kWarps][2][32]
    float *y_sums = reinterpret_cast<float *>(behind);  // down: [kWarps][tokens][kRows]
    Lists lists(behind + (kDown ? kWarps * p.tokens * kRows * 4 : kWarps * 1024), p.experts, p.tokens * p.top);
    const int depth = kDown ? p.ffn : p.hidden;  // K
    const int depth_steps = (depth + kStep - 1) / kStep;
    uint64_t *full = barriers[warp];  // a barrier per stage of the warp's ring
    volatile int *abort_flag = &abort_word;
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
        abort_word = 0;
    }
    if (lane < stages) {
        mbar_init(full + lane, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    for (int e = tid; e < p.experts; e += kThreads) {
        lists.tokens[e] = 0ull;
    }
    if (kDown) {
        for (int i = tid; i < kWarps * p.tokens * kRows; i += kThreads) {
            y_sums[i] = 0.0f;
        }
    }
    __syncthreads();
    if (!kDown) {
        pdl_wait();
        pdl_launch_dependents();  // behind the wait: what the second kernel reads ahead of its own is older than this one
    }
    make_lists<!kDown, kWarps>(lists, p, depth_steps);
    using Place = Cursor<kDown, kWarps>;
    auto start = [&](Place &c) {
        if (kDown) {
            c.start_down(p, lists, warp, depth_steps, shape.cluster);
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

    // ---- the stream: lane i < 4 brings eight rows of weights (up: of the gate, of the up, and the next eight of both), lane 8 + 8 plane + i the
    // row of an expert's i-th token, where those lie on 16-byte boundaries
    const long long pitch = h_pitch(p.ffn);
    const long long plane_step = static_cast<long long>(p.tokens) * p.top * pitch;
    const bool staged = kDown || ((reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && p.x_ld % 8 == 0);
    // the row of x or h of a pair, in bytes
    auto token_row = [&](int pair, int plane) -> const unsigned char * {
        if (kDown) {
            return static_cast<const unsigned char *>(p.h) + (pair * pitch + plane * plane_step) * kTokenElem;
        }
        return static_cast<const unsigned char *>(p.x) + lists.token[pair] * p.x_ld * kTokenElem;
    };
    const int copy_plane = (lane - 8) >> 3, copy_row = lane & 7;
    unsigned char *const copy_to = token_ring + (copy_plane * shape.token_rows + copy_row) * kTokenPitch;
    const unsigned char *copy_from = nullptr;
    bool copies = false;
    int box_row = 0, boxes = 0, token_copies = 0;
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
            const int rows = min(static_cast<int>(lists.count[ahead.rank]), 8);
            token_copies = staged ? rows * kPlanes : 0;
            copies = staged && lane >= 8 && copy_plane < kPlanes && copy_row < rows;
            copy_from = token_row(lists.first[ahead.rank] + min(copy_row, rows - 1), copies ? copy_plane : 0);
        }
    };
    aim();
    bool gave_up = false;
    // weights: those of the step; tokens: theirs
    auto copy_weights = [&](int stage, int k) {
        if (lane < boxes && (waits.skip_step < 0 || k / kStep < waits.skip_step)) {
            tma_load_3d(ring + stage * kStageBytes + lane * kBoxBytes, &map, full + stage, k, box_row, ahead_expert);
        }
    };
    auto copy_tokens = [&](int stage, int k, int bytes) {
        if (copies && bytes > 0) {
            bulk_copy(copy_to + stage * shape.token_bytes, copy_from + static_cast<long long>(k) * kTokenElem, bytes, full + stage);
        }
    };
    // h's rows are whole; of x's last step the whole 16 bytes
    auto token_bytes = [&](int k) { return kDown ? kTokenRow : min(kTokenRow, (depth - k) / 8 * 16); };
    auto issue = [&]() {
        if (ahead_left > 0) {
            const int bytes = token_bytes(ahead_k);
            if (!gave_up) {
                if (lane == 0) {
                    mbar_expect_tx(full + ahead_stage, boxes * kBoxBytes + token_copies * bytes);
                }
                copy_weights(ahead_stage, ahead_k);
                copy_tokens(ahead_stage, ahead_k, bytes);
            }
            ahead_k += ahead.stride * kStep;
            ahead_stage = ahead_stage + 1 == stages ? 0 : ahead_stage + 1;
            if (--ahead_left == 0) {
                aim();
            }
        }
    };
    if (kDown) {
        // the first round's weights, ahead of the wait for h, whose rows follow
        const Place from = ahead;
        const int from_k = ahead_k, from_left = ahead_left, from_expert = ahead_expert, from_boxes = boxes, from_row = box_row, from_copies = token_copies;
        const unsigned char *from_copy = copy_from;
        const bool from_any = copies;
#pragma unroll 1
        for (int i = 0; i < stages && ahead_left > 0; ++i) {
            if (lane == 0) {
                mbar_expect_tx(full + i, boxes * kBoxBytes + token_copies * kTokenRow);
            }
            copy_weights(i, ahead_k);
            ahead_k += ahead.stride * kStep;
            if (--ahead_left == 0) {
                aim();
            }
        }
        pdl_wait();
        pdl_launch_dependents();
        ahead = from;
        ahead_k = from_k;
        ahead_left = from_left;
        ahead_expert = from_expert;
        boxes = from_boxes;
        box_row = from_row;
        token_copies = from_copies;
        copy_from = from_copy;
        copies = from_any;
#pragma unroll 1
        for (int i = 0; i < stages && ahead_left > 0; ++i) {
            copy_tokens(i, ahead_k, kTokenRow);
            ahead_k += ahead.stride * kStep;
            ahead_stage = ahead_stage + 1 == stages ? 0 : ahead_stage + 1;
            if (--ahead_left == 0) {
                aim();
            }
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < stages; ++i) {
            issue();
        }
    }

    // ---- the products
    struct Tokens {
        uint4 q[2][kPlanes][kLoads];  // [which 64 bytes of weights]
    };
    // the fragments of tokens that do not come through the ring; whole: all of the step's elements exist, on 16-byte boundaries
    auto load_tokens = [&](Tokens &b, int pair, int k, bool whole) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int from_k = k + u * 4 * kPiece;
#pragma unroll
            for (int plane = 0; plane < kPlanes; ++plane) {
                const unsigned char *from = token_row(pair, plane) + static_cast<long long>(from_k) * kTokenElem;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    if (kDown || whole) {
                        b.q[u][plane][i] = reinterpret_cast<const uint4 *>(from)[i];
                    } else {
                        b.q[u][plane][i] = load_some(reinterpret_cast<const unsigned short *>(from) + i * 8, depth - from_k - i * 8);
                    }
                }
            }
        }
    };
    const float *scale = kDown ? p.down_scale : p.gate_up_scale;
    const long long ss_e = kDown ? p.ds_se : p.gus_se, ss_n = kDown ? p.ds_sn : p.gus_sn, ss_k = kDown ? p.ds_sk : p.gus_sk;
    // where this lane's fragments of row g lie: chunks t and t + 4, which the copies put in place t ^ g and so on
    const unsigned char *fragment = ring + g * 128 + (t ^ g) * 16;
    const int other = (g & 4) != 0 ? -64 : 64;
    int stage = 0;
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
        const float *scale_at[4];
        if (kW == kE4m3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // rows g + 8 i, or g and g of the up, then 8 on
                const int r = min(kDown ? i * 8 + g : (i >> 1) * 8 + g, now.rows - 1);
                scale_at[i] = scale + lists.expert[now.rank] * ss_e + (now.row + r + (!kDown && (i & 1) != 0 ? p.ffn : 0)) / 128 * ss_n;
            }
        }
        const unsigned char *token_fragment = token_ring + min(g, count - 1) * kTokenPitch + t * 16 * kLoads;
        int step = now.step;
#pragma unroll 1
        for (int s = 0; s < now.steps; ++s, step += now.stride) {
            float of_block[4];
            if (kW == kE4m3) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    of_block[i] = scale_at[i][step * ss_k];
                }
            }
            gave_up = gave_up || !mbar_wait(full + stage, parity, abort_flag, &experts_status, kDown ? 2 : 1, waits.limit);
            const int k = step * kStep + t * kPiece;
            const bool whole = kDown || (staged && (step + 1) * kStep <= depth);
            if (!kDown && staged && !whole) {
                // x's last step: the elements behind the last whole 16 bytes, which the copy did not bring, and zeros behind the last one
                const int left = depth - step * kStep, copied = left & ~7;
#pragma unroll 1
                for (int i = lane; i < min(count, 8) * kStep; i += 32) {
                    const int row = i / kStep, column = i % kStep;
                    if (column >= copied) {
                        const unsigned short *from = reinterpret_cast<const unsigned short *>(token_row(first + row, 0)) + step * kStep + column;
                        reinterpret_cast<unsigned short *>(token_ring + stage * shape.token_bytes + row * kTokenPitch)[column] = column < left ? *from : 0;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            uint4 a[2][4];  // [which 64 bytes][row g + 8 i of the tile's 32]
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned char *at = fragment + stage * kStageBytes + r * 1024;
                a[0][r] = *reinterpret_cast<const uint4 *>(at);
                a[1][r] = *reinterpret_cast<const uint4 *>(at + other);
            }
            Tokens b0;
            if (staged) {
                const unsigned char *at = token_fragment + stage * shape.token_bytes;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int plane = 0; plane < kPlanes; ++plane) {
#pragma unroll
                        for (int i = 0; i < kLoads; ++i) {
                            b0.q[u][plane][i] =
                                reinterpret_cast<const uint4 *>(at + plane * shape.token_rows * kTokenPitch + u * 64 * kLoads)[i];
                        }
                    }
                }
            } else {
                load_tokens(b0, first + min(g, count - 1), k, false);
            }
            __syncwarp();
            issue();  // into the stage that has just been read
            if (++stage == stages) {
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
            // sums of the tokens `b`, in chains in turn: the matrix instructions of one wait for one another.  part: of e4m3 weights this step's,
            // for the scale; of others the products of h's lower half, which count only where they are finite: with an infinite weight the upper
            // half has the infinity, and the lower one, which may be zero or of the other sign, must not make it NaN.
            auto add = [&](float(&sum)[2][4], const Tokens &b) {
                constexpr bool kApart = kDown && kW != kE4m3;
                float part[2][4];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    part[m][0] = part[m][1] = part[m][2] = part[m][3] = 0.0f;
                }
                float(&to)[2][4] = kW == kE4m3 ? part : sum;
                float(&lower)[2][4] = kApart ? part : to;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (kTf32) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint4 &q = b.q[u][0][j / 2 % kLoads];
                            const float2 b0 = split_tf32(__uint_as_float(word(q, j % 2 * 2)));
                            const float2 b1 = split_tf32(__uint_as_float(word(q, j % 2 * 2 + 1)));
                            float2 f[4];
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const uint32_t w = word(a[u][r], j);
                                f[r] = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                            }
                            mma_tf32(lower[0], f[0].x, f[1].x, f[0].y, f[1].y, b0.y, b1.y);
                            mma_tf32(lower[1], f[2].x, f[3].x, f[2].y, f[3].y, b0.y, b1.y);
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
                                    mma_16<kBfMma>(plane > 0 ? lower[m] : to[m], w[m][0], w[m][1], w[m][2], w[m][3], word(q, j % 2 * 2), word(q, j % 2 * 2 + 1));
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
                if (kApart) {
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            sum[m][i] += isfinite(part[m][i]) ? part[m][i] : 0.0f;
                        }
                    }
                }
            };
            add(c[0], b0);
#pragma unroll
            for (int n = 1; n < kN; ++n) {
                Tokens b;
                load_tokens(b, first + min(n * 8 + g, count - 1), k, whole);
                add(c[n], b);
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
        auto put = [&](long long to, float v) {
            if (kW == kF16) {
                static_cast<float *>(p.h)[to] = v;
            } else {
                // next to fp32's largest value the upper half is cut, not rounded, which would make it infinite; the rest is rounded either way
                const float nearest = bf16_bits_to_f32(f32_to_bf16_rne_bits(v));
                const float hi = isfinite(v) && !isfinite(nearest) ? __uint_as_float(__float_as_uint(v) & 0xffff0000u) : nearest;
                unsigned short *planes = static_cast<unsigned short *>(p.h);
                planes[to] = f32_to_bf16_rne_bits(hi);
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
                                    put((first + column) * pitch + now.row + r, expert_gate(c[n][m][j], c[n][m][2 + j]));
                                }
                            }
                        }
                    } else {
                        // the group's sums, eight tokens at a time
                        const int group = warp / group_warps, threads = group_warps * 32;
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            sums[warp * 64 + m * 32 + lane] = make_float4(c[n][m][0], c[n][m][1], c[n][m][2], c[n][m][3]);
                        }
                        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads) : "memory");
                        const float *from = reinterpret_cast<const float *>(sums + group * group_warps * 64);
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
                                put((first + column) * pitch + now.row + r, expert_gate(gate, up));
                            }
                        }
                        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads) : "memory");
                    }
                }
                if (now.row + now.rows == p.ffn && now.offset == 0) {
                    const int some = static_cast<int>(pitch) - p.ffn;
                    for (int i = lane; i < some * count; i += 32) {
                        put((first + i / some) * pitch + p.ffn + i % some, 0.0f);
                    }
                }
            });
        }
    } else {
        cg::cluster_group cluster = cg::this_cluster();
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
            if (shape.cluster > 1) {
                cluster.sync();
            } else {
                __syncthreads();
            }
            // the CTAs of a cluster take turns at the results, all add in the same order
            const int items = p.tokens * kRows;
            for (int i = tid * shape.cluster + static_cast<int>(blockIdx.x) % shape.cluster; i < items; i += kThreads * shape.cluster) {
                float y = 0.0f;
                for (int cta = 0; cta < shape.cluster; ++cta) {
                    const float *from = shape.cluster > 1 ? cluster.map_shared_rank(y_sums, cta) : y_sums;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        y += from[w * items + i];
                    }
                }
                const int token = i / kRows, r = i % kRows;
                if (r < now.rows) {
                    store_exact(p.y, p.x_dtype, token * p.y_ld + now.row + r, round_rne(y, p.x_dtype));
                }
            }
            if (shape.cluster > 1) {
                cluster.sync();
            } else {
                __syncthreads();
            }
            if (now.row + now.rows < now.end) {
                for (int i = tid; i < kWarps * items; i += kThreads) {
                    y_sums[i] = 0.0f;
                }
                __syncthreads();
            }
        }
    }
    if (gave_up) {
        experts_status.where = kDown ? 2 : 1;
        experts_status.block = static_cast<int>(blockIdx.x);
        __threadfence();
        atomicAdd(&experts_gave_up, 1u);  // every lane: some may have been there in time
        // the copies that are still on their way, each for a moment
        for (int i = 0; i < stages; ++i) {
            for (int spin = 0; spin < 2000 && !mbar_try_wait(full + i, parity ^ (i < stage ? 1u : 0u)); ++spin) {
            }
        }
    }
}

constexpr int kMostShared = 227 * 1024 - 2048;            // of a CTA, beside its static part
constexpr int kHalfShared = (228 * 1024) / 2 - 2 * 1024;  // where two CTAs are to fit

template <Weights kW, bool kBf, bool kDown, int kTokens>
cudaError_t launch_one(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    constexpr int kWarps = kWarpsOf<kW, kTokens>, kStep = kW == kE4m3 ? 128 : 64;
    constexpr int kTokenPitch = kStep * (kDown && kW == kF16 ? 4 : 2) + 64;
    Shape shape;
    shape.token_rows = std::min(8, p.tokens);
    shape.token_bytes = shape.token_rows * (kDown && kW != kF16 ? 2 : 1) * kTokenPitch;
    // Two CTAs fit an SM where the registers suffice and half of its shared memory holds the rings.  With much to read both are this kernel's: 16
    // warps hide the latency of their instructions better than 8 (1 token, 8 experts 4096 x 2048: 77 us, with 8 warps 86).  With little, the second
    // place is the next kernel's, which is then set up while this one runs (2 experts 1024 x 704: 12.5 us, otherwise 14.9).
    constexpr bool kHalves = kTokens == 1 && kW != kE4m3;
    const long long most = 6ll * std::min(p.experts, p.tokens * p.top) * p.hidden * p.ffn;  // bytes of the experts that can be chosen
    const int stage = kWarps * (kStageBytes + shape.token_bytes);
    const int fixed = 1024 + (kDown ? kWarps * p.tokens * kRows * 4 : kWarps * 1024) + Lists::bytes(p.experts, p.tokens * p.top);
    // A ring of one step at least, whatever the call (a kernel without a ring would wait for copies that nobody makes)
    constexpr int kMostFixed = 1024 + kWarps * (kDown ? 8 * kTokens * kRows * 4 : 1024) + Lists::bytes(kMostExperts, 8 * kTokens * kMostExpertTop);
    constexpr int kMostStage = kWarps * (kStageBytes + 8 * (kDown && kW != kF16 ? 2 : 1) * kTokenPitch);
    static_assert(8 * kTokens <= kMostExpertTokens && kMostFixed + kMostStage <= kMostShared, "shared memory holds no ring");
    const int in_half = kHalves ? (kHalfShared - fixed) / stage : 0;
    const bool two = most > 64ll << 20 && in_half >= 2;
    const int ctas = two ? 2 * sm_count : sm_count;
    shape.cluster = kDown && p.hidden <= 16 * ctas ? 2 : 1;
    // For 64 experts: 2 to 4 steps of 16-bit weights; of e4m3 weights, with more warps and tokens' rows of 256 bytes, 2, but 1 for 8 tokens and in the
    // second kernel for 5 to 16, and 2 to 4 from 17 on
    shape.stages = std::min(two || in_half >= 3 ? in_half : (kMostShared - fixed) / stage, kMostStages);
    const size_t shared = static_cast<size_t>(fixed) + static_cast<size_t>(shape.stages) * stage;
    alignas(64) CUtensorMap map;
    cudaError_t e = tc_encode_groups(&map, kDown ? p.down : p.gate_up, p.w_dtype, p.experts, kDown ? p.hidden : 2ll * p.ffn, kDown ? p.ffn : p.hidden,
                                     std::max(kDown ? p.d_se : p.gu_se, 16ll), kDown ? p.d_sn : p.gu_sn, kBoxRows);
    if (e == cudaSuccess) {
        e = cudaFuncSetAttribute(experts_stream_kernel<kW, kBf, kDown, kTokens>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    }
    const long long limit = wait_limit.load();
    const Waits waits = {limit > 0 ? limit : kDefaultWaitLimitCycles, wait_skip.load()};
    return e != cudaSuccess ? e
                            : launch_chained(experts_stream_kernel<kW, kBf, kDown, kTokens>, dim3(ctas / shape.cluster * shape.cluster), dim3(kWarps * 32),
                                             shared, stream, shape.cluster, p, map, shape, waits);
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

// K-contiguous rows on 16-byte boundaries; the tokens may begin anywhere.  Sizes whose counts of rows, tiles and steps 32 bits hold: 2^22 rows x
// 296 CTAs, 1024 experts x 2^22 / 16 tiles (and a round or eight more).
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

cudaError_t experts_status_of(unsigned *gave_up, DeviceStatus *last)
{
    const cudaError_t e = cudaMemcpyFromSymbol(gave_up, experts_gave_up, sizeof(unsigned));
    return e == cudaSuccess ? cudaMemcpyFromSymbol(last, experts_status, sizeof(DeviceStatus)) : e;
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
