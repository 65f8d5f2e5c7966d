// The block of experts for few tokens in two kernels that stream the weights once (experts.cuh).
//
// What bounds it is reading the chosen experts' weights; everything here serves to keep as many bytes in flight as HBM wants, without pauses:
//   * Both products are cut by weight rows alone: the rows (gate and up rows in pairs) of all chosen experts are dealt out evenly, one CTA per SM,
//     so that every SM streams the same number of bytes; nothing is added up across CTAs, no atomics, and the same call gives the same bits.
//   * The 16 warps of a CTA stream on their own, without barriers.  First kernel: as many groups of warps as the CTA has tiles of rows, up to 16;
//     a group's warps split K and add up at the end of a tile (with a tile per warp, what large batches have, nothing is added up).  Second
//     kernel: each warp a sixteenth of all steps of all experts at the CTA's rows, with sums of y of its own, added up at the end.
//   * Every lane copies its own 16 bytes of a few rows into a ring in shared memory (cp.async, some steps ahead) and reads back only what it
//     copied itself.  Copies of what lies beyond the last row or column bring zeros.
//   * The lanes' pieces are, as they are, operand fragments of mma.m16n8k16 with a permuted k: weights on the side of 16 rows, tokens on that of 8;
//     four neighbouring lanes hold 64 neighbouring bytes of a row.  The tokens' fragments are read from L1 and L2 in the same permutation.
//   * The second kernel starts its copies of `down` while the first one ends (its CTAs take the place of the first one's as those leave) and
//     waits only before it reads h.
// h is kept as the tensor cores take it without loss: two bf16 halves (of bf16 and e4m3 weights), or fp32 that the second kernel splits into two
// tf32 halves (of fp16 weights: halves of fp16 would overflow beyond 65504 and lose small values).
#include "experts.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostPairs = kMostExpertTokens * kMostExpertTop;

enum Weights { kBf16, kF16, kE4m3 };

// Which tokens the experts have: pairs in order of experts and tokens.
struct Lists {
    unsigned long long tokens[kMostExperts];  // bit t: token t is the expert's
    short start[kMostExperts];                // of its pairs
    short expert[kMostExperts];               // the active experts; what follows is by their rank
    short first[kMostExperts];
    short count[kMostExperts];
    unsigned char token[kMostPairs];
    float p[kMostPairs];
    int ids[kMostPairs];
    int active;
};

// All threads of the CTA.  An id that a token names twice counts once, with both weights.
__device__ __forceinline__ void make_lists(Lists &l, const ExpertsParams &p)
{
    const int pairs = p.tokens * p.top, tid = static_cast<int>(threadIdx.x);
    for (int e = tid; e < p.experts; e += kThreads) {
        l.tokens[e] = 0ull;
    }
    for (int i = tid; i < pairs; i += kThreads) {
        l.ids[i] = p.ids[i];
    }
    __syncthreads();
    for (int i = tid; i < pairs; i += kThreads) {
        const int e = l.ids[i];
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
                sum += same ? p.p[j] : 0.0f;
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

__device__ __forceinline__ void copy_16(uint32_t to, const void *from, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

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

// 8 values of 16 bits from `at`, of which `left` exist, mostly all or (lanes without a token) none; vector: `at` is on a 16-byte boundary
__device__ __forceinline__ uint4 load_8(const unsigned short *at, int left, bool vector)
{
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (vector && left >= 8) {
        q = *reinterpret_cast<const uint4 *>(at);
    } else if (left > 0) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = 2 * i < left ? at[2 * i] : 0u, hi = 2 * i + 1 < left ? at[2 * i + 1] : 0u;
            w[i] = lo | hi << 16;
        }
        q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return q;
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

// A tile has 16 rows of weights, a step 128 bytes of each.
constexpr int kRows = 16;
constexpr int kStageBytes = kRows * 128;

// The kernels for experts of up to 8 kTokens tokens: the ring, and behind it the warps' sums.
template <bool kDown, int kTokens>
struct Layout {
    static constexpr int kTileRows = kDown ? kRows : kRows / 2;  // rows of y, or pairs of a gate's and an up's row
    static constexpr int kStages = kTokens == 8 ? 4 : 5;
    static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
    // up: the sums of 8 tokens of every warp, in two buffers; down: each warp's sums of y
    static constexpr int kSumBytes = kDown ? kWarps * 8 * kTokens * kRows * 4 : 2 * kWarps * 512;
    static constexpr size_t kBytes = kRingBytes + kSumBytes + sizeof(Lists);
};

// A warp's way through the weights, piece by piece: steps of K of up to kTileRows rows of one expert.
template <bool kDown, int kTileRows>
struct Cursor {
    int rank, row, rows;       // the expert, its first row (of the gate, or of down), how many
    int step, steps, stride;   // of K
    long long at, end;         // up: pairs of rows of all active experts, one after the other; down: rows of y
    long long begin, until, position;  // down: the warp's steps of all experts at the same rows
    int depth;                 // steps of an expert
    int offset;                // up: of the warp in its group
    __device__ __forceinline__ void start_up(const ExpertsParams &p, const Lists &l, int warp, int group_warps, int depth_steps)
    {
        const long long all = static_cast<long long>(l.active) * p.ffn;
        const long long from = all * blockIdx.x / gridDim.x, to = all * (blockIdx.x + 1) / gridDim.x;
        const int groups = kWarps / group_warps, group = warp / group_warps;
        at = from + (to - from) * group / groups;
        end = from + (to - from) * (group + 1) / groups;
        offset = warp % group_warps;
        stride = group_warps;
        depth = depth_steps;
        rows = 0;
    }
    __device__ __forceinline__ bool next_up(const ExpertsParams &p)
    {
        at += rows;
        if (at >= end) {
            return false;
        }
        rank = static_cast<int>(at / p.ffn);
        row = static_cast<int>(at - static_cast<long long>(rank) * p.ffn);
        equal_tile(min(end - at, static_cast<long long>(p.ffn - row)));
        step = offset;
        steps = depth > offset ? (depth - offset + stride - 1) / stride : 0;
        return true;
    }
    __device__ __forceinline__ void start_down(const ExpertsParams &p, const Lists &l, int warp, int depth_steps)
    {
        at = static_cast<long long>(p.hidden) * blockIdx.x / gridDim.x;
        end = static_cast<long long>(p.hidden) * (blockIdx.x + 1) / gridDim.x;
        depth = depth_steps;
        const long long all = static_cast<long long>(l.active) * depth;  // at most 1024 x 2^26: 64 bits
        begin = all * warp / kWarps;
        until = all * (warp + 1) / kWarps;
        stride = 1;
        rows = 0;
        position = until;
    }
    // Down: true while the warp has pieces at the present rows.
    __device__ __forceinline__ bool next_down()
    {
        if (position >= until) {
            return false;
        }
        rank = static_cast<int>(position / depth);
        step = static_cast<int>(position - static_cast<long long>(rank) * depth);
        steps = static_cast<int>(min(until - position, static_cast<long long>(depth - step)));
        position += steps;
        return true;
    }
    __device__ __forceinline__ bool next_rows()
    {
        at += rows;
        if (at >= end) {
            return false;
        }
        row = static_cast<int>(at);
        equal_tile(end - at);
        position = begin;
        return true;
    }
    __device__ __forceinline__ void equal_tile(long long left)
    {
        const int tiles = static_cast<int>((left + kTileRows - 1) / kTileRows);
        rows = static_cast<int>((left + tiles - 1) / tiles);
    }
};

// kTokens: an expert's most, in eights.
template <Weights kW, bool kBf, bool kDown, int kTokens>
__global__ void __launch_bounds__(kThreads, 1) experts_stream_kernel(const __grid_constant__ ExpertsParams p)
{
    using L = Layout<kDown, kTokens>;
    constexpr int kStages = L::kStages;
    constexpr int kElem = kW == kE4m3 ? 1 : 2;
    constexpr int kStep = 128 / kElem;                // of K
    constexpr int kPiece = 16 / kElem;                // of a lane, twice in a step
    constexpr bool kTf32 = kDown && kW == kF16;       // h in fp32, products of tf32
    constexpr bool kBfMma = kW == kBf16 || (kW == kE4m3 && (kBf || kDown));
    extern __shared__ __align__(16) unsigned char shared[];
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    unsigned char *ring = shared + warp * kStages * kStageBytes;
    float4 *sums = reinterpret_cast<float4 *>(shared + L::kRingBytes);  // up: [2][kWarps][32]
    float *y_sums = reinterpret_cast<float *>(shared + L::kRingBytes);  // down: [kWarps][tokens][kRows]
    Lists &lists = *reinterpret_cast<Lists *>(shared + L::kRingBytes + L::kSumBytes);
    const int depth = kDown ? p.ffn : p.hidden;  // K
    const char *weights = static_cast<const char *>(kDown ? p.down : p.gate_up);
    const long long se = kDown ? p.d_se : p.gu_se, sn = kDown ? p.d_sn : p.gu_sn;

    if (!kDown) {
        pdl_wait();
        pdl_launch_dependents();  // behind the wait: what the second kernel reads ahead of its own is older than this one
    }
    make_lists(lists, p);

    // up: warps that share a tile, as few as leave no group without one
    int group_warps = 1;
    if (!kDown) {
        const long long pairs = static_cast<long long>(lists.active) * p.ffn / gridDim.x + 1;
        group_warps = kWarps;
        while (group_warps > 1 && pairs > static_cast<long long>(kWarps / group_warps) * L::kTileRows) {
            group_warps /= 2;
        }
    }

    // ---- the stream: copy i of a step brings 128 bytes of rows 4 i .. 4 i + 3, the chunk of 16 bytes in place c ^ 4 (row % 2), so that the
    // fragments are read without bank conflicts
    using Place = Cursor<kDown, L::kTileRows>;
    auto start = [&](Place &c) {
        if (kDown) {
            c.start_down(p, lists, warp, (depth + kStep - 1) / kStep);
        } else {
            c.start_up(p, lists, warp, group_warps, (depth + kStep - 1) / kStep);
        }
    };
    const int copy_row = lane >> 3, chunk = lane & 7;
    const uint32_t copy_to = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) +
                             static_cast<uint32_t>(copy_row * 128 + (chunk ^ (copy_row & 1) * 4) * 16);
    const char *row_at[4];
    int row_here = 0;  // bit i: the row of copy i exists
    int ahead_k = 0, ahead_left = 0, ahead_stage = 0;
    Place ahead;
    start(ahead);
    // the next piece with steps of its own
    auto advance = [&]() {
        do {
            if (kDown) {
                while (!ahead.next_down()) {
                    if (!ahead.next_rows() || ahead.position >= ahead.until) {
                        return;  // no rows are left, or this warp has no steps at any
                    }
                }
            } else if (!ahead.next_up(p)) {
                return;
            }
            ahead_left = ahead.steps;
        } while (ahead_left == 0);
        ahead_k = ahead.step * kStep + chunk * kPiece;
        row_here = 0;
        const char *expert = weights + lists.expert[ahead.rank] * se * kElem;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int in_tile = i * 4 + copy_row, r = kDown ? in_tile : in_tile & 7;  // up: eight of the gate, then their eight of the up
            const bool here = r < ahead.rows;
            const long long row = ahead.row + r + (!kDown && i >= 2 ? p.ffn : 0);
            row_at[i] = here ? expert + row * sn * kElem : weights;
            row_here |= here ? 1 << i : 0;
        }
    };
    advance();
    auto issue = [&]() {
        if (ahead_left > 0) {
            const int bytes = max(0, min(16, (depth - ahead_k) * kElem));
            const uint32_t to = copy_to + static_cast<uint32_t>(ahead_stage * kStageBytes);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = (row_here >> i & 1) != 0 ? bytes : 0;
                copy_16(to + i * 512, row_at[i] + (n > 0 ? static_cast<long long>(ahead_k) * kElem : 0), n);
            }
            ahead_k += ahead.stride * kStep;
            if (--ahead_left == 0) {
                advance();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead_stage = ahead_stage + 1 == kStages ? 0 : ahead_stage + 1;
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) {
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

    // ---- the products
    const long long pitch = h_pitch(p);
    const int h_rows = p.tokens * p.top;
    const unsigned short *x = static_cast<const unsigned short *>(p.x), *h = static_cast<const unsigned short *>(p.h);
    const bool vector = kDown || ((reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && p.x_ld % 8 == 0);
    const float *scale = kDown ? p.down_scale : p.gate_up_scale;
    const long long ss_e = kDown ? p.ds_se : p.gus_se, ss_n = kDown ? p.ds_sn : p.gus_sn, ss_k = kDown ? p.ds_sk : p.gus_sk;
    // where this lane's fragments of rows g and g + 8 lie: chunks t and t + 4
    const unsigned char *fragment = ring + g * 128 + (t ^ (g & 1) * 4) * 16;
    const int other = (g & 1) != 0 ? -64 : 64;
    int stage = 0, turn = 0;
    float c[kTokens][4];

    auto multiply = [&](const Place &now) {
        const int expert = lists.expert[now.rank], first = lists.first[now.rank], count = lists.count[now.rank];
        const int eights = (count + 7) / 8;
#pragma unroll
        for (int n = 0; n < kTokens; ++n) {
            c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
        }
        const float *scale_at[2];
        if (kW == kE4m3) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = min(kDown ? i * 8 + g : g, now.rows - 1);
                scale_at[i] = scale + expert * ss_e + (now.row + r + (!kDown && i != 0 ? p.ffn : 0)) / 128 * ss_n;
            }
        }
        int step = now.step;
#pragma unroll 1
        for (int s = 0; s < now.steps; ++s, step += now.stride) {
            const int k = step * kStep + t * kPiece, left = depth - k;
            float of_block[2];
            if (kW == kE4m3) {
                of_block[0] = scale_at[0][step * ss_k];
                of_block[1] = scale_at[1][step * ss_k];
            }
            uint4 a[2][2];  // [which 64 bytes][row g or g + 8]
            bool arrived = false;
#pragma unroll
            for (int n = 0; n < kTokens; ++n) {
                if (n < eights) {
                    const int column = n * 8 + g;
                    const bool here = column < count;
                    const int have = here ? left : 0;
                    constexpr int kPlanes = kDown ? 2 : 1, kLoads = kPiece / 8;
                    uint4 b[2][kPlanes][kLoads];  // the tokens' fragments; kTf32: 8 values of fp32
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int from_k = k + u * 4 * kPiece, some = have - u * 4 * kPiece;
                        if (kTf32) {
                            const float *from = static_cast<const float *>(p.h) + (first + (here ? column : 0)) * pitch + from_k;
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                if (some >= 4 * i + 4) {
                                    v = reinterpret_cast<const float4 *>(from)[i];
                                } else if (some > 4 * i) {
                                    v.x = from[4 * i];
                                    v.y = some > 4 * i + 1 ? from[4 * i + 1] : 0.0f;
                                    v.z = some > 4 * i + 2 ? from[4 * i + 2] : 0.0f;
                                }
                                b[u][i][0] = *reinterpret_cast<const uint4 *>(&v);
                            }
                        } else {
#pragma unroll
                            for (int plane = 0; plane < kPlanes; ++plane) {
                                const unsigned short *from =
                                    kDown ? h + (static_cast<long long>(plane) * h_rows + first + (here ? column : 0)) * pitch + from_k
                                          : x + lists.token[first + (here ? column : 0)] * p.x_ld + from_k;
#pragma unroll
                                for (int i = 0; i < kLoads; ++i) {
                                    b[u][plane][i] = load_8(from + i * 8, some - i * 8, vector);
                                }
                            }
                        }
                    }
                    if (!arrived) {
                        // the weights, behind the first tokens' loads
                        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
                        __syncwarp();
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const unsigned char *at = fragment + stage * kStageBytes + r * 1024;
                            a[0][r] = *reinterpret_cast<const uint4 *>(at);
                            a[1][r] = *reinterpret_cast<const uint4 *>(at + other);
                        }
                        arrived = true;
                    }
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    float(&to)[4] = kW == kE4m3 ? part : c[n];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (kTf32) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint4 &q = b[u][j / 2][0];
                                const float2 b0 = split_tf32(__uint_as_float(word(q, j % 2 * 2)));
                                const float2 b1 = split_tf32(__uint_as_float(word(q, j % 2 * 2 + 1)));
                                const uint32_t w0 = word(a[u][0], j), w1 = word(a[u][1], j);
                                const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&w0));
                                const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&w1));
                                mma_tf32(to, f0.x, f1.x, f0.y, f1.y, b0.y, b1.y);
                                mma_tf32(to, f0.x, f1.x, f0.y, f1.y, b0.x, b1.x);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 2 * kLoads; ++j) {
                                uint32_t a0, a1, a2, a3;
                                if (kW == kE4m3) {
                                    const uint32_t w0 = word(a[u][0], j), w1 = word(a[u][1], j);
                                    a0 = widen_e4m3<kBfMma>(w0, false);
                                    a1 = widen_e4m3<kBfMma>(w1, false);
                                    a2 = widen_e4m3<kBfMma>(w0, true);
                                    a3 = widen_e4m3<kBfMma>(w1, true);
                                } else {
                                    a0 = word(a[u][0], 2 * j);
                                    a1 = word(a[u][1], 2 * j);
                                    a2 = word(a[u][0], 2 * j + 1);
                                    a3 = word(a[u][1], 2 * j + 1);
                                }
#pragma unroll
                                for (int plane = kPlanes - 1; plane >= 0; --plane) {
                                    const uint4 &q = b[u][plane][j / 2];
                                    mma_16<kBfMma>(to, a0, a1, a2, a3, word(q, j % 2 * 2), word(q, j % 2 * 2 + 1));
                                }
                            }
                        }
                    }
                    if (kW == kE4m3) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            c[n][i] = fmaf(part[i], of_block[i / 2], c[n][i]);
                        }
                    }
                }
            }
            issue();
            stage = stage + 1 == kStages ? 0 : stage + 1;
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
                planes[h_rows * pitch + to] = f32_to_bf16_rne_bits(isfinite(hi) ? v - hi : 0.0f);
            }
        };
        while (now.next_up(p)) {
            multiply(now);
            const int first = lists.first[now.rank], count = lists.count[now.rank], eights = (count + 7) / 8;
#pragma unroll
            for (int n = 0; n < kTokens; ++n) {
                if (n < eights) {
                    if (group_warps == 1) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int column = n * 8 + 2 * t + j;
                            if (g < now.rows && column < count) {
                                store_h((first + column) * pitch + now.row + g, c[n][j], c[n][2 + j]);
                            }
                        }
                    } else {
                        // the group's sums, eight tokens at a time; two buffers take turns, so that one barrier does
                        float4 *buffer = sums + turn * kWarps * 32;
                        turn ^= 1;
                        buffer[warp * 32 + lane] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
                        const int group = warp / group_warps, threads = group_warps * 32;
                        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads) : "memory");
                        const float *from = reinterpret_cast<const float *>(buffer + group * threads);
                        const int i = tid % threads;
                        if (i < 64) {
                            const int of = i >> 1, j = i & 1;  // element j of lane `of`, and the one of the up's row
                            float gate = 0.0f, up = 0.0f;
                            for (int w = 0; w < group_warps; ++w) {
                                const float *at = from + (w * 32 + of) * 4 + j;
                                gate += at[0];
                                up += at[2];
                            }
                            const int r = of >> 2, column = n * 8 + (of & 3) * 2 + j;
                            if (r < now.rows && column < count) {
                                store_h((first + column) * pitch + now.row + r, gate, up);
                            }
                        }
                    }
                }
            }
        }
    } else {
        float *mine = y_sums + warp * p.tokens * kRows;
        while (now.next_rows()) {
            while (now.next_down()) {
                multiply(now);
                const int first = lists.first[now.rank], count = lists.count[now.rank], eights = (count + 7) / 8;
#pragma unroll
                for (int n = 0; n < kTokens; ++n) {
                    if (n < eights) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int column = n * 8 + 2 * t + j;
                            if (column < count) {
                                float *to = mine + lists.token[first + column] * kRows + g;
                                const float weight = lists.p[first + column];
                                to[0] = fmaf(weight, c[n][j], to[0]);
                                to[8] = fmaf(weight, c[n][2 + j], to[8]);
                            }
                        }
                    }
                }
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
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <Weights kW, bool kBf, bool kDown, int kTokens>
cudaError_t launch_one(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    constexpr size_t kShared = Layout<kDown, kTokens>::kBytes;
    static_assert(kShared <= 227 * 1024, "shared memory");
    const cudaError_t e =
        cudaFuncSetAttribute(experts_stream_kernel<kW, kBf, kDown, kTokens>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kShared));
    return e != cudaSuccess ? e : launch_chained(experts_stream_kernel<kW, kBf, kDown, kTokens>, dim3(sm_count), dim3(kThreads), kShared, stream, 1u, p);
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

// K-contiguous rows on 16-byte boundaries; the tokens may begin anywhere
bool experts_stream_takes(const ExpertsParams &p)
{
    const long long elem = p.w_dtype == KUDNN_B200_E4M3 ? 1 : 2;
    auto rows = [&](const void *w, long long se, long long sn, long long sk, long long depth) {
        return (sk == 1 || depth == 1) && (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && se * elem % 16 == 0 && sn * elem % 16 == 0;
    };
    return rows(p.gate_up, p.gu_se, p.gu_sn, p.gu_sk, p.hidden) && rows(p.down, p.d_se, p.d_sn, p.d_sk, p.ffn);
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
