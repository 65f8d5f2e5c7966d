// The block of experts for few tokens in two kernels that stream the weights once (experts.cuh).
//
// What bounds it is reading the chosen experts' weights; everything here serves to keep as many bytes in flight as HBM wants, without pauses:
//   * Both products are cut by weight rows alone: the rows (gate and up rows in pairs) of all chosen experts are dealt out evenly, one CTA per SM,
//     so that every SM streams the same number of bytes; nothing is added up across CTAs, no atomics, and the same call gives the same bits.
//   * The 16 warps of a CTA split K: each takes every sixteenth step of 64 bytes of 32 rows.  Every lane copies its own 16 bytes of 4 rows into a
//     ring in shared memory of its own (cp.async, four steps ahead) and reads back only what it copied, so that no barrier stands in the stream.
//     Copies of what lies beyond the last row or column bring zeros.
//   * The lanes' pieces are, as they are, operand fragments of mma.m16n8k16 with a permuted k: weights on the side of 16 rows, tokens on that of 8;
//     four neighbouring lanes hold 64 neighbouring bytes of a row.  The tokens' fragments are read from L1 and L2 in the same permutation.
//   * Where the warps' sums meet, at the end of 32 rows, the next rows' copies are on their way.
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
constexpr int kTileRows = 32;                     // weight rows of a tile: 16 gate and 16 up rows, or 32 of down
constexpr int kStages = 5;                        // steps of a warp's ring
constexpr int kStageBytes = kTileRows * 64;       // of one warp
constexpr int kRingBytes = kWarps * kStages * kStageBytes;
constexpr int kSumBytes = 2 * kWarps * 2 * 32 * 16;  // the warps' sums of 8 tokens, in two buffers
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

// 8 values of 16 bits from `at`, of which `left` exist; vector: `at` is on a 16-byte boundary
__device__ __forceinline__ uint4 load_8(const unsigned short *at, int left, bool vector)
{
    if (vector && left >= 8) {
        return *reinterpret_cast<const uint4 *>(at);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = 2 * i < left ? at[2 * i] : 0u, hi = 2 * i + 1 < left ? at[2 * i + 1] : 0u;
        w[i] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
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

// Where a CTA stands in its tiles: up to 32 rows of one expert.
template <bool kDown>
struct Cursor {
    long long at, end;  // up: pairs of rows of all active experts, one after the other; down: rows of y
    int rank;           // of the expert
    int row, rows;      // first row (of the gate, or of down) and how many, 16 or 32 at most
    __device__ __forceinline__ void start(const ExpertsParams &p, const Lists &l)
    {
        const long long all = kDown ? p.hidden : static_cast<long long>(l.active) * p.ffn;
        at = all * blockIdx.x / gridDim.x;
        end = all * (blockIdx.x + 1) / gridDim.x;
        rank = kDown ? -1 : 0;
        rows = 0;
        if (kDown) {
            set_rows();
        }
    }
    // down: the rows left are cut into equal tiles
    __device__ __forceinline__ void set_rows()
    {
        const long long left = end - at;
        const int tiles = static_cast<int>((left + kTileRows - 1) / kTileRows);
        row = static_cast<int>(at);
        rows = tiles > 0 ? static_cast<int>((left + tiles - 1) / tiles) : 0;
    }
    // false: no tile is left.  down: a tile is all active experts' turn at the same rows
    __device__ __forceinline__ bool next(const ExpertsParams &p, const Lists &l)
    {
        if (kDown) {
            if (rows == 0 || l.active == 0) {
                return false;
            }
            if (++rank == l.active) {
                rank = 0;
                at += rows;
                set_rows();
                return rows > 0;
            }
            return true;
        }
        at += rows;
        if (at >= end) {
            return false;
        }
        rank = static_cast<int>(at / p.ffn);
        row = static_cast<int>(at - static_cast<long long>(rank) * p.ffn);
        rows = static_cast<int>(min(static_cast<long long>(kTileRows / 2), min(end - at, static_cast<long long>(p.ffn - row))));
        return true;
    }
};

// kTokens: an expert's most, in eights.
template <Weights kW, bool kBf, bool kDown, int kTokens>
__global__ void __launch_bounds__(kThreads, 1) experts_stream_kernel(const __grid_constant__ ExpertsParams p)
{
    constexpr int kStep = kW == kE4m3 ? 64 : 32;      // of K: 64 bytes of a row
    constexpr int kPiece = kStep / 4;                 // of a lane
    constexpr int kElem = kW == kE4m3 ? 1 : 2;
    constexpr bool kTf32 = kDown && kW == kF16;       // h in fp32, products of tf32
    constexpr bool kBfMma = kW == kBf16 || (kW == kE4m3 && (kBf || kDown));
    extern __shared__ __align__(16) unsigned char shared[];
    unsigned char *ring = shared;
    float4 *sums = reinterpret_cast<float4 *>(shared + kRingBytes);  // [2][kWarps][2][32]
    float *y_sums = reinterpret_cast<float *>(shared + kRingBytes + kSumBytes);  // down: [tokens][32]
    Lists &lists = *reinterpret_cast<Lists *>(shared + kRingBytes + kSumBytes + (kDown ? kMostExpertTokens * kTileRows * 4 : 0));
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int depth = kDown ? p.ffn : p.hidden;  // K
    const int steps = (depth + kStep - 1) / kStep, mine = warp < steps ? (steps - warp + kWarps - 1) / kWarps : 0;
    const char *weights = static_cast<const char *>(kDown ? p.down : p.gate_up);
    const long long se = kDown ? p.d_se : p.gu_se, sn = kDown ? p.d_sn : p.gu_sn;

    if (!kDown) {
        pdl_wait();
        pdl_launch_dependents();  // behind the wait: what the second kernel reads ahead of its own is older than this one
    }
    make_lists(lists, p);

    // ---- the stream: this lane's next copies
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + static_cast<uint32_t>(warp * kStages * kStageBytes + lane * 16);
    Cursor<kDown> ahead;
    ahead.start(p, lists);
    bool more = mine > 0 && ahead.next(p, lists);
    int ahead_step = 0, ahead_stage = 0;
    const char *row_at[4];
    int row_here = 0;  // bit i: the lane's i-th row exists
    auto set_rows = [&]() {
        row_here = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // i = 2 * (upper sixteen) + (upper eight)
            const int r = kDown ? i * 8 + g : (i >> 1) * 8 + g;
            const bool here = r < ahead.rows;
            const long long row = ahead.row + r + (!kDown && (i & 1) != 0 ? p.ffn : 0);
            row_at[i] = here ? weights + (lists.expert[ahead.rank] * se + row * sn) * kElem : weights;
            row_here |= here ? 1 << i : 0;
        }
    };
    if (more) {
        set_rows();
    }
    auto issue = [&]() {
        if (more) {
            const int k = (ahead_step * kWarps + warp) * kStep + t * kPiece;
            const int bytes = max(0, min(16, (depth - k) * kElem));
            const uint32_t to = ring_at + static_cast<uint32_t>(ahead_stage * kStageBytes);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = (row_here >> i & 1) != 0 ? bytes : 0;
                copy_16(to + i * 512, row_at[i] + (n > 0 ? static_cast<long long>(k) * kElem : 0), n);
            }
            if (++ahead_step == mine) {
                ahead_step = 0;
                more = ahead.next(p, lists);
                if (more) {
                    set_rows();
                }
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
        for (int i = tid; i < p.tokens * kTileRows; i += kThreads) {
            y_sums[i] = 0.0f;
        }
        pdl_wait();
        pdl_launch_dependents();
    }

    // ---- the products
    const long long pitch = h_pitch(p);
    const int h_rows = p.tokens * p.top;
    const unsigned short *x = static_cast<const unsigned short *>(p.x), *h = static_cast<const unsigned short *>(p.h);
    const bool vector = kDown || ((reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && p.x_ld % 8 == 0);
    const float *scale = kDown ? p.down_scale : p.gate_up_scale;
    const long long ss_e = kDown ? p.ds_se : p.gus_se, ss_n = kDown ? p.ds_sn : p.gus_sn, ss_k = kDown ? p.ds_sk : p.gus_sk;
    Cursor<kDown> now;
    now.start(p, lists);
    int stage = 0, turn = 0;
    while (now.next(p, lists)) {
        const int expert = lists.expert[now.rank], first = lists.first[now.rank], count = lists.count[now.rank];
        const int eights = (count + 7) / 8;
        float c[kTokens][2][4];
#pragma unroll
        for (int n = 0; n < kTokens; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[n][0][i] = c[n][1][i] = 0.0f;
            }
        }
        const float *scale_at[4];
        if (kW == kE4m3) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = kDown ? i * 8 + g : (i >> 1) * 8 + g;
                const long long row = now.row + min(r, now.rows - 1) + (!kDown && (i & 1) != 0 ? p.ffn : 0);
                scale_at[i] = scale + expert * ss_e + row / 128 * ss_n;
            }
        }
#pragma unroll 1
        for (int s = 0; s < mine; ++s) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            const int k = (s * kWarps + warp) * kStep + t * kPiece, left = depth - k;
            uint4 a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = *reinterpret_cast<const uint4 *>(ring + (warp * kStages + stage) * kStageBytes + i * 512 + lane * 16);
            }
            float of_block[4];
            if (kW == kE4m3) {
                const long long block = (s * kWarps + warp) * kStep / 128 * ss_k;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    of_block[i] = scale_at[i][block];
                }
            }
#pragma unroll
            for (int n = 0; n < kTokens; ++n) {
                if (n < eights) {
                    const int column = n * 8 + g;
                    const bool here = column < count;
                    const int have = here ? left : 0;
                    float part[2][4];
                    if (kW == kE4m3) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            part[0][i] = part[1][i] = 0.0f;
                        }
                    }
                    float(&to)[2][4] = kW == kE4m3 ? part : c[n];
                    if (kTf32) {
                        const float *from = static_cast<const float *>(p.h) + (first + (here ? column : 0)) * pitch + k;
                        float v[8];
                        if (have >= 8) {
                            *reinterpret_cast<float4 *>(v) = reinterpret_cast<const float4 *>(from)[0];
                            *reinterpret_cast<float4 *>(v + 4) = reinterpret_cast<const float4 *>(from)[1];
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                v[i] = i < have ? from[i] : 0.0f;
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 b0 = split_tf32(v[2 * j]), b1 = split_tf32(v[2 * j + 1]);
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                const uint32_t w0 = word(a[2 * m], j), w1 = word(a[2 * m + 1], j);
                                const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&w0));
                                const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&w1));
                                mma_tf32(to[m], f0.x, f1.x, f0.y, f1.y, b0.y, b1.y);
                                mma_tf32(to[m], f0.x, f1.x, f0.y, f1.y, b0.x, b1.x);
                            }
                        }
                    } else {
                        constexpr int kPlanes = kDown ? 2 : 1, kLoads = kPiece / 8;
                        uint4 b[kPlanes][kLoads];
#pragma unroll
                        for (int plane = 0; plane < kPlanes; ++plane) {
                            const unsigned short *from =
                                kDown ? h + (static_cast<long long>(plane) * h_rows + first + (here ? column : 0)) * pitch + k
                                      : x + lists.token[first + (here ? column : 0)] * p.x_ld + k;
#pragma unroll
                            for (int i = 0; i < kLoads; ++i) {
                                b[plane][i] = load_8(from + i * 8, have - i * 8, vector);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < kStep / 16; ++j) {
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                uint32_t a0, a1, a2, a3;
                                if (kW == kE4m3) {
                                    const uint32_t w0 = word(a[2 * m], j), w1 = word(a[2 * m + 1], j);
                                    a0 = widen_e4m3<kBfMma>(w0, false);
                                    a1 = widen_e4m3<kBfMma>(w1, false);
                                    a2 = widen_e4m3<kBfMma>(w0, true);
                                    a3 = widen_e4m3<kBfMma>(w1, true);
                                } else {
                                    a0 = word(a[2 * m], 2 * j);
                                    a1 = word(a[2 * m + 1], 2 * j);
                                    a2 = word(a[2 * m], 2 * j + 1);
                                    a3 = word(a[2 * m + 1], 2 * j + 1);
                                }
#pragma unroll
                                for (int plane = kPlanes - 1; plane >= 0; --plane) {
                                    const uint4 &q = b[plane][j / 2];
                                    mma_16<kBfMma>(to[m], a0, a1, a2, a3, word(q, j % 2 * 2), word(q, j % 2 * 2 + 1));
                                }
                            }
                        }
                    }
                    if (kW == kE4m3) {
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                c[n][m][i] = fmaf(part[m][i], of_block[2 * m + i / 2], c[n][m][i]);
                            }
                        }
                    }
                }
            }
            issue();
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        // ---- the warps' sums, eight tokens at a time; buffers take turns, so that one barrier does
#pragma unroll
        for (int n = 0; n < kTokens; ++n) {
            if (n < eights) {
                float4 *buffer = sums + turn * kWarps * 64;
                turn ^= 1;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    buffer[(warp * 2 + m) * 32 + lane] = make_float4(c[n][m][0], c[n][m][1], c[n][m][2], c[n][m][3]);
                }
                __syncthreads();
                // two threads per sum, eight warps' each: half in {0, 1}, element e of lane `of` of half m
                const int half = tid & 1, e = tid >> 1 & 3, of = tid >> 3 & 31, m = tid >> 8;
                const float *from = reinterpret_cast<const float *>(buffer) + (m * 32 + of) * 4 + e;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps / 2; ++w) {
                    sum += from[(half * (kWarps / 2) + w) * 256];
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                const int column = n * 8 + (of & 3) * 2 + (e & 1);
                if (kDown) {
                    const int r = m * 16 + (e >> 1) * 8 + (of >> 2);
                    if (half == 0 && column < count && r < now.rows) {
                        float &y = y_sums[lists.token[first + column] * kTileRows + r];
                        y = fmaf(lists.p[first + column], sum, y);
                    }
                } else {
                    const float up = __shfl_down_sync(0xffffffffu, sum, 4);  // the same column of the row eight further down
                    const int r = m * 8 + (of >> 2);
                    if (half == 0 && e < 2 && column < count && r < now.rows) {
                        const float v = expert_gate(sum, up);
                        const long long to = (first + column) * pitch + now.row + r;
                        if (kW == kF16) {
                            static_cast<float *>(p.h)[to] = v;
                        } else {
                            const float hi = __bfloat162float(__float2bfloat16_rn(v));
                            unsigned short *planes = static_cast<unsigned short *>(p.h);
                            planes[to] = f32_to_bf16_rne_bits(v);
                            planes[h_rows * pitch + to] = f32_to_bf16_rne_bits(isfinite(hi) ? v - hi : 0.0f);
                        }
                    }
                }
            }
        }
        if (kDown && now.rank == lists.active - 1) {
            // the last expert's turn at these rows
            __syncthreads();
            for (int i = tid; i < p.tokens * kTileRows; i += kThreads) {
                const int token = i / kTileRows, r = i % kTileRows;
                if (r < now.rows) {
                    store_exact(p.y, p.x_dtype, token * p.y_ld + now.row + r, round_rne(y_sums[i], p.x_dtype));
                }
                y_sums[i] = 0.0f;
            }
            __syncthreads();
        }
    }
    if (kDown && lists.active == 0) {
        for (long long r = now.at; r < now.end; ++r) {
            for (int token = tid; token < p.tokens; token += kThreads) {
                store_exact(p.y, p.x_dtype, token * p.y_ld + r, 0.0f);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <Weights kW, bool kBf, bool kDown, int kTokens>
cudaError_t launch_one(const ExpertsParams &p, int sm_count, cudaStream_t stream)
{
    constexpr size_t kShared = kRingBytes + kSumBytes + (kDown ? kMostExpertTokens * kTileRows * 4 : 0) + sizeof(Lists);
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
