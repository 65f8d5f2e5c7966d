// The router (experts.cuh): logits in 64 bits, scores, the choice of the largest, in one launch.
//
// The products are those of the tensor cores in 64 bits (8 tokens x 8 experts x 4), which take a value per lane for each operand: it is widening them
// to 64 bits, 16 a cycle and SM, that costs most, and so each serves eight products.
// Few tokens: a cluster of eight CTAs takes eight of them, each CTA an eighth of the experts, so that w is read by many SMs, K split between its warps.
// The logits are gathered through distributed shared memory, and a warp finishes each token.  It is latency throughout: reading w once, two
// cluster barriers, the choice.
// Many tokens: a CTA takes sixteen and all experts, 64 at a time, two warps side by side for each quarter of K.
// 1 token x 64 experts x 4096: 7.8 us; 61 x 128 x 2048: 10.7 us; 4096 x 64 x 4096: 93 us, 23 TFLOP/s in 64 bits, with
// 8 experts 96 us (all 64 are computed), with 96 or 128 experts 180.  All registers that ptxas spills (332 to 664 bytes per instance) are those of
// finish_token for more than 256 experts, 32 keys and scores of 64 bits per lane.
#include "experts.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace kb {

namespace {

namespace cg = cooperative_groups;

constexpr int kCluster = 8;
constexpr int kTokens = 8;  // of a warp, and of a cluster
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// Four consecutive values, as they lie in memory
template <typename T>
struct alignas(4 * sizeof(T)) Four {
    T v[4];
};
// The first `left` of four values (a loop: it is seldom run)
template <typename T>
__device__ __forceinline__ Four<T> load_some(const T *at, int left)
{
    Four<T> q;
    q.v[0] = q.v[1] = q.v[2] = q.v[3] = static_cast<T>(0.0f);
#pragma unroll 1
    for (int i = min(left, 4) - 1; i >= 0; --i) {
        q.v[3] = q.v[2];
        q.v[2] = q.v[1];
        q.v[1] = q.v[0];
        q.v[0] = at[i];
    }
    return q;
}
template <typename T>
__device__ __forceinline__ double widen(T v)
{
    return static_cast<double>(static_cast<float>(v));
}

// c += a b: 8 x 4 by 4 x 8; lane l has a[l / 4][l % 4], b[l % 4][l / 4] and c[l / 4][2 (l % 4)], c[l / 4][2 (l % 4) + 1]
__device__ __forceinline__ void mma_64(double (&c)[2], double a, double b)
{
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

template <typename T>
__device__ __forceinline__ bool whole_fours(const void *at, long long pitch)
{
    return reinterpret_cast<uintptr_t>(at) % (4 * sizeof(T)) == 0 && pitch % 4 == 0;
}

// A warp's products of 8 tokens and 8 kN experts over k = first, first + step, ... of 16 each.  x, w: this lane's rows, of token lane / 4 and of
// expert lane / 4 of every eight; lane % 4 takes four neighbouring k of each sixteen.
template <int kN, typename X, typename W>
__device__ __forceinline__ void products(double (&c)[kN][2], const X *x, const W *const (&w)[kN], int first, int step, int depth, bool x_vector, bool w_vector)
{
    const int mine = static_cast<int>(threadIdx.x & 3u) * 4;
    double more[2] = {0.0, 0.0};  // kN = 1: a second chain of sums
    auto add = [&](const Four<X> &xv, const Four<W> (&wv)[kN]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double a = widen(xv.v[j]);
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                mma_64(kN == 1 && j % 2 != 0 ? more : c[n], a, widen(wv[n].v[j]));
            }
        }
    };
    int k0 = first;
    if (x_vector && w_vector) {
        // some steps' loads ahead of their use: latency is what a warp waits for
        constexpr int kAhead = kN == 1 ? 8 : 2;
        for (; k0 + (kAhead - 1) * step + 16 <= depth; k0 += kAhead * step) {
            Four<X> xv[kAhead];
            Four<W> wv[kAhead][kN];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int k = k0 + i * step + mine;
                xv[i] = *reinterpret_cast<const Four<X> *>(x + k);
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    wv[i][n] = *reinterpret_cast<const Four<W> *>(w[n] + k);
                }
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                add(xv[i], wv[i]);
            }
        }
#pragma unroll 1
        for (; k0 + 16 <= depth; k0 += step) {
            Four<W> wv[kN];
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                wv[n] = *reinterpret_cast<const Four<W> *>(w[n] + k0 + mine);
            }
            add(*reinterpret_cast<const Four<X> *>(x + k0 + mine), wv);
        }
    }
#pragma unroll 1
    for (; k0 < depth; k0 += step) {
        const int k = k0 + mine;
        Four<W> wv[kN];
        const Four<X> xv = load_some(x + k, depth - k);
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            wv[n] = load_some(w[n] + k, depth - k);
        }
        add(xv, wv);
    }
    c[0][0] += more[0];
    c[0][1] += more[1];
}

// A warp finishes token `token`: scores of its experts, kPer per lane, and the choice of the largest keys.  logit(e): the e-th expert's; scores:
// p.experts values of shared memory for this warp.  Keys are compared as integers of the same order, so that a warp's largest takes three
// instructions: its upper half, its lower half, the lowest index that has both.
template <int kPer, typename Logit>
__device__ __forceinline__ void finish_token(const RouteParams &p, int token, int lane, Logit logit, double *scores)
{
    const double lowest = -__longlong_as_double(0x7ff0000000000000ll);
    double v[kPer];
    double most = lowest;
    unsigned long long key[kPer];  // 0: takes no part
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        const bool in = e < p.experts && !(p.bias != nullptr && p.bias[e] == __int_as_float(0xff800000));
        v[i] = in ? logit(e) : lowest;
        key[i] = in ? 1ull : 0ull;
        most = v[i] > most ? v[i] : most;
    }
    double sum = 1.0;
    if (p.sigmoid == 0) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double other = __shfl_xor_sync(0xffffffffu, most, o);
            most = other > most ? other : most;
        }
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (key[i] != 0ull) {
                const bool number = v[i] == v[i];
                v[i] = exp(v[i] - most);
                sum += number ? v[i] : 0.0;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        if (key[i] != 0ull) {
            const double s = p.sigmoid != 0 ? 1.0 / (1.0 + exp(-v[i])) : v[i] / sum;
            const double k = (p.bias != nullptr ? s + static_cast<double>(p.bias[e]) : s) + 0.0;
            const bool ahead = p.nan_first != 0 && k != k;
            scores[e] = ahead ? k : s;
            const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(k));
            key[i] = ahead ? ~0ull : k > lowest ? ((bits >> 63) != 0ull ? ~bits : bits | 0x8000000000000000ull) : 0ull;
        }
    }
    __syncwarp();
    // lane i keeps the places i and i + 32
    double chosen[2] = {0.0, 0.0}, total = 0.0;
    int ids[2] = {-1, -1};
    for (int j = 0; j < p.top; ++j) {
        unsigned long long best = 0ull;
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (key[i] > best) {
                best = key[i];
                at = lane + 32 * i;
            }
        }
        const unsigned hi = static_cast<unsigned>(best >> 32), most_hi = __reduce_max_sync(0xffffffffu, hi);
        const unsigned lo = hi == most_hi ? static_cast<unsigned>(best) : 0u, most_lo = __reduce_max_sync(0xffffffffu, lo);
        if (most_hi == 0u) {
            break;  // nobody is left: a key that takes part has its upper half set
        }
        const int first = __reduce_min_sync(0xffffffffu, hi == most_hi && lo == most_lo ? at : 0x7fffffff);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            key[i] = lane + 32 * i == first ? 0ull : key[i];
        }
        const double s = scores[first];
        total += s;
        if (lane == j % 32) {
            chosen[j / 32] = s;
            ids[j / 32] = first;
        }
    }
    const double factor = p.normalise != 0 ? (total != 0.0 ? static_cast<double>(p.scale) / total : 0.0) : static_cast<double>(p.scale);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = lane + i * 32;
        if (j < p.top) {
            const long long to = static_cast<long long>(token) * p.top + j;
            p.ids[to] = ids[i];
            p.weights[to] = ids[i] < 0 ? 0.0f : static_cast<float>(chosen[i] * factor);
        }
    }
}

template <typename Logit>
__device__ __forceinline__ void finish_any(const RouteParams &p, int token, int lane, Logit logit, double *scores)
{
    if (p.experts <= 64) {
        finish_token<2>(p, token, lane, logit, scores);
    } else if (p.experts <= 256) {
        finish_token<8>(p, token, lane, logit, scores);
    } else {
        finish_token<32>(p, token, lane, logit, scores);
    }
}

template <typename X, typename W>
__global__ void __launch_bounds__(kThreads) route_few_kernel(const __grid_constant__ RouteParams p)
{
    extern __shared__ double shared[];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    const int t0 = static_cast<int>(blockIdx.x) / kCluster * kTokens, count = min(kTokens, p.tokens - t0);
    const int mine = (p.experts + kCluster - 1) / kCluster;  // experts of a CTA
    const int e0 = rank * mine, here = max(0, min(mine, p.experts - e0));
    const int groups = (mine + 7) / 8, splits = max(1, min(kWarps / groups, (p.hidden + 63) / 64));
    double *logits = shared;                  // [kTokens][mine]
    double *parts = logits + kTokens * mine;  // [splits][groups][kTokens][8]; then the scores of a token
    pdl_launch_dependents();
    pdl_wait();
    const X *x = static_cast<const X *>(p.x) + static_cast<long long>(t0 + min(lane >> 2, count - 1)) * p.x_ld;
    for (int unit = warp; unit < groups * splits; unit += kWarps) {
        const int group = unit % groups, split = unit / groups;
        if (group * 8 >= here) {
            continue;
        }
        const W *const w[1] = {static_cast<const W *>(p.w) + static_cast<long long>(e0 + min(group * 8 + (lane >> 2), here - 1)) * p.w_ld};
        double c[1][2] = {};
        products<1, X, W>(c, x, w, split * 16, splits * 16, p.hidden, whole_fours<X>(p.x, p.x_ld), whole_fours<W>(p.w, p.w_ld));
        double *to = parts + ((split * groups + group) * kTokens + (lane >> 2)) * 8 + (lane & 3) * 2;
        to[0] = c[0][0];
        to[1] = c[0][1];
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < kTokens * mine; i += kThreads) {
        const int t = i / mine, e = i % mine;
        double v = 0.0;
        if (e < here && t < count) {
            for (int s = 0; s < splits; ++s) {
                v += parts[((s * groups + e / 8) * kTokens + t) * 8 + e % 8];
            }
        }
        logits[i] = v;
    }
    cluster.sync();
    if (rank < count && warp == 0) {
        finish_any(p, t0 + rank, lane, [&](int e) { return cluster.map_shared_rank(logits, e / mine)[rank * mine + e % mine]; }, parts);
    }
    cluster.sync();  // until here others may read this CTA's logits
}

constexpr int kTile = 16;          // tokens of a CTA
constexpr int kTileThreads = 256;  // two eights of tokens, four quarters of K
constexpr int kTileEights = 8;     // experts at a time, in eights

template <typename X, typename W>
__global__ void __launch_bounds__(kTileThreads, 2) route_many_kernel(const __grid_constant__ RouteParams p)
{
    extern __shared__ double shared[];
    double *logits = shared;  // [kTile][experts]
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
    const int t0 = static_cast<int>(blockIdx.x) * kTile, quarter = warp >> 1, eight = warp & 1;
    pdl_launch_dependents();
    pdl_wait();
    const X *x = static_cast<const X *>(p.x) + static_cast<long long>(min(t0 + eight * 8 + (lane >> 2), p.tokens - 1)) * p.x_ld;
    for (int e0 = 0; e0 < p.experts; e0 += kTileEights * 8) {
        const W *w[kTileEights];
        double c[kTileEights][2];
#pragma unroll
        for (int n = 0; n < kTileEights; ++n) {
            w[n] = static_cast<const W *>(p.w) + static_cast<long long>(min(e0 + n * 8 + (lane >> 2), p.experts - 1)) * p.w_ld;
            c[n][0] = c[n][1] = 0.0;
        }
        products<kTileEights, X, W>(c, x, w, quarter * 16, 64, p.hidden, whole_fours<X>(p.x, p.x_ld), whole_fours<W>(p.w, p.w_ld));
        // the quarters' sums, one after the other
        for (int q = 0; q < 4; ++q) {
            if (quarter == q) {
#pragma unroll
                for (int n = 0; n < kTileEights; ++n) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int t = eight * 8 + (lane >> 2), e = e0 + n * 8 + (lane & 3) * 2 + j;
                        if (e < p.experts) {
                            logits[t * p.experts + e] = q == 0 ? c[n][j] : logits[t * p.experts + e] + c[n][j];
                        }
                    }
                }
            }
            __syncthreads();
        }
    }
    for (int t = warp; t < kTile && t0 + t < p.tokens; t += kTileThreads / 32) {
        // each lane's scores replace the logits that it has read
        finish_any(p, t0 + t, lane, [&](int e) { return logits[t * p.experts + e]; }, logits + t * p.experts);
    }
}

template <typename X, typename W>
cudaError_t launch_typed(const RouteParams &p, cudaStream_t stream)
{
    // x 64 experts x 4096: 64, 256, 512 and 1024 tokens 9, 24, 40 and 71 us by the first kernel, 51 (256) to 57 (1024) by the second; x 128
    // experts 14, 39, 64, 114 and 99 to 101
    if (p.tokens > 768) {
        const size_t shared = sizeof(double) * kTile * p.experts;
        const cudaError_t e = cudaFuncSetAttribute(route_many_kernel<X, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(sizeof(double)) * kTile * kMostExperts);
        return e != cudaSuccess ? e
                                : launch_chained(route_many_kernel<X, W>, dim3((p.tokens + kTile - 1) / kTile), dim3(kTileThreads), shared, stream, 1u, p);
    }
    const int mine = (p.experts + kCluster - 1) / kCluster, groups = (mine + 7) / 8;
    const int splits = std::max(1, std::min(kWarps / groups, (p.hidden + 63) / 64));
    const size_t shared = sizeof(double) * (kTokens * mine + std::max(splits * groups * kTokens * 8, p.experts));
    const int clusters = (p.tokens + kTokens - 1) / kTokens;
    return launch_chained(route_few_kernel<X, W>, dim3(clusters * kCluster), dim3(kThreads), shared, stream, kCluster, p);
}

template <typename X>
cudaError_t launch_x(const RouteParams &p, cudaStream_t stream)
{
    switch (p.w_dtype) {
        case KUDNN_B200_F32: return launch_typed<X, float>(p, stream);
        case KUDNN_B200_F16: return launch_typed<X, __half>(p, stream);
        default: return launch_typed<X, __nv_bfloat16>(p, stream);
    }
}

}  // namespace

cudaError_t launch_route(const RouteParams &p, cudaStream_t stream)
{
    switch (p.x_dtype) {
        case KUDNN_B200_F32: return launch_x<float>(p, stream);
        case KUDNN_B200_F16: return launch_x<__half>(p, stream);
        default: return launch_x<__nv_bfloat16>(p, stream);
    }
}

}  // namespace kb
