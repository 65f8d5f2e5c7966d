// The router (experts.cuh): logits in 64 bits, scores, the choice of the largest, in one launch.
//
// A cluster of eight CTAs takes four tokens: each CTA an eighth of the experts, four experts x four tokens per warp at a time (16 sums in 64 bits
// per lane; a value that is loaded and widened serves four products), K split between warps where the experts are few.  Widening to 64 bits runs
// at a quarter of the rate of 32-bit arithmetic and the products at half, so that both are what bounds large batches; a few tokens are bound
// by the latency of reading w once.  The logits are gathered through distributed shared memory: CTA i finishes token i.
#include "experts.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace kb {

namespace {

namespace cg = cooperative_groups;

constexpr int kCluster = 8;
constexpr int kTokens = 4;   // of a cluster
constexpr int kExperts = 4;  // of a warp at a time
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// Four consecutive values, widened; `left` of them exist.  `vector`: their address is a multiple of four elements' size.
template <typename T>
__device__ __forceinline__ void load_four(const T *at, int left, bool vector, double (&v)[4])
{
    if (vector && left >= 4) {
        if (sizeof(T) == 4) {
            const float4 q = *reinterpret_cast<const float4 *>(at);
            v[0] = q.x;
            v[1] = q.y;
            v[2] = q.z;
            v[3] = q.w;
        } else {
            const uint2 q = *reinterpret_cast<const uint2 *>(at);
            T e[4];
            *reinterpret_cast<uint2 *>(e) = q;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = static_cast<double>(static_cast<float>(e[i]));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = i < left ? static_cast<double>(static_cast<float>(at[i])) : 0.0;
    }
}

// Sixteen sums over the lanes of a warp: half of the values go to the other half of the lanes, and so on.  Afterwards lane l holds value l / 2.
__device__ __forceinline__ double spread_sums(double (&v)[16], int lane)
{
#pragma unroll
    for (int half = 8; half > 0; half >>= 1) {
        const bool upper = (lane & (2 * half)) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const double keep = upper ? v[i + half] : v[i], give = upper ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * half);
        }
    }
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

__device__ __forceinline__ double block_reduce(double v, bool largest, double *scratch)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double other = __shfl_xor_sync(0xffffffffu, v, o);
        v = largest ? fmax(v, other) : v + other;
    }
    if ((threadIdx.x & 31) == 0) {
        scratch[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < kWarps; ++i) {
        v = largest ? fmax(v, scratch[i]) : v + scratch[i];
    }
    __syncthreads();
    return v;
}

template <typename X, typename W>
__global__ void __launch_bounds__(kThreads) route_kernel(const __grid_constant__ RouteParams p)
{
    extern __shared__ double shared[];
    __shared__ double scratch[kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank());
    const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    const int t0 = static_cast<int>(blockIdx.x) / kCluster * kTokens, count = min(kTokens, p.tokens - t0);
    const int mine = (p.experts + kCluster - 1) / kCluster;  // experts of a CTA
    const int e0 = rank * mine, here = max(0, min(mine, p.experts - e0));
    const int groups = (mine + kExperts - 1) / kExperts, splits = max(1, min(kWarps / groups, (p.hidden + 511) / 512));
    double *logits = shared;                                       // [kTokens][mine]
    double *parts = logits + kTokens * mine;                       // [splits][groups][16]
    pdl_launch_dependents();
    pdl_wait();
    const X *x = static_cast<const X *>(p.x) + static_cast<long long>(t0) * p.x_ld;
    const W *w = static_cast<const W *>(p.w);
    const bool x_vector = (reinterpret_cast<uintptr_t>(p.x) % (4 * sizeof(X))) == 0 && p.x_ld % 4 == 0;
    const bool w_vector = (reinterpret_cast<uintptr_t>(p.w) % (4 * sizeof(W))) == 0 && p.w_ld % 4 == 0;
    for (int unit = warp; unit < groups * splits; unit += kWarps) {
        const int group = unit % groups, split = unit / groups;
        const int first = e0 + group * kExperts, experts = min(kExperts, e0 + here - first);
        if (experts <= 0) {
            continue;
        }
        double sum[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sum[i] = 0.0;
        }
        for (int k = (split * 32 + lane) * 4; k < p.hidden; k += splits * 128) {
            double xv[kTokens][4], wv[kExperts][4];
#pragma unroll
            for (int i = 0; i < kExperts; ++i) {
                if (i < experts) {
                    load_four(w + (first + i) * p.w_ld + k, p.hidden - k, w_vector, wv[i]);
                } else {
                    wv[i][0] = wv[i][1] = wv[i][2] = wv[i][3] = 0.0;
                }
            }
#pragma unroll
            for (int t = 0; t < kTokens; ++t) {
                if (t < count) {
                    load_four(x + t * p.x_ld + k, p.hidden - k, x_vector, xv[t]);
#pragma unroll
                    for (int i = 0; i < kExperts; ++i) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            sum[t * kExperts + i] = fma(xv[t][j], wv[i][j], sum[t * kExperts + i]);
                        }
                    }
                }
            }
        }
        const double total = spread_sums(sum, lane);
        if ((lane & 1) == 0) {
            parts[(split * groups + group) * 16 + lane / 2] = total;
        }
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < kTokens * mine; i += kThreads) {
        const int t = i / mine, e = i % mine;
        double v = 0.0;
        if (e < here && t < count) {
            for (int s = 0; s < splits; ++s) {
                v += parts[(s * groups + e / kExperts) * 16 + t * kExperts + e % kExperts];
            }
        }
        logits[i] = v;
    }
    cluster.sync();
    if (rank < count) {
        // the whole row of token `rank`; each expert's key and score side by side in shared memory, where the partial sums were
        double *key = parts, *score = parts + p.experts;
        const double lowest = -__longlong_as_double(0x7ff0000000000000ll);
        double most = lowest;
        for (int e = static_cast<int>(threadIdx.x); e < p.experts; e += kThreads) {
            double v = cluster.map_shared_rank(logits, e / mine)[rank * mine + e % mine];
            if (p.bias != nullptr && p.bias[e] == __int_as_float(0xff800000)) {
                v = lowest;
                key[e] = lowest;
            } else {
                key[e] = 0.0;
            }
            score[e] = v;
            most = v > most ? v : most;
        }
        double sum = 1.0;
        if (p.sigmoid == 0) {
            most = block_reduce(most, true, scratch);
            double s = 0.0;
            for (int e = static_cast<int>(threadIdx.x); e < p.experts; e += kThreads) {
                const double v = score[e];
                score[e] = v == v && key[e] == 0.0 ? exp(v - most) : v;
                s += v == v && key[e] == 0.0 ? score[e] : 0.0;
            }
            sum = block_reduce(s, false, scratch);
        }
        for (int e = static_cast<int>(threadIdx.x); e < p.experts; e += kThreads) {
            if (key[e] == 0.0) {
                const double v = p.sigmoid != 0 ? 1.0 / (1.0 + exp(-score[e])) : score[e] / sum;
                const double k = p.bias != nullptr ? v + static_cast<double>(p.bias[e]) : v;
                score[e] = v;
                key[e] = k == k ? k : lowest;
            }
        }
        __syncthreads();
        if (warp == 0) {
            // the largest keys, one after the other; lane i keeps the places i and i + 32
            double chosen[2] = {0.0, 0.0}, total = 0.0;
            int ids[2] = {-1, -1};
            for (int j = 0; j < p.top; ++j) {
                double best = lowest;
                int at = -1;
                for (int e = lane; e < p.experts; e += 32) {
                    if (key[e] > best) {
                        best = key[e];
                        at = e;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const double other = __shfl_xor_sync(0xffffffffu, best, o);
                    const int other_at = __shfl_xor_sync(0xffffffffu, at, o);
                    if (other > best || (other == best && other_at >= 0 && (at < 0 || other_at < at))) {
                        best = other;
                        at = other_at;
                    }
                }
                if (at < 0) {
                    break;  // nobody is left: in all lanes alike
                }
                const double v = score[at];
                total += v;
                if (lane == j % 32) {
                    chosen[j / 32] = v;
                    ids[j / 32] = at;
                }
                __syncwarp();
                if (lane == 0) {
                    key[at] = lowest;
                }
                __syncwarp();
            }
            const double factor = p.normalise != 0 ? (total != 0.0 ? static_cast<double>(p.scale) / total : 0.0) : static_cast<double>(p.scale);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = lane + i * 32;
                if (j < p.top) {
                    const long long to = static_cast<long long>(t0 + rank) * p.top + j;
                    p.ids[to] = ids[i];
                    p.weights[to] = ids[i] < 0 ? 0.0f : static_cast<float>(chosen[i] * factor);
                }
            }
        }
    }
    cluster.sync();  // until here others may read this CTA's logits
}

template <typename X, typename W>
cudaError_t launch_typed(const RouteParams &p, cudaStream_t stream)
{
    const int mine = (p.experts + kCluster - 1) / kCluster, groups = (mine + kExperts - 1) / kExperts;
    const int splits = std::max(1, std::min(kWarps / groups, (p.hidden + 511) / 512));
    const size_t shared = sizeof(double) * (kTokens * mine + std::max(splits * groups * 16, 2 * p.experts));
    const long long clusters = (static_cast<long long>(p.tokens) + kTokens - 1) / kTokens;
    return launch_chained(route_kernel<X, W>, dim3(static_cast<unsigned>(clusters * kCluster)), dim3(kThreads), shared, stream, kCluster, p);
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
