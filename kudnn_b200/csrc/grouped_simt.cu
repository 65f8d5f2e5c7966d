// Grouped and block-scaled products (grouped.cuh) of operands in any layout: FMAs on 64 x 64 tiles, for what the tensor-core kernel
// does not take (rows that are not K-contiguous or not 16-byte aligned).
//
// Bound by the FMA pipe: 16 FMAs to 8 shared-memory words per thread and k.  K is walked in steps of 32, so that a step lies within one
// block of scales; the sum of a block is kept apart and added with its scale, or as it is: one chain of 8192 additions is 9.5e-7 off in the
// norm, 64 of 128 1.6e-7.
#include "grouped.cuh"

namespace kb {

namespace {

constexpr int kTile = 64, kStep = 32, kThreads = 256;

__device__ __forceinline__ float load_element(const void *p, int dtype, long long i)
{
    if (dtype == KUDNN_B200_E4M3) {
        return e4m3x2_to_f32(static_cast<const unsigned char *>(p)[i]).x;
    }
    return load_as_f32(p, dtype, i);
}

// Rows [row0, row0 + 64) x columns [k0, k0 + 32) of an operand into tile[k][row], zero outside of rows and k.  Consecutive threads
// follow the operand's contiguous dimension.
__device__ __forceinline__ void load_tile(float (*tile)[kTile + 4], const void *src, int dtype, long long s_row, long long s_k, int row0, int rows,
                                          int k0, int k)
{
    const bool k_first = s_k <= s_row;
    for (int i = threadIdx.x; i < kTile * kStep; i += kThreads) {
        const int r = k_first ? i / kStep : i % kTile;
        const int c = k_first ? i % kStep : i / kTile;
        float v = 0.0f;
        if (row0 + r < rows && k0 + c < k) {
            v = load_element(src, dtype, static_cast<long long>(row0 + r) * s_row + static_cast<long long>(k0 + c) * s_k);
        }
        tile[c][r] = v;
    }
}

__global__ void __launch_bounds__(kThreads) grouped_simt_kernel(const __grid_constant__ GroupedParams p)
{
    __shared__ __align__(16) float ta[kStep][kTile + 4];
    __shared__ __align__(16) float tb[kStep][kTile + 4];
    __shared__ int found[4];  // group, first row, end of the group's rows; end of all groups
    const int tiles_n = (p.n + kTile - 1) / kTile;
    const int n0 = static_cast<int>(blockIdx.x % tiles_n) * kTile;
    // tile blockIdx.x / tiles_n of all groups' row tiles, one group after the other
    if (threadIdx.x == 0) {
        int left = static_cast<int>(blockIdx.x / tiles_n), begin = group_offset(p, 0);
        found[0] = -1;
        for (int g = 0; g < p.groups; ++g) {
            const int next = group_offset(p, g + 1), end = next > begin ? next : begin;
            const int tiles = (end - begin + kTile - 1) / kTile;
            if (left >= 0 && left < tiles) {
                found[0] = g;
                found[1] = begin + left * kTile;
                found[2] = end;
            }
            left -= tiles;
            begin = end;
        }
        found[3] = begin;
    }
    __syncthreads();
    if (blockIdx.x / tiles_n == 0) {  // these blocks also clear the rows that no group holds
        const int first = group_offset(p, 0), held = found[3] - first;
        for (long long i = threadIdx.x; i < static_cast<long long>(p.rows - held) * kTile; i += kThreads) {
            const int at = static_cast<int>(i / kTile), n = n0 + static_cast<int>(i % kTile);
            if (n < p.n) {
                store_exact(p.c, p.c_dtype, (at < first ? at : at + held) * p.c_sm + n * p.c_sn, 0.0f);
            }
        }
    }
    const int g = found[0], row0 = found[1], row_end = found[2];
    if (g < 0) {
        return;
    }
    const int elem = p.ab_dtype == KUDNN_B200_E4M3 ? 1 : 2;
    const void *b = static_cast<const char *>(p.b) + static_cast<long long>(g) * p.b_sg * elem;
    const int tr = static_cast<int>(threadIdx.x) / 16 * 4, tn = static_cast<int>(threadIdx.x) % 16 * 4;
    const bool scaled = p.ab_dtype == KUDNN_B200_E4M3;
    float sum[4][4] = {}, part[4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += kStep) {
        load_tile(ta, p.a, p.ab_dtype, p.a_sm, p.a_sk, row0, row_end, k0, p.k);
        load_tile(tb, b, p.ab_dtype, p.b_sn, p.b_sk, n0, p.n, k0, p.k);
        __syncthreads();
#pragma unroll 8
        for (int c = 0; c < kStep; ++c) {
            const float4 x = *reinterpret_cast<const float4 *>(&ta[c][tr]);
            const float4 y = *reinterpret_cast<const float4 *>(&tb[c][tn]);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    part[i][j] = fmaf(xs[i], ys[j], part[i][j]);
                }
            }
        }
        __syncthreads();
        if ((k0 + kStep) % kScaleBlock == 0 || k0 + kStep >= p.k) {
            const int kb = k0 / kScaleBlock;
            float sa[4], sb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sa[i] = !scaled ? 1.0f : row0 + tr + i < row_end ? p.a_scale[(row0 + tr + i) * p.as_sm + kb * p.as_sk] : 0.0f;
                sb[i] = !scaled ? 1.0f : n0 + tn + i < p.n ? p.b_scale[g * p.bs_sg + (n0 + tn + i) / kScaleBlock * p.bs_sn + kb * p.bs_sk] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sum[i][j] = fmaf(part[i][j], sa[i] * sb[j], sum[i][j]);
                    part[i][j] = 0.0f;
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < 4; ++j) {
            const int r = row0 + tr + i, n = n0 + tn + j;
            if (r < row_end && n < p.n) {
                float v = sum[i][j];
                if (p.has_bias) {
                    v += load_as_f32(p.bias, p.bias_dtype, g * p.bias_sg + n * p.bias_sn);
                }
                v = activation_any(v, p.act, p.act_alpha, p.c_dtype == KUDNN_B200_F32 ? 1 : 0);
                store_exact(p.c, p.c_dtype, r * p.c_sm + n * p.c_sn, round_rne(v, p.c_dtype));
            }
        }
    }
}

}  // namespace

cudaError_t launch_grouped_simt(const GroupedParams &p, cudaStream_t stream)
{
    const long long row_tiles = (static_cast<long long>(p.rows) + kTile - 1) / kTile + (p.groups < p.rows ? p.groups : p.rows);
    const long long blocks = (row_tiles > 0 ? row_tiles : 1) * ((p.n + kTile - 1) / kTile);
    if (blocks > 0x7fffffffll) {
        return cudaErrorInvalidConfiguration;
    }
    grouped_simt_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace kb
