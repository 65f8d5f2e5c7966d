// fp32 / fp16 / bf16 -> e4m3 with an fp32 scale per block: q = e4m3(v * (448 / most)), scale = most / 448, most = max(|v| over the block,
// 1e-30).  v is the row itself, the row an index names, or silu(gate) * up of a row's two halves.  A block that holds a NaN is NaN
// throughout, its scale too; with infinities in it the scale is infinite, finite elements become 0 and infinite ones NaN.
#include "grouped.cuh"

namespace kb {

namespace {

constexpr float kE4m3Most = 448.0f;
constexpr float kLeast = 1e-30f;  // below it a block is scaled as if this were its largest magnitude: 448 / 1e-30 is finite

__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// e4m3 of (lo, hi), to nearest even, beyond 448 to 448
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi)
{
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

template <bool kPrecise>
__device__ __forceinline__ float gated(float gate, float up)
{
    return activation<kPrecise>(gate, KUDNN_B200_ACT_SWISH, 1.0f) * up;
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ float widen<__half>(__half v)
{
    return __half2float(v);
}
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}

// 8 lanes per block of 128 columns, 16 columns each.
template <typename T, bool kGate>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantizeParams p)
{
    constexpr bool kPrecise = sizeof(T) == 4;
    const int blocks_k = (p.k + kScaleBlock - 1) / kScaleBlock;
    const long long unit = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / 8;
    const int part = static_cast<int>(threadIdx.x) & 7;
    const long long row = unit / blocks_k;
    const int kb = static_cast<int>(unit % blocks_k);
    if (row >= p.rows) {
        return;
    }
    const long long from = p.index != nullptr ? p.index[row] : row;
    const bool inside = from >= 0 && from < p.x_rows;
    const T *x = static_cast<const T *>(p.x) + (inside ? from : 0) * p.x_ld;
    const int c0 = kb * kScaleBlock + part * 16;
    float v[16];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        v[i] = 0.0f;
        if (inside && c0 + i < p.k) {
            v[i] = widen<T>(x[c0 + i]);
            if (kGate) {
                v[i] = gated<kPrecise>(v[i], widen<T>(x[p.k + c0 + i]));
            }
        }
        most = max_nan(most, fabsf(v[i]));
    }
    const unsigned lanes = 0xffu << (threadIdx.x & 24);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        most = max_nan(most, __shfl_xor_sync(lanes, most, o));
    }
    most = max_nan(most, kLeast);
    const float up = kE4m3Most / most;
    if (part == 0) {
        p.scale[row * p.s_row + kb * p.s_col] = most / kE4m3Most;
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const uint32_t two = e4m3x2(v[i] * up, v[i + 1] * up);
        unsigned char *at = p.q + row * p.q_ld + c0 + i;
        if (c0 + i < p.k) {
            at[0] = static_cast<unsigned char>(two);
        }
        if (c0 + i + 1 < p.k) {
            at[1] = static_cast<unsigned char>(two >> 8);
        }
    }
}

// One CTA per 128 x 128 block, for weights: a warp takes 16 rows, a lane 4 columns.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const __grid_constant__ QuantizeParams p)
{
    __shared__ float warps[8];
    const int blocks_k = (p.k + kScaleBlock - 1) / kScaleBlock;
    const int rb = static_cast<int>(blockIdx.x / blocks_k), kb = static_cast<int>(blockIdx.x % blocks_k);
    const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
    const T *x = static_cast<const T *>(p.x);
    float v[16][4];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long long row = static_cast<long long>(rb) * kScaleBlock + i * 8 + warp;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = kb * kScaleBlock + j * 32 + lane;
            v[i][j] = row < p.rows && c < p.k ? widen<T>(x[row * p.x_ld + c]) : 0.0f;
            most = max_nan(most, fabsf(v[i][j]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    if (lane == 0) {
        warps[warp] = most;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        most = max_nan(most, warps[i]);
    }
    most = max_nan(most, kLeast);
    const float up = kE4m3Most / most;
    if (threadIdx.x == 0) {
        p.scale[rb * p.s_row + kb * p.s_col] = most / kE4m3Most;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const long long row = static_cast<long long>(rb) * kScaleBlock + i * 8 + warp;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = kb * kScaleBlock + j * 32 + lane;
            if (row < p.rows && c < p.k) {
                p.q[row * p.q_ld + c] = static_cast<unsigned char>(e4m3x2(v[i][j] * up, 0.0f));
            }
        }
    }
}

template <typename T>
cudaError_t launch_typed(const QuantizeParams &p, cudaStream_t stream)
{
    const long long blocks_k = (p.k + kScaleBlock - 1) / kScaleBlock;
    const long long blocks = p.block_rows == 1 ? (p.rows * blocks_k * 8 + 255) / 256 : (p.rows + kScaleBlock - 1) / kScaleBlock * blocks_k;
    if (blocks > 0x7fffffffll) {
        return cudaErrorInvalidConfiguration;
    }
    const unsigned grid = static_cast<unsigned>(blocks);
    if (p.block_rows != 1) {
        quantize_blocks_kernel<T><<<grid, 256, 0, stream>>>(p);
    } else if (p.gate != 0) {
        quantize_rows_kernel<T, true><<<grid, 256, 0, stream>>>(p);
    } else {
        quantize_rows_kernel<T, false><<<grid, 256, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize(const QuantizeParams &p, int sm_count, cudaStream_t stream)
{
    (void)sm_count;
    switch (p.x_dtype) {
        case KUDNN_B200_F32: return launch_typed<float>(p, stream);
        case KUDNN_B200_F16: return launch_typed<__half>(p, stream);
        default: return launch_typed<__nv_bfloat16>(p, stream);
    }
}

}  // namespace kb
