// fp32 / fp16 / bf16 -> e4m3 with an fp32 scale per block: q = e4m3(v * (448 / most)), scale = most / 448, most = max(|v| over the block,
// 1e-30).  v is the row itself, the row an index names, or silu(gate) * up of a row's two halves.  A block that holds a NaN is NaN
// throughout, its scale too; with infinities in it the scale is infinite, finite elements become 0 and infinite ones NaN.
#include "grouped.cuh"

#include <type_traits>

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

// silu(gate) * up, as gate / (1 + exp(-gate)) or gate exp(gate) / (1 + exp(gate)): the one that raises e to a power below zero, so that
// the divisor lies in [1, 2].  expf, since two to a rounded multiple of the gate is off in proportion to the gate (up to 2^-18.2, and the
// fp32 scale with it); behind it the hardware's reciprocal, 1 unit in the last place, for 16-bit values: 2^-21.9 off at most, 6.1e-8 in
// the square mean, against 2^-22.1 and 5.9e-8 by divisions.  8192 x 11008 of bf16: 94 us, by divisions 110, with the hardware's
// exponential 82.
template <bool kPrecise>
__device__ __forceinline__ float gated(float gate, float up)
{
    const float e = expf(-fabsf(gate)), over = gate < 0.0f ? gate * e : gate;
    return (kPrecise ? over / (1.0f + e) : over * rcp_approx(1.0f + e)) * up;
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

// 16 consecutive elements, two per word (or one)
template <typename T>
struct Sixteen {
    uint4 w[sizeof(T)];
    __device__ __forceinline__ void load(const T *at)
    {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T); ++i) {
            w[i] = reinterpret_cast<const uint4 *>(at)[i];
        }
    }
    __device__ __forceinline__ float operator[](int i) const
    {
        const uint4 &q = w[i * sizeof(T) / 16];
        const int j = i * static_cast<int>(sizeof(T)) / 4 % 4;
        const uint32_t word = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
        if (sizeof(T) == 4) {
            return __uint_as_float(word);
        }
        if (std::is_same<T, __nv_bfloat16>::value) {
            return __uint_as_float(i % 2 == 0 ? word << 16 : word & 0xffff0000u);
        }
        return f16_bits_to_f32(static_cast<unsigned short>(i % 2 == 0 ? word & 0xffffu : word >> 16));
    }
};

__device__ __forceinline__ const void *source_row(const QuantizeParams &p, int row, int elem, bool *inside)
{
    const long long from = p.index != nullptr ? p.index[row] : row;
    *inside = from >= 0 && from < p.x_rows;
    return static_cast<const char *>(p.x) + (*inside ? from : 0) * p.x_ld * elem;
}

// Rows on 16-byte boundaries: 8 lanes per block of 128 columns, 16 columns each, everything in registers between one read and one write.
//
// Rows as they are are bound by HBM (2 or 4 bytes read and 1.03 written per element): 28672 x 8192 bf16 values take 120 us, 5.9 TB/s, 0.89 of
// a copy's rate.  Gated ones by their instructions (the schedulers issue in 84 % of the cycles): 8192 x 11008 bf16 values take 94 us, 4.8 TB/s;
// read and written element by element 238 us.
template <typename T, bool kGate>
__global__ void __launch_bounds__(128) quantize_rows_kernel(const __grid_constant__ QuantizeParams p)
{
    constexpr bool kPrecise = sizeof(T) == 4;
    const unsigned blocks_k = static_cast<unsigned>(p.k + kScaleBlock - 1) / kScaleBlock;
    const unsigned unit = blockIdx.x * 16u + threadIdx.x / 8u;
    const int row = static_cast<int>(unit / blocks_k), kb = static_cast<int>(unit % blocks_k);
    const int part = static_cast<int>(threadIdx.x) & 7;
    pdl_launch_dependents();
    pdl_wait();
    if (row >= p.rows) {
        return;
    }
    bool inside;
    const T *x = static_cast<const T *>(source_row(p, row, sizeof(T), &inside));
    const int c0 = kb * kScaleBlock + part * 16;
    float v[16];
    float most = 0.0f;
    if (inside && c0 + 16 <= p.k) {
        Sixteen<T> first, second;
        first.load(x + c0);
        if (kGate) {
            second.load(x + p.k + c0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[i] = kGate ? gated<kPrecise>(first[i], second[i]) : first[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[i] = 0.0f;
            if (inside && c0 + i < p.k) {
                v[i] = widen<T>(x[c0 + i]);
                if (kGate) {
                    v[i] = gated<kPrecise>(v[i], widen<T>(x[p.k + c0 + i]));
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
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
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = e4m3x2(v[4 * i] * up, v[4 * i + 1] * up) | e4m3x2(v[4 * i + 2] * up, v[4 * i + 3] * up) << 16;
    }
    unsigned char *to = p.q + row * p.q_ld + c0;
    if (c0 + 16 <= p.k) {
        *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (c0 + i < p.k) {
                to[i] = static_cast<unsigned char>(w[i / 4] >> i % 4 * 8);
            }
        }
    }
}

// Rows that begin anywhere: a warp takes four blocks of columns, every lane each 32nd, so that its accesses lie side by side however they
// are aligned.  Bound by instructions (the schedulers issue in 74 % of the cycles): 9001 rows of 4099 fp16 values, gathered from 1501, take
// 25 us; 41 us where every lane divided for every block and each block was reduced by itself, and no less with four neighbouring columns
// per lane and 4-byte stores.
template <typename T, bool kGate>
__global__ void __launch_bounds__(128) quantize_any_kernel(const __grid_constant__ QuantizeParams p)
{
    constexpr bool kPrecise = sizeof(T) == 4;
    const unsigned spans = static_cast<unsigned>(p.k + 4 * kScaleBlock - 1) / (4 * kScaleBlock);
    const unsigned unit = blockIdx.x * 4u + threadIdx.x / 32u;
    const int row = static_cast<int>(unit / spans), c0 = static_cast<int>(unit % spans) * 4 * kScaleBlock;
    const int lane = static_cast<int>(threadIdx.x) & 31;
    pdl_launch_dependents();
    pdl_wait();
    if (row >= p.rows) {
        return;
    }
    bool inside;
    const T *x = static_cast<const T *>(source_row(p, row, sizeof(T), &inside)) + c0 + lane;
    unsigned char *to = p.q + row * p.q_ld + c0 + lane;
    const int left = p.k - c0 - lane;
    const bool whole = inside && c0 + 4 * kScaleBlock <= p.k;
    float v[16];
    if (whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[i] = widen<T>(x[i * 32]);
        }
        if (kGate) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = gated<kPrecise>(v[i], widen<T>(x[p.k + i * 32]));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            v[i] = 0.0f;
            if (inside && i * 32 < left) {
                v[i] = widen<T>(x[i * 32]);
                if (kGate) {
                    v[i] = gated<kPrecise>(v[i], widen<T>(x[p.k + i * 32]));
                }
            }
        }
    }
    // the four blocks' largest, of a block in each eight lanes: every exchange halves how many a lane carries
    float m[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        m[b] = max_nan(max_nan(fabsf(v[4 * b]), fabsf(v[4 * b + 1])), max_nan(fabsf(v[4 * b + 2]), fabsf(v[4 * b + 3])));
    }
    const bool upper = (lane & 16) != 0, odd = (lane & 8) != 0;
    const float keep0 = upper ? m[2] : m[0], give0 = upper ? m[0] : m[2], keep1 = upper ? m[3] : m[1], give1 = upper ? m[1] : m[3];
    const float two0 = max_nan(keep0, __shfl_xor_sync(0xffffffffu, give0, 16)), two1 = max_nan(keep1, __shfl_xor_sync(0xffffffffu, give1, 16));
    float most = max_nan(odd ? two1 : two0, __shfl_xor_sync(0xffffffffu, odd ? two0 : two1, 8));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    most = max_nan(most, kLeast);
    const float up = kE4m3Most / most;
    const int kb = c0 / kScaleBlock + lane / 8;
    if ((lane & 7) == 0 && kb * kScaleBlock < p.k) {
        p.scale[row * p.s_row + kb * p.s_col] = most / kE4m3Most;
    }
    float up_of[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        up_of[b] = __shfl_sync(0xffffffffu, up, 8 * b);
    }
    if (whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            to[i * 32] = static_cast<unsigned char>(e4m3x2(v[i] * up_of[i / 4], 0.0f));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i * 32 < left) {
                to[i * 32] = static_cast<unsigned char>(e4m3x2(v[i] * up_of[i / 4], 0.0f));
            }
        }
    }
}

// One CTA per 128 x 128 block, for weights, once per layer: a warp takes 16 rows, a lane 4 columns.  11008 x 4096 bf16 values take 352 us
// (0.4 TB/s: elements of 2 bytes read and 1 byte written one by one), more than ten times what rows take; nothing waits for it.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const __grid_constant__ QuantizeParams p)
{
    __shared__ float warps[8];
    const int blocks_k = (p.k + kScaleBlock - 1) / kScaleBlock;
    const int rb = static_cast<int>(blockIdx.x / blocks_k), kb = static_cast<int>(blockIdx.x % blocks_k);
    const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
    const T *x = static_cast<const T *>(p.x);
    pdl_launch_dependents();
    pdl_wait();
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
    if (p.block_rows != 1) {
        const long long blocks = (p.rows + kScaleBlock - 1) / kScaleBlock * blocks_k;
        if (blocks > 0x7fffffffll) {
            return cudaErrorInvalidConfiguration;
        }
        return launch_chained(quantize_blocks_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, 1u, p);
    }
    const long long elem = sizeof(T);
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.q)) & 15u) == 0 && p.x_ld * elem % 16 == 0 &&
                         p.q_ld % 16 == 0 && (p.gate == 0 || p.k * elem % 16 == 0);
    const long long units = aligned ? p.rows * blocks_k : p.rows * ((blocks_k + 3) / 4);
    if (units > 0xffffff00ll) {
        return cudaErrorInvalidConfiguration;
    }
    const dim3 grid(static_cast<unsigned>(aligned ? (units + 15) / 16 : (units + 3) / 4));
    if (aligned) {
        return p.gate != 0 ? launch_chained(quantize_rows_kernel<T, true>, grid, dim3(128), 0, stream, 1u, p)
                           : launch_chained(quantize_rows_kernel<T, false>, grid, dim3(128), 0, stream, 1u, p);
    }
    return p.gate != 0 ? launch_chained(quantize_any_kernel<T, true>, grid, dim3(128), 0, stream, 1u, p)
                       : launch_chained(quantize_any_kernel<T, false>, grid, dim3(128), 0, stream, 1u, p);
}

}  // namespace

cudaError_t launch_quantize(const QuantizeParams &p, cudaStream_t stream)
{
    switch (p.x_dtype) {
        case KUDNN_B200_F32: return launch_typed<float>(p, stream);
        case KUDNN_B200_F16: return launch_typed<__half>(p, stream);
        default: return launch_typed<__nv_bfloat16>(p, stream);
    }
}

}  // namespace kb
