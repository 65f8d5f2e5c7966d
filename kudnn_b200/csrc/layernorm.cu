// Kernels of layer normalisation (layernorm.cuh).  Both directions read every input once and write every output once: a row stays in registers
// between the reduction and the result.  The variance is taken about the mean that is already known, not as a difference of two sums.
//
// Rows are read and written in pieces of 16 bytes that begin on 16-byte boundaries, whatever the row's own address: its first and last piece
// are then partly its neighbours' (read, never written).  All rows of a CTA are a multiple of `period` rows apart, so that they begin equally far
// into a piece and one copy of scale and shift in shared memory, moved by as much, serves all of them.
#include "layernorm.cuh"

#include <algorithm>
#include <type_traits>

namespace kb {

namespace {

constexpr int kMostThreads = 512;
constexpr int kMostShared = 160 * 1024;
constexpr int kRowWarps = 4;     // rows of a CTA at a time where a warp takes a row
constexpr int kMostParts = 592;  // CTAs of a backward pass, each with sums of its own: four per SM

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
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}

template <typename T>
constexpr int kPer = 16 / sizeof(T);  // elements of a piece

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &q, float (&v)[kPer<T>])
{
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (sizeof(T) == 4) {
            v[j] = __uint_as_float(w[j]);
        } else if (std::is_same<T, __nv_bfloat16>::value) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[(2 * j + 1) % kPer<T>] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
            v[2 * j] = f.x;
            v[(2 * j + 1) % kPer<T>] = f.y;
        }
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[kPer<T>])
{
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (sizeof(T) == 4) {
            w[j] = __float_as_uint(v[j]);
        } else if (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[(2 * j + 1) % kPer<T>]);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __floats2half2_rn(v[2 * j], v[(2 * j + 1) % kPer<T>]);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sums of two values over the threads of a row: a warp, or the CTA.  Consecutive calls take turns between two buffers, so that one barrier
// does: who writes a buffer again has passed the barrier of the call in between, which nobody reached before reading it.  Fixed order.
template <bool kWarp>
__device__ __forceinline__ float2 row_sum(float a, float b, float2 (*scratch)[kMostThreads / 32], int &turn)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (kWarp) {
        return make_float2(a, b);
    }
    float2 *buffer = scratch[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
        buffer[threadIdx.x >> 5] = make_float2(a, b);
    }
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    float2 s = lane < warps ? buffer[lane] : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int o = kMostThreads / 64; o > 0; o >>= 1) {
        s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    s.x = __shfl_sync(0xffffffffu, s.x, 0);
    s.y = __shfl_sync(0xffffffffu, s.y, 0);
    return s;
}

// The piece `c` of a row that begins `skew` elements into its first piece: elements [lo, hi) of it are the row's.
template <typename T>
struct Span {
    int lo, hi;
    __device__ __forceinline__ Span(int c, int skew, int axis)
        : lo(c == 0 ? skew : 0), hi(min(kPer<T>, axis + skew - c * kPer<T>))
    {
    }
    __device__ __forceinline__ bool whole() const { return lo == 0 && hi == kPer<T>; }
};

template <typename T>
__device__ __forceinline__ void store_piece(T *row, int c, const Span<T> &s, bool whole, const float (&v)[kPer<T>])
{
    if (whole) {
        reinterpret_cast<uint4 *>(row)[c] = pack<T>(v);
    } else {
#pragma unroll
        for (int j = 0; j < kPer<T>; ++j) {
            if (j >= s.lo && j < s.hi) {
                row[c * kPer<T> + j] = narrow<T>(v[j]);
            }
        }
    }
}

// elements in the pieces of a row wherever it begins
template <typename T>
__host__ __device__ __forceinline__ int most_slots(int axis)
{
    return (axis + 2 * kPer<T> - 2) / kPer<T> * kPer<T>;
}

// Scale or shift, moved by the skew, into shared memory (nothing given: `none`).
template <typename P>
__device__ __forceinline__ void stage(P *to, const void *from, int skew, int axis, int slots, float none, int lane, int lanes)
{
    for (int i = lane; i < slots; i += lanes) {
        const int e = i - skew;
        to[i] = from != nullptr && e >= 0 && e < axis ? static_cast<const P *>(from)[e] : narrow<P>(none);
    }
}

// kPer<T> values of P from shared memory, 16 bytes at a time
template <typename T, typename P>
__device__ __forceinline__ void fetch(const P *from, int c, float (&v)[kPer<T>])
{
    constexpr int kReads = kPer<T> / kPer<P>;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
        float part[kPer<P>];
        unpack<P>(reinterpret_cast<const uint4 *>(from)[c * kReads + i], part);
#pragma unroll
        for (int j = 0; j < kPer<P>; ++j) {
            v[(i * kPer<P> + j) % kPer<T>] = part[j];
        }
    }
}

// Who takes a row: a warp of kRowWarps, or the CTA.
template <bool kWarp>
struct Team {
    int lane, lanes, index;
    long long first, step;
    __device__ __forceinline__ Team()
        : lane(static_cast<int>(threadIdx.x) & (kWarp ? 31 : 0x3ff)),
          lanes(kWarp ? 32 : static_cast<int>(blockDim.x)),
          index(kWarp ? static_cast<int>(threadIdx.x) >> 5 : 0),
          first(kWarp ? blockIdx.x * static_cast<long long>(kRowWarps) + index : blockIdx.x),
          step(kWarp ? gridDim.x * static_cast<long long>(kRowWarps) : gridDim.x)
    {
    }
    __device__ __forceinline__ void sync() const
    {
        if (kWarp) {
            __syncwarp();
        } else {
            __syncthreads();
        }
    }
};

// kWarp: a warp per row, otherwise a CTA; kN pieces per thread.  Two rows at a time: twice the bytes in flight, and scale and shift are read from
// shared memory once for both.  kEdge: some row has pieces that are only partly its own.
template <typename T, typename P, int kN, bool kEdge, bool kWarp>
__global__ void __launch_bounds__(kMostThreads) layernorm_kernel(const __grid_constant__ LayernormParams p)
{
    extern __shared__ uint4 shared[];
    __shared__ float2 scratch[2][kMostThreads / 32];
    constexpr int kV = kPer<T>;
    const Team<kWarp> team;
    const int lane = team.lane, lanes = team.lanes;
    const long long step = team.step;
    long long row = team.first;
    const T *x0 = static_cast<const T *>(p.x);
    T *y0 = static_cast<T *>(p.y);
    const int skew = kEdge ? static_cast<int>(reinterpret_cast<uintptr_t>(x0 + row * p.x_ld) & 15u) / static_cast<int>(sizeof(T)) : 0;
    const int pieces = (p.axis + skew + kV - 1) / kV, slots = pieces * kV;
    // teams of a CTA have copies of their own where their rows may begin elsewhere
    P *scale = reinterpret_cast<P *>(shared) + (kWarp && kEdge ? team.index * 2ll * most_slots<T>(p.axis) : 0);
    P *shift = scale + slots;
    int turn = 0;
    pdl_launch_dependents();
    pdl_wait();
    uint4 q[2][kN];
    auto load = [&](long long r, uint4(&to)[kN]) {
        const uint4 *from = reinterpret_cast<const uint4 *>(x0 + r * p.x_ld - skew);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = lane + i * lanes;
            to[i] = c < pieces ? from[c] : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    bool staged = false;
    const float inv_axis = 1.0f / static_cast<float>(p.axis);
    for (; row < p.rows; row += 2 * step) {
        const bool two = row + step < p.rows;
        load(row, q[0]);
        if (two) {
            load(row + step, q[1]);
        }
        if (!staged) {
            stage(scale, p.scale, skew, p.axis, slots, 1.0f, lane, lanes);
            stage(shift, p.shift, skew, p.axis, slots, 0.0f, lane, lanes);
            staged = true;
            team.sync();
        }
        float mean[2], var[2];
        if (p.given != 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                mean[k] = k == 0 || two ? p.mean[row + k * step] : 0.0f;
                var[k] = k == 0 || two ? p.variance[row + k * step] : 0.0f;
            }
        } else {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (k == 0 || two) {
#pragma unroll
                    for (int i = 0; i < kN; ++i) {
                        float v[kV];
                        unpack<T>(q[k][i], v);
                        const Span<T> span(lane + i * lanes, skew, p.axis);
                        const bool whole = !kEdge || span.whole();
#pragma unroll
                        for (int j = 0; j < kV; ++j) {
                            s[k] += whole || (j >= span.lo && j < span.hi) ? v[j] : 0.0f;
                        }
                    }
                }
            }
            float2 total = row_sum<kWarp>(s[0], s[1], scratch, turn);
            mean[0] = total.x * inv_axis;
            mean[1] = total.y * inv_axis;
            s[0] = s[1] = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (k == 0 || two) {
#pragma unroll
                    for (int i = 0; i < kN; ++i) {
                        float v[kV];
                        unpack<T>(q[k][i], v);
                        const int c = lane + i * lanes;
                        const Span<T> span(c, skew, p.axis);
                        const bool whole = kEdge ? span.whole() : c < pieces;
#pragma unroll
                        for (int j = 0; j < kV; ++j) {
                            const float d = v[j] - mean[k];
                            const bool mine = whole || (kEdge && j >= span.lo && j < span.hi);
                            s[k] = mine ? fmaf(d, d, s[k]) : s[k];
                        }
                    }
                }
            }
            total = row_sum<kWarp>(s[0], s[1], scratch, turn);
            var[0] = total.x * inv_axis;
            var[1] = total.y * inv_axis;
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if ((k == 0 || two) && p.mean != nullptr) {
                        p.mean[row + k * step] = mean[k];
                    }
                    if ((k == 0 || two) && p.variance != nullptr) {
                        p.variance[row + k * step] = var[k];
                    }
                }
            }
        }
        const float r[2] = {1.0f / sqrtf(var[0] + p.eps), 1.0f / sqrtf(var[1] + p.eps)};
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = lane + i * lanes;
            if (c < pieces) {
                float a[kV], b[kV];
                fetch<T, P>(scale, c, a);
                fetch<T, P>(shift, c, b);
                const Span<T> span(c, skew, p.axis);
                const bool whole = !kEdge || span.whole();
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (k == 0 || two) {
                        float v[kV];
                        unpack<T>(q[k][i], v);
#pragma unroll
                        for (int j = 0; j < kV; ++j) {
                            v[j] = fmaf((v[j] - mean[k]) * r[k], a[j], b[j]);
                        }
                        store_piece<T>(y0 + (row + k * step) * p.y_ld - skew, c, span, whole, v);
                    }
                }
            }
        }
    }
}

// Rows longer than the registers of a CTA hold, or whose x and y do not begin equally far into a piece: element by element, x read three times.
template <typename T, typename P>
__global__ void __launch_bounds__(kMostThreads) layernorm_any_kernel(const __grid_constant__ LayernormParams p)
{
    __shared__ float2 scratch[2][kMostThreads / 32];
    int turn = 0;
    pdl_launch_dependents();
    pdl_wait();
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(p.x) + row * p.x_ld;
        T *y = static_cast<T *>(p.y) + row * p.y_ld;
        float mean, var;
        if (p.given != 0) {
            mean = p.mean[row];
            var = p.variance[row];
        } else {
            float s = 0.0f;
            for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
                s += widen<T>(x[i]);
            }
            mean = row_sum<false>(s, 0.0f, scratch, turn).x / static_cast<float>(p.axis);
            s = 0.0f;
            for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
                const float d = widen<T>(x[i]) - mean;
                s = fmaf(d, d, s);
            }
            var = row_sum<false>(s, 0.0f, scratch, turn).x / static_cast<float>(p.axis);
            if (threadIdx.x == 0) {
                if (p.mean != nullptr) {
                    p.mean[row] = mean;
                }
                if (p.variance != nullptr) {
                    p.variance[row] = var;
                }
            }
        }
        const float r = 1.0f / sqrtf(var + p.eps);
        for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
            const float a = p.scale != nullptr ? widen<P>(static_cast<const P *>(p.scale)[i]) : 1.0f;
            const float b = p.shift != nullptr ? widen<P>(static_cast<const P *>(p.shift)[i]) : 0.0f;
            y[i] = narrow<T>(fmaf((widen<T>(x[i]) - mean) * r, a, b));
        }
    }
}

// The gradient: a row at a time per CTA or warp, the next row's x and dy on their way while this one is summed.  The sums over rows of dscale and dshift
// stay in registers, each thread its own columns; every CTA leaves one set of them, added up in a fixed order by column_sums_kernel.
template <typename T, typename P, int kN, bool kEdge, bool kWarp>
__global__ void __launch_bounds__(kMostThreads) layernorm_backward_kernel(const __grid_constant__ LayernormParams p)
{
    extern __shared__ uint4 shared[];
    __shared__ float2 scratch[2][kMostThreads / 32];
    constexpr int kV = kPer<T>;
    const Team<kWarp> team;
    const int lane = team.lane, lanes = team.lanes;
    const long long step = team.step;
    long long row = team.first;
    const T *x0 = static_cast<const T *>(p.x), *dy0 = static_cast<const T *>(p.dy);
    const int skew = kEdge ? static_cast<int>(reinterpret_cast<uintptr_t>(x0 + row * p.x_ld) & 15u) / static_cast<int>(sizeof(T)) : 0;
    const int pieces = (p.axis + skew + kV - 1) / kV, slots = pieces * kV;
    P *scale = reinterpret_cast<P *>(shared) + (kWarp && kEdge ? static_cast<long long>(team.index) * most_slots<T>(p.axis) : 0);
    int turn = 0;
    pdl_launch_dependents();
    pdl_wait();
    uint4 x_next[kN], dy_next[kN];
    float mean_next = 0.0f, var_next = 0.0f;
    auto load = [&](long long r) {
        const uint4 *x = reinterpret_cast<const uint4 *>(x0 + r * p.x_ld - skew), *dy = reinterpret_cast<const uint4 *>(dy0 + r * p.dy_ld - skew);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = lane + i * lanes;
            x_next[i] = c < pieces ? x[c] : make_uint4(0u, 0u, 0u, 0u);
            dy_next[i] = c < pieces ? dy[c] : make_uint4(0u, 0u, 0u, 0u);
        }
        mean_next = p.mean[r];
        var_next = p.variance[r];
    };
    float sum_scale[kN][kV], sum_shift[kN][kV];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
#pragma unroll
        for (int j = 0; j < kV; ++j) {
            sum_scale[i][j] = sum_shift[i][j] = 0.0f;
        }
    }
    if (row < p.rows) {
        load(row);
    }
    stage(scale, p.scale, skew, p.axis, slots, 1.0f, lane, lanes);
    team.sync();
    const float inv_axis = 1.0f / static_cast<float>(p.axis);
    for (; row < p.rows; row += step) {
        uint4 x[kN], dy[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            x[i] = x_next[i];
            dy[i] = dy_next[i];
        }
        const float mean = mean_next, r = 1.0f / sqrtf(var_next + p.eps);
        if (row + step < p.rows) {
            load(row + step);
        }
        float of_g = 0.0f, of_gx = 0.0f;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = lane + i * lanes;
            const Span<T> span(c, skew, p.axis);
            const bool whole = kEdge ? span.whole() : c < pieces;
            if (whole || (kEdge && span.lo < span.hi)) {
                float xv[kV], dv[kV], a[kV];
                unpack<T>(x[i], xv);
                unpack<T>(dy[i], dv);
                fetch<T, P>(scale, c, a);
#pragma unroll
                for (int j = 0; j < kV; ++j) {
                    const bool mine = whole || (j >= span.lo && j < span.hi);
                    const float d = mine ? dv[j] : 0.0f, xh = mine ? (xv[j] - mean) * r : 0.0f, g = d * a[j];
                    of_g += g;
                    of_gx = fmaf(g, xh, of_gx);
                    sum_scale[i][j] = fmaf(d, xh, sum_scale[i][j]);
                    sum_shift[i][j] += d;
                }
            }
        }
        if (p.y != nullptr) {
            if (p.given == 0) {
                const float2 total = row_sum<kWarp>(of_g, of_gx, scratch, turn);
                of_g = total.x * inv_axis;
                of_gx = total.y * inv_axis;
            } else {
                of_g = of_gx = 0.0f;
            }
            T *to = static_cast<T *>(p.y) + row * p.y_ld - skew;
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = lane + i * lanes;
                if (c < pieces) {
                    float xv[kV], dv[kV], a[kV];
                    unpack<T>(x[i], xv);
                    unpack<T>(dy[i], dv);
                    fetch<T, P>(scale, c, a);
                    const Span<T> span(c, skew, p.axis);
#pragma unroll
                    for (int j = 0; j < kV; ++j) {
                        const float xh = (xv[j] - mean) * r, g = dv[j] * a[j];
                        dv[j] = p.given != 0 ? r * g : r * (g - of_g - xh * of_gx);
                    }
                    store_piece<T>(to, c, span, !kEdge || span.whole(), dv);
                }
            }
        }
    }
    if (p.partial == nullptr) {
        return;
    }
    float *to = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.axis;
    float *sums = kWarp ? reinterpret_cast<float *>(shared) : to;  // the warps' sums are added up one after the other
#pragma unroll 1
    for (int turn_of = 0; turn_of < (kWarp ? kRowWarps : 1); ++turn_of) {
        if (kWarp) {
            __syncthreads();
        }
        if (team.index == turn_of) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = lane + i * lanes;
                if (c < pieces) {
#pragma unroll
                    for (int j = 0; j < kV; ++j) {
                        const int e = c * kV + j - skew;
                        if (e >= 0 && e < p.axis) {
                            sums[e] = sum_scale[i][j] + (turn_of == 0 ? 0.0f : sums[e]);
                            sums[p.axis + e] = sum_shift[i][j] + (turn_of == 0 ? 0.0f : sums[p.axis + e]);
                        }
                    }
                }
            }
        }
    }
    if (kWarp) {
        __syncthreads();
        for (int e = static_cast<int>(threadIdx.x); e < 2 * p.axis; e += static_cast<int>(blockDim.x)) {
            to[e] = sums[e];
        }
    }
}

// As layernorm_any_kernel: the sums over a CTA's rows column by column, then dx of them, which may lie where x or dy does.
template <typename T, typename P>
__global__ void __launch_bounds__(kMostThreads) layernorm_backward_any_kernel(const __grid_constant__ LayernormParams p)
{
    __shared__ float2 scratch[2][kMostThreads / 32];
    int turn = 0;
    pdl_launch_dependents();
    pdl_wait();
    const T *x0 = static_cast<const T *>(p.x), *dy0 = static_cast<const T *>(p.dy);
    if (p.partial != nullptr) {
        float *to = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.axis;
        for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
            float of_scale = 0.0f, of_shift = 0.0f;
            for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
                const float d = widen<T>(dy0[row * p.dy_ld + i]), r = 1.0f / sqrtf(p.variance[row] + p.eps);
                of_scale = fmaf(d, (widen<T>(x0[row * p.x_ld + i]) - p.mean[row]) * r, of_scale);
                of_shift += d;
            }
            to[i] = of_scale;
            to[p.axis + i] = of_shift;
        }
    }
    if (p.y != nullptr) {
        for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
            const T *x = x0 + row * p.x_ld, *dy = dy0 + row * p.dy_ld;
            T *dx = static_cast<T *>(p.y) + row * p.y_ld;
            const float mean = p.mean[row], r = 1.0f / sqrtf(p.variance[row] + p.eps);
            float of_g = 0.0f, of_gx = 0.0f;
            if (p.given == 0) {
                for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
                    const float a = p.scale != nullptr ? widen<P>(static_cast<const P *>(p.scale)[i]) : 1.0f;
                    const float g = widen<T>(dy[i]) * a;
                    of_g += g;
                    of_gx = fmaf(g, (widen<T>(x[i]) - mean) * r, of_gx);
                }
                const float2 total = row_sum<false>(of_g, of_gx, scratch, turn);
                of_g = total.x / static_cast<float>(p.axis);
                of_gx = total.y / static_cast<float>(p.axis);
            }
            for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
                const float a = p.scale != nullptr ? widen<P>(static_cast<const P *>(p.scale)[i]) : 1.0f;
                const float g = widen<T>(dy[i]) * a, xh = (widen<T>(x[i]) - mean) * r;
                dx[i] = narrow<T>(p.given != 0 ? r * g : r * (g - of_g - xh * of_gx));
            }
        }
    }
}

// dscale and dshift from `parts` sets of sums: a CTA of 32 columns x 8 threads, which add every eighth set each and are then added in order.
template <typename P>
__global__ void __launch_bounds__(256) column_sums_kernel(const __grid_constant__ LayernormParams p, int parts)
{
    __shared__ float sums[8][33];
    const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
    const int e = static_cast<int>(blockIdx.x) * 32 + lane;
    pdl_launch_dependents();
    pdl_wait();
    P *to = static_cast<P *>(blockIdx.y == 0 ? p.dscale : p.dshift);
    if (to == nullptr) {
        return;
    }
    float s = 0.0f;
    if (e < p.axis) {
        const float *from = p.partial + static_cast<long long>(blockIdx.y) * p.axis + e;
        for (int i = warp; i < parts; i += 8) {
            s += from[static_cast<long long>(i) * 2 * p.axis];
        }
    }
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && e < p.axis) {
        for (int i = 1; i < 8; ++i) {
            s += sums[i][lane];
        }
        to[e] = narrow<P>(s);
    }
}

// Rows a CTA's rows are apart at least, so that all of them begin equally far into a 16-byte piece; 0: x and another tensor do not.
int period_of(const LayernormParams &p, int elem, bool backward)
{
    const long long pitch = p.x_ld * elem;
    auto differs = [&](const void *t, long long ld) {
        return t != nullptr &&
               (((reinterpret_cast<uintptr_t>(t) ^ reinterpret_cast<uintptr_t>(p.x)) & 15u) != 0 || (p.rows > 1 && (ld * elem - pitch) % 16 != 0));
    };
    if (differs(p.y, p.y_ld) || (backward && differs(p.dy, p.dy_ld))) {
        return 0;
    }
    int period = 1;
    while (pitch * period % 16 != 0) {
        period *= 2;
    }
    return period;
}

struct Shape {
    int threads, pieces, grid;
    size_t shared;
    bool edge, warp;
};

// false: the general kernel
bool shape_of(const LayernormParams &p, int elem, int param_elem, bool backward, int sm_count, Shape *s)
{
    const int period = period_of(p, elem, backward);
    if (period == 0) {
        return false;
    }
    const int per = 16 / elem;
    s->edge = period != 1 || (reinterpret_cast<uintptr_t>(p.x) & 15u) != 0 || p.axis % per != 0;
    const long long most = (static_cast<long long>(p.axis) + (s->edge ? 2 * per - 2 : per - 1)) / per;  // pieces of a row
    s->warp = most <= 128;
    s->pieces = most <= 32 ? 1 : most <= 64 ? 2 : s->warp ? 4 : most <= 512 ? 2 : 4;
    const long long threads = s->warp ? 32 * kRowWarps : ((most + s->pieces - 1) / s->pieces + 31) / 32 * 32;
    long long shared = most * per * param_elem * (backward ? 1 : 2) * (s->warp && s->edge ? kRowWarps : 1);
    if (backward && s->warp) {
        shared = std::max<long long>(shared, 8ll * p.axis);
    }
    if (threads > kMostThreads || shared > kMostShared) {
        return false;
    }
    s->threads = static_cast<int>(threads);
    s->shared = static_cast<size_t>(shared);
    const int rows = s->warp ? kRowWarps : 1;
    const long long per_sm = std::min<long long>(std::min<long long>((backward ? 512 : 1536) / threads, (200 * 1024) / (shared + 1024)), 24);
    long long grid = std::max<long long>(1, per_sm) * sm_count;
    if (backward) {
        grid = std::min<long long>(grid, kMostParts);
    }
    grid = grid / period * period;
    s->grid = static_cast<int>(std::min<long long>(grid, (p.rows + rows - 1) / rows));
    return true;
}

template <typename T, typename P, int kN, bool kEdge, bool kWarp>
cudaError_t launch_shape(const LayernormParams &p, const Shape &s, bool backward, cudaStream_t stream)
{
    void (*kernel)(LayernormParams) = backward ? layernorm_backward_kernel<T, P, kN, kEdge, kWarp> : layernorm_kernel<T, P, kN, kEdge, kWarp>;
    if (s.shared > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
        if (e != cudaSuccess) {
            return e;
        }
    }
    return launch_chained(kernel, dim3(s.grid), dim3(s.threads), s.shared, stream, 1u, p);
}

template <typename T, typename P, bool kEdge>
cudaError_t launch_edge(const LayernormParams &p, const Shape &s, bool backward, cudaStream_t stream)
{
    if (s.warp) {
        return s.pieces == 1   ? launch_shape<T, P, 1, kEdge, true>(p, s, backward, stream)
               : s.pieces == 2 ? launch_shape<T, P, 2, kEdge, true>(p, s, backward, stream)
                               : launch_shape<T, P, 4, kEdge, true>(p, s, backward, stream);
    }
    return s.pieces == 2 ? launch_shape<T, P, 2, kEdge, false>(p, s, backward, stream) : launch_shape<T, P, 4, kEdge, false>(p, s, backward, stream);
}

template <typename T, typename P>
cudaError_t launch_typed(const LayernormParams &p, int sm_count, bool backward, cudaStream_t stream)
{
    Shape s;
    cudaError_t e;
    if (shape_of(p, sizeof(T), sizeof(P), backward, sm_count, &s)) {
        e = s.edge ? launch_edge<T, P, true>(p, s, backward, stream) : launch_edge<T, P, false>(p, s, backward, stream);
    } else {
        s.grid = static_cast<int>(std::min<long long>(p.rows, kMostParts));
        e = launch_chained(backward ? layernorm_backward_any_kernel<T, P> : layernorm_any_kernel<T, P>, dim3(s.grid), dim3(kMostThreads), 0, stream, 1u, p);
    }
    if (e != cudaSuccess || !backward || p.partial == nullptr) {
        return e;
    }
    return launch_chained(column_sums_kernel<P>, dim3((p.axis + 31) / 32, 2), dim3(256), 0, stream, 1u, p, s.grid);
}

cudaError_t launch(const LayernormParams &p, int sm_count, bool backward, cudaStream_t stream)
{
    switch (p.dtype) {
        case KUDNN_B200_F32: return launch_typed<float, float>(p, sm_count, backward, stream);
        case KUDNN_B200_F16:
            return p.param_dtype == KUDNN_B200_F32 ? launch_typed<__half, float>(p, sm_count, backward, stream)
                                                   : launch_typed<__half, __half>(p, sm_count, backward, stream);
        default:
            return p.param_dtype == KUDNN_B200_F32 ? launch_typed<__nv_bfloat16, float>(p, sm_count, backward, stream)
                                                   : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, sm_count, backward, stream);
    }
}

}  // namespace

cudaError_t launch_layernorm(const LayernormParams &p, int sm_count, cudaStream_t stream)
{
    return launch(p, sm_count, false, stream);
}

long long layernorm_backward_floats(long long rows, long long axis)
{
    return std::min<long long>(rows, kMostParts) * 2 * axis;
}

cudaError_t launch_layernorm_backward(const LayernormParams &p, int sm_count, cudaStream_t stream)
{
    return launch(p, sm_count, true, stream);
}

}  // namespace kb
