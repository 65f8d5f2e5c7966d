// Kernels of layer normalisation (layernorm.cuh).  Both directions read every input once and write every output once.  The variance is taken about the
// mean that is already known, not as a difference of two sums.
//
// Rows are read and written in pieces of 16 bytes that begin on 16-byte boundaries, whatever the row's own address.  All rows of a CTA are a multiple
// of `period` rows apart, so that they begin equally far into a piece and one copy of scale and shift in shared memory, moved by as much, serves
// all of them.
#include "layernorm.cuh"

#include <algorithm>
#include <type_traits>

namespace kb {

namespace {

constexpr int kMostThreads = 512;
constexpr int kMostShared = 200 * 1024;
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

// Two fp32 values in one 64-bit register pair, for the instructions that take both at once
using Two = unsigned long long;
__device__ __forceinline__ Two two(float lo, float hi)
{
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 both(Two v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ Two add(Two a, Two b)
{
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two mul(Two a, Two b)
{
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c)
{
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &q, Two (&v)[kPer<T> / 2])
{
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < kPer<T> / 2; ++j) {
        if (sizeof(T) == 4) {
            v[j] = two(__uint_as_float(w[2 * j % 4]), __uint_as_float(w[(2 * j + 1) % 4]));
        } else if (std::is_same<T, __nv_bfloat16>::value) {
            v[j] = two(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
            v[j] = two(f.x, f.y);
        }
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const Two (&v)[kPer<T> / 2])
{
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < kPer<T> / 2; ++j) {
        const float2 f = both(v[j]);
        if (sizeof(T) == 4) {
            w[2 * j % 4] = __float_as_uint(f.x);
            w[(2 * j + 1) % 4] = __float_as_uint(f.y);
        } else if (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __floats2half2_rn(f.x, f.y);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sum over a warp, in all its lanes.
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// 1 / sqrt(v): the hardware's and a step of Newton's iteration, 2^-23 off at most; the zero and the infinity of the hardware's stay
__device__ __forceinline__ float inverse_root(float v)
{
    const float r = rsqrtf(v);
    const float better = fmaf(r * 0.5f, fmaf(-v * r, r, 1.0f), r);
    return r > 0.0f && r < 3e38f ? better : r;
}

// Sums of two values over the CTA, in a fixed order.  Consecutive calls take turns between two buffers, so that one barrier does: who writes a
// buffer again has passed the barrier of the call in between, which nobody reached before reading it.
__device__ __forceinline__ float2 block_sum(float a, float b, float2 (*scratch)[kMostThreads / 32], int &turn)
{
    a = warp_sum(a);
    b = warp_sum(b);
    float2 *buffer = scratch[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
        buffer[threadIdx.x >> 5] = make_float2(a, b);
    }
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
    const float2 s = lane < warps ? buffer[lane] : make_float2(0.0f, 0.0f);
    return make_float2(warp_sum(s.x), warp_sum(s.y));
}

// Scale and shift in shared memory: where 16 bytes of a row's type hold more elements than 16 bytes of theirs, the first halves of all pieces'
// worth and behind them the second ones, so that a warp reads 16 bytes per lane side by side.
template <typename T, typename P>
__device__ __forceinline__ int param_slot(int i, int whole)
{
    constexpr int kReads = kPer<T> / kPer<P>;
    return kReads == 1 ? i : i % kPer<T> / kPer<P> * (whole * kPer<P>) + i / kPer<T> * kPer<P> + i % kPer<P>;
}

template <typename T, typename P>
__device__ __forceinline__ void stage_params(P *to, const void *from, int head, int whole, float none)
{
    for (int i = static_cast<int>(threadIdx.x); i < whole * kPer<T>; i += static_cast<int>(blockDim.x)) {
        to[param_slot<T, P>(i, whole)] = from != nullptr ? static_cast<const P *>(from)[head + i] : narrow<P>(none);
    }
}

// kPer<T> values of P, those of piece c
template <typename T, typename P>
__device__ __forceinline__ void fetch(const P *from, int c, int whole, Two (&v)[kPer<T> / 2])
{
    constexpr int kReads = kPer<T> / kPer<P>, kPairs = kPer<P> / 2;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
        Two part[kPairs];
        unpack<P>(reinterpret_cast<const uint4 *>(from)[i * whole + c], part);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            v[(i * kPairs + j) % (kPer<T> / 2)] = part[j];
        }
    }
}

// How rows are dealt out.  A team of `warps` warps takes a row, a CTA has `teams` of them.  CTA b takes rows of the class b % period, so that all
// of its rows begin equally far into a piece.
struct Teams {
    int warps, teams, period;
    int row_bytes;  // of shared memory per row: its whole pieces
    int stages;     // backward: rows of a team in shared memory
};

// A thread's place in them.
template <typename T, bool kEdge>
struct Place {
    int lanes, team, lane;
    long long row, step;    // first row, and from one to the next
    int head, whole, tail;  // elements in front of the first whole piece, whole pieces, elements behind
    bool single;            // this lane has one of those elements: number `at`
    int at;
    __device__ __forceinline__ Place(const LayernormParams &p, const Teams &of)
        : lanes(of.warps * 32), team(static_cast<int>(threadIdx.x) / lanes), lane(static_cast<int>(threadIdx.x) - team * lanes)
    {
        constexpr int kV = kPer<T>;
        const int in_class = static_cast<int>(blockIdx.x) % of.period;
        step = static_cast<long long>(gridDim.x) * of.teams;  // gridDim.x is a multiple of the period
        row = in_class + static_cast<long long>(of.period) * (static_cast<long long>(blockIdx.x) / of.period * of.teams + team);
        const int skew =
            kEdge ? static_cast<int>(reinterpret_cast<uintptr_t>(static_cast<const T *>(p.x) + in_class * p.x_ld) & 15u) / static_cast<int>(sizeof(T)) : 0;
        head = min(p.axis, (kV - skew) % kV);
        whole = (p.axis - head) / kV;
        tail = p.axis - head - whole * kV;
        single = kEdge && (lane < head || (lane >= 16 && lane - 16 < tail));
        at = lane < 16 ? lane : p.axis - tail + lane - 16;
    }
};

// Sum over a team's warps, in a fixed order; consecutive calls take turns between two buffers (see block_sum).
__device__ __forceinline__ float2 team_sum(float a, float b, const Teams &of, int team, float2 (*scratch)[kMostThreads / 32], int &turn)
{
    a = warp_sum(a);
    b = warp_sum(b);
    if (of.warps == 1) {
        return make_float2(a, b);
    }
    float2 *buffer = scratch[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
        buffer[threadIdx.x >> 5] = make_float2(a, b);
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(of.warps * 32) : "memory");
    float2 s = make_float2(0.0f, 0.0f);
    for (int w = 0; w < of.warps; ++w) {
        const float2 v = buffer[team * of.warps + w];
        s.x += v.x;
        s.y += v.y;
    }
    return s;
}

__device__ __forceinline__ void copy_piece(unsigned char *to, const void *from)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}

// A row lies in shared memory (cp.async, the next one on its way meanwhile; each thread reads back only what it copied itself) and is gone through
// three times: mean, squares about it, result.  What bounds it is instructions beside HBM: the fewer threads a row has, the fewer of them compute
// the row's statistics, so teams are as small as sixteen warps per CTA allow, and sums and products are taken two at a time.
// 16384 x 8192 bf16: 101 to 109 us, 4.9 to 5.3 TB/s (a CTA per row, one value at a time: 122); 9001 x 4099 f16 with fp32 scale and shift: 44 us, 3.4 TB/s
// (58); 8 x 4096: 4.2 us; 8192 x 8192 fp32: 96 us, 5.6 TB/s.  kEdge: the elements in front of the first whole piece and behind the
// last one are single lanes' own, in registers.
template <typename T, typename P, bool kEdge>
__global__ void __launch_bounds__(kMostThreads, 2) layernorm_kernel(const __grid_constant__ LayernormParams p, const __grid_constant__ Teams of)
{
    extern __shared__ uint4 shared[];
    __shared__ float2 scratch[2][kMostThreads / 32];
    constexpr int kV = kPer<T>;
    const Place<T, kEdge> place(p, of);
    const int lanes = place.lanes, lane = place.lane, head = place.head, whole = place.whole, at = place.at, slots = whole * kV;
    const bool single = place.single;
    const long long step = place.step;
    long long row = place.row;
    const T *x0 = static_cast<const T *>(p.x);
    T *y0 = static_cast<T *>(p.y);
    P *scale = reinterpret_cast<P *>(shared), *shift = scale + slots;
    unsigned char *ring = reinterpret_cast<unsigned char *>(shared) + (2ll * slots * sizeof(P) + 15) / 16 * 16 + place.team * 2ll * of.row_bytes;
    pdl_launch_dependents();
    pdl_wait();
    auto load = [&](long long r, int stage) {
        if (r < p.rows) {
            const uint4 *from = reinterpret_cast<const uint4 *>(x0 + r * p.x_ld + head);
            unsigned char *to = ring + stage * of.row_bytes;
            for (int c = lane; c < whole; c += lanes) {
                copy_piece(to + c * 16, from + c);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    load(row, 0);
    load(row + step, 1);
    float own = 0.0f, own_next = 0.0f, own_scale = 1.0f, own_shift = 0.0f;
    if (single) {
        own_next = row < p.rows ? widen<T>(x0[row * p.x_ld + at]) : 0.0f;
        own_scale = p.scale != nullptr ? widen<P>(static_cast<const P *>(p.scale)[at]) : 1.0f;
        own_shift = p.shift != nullptr ? widen<P>(static_cast<const P *>(p.shift)[at]) : 0.0f;
    }
    stage_params<T, P>(scale, p.scale, head, whole, 1.0f);
    stage_params<T, P>(shift, p.shift, head, whole, 0.0f);
    __syncthreads();
    int turn = 0;
    const float inv_axis = 1.0f / static_cast<float>(p.axis);
    int stage = 0;
    for (; row < p.rows; row += step) {
        if (kEdge) {
            own = own_next;
            own_next = single && row + step < p.rows ? widen<T>(x0[(row + step) * p.x_ld + at]) : 0.0f;
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        const uint4 *x = reinterpret_cast<const uint4 *>(ring + stage * of.row_bytes);
        float mean, var;
        if (p.given != 0) {
            mean = p.mean[row];
            var = p.variance[row];
        } else {
            Two s = two(kEdge ? own : 0.0f, 0.0f);
#pragma unroll 4
            for (int c = lane; c < whole; c += lanes) {
                Two v[kV / 2];
                unpack<T>(x[c], v);
#pragma unroll
                for (int j = 0; j < kV / 2; ++j) {
                    s = add(s, v[j]);
                }
            }
            float2 halves = both(s);
            mean = team_sum(halves.x + halves.y, 0.0f, of, place.team, scratch, turn).x * inv_axis;
            const float d = single ? own - mean : 0.0f;
            const Two less = two(-mean, -mean);
            s = two(d * d, 0.0f);
#pragma unroll 4
            for (int c = lane; c < whole; c += lanes) {
                Two v[kV / 2];
                unpack<T>(x[c], v);
#pragma unroll
                for (int j = 0; j < kV / 2; ++j) {
                    const Two e = add(v[j], less);
                    s = fma(e, e, s);
                }
            }
            halves = both(s);
            var = team_sum(halves.x + halves.y, 0.0f, of, place.team, scratch, turn).x * inv_axis;
            if (lane == 0) {
                if (p.mean != nullptr) {
                    p.mean[row] = mean;
                }
                if (p.variance != nullptr) {
                    p.variance[row] = var;
                }
            }
        }
        const float r = inverse_root(var + p.eps);
        T *y = y0 + row * p.y_ld;
        uint4 *to = reinterpret_cast<uint4 *>(y + head);
        const Two less = two(-mean, -mean), times = two(r, r);
#pragma unroll 2
        for (int c = lane; c < whole; c += lanes) {
            Two v[kV / 2], a[kV / 2], b[kV / 2];
            unpack<T>(x[c], v);
            fetch<T, P>(scale, c, whole, a);
            fetch<T, P>(shift, c, whole, b);
#pragma unroll
            for (int j = 0; j < kV / 2; ++j) {
                v[j] = fma(mul(add(v[j], less), times), a[j], b[j]);
            }
            to[c] = pack<T>(v);
        }
        if (single) {
            y[at] = narrow<T>(fmaf((own - mean) * r, own_scale, own_shift));
        }
        load(row + 2 * step, stage);
        stage ^= 1;
    }
}

// Rows longer than shared memory holds (fp32 from 12,801 elements on, 16 bit with fp32 parameters from 17,065, 16 bit from 25,601), or whose x and y
// do not begin equally far into a piece: element by element, x read three times.  4096 x 16384 fp32: 205 us, 2.6 TB/s; rows of a view, 16384 x
// 4096 bf16: 211 us, 1.3 TB/s.
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
            mean = block_sum(s, 0.0f, scratch, turn).x / static_cast<float>(p.axis);
            s = 0.0f;
            for (int i = static_cast<int>(threadIdx.x); i < p.axis; i += static_cast<int>(blockDim.x)) {
                const float d = widen<T>(x[i]) - mean;
                s = fmaf(d, d, s);
            }
            var = block_sum(s, 0.0f, scratch, turn).x / static_cast<float>(p.axis);
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

// The gradient, rows as in the forward pass: a thread's kN pieces of x and dy come by way of shared memory, are widened once and kept as xh and g
// between the row's sums and dx (kKeep), unless that takes too many registers (then it is widened again).  The sums over rows of dscale and dshift stay in registers, each
// thread its own columns; every CTA leaves one set of them, added up in a fixed order by column_sums_kernel.
// 16384 x 4096 bf16: 87 to 92 us, 4.4 to 4.7 TB/s; the schedulers issue in 56 % of the cycles and HBM is at 65 %, so that it is the chain of a row
// (load, sums, exchange, dx), of which a team has one at a time, that bounds it; 16 elements per thread 94.
template <typename T, typename P, int kN, bool kEdge>
__global__ void __launch_bounds__(kMostThreads) layernorm_backward_kernel(const __grid_constant__ LayernormParams p, const __grid_constant__ Teams of)
{
    extern __shared__ uint4 shared[];
    __shared__ float2 scratch[2][kMostThreads / 32];
    constexpr int kV = kPer<T>, kH = kV / 2;
    constexpr bool kKeep = kN * kV <= 16;
    const Place<T, kEdge> place(p, of);
    const int lanes = place.lanes, lane = place.lane, head = place.head, whole = place.whole, at = place.at, slots = whole * kV;
    const bool single = place.single;
    const long long step = place.step;
    long long row = place.row;
    const T *x0 = static_cast<const T *>(p.x), *dy0 = static_cast<const T *>(p.dy);
    P *scale = reinterpret_cast<P *>(shared);
    unsigned char *ring = reinterpret_cast<unsigned char *>(shared) + (static_cast<long long>(slots) * sizeof(P) + 15) / 16 * 16 +
                          place.team * 2ll * of.stages * of.row_bytes;  // [stage][x, dy]
    pdl_launch_dependents();
    pdl_wait();
    auto load = [&](long long r, int stage) {
        if (r < p.rows) {
            const uint4 *x = reinterpret_cast<const uint4 *>(x0 + r * p.x_ld + head), *dy = reinterpret_cast<const uint4 *>(dy0 + r * p.dy_ld + head);
            unsigned char *to = ring + stage * 2 * of.row_bytes;
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = lane + i * lanes;
                if (c < whole) {
                    copy_piece(to + c * 16, x + c);
                    copy_piece(to + of.row_bytes + c * 16, dy + c);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    load(row, 0);
    if (of.stages > 1) {
        load(row + step, 1);
    }
    float mean_next = 0.0f, var_next = 0.0f, x_next = 0.0f, dy_next = 0.0f;
    auto ahead = [&](long long r) {
        if (r < p.rows) {
            mean_next = p.mean[r];
            var_next = p.variance[r];
            if (single) {
                x_next = widen<T>(x0[r * p.x_ld + at]);
                dy_next = widen<T>(dy0[r * p.dy_ld + at]);
            }
        }
    };
    ahead(row);
    const float own_scale = single && p.scale != nullptr ? widen<P>(static_cast<const P *>(p.scale)[at]) : 1.0f;
    float own_sum_scale = 0.0f, own_sum_shift = 0.0f;
    Two sum_scale[kN][kH], sum_shift[kN][kH];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
#pragma unroll
        for (int j = 0; j < kH; ++j) {
            sum_scale[i][j] = sum_shift[i][j] = 0ull;
        }
    }
    stage_params<T, P>(scale, p.scale, head, whole, 1.0f);
    __syncthreads();
    const float inv_axis = 1.0f / static_cast<float>(p.axis);
    int turn = 0, stage = 0;
    for (; row < p.rows; row += step) {
        const float mean = mean_next, r = inverse_root(var_next + p.eps), own_xh = single ? (x_next - mean) * r : 0.0f, own_dy = single ? dy_next : 0.0f;
        const Two less = two(-mean, -mean), times = two(r, r);
        ahead(row + step);
        if (of.stages > 1) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        const uint4 *x = reinterpret_cast<const uint4 *>(ring + stage * 2 * of.row_bytes), *dy = x + of.row_bytes / 16;
        Two kept_xh[kKeep ? kN : 1][kH], kept_g[kKeep ? kN : 1][kH];
        const float own_g = own_dy * own_scale;
        Two of_g = two(own_g, 0.0f), of_gx = two(own_g * own_xh, 0.0f);
        if (kEdge) {
            own_sum_scale = fmaf(own_dy, own_xh, own_sum_scale);
            own_sum_shift += own_dy;
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = lane + i * lanes;
            if (c < whole) {
                Two xh[kH], d[kH], a[kH];
                unpack<T>(x[c], xh);
                unpack<T>(dy[c], d);
                fetch<T, P>(scale, c, whole, a);
#pragma unroll
                for (int j = 0; j < kH; ++j) {
                    xh[j] = mul(add(xh[j], less), times);
                    sum_scale[i][j] = fma(d[j], xh[j], sum_scale[i][j]);
                    sum_shift[i][j] = add(sum_shift[i][j], d[j]);
                    const Two g = mul(d[j], a[j]);
                    of_g = add(of_g, g);
                    of_gx = fma(g, xh[j], of_gx);
                    if (kKeep) {
                        kept_xh[kKeep ? i : 0][j] = xh[j];
                        kept_g[kKeep ? i : 0][j] = g;
                    }
                }
            }
        }
        if (p.y != nullptr) {
            float along = 0.0f, level = 0.0f;
            if (p.given == 0) {
                const float2 g = both(of_g), gx = both(of_gx);
                const float2 total = team_sum(g.x + g.y, gx.x + gx.y, of, place.team, scratch, turn);
                level = total.x * inv_axis;
                along = total.y * inv_axis;
            }
            const Two no_level = two(-level, -level), no_along = two(-along, -along);
            T *dx = static_cast<T *>(p.y) + row * p.y_ld;
            uint4 *to = reinterpret_cast<uint4 *>(dx + head);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = lane + i * lanes;
                if (c < whole) {
                    Two xh[kH], g[kH];
                    if (kKeep) {
#pragma unroll
                        for (int j = 0; j < kH; ++j) {
                            xh[j] = kept_xh[kKeep ? i : 0][j];
                            g[j] = kept_g[kKeep ? i : 0][j];
                        }
                    } else {
                        Two a[kH];
                        unpack<T>(x[c], xh);
                        unpack<T>(dy[c], g);
                        fetch<T, P>(scale, c, whole, a);
#pragma unroll
                        for (int j = 0; j < kH; ++j) {
                            xh[j] = mul(add(xh[j], less), times);
                            g[j] = mul(g[j], a[j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kH; ++j) {
                        g[j] = mul(p.given != 0 ? g[j] : fma(xh[j], no_along, add(g[j], no_level)), times);
                    }
                    to[c] = pack<T>(g);
                }
            }
            if (single) {
                dx[at] = narrow<T>((p.given != 0 ? own_g : fmaf(-own_xh, along, own_g - level)) * r);
            }
        }
        load(row + of.stages * step, stage);
        stage = of.stages > 1 ? stage ^ 1 : 0;
    }
    if (p.partial == nullptr) {
        return;
    }
    // the teams' sums, one after the other
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    float *to = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.axis;
    float *sums = of.teams > 1 ? reinterpret_cast<float *>(shared) : to;
    for (int k = 0; k < of.teams; ++k) {
        if (of.teams > 1) {
            __syncthreads();
        }
        if (place.team == k) {
            auto put = [&](int e, float of_scale, float of_shift) {
                sums[e] = of_scale + (k == 0 ? 0.0f : sums[e]);
                sums[p.axis + e] = of_shift + (k == 0 ? 0.0f : sums[p.axis + e]);
            };
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int c = lane + i * lanes;
                if (c < whole) {
#pragma unroll
                    for (int j = 0; j < kH; ++j) {
                        const float2 of_scale = both(sum_scale[i][j]), of_shift = both(sum_shift[i][j]);
                        put(head + c * kV + 2 * j, of_scale.x, of_shift.x);
                        put(head + c * kV + 2 * j + 1, of_scale.y, of_shift.y);
                    }
                }
            }
            if (single) {
                put(at, own_sum_scale, own_sum_shift);
            }
        }
    }
    if (of.teams > 1) {
        __syncthreads();
        for (int e = static_cast<int>(threadIdx.x); e < 2 * p.axis; e += static_cast<int>(blockDim.x)) {
            to[e] = sums[e];
        }
    }
}

// As layernorm_any_kernel (rows from 16,385 elements on): the sums over a CTA's rows column by column, then dx of them, which may lie where x or
// dy does.  4096 x 18432 bf16: 715 us, a tenth of HBM's rate.
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
                const float2 total = block_sum(of_g, of_gx, scratch, turn);
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
        int i = warp;
        for (; i + 56 < parts; i += 64) {  // eight loads at a time
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = from[static_cast<long long>(i + 8 * j) * 2 * p.axis];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s += v[j];
            }
        }
        for (; i < parts; i += 8) {
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

// CTAs that give every row to a team of its own, none of them without rows (in the last round of the classes, fewer than the period).
long long ctas_for(long long rows, int teams, int period)
{
    const long long round = static_cast<long long>(teams) * period, before = (rows - 1) / round;
    return before * period + std::min<long long>(period, rows - before * round);
}

// false: the general kernel
bool teams_of(const LayernormParams &p, int elem, int param_elem, int sm_count, Teams *t, int *grid, size_t *shared)
{
    const int period = period_of(p, elem, false);
    if (period == 0) {
        return false;
    }
    const long long bytes = (static_cast<long long>(p.axis) * elem + 15) / 16 * 16;
    const long long params = 2ll * p.axis * param_elem;
    const long long most = kMostShared - (params + 15) / 16 * 16;
    if (2 * bytes > most) {
        return false;
    }
    // sixteen warps per CTA with as many teams as shared memory has room for; with few rows, a piece per lane
    const long long room = std::max<long long>(1, most / (2 * bytes));
    int warps = 1;
    while (warps < 16 && (warps * room < 16 || (p.rows <= 2ll * sm_count && bytes > warps * 512ll))) {
        warps *= 2;
    }
    int teams = static_cast<int>(std::min<long long>(16 / warps, room));
    const long long need = (p.rows + sm_count - 1) / sm_count;
    while (teams > 1 && teams / 2 >= need) {
        teams /= 2;
    }
    *shared = static_cast<size_t>((params + 15) / 16 * 16 + 2 * bytes * teams);
    const int threads = teams * warps * 32;
    const long long per_sm = std::max<long long>(1, std::min<long long>({1024 / threads, static_cast<long long>(226 * 1024 / (*shared + 1280)), 16ll}));
    const long long enough = ctas_for(p.rows, teams, period);
    *grid = static_cast<int>(std::min<long long>(per_sm * sm_count / period * period, enough));
    *t = {warps, teams, period, static_cast<int>(bytes), 2};
    return true;
}

// The same for the gradient, kN pieces per thread.
bool backward_teams_of(const LayernormParams &p, int elem, int param_elem, int sm_count, Teams *t, int *pieces, int *grid, size_t *shared)
{
    const int period = period_of(p, elem, true);
    if (period == 0) {
        return false;
    }
    const long long bytes = (static_cast<long long>(p.axis) * elem + 15) / 16 * 16, whole = bytes / 16;
    const long long params = (static_cast<long long>(p.axis) * param_elem + 15) / 16 * 16;
    *pieces = whole <= 32 ? 1 : whole <= 64 ? 2 : whole <= 4 * kMostThreads || elem != 4 ? 4 : 8;
    const long long warps = (whole + *pieces * 32 - 1) / (*pieces * 32);
    if (warps * 32 > kMostThreads) {
        return false;
    }
    const int stages = params + 4 * bytes <= kMostShared ? 2 : 1;
    if (params + 2 * stages * bytes > kMostShared) {
        return false;
    }
    int teams = static_cast<int>(std::max<long long>(1, std::min<long long>(8 / warps, (kMostShared - params) / (2 * stages * bytes))));
    const long long need = (p.rows + sm_count - 1) / sm_count;
    while (teams > 1 && teams / 2 >= need) {
        teams /= 2;
    }
    *shared = static_cast<size_t>(std::max(params + 2 * stages * bytes * teams, teams > 1 ? 8ll * p.axis : 0ll));
    const int threads = static_cast<int>(teams * warps * 32);
    const long long per_sm = std::max<long long>(1, std::min<long long>(512 / threads, static_cast<long long>(226 * 1024 / (*shared + 1280))));
    const long long enough = ctas_for(p.rows, teams, period);
    *grid = static_cast<int>(std::min<long long>({per_sm * sm_count / period * period, kMostParts / period * period, enough}));
    *t = {static_cast<int>(warps), teams, period, static_cast<int>(bytes), stages};
    return true;
}

// Raises the kernel's limit of shared memory and launches it.
cudaError_t launch_teams(void (*kernel)(LayernormParams, Teams), const LayernormParams &p, const Teams &t, int grid, size_t shared, cudaStream_t stream)
{
    if (shared > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
        if (e != cudaSuccess) {
            return e;
        }
    }
    return launch_chained(kernel, dim3(grid), dim3(t.teams * t.warps * 32), shared, stream, 1u, p, t);
}

// Whether some row has elements that are not in whole pieces.
template <typename T>
bool has_edges(const LayernormParams &p, const Teams &t)
{
    return t.period != 1 || (reinterpret_cast<uintptr_t>(p.x) & 15u) != 0 || p.axis % kPer<T> != 0;
}

template <typename T, typename P>
cudaError_t launch_forward(const LayernormParams &p, int sm_count, cudaStream_t stream)
{
    Teams t;
    int grid;
    size_t shared;
    if (!teams_of(p, sizeof(T), sizeof(P), sm_count, &t, &grid, &shared)) {
        return launch_chained(layernorm_any_kernel<T, P>, dim3(static_cast<unsigned>(std::min<long long>(p.rows, 4ll * sm_count))), dim3(kMostThreads), 0,
                              stream, 1u, p);
    }
    return launch_teams(has_edges<T>(p, t) ? layernorm_kernel<T, P, true> : layernorm_kernel<T, P, false>, p, t, grid, shared, stream);
}

template <typename T, typename P>
cudaError_t launch_backward(const LayernormParams &p, int sm_count, cudaStream_t stream)
{
    Teams t;
    int pieces, grid;
    size_t shared;
    cudaError_t e;
    if (backward_teams_of(p, sizeof(T), sizeof(P), sm_count, &t, &pieces, &grid, &shared)) {
        const bool edges = has_edges<T>(p, t);
        void (*kernel)(LayernormParams, Teams) = edges ? layernorm_backward_kernel<T, P, 4, true> : layernorm_backward_kernel<T, P, 4, false>;
        if (pieces == 1) {
            kernel = edges ? layernorm_backward_kernel<T, P, 1, true> : layernorm_backward_kernel<T, P, 1, false>;
        } else if (pieces == 2) {
            kernel = edges ? layernorm_backward_kernel<T, P, 2, true> : layernorm_backward_kernel<T, P, 2, false>;
        }
        if constexpr (sizeof(T) == 4) {
            if (pieces == 8) {
                kernel = edges ? layernorm_backward_kernel<T, P, 8, true> : layernorm_backward_kernel<T, P, 8, false>;
            }
        }
        e = launch_teams(kernel, p, t, grid, shared, stream);
    } else {
        grid = static_cast<int>(std::min<long long>(p.rows, kMostParts));
        e = launch_chained(layernorm_backward_any_kernel<T, P>, dim3(grid), dim3(kMostThreads), 0, stream, 1u, p);
    }
    if (e != cudaSuccess || p.partial == nullptr) {
        return e;
    }
    return launch_chained(column_sums_kernel<P>, dim3((p.axis + 31) / 32, 2), dim3(256), 0, stream, 1u, p, grid);
}

template <typename T, typename P>
cudaError_t launch_typed(const LayernormParams &p, int sm_count, bool backward, cudaStream_t stream)
{
    return backward ? launch_backward<T, P>(p, sm_count, stream) : launch_forward<T, P>(p, sm_count, stream);
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
