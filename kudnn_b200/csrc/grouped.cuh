// Products whose rows belong to groups (experts), each with weights of its own, and products of e4m3 operands that carry a scale for
// every block of 128:
//     c[r, :] = act( sum over k of a[r, k] b[g, :, k] + bias[g, :] )        for offsets[g] <= r < offsets[g + 1]
// with a 8-bit product scaled per block of K:  sum over kb of a_scale[r, kb] b_scale[g, n / 128, kb] (sum over k in kb of a b).
// The sums, the scales' products, the bias and the activation are fp32; the result is rounded once, to nearest even.
#pragma once

#include "kernels.cuh"

namespace kb {

constexpr int kScaleBlock = 128;
constexpr int kMaxGroups = 1024;

struct GroupedParams {
    const void *a, *b;
    void *c;
    const void *bias;
    const float *a_scale, *b_scale;
    const void *offsets;  // null: one group of all rows
    long long a_sm, a_sk, b_sg, b_sn, b_sk, c_sm, c_sn, bias_sg, bias_sn;
    long long as_sm, as_sk, bs_sg, bs_sn, bs_sk;
    int rows, n, k, groups;
    int ab_dtype, c_dtype, bias_dtype, has_bias, act, offsets_64;
    float act_alpha;
};

// offsets[i] brought into [0, rows]
__device__ __forceinline__ int group_offset(const GroupedParams &p, int i)
{
    if (p.offsets == nullptr) {
        return i == 0 ? 0 : p.rows;
    }
    const long long v = p.offsets_64 != 0 ? static_cast<const long long *>(p.offsets)[i] : static_cast<const int *>(p.offsets)[i];
    return static_cast<int>(v < 0 ? 0 : v > p.rows ? p.rows : v);
}

// Two e4m3 values, the lower byte first.
__device__ __forceinline__ float2 e4m3x2_to_f32(unsigned short v)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
    return make_float2(f16_bits_to_f32(static_cast<unsigned short>(h)), f16_bits_to_f32(static_cast<unsigned short>(h >> 16)));
}

// Whether the tensor-core kernel (grouped_tc.cuh) takes these operands: rows K-contiguous, 16-byte aligned.
bool grouped_tc_takes(const GroupedParams &p);
// rows of its tiles (0: not chosen yet), whether they stand on the M side, CTAs that cut K
struct GroupedTile {
    int rows, on_m, splits;
};
// Takes the tile that *tile asks for, or chooses one, and says which it was.
cudaError_t launch_grouped_tc(const GroupedParams &p, int sm_count, DeviceStatus *status, long long wait_limit_cycles, int skip_kblock,
                              GroupedTile *tile, cudaStream_t stream);
cudaError_t launch_grouped_simt(const GroupedParams &p, cudaStream_t stream);

// x -> e4m3 with a scale per row and 128 columns (block_rows = 1) or per 128 x 128 (block_rows = 128); see quantize.cu
struct QuantizeParams {
    const void *x;
    unsigned char *q;
    float *scale;
    const int *index;  // null: row r of q is row r of x
    long long x_ld, q_ld, s_row, s_col;
    int rows, k, x_rows;
    int x_dtype, gate, block_rows;
};
cudaError_t launch_quantize(const QuantizeParams &p, cudaStream_t stream);

}  // namespace kb
