// General kernels of the block of experts: any strides, one element at a time.
#include "experts.cuh"

namespace kb {

namespace {

constexpr int kBlock = 128;  // rows and columns per scale

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

__device__ __forceinline__ float weight_at(const void *w, int dtype, long long i)
{
    return dtype == KUDNN_B200_E4M3 ? e4m3_to_f32(static_cast<const unsigned char *>(w)[i]) : load_as_f32(w, dtype, i);
}

// A warp per pair of token and expert and per value of h; the gate's and the up's row side by side.
__global__ void __launch_bounds__(256) experts_any_up_kernel(const __grid_constant__ ExpertsParams p)
{
    const int lane = static_cast<int>(threadIdx.x) & 31;
    pdl_launch_dependents();
    pdl_wait();
    const long long all = static_cast<long long>(p.tokens) * p.top * p.ffn;
    for (long long i = blockIdx.x * 8ll + threadIdx.x / 32; i < all; i += gridDim.x * 8ll) {
        const int pair = static_cast<int>(i / p.ffn), f = static_cast<int>(i % p.ffn), e = p.ids[pair];
        if (e < 0 || e >= p.experts) {
            continue;
        }
        const long long x0 = pair / p.top * p.x_ld, w0 = e * p.gu_se + f * p.gu_sn, w1 = w0 + p.ffn * p.gu_sn;
        const bool scaled = p.gate_up_scale != nullptr;
        const float *s0 = scaled ? p.gate_up_scale + e * p.gus_se + f / kBlock * p.gus_sn : nullptr;
        const float *s1 = scaled ? p.gate_up_scale + e * p.gus_se + (p.ffn + f) / kBlock * p.gus_sn : nullptr;
        float gate = 0.0f, up = 0.0f;
        for (int k0 = 0; k0 < p.hidden; k0 += kBlock) {  // block by block: no long chain of additions
            float g = 0.0f, u = 0.0f;
            for (int k = k0 + lane; k < min(k0 + kBlock, p.hidden); k += 32) {
                const float x = load_as_f32(p.x, p.x_dtype, x0 + k);
                g = fmaf(x, weight_at(p.gate_up, p.w_dtype, w0 + k * p.gu_sk), g);
                u = fmaf(x, weight_at(p.gate_up, p.w_dtype, w1 + k * p.gu_sk), u);
            }
            gate = fmaf(g, scaled ? s0[k0 / kBlock * p.gus_sk] : 1.0f, gate);
            up = fmaf(u, scaled ? s1[k0 / kBlock * p.gus_sk] : 1.0f, up);
        }
        gate = warp_sum(gate);
        up = warp_sum(up);
        if (lane == 0) {
            static_cast<float *>(p.h)[i] = expert_gate(gate, up);
        }
    }
}

// A warp per value of y.
__global__ void __launch_bounds__(256) experts_any_down_kernel(const __grid_constant__ ExpertsParams p)
{
    const int lane = static_cast<int>(threadIdx.x) & 31;
    pdl_launch_dependents();
    pdl_wait();
    const long long all = static_cast<long long>(p.tokens) * p.hidden;
    for (long long i = blockIdx.x * 8ll + threadIdx.x / 32; i < all; i += gridDim.x * 8ll) {
        const int t = static_cast<int>(i / p.hidden), n = static_cast<int>(i % p.hidden);
        float y = 0.0f;
        for (int j = 0; j < p.top; ++j) {
            const int e = p.ids[t * p.top + j];
            if (e < 0 || e >= p.experts) {
                continue;
            }
            const float *h = static_cast<const float *>(p.h) + (static_cast<long long>(t) * p.top + j) * p.ffn;
            const long long w0 = e * p.d_se + n * p.d_sn;
            const float *scale = p.down_scale != nullptr ? p.down_scale + e * p.ds_se + n / kBlock * p.ds_sn : nullptr;
            float sum = 0.0f;
            for (int k0 = 0; k0 < p.ffn; k0 += kBlock) {
                float s = 0.0f;
                for (int k = k0 + lane; k < min(k0 + kBlock, p.ffn); k += 32) {
                    s = fmaf(h[k], weight_at(p.down, p.w_dtype, w0 + k * p.d_sk), s);
                }
                sum = fmaf(s, scale != nullptr ? scale[k0 / kBlock * p.ds_sk] : 1.0f, sum);
            }
            y = fmaf(p.p[t * p.top + j], warp_sum(sum), y);
        }
        if (lane == 0) {
            store_exact(p.y, p.x_dtype, t * p.y_ld + n, round_rne(y, p.x_dtype));
        }
    }
}

}  // namespace

long long experts_workspace_bytes(long long tokens, long long top, long long ffn)
{
    return tokens * top * ((ffn + 127) / 128 * 128) * 4;
}

cudaError_t launch_experts_any(const ExpertsParams &p, cudaStream_t stream)
{
    cudaError_t e = launch_chained(experts_any_up_kernel, dim3(148 * 8), dim3(256), 0, stream, 1u, p);
    return e == cudaSuccess ? launch_chained(experts_any_down_kernel, dim3(148 * 8), dim3(256), 0, stream, 1u, p) : e;
}

}  // namespace kb
