// A router and a block of experts for few tokens:
//     logit[t, e] = x[t] . w[e];  ids, p: the largest scores of each token (see include/kudnn_b200.h)
//     y[t] = sum over j of p[t, j] down[e] (silu(gate[e] x[t]) * (up[e] x[t])),  e = ids[t, j]
#pragma once

#include "kernels.cuh"

namespace kb {

constexpr int kMostExperts = 1024;
constexpr int kMostRouted = 64;       // experts a token is routed to
constexpr int kMostExpertTokens = 64;
constexpr int kMostExpertTop = 16;

struct RouteParams {
    const void *x, *w;
    const float *bias;
    float *weights;
    int *ids;
    long long x_ld, w_ld;
    int tokens, experts, hidden, top;
    int x_dtype, w_dtype, sigmoid, normalise, nan_first;
    float scale;
};
cudaError_t launch_route(const RouteParams &p, cudaStream_t stream);

struct ExpertsParams {
    const void *x;
    const float *p;
    const int *ids;
    const void *gate_up, *down;
    const float *gate_up_scale, *down_scale;
    void *y;
    void *h;  // workspace: the gated values
    long long x_ld, y_ld;
    long long gu_se, gu_sn, gu_sk, d_se, d_sn, d_sk;
    long long gus_se, gus_sn, gus_sk, ds_se, ds_sn, ds_sk;
    int tokens, hidden, ffn, experts, top;
    int x_dtype, w_dtype;
};
long long experts_workspace_bytes(long long tokens, long long top, long long ffn);
// The kernels that stream the weights take K-contiguous rows on 16-byte boundaries; the general ones any.
bool experts_stream_takes(const ExpertsParams &p);
cudaError_t launch_experts_stream(const ExpertsParams &p, int sm_count, cudaStream_t stream);
void experts_set_wait(long long limit_cycles, int skip_step);
// Of the current device, since the program began: how many waits gave up, and which was the last
cudaError_t experts_status_of(unsigned *gave_up, DeviceStatus *last);
cudaError_t launch_experts_any(const ExpertsParams &p, cudaStream_t stream);

// silu(gate) * up in fp32: e raised to a power below zero, so that the divisor lies in [1, 2]
__device__ __forceinline__ float expert_gate(float gate, float up)
{
    const float e = expf(-fabsf(gate));
    return (gate < 0.0f ? gate * e : gate) / (1.0f + e) * up;
}

__device__ __forceinline__ float e4m3_to_f32(unsigned char v)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(v)));
    return f16_bits_to_f32(static_cast<unsigned short>(h));
}

}  // namespace kb
