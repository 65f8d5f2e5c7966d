// Layer normalisation over the last axis and its gradient.
//     m = mean(x)   v = mean((x - m)^2)   r = 1 / sqrt(v + eps)   xh = (x - m) r   y = xh scale + shift
//     g = dy scale  dx = r (g - mean(g) - xh mean(g xh))   dscale = sum over rows of dy xh   dshift = sum over rows of dy
// With given statistics m and v are constants: dx = r g.  All of it is fp32, each result rounded once.
#pragma once

#include "kernels.cuh"

namespace kb {

struct LayernormParams {
    const void *x, *dy, *scale, *shift;  // scale, shift: null for 1 and 0
    void *y;                             // forward: y; backward: dx or null
    float *mean, *variance;              // forward: written unless given (null: not wanted); backward: read
    void *dscale, *dshift;               // null: not wanted
    float *partial;                      // backward: [CTAs][2][axis], null: neither dscale nor dshift
    long long x_ld, y_ld, dy_ld;         // row pitches in elements
    int rows, axis;
    int dtype, param_dtype;
    int given;  // the statistics are given
    float eps;
};

cudaError_t launch_layernorm(const LayernormParams &p, int sm_count, cudaStream_t stream);

// fp32 values of the sums over rows that a backward pass leaves in LayernormParams::partial on its way to dscale and dshift
long long layernorm_backward_floats(long long rows, long long axis);
cudaError_t launch_layernorm_backward(const LayernormParams &p, int sm_count, cudaStream_t stream);

}  // namespace kb
