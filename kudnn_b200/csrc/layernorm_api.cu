// C-ABI of layer normalisation and its gradient (declared in include/kudnn_b200.h).
#include "layernorm.cuh"

#include <cmath>
#include <cstdio>

namespace {

int fail(int code, const char *message)
{
    return kb::set_last_error(code, message);
}

int fail_cuda(cudaError_t e, const char *what)
{
    char text[200];
    (void)cudaGetLastError();
    std::snprintf(text, sizeof(text), "%s: %s", what, cudaGetErrorString(e));
    return fail(e == cudaErrorMemoryAllocation ? KUDNN_B200_ALLOC_FAILED : KUDNN_B200_CUDA_ERROR, text);
}

bool misaligned(const void *p, int size)
{
    return reinterpret_cast<uintptr_t>(p) % size != 0;
}

constexpr int64_t kMostExtent = 0x7fffffffll - 1024;

int current_device(int *sms)
{
    int dev = 0, major = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(KUDNN_B200_NO_DEVICE, "no usable CUDA device is current");
    }
    if (major != 10) {
        return fail(KUDNN_B200_NO_DEVICE, "the current device is not sm_100; this library carries sm_100a code only");
    }
    return KUDNN_B200_OK;
}

// the flags and pointers that both directions share
int common(const kudnn_b200_layernorm_desc &d, const void *x, const void *scale, const float *mean, const float *variance, kb::LayernormParams *p)
{
    const int elem = kb::dtype_size(d.dtype), param = kb::dtype_size(d.param_dtype);
    if (x == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: x must not be null");
    }
    if (((d.flags & KUDNN_B200_NORM_USE_SCALE) != 0) != (scale != nullptr)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: the scale and the descriptor do not agree");
    }
    if (misaligned(x, elem) || misaligned(scale, param) || misaligned(mean, 4) || misaligned(variance, 4)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: a tensor is not aligned to its elements");
    }
    *p = kb::LayernormParams{};
    p->x = x;
    p->scale = scale;
    p->mean = const_cast<float *>(mean);
    p->variance = const_cast<float *>(variance);
    p->x_ld = d.x_ld;
    p->rows = static_cast<int>(d.rows);
    p->axis = static_cast<int>(d.axis);
    p->dtype = d.dtype;
    p->param_dtype = d.param_dtype;
    p->given = (d.flags & KUDNN_B200_NORM_USE_GLOBAL_STATS) != 0 ? 1 : 0;
    p->eps = d.eps;
    return KUDNN_B200_OK;
}

}  // namespace

extern "C" {

int kudnn_b200_layernorm_validate(const kudnn_b200_layernorm_desc *d)
{
    if (d == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: null descriptor");
    }
    if (d->rows < 0 || d->x_ld < 0 || d->y_ld < 0 || d->dy_ld < 0 || d->dx_ld < 0) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: negative extents or pitches");
    }
    if (d->axis <= 0) {
        return fail(KUDNN_B200_UNSUPPORTED, "layernorm: rows without elements are not supported");
    }
    if (d->rows > kMostExtent || d->axis > kMostExtent) {
        return fail(KUDNN_B200_UNSUPPORTED, "layernorm: extents of 2^31 and more are not supported");
    }
    if (d->dtype != KUDNN_B200_F32 && d->dtype != KUDNN_B200_F16 && d->dtype != KUDNN_B200_BF16) {
        return fail(KUDNN_B200_UNSUPPORTED, "layernorm: only F32 / F16 / BF16 tensors are implemented");
    }
    if (d->param_dtype != KUDNN_B200_F32 && d->param_dtype != d->dtype) {
        return fail(KUDNN_B200_UNSUPPORTED, "layernorm: scale and shift are F32 or of the rows' type");
    }
    if ((d->flags & ~(KUDNN_B200_NORM_USE_GLOBAL_STATS | KUDNN_B200_NORM_USE_SCALE | KUDNN_B200_NORM_USE_SHIFT)) != 0) {
        return fail(KUDNN_B200_UNSUPPORTED, "layernorm: the flags are USE_GLOBAL_STATS, USE_SCALE and USE_SHIFT");
    }
    if (!(d->eps >= 0.0f) || std::isinf(d->eps)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: eps is finite and not negative");
    }
    // 0: not used by this call; whoever writes the result looks again
    if (d->rows > 1 && ((d->y_ld != 0 && d->y_ld < d->axis) || (d->dx_ld != 0 && d->dx_ld < d->axis))) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: rows of a result overlap");
    }
    return KUDNN_B200_OK;
}

int kudnn_b200_layernorm_run(const kudnn_b200_layernorm_desc *d, const void *x, const void *scale, const void *shift, void *y, float *mean,
                             float *variance, void *cuda_stream)
{
    int rc = kudnn_b200_layernorm_validate(d);
    if (rc != KUDNN_B200_OK || d->rows == 0) {  // empty tensors often have no address
        return rc;
    }
    kb::LayernormParams p;
    rc = common(*d, x, scale, mean, variance, &p);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    if (y == nullptr || ((d->flags & KUDNN_B200_NORM_USE_SHIFT) != 0) != (shift != nullptr) ||
        (p.given != 0 && (mean == nullptr || variance == nullptr))) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: y, the shift or the given statistics and the descriptor do not agree");
    }
    if (d->rows > 1 && d->y_ld < d->axis) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: rows of a result overlap");
    }
    if (misaligned(y, kb::dtype_size(d->dtype)) || misaligned(shift, kb::dtype_size(d->param_dtype))) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: a tensor is not aligned to its elements");
    }
    int sms = 0;
    rc = current_device(&sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    p.shift = shift;
    p.y = y;
    p.y_ld = d->y_ld;
    const cudaError_t e = kb::launch_layernorm(p, sms, static_cast<cudaStream_t>(cuda_stream));
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "layernorm kernel launch");
}

int kudnn_b200_layernorm_backward_workspace(const kudnn_b200_layernorm_desc *d, int64_t *bytes)
{
    const int rc = kudnn_b200_layernorm_validate(d);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: nowhere to put the number of bytes");
    }
    *bytes = kb::layernorm_backward_floats(d->rows, d->axis) * 4;
    return KUDNN_B200_OK;
}

int kudnn_b200_layernorm_backward_run(const kudnn_b200_layernorm_desc *d, const void *x, const void *dy, const void *scale, const float *mean,
                                      const float *variance, void *dx, void *dscale, void *dshift, void *workspace, int64_t workspace_bytes,
                                      void *cuda_stream)
{
    int rc = kudnn_b200_layernorm_validate(d);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const int param = kb::dtype_size(d->param_dtype);
    if (misaligned(dscale, param) || misaligned(dshift, param)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: a tensor is not aligned to its elements");
    }
    if (d->rows == 0) {  // sums of nothing
        cudaError_t e = cudaSuccess;
        if (dscale != nullptr) e = cudaMemsetAsync(dscale, 0, static_cast<size_t>(d->axis) * param, stream);
        if (e == cudaSuccess && dshift != nullptr) e = cudaMemsetAsync(dshift, 0, static_cast<size_t>(d->axis) * param, stream);
        return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "layernorm: gradients of no rows");
    }
    kb::LayernormParams p;
    rc = common(*d, x, scale, mean, variance, &p);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    if (dy == nullptr || mean == nullptr || variance == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: the gradient needs dy, the mean and the variance");
    }
    const bool sums = dscale != nullptr || dshift != nullptr;
    if (sums && (workspace == nullptr || misaligned(workspace, 4) || workspace_bytes < kb::layernorm_backward_floats(d->rows, d->axis) * 4)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: the workspace is missing, too small or not aligned");
    }
    if (dx != nullptr && d->rows > 1 && d->dx_ld < d->axis) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: rows of a result overlap");
    }
    if (misaligned(dy, kb::dtype_size(d->dtype)) || misaligned(dx, kb::dtype_size(d->dtype))) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "layernorm: a tensor is not aligned to its elements");
    }
    if (!sums && dx == nullptr) {
        return KUDNN_B200_OK;
    }
    int sms = 0;
    rc = current_device(&sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    p.dy = dy;
    p.dy_ld = d->dy_ld;
    p.y = dx;
    p.y_ld = d->dx_ld;
    p.dscale = dscale;
    p.dshift = dshift;
    p.partial = sums ? static_cast<float *>(workspace) : nullptr;
    const cudaError_t e = kb::launch_layernorm_backward(p, sms, stream);
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "layernorm gradient kernel launch");
}

}  // extern "C"
