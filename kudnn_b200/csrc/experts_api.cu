// C-ABI of the router and of the block of experts for few tokens (declared in include/kudnn_b200.h).
#include "experts.cuh"

#include <cmath>
#include <cstdio>
#include <map>
#include <new>

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

bool float_type(int dt)
{
    return dt == KUDNN_B200_F32 || dt == KUDNN_B200_F16 || dt == KUDNN_B200_BF16;
}

bool misaligned(const void *p, int size)
{
    return reinterpret_cast<uintptr_t>(p) % size != 0;
}

constexpr int64_t kMostExtent = 0x7fffffffll - 1024;
constexpr int64_t kMostRouterDepth = 0x7fffffffll - 4096;  // its kernels look up to 2060 elements ahead, in 32 bits

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

}  // namespace

extern "C" {

int kudnn_b200_route_validate(const kudnn_b200_route_desc *d)
{
    if (d == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "route: null descriptor");
    }
    if (d->tokens < 0 || d->x_ld < 0 || d->w_ld < 0) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "route: negative extents or pitches");
    }
    if (d->hidden <= 0 || d->hidden > kMostRouterDepth || d->tokens > kMostExtent / 8) {
        return fail(KUDNN_B200_UNSUPPORTED, "route: rows without elements and extents of 2^28 tokens and more are not supported");
    }
    if (d->experts < 1 || d->experts > kb::kMostExperts) {
        return fail(KUDNN_B200_UNSUPPORTED, "route: 1 to 1024 experts are supported");
    }
    if (d->top < 1 || d->top > d->experts) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "route: a token goes to at least one expert and at most to all of them");
    }
    if (d->top > kb::kMostRouted) {
        return fail(KUDNN_B200_UNSUPPORTED, "route: a token goes to at most 64 experts");
    }
    if (!float_type(d->x_dtype) || !float_type(d->w_dtype)) {
        return fail(KUDNN_B200_UNSUPPORTED, "route: tokens and weights are F32, F16 or BF16");
    }
    if (d->score != KUDNN_B200_SCORE_SOFTMAX && d->score != KUDNN_B200_SCORE_SIGMOID) {
        return fail(KUDNN_B200_UNSUPPORTED, "route: scores are a softmax or a sigmoid");
    }
    if (!std::isfinite(d->scale)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "route: the scale is finite");
    }
    return KUDNN_B200_OK;
}

int kudnn_b200_route_run(const kudnn_b200_route_desc *d, const void *x, const void *w, const float *bias, float *weights, int32_t *ids,
                         void *cuda_stream)
{
    int rc = kudnn_b200_route_validate(d);
    if (rc != KUDNN_B200_OK || d->tokens == 0) {  // empty tensors often have no address
        return rc;
    }
    if (x == nullptr || w == nullptr || weights == nullptr || ids == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "route: x, w, weights and ids must not be null");
    }
    if (misaligned(x, kb::dtype_size(d->x_dtype)) || misaligned(w, kb::dtype_size(d->w_dtype)) || misaligned(bias, 4) || misaligned(weights, 4) ||
        misaligned(ids, 4)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "route: a tensor is not aligned to its elements");
    }
    int sms = 0;
    rc = current_device(&sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    kb::RouteParams p;
    p.x = x;
    p.w = w;
    p.bias = bias;
    p.weights = weights;
    p.ids = ids;
    p.x_ld = d->x_ld;
    p.w_ld = d->w_ld;
    p.tokens = static_cast<int>(d->tokens);
    p.experts = d->experts;
    p.hidden = static_cast<int>(d->hidden);
    p.top = d->top;
    p.x_dtype = d->x_dtype;
    p.w_dtype = d->w_dtype;
    p.sigmoid = d->score == KUDNN_B200_SCORE_SIGMOID ? 1 : 0;
    p.normalise = d->normalise != 0 ? 1 : 0;
    p.nan_first = d->nan_first == 1 ? 1 : 0;  // the place of a field that had no meaning
    p.scale = d->scale;
    const cudaError_t e = kb::launch_route(p, static_cast<cudaStream_t>(cuda_stream));
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "route kernel launch");
}

int kudnn_b200_experts_validate(const kudnn_b200_experts_desc *d)
{
    if (d == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: null descriptor");
    }
    if (d->tokens < 0 || d->experts < 1 || d->top < 1) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: tokens must not be negative, and there is one expert at least");
    }
    if (d->tokens > kb::kMostExpertTokens || d->top > kb::kMostExpertTop) {
        return fail(KUDNN_B200_UNSUPPORTED, "experts: at most 64 tokens and 16 experts per token; larger batches are products by group");
    }
    if (d->experts > kb::kMostExperts) {
        return fail(KUDNN_B200_UNSUPPORTED, "experts: more than 1024 experts are not supported");
    }
    if (d->hidden <= 0 || d->ffn <= 0 || d->hidden > kMostExtent || d->ffn > kMostExtent / 2) {
        return fail(KUDNN_B200_UNSUPPORTED, "experts: empty weights and extents of 2^31 and more are not supported");
    }
    if (d->x_dtype != KUDNN_B200_F16 && d->x_dtype != KUDNN_B200_BF16) {
        return fail(KUDNN_B200_UNSUPPORTED, "experts: tokens are F16 or BF16");
    }
    if (d->w_dtype != d->x_dtype && d->w_dtype != KUDNN_B200_E4M3) {
        return fail(KUDNN_B200_UNSUPPORTED, "experts: weights are of the tokens' type or E4M3");
    }
    const int64_t strides[] = {d->x_ld, d->y_ld, d->gate_up_se, d->gate_up_sn, d->gate_up_sk, d->down_se, d->down_sn, d->down_sk,
                               d->gate_up_scale_se, d->gate_up_scale_sn, d->gate_up_scale_sk, d->down_scale_se, d->down_scale_sn, d->down_scale_sk};
    for (int64_t s : strides) {
        if (s < 0) {
            return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: negative strides");
        }
    }
    if (d->tokens > 1 && d->y_ld < d->hidden) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: rows of y overlap");
    }
    return KUDNN_B200_OK;
}

int kudnn_b200_experts_workspace(const kudnn_b200_experts_desc *d, int64_t *bytes)
{
    const int rc = kudnn_b200_experts_validate(d);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    if (bytes == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: nowhere to put the number of bytes");
    }
    *bytes = kb::experts_workspace_bytes(d->tokens, d->top, d->ffn);
    return KUDNN_B200_OK;
}

int kudnn_b200_experts_run(const kudnn_b200_experts_desc *d, const kudnn_b200_experts_args *a, void *cuda_stream)
{
    int rc = kudnn_b200_experts_validate(d);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    if (a == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: null arguments");
    }
    if (d->tokens == 0) {  // empty tensors often have no address
        return KUDNN_B200_OK;
    }
    if (a->x == nullptr || a->weights == nullptr || a->ids == nullptr || a->gate_up == nullptr || a->down == nullptr || a->y == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: x, weights, ids, gate_up, down and y must not be null");
    }
    const bool e4m3 = d->w_dtype == KUDNN_B200_E4M3;
    if (e4m3 != (a->gate_up_scale != nullptr) || e4m3 != (a->down_scale != nullptr)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: E4M3 weights need both scales, others take none");
    }
    if (misaligned(a->x, 2) || misaligned(a->y, 2) || misaligned(a->weights, 4) || misaligned(a->ids, 4) || misaligned(a->gate_up, e4m3 ? 1 : 2) ||
        misaligned(a->down, e4m3 ? 1 : 2) || misaligned(a->gate_up_scale, 4) || misaligned(a->down_scale, 4)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: a tensor is not aligned to its elements");
    }
    if (a->workspace == nullptr || misaligned(a->workspace, 16) ||
        a->workspace_bytes < kb::experts_workspace_bytes(d->tokens, d->top, d->ffn)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: the workspace is missing, too small or not on a 16-byte boundary");
    }
    int sms = 0;
    rc = current_device(&sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    kb::ExpertsParams p;
    p.x = a->x;
    p.p = a->weights;
    p.ids = a->ids;
    p.gate_up = a->gate_up;
    p.down = a->down;
    p.gate_up_scale = a->gate_up_scale;
    p.down_scale = a->down_scale;
    p.y = a->y;
    p.h = a->workspace;
    p.x_ld = d->x_ld;
    p.y_ld = d->y_ld;
    p.gu_se = d->gate_up_se;
    p.gu_sn = d->gate_up_sn;
    p.gu_sk = d->gate_up_sk;
    p.d_se = d->down_se;
    p.d_sn = d->down_sn;
    p.d_sk = d->down_sk;
    p.gus_se = d->gate_up_scale_se;
    p.gus_sn = d->gate_up_scale_sn;
    p.gus_sk = d->gate_up_scale_sk;
    p.ds_se = d->down_scale_se;
    p.ds_sn = d->down_scale_sn;
    p.ds_sk = d->down_scale_sk;
    p.tokens = static_cast<int>(d->tokens);
    p.hidden = static_cast<int>(d->hidden);
    p.ffn = static_cast<int>(d->ffn);
    p.experts = d->experts;
    p.top = d->top;
    p.x_dtype = d->x_dtype;
    p.w_dtype = d->w_dtype;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = kb::experts_stream_takes(p) ? kb::launch_experts_stream(p, sms, stream) : kb::launch_experts_any(p, stream);
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "experts kernel launch");
}

int kudnn_b200_experts_check(void *cuda_stream)
{
    // What this thread has seen of each device.  Runs of all callers count together: a thread that took another's report away would leave the
    // other with results that are undefined and a check that says nothing.
    static thread_local std::map<int, unsigned> seen;
    int sms = 0, dev = 0;
    const int rc = current_device(&sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    kb::DeviceStatus st;
    unsigned gave_up = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaStreamSynchronize(static_cast<cudaStream_t>(cuda_stream));
    if (e == cudaSuccess) e = kb::experts_status_of(&gave_up, &st);
    if (e != cudaSuccess) {
        return fail_cuda(e, "experts: check");
    }
    bool news = false;
    try {
        unsigned &known = seen[dev];
        news = gave_up != known;
        known = gave_up;
    } catch (const std::bad_alloc &) {
        return fail(KUDNN_B200_ALLOC_FAILED, "experts: check: out of host memory");
    }
    if (news) {
        char text[120];
        std::snprintf(text, sizeof(text), "device-side wait gave up (site %d, block %d)", st.where, st.block);
        return fail(KUDNN_B200_TIMEOUT, text);
    }
    return KUDNN_B200_OK;
}

int kudnn_b200_experts_set_wait(long long wait_limit_cycles, int skip_step)
{
    if (wait_limit_cycles < 0) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "experts: the limit of a wait is not negative");
    }
    kb::experts_set_wait(wait_limit_cycles, skip_step);
    return KUDNN_B200_OK;
}

}  // extern "C"
