// C-ABI of quantisation to e4m3 and of the products by group (declared in include/kudnn_b200.h).
#include "grouped.cuh"

#include <cstdio>
#include <mutex>
#include <new>
#include <numeric>

struct kudnn_b200_grouped_s {
    kudnn_b200_grouped_desc d;
    std::mutex lock;
    int forced_kernel = KUDNN_B200_KERNEL_AUTO;
    int last_kernel = 0;
    kb::GroupedTile forced_tile = {0, 0, 0}, last_tile = {0, 0, 0};
    int device = -1;
    int sm_count = 0;
    kb::DeviceStatus *status = nullptr;
    long long wait_limit = 0;
    int skip_kblock = -1;
};

namespace {

using Handle = kudnn_b200_grouped_s;

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

// whether some address is not a multiple of its elements' size: a load from it would fault
bool misaligned(const void *p, int size)
{
    return reinterpret_cast<uintptr_t>(p) % size != 0;
}

// Whether two elements of a matrix share an address: i * s1 == j * s2 for some i < rows, j < cols, the least of which are s2 / g, s1 / g.
bool overlaps(int64_t rows, int64_t s1, int64_t cols, int64_t s2)
{
    const int64_t g = std::gcd(s1, s2);
    return g == 0 ? rows > 1 || cols > 1 : s2 / g < rows && s1 / g < cols;
}

constexpr int64_t kMostExtent = 0x7fffffffll - 1024;

int current_device(int *dev, int *sms)
{
    int major = 0;
    if (cudaGetDevice(dev) != cudaSuccess || cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *dev) != cudaSuccess ||
        cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(KUDNN_B200_NO_DEVICE, "no usable CUDA device is current");
    }
    if (major != 10) {
        return fail(KUDNN_B200_NO_DEVICE, "the current device is not sm_100; this library carries sm_100a code only");
    }
    return KUDNN_B200_OK;
}

int ensure_device(Handle *h)
{
    std::lock_guard<std::mutex> guard(h->lock);
    int dev = 0;
    if (h->device >= 0) {
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) {
            return fail_cuda(e, "grouped");
        }
        return dev == h->device ? KUDNN_B200_OK : fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: the handle was first used on another device");
    }
    int sms = 0;
    const int rc = current_device(&dev, &sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    // cleared on a stream of its own: the first run may be captured on a stream that the default stream would wait for
    void *status = nullptr;
    cudaStream_t aside = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    (void)cudaThreadExchangeStreamCaptureMode(&mode);
    cudaError_t e = kb::library_malloc(&status, sizeof(kb::DeviceStatus));
    if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&aside, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemsetAsync(status, 0, sizeof(kb::DeviceStatus), aside);
    if (e == cudaSuccess) e = cudaStreamSynchronize(aside);
    if (aside != nullptr) {
        cudaStreamDestroy(aside);
    }
    (void)cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
        cudaFree(status);
        return fail_cuda(e, "grouped: status block");
    }
    h->status = static_cast<kb::DeviceStatus *>(status);
    h->device = dev;
    h->sm_count = sms;
    return KUDNN_B200_OK;
}

}  // namespace

extern "C" {

int kudnn_b200_quantize_validate(const kudnn_b200_quantize_desc *d)
{
    if (d == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: null descriptor");
    }
    if (d->rows < 0 || d->x_rows < 0 || d->x_ld < 0 || d->q_ld < 0 || d->s_row < 0 || d->s_col < 0) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: negative extents or strides");
    }
    if (d->k <= 0) {
        return fail(KUDNN_B200_UNSUPPORTED, "quantize: rows without columns are not supported");
    }
    if (d->rows > kMostExtent || d->x_rows > kMostExtent || d->k > kMostExtent / 2) {
        return fail(KUDNN_B200_UNSUPPORTED, "quantize: extents of 2^31 and more are not supported");
    }
    if (!float_type(d->x_dtype)) {
        return fail(KUDNN_B200_UNSUPPORTED, "quantize: x is F32, F16 or BF16");
    }
    if (d->block_rows != 1 && d->block_rows != kb::kScaleBlock) {
        return fail(KUDNN_B200_UNSUPPORTED, "quantize: blocks are of 1 x 128 or 128 x 128 elements");
    }
    if (d->block_rows != 1 && (d->gate != 0 || d->x_rows != d->rows)) {
        return fail(KUDNN_B200_UNSUPPORTED, "quantize: a gate or an index goes with a scale per row");
    }
    if (d->rows > 1 && d->q_ld < d->k) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: rows of q overlap");
    }
    const int64_t scale_rows = (d->rows + d->block_rows - 1) / d->block_rows, scale_cols = (d->k + kb::kScaleBlock - 1) / kb::kScaleBlock;
    if (overlaps(scale_rows, d->s_row, scale_cols, d->s_col)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: scales overlap");
    }
    return KUDNN_B200_OK;
}

int kudnn_b200_quantize_run(const kudnn_b200_quantize_desc *d, const void *x, void *q, float *scale, const int32_t *index, void *cuda_stream)
{
    int rc = kudnn_b200_quantize_validate(d);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    if (d->rows == 0) {  // ahead of the checks of pointers: empty tensors often have none
        return KUDNN_B200_OK;
    }
    if (index == nullptr && d->x_rows != d->rows) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: x and q have the same rows unless there is an index");
    }
    if (index != nullptr && d->block_rows != 1) {
        return fail(KUDNN_B200_UNSUPPORTED, "quantize: a gate or an index goes with a scale per row");
    }
    if ((x == nullptr && d->x_rows != 0) || q == nullptr || scale == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: x, q and scale must not be null");
    }
    if (misaligned(x, kb::dtype_size(d->x_dtype)) || misaligned(scale, 4) || misaligned(index, 4)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "quantize: x, scale or index is not aligned to its elements");
    }
    int dev = 0, sms = 0;
    rc = current_device(&dev, &sms);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    kb::QuantizeParams p;
    p.x = x;
    p.q = static_cast<unsigned char *>(q);
    p.scale = scale;
    p.index = index;
    p.x_ld = d->x_ld;
    p.q_ld = d->q_ld;
    p.s_row = d->s_row;
    p.s_col = d->s_col;
    p.rows = static_cast<int>(d->rows);
    p.k = static_cast<int>(d->k);
    p.x_rows = static_cast<int>(d->x_rows);
    p.x_dtype = d->x_dtype;
    p.gate = d->gate != 0 ? 1 : 0;
    p.block_rows = d->block_rows;
    const cudaError_t e = kb::launch_quantize(p, static_cast<cudaStream_t>(cuda_stream));
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "quantize kernel launch");
}

int kudnn_b200_grouped_validate(const kudnn_b200_grouped_desc *d)
{
    if (d == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: null descriptor");
    }
    if (d->rows < 0 || d->groups < 1) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: rows must not be negative and there is one group at least");
    }
    if (d->n <= 0 || d->k <= 0) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: empty weights are not supported");
    }
    if (d->rows > kMostExtent || d->n > kMostExtent || d->k > kMostExtent) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: extents of 2^31 and more are not supported");
    }
    if (d->groups > kb::kMaxGroups) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: more than 1024 groups are not supported");
    }
    // work items are counted in 31 bits: tiles of at least 16 rows x 64 columns
    if ((d->rows / 16 + d->groups + 1) * ((d->n + 63) / 64) > 0x7fffffffll) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: c has too many tiles");
    }
    if (d->ab_dtype != KUDNN_B200_F16 && d->ab_dtype != KUDNN_B200_BF16 && d->ab_dtype != KUDNN_B200_E4M3) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: operands are F16, BF16 or E4M3");
    }
    if (!float_type(d->c_dtype) || (d->has_bias != 0 && !float_type(d->bias_dtype))) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: results and bias are F32, F16 or BF16");
    }
    if (d->act != KUDNN_B200_ACT_NONE && kudnn_b200_activation_validate(1, KUDNN_B200_F32, KUDNN_B200_F32, d->act) != KUDNN_B200_OK) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: this activation is not implemented");
    }
    if (d->offsets_dtype != 0 && d->offsets_dtype != KUDNN_B200_S32 && d->offsets_dtype != KUDNN_B200_S64) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: offsets are S32 or S64");
    }
    if (d->offsets_dtype == 0 && d->groups != 1) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: several groups need offsets");
    }
    const int64_t strides[] = {d->a_sm, d->a_sk, d->b_sg, d->b_sn, d->b_sk, d->c_sm, d->c_sn, d->bias_sg, d->bias_sn,
                               d->a_scale_sm, d->a_scale_sk, d->b_scale_sg, d->b_scale_sn, d->b_scale_sk};
    for (int64_t s : strides) {
        if (s < 0) {
            return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: negative strides");
        }
    }
    if (overlaps(d->rows, d->c_sm, d->n, d->c_sn)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: elements of c overlap");
    }
    return KUDNN_B200_OK;
}

int kudnn_b200_grouped_create(const kudnn_b200_grouped_desc *d, kudnn_b200_grouped_t *handle)
{
    if (handle == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: null handle pointer");
    }
    *handle = nullptr;
    const int rc = kudnn_b200_grouped_validate(d);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    Handle *h = new (std::nothrow) Handle;
    if (h == nullptr) {
        return fail(KUDNN_B200_ALLOC_FAILED, "grouped: out of host memory");
    }
    h->d = *d;
    *handle = h;
    return KUDNN_B200_OK;
}

int kudnn_b200_grouped_destroy(kudnn_b200_grouped_t h)
{
    if (h == nullptr) {
        return KUDNN_B200_OK;
    }
    if (h->status != nullptr) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        (void)cudaThreadExchangeStreamCaptureMode(&mode);
        cudaFree(h->status);  // waits for the runs that may still write it
        (void)cudaThreadExchangeStreamCaptureMode(&mode);
    }
    delete h;
    return KUDNN_B200_OK;
}

int kudnn_b200_grouped_run(kudnn_b200_grouped_t h, const kudnn_b200_grouped_args *args, void *cuda_stream)
{
    if (h == nullptr || args == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: null handle or arguments");
    }
    const kudnn_b200_grouped_desc &d = h->d;
    if (d.rows == 0) {  // ahead of the checks of pointers: empty tensors often have none
        return KUDNN_B200_OK;
    }
    if ((d.has_bias != 0) != (args->bias != nullptr)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: the bias and the descriptor do not agree");
    }
    if ((d.ab_dtype == KUDNN_B200_E4M3) != (args->a_scale != nullptr) || (d.ab_dtype == KUDNN_B200_E4M3) != (args->b_scale != nullptr)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: E4M3 operands need both scales, others take none");
    }
    if ((d.offsets_dtype != 0) != (args->offsets != nullptr)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: the offsets and the descriptor do not agree");
    }
    if (args->a == nullptr || args->b == nullptr || args->c == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: a, b and c must not be null");
    }
    const int es = d.ab_dtype == KUDNN_B200_E4M3 ? 1 : 2;
    if (misaligned(args->a, es) || misaligned(args->b, es) || misaligned(args->c, kb::dtype_size(d.c_dtype)) ||
        (d.has_bias != 0 && misaligned(args->bias, kb::dtype_size(d.bias_dtype))) || misaligned(args->a_scale, 4) || misaligned(args->b_scale, 4) ||
        misaligned(args->offsets, d.offsets_dtype == KUDNN_B200_S64 ? 8 : 4)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: an operand is not aligned to its elements");
    }
    const int rc = ensure_device(h);
    if (rc != KUDNN_B200_OK) {
        return rc;
    }
    kb::GroupedParams p;
    p.a = args->a;
    p.b = args->b;
    p.c = args->c;
    p.bias = args->bias;
    p.a_scale = args->a_scale;
    p.b_scale = args->b_scale;
    p.offsets = args->offsets;
    p.a_sm = d.a_sm;
    p.a_sk = d.a_sk;
    p.b_sg = d.b_sg;
    p.b_sn = d.b_sn;
    p.b_sk = d.b_sk;
    p.c_sm = d.c_sm;
    p.c_sn = d.c_sn;
    p.bias_sg = d.bias_sg;
    p.bias_sn = d.bias_sn;
    p.as_sm = d.a_scale_sm;
    p.as_sk = d.a_scale_sk;
    p.bs_sg = d.b_scale_sg;
    p.bs_sn = d.b_scale_sn;
    p.bs_sk = d.b_scale_sk;
    p.rows = static_cast<int>(d.rows);
    p.n = static_cast<int>(d.n);
    p.k = static_cast<int>(d.k);
    p.groups = d.groups;
    p.ab_dtype = d.ab_dtype;
    p.c_dtype = d.c_dtype;
    p.bias_dtype = d.bias_dtype;
    p.has_bias = d.has_bias != 0 ? 1 : 0;
    p.act = d.act;
    p.act_alpha = d.act_alpha;
    p.offsets_64 = d.offsets_dtype == KUDNN_B200_S64 ? 1 : 0;
    const bool takes = kb::grouped_tc_takes(p);
    if (h->forced_kernel == KUDNN_B200_KERNEL_TC && !takes) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: the tensor cores want rows that are K-contiguous and 16-byte aligned");
    }
    const bool tc = takes && h->forced_kernel != KUDNN_B200_KERNEL_SIMT;
    cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    kb::GroupedTile tile = h->forced_tile;
    const cudaError_t e = tc ? kb::launch_grouped_tc(p, h->sm_count, h->status, h->wait_limit, h->skip_kblock, &tile, stream)
                             : kb::launch_grouped_simt(p, stream);
    h->last_tile = tc ? tile : kb::GroupedTile{0, 0, 0};
    h->last_kernel = tc ? KUDNN_B200_KERNEL_TC : KUDNN_B200_KERNEL_SIMT;
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "grouped kernel launch");
}

int kudnn_b200_grouped_check(kudnn_b200_grouped_t h, void *cuda_stream)
{
    if (h == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: null handle");
    }
    std::lock_guard<std::mutex> guard(h->lock);
    if (h->device < 0) {
        return KUDNN_B200_OK;
    }
    kb::DeviceStatus st;
    cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(cuda_stream));
    if (e == cudaSuccess) e = cudaMemcpy(&st, h->status, sizeof(st), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess && st.code != kb::kErrNone) {
        e = cudaMemset(h->status, 0, sizeof(st));
        if (e == cudaSuccess) {
            char text[120];
            std::snprintf(text, sizeof(text), "device-side wait gave up (site %d, block %d)", st.where, st.block);
            return fail(KUDNN_B200_TIMEOUT, text);
        }
    }
    return e == cudaSuccess ? KUDNN_B200_OK : fail_cuda(e, "grouped: check");
}

int kudnn_b200_grouped_force_kernel(kudnn_b200_grouped_t h, int kernel)
{
    if (h == nullptr || (kernel != KUDNN_B200_KERNEL_AUTO && kernel != KUDNN_B200_KERNEL_SIMT && kernel != KUDNN_B200_KERNEL_TC)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: force_kernel takes AUTO, SIMT or TC");
    }
    h->forced_kernel = kernel;
    return KUDNN_B200_OK;
}

int kudnn_b200_grouped_last_kernel(kudnn_b200_grouped_t h)
{
    return h == nullptr ? 0 : h->last_kernel;
}

int kudnn_b200_grouped_force_tile(kudnn_b200_grouped_t h, int tile_rows, int rows_on_m)
{
    if (h == nullptr || (tile_rows != 0 && tile_rows != 32 && tile_rows != 64 && tile_rows != 128 && tile_rows != 256)) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: tiles have 32, 64, 128 or 256 rows");
    }
    if (rows_on_m != 0 && (tile_rows != 256 || h->d.ab_dtype != KUDNN_B200_E4M3)) {
        return fail(KUDNN_B200_UNSUPPORTED, "grouped: the rows stand on the M side in tiles of 256 rows of E4M3 operands only");
    }
    h->forced_tile = {tile_rows, rows_on_m != 0 ? 1 : 0, 0};
    return KUDNN_B200_OK;
}

int kudnn_b200_grouped_last_tile(kudnn_b200_grouped_t h, int *tile_rows, int *rows_on_m, int *splits)
{
    if (h == nullptr || tile_rows == nullptr || rows_on_m == nullptr || splits == nullptr) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: null handle or arguments");
    }
    *tile_rows = h->last_tile.rows;
    *rows_on_m = h->last_tile.on_m;
    *splits = h->last_tile.splits;
    return KUDNN_B200_OK;
}

int kudnn_b200_grouped_set_wait(kudnn_b200_grouped_t h, long long wait_limit_cycles, int skip_kblock)
{
    if (h == nullptr || wait_limit_cycles < 0) {
        return fail(KUDNN_B200_BAD_ARGUMENTS, "grouped: set_wait takes a handle and a limit that is not negative");
    }
    h->wait_limit = wait_limit_cycles;
    h->skip_kblock = skip_kblock;
    return KUDNN_B200_OK;
}

}  // extern "C"
