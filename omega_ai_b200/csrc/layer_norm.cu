// Layer norm of rows, forward and backward.
//
//   mean = sum(x) / d;  var = sum((x - mean)^2) / d;  rstd = 1 / sqrt(var + eps);  h = (x - mean) * rstd
//   y = h * gamma + beta
//   g = dy * gamma;  dx = rstd * (g - sum(g) / d - h * sum(g * h) / d);  dgamma = sum over rows of dy * h;  dbeta = of dy
//
// The variance is taken after the mean: the difference of the mean of squares and the squared mean loses all digits on rows
// whose offset is large against their spread.  All sums are fp32 in a fixed order.
#include "ops.cuh"

namespace omoe {

namespace {

constexpr int kWideThreads = 512;

// Sum over a block of kWideThreads, the same value in every thread.
__device__ __forceinline__ float block_sum(float v, float *s) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWideThreads / 32; i++) sum += s[i];
    return sum;
}

// Any width: a block walks its row three times, from cache after the first.
template <typename XT, typename YT>
__global__ void __launch_bounds__(kWideThreads)
norm_wide_kernel(const XT *__restrict__ x, int64_t ldx, const float *__restrict__ gamma, const float *__restrict__ beta,
                 float eps, YT *__restrict__ y, int64_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out, int d) {
    __shared__ float s[kWideThreads / 32];
    const int64_t t = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    const XT *row = x + t * ldx;
    float sum = 0.f;
    for (int c = threadIdx.x; c < d; c += kWideThreads) sum += (float)row[c];
    const float mean = block_sum(sum, s) / (float)d;
    sum = 0.f;
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float v = (float)row[c] - mean;
        sum = fmaf(v, v, sum);
    }
    const float rstd = 1.f / sqrtf(block_sum(sum, s) / (float)d + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[t] = mean;
        if (rstd_out) rstd_out[t] = rstd;
    }
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float h = ((float)row[c] - mean) * rstd;
        y[t * ldy + c] = (YT)fmaf(h, gamma ? gamma[c] : 1.f, beta ? beta[c] : 0.f);
    }
}

template <typename XT, typename YT>
__global__ void __launch_bounds__(kWideThreads)
norm_bwd_wide_kernel(const YT *__restrict__ dy, int64_t lddy, const XT *__restrict__ x, int64_t ldx,
                     const float *__restrict__ gamma, const float *__restrict__ mean, const float *__restrict__ rstd,
                     XT *__restrict__ dx, int64_t lddx, int d) {
    __shared__ float s[2][kWideThreads / 32];
    const int64_t t = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    const float m = mean[t], r = rstd[t];
    float sum = 0.f, dot = 0.f;
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float g = (float)dy[t * lddy + c] * (gamma ? gamma[c] : 1.f);
        sum += g;
        dot = fmaf(g, ((float)x[t * ldx + c] - m) * r, dot);
    }
    const float mg = block_sum(sum, s[0]) / (float)d, mh = block_sum(dot, s[1]) / (float)d;
    for (int c = threadIdx.x; c < d; c += kWideThreads) {
        const float g = (float)dy[t * lddy + c] * (gamma ? gamma[c] : 1.f), h = ((float)x[t * ldx + c] - m) * r;
        dx[t * lddx + c] = (XT)(r * (g - mg - h * mh));
    }
}

// Column sums of a slice of the rows: partial[slice][0][d] of dy * h, [1][d] of dy.
template <typename XT, typename YT>
__global__ void __launch_bounds__(256)
norm_cols_kernel(const YT *__restrict__ dy, int64_t lddy, const XT *__restrict__ x, int64_t ldx,
                 const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ partial, int T, int d,
                 int slice) {
    __shared__ float s[2][8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    pdl_trigger();
    pdl_wait();
    const int64_t t0 = (int64_t)blockIdx.y * slice, t1 = min((int64_t)T, t0 + slice);
    float a = 0.f, b = 0.f;
    if (c < d)
        for (int64_t t = t0 + warp; t < t1; t += 8) {
            const float g = (float)dy[t * lddy + c];
            a = fmaf(g, ((float)x[t * ldx + c] - mean[t]) * rstd[t], a);
            b += g;
        }
    s[0][warp][lane] = a;
    s[1][warp][lane] = b;
    __syncthreads();
    if (warp < 2 && c < d) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) sum += s[warp][i][lane];
        partial[((int64_t)blockIdx.y * 2 + warp) * d + c] = sum;
    }
}

// dgamma and dbeta from n partial sums: a warp of the block takes every 8th, then the block's sums are joined.
__global__ void __launch_bounds__(256)
norm_join_kernel(const float *__restrict__ partial, int n, int d, float *__restrict__ dgamma, float *__restrict__ dbeta) {
    __shared__ float s[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float *out = blockIdx.y ? dbeta : dgamma;
    pdl_trigger();
    pdl_wait();
    if (!out) return;
    float sum = 0.f;
    if (c < d)
        for (int i = warp; i < n; i += 8) sum += partial[((int64_t)i * 2 + blockIdx.y) * d + c];
    s[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < d) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) sum += s[i][lane];
        out[c] = sum;
    }
}

// Row slices whose column sums are kept apart.
constexpr int kSlicesMax = 64;
int slices_of(int T) { return T < kSlicesMax ? (T < 1 ? 1 : T) : kSlicesMax; }

}  // namespace
}  // namespace omoe

using namespace omoe;

extern "C" {

int omoe_layer_norm(const void *x_dev, int64_t ldx, int32_t x_dtype, const float *gamma_dev, const float *beta_dev, float eps,
                    void *y_dev, int64_t ldy, int32_t y_dtype, float *mean_dev, float *rstd_dev, int32_t T, int32_t d,
                    void *cuda_stream) {
    const char *fn = "omoe_layer_norm";
    if (T < 0) return ops_fail(OMOE_ERR_INVALID, fn, "T must not be negative");
    if (!(eps >= 0.f)) return ops_fail(OMOE_ERR_INVALID, fn, "eps must not be negative");
    const Rows x = {x_dev, ldx, x_dtype, T, d}, y = {y_dev, ldy, y_dtype, T, d};
    if (const char *bad = rows_wrong(x)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (const char *bad = rows_wrong(y)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (rows_overlap(y, x)) return ops_fail(OMOE_ERR_INVALID, fn, "an output overlaps another buffer");
    if (misaligned(gamma_dev, 4) || misaligned(beta_dev, 4) || misaligned(mean_dev, 4) || misaligned(rstd_dev, 4))
        return ops_fail(OMOE_ERR_INVALID, fn, "fp32 buffers must be 4-byte aligned");
    if (T == 0) return ops_ok();
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    return ops_launched(by_types(x_dtype, y_dtype, [&](auto *xt, auto *yt) {
        using XT = std::remove_pointer_t<decltype(xt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        return launch_ex(norm_wide_kernel<XT, YT>, dim3(T), dim3(kWideThreads), 0, s, ops_pdl(), static_cast<const XT *>(x_dev),
                         ldx, gamma_dev, beta_dev, eps, static_cast<YT *>(y_dev), ldy, mean_dev, rstd_dev, d);
    }), fn);
}

int64_t omoe_layer_norm_backward_workspace(int32_t T, int32_t d) {
    if (T < 0 || d < 1) return OMOE_ERR_INVALID;
    return (int64_t)slices_of(T) * 2 * d * sizeof(float);
}

int omoe_layer_norm_backward(const void *dy_dev, int64_t lddy, int32_t dy_dtype, const void *x_dev, int64_t ldx, int32_t x_dtype,
                             const float *gamma_dev, const float *mean_dev, const float *rstd_dev, void *dx_dev, int64_t lddx,
                             float *dgamma_dev, float *dbeta_dev, int32_t T, int32_t d, void *workspace_dev,
                             int64_t workspace_bytes, void *cuda_stream) {
    const char *fn = "omoe_layer_norm_backward";
    if (T < 0) return ops_fail(OMOE_ERR_INVALID, fn, "T must not be negative");
    const Rows dx = {dx_dev, lddx, x_dtype, T, d}, dy = {dy_dev, lddy, dy_dtype, T, d}, x = {x_dev, ldx, x_dtype, T, d};
    for (const Rows *r : {&dx, &dy, &x})
        if (const char *bad = rows_wrong(*r)) return ops_fail(OMOE_ERR_INVALID, fn, bad);
    if (rows_overlap(dx, dy) || rows_overlap(dx, x)) return ops_fail(OMOE_ERR_INVALID, fn, "an output overlaps another buffer");
    if (T > 0 && (!mean_dev || !rstd_dev)) return ops_fail(OMOE_ERR_INVALID, fn, "null buffer");
    if (misaligned(gamma_dev, 4) || misaligned(mean_dev, 4) || misaligned(rstd_dev, 4) || misaligned(dgamma_dev, 4) ||
        misaligned(dbeta_dev, 4))
        return ops_fail(OMOE_ERR_INVALID, fn, "fp32 buffers must be 4-byte aligned");
    if (workspace_bytes < omoe_layer_norm_backward_workspace(T, d) || !workspace_dev || misaligned(workspace_dev, 16))
        return ops_fail(OMOE_ERR_INVALID, fn, "the workspace is missing, misaligned or too small");
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    float *partial = static_cast<float *>(workspace_dev);
    const int slices = slices_of(T), cols = ceil_div(d, 32);
    const bool params = dgamma_dev || dbeta_dev;
    return ops_launched(by_types(x_dtype, dy_dtype, [&](auto *xt, auto *yt) {
        using XT = std::remove_pointer_t<decltype(xt)>;
        using YT = std::remove_pointer_t<decltype(yt)>;
        const YT *g = static_cast<const YT *>(dy_dev);
        const XT *in = static_cast<const XT *>(x_dev);
        cudaError_t e = cudaSuccess;
        if (T > 0) {
            e = launch_ex(norm_bwd_wide_kernel<XT, YT>, dim3(T), dim3(kWideThreads), 0, s, ops_pdl(), g, lddy, in, ldx, gamma_dev,
                          mean_dev, rstd_dev, static_cast<XT *>(dx_dev), lddx, d);
            if (e != cudaSuccess || !params) return e;
        }
        if (!params) return e;
        e = launch_ex(norm_cols_kernel<XT, YT>, dim3(cols, slices), dim3(256), 0, s, ops_pdl(), g, lddy, in, ldx, mean_dev,
                      rstd_dev, partial, T, d, ceil_div(T, slices));
        if (e != cudaSuccess) return e;
        return launch_ex(norm_join_kernel, dim3(cols, 2), dim3(256), 0, s, ops_pdl(), partial, slices, d, dgamma_dev, dbeta_dev);
    }), fn);
}

}  // extern "C"
