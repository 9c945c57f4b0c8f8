// Layer norm and its gradient (b200opt_layernorm_* of include/b200opt.h).
#include "lm_common.cuh"

namespace b200 {
namespace {

template <typename T, typename P>
__global__ void layernorm_fwd_kernel(size_t dim, const T *x, size_t xs, const P *gamma,
                                     const P *beta, float eps, T *y, size_t ys, float *mean,
                                     float *rstd)
{
    __shared__ float red[32];
    const size_t r = blockIdx.x;
    x += r * xs;
    y += r * ys;
    float s = 0.0f;
    for(size_t d = threadIdx.x; d < dim; d += blockDim.x)
        s += lm_load(x + d);
    const float mu = block_sum(s, red) / (float)dim;
    s = 0.0f;
    for(size_t d = threadIdx.x; d < dim; d += blockDim.x) {
        const float c = lm_load(x + d) - mu;
        s += c * c;
    }
    const float rs = 1.0f / sqrtf(block_sum(s, red) / (float)dim + eps);
    for(size_t d = threadIdx.x; d < dim; d += blockDim.x)
        lm_store(y + d, (lm_load(x + d) - mu) * rs * (gamma ? lm_load(gamma + d) : 1.0f) +
                            (beta ? lm_load(beta + d) : 0.0f));
    if(threadIdx.x == 0) {
        if(mean)
            mean[r] = mu;
        if(rstd)
            rstd[r] = rs;
    }
}

template <typename T, typename P>
__global__ void layernorm_bwd_x_kernel(size_t dim, const T *dy, size_t ys, const T *x, size_t xs,
                                       const P *gamma, const float *mean, const float *rstd, T *dx,
                                       size_t dxs)
{
    __shared__ float red[32];
    const size_t r = blockIdx.x;
    const float mu = mean[r], rs = rstd[r];
    float a = 0.0f, b = 0.0f;
    for(size_t d = threadIdx.x; d < dim; d += blockDim.x) {
        const float g = lm_load(dy + r * ys + d) * (gamma ? lm_load(gamma + d) : 1.0f);
        a += g;
        b += g * ((lm_load(x + r * xs + d) - mu) * rs);
    }
    a = block_sum(a, red) / (float)dim;
    b = block_sum(b, red) / (float)dim;
    for(size_t d = threadIdx.x; d < dim; d += blockDim.x) {
        const float g = lm_load(dy + r * ys + d) * (gamma ? lm_load(gamma + d) : 1.0f);
        lm_store(dx + r * dxs + d, rs * (g - a - (lm_load(x + r * xs + d) - mu) * rs * b));
    }
}

template <typename T, typename P>
__global__ void layernorm_bwd_params_kernel(size_t rows, size_t dim, const T *dy, size_t ys,
                                            const T *x, size_t xs, const float *mean,
                                            const float *rstd, P *dgamma, P *dbeta, int accumulate)
{
    const size_t d = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if(d >= dim)
        return;
    float g = 0.0f, b = 0.0f;
    for(size_t r = 0; r < rows; r++) {
        const float v = lm_load(dy + r * ys + d);
        g += v * ((lm_load(x + r * xs + d) - mean[r]) * rstd[r]);
        b += v;
    }
    if(dgamma)
        lm_store(dgamma + d, g + (accumulate ? lm_load(dgamma + d) : 0.0f));
    if(dbeta)
        lm_store(dbeta + d, b + (accumulate ? lm_load(dbeta + d) : 0.0f));
}

template <typename T, typename P>
int fwd(size_t rows, size_t dim, const void *x, size_t xs, const void *gamma, const void *beta,
        float eps, void *y, size_t ys, float *mean, float *rstd, cudaStream_t st)
{
    layernorm_fwd_kernel<<<(unsigned)rows, 256, 0, st>>>(dim, (const T *)x, xs, (const P *)gamma,
                                               (const P *)beta, eps, (T *)y, ys, mean, rstd);
    return lm_launched();
}

template <typename T, typename P>
int bwd(size_t rows, size_t dim, const void *dy, size_t ys, const void *x, size_t xs,
        const void *gamma, const float *mean, const float *rstd, void *dx, size_t dxs, void *dgamma,
        void *dbeta, int accumulate, cudaStream_t st)
{
    if(dx && rows)
        layernorm_bwd_x_kernel<<<(unsigned)rows, 256, 0, st>>>(dim, (const T *)dy, ys, (const T *)x, xs,
                                                     (const P *)gamma, mean, rstd, (T *)dx, dxs);
    if(dgamma || dbeta)
        layernorm_bwd_params_kernel<<<(unsigned)((dim + 255) / 256), 256, 0, st>>>(
            rows, dim, (const T *)dy, ys, (const T *)x, xs, mean, rstd, (P *)dgamma, (P *)dbeta, accumulate);
    return lm_launched();
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200opt_layernorm_fwd(int dtype, int param_dtype, size_t rows, size_t dim, const void *x,
                          size_t x_stride, const void *gamma, const void *beta, float eps, void *y,
                          size_t y_stride, float *mean, float *rstd, void *stream)
{
    if(!lm_dtype(dtype) || !lm_dtype(param_dtype) ||
       (param_dtype == B200OPT_HALF && dtype != B200OPT_HALF) || !(eps >= 0.0f))
        return B200OPT_EINVAL;
    if(rows > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    if(!rows || !dim)
        return B200OPT_OK;
    const size_t e = lm_size(dtype), p = lm_size(param_dtype);
    if(!lm_matrix(x, rows, dim, x_stride, e) || !lm_matrix(y, rows, dim, y_stride, e) ||
       !lm_aligned(gamma, p) || !lm_aligned(beta, p) || !lm_aligned(mean, 4) || !lm_aligned(rstd, 4))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    if(dtype == B200OPT_FLOAT)
        return fwd<float, float>(rows, dim, x, x_stride, gamma, beta, eps, y, y_stride, mean, rstd, st);
    if(param_dtype == B200OPT_FLOAT)
        return fwd<__half, float>(rows, dim, x, x_stride, gamma, beta, eps, y, y_stride, mean, rstd, st);
    return fwd<__half, __half>(rows, dim, x, x_stride, gamma, beta, eps, y, y_stride, mean, rstd, st);
}

int b200opt_layernorm_bwd_workspace(size_t rows, size_t dim, size_t *bytes)
{
    if(!bytes)
        return B200OPT_EINVAL;
    if(rows > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    *bytes = 0;
    return B200OPT_OK;
}

int b200opt_layernorm_bwd(int dtype, int param_dtype, size_t rows, size_t dim, const void *grad_y,
                          size_t grad_y_stride, const void *x, size_t x_stride, const void *gamma,
                          const float *mean, const float *rstd, void *grad_x, size_t grad_x_stride,
                          void *grad_gamma, void *grad_beta, int accumulate, void *workspace,
                          size_t workspace_bytes, void *stream)
{
    if(!lm_dtype(dtype) || !lm_dtype(param_dtype) ||
       (param_dtype == B200OPT_HALF && dtype != B200OPT_HALF))
        return B200OPT_EINVAL;
    size_t need = 0;
    const int rc = b200opt_layernorm_bwd_workspace(rows, dim, &need);
    if(rc)
        return rc;
    if(!dim)
        return B200OPT_OK;
    const size_t e = lm_size(dtype), p = lm_size(param_dtype);
    if(!lm_matrix(grad_y, rows, dim, grad_y_stride, e) || !lm_matrix(x, rows, dim, x_stride, e) ||
       (rows && (!mean || !rstd)) || !lm_aligned(mean, 4) || !lm_aligned(rstd, 4) ||
       (grad_x && !lm_matrix(grad_x, rows, dim, grad_x_stride, e)) || !lm_aligned(gamma, p) ||
       !lm_aligned(grad_gamma, p) || !lm_aligned(grad_beta, p) || workspace_bytes < need ||
       (need && (!workspace || !lm_aligned(workspace, 256))))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    if(dtype == B200OPT_FLOAT)
        return bwd<float, float>(rows, dim, grad_y, grad_y_stride, x, x_stride, gamma, mean, rstd,
                                 grad_x, grad_x_stride, grad_gamma, grad_beta, accumulate, st);
    if(param_dtype == B200OPT_FLOAT)
        return bwd<__half, float>(rows, dim, grad_y, grad_y_stride, x, x_stride, gamma, mean, rstd,
                                  grad_x, grad_x_stride, grad_gamma, grad_beta, accumulate, st);
    return bwd<__half, __half>(rows, dim, grad_y, grad_y_stride, x, x_stride, gamma, mean, rstd,
                               grad_x, grad_x_stride, grad_gamma, grad_beta, accumulate, st);
}

}  // extern "C"
