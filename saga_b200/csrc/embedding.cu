// Embedding lookup and its gradient (b200opt_embedding_* of include/b200opt.h).
#include "lm_common.cuh"

namespace b200 {
namespace {

template <typename T>
__global__ void embedding_fwd_kernel(size_t vocab, size_t dim, const void *ids, int wide,
                                     const T *weight, size_t ws, float scale, T *out, size_t os)
{
    const size_t t = blockIdx.x;
    const int id = lm_index_at(ids, wide, t, vocab);
    for(size_t d = threadIdx.x; d < dim; d += blockDim.x)
        lm_store(out + t * os + d, id < 0 ? 0.0f : scale * lm_load(weight + id * ws + d));
}

// One block per row of the table: looks for its tokens among all ids.
template <typename T>
__global__ void embedding_bwd_kernel(size_t tokens, size_t vocab, size_t dim, const void *ids,
                                     int wide, const T *dy, size_t ys, float scale, T *dw,
                                     size_t ws, int accumulate)
{
    const int v = blockIdx.x;
    const size_t d = (size_t)blockIdx.y * blockDim.x + threadIdx.x;
    float sum = 0.0f;
    bool any = false;
    for(size_t t = 0; t < tokens; t++)
        if(lm_index_at(ids, wide, t, vocab) == v) {
            any = true;
            if(d < dim)
                sum += lm_load(dy + t * ys + d);
        }
    if(d >= dim || (accumulate && !any))
        return;
    T *to = dw + v * ws + d;
    lm_store(to, scale * sum + (accumulate ? lm_load(to) : 0.0f));
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200opt_embedding_fwd(int dtype, size_t tokens, size_t vocab, size_t dim, const void *ids,
                          int index_bytes, const void *weight, size_t weight_stride, float scale,
                          void *out, size_t out_stride, void *stream)
{
    if(!lm_dtype(dtype) || !lm_index(index_bytes))
        return B200OPT_EINVAL;
    if(tokens > B200OPT_LM_MAX || vocab > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    if(!tokens || !dim)
        return B200OPT_OK;
    const size_t e = lm_size(dtype);
    if(!ids || !lm_aligned(ids, index_bytes) ||
       !lm_matrix(weight, vocab, dim, weight_stride, e) || !lm_matrix(out, tokens, dim, out_stride, e))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    if(dtype == B200OPT_HALF)
        embedding_fwd_kernel<<<(unsigned)tokens, 256, 0, st>>>(vocab, dim, ids, index_bytes == 8, (const __half *)weight,
                                                     weight_stride, scale, (__half *)out, out_stride);
    else
        embedding_fwd_kernel<<<(unsigned)tokens, 256, 0, st>>>(vocab, dim, ids, index_bytes == 8, (const float *)weight,
                                                     weight_stride, scale, (float *)out, out_stride);
    return lm_launched();
}

int b200opt_embedding_bwd_workspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes)
{
    if(!bytes)
        return B200OPT_EINVAL;
    if(tokens > B200OPT_LM_MAX || vocab > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    *bytes = 0;
    return B200OPT_OK;
}

int b200opt_embedding_bwd(int dtype, size_t tokens, size_t vocab, size_t dim, const void *ids,
                          int index_bytes, const void *grad_out, size_t grad_out_stride, float scale,
                          void *grad_weight, size_t grad_weight_stride, int accumulate,
                          void *workspace, size_t workspace_bytes, void *stream)
{
    if(!lm_dtype(dtype) || !lm_index(index_bytes))
        return B200OPT_EINVAL;
    size_t need = 0;
    const int rc = b200opt_embedding_bwd_workspace(tokens, vocab, dim, &need);
    if(rc)
        return rc;
    if(!vocab || !dim)
        return B200OPT_OK;
    const size_t e = lm_size(dtype);
    if((tokens && (!ids || !lm_aligned(ids, index_bytes))) ||
       !lm_matrix(grad_out, tokens, dim, grad_out_stride, e) ||
       !lm_matrix(grad_weight, vocab, dim, grad_weight_stride, e) ||
       workspace_bytes < need || (need && (!workspace || !lm_aligned(workspace, 256))))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid((unsigned)vocab, (unsigned)((dim + 255) / 256));
    if(dtype == B200OPT_HALF)
        embedding_bwd_kernel<<<grid, 256, 0, st>>>(tokens, vocab, dim, ids, index_bytes == 8, (const __half *)grad_out,
            grad_out_stride, scale, (__half *)grad_weight, grad_weight_stride, accumulate);
    else
        embedding_bwd_kernel<<<grid, 256, 0, st>>>(tokens, vocab, dim, ids, index_bytes == 8, (const float *)grad_out,
            grad_out_stride, scale, (float *)grad_weight, grad_weight_stride, accumulate);
    return lm_launched();
}

}  // extern "C"
