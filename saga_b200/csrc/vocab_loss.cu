// Softmax cross entropy over the vocabulary with the classifier's product, and
// its gradient (b200opt_vocab_loss_* of include/b200opt.h).
#include <algorithm>

#include "lm_common.cuh"

namespace b200 {
namespace {

constexpr int kTile = 64;
constexpr size_t kPieceBytes = (size_t)256 << 20;  // of p - onehot held at a time
constexpr float kLift = 32768.0f;                  // 2^15: see the header

// acc[i][j] = sum_k A[m][k] B[n][k] for m = m0 + 4 ty + i, n = n0 + 4 tx + j.
__device__ __forceinline__ void tile_product(float acc[4][4], const __half *A, size_t am, size_t ak,
                                             const __half *B, size_t bn, size_t bk, size_t M,
                                             size_t N, size_t K, size_t m0, size_t n0)
{
    __shared__ float sa[16][kTile], sb[16][kTile];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for(int i = 0; i < 4; i++)
        for(int j = 0; j < 4; j++)
            acc[i][j] = 0.0f;
    for(size_t k0 = 0; k0 < K; k0 += 16) {
        for(int e = threadIdx.x; e < 16 * kTile; e += 256) {
            const size_t k = k0 + e / kTile, m = m0 + e % kTile, n = n0 + e % kTile;
            sa[e / kTile][e % kTile] = k < K && m < M ? __half2float(A[m * am + k * ak]) : 0.0f;
            sb[e / kTile][e % kTile] = k < K && n < N ? __half2float(B[n * bn + k * bk]) : 0.0f;
        }
        __syncthreads();
        for(int k = 0; k < 16; k++)
            for(int i = 0; i < 4; i++)
                for(int j = 0; j < 4; j++)
                    acc[i][j] += sa[k][4 * ty + i] * sb[k][4 * tx + j];
        __syncthreads();
    }
}

// Per row and tile of the vocabulary: the maximum and the sum of exp(z - max).
__global__ void logits_stats_kernel(size_t T, size_t V, size_t D, const __half *x, size_t xs,
                                    const __half *w, size_t ws, const void *y, int wide,
                                    float2 *part, float *zt)
{
    __shared__ float z[kTile][kTile + 1];
    const size_t m0 = (size_t)blockIdx.x * kTile, n0 = (size_t)blockIdx.y * kTile;
    float acc[4][4];
    tile_product(acc, x, xs, 1, w, ws, 1, T, V, D, m0, n0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for(int i = 0; i < 4; i++)
        for(int j = 0; j < 4; j++)
            z[4 * ty + i][4 * tx + j] = acc[i][j];
    __syncthreads();
    const size_t t = m0 + threadIdx.x;
    if(threadIdx.x >= kTile || t >= T)
        return;
    const int n = (int)min((size_t)kTile, V - n0), at = lm_index_at(y, wide, t, V);
    float top = -INFINITY, sum = 0.0f;
    for(int j = 0; j < n; j++)
        top = fmaxf(top, z[threadIdx.x][j]);
    for(int j = 0; j < n; j++)
        sum += expf(z[threadIdx.x][j] - top);
    part[blockIdx.y * T + t] = make_float2(top, sum);
    if(at >= 0 && (size_t)at >= n0 && (size_t)at < n0 + n)
        zt[t] = z[threadIdx.x][at - n0];
}

__global__ void loss_kernel(size_t T, size_t V, size_t tiles, const float2 *part, const float *zt,
                            const void *y, int wide, float *loss, float *lse)
{
    const size_t t = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if(t >= T)
        return;
    float top = -INFINITY, sum = 0.0f;
    for(size_t i = 0; i < tiles; i++)
        top = fmaxf(top, part[i * T + t].x);
    for(size_t i = 0; i < tiles; i++)
        sum += part[i * T + t].y * expf(part[i * T + t].x - top);
    const float l = top + logf(sum);
    lse[t] = l;
    loss[t] = lm_index_at(y, wide, t, V) >= 0 ? l - zt[t] : 0.0f;
}

__global__ void stats_kernel(size_t T, size_t V, const float *loss, const void *y, int wide,
                             float *stats)
{
    __shared__ float red[32];
    float s = 0.0f, n = 0.0f;
    for(size_t t = threadIdx.x; t < T; t += blockDim.x) {
        s += loss[t];
        n += lm_index_at(y, wide, t, V) >= 0 ? 1.0f : 0.0f;
    }
    s = block_sum(s, red);
    n = block_sum(n, red);
    if(threadIdx.x == 0) {
        stats[0] = s;
        stats[1] = n;
    }
}

// dz[t][v - first] = 2^15 (p - onehot), 0 for ignored tokens
__global__ void dz_kernel(size_t T, size_t V, size_t D, const __half *x, size_t xs, const __half *w,
                          size_t ws, const void *y, int wide, const float *lse, size_t first,
                          size_t count, __half *dz, size_t dzs)
{
    const size_t m0 = (size_t)blockIdx.x * kTile, n0 = (size_t)blockIdx.y * kTile;
    float acc[4][4];
    tile_product(acc, x, xs, 1, w + first * ws, ws, 1, T, count, D, m0, n0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for(int i = 0; i < 4; i++) {
        const size_t t = m0 + 4 * ty + i;
        if(t >= T)
            continue;
        const int at = lm_index_at(y, wide, t, V);
        for(int j = 0; j < 4; j++) {
            const size_t n = n0 + 4 * tx + j;
            if(n >= count)
                continue;
            const float p = expf(acc[i][j] - lse[t]) - ((size_t)at == first + n ? 1.0f : 0.0f);
            dz[t * dzs + n] = __float2half_rn(at >= 0 ? p * kLift : 0.0f);
        }
    }
}

__device__ __forceinline__ float factor_of(float scale, const float *loss_scale, const float *stats)
{
    const float f = loss_scale ? scale * *loss_scale : scale;
    return stats ? f / fmaxf(stats[1], 1.0f) : f;
}

// sum32 += A B^T; with `out`, out = factor 2^-15 sum instead
__global__ void product_kernel(size_t M, size_t N, size_t K, const __half *A, size_t am, size_t ak,
                               const __half *B, size_t bn, size_t bk, float *sum32, int begin,
                               __half *out, size_t os, int accumulate, float scale,
                               const float *loss_scale, const float *stats)
{
    const size_t m0 = (size_t)blockIdx.x * kTile, n0 = (size_t)blockIdx.y * kTile;
    float acc[4][4];
    tile_product(acc, A, am, ak, B, bn, bk, M, N, K, m0, n0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float f = factor_of(scale, loss_scale, stats) * (1.0f / kLift);
    for(int i = 0; i < 4; i++)
        for(int j = 0; j < 4; j++) {
            const size_t m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
            if(m >= M || n >= N)
                continue;
            float v = acc[i][j];
            if(sum32 && !begin)
                v += sum32[m * N + n];
            if(out)
                out[m * os + n] = __float2half_rn(f * v + (accumulate ? __half2float(out[m * os + n]) : 0.0f));
            else
                sum32[m * N + n] = v;
        }
}

size_t piece_of(size_t T, size_t V)
{
    const size_t most = std::max<size_t>(kPieceBytes / 2 / std::max<size_t>(T, 1) / 256 * 256, 256);
    return std::min(lm_up(V, 8), most);
}

bool lm_head(size_t T, size_t V, size_t D, const void *x, size_t xs, const void *w, size_t ws,
             const void *y, int index_bytes)
{
    return D % 8 == 0 && xs % 8 == 0 && ws % 8 == 0 && lm_aligned(x, 16) && lm_aligned(w, 16) &&
           lm_matrix(x, T, D, xs, 2) && lm_matrix(w, V, D, ws, 2) && (!T || y) &&
           lm_aligned(y, index_bytes);
}

unsigned tiles_of(size_t n) { return (unsigned)((n + kTile - 1) / kTile); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200opt_vocab_loss_fwd_workspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes)
{
    if(!bytes || !vocab || !dim)
        return B200OPT_EINVAL;
    if(tokens > B200OPT_LM_MAX || vocab > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    *bytes = lm_up(tokens * 4, 256) + (size_t)tiles_of(vocab) * tokens * 8;
    return B200OPT_OK;
}

int b200opt_vocab_loss_fwd(size_t tokens, size_t vocab, size_t dim, const void *hidden,
                           size_t hidden_stride, const void *weight, size_t weight_stride,
                           const void *targets, int index_bytes, float *loss, float *lse,
                           float *stats, void *workspace, size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    const int rc = b200opt_vocab_loss_fwd_workspace(tokens, vocab, dim, &need);
    if(rc)
        return rc;
    if(!lm_index(index_bytes) ||
       !lm_head(tokens, vocab, dim, hidden, hidden_stride, weight, weight_stride, targets, index_bytes) ||
       (tokens && (!loss || !lse)) || !lm_aligned(loss, 4) || !lm_aligned(lse, 4) ||
       !lm_aligned(stats, 4) || workspace_bytes < need ||
       (need && (!workspace || !lm_aligned(workspace, 256))))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    const int wide = index_bytes == 8;
    float *zt = (float *)workspace;
    float2 *part = (float2 *)((char *)workspace + lm_up(tokens * 4, 256));
    if(tokens) {
        logits_stats_kernel<<<dim3(tiles_of(tokens), tiles_of(vocab)), 256, 0, st>>>(
            tokens, vocab, dim, (const __half *)hidden, hidden_stride, (const __half *)weight,
            weight_stride, targets, wide, part, zt);
        loss_kernel<<<(unsigned)((tokens + 127) / 128), 128, 0, st>>>(
            tokens, vocab, tiles_of(vocab), part, zt, targets, wide, loss, lse);
    }
    if(stats)
        stats_kernel<<<1, 1024, 0, st>>>(tokens, vocab, loss, targets, wide, stats);
    return lm_launched();
}

int b200opt_vocab_loss_bwd_workspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes)
{
    if(!bytes || !vocab || !dim)
        return B200OPT_EINVAL;
    if(tokens > B200OPT_LM_MAX || vocab > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    *bytes = lm_up(tokens * piece_of(tokens, vocab) * 2, 256) + tokens * dim * 4;
    return B200OPT_OK;
}

int b200opt_vocab_loss_bwd(size_t tokens, size_t vocab, size_t dim, const void *hidden,
                           size_t hidden_stride, const void *weight, size_t weight_stride,
                           const void *targets, int index_bytes, const float *lse,
                           const float *stats, float grad_scale, const float *loss_scale,
                           void *grad_hidden, size_t grad_hidden_stride, void *grad_weight,
                           size_t grad_weight_stride, int accumulate, void *workspace,
                           size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    const int rc = b200opt_vocab_loss_bwd_workspace(tokens, vocab, dim, &need);
    if(rc)
        return rc;
    if(!lm_index(index_bytes) ||
       !lm_head(tokens, vocab, dim, hidden, hidden_stride, weight, weight_stride, targets, index_bytes) ||
       (tokens && !lse) || !lm_aligned(lse, 4) || !lm_aligned(stats, 4) || !lm_aligned(loss_scale, 4) ||
       (grad_hidden && (!lm_matrix(grad_hidden, tokens, dim, grad_hidden_stride, 2) ||
                        !lm_aligned(grad_hidden, 16) || grad_hidden_stride % 8)) ||
       (grad_weight && (!lm_matrix(grad_weight, vocab, dim, grad_weight_stride, 2) ||
                        !lm_aligned(grad_weight, 16) || grad_weight_stride % 8)) ||
       workspace_bytes < need || (need && (!workspace || !lm_aligned(workspace, 256))))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    const int wide = index_bytes == 8;
    const __half *x = (const __half *)hidden, *w = (const __half *)weight;
    __half *dz = (__half *)workspace;
    const size_t piece = piece_of(tokens, vocab);
    float *sum = (float *)((char *)workspace + lm_up(tokens * piece * 2, 256));
    for(size_t first = 0; first < vocab; first += piece) {
        const size_t count = std::min(piece, vocab - first);
        const bool last = first + count == vocab;
        if(tokens)
            dz_kernel<<<dim3(tiles_of(tokens), tiles_of(count)), 256, 0, st>>>(
                tokens, vocab, dim, x, hidden_stride, w, weight_stride, targets, wide, lse, first,
                count, dz, piece);
        if(grad_hidden && tokens)
            product_kernel<<<dim3(tiles_of(tokens), tiles_of(dim)), 256, 0, st>>>(
                tokens, dim, count, dz, piece, 1, w + first * weight_stride, 1, weight_stride, sum,
                first == 0, last ? (__half *)grad_hidden : nullptr, grad_hidden_stride, 0, grad_scale,
                loss_scale, stats);
        if(grad_weight)
            product_kernel<<<dim3(tiles_of(count), tiles_of(dim)), 256, 0, st>>>(
                count, dim, tokens, dz, 1, piece, x, 1, hidden_stride, nullptr, 1,
                (__half *)grad_weight + first * grad_weight_stride, grad_weight_stride, accumulate,
                grad_scale, loss_scale, stats);
    }
    return lm_launched();
}

}  // extern "C"
