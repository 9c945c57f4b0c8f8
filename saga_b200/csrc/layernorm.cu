// Layer norm and its gradient (b200opt_layernorm_* of include/b200opt.h).
#include <algorithm>
#include <type_traits>

#include "lm_common.cuh"

namespace b200 {
namespace {

// threads of a block: eight rows of a warp each, or one row of WARPS warps
__host__ __device__ constexpr int threads_of(int warps) { return warps == 1 ? 256 : 32 * warps; }
__host__ __device__ constexpr int rows_of(int warps) { return warps == 1 ? 8 : 1; }
constexpr int kMaxParts = 444;  // blocks of the gradient kernel at most: three on each of 148 SMs

// Sums over the threads that share a row: a warp, or the block.  `turn` alternates
// between two sets of slots, so that one barrier a sum is enough.
template <int WARPS, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*slots)[16][K], int &turn)
{
#pragma unroll
    for(int k = 0; k < K; k++)
        v[k] = warp_sum(v[k]);
    if(WARPS == 1)
        return;
    const int warp = threadIdx.x >> 5;
    if((threadIdx.x & 31) == 0)
        for(int k = 0; k < K; k++)
            slots[turn][warp][k] = v[k];
    __syncthreads();
#pragma unroll
    for(int k = 0; k < K; k++) {
        v[k] = 0.0f;
#pragma unroll
        for(int w = 0; w < WARPS; w++)
            v[k] += slots[turn][w][k];
    }
    turn ^= 1;
}

// Two sums at once over the WARPS warps of a group that shares a row, of a block of
// BLOCK warps: the halves of a warp exchange, then each carries one of the sums.
template <int WARPS, int BLOCK>
__device__ __forceinline__ float2 row_pair(float a, float b, float (*slots)[2][16], int &turn)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / WARPS;
    const bool low = lane < 16;
    float v = (low ? a : b) + __shfl_xor_sync(0xffffffffu, low ? b : a, 16);
#pragma unroll
    for(int o = 8; o; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    if(WARPS == 1)
        return make_float2(__shfl_sync(0xffffffffu, v, 0), __shfl_sync(0xffffffffu, v, 16));
    if((lane & 15) == 0)
        slots[turn][lane >> 4][warp] = v;
    if(WARPS == BLOCK)
        __syncthreads();
    else
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * WARPS) : "memory");
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for(int w = 0; w < WARPS; w++)
        s.x += slots[turn][0][group * WARPS + w], s.y += slots[turn][1][group * WARPS + w];
    turn ^= 1;
    return s;
}

// Brings a row into L2: 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void prefetch_row(const void *row, uint32_t bytes)
{
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row), "r"(bytes) : "memory");
}

template <typename P, int N>
__device__ __forceinline__ void load_param(const P *p, size_t c, float fill, float (&f)[N])
{
    if(p) {
        reinterpret_cast<const Vec<P, N> *>(p)[c].get(f);
    } else {
#pragma unroll
        for(int i = 0; i < N; i++)
            f[i] = fill;
    }
}

// A row stays in the registers of a warp (WARPS 1) or of the block, NV vectors of
// N elements a thread: it is read once, and the variance is taken around the mean
// in a second pass over the registers.  ROWS rows go through together: they share
// the barriers and the loads of the parameters, whose way through L1 is what bounds
// one row at a time (16384 x 4096 fp16 with fp32 parameters: 53 us one by one, 44 us
// in pairs, 45 in threes; a plain copy of the same bytes takes 45).
template <typename T, typename P, int N, int NV, int WARPS, int ROWS>
__global__ void __launch_bounds__(threads_of(WARPS))
    layernorm_fwd_kernel(size_t rows, size_t dim, const T *x, size_t xs, const P *gamma, const P *beta,
                         float eps, T *y, size_t ys, float *mean, float *rstd)
{
    __shared__ float slots[2][16][ROWS];
    int turn = 0;
    constexpr int L = 32 * WARPS;
    const size_t r0 = ((size_t)blockIdx.x * rows_of(WARPS) + threadIdx.x / L) * ROWS;
    const int l = threadIdx.x % L, vecs = (int)(dim / N);
    if(WARPS == 1 && r0 >= rows)
        return;
    Vec<T, N> v[ROWS][NV];
#pragma unroll
    for(int k = 0; k < ROWS; k++)
#pragma unroll
        for(int i = 0; i < NV; i++)
            if(l + i * L < vecs && r0 + k < rows)
                v[k][i] = reinterpret_cast<const Vec<T, N> *>(x + (r0 + k) * xs)[l + i * L];
    float mu[ROWS], rs[ROWS];
#pragma unroll
    for(int k = 0; k < ROWS; k++) {
        mu[k] = 0.0f;
#pragma unroll
        for(int i = 0; i < NV; i++)
            if(l + i * L < vecs) {
                float f[N];
                v[k][i].get(f);
#pragma unroll
                for(int j = 0; j < N; j++)
                    mu[k] += f[j];
            }
    }
    row_sums<WARPS, ROWS>(mu, slots, turn);
#pragma unroll
    for(int k = 0; k < ROWS; k++) {
        mu[k] /= (float)dim;
        rs[k] = 0.0f;
#pragma unroll
        for(int i = 0; i < NV; i++)
            if(l + i * L < vecs) {
                float f[N];
                v[k][i].get(f);
#pragma unroll
                for(int j = 0; j < N; j++)
                    rs[k] += (f[j] - mu[k]) * (f[j] - mu[k]);
            }
    }
    row_sums<WARPS, ROWS>(rs, slots, turn);
#pragma unroll
    for(int k = 0; k < ROWS; k++)
        rs[k] = 1.0f / sqrtf(rs[k] / (float)dim + eps);
#pragma unroll
    for(int i = 0; i < NV; i++)
        if(l + i * L < vecs) {
            float g[N], b[N];
            load_param<P, N>(gamma, l + i * L, 1.0f, g);
            load_param<P, N>(beta, l + i * L, 0.0f, b);
#pragma unroll
            for(int k = 0; k < ROWS; k++) {
                float f[N];
                v[k][i].get(f);
#pragma unroll
                for(int j = 0; j < N; j++)
                    f[j] = fmaf((f[j] - mu[k]) * rs[k], g[j], b[j]);
                v[k][i].set(f);
                if(r0 + k < rows)
                    reinterpret_cast<Vec<T, N> *>(y + (r0 + k) * ys)[l + i * L] = v[k][i];
            }
        }
    if(l == 0)
#pragma unroll
        for(int k = 0; k < ROWS; k++)
            if(r0 + k < rows) {
                if(mean)
                    mean[r0 + k] = mu[k];
                if(rstd)
                    rstd[r0 + k] = rs[k];
            }
}

// Rows too long for the registers: three passes over memory.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
    layernorm_fwd_long_kernel(size_t dim, const T *x, size_t xs, const P *gamma, const P *beta,
                              float eps, T *y, size_t ys, float *mean, float *rstd)
{
    __shared__ float red[32];
    const size_t r = blockIdx.x;
    x += r * xs;
    y += r * ys;
    float s = 0.0f;
    for(size_t d = threadIdx.x; d < dim; d += 1024)
        s += lm_load(x + d);
    const float mu = block_sum(s, red) / (float)dim;
    s = 0.0f;
    for(size_t d = threadIdx.x; d < dim; d += 1024) {
        const float c = lm_load(x + d) - mu;
        s += c * c;
    }
    const float rs = 1.0f / sqrtf(block_sum(s, red) / (float)dim + eps);
    for(size_t d = threadIdx.x; d < dim; d += 1024)
        lm_store(y + d, fmaf((lm_load(x + d) - mu) * rs, gamma ? lm_load(gamma + d) : 1.0f,
                             beta ? lm_load(beta + d) : 0.0f));
    if(threadIdx.x == 0) {
        if(mean)
            mean[r] = mu;
        if(rstd)
            rstd[r] = rs;
    }
}

// The gradient in one pass over x and grad_y.  A block walks over rows; each
// thread keeps the parameters' sums of its own columns in registers and leaves
// them in `parts` at the end, for params_kernel to join in a fixed order.  The
// next row's vectors are loaded before the present row's sums are waited for.
// Blocks of the gradient kernel: 256 threads, several groups of WARPS warps with a
// row each, or 512; and how many an SM is to hold, by the columns a thread has.
__host__ __device__ constexpr int bwd_warps(int warps) { return warps > 8 ? warps : 8; }
__host__ __device__ constexpr int bwd_blocks(int columns, bool halves)
{
    return columns <= 8 && halves ? 3 : columns <= 16 ? 2 : 1;
}

template <typename T, typename P, int N, int NV, int WARPS>
__global__ void __launch_bounds__(32 * bwd_warps(WARPS), bwd_blocks(N * NV, N == 8))
    layernorm_bwd_kernel(size_t rows, size_t dim, const T *dy, size_t ys, const T *x, size_t xs,
                         const P *gamma, const float *mean, const float *rstd, T *dx, size_t dxs,
                         float *parts)
{
    constexpr int BLOCK = bwd_warps(WARPS), R = BLOCK / WARPS, L = 32 * WARPS, THREADS = 32 * BLOCK;
    __shared__ __align__(16) float slots[2][2][16];
    __shared__ float joined[R > 1 ? 2 * L * NV * N : 1];
    int turn = 0;
    const int l = threadIdx.x % L, vecs = (int)(dim / N);
    const size_t step = (size_t)gridDim.x * R;
    const float inverse = 1.0f / (float)dim;
    float sg[NV][N], sb[NV][N];
#pragma unroll
    for(int i = 0; i < NV; i++)
#pragma unroll
        for(int j = 0; j < N; j++)
            sg[i][j] = sb[i][j] = 0.0f;

    size_t r = (size_t)blockIdx.x * R + threadIdx.x / L;
    Vec<T, N> vx[NV], vy[NV];
    float mu = 0.0f, rs = 0.0f;
    auto fetch = [&](size_t row, Vec<T, N> *a, Vec<T, N> *b, float &m, float &q) {
        if(row >= rows)
            return;
        m = mean[row];
        q = rstd[row];
        const Vec<T, N> *px = reinterpret_cast<const Vec<T, N> *>(x + row * xs);
        const Vec<T, N> *py = reinterpret_cast<const Vec<T, N> *>(dy + row * ys);
#pragma unroll
        for(int i = 0; i < NV; i++)
            if(l + i * L < vecs) {
                a[i] = px[l + i * L];
                b[i] = py[l + i * L];
            }
    };
    // registers for the next row's vectors, and for xh and d between the two passes: not
    // with 512 threads
    constexpr bool kRoom = BLOCK == 8;
    fetch(r, vx, vy, mu, rs);
    // the threads of a group agree on r
    for(; r < rows; r += step) {
        if(N > 1 && l == 0 && r + 2 * step < rows) {  // two rows ahead, as far as L2
            prefetch_row(x + (r + 2 * step) * xs, (uint32_t)(dim * sizeof(T)));
            prefetch_row(dy + (r + 2 * step) * ys, (uint32_t)(dim * sizeof(T)));
        }
        Vec<T, N> nx[kRoom ? NV : 1], ny[kRoom ? NV : 1];
        float nmu = 0.0f, nrs = 0.0f;
        if constexpr(kRoom)
            fetch(r + step, nx, ny, nmu, nrs);
        float s[2] = {0.0f, 0.0f}, xh[kRoom ? NV : 1][N], d[kRoom ? NV : 1][N];
#pragma unroll
        for(int i = 0; i < NV; i++)
            if(l + i * L < vecs) {
                float fx[N], fy[N], g[N];
                const int k = kRoom ? i : 0;
                vx[i].get(fx);
                vy[i].get(fy);
                load_param<P, N>(gamma, l + i * L, 1.0f, g);
#pragma unroll
                for(int j = 0; j < N; j++) {
                    xh[k][j] = (fx[j] - mu) * rs;
                    d[k][j] = fy[j] * g[j];
                    sg[i][j] = fmaf(fy[j], xh[k][j], sg[i][j]);
                    sb[i][j] += fy[j];
                    s[0] += d[k][j];
                    s[1] = fmaf(d[k][j], xh[k][j], s[1]);
                }
            }
        if(dx) {
            const float2 t = row_pair<WARPS, BLOCK>(s[0], s[1], slots, turn);
            const float a = t.x * inverse, b = t.y * inverse;
            Vec<T, N> *to = reinterpret_cast<Vec<T, N> *>(dx + r * dxs);
#pragma unroll
            for(int i = 0; i < NV; i++)
                if(l + i * L < vecs) {
                    float f[N];
                    const int k = kRoom ? i : 0;
                    if constexpr(!kRoom) {
                        vx[i].get(xh[0]);
                        vy[i].get(d[0]);
                        load_param<P, N>(gamma, l + i * L, 1.0f, f);
#pragma unroll
                        for(int j = 0; j < N; j++) {
                            xh[0][j] = (xh[0][j] - mu) * rs;
                            d[0][j] *= f[j];
                        }
                    }
#pragma unroll
                    for(int j = 0; j < N; j++)
                        f[j] = rs * fmaf(-b, xh[k][j], d[k][j] - a);
                    Vec<T, N> o;
                    o.set(f);
                    to[l + i * L] = o;
                }
        }
        if constexpr(kRoom) {
#pragma unroll
            for(int i = 0; i < NV; i++) {
                vx[i] = nx[i];
                vy[i] = ny[i];
            }
            mu = nmu;
            rs = nrs;
        } else {
            fetch(r + step, vx, vy, mu, rs);
        }
    }
    if(!parts)
        return;
    float *pg = parts + (size_t)blockIdx.x * 2 * dim, *pb = pg + dim;
    if(R > 1) {  // the block's groups have the same columns: joined one after the other
        for(int w = 0; w < R; w++) {
            if(threadIdx.x / L == w)
#pragma unroll
                for(int i = 0; i < NV; i++)
                    if(l + i * L < vecs)
#pragma unroll
                        for(int j = 0; j < N; j++) {
                            float *g = joined + (i * L + l) * N + j, *b = g + L * NV * N;
                            *g = w ? *g + sg[i][j] : sg[i][j];
                            *b = w ? *b + sb[i][j] : sb[i][j];
                        }
            __syncthreads();
        }
        for(int d = threadIdx.x; d < (int)dim; d += THREADS) {
            pg[d] = joined[d];
            pb[d] = joined[L * NV * N + d];
        }
    } else {
#pragma unroll
        for(int i = 0; i < NV; i++)
            if(l + i * L < vecs)
#pragma unroll
                for(int j = 0; j < N; j++) {
                    pg[(l + i * L) * N + j] = sg[i][j];
                    pb[(l + i * L) * N + j] = sb[i][j];
                }
    }
}

// Joins the blocks' sums: 32 columns and 8 stretches of blocks a block.
template <typename P>
__global__ void __launch_bounds__(256)
    params_kernel(size_t dim, int blocks, const float *parts, P *dgamma, P *dbeta, int accumulate)
{
    lm_after_previous();
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const size_t d = (size_t)blockIdx.x * 32 + lane;
    P *to = blockIdx.y ? dbeta : dgamma;
    if(!to)
        return;
    float s = 0.0f;
    if(d < dim)
#pragma unroll 8
        for(int b = w; b < blocks; b += 8)
            s += parts[((size_t)b * 2 + blockIdx.y) * dim + d];
    red[w][lane] = s;
    __syncthreads();
    if(w || d >= dim)
        return;
    for(int i = 1; i < 8; i++)
        s += red[i][lane];
    lm_store(to + d, accumulate ? s + lm_load(to + d) : s);
}

// Rows too long for that: grad_x row by row, the parameters' sums column by column.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
    layernorm_bwd_long_kernel(size_t dim, const T *dy, size_t ys, const T *x, size_t xs,
                              const P *gamma, const float *mean, const float *rstd, T *dx, size_t dxs)
{
    __shared__ float red[32];
    const size_t r = blockIdx.x;
    const float mu = mean[r], rs = rstd[r];
    float a = 0.0f, b = 0.0f;
    for(size_t d = threadIdx.x; d < dim; d += 1024) {
        const float g = lm_load(dy + r * ys + d) * (gamma ? lm_load(gamma + d) : 1.0f);
        a += g;
        b += g * ((lm_load(x + r * xs + d) - mu) * rs);
    }
    a = block_sum(a, red) / (float)dim;
    b = block_sum(b, red) / (float)dim;
    for(size_t d = threadIdx.x; d < dim; d += 1024) {
        const float g = lm_load(dy + r * ys + d) * (gamma ? lm_load(gamma + d) : 1.0f);
        lm_store(dx + r * dxs + d, rs * (g - a - (lm_load(x + r * xs + d) - mu) * rs * b));
    }
}

template <typename T, typename P>
__global__ void __launch_bounds__(128)
    layernorm_params_long_kernel(size_t rows, size_t dim, const T *dy, size_t ys, const T *x, size_t xs,
                                 const float *mean, const float *rstd, float *parts)
{
    // blockIdx.y: a stretch of the rows
    const size_t d = (size_t)blockIdx.x * 128 + threadIdx.x;
    if(d >= dim)
        return;
    const size_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
    float g = 0.0f, b = 0.0f;
#pragma unroll 4
    for(size_t r = r0; r < r1; r++) {
        const float v = lm_load(dy + r * ys + d);
        g += v * ((lm_load(x + r * xs + d) - mean[r]) * rstd[r]);
        b += v;
    }
    parts[(size_t)blockIdx.y * 2 * dim + d] = g;
    parts[((size_t)blockIdx.y * 2 + 1) * dim + d] = b;
}

// ---------------------------------------------------------------- host side

struct Args {
    size_t rows, dim, xs, ys, dxs;
    const void *x, *dy, *gamma, *beta;
    float eps;
    void *y, *dx, *dgamma, *dbeta;
    float *mean, *rstd;
    const float *mean_in, *rstd_in;
    int accumulate;
    float *parts;
    cudaStream_t st;
};

// Calls f with the smallest number of vectors a thread, NV times a power of two up
// to MAX, with which WARPS warps hold a row.
template <int WARPS, int NV, int MAX, typename F>
bool pick(size_t vecs, F &&f)
{
    if(vecs <= (size_t)32 * WARPS * NV) {
        f(std::integral_constant<int, NV>(), std::integral_constant<int, WARPS>());
        return true;
    }
    if constexpr(2 * NV <= MAX) {
        return pick<WARPS, 2 * NV, MAX>(vecs, f);
    } else {
        return false;
    }
}

template <typename T, typename P, int N>
int fwd_with(const Args &a)
{
    auto launch = [&](auto nv, auto warps) {
        constexpr int NV = decltype(nv)::value, W = decltype(warps)::value;
        // several rows at a time where that leaves blocks enough
        constexpr int MANY = N == 1 || NV > 4 ? 1 : W > 1 || NV == 4 ? 2 : 4;
        auto go = [&](auto count) {
            constexpr int ROWS = decltype(count)::value;
            const size_t blocks = (a.rows + rows_of(W) * ROWS - 1) / (rows_of(W) * ROWS);
            layernorm_fwd_kernel<T, P, N, NV, W, ROWS><<<(unsigned)blocks, threads_of(W), 0, a.st>>>(
                a.rows, a.dim, (const T *)a.x, a.xs, (const P *)a.gamma, (const P *)a.beta, a.eps,
                (T *)a.y, a.ys, a.mean, a.rstd);
        };
        if(a.rows >= (size_t)592 * rows_of(W) * MANY)
            go(std::integral_constant<int, MANY>());
        else
            go(std::integral_constant<int, 1>());
    };
    const size_t vecs = a.dim / N;
    constexpr int MOST = N == 1 ? 16 : 4;
    if(!pick<1, 1, 4>(vecs, launch) && !pick<4, 2, MOST>(vecs, launch) &&
       !pick<8, MOST, MOST>(vecs, launch) && !pick<16, MOST, 16>(vecs, launch))
        layernorm_fwd_long_kernel<<<(unsigned)a.rows, 1024, 0, a.st>>>(
            a.dim, (const T *)a.x, a.xs, (const P *)a.gamma, (const P *)a.beta, a.eps, (T *)a.y, a.ys,
            a.mean, a.rstd);
    return lm_launched();
}

template <typename T, typename P, int N>
int bwd_with(const Args &a)
{
    const bool want = a.dgamma || a.dbeta;
    float *parts = want ? a.parts : nullptr;
    size_t blocks = 0;
    auto launch = [&](auto nv, auto warps) {
        constexpr int NV = decltype(nv)::value, W = decltype(warps)::value;
        constexpr int R = bwd_warps(W) / W;
        blocks = std::min<size_t>((a.rows + R - 1) / R, std::min(148 * bwd_blocks(N * NV, N == 8), kMaxParts));
        if(blocks)
            layernorm_bwd_kernel<T, P, N, NV, W><<<(unsigned)blocks, 32 * bwd_warps(W), 0, a.st>>>(
                a.rows, a.dim, (const T *)a.dy, a.ys, (const T *)a.x, a.xs, (const P *)a.gamma,
                a.mean_in, a.rstd_in, (T *)a.dx, a.dxs, parts);
    };
    const size_t vecs = a.dim / N;
    // few columns a thread as long as warps can be added, then more.  Two vectors in
    // fp16, where a row's fixed cost weighs more (16384 x 2048: 45 us, with one vector
    // 55; x 1024: 29 and 31), eight columns otherwise (fp32 x 1024: 39 us; a warp a
    // row with 32 columns 53).
    constexpr int FEW = N == 8 ? 2 : 8 / N, MOST = 32 / N;
    bool held = pick<1, 1, FEW>(vecs, launch) || pick<2, FEW, FEW>(vecs, launch) ||
                pick<4, FEW, FEW>(vecs, launch) || pick<8, FEW, MOST>(vecs, launch);
    if constexpr(N == 8)
        held = held || pick<16, 4, 4>(vecs, launch);
    if(!held) {
        if(a.dx && a.rows)
            layernorm_bwd_long_kernel<<<(unsigned)a.rows, 1024, 0, a.st>>>(
                a.dim, (const T *)a.dy, a.ys, (const T *)a.x, a.xs, (const P *)a.gamma, a.mean_in,
                a.rstd_in, (T *)a.dx, a.dxs);
        blocks = std::min<size_t>((a.rows + 63) / 64, kMaxParts);
        if(want && blocks)
            layernorm_params_long_kernel<T, P>
                <<<dim3((unsigned)((a.dim + 127) / 128), (unsigned)blocks), 128, 0, a.st>>>(
                    a.rows, a.dim, (const T *)a.dy, a.ys, (const T *)a.x, a.xs, a.mean_in, a.rstd_in,
                    parts);
    }
    const dim3 grid((unsigned)((a.dim + 31) / 32), 2);
    if(want && blocks)
        lm_launch_next(params_kernel<P>, grid, 256, 0, a.st, a.dim, (int)blocks, parts, (P *)a.dgamma,
                       (P *)a.dbeta, a.accumulate);
    else if(want)
        params_kernel<P><<<grid, 256, 0, a.st>>>(a.dim, 0, parts, (P *)a.dgamma, (P *)a.dbeta, a.accumulate);
    return lm_launched();
}

template <typename T, typename P>
int fwd(const Args &a)
{
    constexpr int N = 16 / sizeof(T);
    const bool v = lm_vectors(a.x, a.xs, sizeof(T), a.dim) && lm_vectors(a.y, a.ys, sizeof(T), a.dim) &&
                   lm_aligned(a.gamma, 16) && lm_aligned(a.beta, 16);
    return v ? fwd_with<T, P, N>(a) : fwd_with<T, P, 1>(a);
}

template <typename T, typename P>
int bwd(const Args &a)
{
    constexpr int N = 16 / sizeof(T);
    const bool v = lm_vectors(a.x, a.xs, sizeof(T), a.dim) && lm_vectors(a.dy, a.ys, sizeof(T), a.dim) &&
                   (!a.dx || lm_vectors(a.dx, a.dxs, sizeof(T), a.dim)) && lm_aligned(a.gamma, 16);
    return v ? bwd_with<T, P, N>(a) : bwd_with<T, P, 1>(a);
}

size_t bwd_bytes(size_t rows, size_t dim)
{
    return std::min<size_t>(rows, kMaxParts) * 2 * dim * 4;
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
    if(!rows || (!dim && !mean && !rstd))
        return B200OPT_OK;
    const size_t e = lm_size(dtype), p = lm_size(param_dtype);
    if(!lm_matrix(x, rows, dim, x_stride, e) || !lm_matrix(y, rows, dim, y_stride, e) ||
       !lm_aligned(gamma, p) || !lm_aligned(beta, p) || !lm_aligned(mean, 4) || !lm_aligned(rstd, 4))
        return B200OPT_EINVAL;
    Args a = {};
    a.rows = rows, a.dim = dim, a.x = x, a.xs = x_stride, a.gamma = gamma, a.beta = beta, a.eps = eps;
    a.y = y, a.ys = y_stride, a.mean = mean, a.rstd = rstd, a.st = (cudaStream_t)stream;
    return dtype == B200OPT_FLOAT         ? fwd<float, float>(a)
           : param_dtype == B200OPT_FLOAT ? fwd<__half, float>(a)
                                          : fwd<__half, __half>(a);
}

int b200opt_layernorm_bwd_workspace(size_t rows, size_t dim, size_t *bytes)
{
    if(!bytes)
        return B200OPT_EINVAL;
    if(rows > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    *bytes = bwd_bytes(rows, dim);
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
    Args a = {};
    a.rows = rows, a.dim = dim, a.x = x, a.xs = x_stride, a.gamma = gamma;
    a.dy = grad_y, a.ys = grad_y_stride, a.mean_in = mean, a.rstd_in = rstd;
    a.dx = grad_x, a.dxs = grad_x_stride, a.dgamma = grad_gamma, a.dbeta = grad_beta;
    a.accumulate = accumulate, a.parts = (float *)workspace, a.st = (cudaStream_t)stream;
    if(!grad_x && !grad_gamma && !grad_beta)
        return B200OPT_OK;
    return dtype == B200OPT_FLOAT         ? bwd<float, float>(a)
           : param_dtype == B200OPT_FLOAT ? bwd<__half, float>(a)
                                          : bwd<__half, __half>(a);
}

}  // extern "C"
