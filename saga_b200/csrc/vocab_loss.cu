// Softmax cross entropy over the vocabulary with the classifier's product, and
// its gradient (b200opt_vocab_loss_* of include/b200opt.h).
#include <algorithm>

#include "tc_gemm.cuh"

namespace b200 {
namespace {

constexpr size_t kPieceBytes = (size_t)256 << 20;  // of p - onehot held at a time
constexpr float kLift = 32768.0f;                  // 2^15: see the header
constexpr float kLog2e = 1.4426950408889634f;

// e^x, to 2^-22 of its size from ex2.approx and about 1.25 |x| 2^-24 from the product
// with log2 e, which is rounded to 32 bits: 2^-20 at x = -10, 2^-17.7 at -60, where the
// value itself is small beside the sum that it enters.  x is a difference from a row's
// maximum or lse, and the callers subtract first and in full: next to a probability of
// 1 what is lost in x is all that is left of the gradient.
__device__ __forceinline__ float exp_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
    return y;
}

// ------------------------------------------------------------------ forward

// What the exponentials of a stretch are taken from: its maximum, and 0 where that is
// infinite.  A stretch of -inf alone (a masked part of the vocabulary) then adds 0, where
// -inf - -inf would make the row NaN, and one with +inf adds +inf.
__device__ __forceinline__ float base_of(float top) { return fabsf(top) == INFINITY ? 0.0f : top; }

// Per row and tile of the vocabulary: the maximum of z and the sum of
// exp(z - base_of(maximum)), in one pass over the accumulator.  The target's logit goes to
// zt.
struct StatsEpilogue {
    int T, V;
    const void *y;
    int wide;
    float2 *part;
    float *zt;
    unsigned *done;  // of loss_kernel's blocks
    struct State {
        float top, sum;
        int at;
    };
    __device__ __forceinline__ int common() const
    {
        if(blockIdx.x == 0 && threadIdx.x == kTcThreads - 1)
            *done = 0;
        return 0;
    }
    __device__ __forceinline__ State begin(int, int row, int, int) const
    {
        return {-INFINITY, 0.0f, row < T ? lm_index_at(y, wide, row, V) : -1};
    }
    __device__ __forceinline__ void columns(int, State &s, int row, int col, float (&v)[32], char *) const
    {
        if(col >= V)
            return;
        const int at = s.at - col;
        if(at >= 0 && at < 32) {
            float z = v[0];
#pragma unroll
            for(int j = 1; j < 32; j++)
                z = at == j ? v[j] : z;
            zt[row] = z;
        }
        if(V - col < 32) {
#pragma unroll
            for(int j = 0; j < 32; j++)
                v[j] = j < V - col ? v[j] : -INFINITY;
        }
        float most[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for(int j = 4; j < 32; j++)
            most[j & 3] = fmaxf(most[j & 3], v[j]);
        const float top = fmaxf(s.top, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
        const float base = base_of(top);
        float sum[4] = {s.sum * exp_fast(s.top - base), 0.0f, 0.0f, 0.0f};
#pragma unroll
        for(int j = 0; j < 32; j++)
            sum[j & 3] += exp_fast(v[j] - base);
        s.top = top;
        s.sum = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    // The four warps that share 32 rows meet; two sets of slots, one for each
    // accumulator, keep a tile's from the next one's.
    __device__ __forceinline__ void end(const State &s, int row, int col, int acc, char *shared) const
    {
        const int quad = (threadIdx.x >> 5) & 3, side = ((threadIdx.x >> 5) - 4) >> 2;
        float2 *slots = reinterpret_cast<float2 *>(shared) + acc * 512 + quad * 32 + (threadIdx.x & 31);
        slots[side * 128] = make_float2(s.top, s.sum);
        asm volatile("bar.sync %0, 128;" ::"r"(1 + quad) : "memory");
        if(side || row >= T)
            return;
        float top = s.top, sum = 0.0f;
#pragma unroll
        for(int i = 1; i < 4; i++)
            top = fmaxf(top, slots[i * 128].x);
        const float base = base_of(top);
#pragma unroll
        for(int i = 0; i < 4; i++)  // a side beyond the vocabulary has -inf and 0
            sum += slots[i * 128].y * exp_fast(slots[i * 128].x - base);
        part[(size_t)(col / kTcTile) * T + row] = make_float2(top, sum);
    }
};

// Joins the parts of kLossRows rows, 64 threads a row.  The block that finishes
// last adds up the blocks' sums of losses, in their order.
constexpr int kLossRows = 8;
__global__ void __launch_bounds__(512)
    loss_kernel(int T, int V, int parts, const float2 *part, const float *zt, const void *y, int wide,
                float *loss, float *lse, float2 *block_sums, unsigned *done, float *stats)
{
    __shared__ float2 red[64][kLossRows];
    __shared__ bool last;
    lm_after_previous();
    const int x = threadIdx.x % kLossRows, w = threadIdx.x / kLossRows;
    const int t = blockIdx.x * kLossRows + x;
    auto add = [](float2 a, float2 b) {  // two (maximum, sum) of disjoint stretches
        const float m = fmaxf(a.x, b.x), base = base_of(m);
        return make_float2(m, a.y * exp_fast(a.x - base) + b.y * exp_fast(b.x - base));
    };
    // asked for now, used at the end
    const bool valid = t < T && lm_index_at(y, wide, t, V) >= 0;
    const float target = t < T ? zt[t] : 0.0f;
    float2 mine = make_float2(-INFINITY, 0.0f);
    if(t < T)
#pragma unroll 4
        for(int i = w; i < parts; i += 64)
            mine = add(mine, part[(size_t)i * T + t]);
    red[w][x] = mine;
    __syncthreads();
    if(threadIdx.x < 32) {  // four threads a row, then one
        float top = mine.x, sum = 0.0f;
#pragma unroll
        for(int i = 1; i < 16; i++)
            top = fmaxf(top, red[w + 4 * i][x].x);
        const float base = base_of(top);
#pragma unroll
        for(int i = 0; i < 16; i++) {
            const float2 p = red[w + 4 * i][x];
            sum += p.y * exp_fast(p.x - base);
        }
        mine = make_float2(top, sum);
#pragma unroll
        for(int o = 16; o >= kLossRows; o >>= 1)
            mine = add(mine, make_float2(__shfl_xor_sync(0xffffffffu, mine.x, o),
                                         __shfl_xor_sync(0xffffffffu, mine.y, o)));
        float own = 0.0f, counted = 0.0f;
        if(t < T && w == 0) {
            const float l = logf(mine.y);
            lse[t] = mine.x + l;
            if(valid) {
                // not from lse: its rounding, at a large logit, would be all of a small loss
                own = (mine.x - target) + l;
                counted = 1.0f;
            }
            loss[t] = own;
        }
        own = warp_sum(own);
        counted = warp_sum(counted);
        if(threadIdx.x == 0 && stats) {
            block_sums[blockIdx.x] = make_float2(own, counted);
            __threadfence();
            last = atomicAdd(done, 1) == gridDim.x - 1;
        }
    }
    if(!stats)
        return;
    __syncthreads();
    if(!last)
        return;
    __threadfence();
    float sum = 0.0f;
    int counted = 0;
    for(int i = threadIdx.x; i < (int)gridDim.x; i += 512) {
        const float2 p = __ldcg(block_sums + i);
        sum += p.x;
        counted += (int)p.y;
    }
    sum = warp_sum(sum);
    counted = __reduce_add_sync(0xffffffffu, counted);
    if((threadIdx.x & 31) == 0)
        red[threadIdx.x >> 5][0] = make_float2(sum, __int_as_float(counted));
    __syncthreads();
    if(threadIdx.x == 0) {
        for(int i = 1; i < 16; i++) {
            sum += red[i][0].x;
            counted += __float_as_int(red[i][0].y);
        }
        stats[0] = sum;
        stats[1] = (float)counted;
    }
}

__global__ void no_stats_kernel(float *stats) { stats[0] = stats[1] = 0.0f; }

// ----------------------------------------------------------------- gradient

// The tokens that are not ignored, moved together in their order: their rows of
// `hidden`, their lse and target, and where they came from.  Ignored tokens then
// cost nothing in the three products, and what stands in their rows (NaN too)
// cannot reach the gradient; their rows of grad_hidden are written as zeros
// here.  Behind the last row, zeros up to the next stage of k.
__global__ void __launch_bounds__(256)
    compact_kernel(int T, int V, int D, int rows_per_block, const __half *x, size_t xs, const void *y,
                   int wide, const float *lse, __half *xc, float *lsec, int *targetc, int *from,
                   int *count, __half *dx, size_t dxs)
{
    __shared__ int before_sum, all_sum, place[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = blockIdx.x * rows_per_block;
    lm_let_next();
    if(tid == 0)
        before_sum = all_sum = 0;
    __syncthreads();
    int before = 0, all = 0;
    for(int t = tid; t < T; t += 256) {
        const int ok = lm_index_at(y, wide, t, V) >= 0;
        all += ok;
        before += t < r0 && ok;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    if(lane == 0) {
        atomicAdd(&before_sum, before);  // whole numbers: any order gives the same
        atomicAdd(&all_sum, all);
    }
    __syncthreads();
    int next = before_sum;
    const int total = all_sum, vecs = D / 8;
    if(blockIdx.x == 0 && tid == 0)
        *count = total;
    const int r1 = min(r0 + rows_per_block, T);
    for(int r = r0; r < r1; r += 32) {
        if(warp == 0) {
            const int t = r + lane, id = t < r1 ? lm_index_at(y, wide, t, V) : -1;
            const unsigned mask = __ballot_sync(0xffffffffu, id >= 0);
            const int at = next + __popc(mask & ((1u << lane) - 1));
            place[lane] = id >= 0 ? at : -1;
            if(id >= 0) {
                lsec[at] = lse[t];
                targetc[at] = id;
                from[at] = t;
            }
        }
        __syncthreads();
        int seen = 0;
        for(int j = 0; j < 32; j++)
            seen += place[j] >= 0;
        for(int j = warp; j < 32; j += 8) {
            const int t = r + j, at = place[j];
            if(t >= r1)
                continue;
            if(at >= 0) {
                const uint4 *s = reinterpret_cast<const uint4 *>(x + (size_t)t * xs);
                uint4 *d = reinterpret_cast<uint4 *>(xc + (size_t)at * D);
                for(int c = lane; c < vecs; c += 32)
                    d[c] = s[c];
            } else if(dx) {
                uint4 *d = reinterpret_cast<uint4 *>(dx + (size_t)t * dxs);
                for(int c = lane; c < vecs; c += 32)
                    d[c] = make_uint4(0, 0, 0, 0);
            }
        }
        next += seen;
        __syncthreads();
    }
    // grad_weight's product runs over whole stages of tokens
    const int pad = max((total + kTcK - 1) / kTcK, 1) * kTcK;
    for(int r = total + blockIdx.x * 8 + warp; r < pad; r += gridDim.x * 8) {
        uint4 *d = reinterpret_cast<uint4 *>(xc + (size_t)r * D);
        for(int c = lane; c < vecs; c += 32)
            d[c] = make_uint4(0, 0, 0, 0);
    }
}

// dz[row][v - first] = 2^15 (p - onehot) in fp16; rows behind the last token are zero.
// The rounding to fp16 is the price of the tensor cores for both gradients' products:
// with few tokens it can be seen beside the results' own rounding (64 x 1000 x 256: the
// gradients are 2.6e-4 off, relative, where rounding exact ones would give 2.1e-4), with
// a thousand it averages out (1001 x 50021 x 1032: 2.1e-4 both).  Two fp16 parts would
// keep the rest, at twice the arithmetic of both products.
struct DzEpilogue {
    const int *count;
    const float *lse;
    const int *target;
    int first;
    __half *dz;
    size_t stride;  // a multiple of 256: whole tiles may be written
    struct State {
        float lse;
        int at;
        bool live;
    };
    __device__ __forceinline__ int common() const { return *count; }
    __device__ __forceinline__ State begin(int tokens, int row, int, int) const
    {
        const bool live = row < tokens;
        return {live ? lse[row] : 0.0f, live ? target[row] - first : -1, live};
    }
    __device__ __forceinline__ void columns(int, State &s, int row, int col, float (&v)[32], char *buf) const
    {
        if((size_t)col >= stride)
            return;
        const int at = s.at - col;
#pragma unroll
        for(int j = 0; j < 32; j++)
            v[j] = s.live ? exp_fast(v[j] - s.lse) * kLift : 0.0f;
        if(at >= 0 && at < 32) {
#pragma unroll
            for(int j = 0; j < 32; j++)
                v[j] -= at == j ? kLift : 0.0f;
        }
        const Turn<4> turn = {buf, (int)(threadIdx.x & 31)};
        __syncwarp();
#pragma unroll
        for(int w = 0; w < 4; w++) {
            uint4 bits;
            __half2 *h = reinterpret_cast<__half2 *>(&bits);
#pragma unroll
            for(int i = 0; i < 4; i++)
                h[i] = __floats2half2_rn(v[8 * w + 2 * i], v[8 * w + 2 * i + 1]);
            turn.put(w, bits);
        }
        __syncwarp();
        __half *to = dz + (size_t)(row - turn.lane) * stride + col + turn.word() * 8;
#pragma unroll
        for(int i = 0; i < turn.kSteps; i++)
            *reinterpret_cast<uint4 *>(to + turn.row(i) * stride) = turn.get(i);
    }
    __device__ __forceinline__ void end(const State &, int, int, int, char *) const {}
};

struct Factor {
    float scale;
    const float *loss_scale, *stats;
    // of the sums of 2^15 (p - onehot)
    __device__ __forceinline__ float get() const
    {
        const float f = loss_scale ? scale * *loss_scale : scale;
        return (stats ? f / fmaxf(stats[1], 1.0f) : f) * (1.0f / kLift);
    }
};

// What a product's result does, MODE:
enum {
    kOut,         // out = factor * acc
    kAccumulate,  // out += factor * acc
    kSums,        // sum[part] = acc, or += acc when it holds earlier pieces
    kLast         // out = factor * (sum + acc): the last piece
};
template <int MODE>
struct OutEpilogue {
    int m;
    const int *count;  // replaces m
    int n;
    float *sum;        // fp32, row stride n, a matrix of the product's rows per part
    int add;           // sum holds earlier pieces
    __half *out;
    size_t stride;
    const int *rows;   // where a row of the result goes; null: its own place
    Factor factor;
    struct Common {
        int live;
        float f;
    };
    struct State {
        int to;         // row of the result; -1: none
        float *sums;    // of this warp's first row and part
        __half *at[4];  // where this thread writes in the four steps of a turn; null: nowhere
    };
    __device__ __forceinline__ Common common() const
    {
        return {count ? *count : m, MODE == kSums ? 0.0f : factor.get()};
    }
    __device__ __forceinline__ State begin(const Common &g, int row, int, int part) const
    {
        State s;
        const int lane = threadIdx.x & 31;
        s.to = row < g.live ? (MODE != kSums && rows ? rows[row] : row) : -1;
        if(MODE == kSums || MODE == kLast)
            s.sums = sum + ((size_t)part * g.live + (row - lane)) * n;
        if(MODE != kSums) {
            const Turn<4> turn = {nullptr, lane};
#pragma unroll
            for(int i = 0; i < 4; i++) {
                const int to = __shfl_sync(0xffffffffu, s.to, turn.row(i));
                s.at[i] = to >= 0 ? out + (size_t)to * stride + turn.word() * 8 : nullptr;
            }
        }
        return s;
    }
    __device__ __forceinline__ void columns(const Common &g, State &s, int, int col, float (&v)[32], char *buf) const
    {
        const int lane = threadIdx.x & 31;
        if(col >= n)
            return;
        if(MODE == kSums || MODE == kLast) {
            const Turn<8> turn = {buf, lane};
            const int c = col + turn.word() * 4;
            __syncwarp();
            if(MODE == kLast || add) {
#pragma unroll
                for(int i = 0; i < turn.kSteps; i++) {
                    const int to = __shfl_sync(0xffffffffu, s.to, turn.row(i));
                    if(to >= 0 && c < n)
                        *turn.at(turn.row(i), turn.word()) =
                            *reinterpret_cast<const uint4 *>(s.sums + (size_t)turn.row(i) * n + c);
                }
                __syncwarp();
#pragma unroll
                for(int w = 0; w < 8; w++) {
                    const float4 a = *reinterpret_cast<const float4 *>(turn.at(lane, w));
                    v[4 * w] += a.x, v[4 * w + 1] += a.y, v[4 * w + 2] += a.z, v[4 * w + 3] += a.w;
                }
                __syncwarp();
            }
            if(MODE == kSums) {
#pragma unroll
                for(int w = 0; w < 8; w++)
                    turn.put(w, make_uint4(__float_as_uint(v[4 * w]), __float_as_uint(v[4 * w + 1]),
                                           __float_as_uint(v[4 * w + 2]), __float_as_uint(v[4 * w + 3])));
                __syncwarp();
#pragma unroll
                for(int i = 0; i < turn.kSteps; i++) {
                    const int to = __shfl_sync(0xffffffffu, s.to, turn.row(i));
                    if(to >= 0 && c < n)
                        *reinterpret_cast<uint4 *>(s.sums + (size_t)turn.row(i) * n + c) = turn.get(i);
                }
            }
        }
        if(MODE == kSums)
            return;
        const Turn<4> turn = {buf, lane};
        const bool inside = col + turn.word() * 8 < n;  // n is a multiple of 8
        __syncwarp();
        if(MODE == kAccumulate) {
#pragma unroll
            for(int i = 0; i < 4; i++)
                if(s.at[i] && inside)
                    *turn.at(turn.row(i), turn.word()) = *reinterpret_cast<const uint4 *>(s.at[i] + col);
            __syncwarp();
        }
#pragma unroll
        for(int w = 0; w < 4; w++) {
            uint4 bits = MODE == kAccumulate ? *turn.at(lane, w) : make_uint4(0, 0, 0, 0);
            __half2 *h = reinterpret_cast<__half2 *>(&bits);
#pragma unroll
            for(int i = 0; i < 4; i++) {
                float a = g.f * v[8 * w + 2 * i], b = g.f * v[8 * w + 2 * i + 1];
                if(MODE == kAccumulate) {
                    const float2 old = __half22float2(h[i]);
                    a += old.x, b += old.y;
                }
                h[i] = __floats2half2_rn(a, b);
            }
            turn.put(w, bits);
        }
        __syncwarp();
#pragma unroll
        for(int i = 0; i < 4; i++)
            if(s.at[i] && inside)
                *reinterpret_cast<uint4 *>(s.at[i] + col) = turn.get(i);
    }
    __device__ __forceinline__ void end(const State &, int, int, int, char *) const {}
};

// A product into its result; false when it could not be launched.
template <bool A_MN, bool B_MN, int NH, int MODE>
bool product(const CUtensorMap &a, const CUtensorMap &b, const TcShape &s, int m, const int *count, int n,
             float *sum, int add, __half *out, size_t stride, const int *rows,
             const Factor &factor, int sms, cudaStream_t st)
{
    const OutEpilogue<MODE> e = {m, count, n, sum, add, out, stride, rows, factor};
    return tc_launch<A_MN, B_MN, NH>(a, b, s, e, sms, st, true);
}

// Joins the parts of a product that was cut along k, in their order.
__global__ void __launch_bounds__(256)
    join_kernel(TcShape shape, const int *count, int n, const float *sum, __half *out, size_t stride,
                const int *rows, int accumulate, Factor factor)
{
    lm_after_previous();
    const int live = count ? *count : shape.m, vecs = n / 8;
    const int parts = (int)tc_parts_of(shape, max(live, 1));
    const size_t part_stride = (size_t)live * n;
    const float f = factor.get();
    const long long total = (long long)live * vecs;
    for(long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total;
        i += (long long)gridDim.x * 256) {
        const int r = (int)(i / vecs), c = (int)(i % vecs) * 8;
        float v[8] = {};
        for(int p = 0; p < parts; p++) {
            const float4 *s = reinterpret_cast<const float4 *>(sum + p * part_stride + (size_t)r * n + c);
            const float4 a = s[0], b = s[1];
            v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
            v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
        }
        uint4 *to = reinterpret_cast<uint4 *>(out + (size_t)(rows ? rows[r] : r) * stride + c);
        uint4 bits = accumulate ? *to : make_uint4(0, 0, 0, 0);
        __half2 *h = reinterpret_cast<__half2 *>(&bits);
#pragma unroll
        for(int j = 0; j < 4; j++) {
            const float2 old = __half22float2(h[j]);
            float a = f * v[2 * j], b = f * v[2 * j + 1];
            if(accumulate)
                a += old.x, b += old.y;
            h[j] = __floats2half2_rn(a, b);
        }
        *to = bits;
    }
}

// ------------------------------------------------------------------ planning

size_t tiles_of(size_t n) { return (n + kTcTile - 1) / kTcTile; }

size_t parts_of(size_t m, size_t n, size_t k)
{
    const size_t tiles = tiles_of(m) * tiles_of(n);
    return tiles > kTcPlanPairs ? 1 : tc_parts((uint32_t)tiles, (uint32_t)((k + kTcK - 1) / kTcK));
}

struct Plan {
    size_t piece;                    // columns of the vocabulary at a time, a multiple of 256
    size_t x_parts, w_parts;         // parts of the two gradients' products
    size_t x_sum, w_sum;             // bytes of their fp32 sums
    size_t at_x, at_dz, at_lse, at_target, at_from, at_count, at_xsum, at_wsum, bytes;
    Plan(size_t T, size_t V, size_t D)
    {
        T = std::max<size_t>(T, 1);
        const size_t rows = lm_up(T, kTcTile);
        const size_t most = std::max<size_t>(kPieceBytes / 2 / rows / kTcTile * kTcTile, kTcTile);
        piece = std::min(lm_up(V, kTcTile), most);
        const bool whole = piece >= V;
        x_parts = parts_of(T, D, std::min(piece, V));
        w_parts = parts_of(std::min(piece, V), D, T);
        x_sum = x_parts > 1 || !whole ? x_parts * T * D * 4 : 0;
        w_sum = w_parts > 1 ? w_parts * std::min(piece, V) * D * 4 : 0;
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t here = at;
            at += lm_up(n, 256);
            return here;
        };
        at_x = take(rows * D * 2);
        at_dz = take(rows * piece * 2);
        at_lse = take(rows * 4);
        at_target = take(rows * 4);
        at_from = take(rows * 4);
        at_count = take(4);
        at_xsum = take(x_sum);
        at_wsum = take(w_sum);
        bytes = at;
    }
};

bool lm_head(size_t T, size_t V, size_t D, const void *x, size_t xs, const void *w, size_t ws,
             const void *y, int index_bytes)
{
    return D % 8 == 0 && xs % 8 == 0 && ws % 8 == 0 && lm_aligned(x, 16) && lm_aligned(w, 16) &&
           lm_matrix(x, T, D, xs, 2) && lm_matrix(w, V, D, ws, 2) && (!T || y) &&
           lm_aligned(y, index_bytes);
}

int head_sizes(size_t T, size_t V, size_t D)
{
    if(!V || !D)
        return B200OPT_EINVAL;
    if(T > B200OPT_LM_MAX || V > B200OPT_LM_MAX || D > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    // the tiles of a product are counted in 31 bits
    const size_t most = std::max(T, std::max(V, D)), rest = std::max(std::min(std::max(T, V), D), std::min(T, V));
    return tiles_of(most) * tiles_of(rest) > 0x7fffffff ? B200OPT_ETOOBIG : B200OPT_OK;
}

// The forward pass's workspace: target logits, blocks' sums, their count, parts.
struct FwdPlan {
    size_t at_sums, at_done, at_part, bytes;
    FwdPlan(size_t T, size_t V)
    {
        at_sums = lm_up(T * 4, 256);
        at_done = at_sums + lm_up((T + kLossRows - 1) / kLossRows * 8, 256);
        at_part = at_done + 256;
        bytes = at_part + tiles_of(V) * T * 8;
    }
};

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200opt_vocab_loss_fwd_workspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes)
{
    if(!bytes)
        return B200OPT_EINVAL;
    if(const int rc = head_sizes(tokens, vocab, dim))
        return rc;
    *bytes = tokens ? FwdPlan(tokens, vocab).bytes : 0;
    return B200OPT_OK;
}

int b200opt_vocab_loss_fwd(size_t tokens, size_t vocab, size_t dim, const void *hidden,
                           size_t hidden_stride, const void *weight, size_t weight_stride,
                           const void *targets, int index_bytes, float *loss, float *lse,
                           float *stats, void *workspace, size_t workspace_bytes, void *stream)
{
    if(const int rc = head_sizes(tokens, vocab, dim))
        return rc;
    const FwdPlan p(tokens, vocab);
    const size_t need = tokens ? p.bytes : 0;
    if(!lm_index(index_bytes) ||
       !lm_head(tokens, vocab, dim, hidden, hidden_stride, weight, weight_stride, targets, index_bytes) ||
       (tokens && (!loss || !lse)) || !lm_aligned(loss, 4) || !lm_aligned(lse, 4) ||
       !lm_aligned(stats, 4) || workspace_bytes < need ||
       (need && (!workspace || !lm_aligned(workspace, 256))))
        return B200OPT_EINVAL;
    cudaStream_t st = (cudaStream_t)stream;
    const int wide = index_bytes == 8, T = (int)tokens, V = (int)vocab;
    if(!tokens && !stats)
        return B200OPT_OK;
    if(tokens) {
        char *ws = (char *)workspace;
        float *zt = (float *)ws;
        unsigned *done = (unsigned *)(ws + p.at_done);
        float2 *part = (float2 *)(ws + p.at_part);
        int sms = 0;
        CUtensorMap mx, mw;
        if(!lm_sms(&sms) || !tc_map(&mx, hidden, tokens, dim, hidden_stride, tc_box(false)) ||
           !tc_map(&mw, weight, vocab, dim, weight_stride, tc_box(false)))
            return B200OPT_ECUDA;
        TcShape s = {T, V, (int)dim, nullptr, 0, 0, 0, 0, 1, 16};
        if(!tc_launch<false, false, 1>(mx, mw, s, StatsEpilogue{T, V, targets, wide, part, zt, done}, sms, st,
                                        false))
            return B200OPT_ECUDA;
        lm_launch_next(loss_kernel, (unsigned)((tokens + kLossRows - 1) / kLossRows), 512, 0, st, T, V,
                       (int)tiles_of(vocab), part, zt, targets, wide, loss, lse, (float2 *)(ws + p.at_sums),
                       done, stats);
    } else {
        no_stats_kernel<<<1, 1, 0, st>>>(stats);
    }
    return lm_launched();
}

int b200opt_vocab_loss_bwd_workspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes)
{
    if(!bytes)
        return B200OPT_EINVAL;
    if(const int rc = head_sizes(tokens, vocab, dim))
        return rc;
    *bytes = tokens ? Plan(tokens, vocab, dim).bytes : 0;
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
    if(const int rc = head_sizes(tokens, vocab, dim))
        return rc;
    const Plan p(tokens, vocab, dim);
    const size_t need = tokens ? p.bytes : 0;
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
    if(!tokens) {
        if(grad_weight && !accumulate &&
           cudaMemset2DAsync(grad_weight, grad_weight_stride * 2, 0, dim * 2, vocab, st) != cudaSuccess)
            return B200OPT_ECUDA;
        return B200OPT_OK;
    }
    if(!grad_hidden && !grad_weight)
        return B200OPT_OK;
    int sms = 0;
    if(!lm_sms(&sms))
        return B200OPT_ECUDA;
    const int wide = index_bytes == 8, T = (int)tokens, V = (int)vocab, D = (int)dim;
    char *ws = (char *)workspace;
    __half *xc = (__half *)(ws + p.at_x), *dz = (__half *)(ws + p.at_dz);
    float *lsec = (float *)(ws + p.at_lse);
    int *target = (int *)(ws + p.at_target), *from = (int *)(ws + p.at_from);
    int *count = (int *)(ws + p.at_count);
    float *xsum = p.x_sum ? (float *)(ws + p.at_xsum) : nullptr;
    float *wsum = p.w_sum ? (float *)(ws + p.at_wsum) : nullptr;
    const size_t rows = lm_up(tokens, kTcTile);
    const Factor factor = {grad_scale, loss_scale, stats};

    const int per = (int)lm_up((tokens + 4 * sms - 1) / (4 * sms), 8);  // a row a warp, at least
    compact_kernel<<<(T + per - 1) / per, 256, 0, st>>>(
        T, V, D, per, (const __half *)hidden, hidden_stride, targets, wide, lse, xc, lsec, target, from,
        count, (__half *)grad_hidden, grad_hidden_stride);

    CUtensorMap x_k, x_mn, w_k, w_mn;
    if(!tc_map(&x_k, xc, rows, dim, dim, tc_box(false)) || !tc_map(&x_mn, xc, rows, dim, dim, tc_box(true)) ||
       !tc_map(&w_k, weight, vocab, dim, weight_stride, tc_box(false)) ||
       !tc_map(&w_mn, weight, vocab, dim, weight_stride, tc_box(true)))
        return B200OPT_ECUDA;
    for(size_t first = 0; first < vocab; first += p.piece) {
        const size_t n = std::min(p.piece, vocab - first);
        const int N = (int)n, at = (int)first;
        const bool begin = first == 0, last = first + n == vocab;
        CUtensorMap dz_k, dz_mn;
        if(!tc_map(&dz_k, dz, rows, n, p.piece, tc_box(false)) ||
           !tc_map(&dz_mn, dz, rows, n, p.piece, tc_box(true)))
            return B200OPT_ECUDA;
        // dz = p - onehot
        TcShape s = {T, N, D, count, 1, 0, 0, at, 1, 16};
        if(!tc_launch<false, false, 1>(x_k, w_k, s, DzEpilogue{count, lsec, target, at, dz, p.piece}, sms, st,
                                        true))
            return B200OPT_ECUDA;
        if(grad_hidden) {  // += dz W
            const bool direct = p.x_parts == 1 && last;
            s = {T, D, N, count, 1, 0, 0, at, (int)p.x_parts, 8, (int)(p.x_parts * tokens),
                 (int)((std::min(p.piece, vocab) + kTcK - 1) / kTcK)};
            auto *run = !direct ? product<false, true, 1, kSums>
                        : begin ? product<false, true, 1, kOut>
                                : product<false, true, 1, kLast>;
            if(!run(dz_k, w_mn, s, T, count, D, xsum, !begin, (__half *)grad_hidden,
                    grad_hidden_stride, from, factor, sms, st))
                return B200OPT_ECUDA;
            if(last && !direct)
                lm_launch_next(join_kernel, sms * 4, 256, 0, st, s, count, D, xsum, (__half *)grad_hidden,
                               grad_hidden_stride, from, 0, factor);
        }
        if(grad_weight) {  // = dz^T X
            __half *to = (__half *)grad_weight + first * grad_weight_stride;
            s = {N, D, T, count, 0, 1, 0, 0, (int)p.w_parts, 8};
            // (by all tokens: how many are ignored is known on the device alone)
            const bool wide_tiles = tc_wide(N, D, T, sms);
            auto *run = p.w_parts > 1 ? product<true, true, 1, kSums>
                        : accumulate  ? (wide_tiles ? product<true, true, 2, kAccumulate>
                                                    : product<true, true, 1, kAccumulate>)
                                      : (wide_tiles ? product<true, true, 2, kOut>
                                                    : product<true, true, 1, kOut>);
            if(!run(dz_mn, x_mn, s, N, nullptr, D, wsum, 0, to, grad_weight_stride, nullptr,
                    factor, sms, st))
                return B200OPT_ECUDA;
            if(p.w_parts > 1)
                lm_launch_next(join_kernel, sms * 4, 256, 0, st, s, nullptr, D, wsum, to, grad_weight_stride,
                               nullptr, accumulate, factor);
        }
    }
    return lm_launched();
}

}  // extern "C"
