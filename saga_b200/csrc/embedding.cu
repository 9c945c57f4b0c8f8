// Embedding lookup and its gradient (b200opt_embedding_* of include/b200opt.h).
//
// Both are bound by memory: the lookup reads and writes `tokens` rows, the
// gradient reads `tokens` rows and writes the whole table.  Rows are moved in
// 16-byte vectors where addresses and strides allow it, else element by element.
#include <algorithm>

#include "lm_common.cuh"

namespace b200 {
namespace {

// ------------------------------------------------------------------- lookup

// `lanes` threads (a power of two) share a row, four vectors each where the row
// is that long, so that the loads behind an id are in flight together.
template <typename T, int N>
__global__ void __launch_bounds__(256)
    embedding_fwd_kernel(size_t tokens, size_t vocab, size_t vecs, int lanes, const void *ids,
                         int wide, const T *weight, size_t ws, float scale, T *out, size_t os)
{
    const int lane = threadIdx.x & (lanes - 1);
    const size_t groups = (size_t)gridDim.x * (256 / lanes);
    for(size_t t = (size_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes; t < tokens; t += groups) {
        const int id = lm_index_at(ids, wide, t, vocab);
        const Vec<T, N> *from = reinterpret_cast<const Vec<T, N> *>(weight + (id < 0 ? 0 : id) * ws);
        Vec<T, N> *to = reinterpret_cast<Vec<T, N> *>(out + t * os);
        for(size_t c0 = lane; c0 < vecs; c0 += 4 * (size_t)lanes) {
            Vec<T, N> v[4];
#pragma unroll
            for(int j = 0; j < 4; j++)
                if(id >= 0 && c0 + j * lanes < vecs)
                    v[j] = from[c0 + j * lanes];
#pragma unroll
            for(int j = 0; j < 4; j++) {
                if(c0 + j * lanes >= vecs)
                    break;
                float f[N];
                if(id >= 0)
                    v[j].get(f);
#pragma unroll
                for(int i = 0; i < N; i++)
                    f[i] = id >= 0 ? scale * f[i] : 0.0f;
                v[j].set(f);
                to[c0 + j * lanes] = v[j];
            }
        }
    }
}

// --------------------------------------------------------- order of the tokens
//
// The gradient of a row is the sum over the row's tokens, in ascending token
// order.  The tokens are brought into that order by a stable radix sort of
// (id, token), least digit first; ids outside the table get the key `vocab` and
// end up last.  A warp ranks 32 keys at a time with one match over their digits;
// a table of counts per warp and digit gives the places.

constexpr int kDigits = 512;      // nine bits a pass: two passes up to 2^18 rows
constexpr int kSortItems = 16;    // keys a thread holds
constexpr int kOneBlock = 1024 * kSortItems;  // tokens that one block sorts by itself
constexpr int kManyThreads = 512;
constexpr int kManyItems = kManyThreads * kSortItems;

__device__ __forceinline__ uint32_t key_of(const void *ids, int wide, size_t t, size_t vocab)
{
    const int id = lm_index_at(ids, wide, t, vocab);
    return id < 0 ? (uint32_t)vocab : (uint32_t)id;
}

// Ranks this warp's keys (items i * 32 + lane, i < trips) among its earlier keys
// of the same digit; count[digit] (this warp's, zeroed) ends as the number of
// keys.  The lanes with the same digit are found by one ballot per bit of it.
__device__ __forceinline__ void warp_rank(const uint32_t (&key)[kSortItems], int shift, int bits,
                                          int trips, unsigned live, uint16_t *count,
                                          uint16_t (&rank)[kSortItems])
{
    const int lane = threadIdx.x & 31;
    const uint32_t mask = (1u << bits) - 1;
#pragma unroll
    for(int i = 0; i < kSortItems; i++) {
        if(i >= trips)
            break;
        const bool here = live >> i & 1;
        const uint32_t d = here ? (key[i] >> shift) & mask : 0;
        unsigned same = __ballot_sync(0xffffffffu, here);
        for(int b = 0; b < bits; b++) {
            const unsigned set = __ballot_sync(0xffffffffu, d >> b & 1);
            same &= d >> b & 1 ? set : ~set;
        }
        const int before = __popc(same & ((1u << lane) - 1));
        if(here)
            rank[i] = count[d] + before;
        __syncwarp();
        if(here && before == 0)
            count[d] += __popc(same);
        __syncwarp();
    }
}

// One block sorts up to kOneBlock tokens in shared memory.
__device__ void sort_one_block(int tokens, size_t vocab, int bits, const void *ids, int wide,
                               char *smem, uint32_t *keys_out, int *order_out)
{
    uint32_t *keys = reinterpret_cast<uint32_t *>(smem);
    uint16_t *order = reinterpret_cast<uint16_t *>(smem + kOneBlock * 4);
    uint16_t *count = reinterpret_cast<uint16_t *>(smem + kOneBlock * 6);  // [32 warps][kDigits]
    int *total = reinterpret_cast<int *>(smem + kOneBlock * 6 + 32 * kDigits * 2);  // [kDigits]
    __shared__ int warp_total[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int trips = (tokens + 1023) / 1024;
    const int first = warp * trips * 32 + lane;  // of this thread's keys
    unsigned live = 0;
    uint32_t key[kSortItems];
    uint16_t item[kSortItems], rank[kSortItems];
#pragma unroll
    for(int i = 0; i < kSortItems; i++) {
        const int t = first + 32 * i;
        if(i < trips && t < tokens) {
            live |= 1u << i;
            key[i] = key_of(ids, wide, t, vocab);
            item[i] = (uint16_t)t;
        }
    }
    const int passes = (bits + 8) / 9, step = (bits + passes - 1) / passes;
    for(int p = 0; p < passes; p++) {
        const int shift = p * step;
        const uint32_t mask = (1u << step) - 1;
        for(int i = tid; i < 32 * kDigits / 2; i += 1024)
            reinterpret_cast<uint32_t *>(count)[i] = 0;
        __syncthreads();
        warp_rank(key, shift, step, trips, live, count + warp * kDigits, rank);
        __syncthreads();
        // exclusive sums: digit by digit, within a digit warp by warp
        int sum = 0;
        if(tid < kDigits) {
            int c[32];
#pragma unroll
            for(int w = 0; w < 32; w++)
                c[w] = count[w * kDigits + tid];
#pragma unroll
            for(int w = 0; w < 32; w++) {
                count[w * kDigits + tid] = (uint16_t)sum;
                sum += c[w];
            }
            int run = sum;
#pragma unroll
            for(int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, run, o);
                run += lane >= o ? v : 0;
            }
            total[tid] = run - sum;
            if(lane == 31)
                warp_total[warp] = run;
        }
        __syncthreads();
        if(tid < kDigits) {
            int ahead = 0;
            for(int w = 0; w < warp; w++)
                ahead += warp_total[w];
            total[tid] += ahead;
        }
        __syncthreads();
#pragma unroll
        for(int i = 0; i < kSortItems; i++)
            if(live >> i & 1) {
                const uint32_t d = (key[i] >> shift) & mask;
                const int at = total[d] + count[warp * kDigits + d] + rank[i];
                keys[at] = key[i];
                order[at] = item[i];
            }
        __syncthreads();
        if(p + 1 < passes) {
#pragma unroll
            for(int i = 0; i < kSortItems; i++)
                if(live >> i & 1) {
                    key[i] = keys[first + 32 * i];
                    item[i] = order[first + 32 * i];
                }
        }
    }
    for(int i = tid; i < tokens; i += 1024) {
        keys_out[i] = keys[i];
        order_out[i] = order[i];
    }
}

constexpr int kSortSmem = kOneBlock * 6 + 32 * kDigits * 2 + kDigits * 4;

// More tokens: per pass, counts of every block of keys, their sums, the move.
// The first pass reads the ids themselves.
__device__ __forceinline__ unsigned load_keys(size_t tokens, size_t vocab, const void *ids, int wide,
                                              const uint32_t *keys, const int *order,
                                              uint32_t (&key)[kSortItems], int (&item)[kSortItems])
{
    const size_t first = (size_t)blockIdx.x * kManyItems + (threadIdx.x >> 5) * (32 * kSortItems) +
                         (threadIdx.x & 31);
    unsigned live = 0;
#pragma unroll
    for(int i = 0; i < kSortItems; i++) {
        const size_t t = first + 32 * i;
        if(t < tokens) {
            live |= 1u << i;
            key[i] = keys ? keys[t] : key_of(ids, wide, t, vocab);
            item[i] = keys ? order[t] : (int)t;
        }
    }
    return live;
}

__global__ void __launch_bounds__(kManyThreads)
    sort_count_kernel(size_t tokens, size_t vocab, const void *ids, int wide, const uint32_t *keys,
                      const int *order, int shift, uint32_t mask, int *counts, int blocks)
{
    __shared__ int count[kDigits];
    for(int i = threadIdx.x; i < kDigits; i += kManyThreads)
        count[i] = 0;
    __syncthreads();
    uint32_t key[kSortItems];
    int item[kSortItems];
    const unsigned live = load_keys(tokens, vocab, ids, wide, keys, order, key, item);
#pragma unroll
    for(int i = 0; i < kSortItems; i++)
        if(live >> i & 1)
            atomicAdd(&count[(key[i] >> shift) & mask], 1);  // whole numbers: no order
    __syncthreads();
    for(int i = threadIdx.x; i < kDigits; i += kManyThreads)
        counts[(size_t)i * blocks + blockIdx.x] = count[i];
}

__global__ void __launch_bounds__(1024) sort_sums_kernel(int *counts, int n)
{
    __shared__ int warp_total[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int base = 0;
    for(int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + tid, c = i < n ? counts[i] : 0;
        int run = c;
#pragma unroll
        for(int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            run += lane >= o ? v : 0;
        }
        if(lane == 31)
            warp_total[warp] = run;
        __syncthreads();
        int ahead = 0, all = 0;
        for(int w = 0; w < 32; w++) {
            ahead += w < warp ? warp_total[w] : 0;
            all += warp_total[w];
        }
        if(i < n)
            counts[i] = base + ahead + run - c;
        base += all;
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kManyThreads)
    sort_move_kernel(size_t tokens, size_t vocab, const void *ids, int wide, const uint32_t *keys,
                     const int *order, int shift, int bits, const int *counts, int blocks,
                     uint32_t *keys_out, int *order_out)
{
    constexpr int kWarps = kManyThreads / 32;
    const uint32_t mask = (1u << bits) - 1;
    __shared__ uint16_t count[kWarps * kDigits];
    for(int i = threadIdx.x; i < kWarps * kDigits / 2; i += kManyThreads)
        reinterpret_cast<uint32_t *>(count)[i] = 0;
    __syncthreads();
    uint32_t key[kSortItems];
    int item[kSortItems];
    uint16_t rank[kSortItems];
    const int warp = threadIdx.x >> 5;
    const unsigned live = load_keys(tokens, vocab, ids, wide, keys, order, key, item);
    warp_rank(key, shift, bits, kSortItems, live, count + warp * kDigits, rank);
    __syncthreads();
    for(int d = threadIdx.x; d < kDigits; d += kManyThreads) {
        int sum = 0;
        for(int w = 0; w < kWarps; w++) {
            const int c = count[w * kDigits + d];
            count[w * kDigits + d] = (uint16_t)sum;
            sum += c;
        }
    }
    __syncthreads();
#pragma unroll
    for(int i = 0; i < kSortItems; i++)
        if(live >> i & 1) {
            const uint32_t d = (key[i] >> shift) & mask;
            const int at = counts[(size_t)d * blocks + blockIdx.x] + count[warp * kDigits + d] + rank[i];
            keys_out[at] = key[i];
            order_out[at] = item[i];
        }
}

// --------------------------------------------------------- rows without tokens

constexpr int kFillRows = 32768;  // rows that a block marks at a time

// Zeros into the rows [v0, v1) that no id names.  With `sorted` the keys are in
// order and only their stretch of the range is looked at.
template <typename T, int N>
__device__ void fill_rows(size_t v0, size_t v1, size_t tokens, size_t vocab, const void *ids, int wide,
                          const uint32_t *sorted, T *dw, size_t ws, size_t vecs)
{
    __shared__ uint32_t named[kFillRows / 32];
    for(size_t a = v0; a < v1; a += kFillRows) {
        const size_t b = min(a + kFillRows, v1);
        for(int i = threadIdx.x; i < kFillRows / 32; i += blockDim.x)
            named[i] = 0;
        __syncthreads();
        size_t lo = 0, hi = tokens;
        if(sorted) {  // first key >= a
            while(lo < hi) {
                const size_t mid = (lo + hi) / 2;
                if(sorted[mid] < a)
                    lo = mid + 1;
                else
                    hi = mid;
            }
        }
        for(size_t t = lo + threadIdx.x; t < tokens; t += blockDim.x) {
            const size_t k = sorted ? sorted[t] : key_of(ids, wide, t, vocab);
            if(k >= a && k < b)
                atomicOr(&named[(k - a) / 32], 1u << ((k - a) & 31));
            else if(sorted)
                break;
        }
        __syncthreads();
        Vec<T, N> zero;
        float f[N] = {};
        zero.set(f);
        if(vecs <= 0xffffffffu / kFillRows) {
            const uint32_t n = (uint32_t)(b - a) * (uint32_t)vecs, per = (uint32_t)vecs;
            for(uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
                const uint32_t r = i / per, c = i - r * per;
                if(!(named[r / 32] >> (r & 31) & 1))
                    reinterpret_cast<Vec<T, N> *>(dw + (a + r) * ws)[c] = zero;
            }
        } else {
            for(size_t r = 0; r < b - a; r++)
                if(!(named[r / 32] >> (r & 31) & 1))
                    for(size_t c = threadIdx.x; c < vecs; c += blockDim.x)
                        reinterpret_cast<Vec<T, N> *>(dw + (a + r) * ws)[c] = zero;
        }
        __syncthreads();
    }
}

// Block 0 sorts; the others, meanwhile, write the rows without tokens.
template <typename T, int N>
__global__ void __launch_bounds__(1024)
    sort_fill_kernel(int tokens, size_t vocab, int bits, const void *ids, int wide, uint32_t *keys,
                     int *order, T *dw, size_t ws, size_t vecs)
{
    extern __shared__ __align__(16) char sort_smem[];
    if(blockIdx.x == 0) {
        sort_one_block(tokens, vocab, bits, ids, wide, sort_smem, keys, order);
    } else {
        const size_t blocks = gridDim.x - 1, b = blockIdx.x - 1;
        fill_rows<T, N>(vocab * b / blocks, vocab * (b + 1) / blocks, tokens, vocab, ids, wide, nullptr,
                        dw, ws, vecs);
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(1024)
    fill_kernel(size_t tokens, size_t vocab, const uint32_t *sorted, T *dw, size_t ws, size_t vecs)
{
    const size_t blocks = gridDim.x, b = blockIdx.x;
    fill_rows<T, N>(vocab * b / blocks, vocab * (b + 1) / blocks, tokens, vocab, nullptr, 0, sorted, dw,
                    ws, vecs);
}

// ----------------------------------------------------------- sums of the rows
//
// The sorted tokens are cut into chunks of kChunk whatever their ids are, so a
// token that fills half the batch is summed by as many groups of threads as any
// other half.  A run of equal ids that lies inside a chunk is summed and written;
// of one that does not, each chunk leaves its part: slot 0 for a run that came
// from the chunk before, slot 1 for one that begins here.  join_kernel adds up
// the parts, in order.

constexpr int kChunk = 16;  // all rows of a chunk are in flight at once

template <typename T, int N>
__device__ __forceinline__ void write_row(T *row, size_t c, float (&sum)[N], float scale, int accumulate)
{
    Vec<T, N> *to = reinterpret_cast<Vec<T, N> *>(row) + c;
    float f[N], old[N] = {};
    if(accumulate)
        to->get(old);
#pragma unroll
    for(int i = 0; i < N; i++)
        f[i] = accumulate ? fmaf(scale, sum[i], old[i]) : scale * sum[i];
    Vec<T, N> v;
    v.set(f);
    *to = v;
}

template <typename T, int N>
__global__ void __launch_bounds__(256)
    sum_kernel(size_t tokens, size_t vocab, size_t vecs, int lanes, const uint32_t *keys,
               const int *order, const T *dy, size_t ys, float scale, T *dw, size_t ws,
               int accumulate, float *parts)
{
    const size_t chunk = (size_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    const size_t c = (size_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    const size_t e0 = chunk * kChunk;
    if(e0 >= tokens || c >= vecs)
        return;
    const int n = (int)min((size_t)kChunk, tokens - e0);
    // keys and order of the chunk as whole words; behind the last token stands
    // what the workspace held, which no sum uses
    union {
        uint4 q[kChunk / 4];
        uint32_t k[kChunk];
    } key;
    union {
        int4 q[kChunk / 4];
        int t[kChunk];
    } from;
#pragma unroll
    for(int i = 0; i < kChunk / 4; i++) {
        key.q[i] = reinterpret_cast<const uint4 *>(keys + e0)[i];
        from.q[i] = reinterpret_cast<const int4 *>(order + e0)[i];
    }
    const uint32_t behind = e0 + kChunk < tokens ? keys[e0 + kChunk] : 0xffffffffu;
    bool came = e0 > 0 && keys[e0 - 1] == key.k[0];  // the run began in an earlier chunk
    Vec<T, N> v[kChunk];
#pragma unroll
    for(int i = 0; i < kChunk; i++)
        if(i < n && key.k[i] < vocab)
            v[i] = reinterpret_cast<const Vec<T, N> *>(dy + (size_t)from.t[i] * ys)[c];
    float sum[N] = {};
#pragma unroll
    for(int i = 0; i < kChunk; i++) {
        const uint32_t run = key.k[i];
        if(i >= n || run >= vocab)  // ids outside the table: all that follow are
            return;
        float f[N];
        v[i].get(f);
#pragma unroll
        for(int j = 0; j < N; j++)
            sum[j] += f[j];
        const uint32_t next = i + 1 < n ? key.k[i + 1 < kChunk ? i + 1 : i] : behind;
        const bool ends = next != run;
        if(ends || i + 1 == n) {
            if(ends && !came) {
                write_row<T, N>(dw + (size_t)run * ws, c, sum, scale, accumulate);
            } else {
                Vec<float, N> part;
                part.set(sum);
                *reinterpret_cast<Vec<float, N> *>(
                    parts + ((chunk * 2 + (came ? 0 : 1)) * vecs + c) * N) = part;
            }
#pragma unroll
            for(int j = 0; j < N; j++)
                sum[j] = 0.0f;
            came = false;
        }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(256)
    join_rows_kernel(size_t tokens, size_t vocab, size_t vecs, int lanes, const uint32_t *keys,
                     float scale, T *dw, size_t ws, int accumulate, const float *parts)
{
    const size_t chunk = (size_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    const size_t c = (size_t)blockIdx.y * lanes + (threadIdx.x & (lanes - 1));
    const size_t e0 = chunk * kChunk, e1 = e0 + kChunk;
    if(e1 >= tokens || c >= vecs)
        return;
    const uint32_t run = keys[e1 - 1];
    // the run that leaves this chunk, if it began here
    if(run >= vocab || keys[e1] != run || (e0 > 0 && keys[e0] == run && keys[e0 - 1] == run))
        return;
    // the chunk it ends in: the first whose next chunk does not begin with it
    const size_t chunks = (tokens + kChunk - 1) / kChunk;
    auto inside = [&](size_t k) { return k + 1 < chunks && keys[(k + 1) * kChunk] == run; };
    size_t last = chunk + 1, hop = 1;
    while(inside(last + hop - 1)) {
        last += hop;
        hop *= 2;
    }
    while(hop > 1) {  // inside(last - 1) holds
        hop /= 2;
        if(inside(last + hop - 1))
            last += hop;
    }
    float sum[N];
    reinterpret_cast<const Vec<float, N> *>(parts + ((chunk * 2 + 1) * vecs + c) * N)->get(sum);
    const float *p = parts + ((chunk + 1) * 2 * vecs + c) * N;
#pragma unroll 8
    for(size_t k = chunk + 1; k <= last; k++, p += 2 * vecs * N) {
        Vec<float, N> v;
        float f[N];
        v = *reinterpret_cast<const Vec<float, N> *>(p);
        v.get(f);
#pragma unroll
        for(int j = 0; j < N; j++)
            sum[j] += f[j];
    }
    write_row<T, N>(dw + (size_t)run * ws, c, sum, scale, accumulate);
}

// ---------------------------------------------------------------- host side

// Threads that share a row of `vecs` vectors with `each` of them per thread.
int lanes_of(size_t vecs, size_t each)
{
    int lanes = 1;
    while(lanes < 256 && lanes * each < vecs)
        lanes *= 2;
    return lanes;
}

template <typename T, int N>
int lookup(size_t tokens, size_t vocab, size_t dim, const void *ids, int wide, const void *weight,
           size_t ws, float scale, void *out, size_t os, cudaStream_t st)
{
    const size_t vecs = dim / N;
    const int lanes = lanes_of(vecs, 4);
    const size_t blocks = std::min<size_t>((tokens * lanes + 255) / 256, 1 << 20);
    embedding_fwd_kernel<T, N><<<(unsigned)blocks, 256, 0, st>>>(
        tokens, vocab, vecs, lanes, ids, wide, (const T *)weight, ws, scale, (T *)out, os);
    return lm_launched();
}

struct Work {
    size_t blocks;  // of the sort
    size_t at_keys, at_order, at_keys2, at_order2, at_counts, at_parts, bytes;
    Work(size_t tokens, size_t dim)
    {
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t here = at;
            at += lm_up(n, 256);
            return here;
        };
        const bool many = tokens > kOneBlock;
        blocks = (tokens + kManyItems - 1) / kManyItems;
        at_keys = take(lm_up(tokens, kChunk) * 4);
        at_order = take(lm_up(tokens, kChunk) * 4);
        at_keys2 = take(many ? lm_up(tokens, kChunk) * 4 : 0);
        at_order2 = take(many ? lm_up(tokens, kChunk) * 4 : 0);
        at_counts = take(many ? blocks * kDigits * 4 : 0);
        at_parts = take((tokens + kChunk - 1) / kChunk * 2 * dim * 4);
        bytes = at;
    }
};

template <typename T, int N>
int gradient(size_t tokens, size_t vocab, size_t dim, const void *ids, int wide, const void *dy,
             size_t ys, float scale, void *dw, size_t ws, int accumulate, char *work, cudaStream_t st)
{
    const Work w(tokens, dim);
    const size_t vecs = dim / N;
    uint32_t *keys = (uint32_t *)(work + w.at_keys);
    int *order = (int *)(work + w.at_order);
    int sms = 0;
    if(!lm_sms(&sms))
        return B200OPT_ECUDA;
    int bits = 0;  // of the largest key, `vocab`
    while(vocab >> bits)
        bits++;
    const unsigned fill = (unsigned)std::min<size_t>(sms, vocab);
    if(tokens <= kOneBlock) {
        if(cudaFuncSetAttribute(sort_fill_kernel<T, N>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kSortSmem) != cudaSuccess)
            return B200OPT_ECUDA;
        sort_fill_kernel<T, N><<<1 + (accumulate ? 0 : fill), 1024, kSortSmem, st>>>(
            (int)tokens, vocab, bits, ids, wide, keys, order, (T *)dw, ws, vecs);
    } else {
        uint32_t *from_k = nullptr, *to_k = (uint32_t *)(work + w.at_keys2);
        int *from_o = nullptr, *to_o = (int *)(work + w.at_order2), *counts = (int *)(work + w.at_counts);
        const int passes = (bits + 8) / 9, step = (bits + passes - 1) / passes;
        const unsigned blocks = (unsigned)w.blocks;
        if(passes & 1)  // the last pass ends in keys, order
            std::swap(keys, to_k), std::swap(order, to_o);
        for(int p = 0; p < passes; p++) {
            const uint32_t mask = (1u << step) - 1;
            sort_count_kernel<<<blocks, kManyThreads, 0, st>>>(tokens, vocab, ids, wide, from_k, from_o,
                                                               p * step, mask, counts, (int)blocks);
            sort_sums_kernel<<<1, 1024, 0, st>>>(counts, (int)blocks * kDigits);
            sort_move_kernel<<<blocks, kManyThreads, 0, st>>>(tokens, vocab, ids, wide, from_k, from_o,
                                                              p * step, step, counts, (int)blocks, to_k,
                                                              to_o);
            from_k = to_k, from_o = to_o;
            std::swap(keys, to_k), std::swap(order, to_o);
        }
        keys = from_k, order = from_o;
        if(!accumulate)
            fill_kernel<T, N><<<fill, 1024, 0, st>>>(tokens, vocab, keys, (T *)dw, ws, vecs);
    }
    if(tokens) {
        const int lanes = lanes_of(vecs, 1);
        const size_t chunks = (tokens + kChunk - 1) / kChunk, per = 256 / lanes;
        const dim3 grid((unsigned)((chunks + per - 1) / per), (unsigned)((vecs + lanes - 1) / lanes));
        float *parts = (float *)(work + w.at_parts);
        sum_kernel<T, N><<<grid, 256, 0, st>>>(tokens, vocab, vecs, lanes, keys, order, (const T *)dy, ys,
                                               scale, (T *)dw, ws, accumulate, parts);
        if(chunks > 1)
            join_rows_kernel<T, N><<<grid, 256, 0, st>>>(tokens, vocab, vecs, lanes, keys, scale, (T *)dw,
                                                         ws, accumulate, parts);
    }
    return lm_launched();
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
    const bool v = lm_vectors(weight, weight_stride, e, dim) && lm_vectors(out, out_stride, e, dim);
    auto *f = dtype == B200OPT_HALF ? (v ? lookup<__half, 8> : lookup<__half, 1>)
                                    : (v ? lookup<float, 4> : lookup<float, 1>);
    return f(tokens, vocab, dim, ids, index_bytes == 8, weight, weight_stride, scale, out, out_stride,
             (cudaStream_t)stream);
}

int b200opt_embedding_bwd_workspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes)
{
    if(!bytes)
        return B200OPT_EINVAL;
    if(tokens > B200OPT_LM_MAX || vocab > B200OPT_LM_MAX || dim > B200OPT_LM_MAX)
        return B200OPT_ETOOBIG;
    *bytes = Work(tokens, dim).bytes;
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
    if(!vocab || !dim || (!tokens && accumulate))
        return B200OPT_OK;
    const size_t e = lm_size(dtype);
    if((tokens && (!ids || !lm_aligned(ids, index_bytes))) ||
       !lm_matrix(grad_out, tokens, dim, grad_out_stride, e) ||
       !lm_matrix(grad_weight, vocab, dim, grad_weight_stride, e) ||
       workspace_bytes < need || (need && (!workspace || !lm_aligned(workspace, 256))))
        return B200OPT_EINVAL;
    const bool v = lm_vectors(grad_out, grad_out_stride, e, dim) &&
                   lm_vectors(grad_weight, grad_weight_stride, e, dim);
    auto *f = dtype == B200OPT_HALF ? (v ? gradient<__half, 8> : gradient<__half, 1>)
                                    : (v ? gradient<float, 4> : gradient<float, 1>);
    return f(tokens, vocab, dim, ids, index_bytes == 8, grad_out, grad_out_stride, scale, grad_weight,
             grad_weight_stride, accumulate, (char *)workspace, (cudaStream_t)stream);
}

}  // extern "C"
