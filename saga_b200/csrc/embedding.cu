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
// order, so the tokens are brought together by id.  Block b takes the ids that
// are b modulo the number of blocks: neighbouring ids, frequent ones among them,
// fall to different blocks.  Every block looks at all ids (64 KB of int32 for 16384
// tokens, from L2), counts its own by their quotient, knows from the count of
// smaller remainders where its tokens begin, and moves them there by one stable
// counting pass: ranks within a warp's stretch, then sums over warps and digits.

constexpr int kChunk = 16;  // tokens summed by one group of threads
constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;
constexpr int kStretch = 512;                             // consecutive tokens of a warp
constexpr int kOrderChunk = kOrderWarps * kStretch;       // tokens at a time
constexpr int kDigits = 512;                              // rows a block can have
constexpr size_t kOrderBlocks = 148;
constexpr int kOrderSmem = kOrderChunk * 4 + kOrderWarps * kDigits * 2;

// Threads of all blocks together, which is how far a thread steps: 2^32 for the
// largest table, so not a 32-bit number.
__host__ __device__ constexpr size_t order_step(uint32_t blocks) { return (size_t)blocks * kOrderThreads; }

// Many tokens: that every block looks at all of them would be most of the work
// (65536 tokens: 42 us, 262144: 153 us).  They are then first dealt out by remainder, three
// launches of a stable counting pass, and a block looks at its own alone: 23 and 52 us
// together.  At 32768 tokens both ways take 22 us.  The dealing has counters for kDigits
// blocks, so it ends where kDigits rows a block need more of them, at kDigits * kDigits =
// 262144 rows.  Beyond, all blocks (one for every 512 rows, several turns of the GPU) look
// at all ids: the whole gradient of 65536 tokens x 16 takes 47 us with 262144 rows and
// 163 us with 262145, of 262144 tokens 73 and 573 us.

constexpr size_t kSplitTokens = 32768;
constexpr int kDealTokens = 2048;  // of a block: 32 warps, 64 each (8192: the move takes 23 us, not 7.5)

__device__ __forceinline__ int remainder_of(const void *ids, int wide, size_t t, size_t tokens,
                                            size_t vocab, uint32_t blocks, int &id)
{
    id = t < tokens ? lm_index_at(ids, wide, t, vocab) : -1;
    return id < 0 ? -1 : (int)((uint32_t)id % blocks);
}

// How many ids of each remainder a chunk has; counts[remainder][chunk].
__global__ void __launch_bounds__(1024)
    deal_count_kernel(size_t tokens, size_t vocab, const void *ids, int wide, uint32_t blocks, int *counts)
{
    __shared__ int count[kDigits];
    lm_let_next();
    for(int i = threadIdx.x; i < kDigits; i += 1024)
        count[i] = 0;
    __syncthreads();
#pragma unroll
    for(int i = 0; i < kDealTokens / 1024; i++) {
        int id;
        const int r = remainder_of(ids, wide, (size_t)blockIdx.x * kDealTokens + i * 1024 + threadIdx.x,
                                   tokens, vocab, blocks, id);
        if(r >= 0)
            atomicAdd(&count[r], 1);  // whole numbers: any order gives the same
    }
    __syncthreads();
    for(int i = threadIdx.x; i < (int)blocks; i += 1024)
        counts[(size_t)i * gridDim.x + blockIdx.x] = count[i];
}

// n numbers to the sums of those before them; counts[n] gets the sum of all.  It has
// room for kEach more behind that, since numbers are read and written four at a time.
constexpr int kEach = 8;  // of a thread, in a row

__global__ void __launch_bounds__(1024) deal_sums_kernel(int *counts, size_t n)
{
    __shared__ int warp_sums[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int base = 0;
    lm_let_next();
    lm_after_previous();
    for(size_t i0 = 0; i0 < n; i0 += 1024 * kEach) {
        const size_t i = i0 + threadIdx.x * kEach;
        int4 *mine = reinterpret_cast<int4 *>(counts + i);
        int c[kEach], sum = 0;
#pragma unroll
        for(int j = 0; j < kEach; j += 4) {
            const int4 v = i < n ? mine[j / 4] : int4{0, 0, 0, 0};
            c[j] = v.x, c[j + 1] = v.y, c[j + 2] = v.z, c[j + 3] = v.w;
        }
#pragma unroll
        for(int j = 0; j < kEach; j++)
            sum += c[j] = i + j < n ? c[j] : 0;
        int run = sum;
#pragma unroll
        for(int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            run += lane >= o ? v : 0;
        }
        if(lane == 31)
            warp_sums[warp] = run;
        __syncthreads();
        const int w = warp_sums[lane];
        int at = base + __reduce_add_sync(0xffffffffu, lane < warp ? w : 0) + run - sum;
#pragma unroll
        for(int j = 0; j < kEach; j += 4) {
            const int4 v = {at, at + c[j], at + c[j] + c[j + 1], at + c[j] + c[j + 1] + c[j + 2]};
            if(i < n)
                mine[j / 4] = v;
            at = v.w + c[j + 3];
        }
        base += __reduce_add_sync(0xffffffffu, w);
        __syncthreads();
    }
    if(threadIdx.x == 0)
        counts[n] = base;
}

__global__ void __launch_bounds__(1024)
    deal_move_kernel(size_t tokens, size_t vocab, const void *ids, int wide, uint32_t blocks,
                     const int *counts, int *dealt, int *dealt_token)
{
    constexpr int kTrips = kDealTokens / 1024;
    __shared__ uint16_t count[32][kDigits];
    lm_let_next();
    lm_after_previous();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for(int i = lane; i < kDigits / 2; i += 32)
        reinterpret_cast<uint32_t *>(count[warp])[i] = 0;
    __syncwarp();
    const size_t first = (size_t)blockIdx.x * kDealTokens + warp * (32 * kTrips) + lane;
    int id[kTrips], r[kTrips], rank[kTrips];
#pragma unroll
    for(int i = 0; i < kTrips; i++)
        r[i] = remainder_of(ids, wide, first + 32 * i, tokens, vocab, blocks, id[i]);
#pragma unroll
    for(int i = 0; i < kTrips; i++) {  // as in order_kernel
        const unsigned same = __match_any_sync(0xffffffffu, r[i]);
        const int lower = __popc(same & ((1u << lane) - 1));
        rank[i] = r[i] >= 0 ? count[warp][r[i]] + lower : 0;
        __syncwarp();
        if(r[i] >= 0 && lower == 0)
            count[warp][r[i]] += (uint16_t)__popc(same);
        __syncwarp();
    }
    __syncthreads();
    for(int d = threadIdx.x; d < (int)blocks; d += 1024) {
        int total = 0;
        for(int w = 0; w < 32; w++) {
            const int c = count[w][d];
            count[w][d] = (uint16_t)total;
            total += c;
        }
    }
    __syncthreads();
#pragma unroll
    for(int i = 0; i < kTrips; i++)
        if(r[i] >= 0) {
            const int at = counts[(size_t)r[i] * gridDim.x + blockIdx.x] + count[warp][r[i]] + rank[i];
            dealt[at] = id[i];
            dealt_token[at] = (int)(first + 32 * i);
        }
}

// keys: the ids in their new order, `vocab` behind the last; order: the tokens;
// ends: where a run of equal ids ends (at its first kChunk tokens).  named: for
// each row, whether it has a token.  DEALT: ids (and dealt_token) are dealt
// out, block b's from starts[b * pitch].
//
// The loops stay rolled: the code runs once per block, so its length, fetched cold,
// would cost more than the branches (unrolled over the ids of a thread it took 9 us
// for 64 tokens).
template <bool DEALT>
__global__ void __launch_bounds__(kOrderThreads, 1)
    order_kernel(size_t tokens, size_t vocab, const void *ids, int wide, const int *starts, size_t pitch,
                 const int *dealt_token, uint32_t *keys, int *order, int *ends, unsigned char *named)
{
    extern __shared__ __align__(16) char order_smem[];
    // this block's tokens, in order, for each warp: place in its stretch << 20 | rank << 9 | digit
    uint32_t *list = reinterpret_cast<uint32_t *>(order_smem) + (threadIdx.x >> 5) * kStretch;
    uint16_t *counts = reinterpret_cast<uint16_t *>(order_smem + kOrderChunk * 4);
    __shared__ int base[kDigits], warp_sums[kOrderWarps], before_sum, valid_sum;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t blocks = gridDim.x, me = blockIdx.x;
    // id / blocks by a rounded-down reciprocal: at most one too small below 2^31
    const uint32_t inverse = 0xffffffffu / blocks;
    const int digits = (int)((vocab - me + blocks - 1) / blocks);  // this block's rows
    uint16_t *count = counts + warp * kDigits;
    lm_let_next();
    if(DEALT)
        lm_after_previous();
    const size_t t0 = DEALT ? starts[me * pitch] : 0, t1 = DEALT ? starts[(me + 1) * pitch] : tokens;
    // a warp's stretch: shorter where there are few tokens, so that all warps have some
    const int stretch =
        (int)min((t1 - t0 + kOrderThreads - 1) / kOrderThreads * 32, (size_t)kStretch);
    const size_t step = (size_t)stretch * kOrderWarps;
    if(tid < kDigits)
        base[tid] = 0;
    if(tid == 0) {
        before_sum = (int)t0;
        valid_sum = DEALT ? starts[blocks * pitch] : 0;
    }
    __syncthreads();

    int n = 0, before = 0, valid = 0, my_start = 0, my_end = 0;
    for(int pass = 0; pass < 2; pass++) {
        for(size_t c0 = t0; c0 < t1; c0 += step) {
            const size_t first = c0 + warp * stretch;
            if(pass == 0 || t1 - t0 > step) {
                n = 0;
                // the stretch's ids, many loads in flight; the block's own replace them
                const int here = (int)min((size_t)stretch, t1 > first ? t1 - first : 0);
                __syncwarp();
#pragma unroll 16
                for(int i = lane; i < here; i += 32)
                    list[i] = (uint32_t)lm_index_at(ids, wide, first + i, vocab);
                __syncwarp();
                for(int i = lane; i - lane < here; i += 32) {
                    const int id = i < here ? (int)list[i] : -1;
                    uint32_t q = __umulhi((uint32_t)id, inverse), r = (uint32_t)id - q * blocks;
                    if(r >= blocks)
                        q++, r -= blocks;
                    const bool mine = id >= 0 && r == me;
                    if(pass == 0) {
                        before += id >= 0 && r < me;
                        valid += id >= 0 && !DEALT;
                        if(mine)
                            atomicAdd(&base[q], 1);  // whole numbers: any order gives the same
                    }
                    const unsigned who = __ballot_sync(0xffffffffu, mine);
                    if(mine)
                        list[n + __popc(who & ((1u << lane) - 1))] = (uint32_t)i << 20 | q;
                    n += __popc(who);
                }
            }
            if(pass == 0)
                continue;
            for(int i = lane; i < kDigits / 2; i += 32)
                reinterpret_cast<uint32_t *>(count)[i] = 0;
            __syncwarp();
            for(int i = 0; i < n; i += 32) {  // ranks among the warp's tokens of the same digit
                const bool have = i + lane < n;  // the others' digit is like no token's
                const uint32_t e = have ? list[i + lane] : 0, d = have ? e & (kDigits - 1) : kDigits;
                const unsigned same = __match_any_sync(0xffffffffu, d);
                const int lower = __popc(same & ((1u << lane) - 1)), seen = have ? count[d] : 0;
                __syncwarp();
                if(have) {
                    if(lower == 0)
                        count[d] = (uint16_t)(seen + __popc(same));
                    list[i + lane] = e | (uint32_t)(seen + lower) << 9;
                }
                __syncwarp();
            }
            __syncthreads();
            int total = 0;
            if(tid < kDigits)
                for(int w = 0; w < kOrderWarps; w += 8) {
                    int c[8];
#pragma unroll
                    for(int k = 0; k < 8; k++)
                        c[k] = counts[(w + k) * kDigits + tid];
#pragma unroll
                    for(int k = 0; k < 8; k++) {
                        counts[(w + k) * kDigits + tid] = (uint16_t)total;
                        total += c[k];
                    }
                }
            __syncthreads();
            for(int i = lane; i < n; i += 32) {
                const uint32_t e = list[i], d = e & (kDigits - 1);
                const int at = base[d] + count[d] + (int)(e >> 9 & 0x7ff);
                keys[at] = d * blocks + me;
                const size_t from = first + (e >> 20);
                order[at] = DEALT ? dealt_token[from] : (int)from;
            }
            __syncthreads();
            if(tid < kDigits)
                base[tid] += total;
        }
        if(pass)
            break;
        // base: from numbers to places
        before = __reduce_add_sync(0xffffffffu, before);
        valid = __reduce_add_sync(0xffffffffu, valid);
        if(lane == 0) {
            atomicAdd(&before_sum, before);
            atomicAdd(&valid_sum, valid);
        }
        __syncthreads();
        const int mine = tid < kDigits ? base[tid] : 0;
        int run = mine;
#pragma unroll
        for(int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            run += lane >= o ? v : 0;
        }
        if(lane == 31)
            warp_sums[warp] = run;
        __syncthreads();
        my_end = before_sum + run +
                 __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0);
        my_start = my_end - mine;
        if(tid < kDigits)
            base[tid] = my_start;
        if(tid < digits)
            named[(size_t)tid * blocks + me] = mine > 0;
    }
    // where a run ends, at its first tokens: as far as the chunk it begins in can reach
    if(tid < kDigits)
        for(int i = my_start; i < min(my_end, my_start + kChunk); i++)
            ends[i] = my_end;
    for(size_t i = (size_t)valid_sum + order_step(me) + tid; i < tokens; i += order_step(blocks))
        keys[i] = (uint32_t)vocab;
}

// ----------------------------------------------------------- sums of the rows
//
// The sorted tokens are cut into chunks of kChunk whatever their ids are, so a
// token that fills half the batch is summed by as many groups of threads as any
// other half.  A run of equal ids that lies inside a chunk is summed and written;
// of one that does not, each chunk leaves its part: slot 0 for a run that came
// from the chunk before, slot 1 for one that begins here.  join_kernel adds up
// the parts, in order.

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

// Zeros into the rows that no token names, three ways, all in the same grid as the
// sums.  Rows of whole vectors and at least kBulkRow bytes: bulk copies of a zeroed
// buffer, kBulkBytes of the table a block (the whole gradient for 50021 rows of
// 4 KB: 65 us, with the threads' own stores 73; of 1 KB: 20.9 and 21.9; below that
// they are even).
// Shorter rows of whole vectors: kFill vectors of the table a block.  Other rows: a
// warp a row, kFillRows rows a block.
constexpr int kFill = 4096;
constexpr int kFillRows = 32;
constexpr size_t kBulkRow = 1024, kBulkBytes = 128 << 10;
constexpr int kZeros = 4096;  // bytes of the buffer

__host__ __device__ inline size_t bulk_rows(size_t row_bytes)
{
    return row_bytes < kBulkRow ? 0 : row_bytes < kBulkBytes ? kBulkBytes / row_bytes : 1;
}

// The zeroed buffer; all 256 threads of a block, then a barrier.
__device__ __forceinline__ void make_zeros(uint4 *zeros)
{
    static_assert(kZeros == 256 * 16, "a word a thread");
    zeros[threadIdx.x] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Starts the bulk copies of one row's zeros, by one thread.
__device__ __forceinline__ void start_zeros(void *row, size_t bytes, const uint4 *zeros)
{
    const uint32_t from = (uint32_t)__cvta_generic_to_shared(zeros);
    for(size_t at = 0; at < bytes; at += kZeros)
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                         static_cast<char *>(row) + at),
                     "r"(from), "r"((uint32_t)min((size_t)kZeros, bytes - at))
                     : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

__device__ __forceinline__ void wait_zeros()
{
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// A row's zeros by one warp: element by element up to the first 16-byte boundary,
// whole words, the rest.
template <typename T>
__device__ __forceinline__ void zero_row(T *row, size_t n)
{
    const int lane = threadIdx.x & 31;
    const size_t head = min(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T), n);
    const size_t words = (n - head) * sizeof(T) / 16, tail = head + words * (16 / sizeof(T));
    if(lane < head)
        lm_store(row + lane, 0.0f);
    for(size_t w = lane; w < words; w += 32)
        reinterpret_cast<uint4 *>(row + head)[w] = make_uint4(0, 0, 0, 0);
    if(tail + lane < n)
        lm_store(row + tail + lane, 0.0f);
}

template <typename T, int N>
__device__ __forceinline__ void fill_rows(size_t block, size_t vocab, size_t vecs,
                                          const unsigned char *named, T *dw, size_t ws)
{
    if(N > 1) {
        const size_t per_block = bulk_rows(vecs * 16);
        if(per_block) {
            __shared__ __align__(128) uint4 zeros[kZeros / 16];
            make_zeros(zeros);
            __syncthreads();
            const size_t r = block * per_block + threadIdx.x;
            if(threadIdx.x < per_block && r < vocab && !named[r]) {
                start_zeros(dw + r * ws, vecs * 16, zeros);
                wait_zeros();
            }
            return;
        }
        const size_t at = block * kFill, row0 = at / vecs;
        const uint32_t col0 = (uint32_t)(at - row0 * vecs), per = (uint32_t)vecs;
        const uint32_t n = (uint32_t)min((size_t)kFill, vocab * vecs - at);
#pragma unroll 4
        for(uint32_t i = threadIdx.x; i < n; i += 256) {
            const uint32_t r = (col0 + i) / per, c = col0 + i - r * per;
            if(!named[row0 + r])
                reinterpret_cast<uint4 *>(dw + (row0 + r) * ws)[c] = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    for(int i = threadIdx.x >> 5; i < kFillRows; i += 8) {
        const size_t r = block * kFillRows + i;
        if(r < vocab && !named[r])
            zero_row(dw + r * ws, vecs);
    }
}

// `sums` blocks add up rows of grad_out, the others write zeros; both kinds are
// spread evenly over the grid, so that the reads of the one run beside the writes
// of the other.
template <typename T, int N>
__global__ void __launch_bounds__(256, 2)
    sum_kernel(size_t tokens, size_t vocab, size_t vecs, int lanes, size_t sums, size_t slices,
               const uint32_t *keys, const int *order, const unsigned char *named, const T *dy,
               size_t ys, float scale, T *dw, size_t ws, int accumulate, float *parts)
{
    lm_let_next();
    lm_after_previous();
    const size_t block = blockIdx.x * sums / gridDim.x;  // sum blocks before this one
    if((blockIdx.x + 1) * sums / gridDim.x == block) {
        fill_rows<T, N>(blockIdx.x - block, vocab, vecs, named, dw, ws);
        return;
    }
    const size_t chunk = block / slices * (256 / lanes) + threadIdx.x / lanes;
    const size_t c = block % slices * lanes + (threadIdx.x & (lanes - 1));
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

// A warp looks at one chunk and 32 vectors of the row, a block at eight chunks.  A
// run of a few parts is joined by its warp, a long one by the block: each warp
// adds up every eighth part, then the eight sums are added in order.
constexpr size_t kWarpParts = 16;

template <typename T, int N>
__global__ void __launch_bounds__(256, 4)
    join_rows_kernel(size_t tokens, size_t vocab, size_t vecs, size_t slices, const uint32_t *keys,
                     const int *ends, float scale, T *dw, size_t ws, int accumulate,
                     const float *parts)
{
    lm_after_previous();
    __shared__ size_t last_of[8];
    __shared__ Vec<float, N> joined[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t chunk0 = blockIdx.x / slices * 8, chunk = chunk0 + warp;
    const size_t c = blockIdx.x % slices * 32 + lane;
    const size_t e0 = chunk * kChunk, e1 = e0 + kChunk;
    size_t last = 0;  // the chunk that a run ends in which leaves this one and began here
    uint32_t run = 0;
    if(e1 < tokens) {
        run = keys[e1 - 1];
        const uint32_t next = keys[e1], first = keys[e0];
        const uint32_t earlier = e0 > 0 ? keys[e0 - 1] : 0xffffffffu;
        const int end = ends[e1 - 1];
        if(run < vocab && next == run && !(first == run && earlier == run))
            last = (size_t)(end - 1) / kChunk;
    }
    auto part = [&](size_t from, size_t k) {  // part k of the run that begins in chunk `from`
        const size_t slot = (from + k) * 2 + (k ? 0 : 1);
        return reinterpret_cast<const Vec<float, N> *>(parts)[slot * vecs + c];
    };
    auto add_parts = [&](size_t from, size_t k0, size_t n, size_t step, float (&sum)[N]) {
        for(; k0 < n; k0 += 4 * step) {
            Vec<float, N> v[4];
#pragma unroll
            for(int i = 0; i < 4; i++)
                if(k0 + i * step < n)
                    v[i] = part(from, k0 + i * step);
#pragma unroll
            for(int i = 0; i < 4; i++)
                if(k0 + i * step < n) {
                    float f[N];
                    v[i].get(f);
#pragma unroll
                    for(int j = 0; j < N; j++)
                        sum[j] += f[j];
                }
        }
    };
    if(last && last - chunk < kWarpParts) {
        if(c < vecs) {
            float sum[N] = {};
            add_parts(chunk, 0, last - chunk + 1, 1, sum);
            write_row<T, N>(dw + (size_t)run * ws, c, sum, scale, accumulate);
        }
        last = 0;
    }
    if(lane == 0)
        last_of[warp] = last;
    if(!__syncthreads_or(last != 0))
        return;
    for(int i = 0; i < 8; i++) {
        const size_t end = last_of[i], from = chunk0 + i;
        if(!end)
            continue;
        float sum[N] = {};
        if(c < vecs)
            add_parts(from, warp, end - from + 1, 8, sum);
        joined[warp][lane].set(sum);
        __syncthreads();
        if(warp == i && c < vecs) {
#pragma unroll
            for(int w = 0; w < 8; w++) {
                float f[N];
                joined[w][lane].get(f);
#pragma unroll
                for(int j = 0; j < N; j++)
                    sum[j] = w ? sum[j] + f[j] : f[j];
            }
            write_row<T, N>(dw + (size_t)run * ws, c, sum, scale, accumulate);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ few tokens
//
// Up to kFewTokens tokens: all of it in one launch, without a workspace, where the
// three launches above would be most of the time (64 tokens, 32000 x 512 fp16: 9.6 us
// here, 13.4 there; at worst 128 tokens of one id, which one block adds up: 50021 x
// 2048 takes 50 us here, 43 there).  A block again has the ids of one remainder,
// finds its tokens among all, writes its rows without tokens, and sums the others
// itself: runs of up to kWarpRun tokens a warp each, longer ones by the whole block.

constexpr int kFewTokens = 128;
constexpr int kFewBlocks = 593;   // a prime: ids at a regular distance do not meet in one block
constexpr int kFewDigits = 2048;  // rows a block can have
constexpr int kWarpRun = 8;

template <typename T, int N>
__global__ void __launch_bounds__(256)
    few_tokens_kernel(int tokens, size_t vocab, size_t vecs, const void *ids, int wide, const T *dy,
                      size_t ys, float scale, T *dw, size_t ws, int accumulate)
{
    __shared__ __align__(128) uint4 zeros[kZeros / 16];
    __shared__ Vec<float, N> joined[8][32];
    __shared__ uint32_t named[kFewDigits / 32];
    __shared__ uint16_t digit[kFewTokens], token[kFewTokens], run_of[kFewTokens], run[kFewTokens],
        list[8][kWarpRun];
    __shared__ int warp_count[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t blocks = gridDim.x, me = blockIdx.x;
    const int digits = (int)((vocab - me + blocks - 1) / blocks);
    const int id = tid < tokens ? lm_index_at(ids, wide, tid, vocab) : -1;
    const uint32_t q = (uint32_t)id / blocks;
    const bool mine = id >= 0 && (uint32_t)id - q * blocks == me;
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    if(lane == 0)
        warp_count[warp] = __popc(who);
    if(tid < kFewDigits / 32)
        named[tid] = 0;
    make_zeros(zeros);
    __syncthreads();
    int m = 0, at = __popc(who & ((1u << lane) - 1));
    for(int w = 0; w < 8; w++) {
        at += w < warp ? warp_count[w] : 0;
        m += warp_count[w];
    }
    if(mine) {
        digit[at] = (uint16_t)q;
        token[at] = (uint16_t)tid;
        atomicOr(&named[q >> 5], 1u << (q & 31));
    }
    __syncthreads();
    const bool bulk = N > 1 && vecs * 16 >= kBulkRow;
    if(!accumulate) {
        if(bulk) {
            for(int r = tid; r < digits; r += 256)
                if(!(named[r >> 5] >> (r & 31) & 1))
                    start_zeros(dw + ((size_t)r * blocks + me) * ws, vecs * 16, zeros);
        } else {
            for(int r = warp; r < digits; r += 8)
                if(!(named[r >> 5] >> (r & 31) & 1))
                    zero_row(dw + ((size_t)r * blocks + me) * ws, vecs * N);
        }
    }
    // the length of the run that begins at each token, 0 where none does, and a token's
    // place in its run
    int rank = 0;
    if(tid < m) {
        int same = 0;
        for(int j = 0; j < m; j++) {
            const bool s = digit[j] == digit[tid];
            same += s;
            rank += s && j < tid;
        }
        run_of[tid] = (uint16_t)(rank ? 0 : same);
    }
    __syncthreads();
    auto row = [&](int i) { return dw + ((size_t)digit[i] * blocks + me) * ws; };
    auto load = [&](int t, size_t c) { return reinterpret_cast<const Vec<T, N> *>(dy + (size_t)t * ys)[c]; };
    for(int i = warp; i < m; i += 8) {
        const int n = run_of[i];
        if(n == 0 || n > kWarpRun)
            continue;
        int found = 0;
        for(int j = 0; j < m; j += 32) {
            const bool s = j + lane < m && digit[j + lane] == digit[i];
            const unsigned same = __ballot_sync(0xffffffffu, s);
            if(s)
                list[warp][found + __popc(same & ((1u << lane) - 1))] = token[j + lane];
            found += __popc(same);
        }
        __syncwarp();
        for(size_t c = lane; c < vecs; c += 32) {
            float sum[N] = {};
            for(int k = 0; k < n; k += 4) {
                Vec<T, N> v[4];
#pragma unroll
                for(int u = 0; u < 4; u++)
                    if(k + u < n)
                        v[u] = load(list[warp][k + u], c);
#pragma unroll
                for(int u = 0; u < 4; u++)
                    if(k + u < n) {
                        float f[N];
                        v[u].get(f);
#pragma unroll
                        for(int x = 0; x < N; x++)
                            sum[x] += f[x];
                    }
            }
            write_row<T, N>(row(i), c, sum, scale, accumulate);
        }
        __syncwarp();
    }
    // long runs: the warps share out stretches of 32 vectors, and the tokens where
    // there are fewer than eight stretches
    const size_t slices = (vecs + 31) / 32;
    const int split = slices >= 8 ? 1 : slices >= 4 ? 2 : slices >= 2 ? 4 : 8;
    for(int i = 0; i < m; i++) {
        const int n = run_of[i];
        if(n <= kWarpRun)
            continue;
        if(tid < m && digit[tid] == digit[i])
            run[rank] = token[tid];
        __syncthreads();
        for(size_t s0 = 0; s0 < slices; s0 += 8 / split) {
            const size_t c = (s0 + warp / split) * 32 + lane;
            float sum[N] = {};
            if(c < vecs)
                for(int k = warp % split; k < n; k += 8 * split) {
                    Vec<T, N> v[8];
#pragma unroll
                    for(int u = 0; u < 8; u++)
                        if(k + u * split < n)
                            v[u] = load(run[k + u * split], c);
#pragma unroll
                    for(int u = 0; u < 8; u++)
                        if(k + u * split < n) {
                            float f[N];
                            v[u].get(f);
#pragma unroll
                            for(int x = 0; x < N; x++)
                                sum[x] += f[x];
                        }
                }
            if(split > 1) {
                joined[warp][lane].set(sum);
                __syncthreads();
                if(warp % split == 0)
                    for(int w = 1; w < split; w++) {
                        float f[N];
                        joined[warp + w][lane].get(f);
#pragma unroll
                        for(int x = 0; x < N; x++)
                            sum[x] += f[x];
                    }
            }
            if(warp % split == 0 && c < vecs)
                write_row<T, N>(row(i), c, sum, scale, accumulate);
            __syncthreads();
        }
    }
    if(bulk)
        wait_zeros();
}

// ---------------------------------------------------------------- host side

// Threads that share a row of `vecs` vectors with `each` of them per thread.
int lanes_of(size_t vecs, size_t each)
{
    size_t lanes = 1;
    while(lanes < 256 && lanes * each < vecs)
        lanes *= 2;
    // not with more than an eighth of the threads idle in the last stretch of a row
    while(lanes > 32 && (vecs + lanes - 1) / lanes * lanes - vecs > vecs / 8)
        lanes /= 2;
    return (int)lanes;
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

bool few_tokens(size_t tokens, size_t vocab)
{
    return tokens <= kFewTokens && vocab <= (size_t)kFewBlocks * kFewDigits;
}

struct Work {
    bool split;
    size_t blocks, deals;  // of order_kernel; of the dealing
    size_t at_keys, at_order, at_ends, at_named, at_parts, at_dealt, at_token, at_counts, bytes;
    Work(size_t tokens, size_t vocab, size_t dim)
    {
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t here = at;
            at += lm_up(n, 256);
            return here;
        };
        at_keys = take(lm_up(tokens, kChunk) * 4);
        at_order = take(lm_up(tokens, kChunk) * 4);
        at_ends = take(lm_up(tokens, kChunk) * 4);
        at_named = take(vocab);
        at_parts = take((tokens + kChunk - 1) / kChunk * 2 * dim * 4);
        // one block an SM, more where a block would get more rows than it has digits for
        blocks = std::min(vocab, std::max<size_t>(kOrderBlocks, (vocab + kDigits - 1) / kDigits));
        split = tokens > kSplitTokens && blocks <= kDigits;
        deals = (tokens + kDealTokens - 1) / kDealTokens;
        at_dealt = take(split ? tokens * 4 : 0);
        at_token = take(split ? tokens * 4 : 0);
        at_counts = take(split ? (blocks * deals + 1 + kEach) * 4 : 0);
        bytes = at;
    }
};

template <typename T, int N>
int gradient(size_t tokens, size_t vocab, size_t dim, const void *ids, int wide, const void *dy,
             size_t ys, float scale, void *dw, size_t ws, int accumulate, char *work, cudaStream_t st)
{
    const size_t vecs = dim / N;
    if(few_tokens(tokens, vocab)) {
        few_tokens_kernel<T, N><<<(unsigned)std::min<size_t>(vocab, kFewBlocks), 256, 0, st>>>(
            (int)tokens, vocab, vecs, ids, wide, (const T *)dy, ys, scale, (T *)dw, ws, accumulate);
        return lm_launched();
    }
    const Work w(tokens, vocab, dim);
    uint32_t *keys = (uint32_t *)(work + w.at_keys);
    int *order = (int *)(work + w.at_order), *ends = (int *)(work + w.at_ends);
    unsigned char *named = (unsigned char *)(work + w.at_named);
    float *parts = (float *)(work + w.at_parts);
    static std::atomic<uint64_t> allowed{0};
    static std::atomic<uint64_t> allowed_dealt{0};
    if(!lm_allow_smem(order_kernel<false>, kOrderSmem, allowed) ||
       !lm_allow_smem(order_kernel<true>, kOrderSmem, allowed_dealt))
        return B200OPT_ECUDA;
    const int lanes = lanes_of(vecs, 1);
    const size_t chunks = (tokens + kChunk - 1) / kChunk, per = 256 / lanes;
    const size_t groups = (chunks + per - 1) / per, slices = (vecs + lanes - 1) / lanes;
    const size_t bulk = N > 1 ? bulk_rows(vecs * 16) : 0;
    const size_t fills = accumulate ? 0
                         : bulk     ? (vocab + bulk - 1) / bulk
                         : N > 1    ? (vocab * vecs + kFill - 1) / kFill
                                    : (vocab + kFillRows - 1) / kFillRows;
    const size_t cuts = (vecs + 31) / 32, joins = (chunks + 7) / 8 * cuts;
    if(groups * slices + fills > 0x7fffffff || joins > 0x7fffffff)
        return B200OPT_ETOOBIG;
    const uint32_t blocks = (uint32_t)w.blocks;
    if(w.split) {
        int *dealt = (int *)(work + w.at_dealt), *token = (int *)(work + w.at_token);
        int *counts = (int *)(work + w.at_counts);
        deal_count_kernel<<<(unsigned)w.deals, 1024, 0, st>>>(tokens, vocab, ids, wide, blocks, counts);
        lm_launch_next(deal_sums_kernel, 1, 1024, 0, st, counts, w.blocks * w.deals);
        lm_launch_next(deal_move_kernel, (unsigned)w.deals, 1024, 0, st, tokens, vocab, ids, wide, blocks,
                       counts, dealt, token);
        lm_launch_next(order_kernel<true>, blocks, kOrderThreads, kOrderSmem, st, tokens, vocab, dealt, 0,
                       counts, w.deals, token, keys, order, ends, named);
    } else {
        order_kernel<false><<<blocks, kOrderThreads, kOrderSmem, st>>>(
            tokens, vocab, ids, wide, nullptr, 0, nullptr, keys, order, ends, named);
    }
    lm_launch_next(sum_kernel<T, N>, (unsigned)(groups * slices + fills), 256, 0, st, tokens, vocab, vecs, lanes,
                   groups * slices, slices, keys, order, named, (const T *)dy, ys, scale, (T *)dw, ws, accumulate,
                   parts);
    if(chunks > 1)
        lm_launch_next(join_rows_kernel<T, N>, (unsigned)joins, 256, 0, st, tokens, vocab, vecs, cuts, keys, ends,
                       scale, (T *)dw, ws, accumulate, parts);
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
    *bytes = few_tokens(tokens, vocab) ? 0 : Work(tokens, vocab, dim).bytes;
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
