// The matrix product of the vocabulary loss: fp16 operands, fp32 accumulation
// on the tensor cores (tcgen05), with the loss's own epilogues.
//
//   acc[m][n] = sum_k A[m][k] B[n][k]
//
// A pair of CTAs (a cluster of two) computes a 256 x 256 tile with one
// cta_group::2 instruction stream: each CTA holds 128 rows of A and 128 rows of
// B in shared memory and 128 rows x 256 columns of the result in its tensor
// memory.  A single CTA's 128 x 256 tile would fetch 1.5 times as many bytes from
// L2 for the same arithmetic (85 against 128 flops a byte).  At 4096 x 50021 x 2048
// the product with the losses in its epilogue takes 577 us, 1.45 PFLOP/s or 0.88 of
// the measured bf16 rate; long runs are bound by the power limit (8192 x 128000 x
// 4096: 6.7 ms, 1.28 PFLOP/s, 0.90 of the measured sustained rate).
//
// Either operand may be "K-major" (k contiguous in memory) or "MN-major" (m or n
// contiguous): TMA brings boxes of 64 contiguous elements (128 bytes, swizzled)
// and the shared-memory descriptors say which way they lie, so that no operand
// is ever transposed in memory.
//
// Warps: 0 issues the TMA loads, 1 (of the even CTA) the MMAs, 2 owns the tensor
// memory, 4..19 are the epilogue.  Two accumulators alternate, so the epilogue
// of a tile runs beside the main loop of the next one; a wide tile has both, and
// its halves are skewed to the same end.
//
// Every wait is bounded: one that runs out makes the epilogue write NaN for the
// tiles it did not get, which the loss and the optimizer's overflow flags show.
#pragma once

#include <cuda.h>

#include "lm_common.cuh"

namespace b200 {

constexpr int kTcTile = 256;    // tile of a CTA pair, both ways; a wide one is 256 x 512
constexpr int kTcHalf = 128;    // a CTA's rows of A, of B and of the result
constexpr int kTcK = 64;        // k per stage: 128 bytes, the swizzle's span
constexpr int kTcOperand = kTcHalf * kTcK * 2;  // bytes of one operand of a stage in a CTA
constexpr int kTcEpilogue = 16;  // warps: four for each 32 rows, 64 columns each
constexpr int kTcColumns = kTcTile / (kTcEpilogue / 4);
constexpr int kTcThreads = 128 + 32 * kTcEpilogue;
// Stages of A and of NH times 128 rows of B, the bytes in which each epilogue warp
// turns its columns around, and the dynamic shared memory of it all.
__host__ __device__ constexpr int tc_stages(int nh) { return nh == 1 ? 5 : 4; }
__host__ __device__ constexpr int tc_staging(int nh) { return nh == 1 ? 4096 : 2048; }
__host__ __device__ constexpr int tc_stage_bytes(int nh) { return (1 + nh) * kTcOperand; }
constexpr int tc_smem(int nh)
{
    return tc_stages(nh) * tc_stage_bytes(nh) + kTcEpilogue * tc_staging(nh) + 1024;
}

struct TcShape {
    // sizes in elements; a dynamic size is read from *count on the device
    // and held to at least one row (which the operands then hold as zeros)
    int m, n, k;
    const int *count;   // replaces m (dyn_m) or k (dyn_k)
    int dyn_m, dyn_k;
    int a_row0, b_row0;  // first row of the tensor maps' outer dimension that is used
    int splits;          // the k range is cut into so many parts
    int group;           // m tiles that are walked through before the next n tile
    int sum_rows;        // dyn_m and splits > 1: rows that the parts' sums have room for
    int plan_stages;     // and the stages of k that the parts are planned for
};

constexpr int kTcPlanPairs = 74;  // CTA pairs that a product is cut for: 148 SMs

// How many parts the k range of a product is cut into: as many as fill the GPU
// when its tiles alone do not, each with at least 16 stages of k (a part of eight
// saves 2 us of main loop, which the launch that joins the parts costs again).
__host__ __device__ inline uint32_t tc_parts(uint32_t tiles, uint32_t stages)
{
    const uint32_t fill = kTcPlanPairs / tiles, most = stages / 16;
    const uint32_t parts = fill < most ? fill : most;
    return parts ? parts : 1;
}

// The same on the device, where the number of rows is known: fewer rows than
// planned leave room for more parts.
__device__ __forceinline__ uint32_t tc_parts_of(const TcShape &s, int rows)
{
    if(s.splits <= 1 || !s.dyn_m)
        return s.splits;
    const uint32_t tiles = ((rows + kTcTile - 1) / kTcTile) * ((s.n + kTcTile - 1) / kTcTile);
    return min(tc_parts(tiles, s.plan_stages), (uint32_t)s.sum_rows / (uint32_t)rows);
}

// --------------------------------------------------------------- primitives

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Address of the same shared variable in another CTA of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::
                     : "memory");
}

// A box of the tensor into this CTA's shared memory; its bytes count on `bar`,
// a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y,
                                         uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// Shared-memory descriptor of an operand: 128-byte swizzle.  K-major: rows of
// 128 bytes, groups of eight rows 1024 bytes apart.  MN-major: one row of 128
// bytes (64 elements of m or n) per k, groups of eight k 1024 bytes apart, the
// next 64 elements of m or n 8192 bytes further (one box of 64 k).
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr)
{
    uint64_t d = (uint64_t)((addr & 0x3ffff) >> 4);
    d |= (uint64_t)(MN ? 8192 >> 4 : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// 16 elements of k further within a stage
template <bool MN>
__device__ __forceinline__ uint64_t k_step()
{
    return (MN ? 16 * 128 : 16 * 2) >> 4;
}

// kind::f16, fp32 accumulator, fp16 operands, 256 x 256
template <bool A_MN, bool B_MN>
__device__ __forceinline__ constexpr uint32_t instruction_desc()
{
    return (1u << 4) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u) |
           ((uint32_t)(kTcTile >> 3) << 17) | ((uint32_t)(kTcTile >> 4) << 24);
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}

// Arrives on this barrier of both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

// 32 columns of this thread's row of the accumulator
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32])
{
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}

// Waits for the loads issued so far.  The registers pass through it, so that no use
// of them can be moved in front of the wait.
__device__ __forceinline__ void tmem_wait(float (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for(int j = 0; j < 32; j++)
        asm volatile("" : "+f"(v[j]));
}

// A part of the sum without a share of k is 0, a tile whose wait ran out NaN.
__device__ __forceinline__ void no_result(float (&v)[32], bool ok)
{
#pragma unroll
    for(int j = 0; j < 32; j++)
        v[j] = ok ? 0.0f : __int_as_float(0x7fffffff);
}

// ------------------------------------------------------------- epilogue's turn
//
// A thread has 32 columns of one row; written straight to memory that would be a
// scattered 16 bytes a thread.  A warp therefore passes its 32 rows through shared
// memory (16-byte words, their places permuted so that neither side meets a bank
// twice) and comes out with rows side by side: `put` takes word w of this thread's
// row, `get` gives a word of row `row()`, step by step.
template <int WORDS>  // 16-byte words of a row: 4 (fp16) or 8 (fp32)
struct Turn {
    char *buf;
    int lane;
    static constexpr int kSteps = WORDS;  // 32 / WORDS rows a step
    __device__ __forceinline__ uint4 *at(int row, int word) const
    {
        const int key = WORDS == 8 ? row & 7 : (row >> 1) & 3;
        return reinterpret_cast<uint4 *>(buf + row * (WORDS * 16) + ((word ^ key) << 4));
    }
    __device__ __forceinline__ void put(int word, uint4 v) const { *at(lane, word) = v; }
    __device__ __forceinline__ int row(int step) const { return step * (32 / WORDS) + lane / WORDS; }
    __device__ __forceinline__ int word() const { return lane % WORDS; }
    __device__ __forceinline__ uint4 get(int step) const { return *at(row(step), word()); }
};

// ------------------------------------------------------------------- kernel

// Which tile is the i-th: groups of `group` m tiles, within a group n by n.  The
// host has made sure that their number fits 31 bits.
struct TcTiles {
    uint32_t mt, nt, group, splits, kblocks;
    __device__ __forceinline__ TcTiles(const TcShape &s, int columns)
    {
        const int c = s.dyn_m || s.dyn_k ? max(*s.count, 1) : 0;
        const int m = s.dyn_m ? c : s.m, k = s.dyn_k ? c : s.k;
        mt = (m + kTcTile - 1) / kTcTile;
        nt = (s.n + columns - 1) / columns;
        kblocks = (k + kTcK - 1) / kTcK;
        group = s.group;
        splits = tc_parts_of(s, m);
    }
    __device__ __forceinline__ uint32_t count() const { return mt * nt * splits; }
    __device__ __forceinline__ void at(uint32_t i, int &m, int &n, int &part, int &k0, int &k1) const
    {
        const uint32_t tiles = mt * nt;
        uint32_t t = i;
        part = 0, k0 = 0, k1 = (int)kblocks;
        if(splits > 1) {
            part = (int)(i / tiles);
            t = i - part * tiles;
            k0 = (int)((uint64_t)kblocks * part / splits);
            k1 = (int)((uint64_t)kblocks * (part + 1) / splits);
        }
        const uint32_t per = group * nt, g = t / per;
        const uint32_t rows = min(group, mt - g * group), r = t - g * per, c = r / rows;
        m = (int)(g * group + r - c * rows);
        n = (int)c;
    }
};

// Epi: the epilogue.  common() is what all tiles share; begin(common, row, col,
// part) gives a thread's state for its row of a tile and the kTcColumns columns from
// col; columns(common, state, row, col, v, staging) gets 32 columns at a time, all
// lanes of a warp together; end(state, row, col, acc, shared) closes them, where
// `shared` is the staging memory of all epilogue warps.  Rows and columns beyond the matrix come too and are for the epilogue to
// leave out.
template <bool A_MN, bool B_MN, int NH, typename Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTcThreads, 1)
    tc_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const TcShape shape, const Epi epi)
{
    constexpr int kTcStages = tc_stages(NH), kStageBytes = tc_stage_bytes(NH);
    extern __shared__ char smem_raw[];
    __shared__ __align__(8) uint64_t full[kTcStages], empty[kTcStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int dead_word;
    volatile int *dead = &dead_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;

    if(threadIdx.x == 0) {
        dead_word = 0;
        for(int i = 0; i < kTcStages; i++) {
            mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&empty[i]), 1);
        }
        for(int i = 0; i < 2; i++) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 2 * kTcEpilogue);  // the epilogue warps of both CTAs
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if(warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(&tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *(volatile uint32_t *)&tmem_slot;
    lm_after_previous();

    const TcTiles tiles(shape, NH * kTcTile);
    const uint32_t total = tiles.count(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if(warp == 0 && lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for(uint32_t i = pair; ok && i < total; i += pairs) {
            int m, n, part, k0, k1;
            tiles.at(i, m, n, part, k0, k1);
            const int am = m * kTcTile + (int)rank * kTcHalf, bn = n * NH * kTcTile + (int)rank * kTcHalf;
            for(int kb = k0; kb < k1; kb++) {
                if(!(ok = mbar_wait(smem_u32(&empty[stage]), phase ^ 1, dead)))
                    break;
                const uint32_t a = base + stage * kStageBytes;
                const uint32_t bar = map_to(smem_u32(&full[stage]), 0);
                if(rank == 0)
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                                     smem_u32(&full[stage])),
                                 "r"(2 * kStageBytes)
                                 : "memory");
                const int k = kb * kTcK;
                if(A_MN) {
                    tma_load(a, &map_a, am, shape.a_row0 + k, bar);
                    tma_load(a + kTcOperand / 2, &map_a, am + 64, shape.a_row0 + k, bar);
                } else {
                    tma_load(a, &map_a, k, shape.a_row0 + am, bar);
                }
#pragma unroll
                for(int h = 0; h < NH; h++) {
                    const uint32_t b = a + (1 + h) * kTcOperand;
                    const int at = bn + h * kTcTile;
                    if(B_MN) {
                        tma_load(b, &map_b, at, shape.b_row0 + k, bar);
                        tma_load(b + kTcOperand / 2, &map_b, at + 64, shape.b_row0 + k, bar);
                    } else {
                        tma_load(b, &map_b, k, shape.b_row0 + at, bar);
                    }
                }
                if(++stage == kTcStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        if(!ok)  // let the copies in flight land before the CTA's memory goes
            for(int i = 0; i < 1000; i++)
                __nanosleep(1000);
    } else if(warp == 1 && lane == 0 && rank == 0) {
        constexpr uint32_t idesc = instruction_desc<A_MN, B_MN>();
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        // one stage's product into accumulator `to`, with B's half h
        auto multiply = [&](int of, int h, int to, bool add) {
            const uint32_t a = base + of * kStageBytes;
            uint64_t da = operand_desc<A_MN>(a), db = operand_desc<B_MN>(a + (1 + h) * kTcOperand);
#pragma unroll
            for(int s = 0; s < kTcK / 16; s++) {
                mma(tmem + to * kTcTile, da, db, idesc, add || s);
                da += k_step<A_MN>();
                db += k_step<B_MN>();
            }
        };
        auto arrived = [&](int of, uint32_t parity) {
            const bool got = mbar_wait(smem_u32(&full[of]), parity, dead);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return got;
        };
        auto next = [&](int &of, uint32_t &parity) {
            if(++of == kTcStages) {
                of = 0;
                parity ^= 1;
            }
        };
        auto emptied = [&](int which, uint32_t parity) {
            const bool got = mbar_wait(smem_u32(&acc_empty[which]), parity, dead);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return got;
        };
        for(uint32_t i = pair; ok && i < total; i += pairs) {
            int m, n, part, k0, k1;
            tiles.at(i, m, n, part, k0, k1);
            if constexpr(NH == 1) {
                if(!(ok = emptied(acc, acc_phase ^ 1)))
                    break;
                for(int kb = k0; kb < k1; kb++) {
                    if(!(ok = arrived(stage, phase)))
                        break;
                    multiply(stage, 0, acc, kb > k0);
                    mma_commit(smem_u32(&empty[stage]));
                    next(stage, phase);
                }
                if(ok)
                    mma_commit(smem_u32(&acc_full[acc]));
                if(++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            } else {
                // Both accumulators are one tile's.  At its start and at its end the
                // first half runs ahead by as many stages as there are: the epilogue of
                // one half then runs beside the main loop of the other.
                const int all = k1 - k0, head = min(all, kTcStages), tail = min(all - head, kTcStages);
                int done = 0;
                auto skewed = [&](int count, bool first) {
                    int of = stage;
                    uint32_t parity = phase;
                    for(int j = 0; ok && j < count; j++) {
                        if((ok = arrived(of, parity)))
                            multiply(of, 0, 0, !first || j);
                        next(of, parity);
                    }
                    if(ok && done + count == all)
                        mma_commit(smem_u32(&acc_full[0]));
                    if(first)
                        ok = ok && emptied(1, acc_phase ^ 1);
                    for(int j = 0; ok && j < count; j++) {
                        multiply(stage, 1, 1, !first || j);
                        mma_commit(smem_u32(&empty[stage]));
                        next(stage, phase);
                    }
                    done += count;
                    if(ok && done == all)
                        mma_commit(smem_u32(&acc_full[1]));
                };
                if(!(ok = emptied(0, acc_phase ^ 1)))
                    break;
                skewed(head, true);
                for(int j = head; ok && j < all - tail; j++) {
                    if(!(ok = arrived(stage, phase)))
                        break;
                    multiply(stage, 0, 0, true);
                    multiply(stage, 1, 1, true);
                    mma_commit(smem_u32(&empty[stage]));
                    next(stage, phase);
                    done++;
                }
                if(ok && tail)
                    skewed(tail, false);
                acc_phase ^= 1;
            }
        }
    } else if(warp >= 4) {
        const int quad = warp & 3, side = (warp - 4) >> 2;
        char *const shared = smem_raw + (base - smem_u32(smem_raw)) + kTcStages * kStageBytes;
        char *const staging = shared + (warp - 4) * tc_staging(NH);
        const auto common = epi.common();
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for(uint32_t i = pair; i < total; i += pairs) {
            int m, n, part, k0, k1;
            tiles.at(i, m, n, part, k0, k1);
            const int row = m * kTcTile + (int)rank * kTcHalf + quad * 32 + lane;
#pragma unroll 1
            for(int h = 0; h < NH; h++) {
                const int col = (n * NH + h) * kTcTile + side * kTcColumns;
                const uint32_t from =
                    tmem + ((uint32_t)(quad * 32) << 16) + acc * kTcTile + side * kTcColumns;
                auto state = epi.begin(common, row, col, part);  // its loads run during the wait
                ok = ok && mbar_wait(smem_u32(&acc_full[acc]), acc_phase, dead);
                ok = __all_sync(0xffffffffu, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                for(int c = 0; c < kTcColumns; c += 32) {
                    float v[32];
                    tmem_load(from + c, v);
                    tmem_wait(v);
                    if(!ok || k1 == k0)
                        no_result(v, ok);
                    epi.columns(common, state, row, col + c, v, staging);
                }
                epi.end(state, row, col, acc, shared);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if(lane == 0)
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                     map_to(smem_u32(&acc_empty[acc]), 0))
                                 : "memory");
                if(++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1;
                }
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if(warp == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// --------------------------------------------------------------------- host

// Tensor map of a row-major fp16 matrix, boxes of 64 columns x box_rows rows.
inline bool tc_map(CUtensorMap *map, const void *p, size_t rows, size_t cols, size_t stride,
                   unsigned box_rows)
{
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                               const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) !=
               cudaSuccess ||
           q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return (Encode)fn;
    }();
    if(!encode)
        return false;
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {stride * 2};
    const cuuint32_t box[2] = {64, box_rows}, steps[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(p), dims, strides, box,
                  steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows of a box: an operand's 128 rows when k is contiguous, 64 k otherwise
constexpr unsigned tc_box(bool mn) { return mn ? kTcK : kTcHalf; }

// Whether a product of two MN-major operands is faster in wide tiles, which fetch a
// quarter less per flop but have four stages of k instead of five, and both
// accumulators, so that a tile's epilogue overlaps less of the next one.  That pays for
// itself with a long k (grad_weight's product, m = 16384, n = 4096, as many turns both ways;
// us narrow and wide: k = 512 63 and 76, 1024 110 and 113, 1280 125 and 125, 1536 146 and
// 143, 2048 202 and 194, 8192 803 and 717).  There are half as many wide tiles to spread
// over the pairs, so the turns that the pairs make, counted in narrow tiles, can grow:
// by 5 % is as much as a k of 2048 allows (48640 x 2048: 305 and 303), by 9 % from 4096 on
// (15360 x 4096, 8 % more turns: k = 2048 188 and 191, 4096 360 and 356, 8192 747 and 708).
// K-major operands gain nothing, and their callers keep to narrow tiles (losses of 8192 x
// 128000, 512 columns: 876 us narrow, 982 wide).
inline bool tc_wide(long long m, long long n, long long k, int sms)
{
    if(k < 1536)
        return false;
    const long long mt = (m + kTcTile - 1) / kTcTile, pairs = sms / 2 > 0 ? sms / 2 : 1;
    const long long narrow = mt * ((n + kTcTile - 1) / kTcTile);
    const long long wide = mt * ((n + 2 * kTcTile - 1) / (2 * kTcTile));
    const long long turns = (narrow + pairs - 1) / pairs, turns2 = 2 * ((wide + pairs - 1) / pairs);
    return 100 * turns2 <= (k < 4096 ? 105 : 109) * turns;
}

template <bool A_MN, bool B_MN, int NH, typename Epi>
bool tc_launch(const CUtensorMap &a, const CUtensorMap &b, const TcShape &s, const Epi &epi, int sms,
               cudaStream_t st, bool next)
{
    auto *kernel = tc_gemm_kernel<A_MN, B_MN, NH, Epi>;
    static std::atomic<uint64_t> allowed{0};
    if(!lm_allow_smem(kernel, tc_smem(NH), allowed))
        return false;
    // (as many pairs as planned for, where the device may find more parts)
    const long long tiles = s.splits > 1 && s.dyn_m
                                ? kTcPlanPairs
                                : (s.m + kTcTile - 1ll) / kTcTile *
                                      ((s.n + NH * kTcTile - 1ll) / (NH * kTcTile)) * s.splits;
    const long long pairs = tiles < sms / 2 ? tiles : sms / 2;
    if(tiles > 0x7fffffff)
        return false;
    if(next)
        lm_launch_next(kernel, (unsigned)(2 * pairs), kTcThreads, tc_smem(NH), st, a, b, s, epi);
    else
        kernel<<<(unsigned)(2 * pairs), kTcThreads, tc_smem(NH), st>>>(a, b, s, epi);
    return true;
}

}  // namespace b200
