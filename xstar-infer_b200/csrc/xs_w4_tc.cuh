// Products with 4-bit weights on the tensor core, for larger batches: out = x W^T (or act(x Wg^T) * (x Wu^T)).
//
// tcgen05.mma with the WEIGHTS as its M rows, taken from TMEM, and the tokens as its N columns, taken from shared memory.  The codes
// arrive by TMA as they lie in memory; sixteen warps turn them into f16, thread = weight row, and store them with tcgen05.st
// straight into TMEM columns, so a dequantised weight never passes through shared memory, whose bandwidth the tokens need.
// Weights in TMEM also make the group scale a scalar of the thread.  Tokens, and the scales of a weight row, have been given a
// common exponent (xs_w4_prepare.cuh); q - z is exact, and times its scale it is rounded once, to the eleven bits of f16.
// Sums are f32 in TMEM; the epilogue multiplies them by the powers of two of their row and token.
//
// CG = 2 pairs two SMs on a 256 x 256 tile (cta_group::2): each dequantises its 128 rows and loads its 128 tokens, so the
// traffic out of L2 and the dequantisation per product halve against two 128 x 256 tiles.  CG = 1 serves smaller batches, where
// the weights' bytes are the work: tiles of 128 rows x up to 128 tokens, K split over a cluster of C blocks that sum through
// distributed shared memory when there are too few tiles for the SMs.
//
// Warps: 0, 3 token loads, alternate blocks (3 owns the TMEM allocation) | 1 MMA | 2 code loads | 4..19 dequantisation (four
// warpgroups, one for each stage of operands, lane quarter = warp % 4) | 20..27 epilogue (lane quarter = warp % 4, half of the
// token columns each).
//
// An operand block is 128 columns because every hand-over costs its roles a few hundred cycles (a poll of a barrier about 110, a
// parked wait about 300, an expect or a load 100 each): with 64 columns one loading thread took 600 cycles a block, whatever the
// tile, and everybody else waited for it.
//
// Measured: 4096 x 4096 x 8192 194 us with the preparation at 1965 MHz, 1.42 PFLOP/s of the 1.66 that the library reaches there, and 226 us
// in a long run under the power cap (about 1480 MHz), 1.22 of 1.37; 8192 x 8192 x 8192 739 us (1.49).  With few tokens the conversion of the codes is the work, 0.42 to 0.46 us for a block of 128 x
// 128 weights: the sixteen warps use half of the issue slots, the tensor pipe is active 19 % of the time, and six stages instead of four gain 1 %.
// 45 x 4096 x 20480 takes 38 us, 83 x 11264 x 4096 25 us, where the bytes would take 8 and 5.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"
#include "xs_w4_common.cuh"
#include "xs_w4_prepare.cuh"

namespace xs {

constexpr int kTcDequantWarps = 16;
constexpr int kTcEpilogueWarp = 4 + kTcDequantWarps;
constexpr int kTcThreads = 32 * (kTcEpilogueWarp + 8);
constexpr int kTcRows = 128;       // weight rows (TMEM lanes) of a block's tile
constexpr int kTcBlockK = 128;     // columns of one operand block: two 128-byte pieces of a token's row
constexpr int kTcRawBlocks = 2;    // operand blocks in one load of codes: 256 columns, 128 bytes a row
constexpr int kTcRawBytes = kTcRows * 128;
constexpr int kTcStages = 4;       // operand blocks in flight: TMEM columns of weights, shared memory of tokens
constexpr int kTcAccCol = kTcStages * (kTcBlockK / 2);

__host__ __device__ constexpr int tc_x_bytes(int cg, int n_tile)
{
    return n_tile / cg * kTcBlockK * 2;
}
// loads of codes in flight: what the tokens leave of shared memory
__host__ __device__ constexpr int tc_raw_stages(int cg, int n_tile)
{
    return n_tile / cg >= 128 ? 4 : 8;
}
__host__ __device__ constexpr int tc_smem_bytes(int cg, int n_tile)
{
    return 1024 + tc_raw_stages(cg, n_tile) * kTcRawBytes + kTcStages * tc_x_bytes(cg, n_tile) + 512 + 2 * 256 * 4; // barriers; factors of two tiles' tokens
}

__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
template <int CG>
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
}
// arrive on the barrier (CG = 2: on that of both blocks) when the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void tc_done(uint64_t *bar)
{
    if constexpr (CG == 1)
        tc_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"(static_cast<uint16_t>(3))
                     : "memory");
}
// the address of the leading block's copy of a barrier
__device__ __forceinline__ uint32_t leader_addr(uint64_t *bar)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
    return a;
}
template <int CG>
__device__ __forceinline__ void tc_arrive_leader(uint64_t *bar)
{
    if constexpr (CG == 1)
        mbar_arrive(bar);
    else
        // what is handed over lies in TMEM, ordered by the tcgen05 fences around the barrier; a release at cluster scope would
        // hold the warp for more than a thousand cycles
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
}
// 2-D tiled load into this block's shared memory; CG = 2: the bytes are counted on the leading block's barrier
template <int CG>
__device__ __forceinline__ void tc_load_x(void *dst, const CUtensorMap *m, uint64_t *bar, int32_t c0, int32_t c1, uint64_t policy)
{
    if constexpr (CG == 1)
        tma_load_2d(dst, m, bar, c0, c1, policy);
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
                     " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
                     "l"(reinterpret_cast<uint64_t>(m)), "r"(leader_addr(bar)), "r"(c0), "r"(c1), "l"(policy)
                     : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait()
{
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel)
{
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// Byte c of a word of codes as a pair: its low nibble (the even column) in the first half, sixteen times its high nibble in the
// second.  The upper byte of each half is the sign of a low nibble's byte, replicated: zero.
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int c)
{
    const uint32_t low = word & 0x0f0f0f0fu, high = word & 0xf0f0f0f0u;
    return prmt(low, high, c | (8 | c) << 4 | (4 + c) << 8 | (8 | c) << 12);
}
// Barrier 1 among the eight epilogue warps; the conjunction of their predicates.
__device__ __forceinline__ bool named_barrier_and(bool ok)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(ok ? 1u : 0u) : "memory");
    return r != 0;
}

// What w4_prepare_kernel made of the scales and tokens, and how the result is written.
struct TcOperands {
    const uint16_t *scales; // f16 (rows, pitch)
    const uint8_t *zeros;   // (rows, pitch) or null: 8
    const float *row;       // factor of a weight row's sums; negative: its scales are of wide range
    const float *token;     // factor of a token
    int pitch;
};

struct TcShape {
    int n_out, T, K, G_log; // G_log: log2 of the group
    int w_tiles, t_tiles;   // tiles along the features and along the tokens
    int split;              // blocks that share a tile (CG = 1)
    int f0;                 // first feature of this launch
};

// Work item -> tile.  Eight token tiles go with each weight tile before the next one, so that what runs at one time shares both.
__device__ __forceinline__ void tc_tile(const TcShape &s, int item, int &wt, int &tt)
{
    constexpr int kGroup = 8;
    const int per = kGroup * s.w_tiles, g = item / per, first = g * kGroup;
    const int width = s.t_tiles - first < kGroup ? s.t_tiles - first : kGroup, r = item - g * per;
    wt = r / width;
    tt = first + r - wt * width;
}

// The factor of a weight row in two: a sum is multiplied by what shrinks it, then by its token's factor, then by what makes it grow, so that
// neither a token near the largest number against a row of small scales nor the reverse leaves the range of f32 on the way.
struct RowFactor {
    float shrink, grow;
    __device__ __forceinline__ explicit RowFactor(float f) : shrink(fminf(fabsf(f), 1.0f)), grow(fmaxf(fabsf(f), 1.0f)) {}
    __device__ __forceinline__ float of(float v, float token) const
    {
        return v * shrink * token * grow;
    }
};
// One element of the result: v, or act(v) u; in bf16, or in f32 for the product that follows.
template <bool GATED, typename Out>
__device__ __forceinline__ Out tc_result(int act, float v, float u)
{
    if constexpr (GATED)
        v = w4_activation(v, act) * u;
    if constexpr (sizeof(Out) == 4)
        return v;
    else
        return __float2bfloat16_rn(v);
}

template <int CG, int N_TILE, bool GATED, typename Out>
__global__ void __launch_bounds__(kTcThreads, 1)
w4_tc_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const TcOperands w, Out *__restrict__ out,
             const TcShape s, int act, int32_t *__restrict__ status)
{
    constexpr int RAW = tc_raw_stages(CG, N_TILE), X_BYTES = tc_x_bytes(CG, N_TILE);
    constexpr int FEATURES = GATED ? kTcRows / 2 : kTcRows; // of a block
    constexpr int NBUF = N_TILE <= 128 ? 2 : 1;             // accumulators
    constexpr uint32_t IDESC = make_idesc(0, 0, kTcRows * CG, N_TILE); // f16

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *x_smem = smem + RAW * kTcRawBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(x_smem + kTcStages * X_BYTES);
    uint64_t *raw_full = bars, *raw_empty = raw_full + RAW;
    uint64_t *full = raw_empty + RAW, *empty = full + kTcStages; // full: both operands of a block are there
    uint64_t *acc_full = empty + kTcStages, *acc_empty = acc_full + NBUF;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + NBUF);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    float *token_smem = reinterpret_cast<float *>(bars) + 128; // [tile parity][256]

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31; // warp: known to be uniform
    const int rank = CG > 1 || s.split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const bool leader = CG == 1 || rank == 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < RAW; i++) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 8); // two blocks, four warps each
        }
        for (int i = 0; i < kTcStages; i++) {
            mbar_init(&full[i], 4 * CG + 1); // the dequantising warps, and the token load with its bytes
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < NBUF; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 8 * CG);
        }
        *abort_flag = 0;
        fence_mbar_init();
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_x);
    }
    if (warp == 3) {
        if constexpr (CG == 1) {
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    if constexpr (CG > 1)
        cluster_barrier(); // the other block arrives on barriers of this one
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Everything above touches only shared memory and TMEM.  The codes may be loaded at once: what runs before this kernel in its
    // stream is the preparation of the tokens (or the product that made them), and the codes were there before that began.
    if (warp != 2)
        pdl_wait();

    const int all_raw = (s.K + kTcRawBlocks * kTcBlockK - 1) / (kTcRawBlocks * kTcBlockK);
    const int raw_per = (all_raw + s.split - 1) / s.split;
    const int raw0 = CG == 1 ? rank * raw_per : 0, raw1 = min(raw0 + raw_per, all_raw); // this block's loads of codes
    const int kb0 = raw0 * kTcRawBlocks, kb1 = min(raw1 * kTcRawBlocks, (s.K + kTcBlockK - 1) / kTcBlockK);
    const int n_kb = kb1 - kb0;
    const int per_item = CG > 1 ? CG : s.split; // blocks working on one item
    const int items = s.w_tiles * s.t_tiles, item0 = blockIdx.x / per_item, item_step = gridDim.x / per_item;
    // first feature of this block's part of a weight tile, first token of its part of a token tile
    const int block_feature = CG > 1 ? rank * FEATURES : 0, block_token = CG > 1 ? rank * (N_TILE / CG) : 0;

    bool ok = true;
    if ((warp == 0 || warp == 3) && lane == 0) {
        const uint64_t policy = policy_evict_last();
        uint32_t n = 0;
        for (int item = item0; item < items && ok; item += item_step) {
            int wt, tt;
            tc_tile(s, item, wt, tt);
            const int token = tt * N_TILE + block_token;
            for (int kb = kb0; kb < kb1; kb++, n++) {
                if ((n & 1) != (warp == 3 ? 1u : 0u))
                    continue;
                const uint32_t st = n % kTcStages;
                if (!mbar_wait(&empty[st], ((n / kTcStages) & 1) ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                if (leader)
                    mbar_arrive_expect_tx(&full[st], X_BYTES * CG);
                tc_load_x<CG>(x_smem + st * X_BYTES, &tmap_x, &full[st], kb * kTcBlockK, token, policy);
                tc_load_x<CG>(x_smem + st * X_BYTES + X_BYTES / 2, &tmap_x, &full[st], kb * kTcBlockK + 64, token, policy);
            }
        }
    } else if (warp == 2 && lane == 0) {
        const uint64_t policy = s.t_tiles > 1 ? policy_evict_last() : policy_evict_first();
        uint32_t n = 0;
        for (int item = item0; item < items && ok; item += item_step) {
            int wt, tt;
            tc_tile(s, item, wt, tt);
            for (int r = raw0; r < raw1; r++, n++) {
                const uint32_t st = n % RAW;
                // The ring is full, and empties once the other warps begin, behind the kernel before this one: however long that takes, it is
                // not for the bounded wait below to count.
                if (n == RAW)
                    pdl_wait();
                if (!mbar_wait(&raw_empty[st], ((n / RAW) & 1) ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(&raw_full[st], kTcRawBytes);
                tma_load_3d(smem + st * kTcRawBytes, &tmap_w, &raw_full[st], r * 128, s.f0 + wt * FEATURES * CG + block_feature, 0, policy);
            }
        }
    } else if (warp == 1 && leader) {
        // The whole warp walks the loop and one elected lane issues, so that addresses and descriptors stay in uniform registers;
        // the waits poll without parking the warp.  What this warp does between blocks is time the tensor pipe may stand still.
        const bool elected = elect_one();
        const uint64_t desc0 = make_desc_sw128(smem_u32(x_smem));
        uint32_t st = 0, ph = 0, use = 0;
        for (int item = item0; item < items && ok; item += item_step, use++) {
            const uint32_t buf = use % NBUF, acc = tmem + kTcAccCol + buf * N_TILE;
            if (!mbar_spin_wait(&acc_empty[buf], ((use / NBUF) & 1) ^ 1, abort_flag)) {
                ok = false;
                break;
            }
            for (int kb = 0; kb < n_kb; kb++) {
                if (!mbar_spin_wait(&full[st], ph, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t db = desc0 + st * (X_BYTES >> 4);
                const uint32_t a = tmem + st * (kTcBlockK / 2);
                if (elected) {
#pragma unroll
                    for (int kk = 0; kk < kTcBlockK / 16; kk++)
                        tc_mma<CG>(acc, a + kk * 8, db + (kk / 4) * (X_BYTES / 2 >> 4) + 2 * (kk % 4), IDESC, (kb | kk) ? 1u : 0u);
                    tc_done<CG>(&empty[st]);
                }
                if (++st == kTcStages) {
                    st = 0;
                    ph ^= 1;
                }
            }
            if (ok && elected)
                tc_done<CG>(&acc_full[buf]);
        }
    } else if (warp >= 4 && warp < kTcEpilogueWarp) {
        // Of the operand blocks, counted over all items, this warpgroup has every fourth, so that one warpgroup alone fills a stage.
        // A parity tells one use of a stage from the next, not from the one after that: nobody may come to a stage two uses early.
        const int wg = (warp - 4) >> 2, q = warp & 3;
        // the row of the codes (as the load laid them out) that this thread's TMEM lane holds; GATED: 16 gate rows, then their 16 up rows
        const int raw_row = GATED ? (lane >> 4) * 64 + q * 16 + (lane & 15) : q * 32 + lane;
        const int feature = GATED ? q * 16 + (lane & 15) : raw_row;
        const uint32_t raw_addr = smem_u32(smem) + raw_row * 128, swz = (raw_row & 7) << 4;
        // Groups of a block (4, 2 or 1) with their scales and zero points, loaded two of this warpgroup's blocks ahead.
        const int per_block = 1 << (7 - s.G_log);
        const bool zeros = w.zeros != nullptr;
        struct Scales {
            uint2 s;    // 16 bits each
            uint32_t z; // 8 bits each
        };
        auto row_at = [&](int item) {
            int wt, tt;
            tc_tile(s, item, wt, tt);
            return static_cast<size_t>(min(s.f0 + wt * FEATURES * CG + block_feature + feature, s.n_out - 1)) + (GATED && lane >= 16 ? s.n_out : 0);
        };
        int ld_item = item0, ld_kb = wg; // kb here and below: within the item
        for (; ld_kb >= n_kb; ld_kb -= n_kb)
            ld_item += item_step;
        int item = ld_item, kb = ld_kb;
        size_t ld_row = ld_item < items ? row_at(ld_item) * w.pitch : 0; // first group of the row
        auto load_scales = [&]() {
            Scales r;
            r.s = make_uint2(0, 0);
            r.z = 0;
            if (ld_item < items) {
                const uint16_t *sp = w.scales + ld_row + (kb0 + ld_kb) * per_block;
                const uint8_t *zp = w.zeros + ld_row + (kb0 + ld_kb) * per_block;
                if (per_block == 4)
                    r.s = __ldg(reinterpret_cast<const uint2 *>(sp));
                else if (per_block == 2)
                    r.s.x = __ldg(reinterpret_cast<const uint32_t *>(sp));
                else
                    r.s.x = __ldg(sp);
                if (zeros)
                    r.z = per_block == 4 ? __ldg(reinterpret_cast<const uint32_t *>(zp)) : per_block == 2 ? __ldg(reinterpret_cast<const uint16_t *>(zp)) : __ldg(zp);
                ld_kb += 4;
                if (ld_kb >= n_kb) {
                    for (; ld_kb >= n_kb; ld_kb -= n_kb)
                        ld_item += item_step;
                    if (ld_item < items)
                        ld_row = row_at(ld_item) * w.pitch;
                }
            }
            return r;
        };
        Scales cur, next, after;
#pragma unroll 1
        for (int i = 0; i < 2; i++) {
            next = after;
            after = load_scales();
        }
        const uint32_t dst = tmem + (static_cast<uint32_t>(q * 32) << 16) + wg * (kTcBlockK / 2);
        uint32_t free = 1, nr = (item - item0) / item_step * (raw1 - raw0); // parity of the stage's release; loads of codes before this item
        while (item < items && ok) {
            // Zero point 8 and scales of narrow range in the warp's 32 rows: one multiply-add a pair, n (2^15 s) 2^-24 - 8 s 2^-9, whose
            // parts are exact; else (q - z) 2^-9 first, exactly, then times s.
            const bool one_step = !zeros && __all_sync(0xffffffffu, __ldg(w.row + row_at(item)) > 0.0f);
            for (; kb < n_kb; kb += 4, free ^= 1) {
                const uint32_t rc = nr + (kb >> 1), rs = rc % RAW;
                const bool is_free = mbar_test_wait(&empty[wg], free), raw_there = mbar_test_wait(&raw_full[rs], (rc / RAW) & 1);
                cur = next;
                next = after;
                after = load_scales();
                // In this order: once the stage is free, the blocks up to four back have been multiplied, so the use of this place of
                // the codes' ring before this one is over, and the parity cannot be that of the one before it.
                ok = __all_sync(0xffffffffu, is_free || mbar_wait(&empty[wg], free, abort_flag));
                if (ok)
                    ok = __all_sync(0xffffffffu, (is_free && raw_there) || mbar_wait(&raw_full[rs], (rc / RAW) & 1, abort_flag));
                if (!ok)
                    break;
                tc_fence_after();
                const uint32_t codes = raw_addr + rs * kTcRawBytes;
#pragma unroll
                for (int h = 0; h < 4; h++) { // 32 columns: one 16-byte piece of codes, one group
                    const int e = (h * per_block) >> 2;
                    // past the end of K the codes read as zero, and so must the weight, whatever the zero point
                    uint32_t sv = prmt(cur.s.x, cur.s.y, 0x1010u + 0x2222u * e);
                    if ((kb0 + kb) * kTcBlockK + h * 32 >= s.K)
                        sv = 0;
                    const uint4 qv = lds128(codes + ((((kb & 1) * 4 + h) << 4) ^ swz));
                    const uint32_t words[4] = {qv.x, qv.y, qv.z, qv.w};
                    uint32_t a[16];
                    if (one_step) {
                        const uint32_t mul = f16x2_mul(sv, kW4PairMul), add = f16x2_mul(sv, kW4HalfMinus8);
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                a[j * 4 + c] = f16x2_fma(w4_pair(words[j], c), mul, add);
                    } else {
                        const uint32_t mz = zeros ? w4_half_minus_zero((cur.z >> (8 * e)) & 15u) : kW4HalfMinus8;
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                a[j * 4 + c] = f16x2_mul(f16x2_fma(w4_pair(words[j], c), kW4PairMul, mz), sv);
                    }
                    tmem_st16(dst + h * 16, a);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    tc_arrive_leader<CG>(&full[wg]);
                    mbar_arrive(&raw_empty[rs]);
                    if (kb + 1 == n_kb && !(kb & 1))
                        mbar_arrive(&raw_empty[rs]); // the load's second block is not there
                }
            }
            for (; kb >= n_kb; kb -= n_kb) {
                item += item_step;
                nr += raw1 - raw0;
            }
        }
    } else if (warp >= kTcEpilogueWarp) {
        const int q = warp & 3, part = (warp - kTcEpilogueWarp) >> 2;
        constexpr int COLS = N_TILE / 2; // of this warp
        const int lane_feature = GATED ? q * 16 + (lane & 15) : q * 32 + lane;
        uint32_t use = 0;
        for (int item = item0; item < items; item += item_step, use++) {
            int wt, tt;
            tc_tile(s, item, wt, tt);
            const uint32_t buf = use % NBUF;
            // the factors of this tile's tokens, into the place the tile before last has left
            float *factor = token_smem + (use & 1) * 256;
            if (const int j = threadIdx.x - 32 * kTcEpilogueWarp; j < N_TILE)
                factor[j] = __ldg(w.token + min(tt * N_TILE + j, s.T - 1));
            // one warp asks, sleeping in between, and the others wait at a barrier that costs no issue slots
            if (warp == kTcEpilogueWarp)
                ok = warp_sleep_wait(&acc_full[buf], (use / NBUF) & 1, abort_flag, n_kb);
            if (!named_barrier_and(ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + kTcAccCol + buf * N_TILE + part * COLS;
            const int feature = s.f0 + wt * FEATURES * CG + block_feature + lane_feature, token0 = tt * N_TILE + part * COLS;
            const int f0 = min(feature, s.n_out - 1);
            const RowFactor row_f(__ldg(w.row + f0)), row_u(GATED ? __ldg(w.row + s.n_out + f0) : 0.0f);
            if (CG == 1 && s.split > 1) {
                // the sums of this block's slice of K, [token][lane], over the operand ring, which nothing reads or fills any more
                float *red = reinterpret_cast<float *>(smem);
                for (int c = 0; c < COLS; c += 16) {
                    uint32_t v[16];
                    tmem_ld16(acc + c, v);
                    tmem_ld_wait_16(v);
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        red[(part * COLS + c + i) * kTcRows + q * 32 + lane] = __uint_as_float(v[i]);
                }
                break; // one tile a block; summed below
            }
            const bool whole = token0 + COLS <= s.T && feature - lane_feature + FEATURES <= s.n_out;
            Out *o = out + static_cast<size_t>(token0 + (GATED && lane >= 16 ? 1 : 0)) * s.n_out + feature;
            for (int c = 0; c < COLS; c += 16) {
                uint32_t v[16];
                tmem_ld16(acc + c, v);
                float tf[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(factor + part * COLS + c + i);
                    tf[i] = f.x, tf[i + 1] = f.y, tf[i + 2] = f.z, tf[i + 3] = f.w;
                }
                tmem_ld_wait_16(v);
                if (c + 16 == COLS) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0)
                        tc_arrive_leader<CG>(&acc_empty[buf]);
                }
                if constexpr (GATED) {
                    // lanes 0..15 hold gate sums and 16..31 the up sums of the same features: of each pair of tokens the first half
                    // of the warp finishes the even one, the second half the odd one
                    const bool up = lane >= 16;
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float even = __uint_as_float(v[i]), uneven = __uint_as_float(v[i + 1]);
                        const float got = __shfl_xor_sync(0xffffffffu, up ? even : uneven, 16), f = up ? tf[i + 1] : tf[i];
                        const int t = token0 + c + i + (up ? 1 : 0);
                        if (whole || (feature < s.n_out && t < s.T))
                            *o = tc_result<true, Out>(act, row_f.of(up ? got : even, f), row_u.of(up ? uneven : got, f));
                        o += 2 * static_cast<size_t>(s.n_out);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        if (whole || (feature < s.n_out && token0 + c + i < s.T))
                            *o = tc_result<false, Out>(act, row_f.of(__uint_as_float(v[i]), tf[i]), 0.0f);
                        o += s.n_out;
                    }
                }
            }
        }
    }
    if (!ok) {
        *abort_flag = 1;
        atomicOr(status, kStatusWaitTimeout);
    }
    __syncwarp();
    if (warp == 2)
        pdl_wait();
    if (CG == 1 && s.split > 1)
        cluster_barrier();
    if (CG == 1 && s.split > 1) {
        // this block's tokens of the tile, four features a thread: the slices' sums in the order of the slices
        int wt, tt;
        tc_tile(s, item0, wt, tt);
        const uint32_t red = smem_u32(smem);
        const int share = N_TILE / s.split;
        for (int i = threadIdx.x; i < share * (FEATURES / 4); i += kTcThreads) {
            const int c = rank * share + i / (FEATURES / 4), f = i % (FEATURES / 4) * 4, feature = s.f0 + wt * FEATURES + f, token = tt * N_TILE + c;
            if (feature >= s.n_out || token >= s.T)
                continue;
            const uint32_t at = red + (c * kTcRows + (GATED ? (f >> 4) * 32 + (f & 15) : f)) * 4;
            float4 v[8], u[GATED ? 8 : 1];
#pragma unroll
            for (int r = 0; r < 8; r++)
                if (r < s.split) {
                    v[r] = ld_cluster_f32x4(at, r);
                    if constexpr (GATED)
                        u[r] = ld_cluster_f32x4(at + 64, r);
                }
            float sv[4] = {}, su[4] = {};
#pragma unroll
            for (int r = 0; r < 8; r++)
                if (r < s.split) {
                    sv[0] += v[r].x, sv[1] += v[r].y, sv[2] += v[r].z, sv[3] += v[r].w;
                    if constexpr (GATED)
                        su[0] += u[r].x, su[1] += u[r].y, su[2] += u[r].z, su[3] += u[r].w;
                }
            const float t = token_smem[c]; // the one tile's
            Out *o = out + static_cast<size_t>(token) * s.n_out + feature;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (feature + j < s.n_out)
                    o[j] = tc_result<GATED, Out>(act, RowFactor(__ldg(w.row + feature + j)).of(sv[j], t),
                                                 GATED ? RowFactor(__ldg(w.row + s.n_out + feature + j)).of(su[j], t) : 0.0f);
        }
    }
    if (*abort_flag)
        for (int i = 0; i < 64; i++)
            __nanosleep(4096); // copies in flight land before the shared memory is given up
    tc_fence_before();
    if (CG > 1 || s.split > 1)
        cluster_barrier(); // nobody leaves while the other block may read its shared memory or write its TMEM
    else
        __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        if constexpr (CG == 1)
            tmem_dealloc(tmem, 512);
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

} // namespace xs
