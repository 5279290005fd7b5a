// Products with 4-bit weights for up to sixteen tokens: out[t][n] = sum_k (q[n][k] - z[n][k/G]) * s[n][k/G] * x[t][k].
//
// The weights are read once and nothing else is large, so the kernel is a stream.  A warp works on 32 weight rows in chunks of
// 256 columns, and owns a ring of such chunks (32 rows x 128 bytes) that TMA fills ahead, across tiles.  Scales come from memory as
// well and are loaded two chunks ahead into registers.  The tokens' columns are laid out once in shared memory.  Of a block's
// sixteen warps, `ways` share the same rows and take alternate chunks of them; they meet once per tile, in shared memory, in a
// fixed order, and no other block-wide barrier stands between a load and its use.  Where the tokens' columns would not fit, or
// where there are too few tiles for the SMs, a cluster of 2, 4 or 8 blocks shares a tile, each with a slice of K, and sums
// through distributed shared memory.  The host picks ways and cluster (plan_small).
//
// The arithmetic must stay below the rate that the stream allows: at 6.5 TB/s an SM receives 46 weights a cycle, and its
// schedulers issue 128 lanes a cycle.  So the products go to mma.m16n8k16 with the weights as the 16 rows and the tokens as the 8
// columns (from the ninth token on: of a second MMA over the same converted weights), and eight codes become (q - z) / 64 with
// nine instructions (w4_unpack).  The order of k inside an MMA is free as long as both operands agree: a lane's 32-bit word holds
// columns 8t .. 8t+7, which come out as the pairs (0,4) (1,5) (2,6) (3,7), and x is laid out in the same pairs.  ldmatrix hands
// word t of row g to lane (g, t), which is the fragment layout.  The MMA sums (q - z) x in f32; the scale multiplies the f32 sum of
// a group, so the weights are never rounded.
//
// Measured: 1 x 4096 x 4096 5.4 us, of which some 4 are launch, first load and sums; 7 x 4096 x 32003 with zero points 24 us, 3.0
// TB/s, half of the issue slots used: registers hold sixteen warps an SM, with chains of conversion and MMA between their loads.
//
// An MLP hands its gated product on in f32 (HALF): rounded to bf16 it would add as much error as the result's own rounding.  The
// second product brings each token, or its slice of one, to a largest element of 2^13 .. 2^14 by a power of two, rounds it once to
// the eleven bits of f16, and multiplies with f16 codes, which are as exact as those in bf16.  Against bf16 rows that costs 0.3 to 0.5 us
// (one token of 4096 x 2048: 10.0 us in all, with an error of 0.0017 for 0.0025); as a second bf16 row of what the first leaves it
// cost 0.7, and half as much K fits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"
#include "xs_w4_common.cuh"

namespace xs {

constexpr int kSwTokens = 16; // at most: two MMAs' columns
constexpr int kSwWarps = 16;
constexpr int kSwChunk = 256;               // columns of one stage: 128 bytes a row
constexpr int kSwStageBytes = 32 * 128;     // 32 rows
constexpr int kSwPartStride = 33;           // floats between tokens in the partial sums of a warp
constexpr int kSwMaxStages = 4;

// in 64 bits: the host asks for rows of any length, most of which do not fit
__host__ __device__ constexpr int64_t sw_x_bytes(int T, int chunks_per_block)
{
    return static_cast<int64_t>(T) * chunks_per_block * kSwChunk * 2;
}
// two halves, for alternate tiles, as long as they leave room for the tokens
__host__ __device__ constexpr int sw_part_bytes(int T)
{
    return (T > 8 ? 1 : 2) * kSwWarps * T * kSwPartStride * 4;
}
__host__ __device__ constexpr int64_t sw_smem_bytes(int T, int chunks_per_block, int stages)
{
    return 1024 + kSwWarps * stages * (kSwStageBytes + 8) + sw_x_bytes(T, chunks_per_block) + sw_part_bytes(T) + 16 + kSwTokens * 4;
}

template <bool HALF>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four 8 x 8 matrices of 16-bit elements: lane (g, t) receives the 32-bit word t of row g of each.  Lane l gives the address of row l % 8 of
// matrix l / 8.
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// GATED: a warp's 32 rows are the 16 gate rows and the 16 up rows of 16 features.  SUB: 32-column steps in a scale group.
// early: the weights were complete before the predecessor began.  Cluster size C, chunks_per_block: K in slices.  HALF: x is
// f32 and enters as f16; out_f32 (GATED): out is written so.
// NT: MMAs' columns, of eight tokens each.
template <bool GATED, int SUB, bool ZEROS, bool HALF, int NT>
__global__ void __launch_bounds__(32 * kSwWarps, 1)
w4_small_kernel(const __grid_constant__ CUtensorMap tmap, const W4Matrix w, const void *x, void *out, int n_out, int T, int K,
                int act, int out_f32, int early, int ways, int C, int chunks_per_block, int stages, int32_t *status)
{
    constexpr int G = 32 * SUB, GROUPS = kSwChunk / G, SLOTS = (GROUPS + 3) / 4; // scale slots a lane holds per row and chunk
    constexpr int ROWS = GATED ? 16 : 32; // features a warp works on
    constexpr float UNIT = HALF ? kW4HalfUnit : kW4Unit;

    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int bands = kSwWarps / ways, band = warp % bands, way = warp / bands; // 32-row bands of a tile
    const int features = bands * ROWS;
    uint8_t *x_smem = smem + kSwWarps * stages * kSwStageBytes;
    float *part = reinterpret_cast<float *>(x_smem + sw_x_bytes(T, chunks_per_block));
    uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(part) + (sw_part_bytes(T) + 7) / 8 * 8);
    volatile uint32_t *abort_flag = reinterpret_cast<uint32_t *>(bars + kSwWarps * stages);
    float *factor = reinterpret_cast<float *>(bars + kSwWarps * stages) + 4; // HALF: of each token
    const uint32_t ring = smem_u32(smem) + warp * stages * kSwStageBytes;
    uint64_t *full = bars + warp * stages;

    const int groups = K / G, part_floats = T * kSwPartStride;
    const int tiles = (n_out + features - 1) / features, all_chunks = (K + kSwChunk - 1) / kSwChunk;
    const int rank = C > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int chunk0 = rank * chunks_per_block, chunk_end = min(chunk0 + chunks_per_block, all_chunks);
    const int first = chunk0 + way; // this warp's chunks: first, first + ways, ... below chunk_end
    const int tile0 = blockIdx.x / C, tile_step = gridDim.x / C;

    if (lane == 0) {
        for (int i = 0; i < stages; i++)
            mbar_init(&full[i], 1);
        if (warp == 0) {
            *abort_flag = 0;
            prefetch_tmap(&tmap);
        }
        fence_mbar_init();
    }
    __syncwarp();

    // Everything past the end of K or of the rows counts as zero: codes that TMA did not find, x and scales.
    struct Place { // one chunk of one tile
        int tile, chunk;
    };
    auto advance = [&](Place &p) {
        p.chunk += ways;
        if (p.chunk >= chunk_end) {
            p.chunk = first;
            p.tile += tile_step;
        }
    };
    const Place begin{first < chunk_end ? tile0 : tiles, first};
    Place ld = begin, ls = begin;
    const uint64_t policy = policy_evict_first(); // every weight is read once
    auto fetch = [&](int stage) {
        if (lane == 0 && ld.tile < tiles) {
            mbar_arrive_expect_tx(&full[stage], kSwStageBytes);
            tma_load_3d(smem + (warp * stages + stage) * kSwStageBytes, &tmap, &full[stage], ld.chunk * (kSwChunk / 2), ld.tile * features + band * ROWS, 0, policy);
        }
        advance(ld);
    };
    // scale (bits 16..31) and zero point (bits 0..3) of a chunk: lane t of a quad holds groups t and t + 4 of rows g + 8 h of the
    // band, h = 0 .. 3 (GATED: h = 2, 3 are the up rows)
    const size_t up_groups = static_cast<size_t>(n_out) * groups;
    auto load_scales = [&](uint32_t (&v)[4][SLOTS]) {
        const int gi = ls.chunk * GROUPS + t % GROUPS, row = ls.tile * features + band * ROWS + g;
        const size_t o = static_cast<size_t>(row) * groups + gi;
        const uint16_t *sp = reinterpret_cast<const uint16_t *>(w.scales) + o;
        const uint8_t *zp = ZEROS ? w.zeros + o : nullptr;
        const int rows = ls.tile < tiles ? n_out - row : 0;
        const bool whole = rows > ROWS - 8 && gi + (SLOTS - 1) * 4 < groups; // every one of them is there
#pragma unroll
        for (int h = 0; h < 4; h++) {
            if (h > 0) {
                const size_t step = GATED && h == 2 ? up_groups - 8 * groups : static_cast<size_t>(8) * groups;
                sp += step;
                if (ZEROS)
                    zp += step;
            }
#pragma unroll
            for (int j = 0; j < SLOTS; j++) {
                v[h][j] = 0u;
                if (whole || ((GATED ? h % 2 : h) * 8 < rows && gi + j * 4 < groups))
                    v[h][j] = static_cast<uint32_t>(sp[j * 4]) << 16 | (ZEROS ? zp[j * 4] & 15u : 0u);
            }
        }
        advance(ls);
    };

    if (!early)
        pdl_wait();
    for (int i = 0; i < stages - 1; i++)
        fetch(i);
    uint32_t sc[4][SLOTS], sc_next[4][SLOTS];
    load_scales(sc);
    load_scales(sc_next);
    if (early)
        pdl_wait();
    pdl_launch_dependents(); // after the wait: what the next kernel may load early was complete before this one began
    // x as the MMA's second operand: [32-column step][token][t] pieces of 16 bytes, the pairs (0,4) (1,5) (2,6) (3,7) of columns 8t ..
    {
        // the warps of a token: two for each of eight, all for a single one; a thread has BATCH pieces of eight columns on their way
        constexpr int BATCH = 4;
        const int spread = NT > 1 ? 1 : T > 4 ? 2 : T > 2 ? 4 : T > 1 ? 8 : 16, n = warp / spread, step = spread * 32, first_p = (warp & (spread - 1)) * 32 + lane;
        const int pieces = n < T ? (chunk_end - chunk0) * (kSwChunk / 8) : 0;
        const int there = min(pieces, K / 8 - chunk0 * (kSwChunk / 8)); // the last slice may end inside a chunk
        const size_t row = static_cast<size_t>(n) * K + chunk0 * kSwChunk;
        auto place = [&](int p) { return reinterpret_cast<uint4 *>(x_smem + (((p >> 2) * T + n) * 4 + (p & 3)) * 16); };
        if constexpr (HALF) {
            auto load = [&](int p, float4 (&v)[BATCH][2]) {
#pragma unroll
                for (int j = 0; j < BATCH; j++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        v[j][i] = p + j * step < there ? reinterpret_cast<const float4 *>(static_cast<const float *>(x) + row)[(p + j * step) * 2 + i]
                                                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            };
            // the first batch is kept, the rest of a long slice loaded twice
            float4 kept[BATCH][2];
            load(first_p, kept);
            float top = 0.0f;
            auto most = [&](const float4 (&v)[BATCH][2]) {
#pragma unroll
                for (int j = 0; j < BATCH; j++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        top = fmaxf(top, fmaxf(fmaxf(finite_abs(v[j][i].x), finite_abs(v[j][i].y)), fmaxf(finite_abs(v[j][i].z), finite_abs(v[j][i].w))));
            };
            most(kept);
#pragma unroll 1
            for (int p = first_p + BATCH * step; p < there; p += BATCH * step) {
                float4 v[BATCH][2];
                load(p, v);
                most(v);
            }
            // floats that are not negative are ordered like their bits
            const uint32_t of_warp = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
            if (lane == 0)
                part[warp] = __uint_as_float(of_warp);
            __syncthreads();
            const uint32_t of_token = __reduce_max_sync(0xffffffffu, __float_as_uint(part[n * spread + (lane & (spread - 1))]));
            const int e = token_exponent(__uint_as_float(of_token));
            const float down = pow2f(-e);
            if (lane == 0 && n < T)
                factor[n] = pow2f(e);
            auto store = [&](int p, const float4 (&v)[BATCH][2]) {
#pragma unroll
                for (int j = 0; j < BATCH; j++) {
                    const float4 &a = v[j][0], &b = v[j][1];
                    const __half2 o[4] = {__floats2half2_rn(a.x * down, b.x * down), __floats2half2_rn(a.y * down, b.y * down),
                                          __floats2half2_rn(a.z * down, b.z * down), __floats2half2_rn(a.w * down, b.w * down)};
                    if (p + j * step < pieces)
                        *place(p + j * step) = *reinterpret_cast<const uint4 *>(o);
                }
            };
            store(first_p, kept);
#pragma unroll 1
            for (int p = first_p + BATCH * step; p < pieces; p += BATCH * step) {
                float4 v[BATCH][2];
                load(p, v);
                store(p, v);
            }
        } else {
#pragma unroll 1
            for (int p = first_p; p < pieces; p += BATCH * step) {
                uint4 v[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; j++)
                    v[j] = p + j * step < there ? reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(x) + row)[p + j * step]
                                                : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < BATCH; j++)
                    if (p + j * step < pieces)
                        *place(p + j * step) = make_uint4(__byte_perm(v[j].x, v[j].z, 0x5410), __byte_perm(v[j].x, v[j].z, 0x7632),
                                                          __byte_perm(v[j].y, v[j].w, 0x5410), __byte_perm(v[j].y, v[j].w, 0x7632));
            }
        }
    }
    __syncthreads();

    // lane l addresses row l % 8 of matrix l / 8; TMA swizzles the 16-byte pieces of a row with the row, and a stage begins at a
    // multiple of 1024, so piece j is one XOR away
    const uint32_t frag = lane * 128 + ((lane & 7) << 4);
    // lanes of tokens that are not there read the last one: a column of its own, which is not stored
    uint32_t x_lane[NT];
#pragma unroll
    for (int i = 0; i < NT; i++)
        x_lane[i] = smem_u32(x_smem) + (min(i * 8 + g, T - 1) * 4 + t) * 16;
    const int x_step = T * 64;
    const int share = features / C, share_log = 31 - __clz(share); // features of a tile that this block finishes: a power of two
    int stage = 0, parity = 0;
    uint32_t phase = 0;
    for (int tile = tile0; tile < tiles; tile += tile_step, parity ^= NT == 1 ? 1 : 0) {
        float acc[2][NT][4] = {};
        for (int chunk = first; chunk < chunk_end; chunk += ways) {
            fetch(stage == 0 ? stages - 1 : stage - 1);
            uint32_t sc_after[4][SLOTS];
            load_scales(sc_after);
            if (!warp_wait(&full[stage], phase, abort_flag)) {
                *abort_flag = 1;
                atomicOr(status, kStatusWaitTimeout);
            }
            const uint32_t st = ring + stage * kSwStageBytes + frag;
            uint32_t xa = (chunk - chunk0) * (kSwChunk / 32) * x_step;
            float c[2][NT][4], s[2][2];
            uint32_t z[2][2];
#pragma unroll
            for (int j = 0; j < kSwChunk / 32; j++) {
                uint4 b[NT];
#pragma unroll
                for (int i = 0; i < NT; i++)
                    b[i] = lds128(x_lane[i] + xa);
                xa += x_step;
                uint32_t q[4];
                ldmatrix_x4(q, st ^ (j << 4));
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    if (j % SUB == 0) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t v = __shfl_sync(0xffffffffu, sc[m * 2 + h][(j / SUB) / 4], (lane & ~3) | ((j / SUB) & 3));
                            s[m][h] = __uint_as_float(ZEROS ? v & 0xffff0000u : v);
                            z[m][h] = HALF ? ZEROS ? w4_half_minus_zero(v & 15u) : kW4HalfMinus8 : ZEROS ? w4_minus_zero(v & 15u) : kW4Minus8;
                        }
                    }
                    uint32_t a[2][4];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if constexpr (HALF)
                            w4_unpack_half(a[h], q[m * 2 + h], z[m][h]);
                        else
                            w4_unpack(a[h], q[m * 2 + h], z[m][h]);
                    }
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        float (&sum)[4] = c[m][i], (&total)[4] = acc[m][i];
                        if (j % SUB == 0)
                            sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
                        mma_16816<HALF>(sum, a[0][0], a[1][0], a[0][1], a[1][1], b[i].x, b[i].y);
                        mma_16816<HALF>(sum, a[0][2], a[1][2], a[0][3], a[1][3], b[i].z, b[i].w);
                        if (j % SUB == SUB - 1) {
                            total[0] = fmaf(s[m][0], sum[0], total[0]);
                            total[1] = fmaf(s[m][0], sum[1], total[1]);
                            total[2] = fmaf(s[m][1], sum[2], total[2]);
                            total[3] = fmaf(s[m][1], sum[3], total[3]);
                        }
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int j = 0; j < SLOTS; j++) {
                    sc[h][j] = sc_next[h][j];
                    sc_next[h][j] = sc_after[h][j];
                }
            __syncwarp(); // every lane has read the stage before the next fetch may fill it again
            if (++stage == stages) {
                stage = 0;
                phase ^= 1;
            }
        }
        float *mine = part + (parity * kSwWarps + warp) * part_floats;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int token = i * 8 + 2 * t + e;
                if (token < T) {
                    const float f = HALF ? factor[token] : 1.0f;
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        mine[token * kSwPartStride + m * 16 + g] = acc[m][i][e] * f;
                        mine[token * kSwPartStride + m * 16 + 8 + g] = acc[m][i][2 + e] * f;
                    }
                }
            }
        // one barrier a tile: the next tile's sums go to the other half of `part`, if it has two
        if (C > 1)
            cluster_barrier();
        else
            __syncthreads();
        for (int i = threadIdx.x; i < share * T; i += 32 * kSwWarps) {
            const int token = i >> share_log, f = rank * share + (i & (share - 1)), feature = tile * features + f;
            const float *p = part + (parity * kSwWarps + f / ROWS) * part_floats + token * kSwPartStride + f % ROWS;
            float v = 0.0f, u = 0.0f;
            for (int r = 0; r < C; r++)
                for (int k = 0; k < ways; k++) {
                    const float *pk = p + k * bands * part_floats;
                    v += C > 1 ? ld_cluster_f32(smem_u32(pk), r) : *pk;
                    if (GATED)
                        u += C > 1 ? ld_cluster_f32(smem_u32(pk + 16), r) : pk[16];
                }
            if (feature < n_out) {
                const float r = GATED ? w4_activation(UNIT * v, act) * (UNIT * u) : UNIT * v;
                const size_t o = static_cast<size_t>(token) * n_out + feature;
                if (GATED && out_f32)
                    static_cast<float *>(out)[o] = r;
                else
                    static_cast<__nv_bfloat16 *>(out)[o] = __float2bfloat16_rn(r);
            }
        }
        if (NT > 1 && tile + tile_step < tiles) {
            if (C > 1)
                cluster_barrier();
            else
                __syncthreads();
        }
    }
    if (C > 1)
        cluster_barrier(); // nobody leaves while its sums may still be read
    if (*abort_flag)
        for (int i = 0; i < 64; i++)
            __nanosleep(4096);
}

} // namespace xs
