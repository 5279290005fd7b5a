// Products with 4-bit weights for up to eight tokens: out[t][n] = sum_k (q[n][k] - z[n][k/G]) * s[n][k/G] * x[t][k].
//
// The weights are read once and nothing else is large, so the kernel is a stream: every warp owns a ring of 256-column chunks of
// 16 weight rows (32 for MT = 2), with the tokens' 256 columns beside them, that cp.async fills ahead across row tiles; scales
// are loaded one chunk ahead into registers, since they come from memory as well.  No block-wide barrier stands between a
// load and its use.  The eight warps of a block take alternate chunks of the same rows (the split over K) and meet once per
// row tile, in shared memory, in a fixed order.
//
// The arithmetic must stay below the rate that the stream allows: at 6.5 TB/s an SM receives 46 weights a cycle, while its
// integer pipe does 64 lanes and its schedulers issue 128.  So the products go to mma.m16n8k16 with the weights as the 16 rows
// and the tokens as the 8 columns, and a weight costs less than one integer instruction: four nibbles of two columns are cut
// out with one AND-OR that plants the exponent of 128 (0x4300 | q is 128 + q in bf16), and subtracting 128 + z, exact in
// bf16, leaves q - z.  The order of k inside an MMA is free as long as both operands agree: a lane's 32-bit word holds columns
// 8t .. 8t+7, which come out as the pairs (0,4) (1,5) (2,6) (3,7), and x is paired the same way.  ldmatrix hands word t of
// row g to lane (g, t), which is the fragment layout.  The MMA sums q - z times x in f32; the scale multiplies the f32 sum
// of a group, so the weights are never rounded.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"
#include "xs_w4_common.cuh"

namespace xs {

constexpr int kSwTokens = 8;
constexpr int kSwWarps = 8;
constexpr int kSwChunk = 256; // columns of one stage: 128 bytes a row

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool in_range)
{
    // out of range: nothing is read, the 16 bytes become zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in_range ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
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
                 : "r"(addr));
}
__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

// chunks of a warp's ring, one in use and the others on their way: 48 to 64 KB of weights in flight an SM
__host__ __device__ constexpr int sw_stages(int mt)
{
    return mt == 1 ? 4 : 3;
}
__host__ __device__ constexpr int sw_stage_bytes(int mt, int T)
{
    return mt * 16 * (kSwChunk / 2) + T * kSwChunk * 2;
}
__host__ __device__ constexpr int sw_part_stride(int mt)
{
    return mt * 16 + 4; // tokens apart in the partial sums; + 4: the fragments' stores meet no bank twice
}
__host__ __device__ constexpr int sw_smem_bytes(int mt, int T)
{
    return kSwWarps * (sw_stages(mt) * sw_stage_bytes(mt, T) + 2 * T * sw_part_stride(mt) * 4);
}

// MT: 16-row groups of a tile; GATED: MT = 2, the 16 gate rows and the 16 up rows of one feature block.  SUB: 32-column steps
// in a scale group.  early: the weights were complete before the predecessor began.
template <int MT, bool GATED, int SUB, bool ZEROS>
__global__ void __launch_bounds__(32 * kSwWarps)
w4_small_kernel(const W4Matrix w, const __nv_bfloat16 *x, __nv_bfloat16 *out, int n_out, int T, int K, int act, int early)
{
    static_assert(!GATED || MT == 2, "a gated tile is one gate group and one up group");
    constexpr int G = 32 * SUB, GROUPS = kSwChunk / G, SLOTS = (GROUPS + 3) / 4; // scale slots a lane holds per row and chunk
    constexpr int FEATURES = GATED ? 16 : 16 * MT;
    constexpr int STAGES = sw_stages(MT);
    constexpr int W_BYTES = MT * 16 * (kSwChunk / 2);

    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int stage_bytes = sw_stage_bytes(MT, T);
    const uint32_t ring = smem_u32(smem) + warp * STAGES * stage_bytes;
    float *part = reinterpret_cast<float *>(smem + kSwWarps * STAGES * stage_bytes);
    const int groups = K / G, part_floats = T * sw_part_stride(MT);
    const int tiles = (n_out + FEATURES - 1) / FEATURES, chunks = (K + kSwChunk - 1) / kSwChunk;
    const int row_bytes = K / 2;
    const size_t half_rows = GATED ? static_cast<size_t>(n_out) - 16 : 0; // rows 16.. of a gated tile lie n_out below the first

    // Everything past the end of K or of the rows reads as zero: codes, x and scales, so that it adds 0 * 0 * 0.
    // The load side of codes and x: one chunk of one tile.
    struct {
        int tile, chunk;
        const uint8_t *w; // this lane's piece of row lane / 8
    } ld{};
    auto ld_start = [&](int tile) {
        ld.tile = tile;
        ld.chunk = warp;
        ld.w = w.codes + (static_cast<size_t>(tile) * FEATURES + (lane >> 3)) * row_bytes + warp * (kSwChunk / 2) + (lane & 7) * 16;
    };
    auto ld_next = [&]() {
        ld.chunk += kSwWarps;
        ld.w += kSwWarps * (kSwChunk / 2);
        if (ld.chunk >= chunks)
            ld_start(ld.tile + gridDim.x);
    };
    const int lane_dst = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4), lane_dst4 = lane_dst ^ 64; // rows 4 .. 7 of every 8
    auto fetch_w = [&](int stage) {
        if (ld.tile < tiles) {
            const uint32_t dst = ring + stage * stage_bytes;
            const bool in = ld.chunk * (kSwChunk / 2) + (lane & 7) * 16 < row_bytes;
            const int rows = n_out - ld.tile * FEATURES - (lane >> 3); // rows from this lane's first to the end
            const uint8_t *src = ld.w;
#pragma unroll
            for (int i = 0; i < 4 * MT; i++) {
                if (GATED && i == 4)
                    src += half_rows * row_bytes;
                const bool ok = in && (GATED ? i % 4 : i) * 4 < rows;
                cp_async16(dst + (i / 2) * 1024 + (i % 2 ? 512 + lane_dst4 : lane_dst), ok ? src : w.codes, ok);
                src += 4 * static_cast<size_t>(row_bytes);
            }
        }
    };
    // 16-byte piece c of a token's 512: at c, or c ^ 4 for odd tokens, so that the eight lanes of a quarter read meet no bank twice
    auto fetch_x = [&](int stage) {
        if (ld.tile < tiles) {
            uint32_t dst = ring + stage * stage_bytes + W_BYTES + (lane << 4);
            const int k = ld.chunk * kSwChunk + lane * 8;
            const bool in = k < K;
            const __nv_bfloat16 *src = x + (in ? k : 0);
            const int odd = lane & 4 ? -64 : 64;
            for (int n = 0; n < T; n++) {
                cp_async16(dst + (n & 1 ? odd : 0), src, in);
                dst += kSwChunk * 2;
                src += K;
            }
        }
        cp_async_commit(); // a group for every call, so that counting groups counts chunks
    };
    // scale (bits 16..31) and zero point (bits 0..3) of a chunk: lane t of a quad holds groups t and t + 4 of rows g and g + 8
    struct {
        int tile, chunk;
    } ls{};
    auto load_scales = [&](uint32_t (&v)[MT][2][SLOTS]) {
        const int gi = ls.chunk * GROUPS + t % GROUPS, rows = ls.tile < tiles ? n_out - ls.tile * FEATURES - g : 0;
        const size_t o = (static_cast<size_t>(ls.tile) * FEATURES + g) * groups + gi;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const size_t oh = o + (GATED && m ? half_rows * groups : 0) + static_cast<size_t>((m * 2 + h) * 8 * groups);
#pragma unroll
                for (int j = 0; j < SLOTS; j++) {
                    v[m][h][j] = 0u;
                    if (((GATED ? 0 : m * 2) + h) * 8 < rows && gi + j * 4 < groups)
                        v[m][h][j] = static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(w.scales)[oh + j * 4]) << 16 |
                                     (ZEROS ? w.zeros[oh + j * 4] & 15u : 0u);
                }
            }
        ls.chunk += kSwWarps;
        if (ls.chunk >= chunks) {
            ls.chunk = warp;
            ls.tile += gridDim.x;
        }
    };

    // a warp without chunks of its own (K <= 256 warp) only joins the sums
    const int first_tile = warp < chunks ? static_cast<int>(blockIdx.x) : tiles;
    if (!early)
        pdl_wait();
    uint32_t sc[MT][2][SLOTS], sc_next[MT][2][SLOTS];
    ld_start(first_tile);
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++, ld_next())
        fetch_w(i);
    ls.tile = first_tile;
    ls.chunk = warp;
    load_scales(sc);
    load_scales(sc_next);
    if (early)
        pdl_wait();
    ld_start(first_tile);
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++, ld_next())
        fetch_x(i);
    pdl_launch_dependents(); // after the wait: what the next kernel may load early was complete before this one began

    // lane l addresses row l % 8 of matrix l / 8: rows 0..7 and 8..15 of two groups (MT = 2), or of two 32-column steps (MT = 1)
    const int mat = lane >> 3, mrow = lane & 7;
    const uint32_t frag = ((MT == 2 ? mat : mat & 1) * 8 + mrow) * 128;
    // lanes of tokens that are not there read the last one: a column of its own, which is not stored
    const int xg = g < T ? g : T - 1;
    const uint32_t x_even = W_BYTES + xg * (kSwChunk * 2) + (t << 4) + ((xg & 1) << 6), x_odd = x_even + 64 - ((xg & 1) << 7);
    int stage = 0, parity = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, parity ^= 1) {
        float acc[MT][4] = {};
        for (int chunk = warp; chunk < chunks; chunk += kSwWarps) {
            const int fill = stage == 0 ? STAGES - 1 : stage - 1;
            fetch_w(fill);
            fetch_x(fill);
            ld_next();
            uint32_t sc_after[MT][2][SLOTS];
            load_scales(sc_after);
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t st = ring + stage * stage_bytes;
            float c[MT][4];
            uint32_t qq[4];
            float s[MT][2];
            uint32_t z[MT][2];
#pragma unroll
            for (int j = 0; j < kSwChunk / 32; j++) {
                const uint4 xv = lds128(st + (j % 2 ? x_odd : x_even) + (j / 2) * 128);
                const uint32_t b[4] = {__byte_perm(xv.x, xv.z, 0x5410), __byte_perm(xv.x, xv.z, 0x7632), __byte_perm(xv.y, xv.w, 0x5410),
                                       __byte_perm(xv.y, xv.w, 0x7632)};
                if (MT == 2)
                    ldmatrix_x4(qq, st + frag + ((j ^ mrow) << 4));
                else if (j % 2 == 0)
                    ldmatrix_x4(qq, st + frag + (((j + (mat >> 1)) ^ mrow) << 4));
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    if (j % SUB == 0) {
                        c[m][0] = c[m][1] = c[m][2] = c[m][3] = 0.0f;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t v = __shfl_sync(0xffffffffu, sc[m][h][(j / SUB) / 4], (lane & ~3) | ((j / SUB) & 3));
                            s[m][h] = __uint_as_float(ZEROS ? v & 0xffff0000u : v);
                            z[m][h] = ZEROS ? (v & 15u) * 0x00010001u + 0x43004300u : 0x43084308u;
                        }
                    }
                    uint32_t a[2][4];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t q = qq[(MT == 2 ? m * 2 : (j % 2) * 2) + h];
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            a[h][i] = w4_minus(w4_magic(q >> (4 * i)), z[m][h]);
                    }
                    mma_16816(c[m], a[0][0], a[1][0], a[0][1], a[1][1], b[0], b[1]);
                    mma_16816(c[m], a[0][2], a[1][2], a[0][3], a[1][3], b[2], b[3]);
                    if (j % SUB == SUB - 1) {
                        acc[m][0] = fmaf(s[m][0], c[m][0], acc[m][0]);
                        acc[m][1] = fmaf(s[m][0], c[m][1], acc[m][1]);
                        acc[m][2] = fmaf(s[m][1], c[m][2], acc[m][2]);
                        acc[m][3] = fmaf(s[m][1], c[m][3], acc[m][3]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int j = 0; j < SLOTS; j++) {
                        sc[m][h][j] = sc_next[m][h][j];
                        sc_next[m][h][j] = sc_after[m][h][j];
                    }
            __syncwarp(); // every lane has read the stage before the next fetch may fill it again
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        float *mine = part + (parity * kSwWarps + warp) * part_floats;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (2 * t + (e & 1) < T)
                    mine[(2 * t + (e & 1)) * sw_part_stride(MT) + m * 16 + (e >> 1) * 8 + g] = acc[m][e];
        __syncthreads(); // one barrier a tile: the next tile's sums go to the other half of `part`
        for (int i = threadIdx.x; i < FEATURES * T; i += 32 * kSwWarps) {
            const int token = i / FEATURES, f = i - token * FEATURES, feature = tile * FEATURES + f;
            const float *p = part + parity * kSwWarps * part_floats + token * sw_part_stride(MT) + f;
            float v = 0.0f, u = 0.0f;
#pragma unroll
            for (int k = 0; k < kSwWarps; k++) {
                v += p[k * part_floats];
                if (GATED)
                    u += p[k * part_floats + 16];
            }
            if (feature < n_out)
                out[static_cast<size_t>(token) * n_out + feature] = __float2bfloat16_rn(GATED ? w4_activation(v, act) * u : v);
        }
    }
    cp_async_wait<0>();
}

} // namespace xs
