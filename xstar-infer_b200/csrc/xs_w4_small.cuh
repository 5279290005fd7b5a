// Products with 4-bit weights for a handful of tokens: out[t][n] = sum_k (q[n][k] - z[n][k/G]) * s[n][k/G] * x[t][k].
//
// The weights are read once and nothing else is large, so the kernel is a stream: every warp owns a ring of 256-column chunks of
// 16 weight rows (32 for MT = 2) that cp.async fills ahead, four stages deep, across row tiles; no block-wide barrier stands between a load
// and its use.  The eight warps of a block take alternate chunks of the same rows (the split over K) and meet once per row
// tile, in shared memory, in a fixed order.
//
// The arithmetic must stay below the issue rate that the stream allows (at 6.5 TB/s an SM receives 46 weights a cycle, its
// schedulers issue 128 lanes a cycle), so the products go to mma.m16n8k16 with the weights as the 16 rows and 8 tokens as
// columns, and a weight costs one instruction and a half: four nibbles of two columns are cut out with one
// AND-OR that plants the exponent of 128 (0x4300 | q is 128 + q in bf16), and subtracting 128 + z, exact in bf16, leaves q - z.
// The order of k inside an MMA is free as long as both operands agree: a lane's 32-bit word holds columns 8t .. 8t+7, which
// come out as the pairs (0,4) (1,5) (2,6) (3,7), and x is paired the same way.  The MMA sums q - z times x exactly as f32 does;
// the scale multiplies the f32 sum of a group, so the weights are never rounded.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"
#include "xs_w4_common.cuh"

namespace xs {

constexpr int kSwWarps = 8;
constexpr int kSwStages = 4;
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
__device__ __forceinline__ uint32_t lds32(uint32_t a)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

__host__ __device__ constexpr int sw_stage_bytes(int mt)
{
    return mt * 16 * (kSwChunk / 2);
}
__host__ __device__ constexpr int sw_part_stride(int mt)
{
    return mt * 16 + 4; // tokens apart in the partial sums; + 4: the fragments' stores meet no bank twice
}
__host__ __device__ constexpr int sw_smem_bytes(int mt, int tn)
{
    return kSwWarps * (kSwStages * sw_stage_bytes(mt) + 2 * tn * 8 * sw_part_stride(mt) * 4);
}

// TN: 8-token columns (T <= 8 TN).  MT: 16-row groups of a tile; GATED: MT = 2, the 16 gate rows and the 16 up rows of one
// feature block.  SUB: 32-column steps in a scale group.  early: the weights were complete before the predecessor began.
template <int TN, int MT, bool GATED, int SUB, bool ZEROS>
__global__ void __launch_bounds__(32 * kSwWarps)
w4_small_kernel(const W4Matrix w, const __nv_bfloat16 *x, __nv_bfloat16 *out, int n_out, int T, int K, int act, int early)
{
    static_assert(!GATED || MT == 2, "a gated tile is one gate group and one up group");
    constexpr int G = 32 * SUB, GROUPS = kSwChunk / G, SLOTS = (GROUPS + 3) / 4; // scale slots a lane holds per row and chunk
    constexpr int FEATURES = GATED ? 16 : 16 * MT;
    constexpr int PART = TN * 8 * sw_part_stride(MT);

    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * kSwStages * sw_stage_bytes(MT);
    float *part = reinterpret_cast<float *>(smem + kSwWarps * kSwStages * sw_stage_bytes(MT));
    const int n_rows = GATED ? 2 * n_out : n_out, groups = K / G;
    const int tiles = (n_out + FEATURES - 1) / FEATURES, chunks = (K + kSwChunk - 1) / kSwChunk;
    const size_t row_bytes = static_cast<size_t>(K) / 2;

    // weight row of row r (0 .. 16 MT - 1) of a tile; rows past the end read the last one and are not stored
    auto row_of = [&](int tile, int r) {
        const int f = tile * FEATURES + (GATED ? r & 15 : r);
        const int n = (GATED && r >= 16) ? n_out + (f < n_out ? f : n_out - 1) : (f < n_out ? f : n_out - 1);
        return n < n_rows ? n : n_rows - 1;
    };
    // the load side: the next chunk this warp fetches
    int ld_tile = blockIdx.x, ld_chunk = warp, ld_stage = 0;
    auto fetch = [&]() {
        if (ld_chunk < chunks && ld_tile < tiles) {
            const uint32_t dst = ring + ld_stage * sw_stage_bytes(MT);
            const int byte = ld_chunk * (kSwChunk / 2) + (lane & 7) * 16;
            const bool in = byte < static_cast<int>(row_bytes);
#pragma unroll
            for (int i = 0; i < 4 * MT; i++) {
                const int r = i * 4 + (lane >> 3);
                const uint8_t *src = w.codes + static_cast<size_t>(row_of(ld_tile, r)) * row_bytes + (in ? byte : 0);
                cp_async16(dst + r * 128 + (((lane & 7) ^ (r & 7)) << 4), src, in);
            }
            ld_chunk += kSwWarps;
            if (ld_chunk >= chunks) {
                ld_chunk = warp;
                ld_tile += gridDim.x;
            }
        }
        cp_async_commit(); // a group for every call, so that counting groups counts chunks
        ld_stage = ld_stage + 1 == kSwStages ? 0 : ld_stage + 1;
    };

    if (!early)
        pdl_wait();
#pragma unroll
    for (int i = 0; i < kSwStages - 1; i++)
        fetch();
    if (early)
        pdl_wait();
    pdl_launch_dependents(); // after the wait: what the next kernel may load early was complete before this one began

    int stage = 0, parity = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, parity ^= 1) {
        float acc[MT][TN][4] = {};
        const uint16_t *sp[MT][2];
        const uint8_t *zp[MT][2];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const size_t o = static_cast<size_t>(row_of(tile, m * 16 + h * 8 + g)) * groups;
                sp[m][h] = reinterpret_cast<const uint16_t *>(w.scales) + o;
                zp[m][h] = ZEROS ? w.zeros + o : nullptr;
            }
        for (int chunk = warp; chunk < chunks; chunk += kSwWarps) {
            // scales and zero points of the chunk: lane t of a quad holds groups t and t + 4 of rows g and g + 8
            uint32_t sv[MT][2][SLOTS], zv[MT][2][SLOTS];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int j = 0; j < SLOTS; j++) {
                        const int gi = chunk * GROUPS + j * 4 + (t < GROUPS ? t : 0);
                        const bool ok = gi < groups;
                        sv[m][h][j] = ok ? static_cast<uint32_t>(sp[m][h][gi]) << 16 : 0u;
                        zv[m][h][j] = ZEROS ? (ok ? 0x43004300u | ((zp[m][h][gi] & 15u) * 0x00010001u) : 0u) : 0u;
                    }
            fetch();
            cp_async_wait<kSwStages - 1>();
            __syncwarp();
            const uint32_t st = ring + stage * sw_stage_bytes(MT);
            float c[MT][TN][4];
#pragma unroll
            for (int j = 0; j < kSwChunk / 32; j++) {
                const int k0 = chunk * kSwChunk + j * 32;
                if (k0 < K) {
                    uint32_t b[TN][4];
#pragma unroll
                    for (int n = 0; n < TN; n++) {
                        uint4 xv = make_uint4(0, 0, 0, 0);
                        const int token = n * 8 + g;
                        if (token < T)
                            xv = *reinterpret_cast<const uint4 *>(x + static_cast<size_t>(token) * K + k0 + t * 8);
                        b[n][0] = __byte_perm(xv.x, xv.z, 0x5410);
                        b[n][1] = __byte_perm(xv.x, xv.z, 0x7632);
                        b[n][2] = __byte_perm(xv.y, xv.w, 0x5410);
                        b[n][3] = __byte_perm(xv.y, xv.w, 0x7632);
                    }
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        if (j % SUB == 0)
#pragma unroll
                            for (int n = 0; n < TN; n++)
                                c[m][n][0] = c[m][n][1] = c[m][n][2] = c[m][n][3] = 0.0f;
                        uint32_t a[2][4];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint32_t q = lds32(st + (m * 16 + h * 8 + g) * 128 + ((j ^ g) << 4) + t * 4);
                            const uint32_t z = ZEROS ? __shfl_sync(0xffffffffu, zv[m][h][(j / SUB) / 4], (lane & ~3) | ((j / SUB) & 3)) : 0x43084308u;
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                a[h][i] = w4_minus(w4_magic(q >> (4 * i)), z);
                        }
#pragma unroll
                        for (int n = 0; n < TN; n++) {
                            mma_16816(c[m][n], a[0][0], a[1][0], a[0][1], a[1][1], b[n][0], b[n][1]);
                            mma_16816(c[m][n], a[0][2], a[1][2], a[0][3], a[1][3], b[n][2], b[n][3]);
                        }
                        if (j % SUB == SUB - 1) {
                            const int gi = j / SUB;
                            const float s0 = __uint_as_float(__shfl_sync(0xffffffffu, sv[m][0][gi / 4], (lane & ~3) | (gi & 3)));
                            const float s1 = __uint_as_float(__shfl_sync(0xffffffffu, sv[m][1][gi / 4], (lane & ~3) | (gi & 3)));
#pragma unroll
                            for (int n = 0; n < TN; n++) {
                                acc[m][n][0] = fmaf(s0, c[m][n][0], acc[m][n][0]);
                                acc[m][n][1] = fmaf(s0, c[m][n][1], acc[m][n][1]);
                                acc[m][n][2] = fmaf(s1, c[m][n][2], acc[m][n][2]);
                                acc[m][n][3] = fmaf(s1, c[m][n][3], acc[m][n][3]);
                            }
                        }
                    }
                }
            }
            __syncwarp(); // every lane has read the stage before the next fetch may fill it again
            stage = stage + 1 == kSwStages ? 0 : stage + 1;
        }
        float *mine = part + (parity * kSwWarps + warp) * PART;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    mine[(n * 8 + 2 * t + (e & 1)) * sw_part_stride(MT) + m * 16 + (e >> 1) * 8 + g] = acc[m][n][e];
        __syncthreads(); // one barrier a tile: the next tile's sums go to the other half of `part`
        for (int i = threadIdx.x; i < FEATURES * T; i += 32 * kSwWarps) {
            const int token = i / FEATURES, f = i - token * FEATURES, feature = tile * FEATURES + f;
            const float *p = part + parity * kSwWarps * PART + token * sw_part_stride(MT) + f;
            float v = 0.0f, u = 0.0f;
#pragma unroll
            for (int k = 0; k < kSwWarps; k++) {
                v += p[k * PART];
                if (GATED)
                    u += p[k * PART + 16];
            }
            if (feature < n_out)
                out[static_cast<size_t>(token) * n_out + feature] = __float2bfloat16_rn(GATED ? w4_activation(v, act) * u : v);
        }
    }
    cp_async_wait<0>();
}

} // namespace xs
