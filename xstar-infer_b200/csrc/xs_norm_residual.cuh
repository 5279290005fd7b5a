// The step between two blocks: r' = r + c * gate . N(y; w_post), n = N(r'; w_next), N(v; w) = v / sqrt(mean(v^2) + eps) * (o + w).
//
// Bytes decide: y and r (and a full gate) are read once, r' and n written once, and everything between stays in registers as
// f32, both sums of squares included.  A row belongs to a warp, a few or a block; all of a row's loads are issued before the
// first sum, several rows are in work on an SM and hide one another's sums, and a sum costs one barrier of the row's warps (the
// partial sums alternate between two places).  The weights stay in L1 rather than in registers: more rows fit an SM.
//
// Measured: 8192 x 4096 with a full gate 54 us, 6.2 TB/s (96 % of a copy); 777 x 2885 at odd addresses 8.1 us (2.2 TB/s: one wave of rows,
// whose two sums and the loads of weights behind each follow one another); one row 2.2 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"

namespace xs {

struct NormResidualArgs {
    const __nv_bfloat16 *y, *r, *w_post, *gate, *w_next;
    __nv_bfloat16 *r_out, *n_out;
    int gate_kind, rows, H;
    float eps, c, offset;
};

// One block per row, the row's r' in shared memory as f32, columns one by one: the widths and alignments the kernel below does not take.
constexpr int kNrLoopThreads = 256;
__global__ void __launch_bounds__(kNrLoopThreads) norm_residual_loop_kernel(const NormResidualArgs a)
{
    extern __shared__ float row[];
    __shared__ float part[kNrLoopThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const size_t base = static_cast<size_t>(blockIdx.x) * a.H;
    auto block_sum = [&](float v) {
        for (int o = 16; o; o >>= 1)
            v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0)
            part[threadIdx.x >> 5] = v;
        __syncthreads();
        float s = 0.0f;
        for (int i = 0; i < kNrLoopThreads / 32; i++)
            s += part[i];
        return s;
    };
    if (a.y) {
        float ss = 0.0f;
        for (int i = threadIdx.x; i < a.H; i += kNrLoopThreads) {
            const float v = __bfloat162float(a.y[base + i]);
            row[i] = v;
            ss += v * v;
        }
        const float inv = a.w_post ? rsqrtf(block_sum(ss) / a.H + a.eps) : 1.0f;
        for (int i = threadIdx.x; i < a.H; i += kNrLoopThreads) {
            float v = row[i];
            if (a.w_post)
                v = v * inv * (a.offset + __bfloat162float(a.w_post[i]));
            if (a.gate_kind)
                v *= __bfloat162float(a.gate[a.gate_kind == 1 ? i : a.gate_kind == 2 ? blockIdx.x : base + i]);
            v = __bfloat162float(a.r[base + i]) + a.c * v;
            row[i] = v;
            a.r_out[base + i] = __float2bfloat16_rn(v);
        }
    } else {
        for (int i = threadIdx.x; i < a.H; i += kNrLoopThreads)
            row[i] = __bfloat162float(a.r[base + i]);
    }
    if (a.n_out) {
        float ss = 0.0f;
        for (int i = threadIdx.x; i < a.H; i += kNrLoopThreads)
            ss += row[i] * row[i];
        const float inv = rsqrtf(block_sum(ss) / a.H + a.eps);
        for (int i = threadIdx.x; i < a.H; i += kNrLoopThreads)
            a.n_out[base + i] = __float2bfloat16_rn(row[i] * inv * (a.offset + __bfloat162float(a.w_next[i])));
    }
}

// Eight bf16 of a row, of which [lo, hi) belong to it.
__device__ __forceinline__ uint4 nr_load(const __nv_bfloat16 *p, int lo, int hi)
{
    if (lo == 0 && hi == 8)
        return *reinterpret_cast<const uint4 *>(p);
    uint32_t v[4] = {};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i >= lo && i < hi)
            v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[i]) << (i % 2 * 16);
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void nr_store(__nv_bfloat16 *p, int lo, int hi, const float (&f)[8])
{
    __nv_bfloat162 o[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    if (lo == 0 && hi == 8) {
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= lo && i < hi)
                p[i] = i % 2 ? o[i / 2].y : o[i / 2].x;
    }
}
__device__ __forceinline__ float nr_get(const uint4 &v, int i)
{
    const uint32_t u = i / 2 == 0 ? v.x : i / 2 == 1 ? v.y : i / 2 == 2 ? v.z : v.w;
    return __uint_as_float(i % 2 ? u & 0xffff0000u : u << 16);
}

// Columns c .. c + 7 of a vector of H, of which [lo, hi) are wanted; c may be odd, or outside where nothing is wanted.
template <bool ALIGNED>
__device__ __forceinline__ uint4 nr_load_columns(const __nv_bfloat16 *p, int c, int lo, int hi)
{
    if (ALIGNED)
        return *reinterpret_cast<const uint4 *>(p + c);
    if (lo != 0 || hi != 8) {
        const __nv_bfloat16 *q = p + c;
        uint32_t v[4] = {};
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= lo && i < hi)
                v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(q)[i]) << (i % 2 * 16);
        return make_uint4(v[0], v[1], v[2], v[3]);
    }
    const uint32_t *q = reinterpret_cast<const uint32_t *>(p) + (c >> 1);
    const uint32_t w0 = q[0], w1 = q[1], w2 = q[2], w3 = q[3];
    if ((c & 1) == 0)
        return make_uint4(w0, w1, w2, w3);
    const uint32_t last = reinterpret_cast<const uint16_t *>(p)[c + 7]; // its pair may lie behind the vector
    return make_uint4(__funnelshift_r(w0, w1, 16), __funnelshift_r(w1, w2, 16), __funnelshift_r(w2, w3, 16), __funnelshift_r(w3, last, 16));
}

// GROUP threads a row, ITER pieces of eight columns a thread.  ALIGNED: H % 8 == 0.  Otherwise the pieces are those of the whole
// tensor, so that loads and stores of y, r, gate, r' and n are aligned for every row; a row's first and last piece is cut, and the
// weights lie differently for each row.  All tensors are 16-byte aligned.
template <int GROUP, int ITER, bool ALIGNED>
__global__ void __launch_bounds__(GROUP < 256 ? 256 : GROUP) norm_residual_kernel(const NormResidualArgs a)
{
    constexpr int WARPS = GROUP / 32, THREADS = GROUP < 256 ? 256 : GROUP;
    __shared__ float part[2][THREADS / 32];
    const int t = threadIdx.x % GROUP, group = threadIdx.x / GROUP;
    constexpr int rows_per_block = THREADS / GROUP;
    pdl_wait();
    pdl_launch_dependents();
    int place = 0;
    auto row_sum = [&](float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            v += __shfl_xor_sync(0xffffffffu, v, o);
        if constexpr (GROUP > 32) {
            if ((threadIdx.x & 31) == 0)
                part[place][threadIdx.x >> 5] = v;
            asm volatile("barrier.sync %0, %1;" ::"r"(group + 1), "n"(GROUP) : "memory"); // the warps of this row
            v = 0.0f;
#pragma unroll
            for (int i = 0; i < WARPS; i++)
                v += part[place][group * WARPS + i];
            place ^= 1;
        }
        return v;
    };
    const float inv_h = 1.0f / static_cast<float>(a.H);
    for (int row = blockIdx.x * rows_per_block + group; row < a.rows; row += gridDim.x * rows_per_block) {
        const size_t base = static_cast<size_t>(row) * a.H;
        const int shift = ALIGNED ? 0 : static_cast<int>(base & 7); // columns of the first piece that belong to the row before
        const size_t piece0 = base - shift;
        uint4 y[ITER], r[ITER], g[ITER];
        int lo[ITER], hi[ITER];
#pragma unroll
        for (int k = 0; k < ITER; k++) {
            const int c = (k * GROUP + t) * 8; // first column of the piece, plus shift
            lo[k] = ALIGNED ? 0 : max(0, shift - c);
            hi[k] = ALIGNED ? (c < a.H ? 8 : 0) : max(0, min(8, a.H + shift - c));
            y[k] = r[k] = g[k] = make_uint4(0, 0, 0, 0);
            if (hi[k] > 0) {
                if (a.y)
                    y[k] = nr_load(a.y + piece0 + c, lo[k], hi[k]);
                r[k] = nr_load(a.r + piece0 + c, lo[k], hi[k]);
                if (a.gate_kind == 3)
                    g[k] = nr_load(a.gate + piece0 + c, lo[k], hi[k]);
                else if (a.gate_kind == 1)
                    g[k] = nr_load_columns<ALIGNED>(a.gate, c - shift, lo[k], hi[k]);
            }
        }
        float f[ITER][8]; // r'
        if (a.y) {
            float scale = a.c;
            if (a.gate_kind == 2)
                scale *= __bfloat162float(a.gate[row]);
            float inv = 1.0f;
            if (a.w_post) {
                float ss = 0.0f;
#pragma unroll
                for (int k = 0; k < ITER; k++)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        ss = fmaf(nr_get(y[k], i), nr_get(y[k], i), ss);
                inv = rsqrtf(row_sum(ss) * inv_h + a.eps);
            }
#pragma unroll
            for (int k = 0; k < ITER; k++) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (a.w_post && hi[k] > 0)
                    w = nr_load_columns<ALIGNED>(a.w_post, (k * GROUP + t) * 8 - shift, lo[k], hi[k]);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float v = nr_get(y[k], i);
                    if (a.w_post)
                        v = v * inv * (a.offset + nr_get(w, i));
                    if (a.gate_kind == 1 || a.gate_kind == 3)
                        v *= nr_get(g[k], i);
                    f[k][i] = fmaf(scale, v, nr_get(r[k], i));
                }
                if (hi[k] > 0)
                    nr_store(a.r_out + piece0 + (k * GROUP + t) * 8, lo[k], hi[k], f[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < ITER; k++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    f[k][i] = nr_get(r[k], i);
        }
        if (a.n_out) {
            float ss = 0.0f;
#pragma unroll
            for (int k = 0; k < ITER; k++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    ss = fmaf(f[k][i], f[k][i], ss); // what is not of this row was loaded as zero
            const float inv = rsqrtf(row_sum(ss) * inv_h + a.eps);
#pragma unroll
            for (int k = 0; k < ITER; k++)
                if (hi[k] > 0) {
                    const uint4 w = nr_load_columns<ALIGNED>(a.w_next, (k * GROUP + t) * 8 - shift, lo[k], hi[k]);
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        o[i] = f[k][i] * inv * (a.offset + nr_get(w, i));
                    nr_store(a.n_out + piece0 + (k * GROUP + t) * 8, lo[k], hi[k], o);
                }
        }
    }
}

} // namespace xs
