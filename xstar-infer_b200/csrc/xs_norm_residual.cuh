// The step between two blocks: r' = r + c * gate . N(y; w_post), n = N(r'; w_next), N(v; w) = v / sqrt(mean(v^2) + eps) * (o + w).
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

// One block per row, the row's r' in shared memory as f32: any width and alignment.
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
        const float inv = a.w_post ? 1.0f / sqrtf(block_sum(ss) / a.H + a.eps) : 1.0f;
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
        const float inv = 1.0f / sqrtf(block_sum(ss) / a.H + a.eps);
        for (int i = threadIdx.x; i < a.H; i += kNrLoopThreads)
            a.n_out[base + i] = __float2bfloat16_rn(row[i] * inv * (a.offset + __bfloat162float(a.w_next[i])));
    }
}

} // namespace xs
