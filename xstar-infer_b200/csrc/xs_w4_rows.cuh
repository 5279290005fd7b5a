// Products with 4-bit weights, W[n][k] = (q - z) * s.  One warp per weight row (or gate / up pair) and eight tokens.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"
#include "xs_w4_common.cuh"

namespace xs {

template <bool GATED>
__global__ void __launch_bounds__(256)
w4_rows_kernel(const W4Matrix w, const __nv_bfloat16 *__restrict__ x, __nv_bfloat16 *__restrict__ out, int n_out, int T, int K, int G, int act)
{
    pdl_wait();
    const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int t0 = blockIdx.y * 8, nt = T - t0 < 8 ? T - t0 : 8;
    if (n >= n_out)
        return;
    float res[2][8];
    for (int half = 0; half < (GATED ? 2 : 1); half++) {
        const size_t row = static_cast<size_t>(n) + static_cast<size_t>(half) * n_out;
        float acc[8] = {};
        for (int k = lane * 8; k < K; k += 256) {
            const uint32_t q = *reinterpret_cast<const uint32_t *>(w.codes + row * (K / 2) + k / 2);
            const size_t g = row * (K / G) + k / G;
            const float s = __bfloat162float(w.scales[g]), z = w.zeros ? static_cast<float>(w.zeros[g] & 15) : 8.0f;
            for (int t = 0; t < nt; t++)
                for (int j = 0; j < 8; j++)
                    acc[t] += (static_cast<float>((q >> (4 * j)) & 15) - z) * s * __bfloat162float(x[static_cast<size_t>(t0 + t) * K + k + j]);
        }
        for (int t = 0; t < 8; t++) {
            for (int o = 16; o; o >>= 1)
                acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
            res[half][t] = acc[t];
        }
    }
    if (lane == 0)
        for (int t = 0; t < nt; t++)
            out[static_cast<size_t>(t0 + t) * n_out + n] = __float2bfloat16_rn(GATED ? w4_activation(res[0][t], act) * res[1][t] : res[0][t]);
}

} // namespace xs
