// What the kernels with 4-bit integer weights share: the matrix, the conversion of codes, the activations.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace xs {

struct W4Matrix {
    const uint8_t *codes;        // (rows, K / 2), the even column in the low nibble
    const __nv_bfloat16 *scales; // (rows, K / G)
    const uint8_t *zeros;        // (rows, K / G) or null: 8
};

// Nibbles 0 and 4 of v as two bf16 numbers 128 + q: the 7 mantissa bits of a bf16 in [128, 256) count ones.
__device__ __forceinline__ uint32_t w4_magic(uint32_t v)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(v)); // (v & m) | e
    return r;
}
// (128 + q) - (128 + z), both pairs: small integers, exact in bf16
__device__ __forceinline__ uint32_t w4_minus(uint32_t q, uint32_t z)
{
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(q), "r"(z));
    return r;
}

// silu: v / (1 + exp(-v)); gelu: v / 2 * (1 + tanh(c (v + 0.044715 v^3))).
__device__ __forceinline__ float w4_activation(float v, int act)
{
    if (act == 0)
        return v / (1.0f + expf(-v));
    return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
}

} // namespace xs
