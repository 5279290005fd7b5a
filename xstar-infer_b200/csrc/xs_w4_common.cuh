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

// Codes to bf16 without an integer-to-float conversion.  A bf16 whose bits are an integer below 256 has the exponent field 0 or
// 1, and both stand for the same scale: its value is that integer times 2^-133.  So the nibbles 0 and 4 of a word (bits 0..3
// of each half) and the nibbles 1 and 5 (bits 4..7: sixteen times the code) are numbers as they stand, and one fused
// multiply-add per pair brings them to (q - z) / 64, exactly: f * 2^-133 * 2^127 = f / 64, with 2^123 for the second pair.
// Nibbles 2, 3, 6, 7 are those of the word shifted by 8.
constexpr uint32_t kW4MulLow = 0x7f007f00u, kW4MulHigh = 0x7d007d00u; // 2^127, 2^123
constexpr uint32_t kW4Minus8 = 0xbe00be00u;                // -8 / 64
constexpr float kW4Unit = 64.0f;
__device__ __forceinline__ uint32_t w4_fma(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// a[0..3]: the pairs (0,4) (1,5) (2,6) (3,7) of a word's codes as (q - z) / 64; mz = -z / 64 twice
__device__ __forceinline__ void w4_unpack(uint32_t (&a)[4], uint32_t q, uint32_t mz)
{
    const uint32_t h = q >> 8;
    a[0] = w4_fma(q & 0x000f000fu, kW4MulLow, mz);
    a[1] = w4_fma(q & 0x00f000f0u, kW4MulHigh, mz);
    a[2] = w4_fma(h & 0x000f000fu, kW4MulLow, mz);
    a[3] = w4_fma(h & 0x00f000f0u, kW4MulHigh, mz);
}
// -z / 64 twice
__device__ __forceinline__ uint32_t w4_minus_zero(uint32_t z)
{
    return w4_fma(z * 0x00010001u, 0xff00ff00u, 0u); // times -2^127
}

// silu: v / (1 + exp(-v)); gelu: v / 2 * (1 + tanh(c (v + 0.044715 v^3))).
__device__ __forceinline__ float w4_activation(float v, int act)
{
    if (act == 0)
        return v / (1.0f + expf(-v));
    return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
}

} // namespace xs
