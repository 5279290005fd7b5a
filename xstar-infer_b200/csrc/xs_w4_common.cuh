// What the kernels with 4-bit integer weights share: the matrix, the conversion of codes, the activations.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "xs_ptx.cuh"

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

__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_fma(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// The same in f16, whose bits are an integer below 1024 times 2^-24: 2^15 brings a nibble, and 2^11 sixteen times one, to the code
// times 2^-9.  kW4PairMul: for a pair of both kinds.
constexpr uint32_t kW4HalfMulLow = 0x78007800u, kW4HalfMulHigh = 0x68006800u, kW4PairMul = 0x68007800u;
constexpr uint32_t kW4HalfMinus8 = 0xa400a400u; // -8 * 2^-9
constexpr float kW4HalfUnit = 512.0f;
__device__ __forceinline__ uint32_t w4_half_minus_zero(uint32_t z)
{
    return f16x2_mul(z * 0x00010001u, 0xf800f800u); // -2^15
}
__device__ __forceinline__ void w4_unpack_half(uint32_t (&a)[4], uint32_t q, uint32_t mz)
{
    const uint32_t h = q >> 8;
    a[0] = f16x2_fma(q & 0x000f000fu, kW4HalfMulLow, mz);
    a[1] = f16x2_fma(q & 0x00f000f0u, kW4HalfMulHigh, mz);
    a[2] = f16x2_fma(h & 0x000f000fu, kW4HalfMulLow, mz);
    a[3] = f16x2_fma(h & 0x00f000f0u, kW4HalfMulHigh, mz);
}

// Powers of two that bring tokens and scales into the range of f16.
constexpr int kExpMin = -112, kExpMax = 114;
__device__ __forceinline__ float pow2f(int e) // -126 <= e <= 127
{
    return __int_as_float((e + 127) << 23);
}
// floor(log2 v) of a positive normal v; subnormal numbers count as 2^-127
__device__ __forceinline__ int log2_floor(float v)
{
    return ((__float_as_int(v) >> 23) & 255) - 127;
}
__device__ __forceinline__ float finite_abs(float v)
{
    const float a = fabsf(v);
    return a <= FLT_MAX ? a : 0.0f; // infinities and NaN do not count
}

// The power of two that brings a token whose largest element is `top` to 2^13 .. 2^14.
__device__ __forceinline__ int token_exponent(float top)
{
    return max(kExpMin, min(kExpMax, log2_floor(top) - 13));
}

// silu: v / (1 + exp(-v)); gelu: v / 2 * (1 + tanh(c (v + 0.044715 v^3))), and (1 + tanh(a)) / 2 = 1 / (1 + exp(-2 a)).  The fast
// exponential and division are off by a few f32 steps, far below the step of the result; far below zero, where the
// exponential leaves f32, the division gives the zero that the result is.
__device__ __forceinline__ float w4_activation(float v, int act)
{
    const float a = act == 0 ? v : 1.5957691216057308f * fmaf(0.044715f * v * v, v, v);
    return __fdividef(v, 1.0f + __expf(-a));
}

// A bounded wait of a whole warp with one outcome.  Every lane asks, since what one of them has seen of memory orders nothing for
// the others.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag)
{
    const bool there = mbar_try_wait(bar, parity);
    return __all_sync(0xffffffffu, there || mbar_wait(bar, parity, abort_flag));
}
// The same for waits that are long by nature: sleeps between polls, so that the warp takes no issue slots from those that work.
// Gives up after about a quarter of a second and 8 us more for each of the `steps` that the wait is for.
__device__ __forceinline__ bool warp_sleep_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *abort_flag, uint32_t steps)
{
    bool ok = true;
    if ((threadIdx.x & 31) == 0) {
        ok = false;
        for (uint32_t i = 0; i < (1u << 21) + 64 * steps; i++) {
            if (mbar_test_wait(bar, parity)) {
                ok = true;
                break;
            }
            if (*abort_flag)
                break;
            __nanosleep(128);
        }
    }
    return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}
__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
// 3-D tiled load: c0 and c1 as in tma_load_2d, c2 the outermost coordinate.
__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *m, uint64_t *bar, int32_t c0, int32_t c1, int32_t c2, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5}], [%2], %6;"
        :
        : "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
        : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank)
{
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr, uint32_t rank)
{
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr), "r"(rank)
                 : "memory");
    return v;
}

} // namespace xs
