// What the tensor-core kernel of the 4-bit products needs before it starts: the tokens and the size of the scales.
//
// Its operands are f16, not bf16: (q - z) s has twelve significant bits, and f16 keeps eleven of them where bf16 keeps eight (the rounding
// of a weight is then an eighth of the rounding of a result, instead of as large), while a bf16 token is exact in f16 once its
// exponent fits.  So every token is scaled by a power of two that brings its largest element to 2^13 .. 2^14: elements down to
// 2^-27 of that are exact, smaller ones are off by 2^-39 of it at most.  The scales of each weight row are brought to f16 in the
// same way, into rows of a padded pitch (with the zero points), which the kernel reads in one piece per block whatever the
// alignment of the originals; a row whose scales differ by less than 2^4 is marked, and takes a shorter conversion there.  The powers of
// two come back in the kernel's epilogue.
//
// The gated product's own result becomes the next product's token.  It is handed on in f32 and scaled like a token, by its own
// largest element (w4_rescale_kernel): a bound from the norms of token and weights, with which it could be written in f16 at
// once, may lie any distance above what occurs, where the weights do not take a large element of the token or the gate closes.
//
// Bytes decide: tokens are read once and written once; the scales are a fiftieth of the weights.  With `norm_w` the tokens are
// normed on the way (the first norm of a block): v / sqrt(mean v^2 + eps) * (offset + w), rounded once, to f16.  8192 tokens of
// 4096 and the scales of 24576 x 4096 and 4096 x 12288: 22 us (6.3 TB/s); with a few tokens 3 to 4 us, most of them latency.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "xs_ptx.cuh"
#include "xs_w4_common.cuh"

namespace xs {

struct PrepareScales {
    const uint16_t *scales; // bf16 (rows, groups)
    const uint8_t *zeros;   // (rows, groups) or null
    uint16_t *scales16;     // f16 (rows, pitch): scale = scales16 * 2^c
    uint8_t *zeros8;        // (rows, pitch)
    float *factor;          // 2^(c + 9) of a row: what its sums are multiplied by; negative for a row of wide range
    int rows, groups, pitch;
    int per_block, blocks; // rows of a block
    int lanes;             // lanes on a row: a power of two; 8 groups each at a time if `vec`
    int vec;
};
struct PrepareArgs {
    const __nv_bfloat16 *x, *norm_w;
    __half *x16;
    float *factor; // token = x16 * factor
    int T, K;
    float eps, offset;
    PrepareScales m[2];   // the second may be empty (blocks = 0)
};

constexpr int kPrepThreads = 128;
constexpr int kPrepRows = 128;     // weight rows of a block at most
constexpr int kPrepKeep = 4;       // pieces of eight columns a thread keeps in registers
constexpr int kTcUnitExp = 9; // the codes enter as (q - z) 2^-9

__device__ __forceinline__ float prep_get(const uint4 &v, int i)
{
    const uint32_t u = i / 2 == 0 ? v.x : i / 2 == 1 ? v.y : i / 2 == 2 ? v.z : v.w;
    return __uint_as_float(i % 2 ? u & 0xffff0000u : u << 16);
}
__global__ void __launch_bounds__(kPrepThreads) w4_prepare_kernel(const PrepareArgs a)
{
    constexpr int WARPS = kPrepThreads / 32;
    __shared__ float part[2][WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    if (static_cast<int>(blockIdx.x) < a.T) {
        const int t = blockIdx.x, pieces = a.K / 8;
        const uint4 *x = reinterpret_cast<const uint4 *>(a.x + static_cast<size_t>(t) * a.K);
        uint4 keep[kPrepKeep];
#pragma unroll
        for (int i = 0; i < kPrepKeep; i++) {
            keep[i] = make_uint4(0, 0, 0, 0);
            if (threadIdx.x + i * kPrepThreads < pieces)
                keep[i] = x[threadIdx.x + i * kPrepThreads];
        }
        // f(piece, its columns) over this thread's pieces: those kept, then the rest of a long row from memory again
        auto each = [&](auto &&f) {
#pragma unroll
            for (int i = 0; i < kPrepKeep; i++)
                if (threadIdx.x + i * kPrepThreads < pieces)
                    f(threadIdx.x + i * kPrepThreads, keep[i]);
            for (int p = threadIdx.x + kPrepKeep * kPrepThreads; p < pieces; p += kPrepThreads)
                f(p, x[p]);
        };
        float inv = 1.0f;
        if (a.norm_w) {
            float ss = 0.0f;
            each([&](int, const uint4 &v) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    ss = fmaf(prep_get(v, i), prep_get(v, i), ss);
            });
#pragma unroll
            for (int o = 16; o; o >>= 1)
                ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (lane == 0)
                part[1][warp] = ss;
            __syncthreads();
            ss = 0.0f;
#pragma unroll
            for (int i = 0; i < WARPS; i++)
                ss += part[1][i];
            inv = rsqrtf(ss / static_cast<float>(a.K) + a.eps);
        }
        // the eight columns of a piece, normed
        auto values = [&](int p, const uint4 &v, float (&f)[8]) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                f[i] = prep_get(v, i);
            if (a.norm_w) {
                const __nv_bfloat16 *w = a.norm_w + p * 8;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    f[i] = f[i] * inv * (a.offset + __bfloat162float(w[i]));
            }
        };
        float top = 0.0f;
        each([&](int p, const uint4 &v) {
            float f[8];
            values(p, v, f);
#pragma unroll
            for (int i = 0; i < 8; i++)
                top = fmaxf(top, finite_abs(f[i]));
        });
#pragma unroll
        for (int o = 16; o; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0)
            part[0][warp] = top;
        __syncthreads();
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < WARPS; i++)
            top = fmaxf(top, part[0][i]);
        const int e = token_exponent(top);
        const float down = pow2f(-e);
        uint4 *out = reinterpret_cast<uint4 *>(a.x16 + static_cast<size_t>(t) * a.K);
        each([&](int p, const uint4 &v) {
            float f[8];
            values(p, v, f);
            __half2 o[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                o[i] = __floats2half2_rn(f[2 * i] * down, f[2 * i + 1] * down);
            out[p] = *reinterpret_cast<uint4 *>(o);
        });
        if (threadIdx.x == 0)
            a.factor[t] = pow2f(e);
    } else {
        int b = blockIdx.x - a.T;
        const int which = b >= a.m[0].blocks ? 1 : 0;
        if (which)
            b -= a.m[0].blocks;
        const PrepareScales m = which ? a.m[1] : a.m[0];
        const int sub = lane & (m.lanes - 1);
        const int stride = kPrepThreads / m.lanes;
        struct Row {
            bool there;
            size_t row;
            uint4 s0; // scales of this lane's first groups; a row of more than 256 groups is read again below
            uint2 z0;
        };
        auto scales = [&](const Row &w, int g) { // of groups g .. g + 7, zero behind the last one
            const uint16_t *s = m.scales + w.row * m.groups;
            if (m.vec)
                return *reinterpret_cast<const uint4 *>(s + g);
            uint32_t u[4] = {};
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (g + j < m.groups)
                    u[j / 2] |= static_cast<uint32_t>(s[g + j]) << (j % 2 * 16);
            return make_uint4(u[0], u[1], u[2], u[3]);
        };
        auto zeros = [&](const Row &w, int g) {
            const uint8_t *z = m.zeros + w.row * m.groups;
            if (m.vec)
                return *reinterpret_cast<const uint2 *>(z + g);
            uint32_t u[2] = {};
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (g + j < m.groups)
                    u[j / 4] |= static_cast<uint32_t>(z[g + j]) << (j % 4 * 8);
            return make_uint2(u[0], u[1]);
        };
        auto load = [&](int r) {
            Row w;
            const int i = b * m.per_block + r;
            w.there = r < m.per_block && i < m.rows;
            w.row = w.there ? static_cast<size_t>(i) : 0;
            w.s0 = make_uint4(0, 0, 0, 0);
            w.z0 = make_uint2(0, 0);
            if (w.there && sub * 8 < m.groups) {
                w.s0 = scales(w, sub * 8);
                if (m.zeros)
                    w.z0 = zeros(w, sub * 8);
            }
            return w;
        };
        auto finish = [&](const Row &w) {
            float top = 0.0f, low = FLT_MAX;
            bool odd = false; // an infinity or NaN
            for (int g = sub * 8; g < m.groups; g += m.lanes * 8) {
                const uint4 v = g == sub * 8 ? w.s0 : scales(w, g);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float f = fabsf(prep_get(v, j)), c = finite_abs(f);
                    odd |= !(f <= FLT_MAX);
                    top = fmaxf(top, c);
                    low = c > 0.0f ? fminf(low, c) : low;
                }
            }
            for (int o = m.lanes / 2; o; o >>= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
                odd |= __shfl_xor_sync(0xffffffffu, odd ? 1 : 0, o) != 0;
            }
            // narrow: scales below 1 and not below 2^-4, so that (q - 8) scale 2^-9 is a normal f16 and the scale times 2^15 one as well;
            // wide: below 2^15, which leaves 2^20 down to the first lost bit
            const int top_exp = log2_floor(top);
            const bool narrow = !odd && top_exp < 100 && top_exp - log2_floor(fminf(low, top)) < 4;
            const int c = max(kExpMin, min(kExpMax, narrow ? top_exp + 1 : top_exp - 14));
            const float down = pow2f(-c);
            if (w.there) {
                for (int g = sub * 8; g < m.groups; g += m.lanes * 8) {
                    const uint4 v = g == sub * 8 ? w.s0 : scales(w, g);
                    __half2 o[4];
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[j] = __floats2half2_rn(prep_get(v, 2 * j) * down, prep_get(v, 2 * j + 1) * down);
                    *reinterpret_cast<uint4 *>(m.scales16 + w.row * m.pitch + g) = *reinterpret_cast<uint4 *>(o);
                    if (m.zeros)
                        *reinterpret_cast<uint2 *>(m.zeros8 + w.row * m.pitch + g) = g == sub * 8 ? w.z0 : zeros(w, g);
                }
                if (sub == 0)
                    m.factor[w.row] = narrow ? pow2f(c + kTcUnitExp) : -pow2f(c + kTcUnitExp);
            }
        };
        // four rows' loads on their way before the first is worked on
        for (int r = static_cast<int>(threadIdx.x) / m.lanes; r - static_cast<int>(threadIdx.x) / m.lanes < m.per_block; r += 4 * stride) {
            Row w[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = load(r + i * stride);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i * stride + r - static_cast<int>(threadIdx.x) / m.lanes < m.per_block)
                    finish(w[i]);
        }
    }
}

// f32 rows (T, K) to f16, each scaled by its own largest element like a token above.  One block a row, which it reads once: kept in
// registers up to 12288 columns, the rest of a longer row from memory again.  Bytes decide: 8192 rows of 12288 in 80 us (7.5 TB/s, some
// of them still in L2).
constexpr int kRescaleThreads = 256;
constexpr int kRescaleKeep = 6;
__global__ void __launch_bounds__(kRescaleThreads) w4_rescale_kernel(const float *__restrict__ h, __half *__restrict__ h16, float *__restrict__ factor, int K)
{
    __shared__ float part[kRescaleThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const int pieces = K / 8;
    const float4 *row = reinterpret_cast<const float4 *>(h + static_cast<size_t>(blockIdx.x) * K);
    uint4 *out = reinterpret_cast<uint4 *>(h16 + static_cast<size_t>(blockIdx.x) * K);
    float4 keep[kRescaleKeep][2];
#pragma unroll
    for (int i = 0; i < kRescaleKeep; i++) {
        const int p = threadIdx.x + i * kRescaleThreads;
        keep[i][0] = keep[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p < pieces) {
            keep[i][0] = row[2 * p];
            keep[i][1] = row[2 * p + 1];
        }
    }
    auto most = [](const float4 &v) { return fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))); };
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kRescaleKeep; i++)
        top = fmaxf(top, fmaxf(most(keep[i][0]), most(keep[i][1])));
    for (int p = threadIdx.x + kRescaleKeep * kRescaleThreads; p < pieces; p += kRescaleThreads)
        top = fmaxf(top, fmaxf(most(row[2 * p]), most(row[2 * p + 1])));
    const uint32_t of_warp = __reduce_max_sync(0xffffffffu, __float_as_uint(top)); // floats that are not negative are ordered like their bits
    if ((threadIdx.x & 31) == 0)
        part[threadIdx.x >> 5] = __uint_as_float(of_warp);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRescaleThreads / 32; i++)
        top = fmaxf(top, part[i]);
    const int e = token_exponent(top);
    const float down = pow2f(-e);
    auto store = [&](int p, const float4 &a, const float4 &b) {
        const __half2 o[4] = {__floats2half2_rn(a.x * down, a.y * down), __floats2half2_rn(a.z * down, a.w * down),
                              __floats2half2_rn(b.x * down, b.y * down), __floats2half2_rn(b.z * down, b.w * down)};
        out[p] = *reinterpret_cast<const uint4 *>(o);
    };
#pragma unroll
    for (int i = 0; i < kRescaleKeep; i++)
        if (static_cast<int>(threadIdx.x) + i * kRescaleThreads < pieces)
            store(threadIdx.x + i * kRescaleThreads, keep[i][0], keep[i][1]);
    for (int p = threadIdx.x + kRescaleKeep * kRescaleThreads; p < pieces; p += kRescaleThreads)
        store(p, row[2 * p], row[2 * p + 1]);
    if (threadIdx.x == 0)
        factor[blockIdx.x] = pow2f(e);
}

} // namespace xs
