// Dense operators with 4-bit integer weights, and the norm / gate / residual step between two blocks.  Same op conventions as
// ops/moe.h: borrowed const inputs, optional inputs as pointers, a new owned Tensor by value, std::runtime_error with the
// reference's short messages, and `_into` stream forms that enqueue on a stream of the caller's and return.
//
// This header is CUDA-free; the device work is reached through the C ABI in include/xs_moe_dense.h, which states the formulas.
//
//   W4Weight      W[n][k] = (code - zero) * scale
//     codes       (N, K/2)   UInt4x2   (the last dimension counts bytes; the even column is the low nibble)
//     scales      (N, K/g)   BFloat16  g = 32, 64 or 128, read off the shapes
//     zeros       (N, K/g)   UInt8     or null: 8
//   x             (..., K)   bf16, leading dims collapsed to T rows
//
// Device::CPU inputs are rejected ("unsupported device").
#pragma once
#include <cstdint>
#include <string>

#include "ops/moe.h"
#include "tensor.h"

struct W4Weight {
    const Tensor *codes = nullptr;
    const Tensor *scales = nullptr;
    const Tensor *zeros = nullptr;
};

enum class Activation { Silu, GeluTanh };
Activation activation_of(const std::string &name); // "silu" | "gelu"; throws "unknown activation"

// x W^T: the engine's linear(x, weight) (reference xstar_cpp/include/ops/linear.h) with a 4-bit weight; (..., N) bf16.
Tensor linear_w4(const Tensor &x, const W4Weight &weight);
void linear_w4_into(const Tensor &x, const W4Weight &weight, Tensor &out, MoEScratch &scratch, void *stream);

// (act(x Wg^T) * (x Wu^T)) Wd^T: the engine's mlp(x, gate_up_weight, down_weight) (reference xstar_cpp/include/ops/mlp.h:51) with
// 4-bit weights, gate_up (2I, H) with the gate rows first, down (H, I).
Tensor mlp_w4(const Tensor &x, const W4Weight &gate_up, const W4Weight &down, Activation act = Activation::Silu);
void mlp_w4_into(const Tensor &x, const W4Weight &gate_up, const W4Weight &down, Activation act, Tensor &out, MoEScratch &scratch, void *stream);

// r' = residual + residual_scale * gate . N(y; post_norm_weight);  n = N(r'; next_norm_weight)
// with N(v; w) = v / sqrt(mean(v^2) + eps) * (weight_offset + w).  The gate's shape says what it is: (H) or (1, H) per channel,
// (rows, 1) per row, the shape of y per element.  Shapes that fit two of these say the same thing both ways.
struct NormResidual {
    float eps = 1e-6f;
    const Tensor *post_norm_weight = nullptr;
    const Tensor *gate = nullptr;
    float residual_scale = 1.0f;
    float weight_offset = 0.0f;
    const Tensor *next_norm_weight = nullptr;
};
// next_out: written when p.next_norm_weight is given (then it must not be null).  out may be residual or y itself.
void norm_residual_into(const Tensor &y, const Tensor &residual, const NormResidual &p, Tensor &out, Tensor *next_out, void *stream);
struct NormResidualResult {
    Tensor residual;
    Tensor next; // empty without next_norm_weight
};
NormResidualResult norm_residual(const Tensor &y, const Tensor &residual, const NormResidual &p);

// One feed-forward half block, x + residual_scale * gate . N(F(N(x; pre_norm_weight)); post_norm_weight) with F = mlp_w4
// (p.next_norm_weight is not used), and the same around the MoE layer: moe_block with a norm, a gate and a scale on its branch.
Tensor mlp_w4_block(const Tensor &x, const Tensor &pre_norm_weight, const W4Weight &gate_up, const W4Weight &down, Activation act,
                    const NormResidual &p);
void mlp_w4_block_into(const Tensor &x, const Tensor &pre_norm_weight, const W4Weight &gate_up, const W4Weight &down, Activation act,
                       const NormResidual &p, Tensor &out, MoEScratch &scratch, void *stream);
Tensor moe_block(const Tensor &x, const Tensor &pre_norm_weight, const MoEWeights &weights, const MoEConfig &config, const NormResidual &p);
void moe_block_into(const Tensor &x, const Tensor &pre_norm_weight, const MoEWeights &weights, const MoEConfig &config, const NormResidual &p,
                    Tensor &out, MoEScratch &scratch, void *stream);
