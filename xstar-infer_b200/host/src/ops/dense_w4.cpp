#include "ops/dense_w4.h"

#include <limits>
#include <stdexcept>

#include "cuda/cuda_allocator.h"
#include "ops/moe_checked.h"
#include "xs_moe_dense.h"

using moe_detail::raise_if;

namespace {

std::int32_t as_int32(std::int64_t v)
{
    if (v > std::numeric_limits<std::int32_t>::max())
        throw std::runtime_error("dimension too large");
    return static_cast<std::int32_t>(v);
}

std::int64_t rows_of(const Tensor &x)
{
    return x.dim(-1) ? x.numel() / x.dim(-1) : 0;
}

void check_x(const Tensor &x)
{
    if (x.dtype() != DType::BFloat16)
        throw std::runtime_error("dtype mismatch");
    if (x.rank() < 1)
        throw std::runtime_error("rank mismatch");
}

// dtype, rank, shape, device: the order of the other ops.  K: the columns the caller's operand asks for.
XsMoeW4 checked(const W4Weight &w, const Tensor &x, std::int64_t K)
{
    if (!w.codes || !w.scales)
        throw std::runtime_error("missing weight");
    const Tensor &c = *w.codes, &s = *w.scales;
    if (c.dtype() != DType::UInt4x2 || s.dtype() != DType::BFloat16 || (w.zeros && w.zeros->dtype() != DType::UInt8))
        throw std::runtime_error("dtype mismatch");
    if (c.rank() != 2 || s.rank() != 2 || (w.zeros && w.zeros->rank() != 2))
        throw std::runtime_error("rank mismatch");
    const std::int64_t N = c.dim(0), groups = s.dim(1);
    if (c.dim(1) * 2 != K || K <= 0 || N <= 0 || s.dim(0) != N || groups <= 0 || K % groups != 0 || (w.zeros && w.zeros->shape() != s.shape()))
        throw std::runtime_error("shape mismatch");
    if (c.device() != x.device() || s.device() != x.device() || (w.zeros && w.zeros->device() != x.device()))
        throw std::runtime_error("device mismatch");
    XsMoeW4 m{};
    m.codes_dev = c.data();
    m.scales_dev = s.data();
    m.zeros_dev = w.zeros ? w.zeros->data<std::uint8_t>() : nullptr;
    m.rows = as_int32(N);
    m.cols = as_int32(K);
    m.group = as_int32(K / groups);
    return m;
}

struct Mlp {
    XsMoeW4 gate_up{}, down{};
    std::int32_t tokens = 0, act = 0;
};

Mlp checked_mlp(const Tensor &x, const W4Weight &gate_up, const W4Weight &down, Activation act)
{
    check_x(x);
    Mlp m;
    m.gate_up = checked(gate_up, x, x.dim(-1));
    if (m.gate_up.rows % 2 != 0)
        throw std::runtime_error("gate_up out must be even");
    m.down = checked(down, x, m.gate_up.rows / 2);
    if (m.down.rows != m.gate_up.cols)
        throw std::runtime_error("shape mismatch");
    m.tokens = as_int32(rows_of(x));
    m.act = act == Activation::Silu ? XS_MOE_SILU : XS_MOE_GELU_TANH;
    return m;
}

void check_out(const Tensor &x, const Tensor &out, std::int64_t numel)
{
    if (out.dtype() != DType::BFloat16)
        throw std::runtime_error("dtype mismatch");
    if (out.numel() != numel)
        throw std::runtime_error("shape mismatch");
    if (out.device() != Device::CUDA || x.device() != Device::CUDA)
        throw std::runtime_error("unsupported device");
}

// A scratch that has to grow gives its block back to the pool: wait for the caller's stream first, which may be one that the
// default stream does not wait for.
void prepare(MoEScratch &scratch, std::size_t need, void *stream)
{
    if (scratch.data() && scratch.bytes() < need)
        raise_if(xs_moe_stream_synchronize(stream));
    scratch.reserve(need);
}

std::int32_t gate_kind(const Tensor *gate, const Tensor &x)
{
    if (!gate)
        return XS_MOE_GATE_NONE;
    const std::int64_t H = x.dim(-1), rows = rows_of(x);
    if (gate->dtype() != DType::BFloat16)
        throw std::runtime_error("dtype mismatch");
    if (gate->device() != x.device())
        throw std::runtime_error("device mismatch");
    if (gate->rank() < 1)
        throw std::runtime_error("rank mismatch");
    if (gate->dim(-1) == H && gate->numel() == H)
        return XS_MOE_GATE_CHANNEL;
    if (gate->dim(-1) == H && gate->numel() == x.numel())
        return XS_MOE_GATE_FULL;
    if (gate->dim(-1) == 1 && gate->numel() == rows)
        return XS_MOE_GATE_ROW;
    throw std::runtime_error("shape mismatch");
}

void check_norm_weight(const Tensor *w, const Tensor &x)
{
    if (!w)
        return;
    if (w->dtype() != DType::BFloat16)
        throw std::runtime_error("dtype mismatch");
    if (w->rank() != 1)
        throw std::runtime_error("rank mismatch");
    if (w->dim(0) != x.dim(-1))
        throw std::runtime_error("shape mismatch");
    if (w->device() != x.device())
        throw std::runtime_error("device mismatch");
}

const void *data_of(const Tensor *t)
{
    return t ? t->data() : nullptr;
}

XsMoeBlockNorms block_norms(const Tensor &x, const Tensor &pre, const NormResidual &p)
{
    check_norm_weight(&pre, x);
    check_norm_weight(p.post_norm_weight, x);
    XsMoeBlockNorms n{};
    n.pre_weight_dev = pre.data();
    n.post_weight_dev = data_of(p.post_norm_weight);
    n.gate_dev = data_of(p.gate);
    n.gate_kind = gate_kind(p.gate, x);
    n.eps = p.eps;
    n.residual_scale = p.residual_scale;
    n.weight_offset = p.weight_offset;
    return n;
}

void require_cuda(const Tensor &x)
{
    if (x.device() != Device::CUDA)
        throw std::runtime_error("unsupported device");
}

Tensor::Shape with_last(Tensor::Shape s, std::int64_t n)
{
    s.back() = n;
    return s;
}

} // namespace

Activation activation_of(const std::string &name)
{
    if (name == "silu")
        return Activation::Silu;
    if (name == "gelu")
        return Activation::GeluTanh;
    throw std::runtime_error("unknown activation");
}

void linear_w4_into(const Tensor &x, const W4Weight &weight, Tensor &out, MoEScratch &scratch, void *stream)
{
    check_x(x);
    const XsMoeW4 w = checked(weight, x, x.dim(-1));
    const std::int32_t T = as_int32(rows_of(x));
    check_out(x, out, static_cast<std::int64_t>(T) * w.rows);
    std::size_t need = 0;
    raise_if(xs_moe_linear_w4_workspace_bytes(&w, T, &need));
    prepare(scratch, need, stream);
    raise_if(xs_moe_linear_w4(&w, x.data(), T, out.data(), scratch.data(), scratch.bytes(), stream));
}

Tensor linear_w4(const Tensor &x, const W4Weight &weight)
{
    check_x(x);
    const XsMoeW4 w = checked(weight, x, x.dim(-1));
    require_cuda(x);
    const std::int32_t T = as_int32(rows_of(x));
    std::size_t need = 0;
    raise_if(xs_moe_linear_w4_workspace_bytes(&w, T, &need));
    Tensor out = Tensor::result(with_last(x.shape(), w.rows), DType::BFloat16);
    Workspace ws(need);
    raise_if(xs_moe_linear_w4(&w, x.data(), T, out.data(), ws.data(), ws.bytes(), nullptr));
    raise_if(xs_moe_check_flags(ws.data(), nullptr));
    return out;
}

void mlp_w4_into(const Tensor &x, const W4Weight &gate_up, const W4Weight &down, Activation act, Tensor &out, MoEScratch &scratch, void *stream)
{
    const Mlp m = checked_mlp(x, gate_up, down, act);
    check_out(x, out, x.numel());
    std::size_t need = 0;
    raise_if(xs_moe_mlp_w4_workspace_bytes(&m.gate_up, &m.down, m.tokens, &need));
    prepare(scratch, need, stream);
    raise_if(xs_moe_mlp_w4(&m.gate_up, &m.down, m.act, x.data(), m.tokens, out.data(), scratch.data(), scratch.bytes(), stream));
}

Tensor mlp_w4(const Tensor &x, const W4Weight &gate_up, const W4Weight &down, Activation act)
{
    const Mlp m = checked_mlp(x, gate_up, down, act);
    require_cuda(x);
    std::size_t need = 0;
    raise_if(xs_moe_mlp_w4_workspace_bytes(&m.gate_up, &m.down, m.tokens, &need));
    Tensor out = Tensor::result(x.shape(), DType::BFloat16);
    Workspace ws(need);
    raise_if(xs_moe_mlp_w4(&m.gate_up, &m.down, m.act, x.data(), m.tokens, out.data(), ws.data(), ws.bytes(), nullptr));
    raise_if(xs_moe_check_flags(ws.data(), nullptr));
    return out;
}

void norm_residual_into(const Tensor &y, const Tensor &residual, const NormResidual &p, Tensor &out, Tensor *next_out, void *stream)
{
    check_x(y);
    if (residual.dtype() != DType::BFloat16)
        throw std::runtime_error("dtype mismatch");
    if (residual.shape() != y.shape())
        throw std::runtime_error("shape mismatch");
    if (residual.device() != y.device())
        throw std::runtime_error("device mismatch");
    check_norm_weight(p.post_norm_weight, y);
    check_norm_weight(p.next_norm_weight, y);
    if ((p.next_norm_weight != nullptr) != (next_out != nullptr))
        throw std::runtime_error("next_norm_weight and next_out go together");
    const std::int32_t kind = gate_kind(p.gate, y);
    check_out(y, out, y.numel());
    if (next_out)
        check_out(y, *next_out, y.numel());
    XsMoeNormResidual a{};
    a.y_dev = y.data();
    a.residual_dev = residual.data();
    a.post_weight_dev = data_of(p.post_norm_weight);
    a.gate_dev = data_of(p.gate);
    a.next_weight_dev = data_of(p.next_norm_weight);
    a.residual_out_dev = out.data();
    a.next_out_dev = next_out ? next_out->data() : nullptr;
    a.gate_kind = kind;
    a.rows = as_int32(rows_of(y));
    a.hidden = as_int32(y.dim(-1));
    a.eps = p.eps;
    a.residual_scale = p.residual_scale;
    a.weight_offset = p.weight_offset;
    if (a.rows == 0)
        return;
    raise_if(xs_moe_norm_residual(&a, stream));
}

NormResidualResult norm_residual(const Tensor &y, const Tensor &residual, const NormResidual &p)
{
    check_x(y);
    require_cuda(y);
    NormResidualResult r{Tensor::result(y.shape(), DType::BFloat16), Tensor()};
    if (p.next_norm_weight)
        r.next = Tensor::result(y.shape(), DType::BFloat16);
    norm_residual_into(y, residual, p, r.residual, p.next_norm_weight ? &r.next : nullptr, nullptr);
    raise_if(xs_moe_stream_synchronize(nullptr));
    return r;
}

void mlp_w4_block_into(const Tensor &x, const Tensor &pre_norm_weight, const W4Weight &gate_up, const W4Weight &down, Activation act,
                       const NormResidual &p, Tensor &out, MoEScratch &scratch, void *stream)
{
    const Mlp m = checked_mlp(x, gate_up, down, act);
    const XsMoeBlockNorms n = block_norms(x, pre_norm_weight, p);
    check_out(x, out, x.numel());
    std::size_t need = 0;
    raise_if(xs_moe_mlp_w4_block_workspace_bytes(&m.gate_up, &m.down, m.tokens, &need));
    prepare(scratch, need, stream);
    raise_if(xs_moe_mlp_w4_block(&m.gate_up, &m.down, m.act, &n, x.data(), m.tokens, out.data(), scratch.data(), scratch.bytes(), stream));
}

Tensor mlp_w4_block(const Tensor &x, const Tensor &pre_norm_weight, const W4Weight &gate_up, const W4Weight &down, Activation act,
                    const NormResidual &p)
{
    const Mlp m = checked_mlp(x, gate_up, down, act);
    const XsMoeBlockNorms n = block_norms(x, pre_norm_weight, p);
    require_cuda(x);
    std::size_t need = 0;
    raise_if(xs_moe_mlp_w4_block_workspace_bytes(&m.gate_up, &m.down, m.tokens, &need));
    Tensor out = Tensor::result(x.shape(), DType::BFloat16);
    Workspace ws(need);
    raise_if(xs_moe_mlp_w4_block(&m.gate_up, &m.down, m.act, &n, x.data(), m.tokens, out.data(), ws.data(), ws.bytes(), nullptr));
    raise_if(xs_moe_check_flags(ws.data(), nullptr));
    return out;
}

void moe_block_into(const Tensor &x, const Tensor &pre_norm_weight, const MoEWeights &weights, const MoEConfig &config, const NormResidual &p,
                    Tensor &out, MoEScratch &scratch, void *stream)
{
    moe_detail::Checked c = moe_detail::validate(x, weights, config, true);
    const XsMoeBlockNorms n = block_norms(x, pre_norm_weight, p);
    check_out(x, out, x.numel());
    std::size_t need = 0;
    raise_if(xs_moe_normed_block_workspace_bytes(&c.cfg, &need));
    prepare(scratch, need, stream);
    raise_if(xs_moe_normed_block_forward(&c.cfg, &c.w, &n, x.data(), out.data(), scratch.data(), scratch.bytes(), stream));
}

Tensor moe_block(const Tensor &x, const Tensor &pre_norm_weight, const MoEWeights &weights, const MoEConfig &config, const NormResidual &p)
{
    moe_detail::Checked c = moe_detail::validate(x, weights, config, true);
    const XsMoeBlockNorms n = block_norms(x, pre_norm_weight, p);
    require_cuda(x);
    std::size_t need = 0;
    raise_if(xs_moe_normed_block_workspace_bytes(&c.cfg, &need));
    Tensor out = Tensor::result(x.shape(), DType::BFloat16);
    Workspace ws(need);
    raise_if(xs_moe_normed_block_forward(&c.cfg, &c.w, &n, x.data(), out.data(), ws.data(), ws.bytes(), nullptr));
    raise_if(xs_moe_check_flags(ws.data(), nullptr));
    return out;
}
