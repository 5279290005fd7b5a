"""Calls of the dense operators on torch tensors, their definitions in 64 bits, and how far a result may be off."""
import ctypes as C
import math

import torch

from xstar_moe import capi, synth

from gpu_util import stream_ptr

F = torch.float64
HALF = 2.0**-8  # half a bf16 step, relative to the value
ACT = {"silu": capi.SILU, "gelu": capi.GELU_TANH}
GATE = {"none": capi.GATE_NONE, "channel": capi.GATE_CHANNEL, "row": capi.GATE_ROW, "full": capi.GATE_FULL}
EXACT_WEIGHT_TOKENS = 16  # up to here the weights of matrices of up to 8192 columns enter the products unrounded


def workspace(nbytes):
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    capi.check(capi.lib().xs_moe_workspace_init(capi.ptr(ws), nbytes, stream_ptr()))
    return ws


def _bytes(fn, *args):
    n = C.c_size_t(0)
    capi.check(fn(*args, C.byref(n)))
    return n.value


def bf16(gen, shape, std=1.0, mean=0.0, device="cuda"):
    return (torch.randn(shape, generator=gen, device=gen.device) * std + mean).to(torch.bfloat16).to(device)


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def weight(g, rows, cols, group, zeros, std=0.02):
    return synth.int4_groups((rows, cols), group, zeros, std, g, g.device)


def linear(w, x, out=None, ws=None):
    L, m, T = capi.lib(), capi.make_w4(w), x.shape[0]
    ws = workspace(_bytes(L.xs_moe_linear_w4_workspace_bytes, C.byref(m), T)) if ws is None else ws
    out = torch.empty(T, m.rows, dtype=torch.bfloat16, device="cuda") if out is None else out
    capi.check(L.xs_moe_linear_w4(C.byref(m), capi.ptr(x), T, capi.ptr(out), capi.ptr(ws), ws.numel(), stream_ptr()))
    return out, ws


def gated(w, x, act, out=None):
    L, m, T = capi.lib(), capi.make_w4(w), x.shape[0]
    ws = workspace(_bytes(L.xs_moe_linear_w4_workspace_bytes, C.byref(m), T))
    out = torch.empty(T, m.rows // 2, dtype=torch.bfloat16, device="cuda") if out is None else out
    capi.check(L.xs_moe_gated_w4(C.byref(m), ACT[act], capi.ptr(x), T, capi.ptr(out), capi.ptr(ws), ws.numel(), stream_ptr()))
    return out, ws


def mlp(gu, dn, x, act, out=None, ws=None):
    L, a, b, T = capi.lib(), capi.make_w4(gu), capi.make_w4(dn), x.shape[0]
    ws = workspace(_bytes(L.xs_moe_mlp_w4_workspace_bytes, C.byref(a), C.byref(b), T)) if ws is None else ws
    out = torch.empty_like(x) if out is None else out
    capi.check(L.xs_moe_mlp_w4(C.byref(a), C.byref(b), ACT[act], capi.ptr(x), T, capi.ptr(out), capi.ptr(ws), ws.numel(), stream_ptr()))
    return out, ws


def block_norms(pre, post=None, gate=None, kind="none", eps=1e-6, scale=1.0, offset=0.0):
    n = capi.XsMoeBlockNorms()
    n.pre_weight_dev, n.post_weight_dev, n.gate_dev, n.gate_kind = capi.ptr(pre), capi.ptr(post), capi.ptr(gate), GATE[kind]
    n.eps, n.residual_scale, n.weight_offset = eps, scale, offset
    return n


def mlp_block(gu, dn, norms, x, act, out=None, ws=None):
    L, a, b, T = capi.lib(), capi.make_w4(gu), capi.make_w4(dn), x.shape[0]
    ws = workspace(_bytes(L.xs_moe_mlp_w4_block_workspace_bytes, C.byref(a), C.byref(b), T)) if ws is None else ws
    out = torch.empty_like(x) if out is None else out
    capi.check(L.xs_moe_mlp_w4_block(C.byref(a), C.byref(b), ACT[act], C.byref(norms), capi.ptr(x), T, capi.ptr(out), capi.ptr(ws), ws.numel(),
                                     stream_ptr()))
    return out, ws


def flags(ws):
    capi.check(capi.lib().xs_moe_check_flags(capi.ptr(ws), stream_ptr()))


def norm_args(y, r, post=None, gate=None, kind="none", nxt=None, out=None, next_out=None, eps=1e-6, scale=1.0, offset=0.0):
    a = capi.XsMoeNormResidual()
    a.y_dev, a.residual_dev, a.post_weight_dev, a.gate_dev = capi.ptr(y), capi.ptr(r), capi.ptr(post), capi.ptr(gate)
    a.next_weight_dev, a.residual_out_dev, a.next_out_dev = capi.ptr(nxt), capi.ptr(out), capi.ptr(next_out)
    a.gate_kind, a.rows, a.hidden = GATE[kind], r.shape[0], r.shape[1]
    a.eps, a.residual_scale, a.weight_offset = eps, scale, offset
    return a


def norm_residual(args):
    capi.check(capi.lib().xs_moe_norm_residual(C.byref(args), stream_ptr()))


# ---- definitions in 64 bits -----------------------------------------------------------------------------------------
def matrix(w):
    q = w["q"]
    m = torch.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1).to(F)
    groups = w["s"].shape[1]
    g = m.shape[1] // groups
    z = 8.0 if w["z"] is None else (w["z"] & 15).to(F).repeat_interleave(g, 1)
    return (m - z) * w["s"].to(F).repeat_interleave(g, 1)


def activation(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    return v / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))


def rms(v, w, eps, offset):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * (offset + w.to(F))


def ref_norm_residual(y, r, post=None, gate=None, nxt=None, eps=1e-6, scale=1.0, offset=0.0):
    y, r = y.to(F), r.to(F)
    if post is not None:
        y = rms(y, post, eps, offset)
    if gate is not None:
        y = y * (gate.to(F).view(-1, 1) if gate.numel() == r.shape[0] and gate.shape[-1] == 1 else gate.to(F))
    r = r + scale * y
    return r, None if nxt is None else rms(r, nxt, eps, offset)


# ---- how far off ----------------------------------------------------------------------------------------------------
# A sum of K products in f32, in any order, is off by at most K * 2^-23 * sum |product| (2^-23 a step: additions that cut off
# instead of rounding).  Beyond EXACT_WEIGHT_TOKENS the operands are f16: a weight is off by half a step, 2^-11 of itself, and a
# token, scaled to a largest element of 2^13 at least, by 2^-25 in that unit: 2^-38 of its largest element.
F16 = 2.0**-11


def _sum_error(X, W, tokens):
    magnitude = X.abs() @ W.abs().T
    err = X.shape[1] * 2.0**-23 * magnitude
    if tokens > EXACT_WEIGHT_TOKENS or (tokens > 8 and X.shape[1] > 8192):
        err = err + F16 * magnitude + 2.0**-38 * X.abs().amax(-1, keepdim=True) * W.abs().sum(-1)
    return err


def linear_reference(w, x):
    """out in 64 bits and the largest error of each of its elements"""
    W, X = matrix(w), x.to(F)
    ref = X @ W.T
    err = _sum_error(X, W, x.shape[0])
    return ref, HALF * ref.abs() + err * (1 + HALF) + 1e-37


def _gated(w, X, act, tokens, dx=None):
    """h before its rounding, and its error; dx: the error of the elements of X"""
    W = matrix(w)
    I = W.shape[0] // 2
    gu = X @ W.T
    err = _sum_error(X, W, tokens)
    if dx is not None:
        err = err + dx @ W.abs().T * (1 + HALF)
    g, u, dg, du = gu[:, :I], gu[:, I:], err[:, :I], err[:, I:]
    a = activation(g, act)
    # |act'| < 1.13 for both; evaluating it in f32 costs a few steps of its terms (2^-20 of |g| is 16 of them)
    da = 1.13 * dg + 2.0**-20 * g.abs()
    return a * u, da * u.abs() + a.abs() * du + da * du


def gated_reference(w, x, act):
    h, dh = _gated(w, x.to(F), act, x.shape[0])
    return h, HALF * h.abs() + dh * (1 + HALF) + 1e-37


def mlp_reference(gu, dn, x, act, dx=None):
    X = x.to(F)
    h, dh = _gated(gu, X, act, x.shape[0], dx)
    if x.shape[0] > EXACT_WEIGHT_TOKENS:
        # h in f16, scaled by a bound of its row: 2^15 of |x|^2 K max(s_gate s_up) at most, of which f16 keeps 2^-40
        s = gu["s"].to(F).abs().amax(-1)
        bound = 2.0**15 * X.square().sum(-1, keepdim=True) * X.shape[1] * (s[: h.shape[1]] * s[h.shape[1]:]).amax()
        dh = F16 * h.abs() + 2.0**-40 * bound + dh * (1 + F16)
    else:  # h in f16, each token, or its part that is summed together, scaled to a largest element of 2^13 at least
        dh = F16 * h.abs() + 2.0**-38 * (h.abs() + dh).amax(-1, keepdim=True) + dh * (1 + F16)
    D = matrix(dn)
    ref = h @ D.T
    err = _sum_error(h.abs() + dh, D, x.shape[0]) + dh @ D.abs().T
    return ref, HALF * ref.abs() + err * (1 + HALF) + 1e-37


def assert_close(got, ref, tol):
    got = got.to(F)
    bad = (got - ref).abs() > tol
    assert torch.isfinite(got).all(), "not finite"
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got - ref).abs() / tol).max().item():.2f} of the bound"


def rel_l2(got, ref):
    return float((got.to(F) - ref).norm() / ref.norm().clamp_min(1e-300))
