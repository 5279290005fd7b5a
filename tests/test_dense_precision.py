"""How exact the dense operators are beyond the rounding of their result.

A result is compared with its definition in 64 bits.  Rounding that definition to bf16 costs e, measured on the definition itself
(2^-8 / sqrt(3) relative at most in the root mean square, about 0.0017).  What the operator may add to it is d, from the roundings
that it makes on the way, each uniform within half a step:
  a weight in f16          2^-11 / sqrt(3) of itself = 2.8e-4      (more than 16 tokens)
  the gated product in f16 2^-11 / sqrt(3) = 2.8e-4
The errors of a sum's terms are independent of one another and of the tokens, so a sum is off by as much relative to its own root mean square.  A linear
product of rounded weights: 2.8e-4.  An MLP: gate and up, each a product (the slope of the activation times its argument is at
most 1.1 times its value in the root mean square), the rounding of h, and the down product: 2.8e-4 * sqrt(1.1^2 + 1 + 1 + 1) = 5.7e-4.
f32 sums add 2^-24 sqrt(K) at most.  D below is the next power of two above these; weights of eight bits instead of eleven would add
2^-9 / sqrt(3) = 1.1e-3 a product.  The two add in quadrature, and 1.05 covers the spread of e over 1024 elements and more (1 / sqrt(2 * 1024) = 2 %)."""
import pytest
import torch

import dense_util as du

D_LINEAR = 2.0**-11
D_MLP = 2.0**-10


def allowed(ref, d):
    """largest relative L2 error of each row"""
    ref = ref.to(du.F)
    e = (ref.to(torch.bfloat16).to(du.F) - ref).norm(dim=-1) / ref.norm(dim=-1)
    return torch.sqrt((1.05 * e) ** 2 + d * d)


def rows_off(got, ref):
    return (got.to(du.F) - ref).norm(dim=-1) / ref.norm(dim=-1)


def assert_exact(got, ref, d):
    off, most = rows_off(got, ref), allowed(ref, d)
    assert torch.isfinite(got).all()
    assert (off <= most).all(), f"worst row {(off / most).max().item():.2f} of the bound, off by {off.max().item():.2e}"


def mlp_exact(gu, dn, x, act):
    W, I = du.matrix(gu), gu["q"].shape[0] // 2
    g, u = x.to(du.F) @ W[:I].T, x.to(du.F) @ W[I:].T
    return (du.activation(g, act) * u) @ du.matrix(dn).T


H, I = 1024, 768


def _mlp(seed, zeros):
    g = du.gen(seed)
    return du.weight(g, 2 * I, H, 128, zeros), du.weight(g, H, I, 128, zeros), g


def _silence_column(w, k):
    """weights of column k exactly zero: its codes become the zero point"""
    group = 2 * w["q"].shape[1] // w["s"].shape[1]
    z = torch.full_like(w["q"][:, 0], 8) if w["z"] is None else w["z"][:, k // group] & 15
    byte = w["q"][:, k // 2]
    w["q"][:, k // 2] = (byte & 0x0F) | (z << 4) if k % 2 else (byte & 0xF0) | z


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("power", [0, 8, 12, 16, 20, 24])
def test_mlp_beside_a_large_element_of_a_token_that_no_weight_takes(power, zeros):
    # the norm of a token says nothing about the size of its gated product
    gu, dn, g = _mlp(power, zeros)
    _silence_column(gu, 77)
    x = du.bf16(g, (300, H))
    x[:, 77] = 2.0**power
    ref = mlp_exact(gu, dn, x, "silu")
    for T in (1, 16, 17, 40, 130, 300):
        out, ws = du.mlp(gu, dn, x[:T], "silu")
        du.flags(ws)
        assert_exact(out, ref[:T], D_MLP)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [0, 12, 16, 24, 40])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_mlp_beside_a_large_gate_row_whose_product_vanishes(power, act):
    # nor does the largest scale of a row: here the feature's up row is zero
    gu, dn, g = _mlp(100 + power, False)
    gu["s"][5] *= 2.0**power
    gu["q"][I + 5] = 0x88
    x = du.bf16(g, (300, H))
    ref = mlp_exact(gu, dn, x, act)
    for T in (1, 16, 17, 40, 130, 300):
        out, ws = du.mlp(gu, dn, x[:T], act)
        du.flags(ws)
        assert_exact(out, ref[:T], D_MLP)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [16, 17, 90, 300])
def test_mlp_with_strongly_negative_gates(T):
    # silu(g) u of order e^-30: far below what the norms of token and weights allow
    gu, dn, g = _mlp(200, False)
    gu["q"][:I] = 0x99  # every gate weight is its scale
    gu["s"][:I] = 2.0**-6
    x = (du.bf16(g, (T, H)).float() * 0.05 - 2.0).to(torch.bfloat16)  # gates near -2 * 1024 / 64 = -32
    out, ws = du.mlp(gu, dn, x, "silu")
    du.flags(ws)
    ref = mlp_exact(gu, dn, x, "silu")
    # the exponential turns an error of the argument into one of the value: f32 sums of 1024 terms of one sign are off by at most 1024 * 2^-23 * 32
    assert_exact(out, ref, D_MLP + 1024 * 2.0**-23 * 32)
