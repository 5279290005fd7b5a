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


# ---- every kernel and both conversions, at the precision that they state ---------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_and_gated_add_little_to_the_rounding_of_their_result(group, zeros):
    g = du.gen(group)
    K, N = 2048, 2 * I
    w, x = du.weight(g, N, K, group, zeros), du.bf16(g, (530, K))
    wide = dict(w, s=(w["s"].float() * 2.0 ** torch.randint(-6, 7, w["s"].shape, generator=g, device="cuda")).to(torch.bfloat16))
    for m in (w, wide):
        W = du.matrix(m)
        ref = x.to(du.F) @ W.T
        h = {act: du.activation(ref[:, :I], act) * ref[:, I:] for act in ("silu", "gelu")}
        for T in (1, 5, 9, 16, 17, 64, 65, 128, 260, 530):
            out, ws = du.linear(m, x[:T])
            du.flags(ws)
            assert_exact(out, ref[:T], D_LINEAR)
            for act in h:
                out, ws = du.gated(m, x[:T], act)
                du.flags(ws)
                assert_exact(out, h[act][:T], D_MLP)


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T", [3, 16, 17, 90, 300])
def test_linear_with_scales_a_millionth_of_their_rows_largest(T, zeros):
    # groups of small scales meet tokens that are large there, so that every group counts alike: 2^20 is what the weights' eleven bits reach down to
    g = du.gen(T)
    K, N, group = 1024, 1024, 32
    w, x = du.weight(g, N, K, group, zeros), du.bf16(g, (T, K))
    power = torch.arange(K // group, device="cuda") % 21
    # every row has a largest scale of its own and no scale more than 2^20 below it
    w["s"] = (w["s"].float().clamp(2.0**-8, 2.0**-7) * 2.0**-power).to(torch.bfloat16)
    x = (x.float() * 2.0 ** power.repeat_interleave(group)).to(torch.bfloat16)
    out, ws = du.linear(w, x)
    du.flags(ws)
    assert_exact(out, x.to(du.F) @ du.matrix(w).T, D_LINEAR)


@pytest.mark.gpu
@pytest.mark.parametrize("T, H, I", [(20, 64, 12288), (20, 64, 12320), (200, 32, 16416), (17, 128, 40000)])
def test_mlp_with_a_long_gated_product(T, H, I):
    # more of it than a block keeps in registers while it finds its scale
    g = du.gen(I)
    gu, dn = du.weight(g, 2 * I, H, 32, False, std=H**-0.5), du.weight(g, H, I, 32, True, std=I**-0.5)
    x = du.bf16(g, (T, H))
    x[1] *= 2.0**-9
    x[2] = 0.0
    out, ws = du.mlp(gu, dn, x, "gelu")
    du.flags(ws)
    ref = mlp_exact(gu, dn, x, "gelu")
    assert (out[2] == 0).all()
    keep = torch.arange(T, device="cuda") != 2
    got, ref = out[keep].to(du.F), ref[keep]
    # few columns a row: all rows but the small one together, then the small one by the largest that its rounding may cost
    assert du.rel_l2(got[2:], ref[2:]) < allowed(ref[2:].reshape(1, -1), D_MLP).item()
    assert du.rel_l2(got[1], ref[1]) < du.HALF + D_MLP


@pytest.mark.gpu
def test_mlp_whose_gated_product_goes_through_memory_in_parts():
    # 2^19 columns: 256 tokens at a time; the second part has 44
    T, H, I = 300, 32, 2**19
    g = du.gen(19)
    gu, dn = du.weight(g, 2 * I, H, 32, False, std=H**-0.5), du.weight(g, H, I, 128, False, std=I**-0.5)
    x = (du.bf16(g, (T, H)).float() * 2.0 ** torch.randint(-3, 4, (T, 1), generator=g, device="cuda")).to(torch.bfloat16)
    out, ws = du.mlp(gu, dn, x, "gelu")
    du.flags(ws)
    ref = mlp_exact(gu, dn, x, "gelu")
    for rows in (slice(0, 256), slice(256, T)):  # a tensor of rows of its own size, each brought to its norm
        unit = ref[rows].norm(dim=-1, keepdim=True)
        assert du.rel_l2(out[rows].to(du.F) / unit, ref[rows] / unit) < allowed(ref[rows].reshape(1, -1), D_MLP + I**0.5 * 2.0**-23).item()
    few = du.mlp(gu, dn, x[256:].contiguous(), "gelu")[0]  # a tile of another shape sums in another order
    assert du.rel_l2(few, out[256:].to(du.F)) < du.HALF


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 17, 300])
def test_mlp_gives_the_same_bits_each_time_and_for_each_token(T):
    gu, dn, g = _mlp(300 + T, True)
    x = du.bf16(g, (T, H))
    a, ws = du.mlp(gu, dn, x, "silu")
    for _ in range(5):
        assert torch.equal(du.mlp(gu, dn, x, "silu", ws=ws)[0], a)
    x[T // 2] = 3.0e4  # a token's scale, and its result, are its own
    b, _ = du.mlp(gu, dn, x, "silu", ws=ws)
    b[T // 2] = a[T // 2]
    assert torch.equal(a, b)


E = 0.0017  # rounding to bf16, in the root mean square


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 16, 17, 130, 300])
@pytest.mark.parametrize("post", [False, True])
def test_block_adds_the_roundings_that_it_states(T, post):
    """The branch is rounded to bf16 before it is added, and up to 16 tokens the normed rows before they are multiplied: E relative to
    the branch, and E through gate and up.  The sum's own rounding is e of the sum, as above.
    An element's error is in proportion to gate times branch, both normal: the squares of these errors have the fourth moment 3 * 3, and
    uniform roundings 1.8, so that the sum over 1024 of them spreads by sqrt((9 * 1.8 - 1) / 1024) = 0.12, its root by 0.06: 1.2 is three times that."""
    gu, dn, g = _mlp(400 + T, True)
    x = du.bf16(g, (T, H), 0.5)
    pre, after = du.bf16(g, (H,), 0.1, 1.0), du.bf16(g, (H,), 0.1, 1.0)
    gate = du.bf16(g, (H,))
    out, ws = du.mlp_block(gu, dn, du.block_norms(pre, after if post else None, gate, "channel", 1e-6, 0.5), x, "silu")
    du.flags(ws)
    y = mlp_exact(gu, dn, du.rms(x.to(du.F), pre, 1e-6, 0.0), "silu")
    branch = 0.5 * gate.to(du.F) * (du.rms(y, after, 1e-6, 0.0) if post else y)
    ref = x.to(du.F) + branch
    d = (D_MLP**2 + E**2 * (1 + (1.1**2 + 1 if T <= 16 else 0))) ** 0.5
    e = (ref.to(torch.bfloat16).to(du.F) - ref).norm(dim=-1)
    off = (out.to(du.F) - ref).norm(dim=-1)
    most = torch.sqrt((1.05 * e) ** 2 + (1.2 * d * branch.norm(dim=-1)) ** 2)
    assert (off <= most).all(), f"worst row {(off / most).max().item():.2f} of the bound"
