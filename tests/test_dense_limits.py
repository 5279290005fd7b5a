"""The dense operators at the edges of what they accept: the longest rows, empty batches, the largest and smallest factors."""
import ctypes as C

import pytest
import torch

from xstar_moe import capi

import dense_util as du
from bridge import xstar_cpp as xs


def _w4(rows, cols, group=128):
    w = capi.XsMoeW4()
    w.codes_dev = w.scales_dev = 4096
    w.rows, w.cols, w.group = rows, cols, group
    return w


# ---- no GPU needed ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 12, 16])
@pytest.mark.parametrize("cols", [2**24, 2**27, 2**28 - 2048, 2**28, 400_000_000, 480_000_000, 2**29, 2**30 - 2**16, 2**30 - 128, 2**30])
def test_rows_that_no_shared_memory_holds_ask_for_the_scratch_of_larger_batches(tokens, cols):
    """a token of 2^24 columns is 32 MB: such a batch is made ready in the workspace (two bytes a column), whatever 32 bits make of its size"""
    L, n = capi.lib(), C.c_size_t(0)
    w = _w4(8, cols // 128 * 128)
    assert L.xs_moe_linear_w4_workspace_bytes(C.byref(w), tokens, C.byref(n)) == 0
    assert n.value > 2 * tokens * w.cols
    if 2 * w.cols <= 2**30:  # rows of the gate and up matrix
        gate_up, down = _w4(2 * w.cols, 128), _w4(128, w.cols)
        assert L.xs_moe_mlp_w4_workspace_bytes(C.byref(gate_up), C.byref(down), tokens, C.byref(n)) == 0
        assert n.value > 2 * tokens * w.cols + 2 * gate_up.rows


def test_the_workspace_of_an_mlp_grows_by_what_its_tokens_need():
    """tokens and gated product in 16 bits, and no more than half a gigabyte of that product in 32"""
    L, n, h, i = capi.lib(), C.c_size_t(0), 4096, 12288
    last = 0
    for tokens in (1, 16, 17, 512, 8192, 10752, 10753, 16384, 65536, 2**20):
        assert L.xs_moe_mlp_w4_workspace_bytes(C.byref(_w4(2 * i, h)), C.byref(_w4(h, i)), tokens, C.byref(n)) == 0
        assert last <= n.value, "a workspace for more tokens serves fewer"
        last = n.value
        weights = 3 * h * i // 128 * 3 + 4 * (2 * i + h)
        assert n.value <= tokens * (2 * h + 2 * i + 4) + min(4 * tokens * i, 2**29) + weights + 2**14


# ---- no tokens --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["none", "channel", "row", "full"])
def test_empty_batches_do_nothing_and_need_no_addresses(kind):
    """a tensor without elements has no address: the gate of an empty batch, its rows and its result"""
    L = capi.lib()
    gate = 4096 if kind == "channel" else None
    a = capi.XsMoeNormResidual()
    a.gate_dev, a.gate_kind, a.rows, a.hidden, a.eps = gate, du.GATE[kind], 0, 64, 1e-6
    a.post_weight_dev = a.next_weight_dev = 4096
    assert L.xs_moe_norm_residual(C.byref(a), None) == 0
    n = capi.XsMoeBlockNorms()
    n.pre_weight_dev, n.gate_dev, n.gate_kind, n.eps = 4096, gate, du.GATE[kind], 1e-6
    assert L.xs_moe_mlp_w4_block(C.byref(_w4(256, 64, 64)), C.byref(_w4(64, 128, 64)), 0, C.byref(n), None, 0, None, None, 0, None) == 0
    cfg = capi.make_config(T=0, H=512, E=16, K=4, I=256, S=0)
    assert L.xs_moe_normed_block_forward(C.byref(cfg), C.byref(capi.XsMoeWeights()), C.byref(n), None, None, None, 0, None) == 0
    # what is wrong without tokens is wrong all the same
    n.gate_kind = 4
    assert L.xs_moe_mlp_w4_block(C.byref(_w4(256, 64, 64)), C.byref(_w4(64, 128, 64)), 0, C.byref(n), None, 0, None, None, 0, None) == -1
    if kind != "none":
        n.gate_dev, n.gate_kind = None, du.GATE[kind]
        assert L.xs_moe_mlp_w4_block(C.byref(_w4(256, 64, 64)), C.byref(_w4(64, 128, 64)), 0, C.byref(n), 4096, 3, 4096, None, 0, None) == -1


@pytest.mark.gpu
def test_host_ops_take_empty_tensors_without_an_address():
    g = du.gen(1)
    gu_, dn, w = du.weight(g, 256, 512, 64, False), du.weight(g, 512, 128, 64, False), du.bf16(g, (512,))
    view = lambda t, kind=xs.DType.BFloat16: xs.from_device_ptr(t.data_ptr(), list(t.shape), kind)
    none = lambda *shape: xs.from_device_ptr(0, list(shape), xs.DType.BFloat16)
    mats = [view(gu_["q"], xs.DType.UInt4x2), view(gu_["s"]), view(dn["q"], xs.DType.UInt4x2), view(dn["s"])]
    for gate in (None, view(w), none(0, 1), none(0, 512)):
        assert xs.mlp_w4_block(none(0, 512), view(w), *mats, gate=gate).shape() == [0, 512]
        r, n = xs.norm_residual(none(0, 512), none(0, 512), gate=gate, next_norm_weight=view(w))
        assert r.shape() == n.shape() == [0, 512]
    assert xs.linear_w4(none(2, 0, 512), *mats[:2]).shape() == [2, 0, 256]
    assert xs.mlp_w4(none(0, 512), *mats).shape() == [0, 512]


# ---- long rows --------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("T, K", [(1, 2**30), (9, 480_000_000)])
def test_the_longest_rows(T, K):
    # a tile of the first takes 0.4 s, in one wait of its epilogue
    N, group = 5, 128
    q = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device="cuda")
    s = torch.ones(N, K // group, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    want = torch.zeros(T, N, dtype=torch.float64)
    columns = [0, 255, 256, 100_001, K // 8 - 1, K // 8, K // 2 - 1, K // 2 + 77, K - 257, K - 1]
    for i, k in enumerate(columns):
        for n in range(N):
            code = (3 * i + 5 * n) % 16
            byte = int(q[n, k // 2])
            q[n, k // 2] = (byte & 0x0F) | code << 4 if k % 2 else (byte & 0xF0) | code
            for t in range(T):
                want[t, n] += (code - 8) * 2.0 ** ((i + t) % 3)
        for t in range(T):
            x[t, k] = 2.0 ** ((i + t) % 3)
    out, ws = du.linear(dict(q=q, s=s, z=None), x)
    du.flags(ws)
    assert torch.equal(out.cpu().to(torch.float64), want)  # small whole numbers: exact in every step


# ---- the range of f32 -------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("T", [4, 17, 40, 130, 300])
@pytest.mark.parametrize("x_power, s_power", [(122, -70), (-100, 90), (60, -60), (-60, 50), (118, -6)])
def test_tokens_and_scales_at_opposite_ends_of_the_range(T, x_power, s_power):
    # the result is within f32, whatever the order of its factors would give (the last pair: up to 1e38)
    g = du.gen(T)
    N, K = 200, 512
    w, x = du.weight(g, N, K, 32, True), du.bf16(g, (T, K))
    x = (x.float().clamp(-3.9, 3.9) * 2.0**x_power).to(torch.bfloat16)
    # every other row of even scales, and of scales 2^14 apart: both kinds that the conversion knows
    spread = torch.randint(0, 15, w["s"].shape, generator=g, device="cuda") * (torch.arange(N, device="cuda") % 2).view(N, 1)
    w["s"] = (w["s"].float() * 2.0 ** (spread + s_power)).to(torch.bfloat16)
    out, ws = du.linear(w, x)
    du.flags(ws)
    ref, tol = du.linear_reference(w, x)
    du.assert_close(out, ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 17, 130])
def test_a_gated_product_just_below_the_largest_number(T):
    # 2 a a = 3.4021e38, between 3.4e38 and the largest f32: a number like any other
    H = I = 32
    a = 181 / 128 * 2.0**63
    gu = dict(q=torch.full((2 * I, H // 2), 0x88, dtype=torch.uint8, device="cuda"), s=torch.ones(2 * I, 1, dtype=torch.bfloat16, device="cuda"), z=None)
    dn = dict(q=torch.full((H, I // 2), 0x88, dtype=torch.uint8, device="cuda"), s=torch.full((H, 1), 2.0**-64, dtype=torch.bfloat16, device="cuda"), z=None)
    gu["q"][0, 0] = gu["q"][I, 0] = 0x89  # gate and up of the first feature: 1 times their scale
    gu["s"][0] = 2.0
    dn["q"][:, 0] = 0x89
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = a
    out, ws = du.mlp(gu, dn, x, "silu")
    du.flags(ws)
    want = 2 * a * a * 2.0**-64
    assert ((out.to(du.F) - want).abs() <= (du.HALF + 2.0**-11) * want).all()
