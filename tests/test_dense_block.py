"""The dense operators as a layer uses them: one after the other, on streams, in graphs, through the host ops, around the MoE layer."""
import ctypes as C

import pytest
import torch

from xstar_moe import capi, synth

import dense_util as du
import gpu_util as gu
from bridge import xstar_cpp as xs

pytestmark = pytest.mark.gpu
L2 = 2.0**-7


def view(t, kind=None):
    return None if t is None else xs.from_device_ptr(t.data_ptr(), list(t.shape), xs.DType.BFloat16 if kind is None else kind)


def w4_views(w):
    return view(w["q"], xs.DType.UInt4x2), view(w["s"]), view(w["z"], xs.DType.UInt8)


def to_torch(t, shape):
    return torch.from_numpy(xs.to_numpy_raw(xs.to_cpu(t)).view("uint16").copy()).view(torch.bfloat16).view(shape)


def layer(seed, H, I, group, zeros):
    g = du.gen(seed)
    return dict(gu=du.weight(g, 2 * I, H, group, zeros, std=H**-0.5), dn=du.weight(g, H, I, group, zeros, std=I**-0.5),
                pre=du.bf16(g, (H,), 0.1, 1.0), post=du.bf16(g, (H,), 0.1, 1.0)), g


def by_definition(p, x, act, post, gate, scale, offset, eps):
    """the block in 64 bits, rounded only where its parts hand rows to one another"""
    bf = lambda t: t.to(torch.bfloat16).to(du.F)
    xn = bf(du.rms(x.to(du.F), p["pre"], eps, offset))
    gu_, I = xn @ du.matrix(p["gu"]).T, p["gu"]["q"].shape[0] // 2
    y = bf(bf(du.activation(gu_[:, :I], act) * gu_[:, I:]) @ du.matrix(p["dn"]).T)
    return du.ref_norm_residual(y, x, p["post"] if post else None, gate, None, eps, scale, offset)[0]


def branch_error(out, ref, x):
    """distance relative to what the block adds to x, less the rounding of the sum"""
    return float(((out.to(du.F) - ref).abs() - du.HALF * ref.abs()).clamp_min(0).norm() / (ref - x.to(du.F)).norm())


@pytest.mark.parametrize("T", [1, 4, 16, 17, 130, 700])
@pytest.mark.parametrize("kind, post, act, scale, offset", [("none", False, "silu", 1.0, 0.0), ("channel", True, "gelu", 0.5, 1.0), ("row", True, "silu", 0.22, 0.0),
                                                            ("full", True, "silu", 1.0, 0.0)])
def test_block_is_its_parts_and_its_definition(T, kind, post, act, scale, offset):
    p, g = layer(T, 640, 896, 64, kind != "row")
    x = du.bf16(g, (T, 640), 1.5)
    shape = {"none": None, "channel": (640,), "row": (T, 1), "full": (T, 640)}[kind]
    gate = None if shape is None else du.bf16(g, shape)
    norms = du.block_norms(p["pre"], p["post"] if post else None, gate, kind, 1e-5, scale, offset)
    out, ws = du.mlp_block(p["gu"], p["dn"], norms, x, act)
    du.flags(ws)
    # the parts, called one by one
    xn, r = torch.empty_like(x), torch.empty_like(x)
    du.norm_residual(du.norm_args(None, x, nxt=p["pre"], next_out=xn, eps=1e-5, offset=offset))
    y, _ = du.mlp(p["gu"], p["dn"], xn, act)
    du.norm_residual(du.norm_args(y, x, p["post"] if post else None, gate, kind, None, r, eps=1e-5, scale=scale, offset=offset))
    if T <= du.EXACT_WEIGHT_TOKENS:  # larger batches are normed on the way to the tensor core, without a rounding to bf16
        assert torch.equal(out, r)
    else:
        assert branch_error(out, r.to(du.F), x) < 2 * L2
    ref = by_definition(p, x, act, post, None if gate is None else gate.expand(T, 640), scale, offset, 1e-5)
    assert branch_error(out, ref, x) < L2
    # over its own input, as a residual stream is kept
    x2 = x.clone()
    du.mlp_block(p["gu"], p["dn"], norms, x2, act, out=x2)
    assert torch.equal(x2, out)


@pytest.mark.parametrize("T", [2, 30])
def test_block_takes_norm_weights_at_any_even_address(T):
    p, g = layer(50, 512, 640, 32, True)
    x = du.bf16(g, (T, 512))
    odd = lambda t: torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")[3: 3 + t.numel()].view_as(t).copy_(t)
    want, _ = du.mlp_block(p["gu"], p["dn"], du.block_norms(p["pre"], p["post"]), x, "silu")
    pre, post = odd(p["pre"]), odd(p["post"])
    out, _ = du.mlp_block(p["gu"], p["dn"], du.block_norms(pre, post), x, "silu")
    assert branch_error(out, want.to(du.F), x) < 2 * L2


@pytest.mark.parametrize("T", [1, 30])
def test_a_stack_of_layers_with_each_tail_doing_the_next_first_norm(T):
    H, I, layers = 512, 768, 3
    stack = [layer(100 + i, H, I, 128, False)[0] for i in range(layers)]
    x = du.bf16(du.gen(9), (T, H), 1.5)
    ref = x.to(du.F)
    for p in stack:
        ref = by_definition(p, ref, "silu", True, None, 1.0, 0.0, 1e-6)
    r, n = x.clone(), torch.empty_like(x)
    du.norm_residual(du.norm_args(None, r, nxt=stack[0]["pre"], next_out=n))
    for i, p in enumerate(stack):
        y, _ = du.mlp(p["gu"], p["dn"], n, "silu")
        nxt = stack[i + 1]["pre"] if i + 1 < layers else None
        du.norm_residual(du.norm_args(y, r, p["post"], None, "none", nxt, r, None if nxt is None else n))
    # three layers of at most six roundings each, every one of them of a part of r
    assert du.rel_l2(r, ref) < 3 * L2


def test_host_ops_agree_with_the_c_abi_and_keep_leading_dimensions():
    p, g = layer(1, 512, 640, 128, True)
    x = du.bf16(g, (2, 9, 512))
    flat, gate = x.view(18, 512), du.bf16(g, (18, 1))
    gu_v, dn_v = w4_views(p["gu"]), w4_views(p["dn"])
    out = xs.linear_w4(view(x), *gu_v)
    assert out.shape() == [2, 9, 1280]
    assert torch.equal(to_torch(out, (18, 1280)).cuda(), du.linear(p["gu"], flat)[0])
    kw = dict(gate_up_zeros=gu_v[2], down_zeros=dn_v[2], activation="gelu")
    out = xs.mlp_w4(view(x), *gu_v[:2], *dn_v[:2], **kw)
    assert out.shape() == [2, 9, 512]
    assert torch.equal(to_torch(out, (18, 512)).cuda(), du.mlp(p["gu"], p["dn"], flat, "gelu")[0])
    tail = dict(eps=1e-5, post_norm_weight=view(p["post"]), gate=view(gate.view(2, 9, 1)), residual_scale=0.5)
    out = xs.mlp_w4_block(view(x), view(p["pre"]), *gu_v[:2], *dn_v[:2], **kw, **tail)
    want, _ = du.mlp_block(p["gu"], p["dn"], du.block_norms(p["pre"], p["post"], gate, "row", 1e-5, 0.5), flat, "gelu")
    assert out.shape() == [2, 9, 512] and torch.equal(to_torch(out, (18, 512)).cuda(), want)
    y = du.bf16(g, (2, 9, 512))
    r, n = xs.norm_residual(view(y), view(x), **tail, next_norm_weight=view(p["pre"]))
    a, b = torch.empty_like(flat), torch.empty_like(flat)
    du.norm_residual(du.norm_args(y.view(18, 512), flat, p["post"], gate, "row", p["pre"], a, b, 1e-5, 0.5))
    assert torch.equal(to_torch(r, (18, 512)).cuda(), a) and torch.equal(to_torch(n, (18, 512)).cuda(), b)
    assert xs.norm_residual(view(y), view(x))[1] is None
    # no tokens
    empty = xs.from_device_ptr(x.data_ptr(), [0, 512], xs.DType.BFloat16)
    assert xs.linear_w4(empty, *gu_v).shape() == [0, 1280]
    assert xs.mlp_w4_block(empty, view(p["pre"]), *gu_v[:2], *dn_v[:2], **kw).shape() == [0, 512]
    assert xs.norm_residual(empty, empty)[0].shape() == [0, 512]


def test_stream_forms_share_one_scratch_that_grows():
    p, g = layer(2, 512, 640, 64, False)
    gu_v, dn_v = w4_views(p["gu"]), w4_views(p["dn"])
    scratch, s = xs.MoEScratch(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    runs = []
    for T in (1, 5, 40, 333, 2):
        x = du.bf16(g, (T, 512))
        s.wait_stream(torch.cuda.current_stream())
        out = torch.empty_like(x)
        with torch.cuda.stream(s):
            xs.mlp_w4_into(view(x), *gu_v[:2], *dn_v[:2], view(out), scratch, s.cuda_stream)
            xs.norm_residual_into(view(out), view(x), view(out), s.cuda_stream, post_norm_weight=view(p["post"]))
        runs.append((x, out))
    xs.moe_check(scratch, s.cuda_stream)
    for x, out in runs:
        y, _ = du.mlp(p["gu"], p["dn"], x, "silu")
        want = torch.empty_like(x)
        du.norm_residual(du.norm_args(y, x, p["post"], None, "none", None, want))
        assert torch.equal(out, want)


@pytest.mark.parametrize("T", [1, 16, 60, 300])
def test_two_captured_graphs_replay_at_once_and_beside_eager_calls(T):
    p, g = layer(3, 1024, 1280, 128, True)
    norms = du.block_norms(p["pre"], p["post"])
    xs_ = [du.bf16(g, (T, 1024)) for _ in range(2)]
    outs = [torch.zeros_like(x) for x in xs_]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, wss = [], []
    for x, out, s in zip(xs_, outs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _, ws = du.mlp_block(p["gu"], p["dn"], norms, x, "silu", out=out)  # a workspace for each graph
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            du.mlp_block(p["gu"], p["dn"], norms, x, "silu", out=out, ws=ws)
        graphs.append(graph)
        wss.append(ws)
    eager_x = du.bf16(g, (T, 1024))
    eager_ws = du.mlp_block(p["gu"], p["dn"], norms, eager_x, "silu")[1]
    for _ in range(4):
        fresh = [du.bf16(g, (T, 1024)) for _ in range(2)]
        want = [du.mlp_block(p["gu"], p["dn"], norms, x, "silu")[0] for x in fresh]
        for x, f in zip(xs_, fresh):
            x.copy_(f)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager, _ = du.mlp_block(p["gu"], p["dn"], norms, eager_x, "silu", ws=eager_ws)
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
        assert torch.equal(eager, du.mlp_block(p["gu"], p["dn"], norms, eager_x, "silu")[0])
    for ws in wss:
        du.flags(ws)


def test_weights_written_just_before_the_call_on_the_same_stream_are_seen():
    """the second half of the MLP loads weights early: never before they are there"""
    p, g = layer(4, 1024, 2048, 128, False)
    q, _ = layer(5, 1024, 2048, 128, False)
    x = du.bf16(g, (1, 1024))
    want = [du.mlp(w["gu"], w["dn"], x, "silu")[0] for w in (p, q)]
    live = {k: {n: t.clone() for n, t in p[k].items() if t is not None} | {"z": None} for k in ("gu", "dn")}
    ws = du.mlp(live["gu"], live["dn"], x, "silu")[1]
    for i in range(20):
        src = (p, q)[i % 2]
        for k in ("gu", "dn"):
            for n in ("q", "s"):
                live[k][n].copy_(src[k][n])
        assert torch.equal(du.mlp(live["gu"], live["dn"], x, "silu", ws=ws)[0], want[i % 2])


@pytest.mark.parametrize("T", [3, 70])
def test_moe_block_with_a_norm_a_gate_and_a_scale_on_its_branch(T):
    dims = dict(T=T, H=512, E=16, K=4, I=256, S=1, fmt="bf16", bias=None)
    d = synth.make_inputs(dims, seed=6, device="cuda")
    g = du.gen(7)
    pre, post, gate = du.bf16(g, (512,), 0.1, 1.0), du.bf16(g, (512,), 0.1, 1.0), du.bf16(g, (512,))
    names = dict(router_weight="router_w", gate_up_weight="gate_up_w", down_weight="down_w", shared_gate_up_weight="shared_gate_up_w",
                 shared_down_weight="shared_down_w")
    kw = {k: view(d[v]) for k, v in names.items()}
    y = gu.forward(dims, dict(d, x=gu.rmsnorm(d["x"], pre, 1e-6)))
    want = torch.empty_like(y)
    du.norm_residual(du.norm_args(y, d["x"], post, gate, "channel", None, want, scale=0.5))
    out = xs.moe_block(view(d["x"]), view(pre), 1e-6, top_k=4, post_norm_weight=view(post), gate=view(gate), residual_scale=0.5, **kw)
    assert torch.equal(to_torch(out, (T, 512)).cuda(), want)
    # without any of them it is the block that was there
    plain = xs.moe_block(view(d["x"]), view(pre), 1e-6, top_k=4, **kw)
    assert torch.equal(to_torch(plain, (T, 512)).cuda(), gu.block_forward(dims, d, pre, 1e-6))
    # the stream form, over its input; weights stored as w - 1
    x2, scratch = d["x"].clone(), xs.MoEScratch()
    st = torch.cuda.current_stream().cuda_stream
    xs.moe_block_into(view(x2), view(pre), view(x2), scratch, st, 1e-6, top_k=4, post_norm_weight=view(post), gate=view(gate), residual_scale=0.5, **kw)
    xs.moe_check(scratch, st)
    assert torch.equal(x2, want)
    one = (pre.float() - 1).to(torch.bfloat16)
    xn = torch.empty_like(d["x"])
    du.norm_residual(du.norm_args(None, d["x"], nxt=one, next_out=xn, offset=1.0))
    y = gu.forward(dims, dict(d, x=xn))
    du.norm_residual(du.norm_args(y, d["x"], None, None, "none", None, want, offset=1.0))
    out = xs.moe_block(view(d["x"]), view(one), 1e-6, top_k=4, weight_offset=1.0, **kw)
    assert torch.equal(to_torch(out, (T, 512)).cuda(), want)


def test_block_refuses_what_it_would_overwrite():
    p, g = layer(8, 256, 128, 64, False)
    x = du.bf16(g, (4, 256))
    L, a, b = capi.lib(), capi.make_w4(p["gu"]), capi.make_w4(p["dn"])
    out, ws = du.mlp_block(p["gu"], p["dn"], du.block_norms(p["pre"], p["post"]), x, "silu")

    def call(norms, x=x, out=out, n=ws.numel()):
        return L.xs_moe_mlp_w4_block(C.byref(a), C.byref(b), 0, C.byref(norms), capi.ptr(x), 4, capi.ptr(out), capi.ptr(ws), n, du.stream_ptr())

    assert call(du.block_norms(p["pre"], p["post"])) == 0
    assert call(du.block_norms(p["pre"], out[0])) == -1 and b"overlaps" in L.xs_moe_last_error()
    assert call(du.block_norms(p["pre"], gate=out, kind="full")) == -1
    assert call(du.block_norms(None)) == -1
    assert call(du.block_norms(p["pre"]), out=ws[256:]) == -1
    assert call(du.block_norms(p["pre"]), n=ws.numel() - 256) == -3
    assert call(du.block_norms(p["pre"].cpu())) == -1 and b"device mismatch" in L.xs_moe_last_error()
    bad = du.block_norms(p["pre"])
    bad.reserved[0] = 1
    assert call(bad) == -1
