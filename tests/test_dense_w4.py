"""4-bit dense operators and the step between two blocks: refusals (no GPU needed) and results against 64-bit definitions.

Tolerances: element by element from the roundings the operators are documented to make (dense_util), and in the norm: the
roundings to bf16 (output, the gated product, the intermediate rows of a block) are off by at most half a step each, 2^-8,
spread evenly, so each adds at most 2^-8 / sqrt(3) of the result in the root mean square, and no chain here has more than six:
sqrt(6 / 3) * 2^-8 < 2^-7."""
import ctypes as C
import threading

import pytest
import torch

from xstar_moe import capi

import dense_util as du
from bridge import torch_to_cpp, xstar_cpp as xs

L2 = 2.0**-7


# ---- refusals ---------------------------------------------------------------------------------------------------------
def _w4(rows=8, cols=256, group=64, codes=4096, scales=4096, zeros=None, reserved=0):
    w = capi.XsMoeW4()
    w.codes_dev, w.scales_dev, w.zeros_dev, w.rows, w.cols, w.group, w.reserved = codes, scales, zeros, rows, cols, group, reserved
    return w


@pytest.mark.parametrize("kw, tokens, code, text", [
    (dict(rows=0), 1, -1, "non-positive"), (dict(cols=-64), 1, -1, "non-positive"), (dict(), -1, -1, "non-positive"),
    (dict(group=16), 1, -2, "group must be"), (dict(group=0), 1, -2, "group must be"), (dict(group=256), 1, -2, "group must be"),
    (dict(cols=288, group=64), 1, -1, "multiple of the group"), (dict(reserved=1), 1, -1, "reserved"),
    (dict(rows=2**30 + 1), 1, -2, "at most 2"), (dict(cols=2**31 - 64), 1, -2, "at most 2"), (dict(), 2**31 - 1, -2, "at most 2"),
])
def test_matrix_shapes_are_checked(kw, tokens, code, text):
    L, n = capi.lib(), C.c_size_t(0)
    assert L.xs_moe_linear_w4_workspace_bytes(C.byref(_w4(**kw)), tokens, C.byref(n)) == code
    assert text in L.xs_moe_last_error().decode()
    assert L.xs_moe_linear_w4(C.byref(_w4(**kw)), None, tokens, None, None, 0, None) == code
    assert L.xs_moe_linear_w4_workspace_bytes(None, 1, C.byref(n)) == -1
    assert L.xs_moe_linear_w4_workspace_bytes(C.byref(_w4()), 1, None) == -1


def test_gated_and_mlp_shapes_are_checked():
    L, n = capi.lib(), C.c_size_t(0)
    assert L.xs_moe_gated_w4(C.byref(_w4(rows=7)), 0, None, 1, None, None, 0, None) == -1
    assert b"must be even" in L.xs_moe_last_error()
    assert L.xs_moe_gated_w4(C.byref(_w4()), 2, None, 1, None, None, 0, None) == -2
    assert b"activation" in L.xs_moe_last_error()
    gu, dn = _w4(rows=128, cols=256), _w4(rows=256, cols=64)
    assert L.xs_moe_mlp_w4_workspace_bytes(C.byref(gu), C.byref(dn), 3, C.byref(n)) == 0 and n.value >= 256 + 3 * 64 * 2
    for bad in (_w4(rows=256, cols=128), _w4(rows=255, cols=64)):
        assert L.xs_moe_mlp_w4_workspace_bytes(C.byref(gu), C.byref(bad), 3, C.byref(n)) == -1
        assert b"down must be" in L.xs_moe_last_error()


def test_workspaces_and_null_pointers_are_refused_before_any_device_work():
    L = capi.lib()
    w = _w4()
    assert L.xs_moe_linear_w4(C.byref(w), None, 0, None, None, 0, None) == 0  # no tokens: nothing to do
    assert L.xs_moe_linear_w4(C.byref(w), 4096, 1, 8192, None, 0, None) == -3
    assert L.xs_moe_linear_w4(C.byref(w), 4096, 1, 8192, 1 << 20, 255, None) == -3
    assert L.xs_moe_linear_w4(C.byref(w), 4096, 1, 8192, (1 << 20) + 16, 4096, None) == -3
    gu, dn = _w4(rows=128, cols=256), _w4(rows=256, cols=64)
    assert L.xs_moe_mlp_w4(C.byref(gu), C.byref(dn), 0, 4096, 3, 8192, 1 << 20, 256, None) == -3


@pytest.mark.parametrize("kw, code, text", [
    (dict(gate_kind=9), -1, "gate kind"), (dict(gate_kind=1), -1, "disagree"), (dict(gate_dev=4096), -1, "disagree"),
    (dict(rows=-1), -1, "non-positive"), (dict(hidden=0), -1, "non-positive"), (dict(hidden=60000), -2, "at most"),
    (dict(rows=2**30 + 1), -2, "at most"),
    (dict(residual_dev=None), -1, "null"), (dict(next_weight_dev=4096), -1, "go together"), (dict(next_out_dev=4096), -1, "go together"),
    (dict(residual_out_dev=None), -1, "go together"), (dict(y_dev=None), -1, "go together"),
])
def test_norm_residual_arguments_are_checked(kw, code, text):
    L, a = capi.lib(), capi.XsMoeNormResidual()
    a.y_dev, a.residual_dev, a.residual_out_dev, a.rows, a.hidden, a.eps = 1 << 20, 2 << 20, 3 << 20, 4, 64, 1e-6
    for k, v in kw.items():
        setattr(a, k, v)
    assert L.xs_moe_norm_residual(C.byref(a), None) == code
    assert text in L.xs_moe_last_error().decode()
    a.reserved[1] = 1
    assert L.xs_moe_norm_residual(C.byref(a), None) == -1
    assert L.xs_moe_norm_residual(None, None) == -1


def _cpu_w4(rows, cols, group, zeros=False, seed=0):
    w = du.weight(du.gen(seed, "cpu"), rows, cols, group, zeros)
    return (torch_to_cpp(w["q"], xs.DType.UInt4x2), torch_to_cpp(w["s"]), torch_to_cpp(w["z"], xs.DType.UInt8) if zeros else None)


def test_host_ops_refuse_with_the_usual_words():
    x = torch_to_cpp(torch.zeros(3, 256).to(torch.bfloat16))
    q, s, z = _cpu_w4(128, 256, 64, True)
    for args, text in [((torch_to_cpp(torch.zeros(3, 256)), q, s), "dtype mismatch"), ((x, s, s), "dtype mismatch"), ((x, q, q), "dtype mismatch"),
                       ((x, q, s, s), "dtype mismatch"), ((x, torch_to_cpp(torch.zeros(2, 64, 128, dtype=torch.uint8), xs.DType.UInt4x2), s), "rank mismatch"),
                       ((torch_to_cpp(torch.zeros(3, 128).to(torch.bfloat16)), q, s), "shape mismatch"), ((x, q, _cpu_w4(64, 256, 64)[1]), "shape mismatch"),
                       ((x, q, s, _cpu_w4(128, 256, 128, True)[2]), "shape mismatch"), ((x, q, s, z), "unsupported device")]:
        with pytest.raises(RuntimeError, match=text):
            xs.linear_w4(*args)
    gq, gs, _ = _cpu_w4(128, 256, 64)
    dq, ds, _ = _cpu_w4(256, 64, 64)
    with pytest.raises(RuntimeError, match="unsupported device"):
        xs.mlp_w4(x, gq, gs, dq, ds)
    with pytest.raises(RuntimeError, match="unknown activation"):
        xs.mlp_w4(x, gq, gs, dq, ds, activation="relu")
    with pytest.raises(RuntimeError, match="shape mismatch"):
        xs.mlp_w4(x, gq, gs, gq, gs)
    with pytest.raises(RuntimeError, match="must be even"):
        xs.mlp_w4(x, *_cpu_w4(127, 256, 64)[:2], dq, ds)
    w = torch_to_cpp(torch.ones(256).to(torch.bfloat16))
    with pytest.raises(RuntimeError, match="unsupported device"):
        xs.mlp_w4_block(x, w, gq, gs, dq, ds)
    with pytest.raises(RuntimeError, match="shape mismatch"):
        xs.mlp_w4_block(x, torch_to_cpp(torch.ones(255).to(torch.bfloat16)), gq, gs, dq, ds)
    out, scratch = torch_to_cpp(torch.zeros(3, 256).to(torch.bfloat16)), xs.MoEScratch()
    bf = lambda *shape: torch_to_cpp(torch.ones(*shape).to(torch.bfloat16))
    with pytest.raises(RuntimeError, match="unsupported device"):
        xs.norm_residual_into(x, x, out, 0)
    with pytest.raises(RuntimeError, match="go together"):
        xs.norm_residual_into(x, x, out, 0, next_norm_weight=w)
    for gate in (bf(2, 1), bf(3, 255), bf(6, 128)):
        with pytest.raises(RuntimeError, match="shape mismatch"):
            xs.norm_residual_into(x, x, out, 0, gate=gate)
    with pytest.raises(RuntimeError, match="dtype mismatch"):
        xs.norm_residual_into(x, x, out, 0, gate=torch_to_cpp(torch.ones(256)))
    with pytest.raises(RuntimeError, match="shape mismatch"):
        xs.norm_residual_into(x, bf(2, 256), out, 0)
    with pytest.raises(RuntimeError, match="unsupported device"):
        xs.linear_w4_into(x, gq, gs, bf(3, 128), scratch, 0)


def test_the_bounds_notice_a_wrong_zero_point_and_a_shifted_scale():
    g = du.gen(5, "cpu")
    w, x = du.weight(g, 24, 512, 32, True), du.bf16(g, (20, 512), device="cpu")
    ref, tol = du.linear_reference(w, x)
    du.assert_close(ref.to(torch.bfloat16), ref, tol)
    wrong = dict(w, z=w["z"].clone())
    wrong["z"][:, 3] ^= 1
    assert du.rel_l2(du.linear_reference(wrong, x)[0], ref) > 4 * L2
    wrong = dict(w, s=w["s"].roll(1, 1))
    assert du.rel_l2(du.linear_reference(wrong, x)[0], ref) > 4 * L2
    with pytest.raises(AssertionError):
        du.assert_close(du.linear_reference(wrong, x)[0], ref, tol)


# ---- linear_w4 --------------------------------------------------------------------------------------------------------
SHAPES = [(1, 32, 32), (5, 64, 64), (16, 128, 128), (33, 160, 32), (127, 384, 128), (130, 1088, 64), (257, 1056, 32), (600, 2048, 128), (264, 2560, 64)]
TOKENS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 129, 200, 257, 600]


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N, K, group", SHAPES)
def test_linear_matches_its_definition(N, K, group, zeros):
    g = du.gen(N * 7 + K)
    w = du.weight(g, N, K, group, zeros)
    for T in TOKENS:
        x = du.bf16(g, (T, K))
        buf = torch.full((T * N + 64,), 77.0, dtype=torch.bfloat16, device="cuda")
        out, ws = du.linear(w, x, out=buf[: T * N].view(T, N))
        du.flags(ws)
        ref, tol = du.linear_reference(w, x)
        du.assert_close(out, ref, tol)
        assert du.rel_l2(out, ref) < L2, T
        assert (buf[T * N:] == 77.0).all(), "wrote behind the last row"


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 16, 40, 300])
@pytest.mark.parametrize("offset", [1, 3])
def test_linear_writes_to_any_even_address_and_reads_any_scale_address(T, offset):
    g = du.gen(T)
    N, K = 136, 512
    w, x = du.weight(g, N, K, 64, True), du.bf16(g, (T, K))
    s = torch.empty(w["s"].numel() + 8, dtype=torch.bfloat16, device="cuda")[offset: offset + w["s"].numel()].view_as(w["s"]).copy_(w["s"])
    z = torch.empty(w["z"].numel() + 8, dtype=torch.uint8, device="cuda")[offset: offset + w["z"].numel()].view_as(w["z"]).copy_(w["z"])
    out = torch.empty(T * N + 8, dtype=torch.bfloat16, device="cuda")[offset: offset + T * N].view(T, N)
    du.linear(dict(q=w["q"], s=s, z=z), x, out=out)
    same, _ = du.linear(w, x)
    assert torch.equal(out, same)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 16, 17, 130])
def test_linear_keeps_every_code_zero_point_and_scale_apart(T):
    """each row of W holds one code, each column group another zero point and scale; x picks single columns"""
    K, N, group = 512, 48, 32
    code = torch.arange(N, device="cuda") % 16
    q = (code | (code << 4)).to(torch.uint8).view(N, 1).expand(N, K // 2).contiguous()
    z = (torch.arange(N * (K // group), device="cuda").view(N, -1) * 7 % 16 + 32).to(torch.uint8)  # the high bits do not count
    s = (2.0 ** (torch.arange(N * (K // group), device="cuda").view(N, -1) % 9 - 4)).to(torch.bfloat16)
    w = dict(q=q, s=s, z=z)
    W = du.matrix(w)
    for k0 in (0, 1, 2, 3, 4, 5, 6, 7, 31, 32, 100, 255, 256, 511):
        x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
        for t in range(T):
            x[t, (k0 + 37 * t) % K] = 2.0
        out, _ = du.linear(w, x)
        assert torch.equal(out.to(du.F), x.to(du.F) @ W.T)  # powers of two times small integers: no rounding anywhere


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 16, 17, 64, 300])
def test_linear_with_infinities_nans_and_zero_scales(T):
    g = du.gen(11)
    K, N = 640, 72
    w, x = du.weight(g, N, K, 128, True), du.bf16(g, (T, K))
    clean, _ = du.linear(w, x)
    w["s"][7] = 0.0
    x2 = x.clone()
    x2[T - 1, 130] = float("nan")
    out, _ = du.linear(w, x2)
    assert out[T - 1].isnan().all()  # NaN * 0 is NaN, so the row of zero scales as well
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[7] = False
    assert torch.equal(out[: T - 1][:, keep], clean[: T - 1][:, keep]) and (out[: T - 1, 7] == 0).all()
    x2 = x.clone()
    x2[0, 5] = float("inf")
    out, _ = du.linear(w, x2)
    want = x2[0].to(du.F) @ du.matrix(w).T
    assert torch.equal(out[0].isnan(), want.isnan()) and torch.equal(out[0].isposinf(), want.isposinf())
    assert torch.equal(out[1:][:, keep], clean[1:][:, keep])
    w["s"][9, 1] = float("inf")
    out, _ = du.linear(w, x)
    assert not out[:, 9].isfinite().any() and torch.equal(out[:, 10:], clean[:, 10:])


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T", [1, 8, 20, 150, 520])
def test_linear_with_scales_and_tokens_of_very_different_size(T, zeros):
    """groups of a row 2^14 apart, rows 2^60 apart, tokens 2^80 apart and their elements 2^20: the powers of two that bring them
    into f16 are each row's and each token's own"""
    g = du.gen(31 + T)
    N, K, group = 200, 1024, 32
    w, x = du.weight(g, N, K, group, zeros), du.bf16(g, (T, K))
    power = torch.randint(-7, 8, w["s"].shape, generator=g, device="cuda") + torch.randint(-30, 31, (N, 1), generator=g, device="cuda")
    w["s"] = (w["s"].float() * 2.0 ** power).to(torch.bfloat16)
    w["s"][3] = 0.0
    w["s"][5, ::2] = 0.0
    x = (x.float() * 2.0 ** torch.randint(-10, 11, (T, K), generator=g, device="cuda") * 2.0 ** torch.randint(-40, 41, (T, 1), generator=g, device="cuda")).to(torch.bfloat16)
    if T > 1:
        x[T // 2] = 0.0
    out, ws = du.linear(w, x)
    du.flags(ws)
    ref, tol = du.linear_reference(w, x)
    du.assert_close(out, ref, tol)
    assert (out[:, 3] == 0).all() and (T == 1 or (out[T // 2] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 100])
def test_linear_with_a_few_more_tiles_than_sms(T):
    g = du.gen(33)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    N, K = sms * 128 + 200, 4096
    w, x = du.weight(g, N, K, 128, True), du.bf16(g, (T, K))
    out, ws = du.linear(w, x)
    du.flags(ws)
    ref, tol = du.linear_reference(w, x)
    du.assert_close(out, ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("T, N", [(20, 50000), (60, 41000), (100, 60001), (700, 9000), (2600, 4000)])
@pytest.mark.parametrize("K", [96, 256, 320, 576, 768, 832, 1152, 1408, 1696])
def test_rows_of_few_blocks_over_many_tiles(T, N, K):
    # an SM goes through several tiles, whose operand blocks are no multiple of the ring's stages
    g = du.gen(K + T)
    w, x = du.weight(g, N, K, 32, K % 3 == 0), du.bf16(g, (T, K))
    out, ws = du.linear(w, x)
    du.flags(ws)
    ref, tol = du.linear_reference(w, x)
    du.assert_close(out, ref, tol)
    for _ in range(10):
        assert torch.equal(du.linear(w, x)[0], out)


@pytest.mark.gpu
@pytest.mark.parametrize("T, H, I, group", [(5121, 576, 2752, 64), (1300, 1152, 4096, 128), (2000, 832, 3000 // 32 * 32, 32)])
def test_mlp_of_short_rows_over_many_tiles(T, H, I, group):
    g = du.gen(T)
    gu, dn, x = du.weight(g, 2 * I, H, group, False, std=H**-0.5), du.weight(g, H, I, group, False, std=I**-0.5), du.bf16(g, (T, H))
    out, ws = du.mlp(gu, dn, x, "gelu")
    du.flags(ws)
    ref, tol = du.mlp_reference(gu, dn, x, "gelu")
    du.assert_close(out, ref, tol)
    for _ in range(10):
        assert torch.equal(du.mlp(gu, dn, x, "gelu")[0], out)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20])
def test_linear_with_offsets_beyond_32_bits(T):
    K, N, group = 65536, 70001, 128  # 2.3 GB of codes
    g = du.gen(3)
    q = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device="cuda")
    s = torch.full((N, K // group), 0.125, dtype=torch.bfloat16, device="cuda")
    rows = [0, 12345, 65535, 65536, N - 2, N - 1]
    part = du.weight(g, len(rows), K, group, False)
    for i, r in enumerate(rows):
        q[r], s[r] = part["q"][i], part["s"][i]
    x = du.bf16(g, (T, K))
    out, ws = du.linear(dict(q=q, s=s, z=None), x)
    du.flags(ws)
    ref, tol = du.linear_reference(part, x)
    du.assert_close(out[:, rows], ref, tol)
    rest = torch.ones(N, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert (out[:, rest] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T, K", [(8, 32768), (8, 33024), (6, 65536 + 128), (1, 300032)])
def test_linear_with_few_tokens_and_long_rows(T, K):
    # tokens that no longer fit into shared memory go the way of larger batches
    g = du.gen(K)
    w, x = du.weight(g, 300, K, 64, True), du.bf16(g, (T, K))
    out, ws = du.linear(w, x)
    du.flags(ws)
    ref, _ = du.linear_reference(w, x)
    many, tol = du.linear_reference(w, torch.cat([x, x.new_zeros(17, K)]))
    assert torch.equal(many[:T], ref)
    du.assert_close(out, ref, tol[:T])


@pytest.mark.gpu
def test_threads_with_calls_of_different_size():
    # the same kernel with little and with much shared memory, from two threads on two streams
    g = du.gen(44)
    cases = [(du.weight(g, 256, K, 64, False), du.bf16(g, (T, K))) for T, K in ((1, 256), (8, 16384), (3, 4096))]
    want = [du.linear(w, x)[0] for w, x in cases]
    torch.cuda.synchronize()
    failed = []

    def work(w, x, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                out, ws = du.linear(w, x)
                for _ in range(300):
                    du.linear(w, x, out, ws)
                torch.cuda.current_stream().synchronize()
                assert torch.equal(out, ref)
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(*c, r)) for c, r in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 16, 90, 520])
def test_linear_gives_the_same_bits_each_time_and_for_each_token(T):
    g = du.gen(21)
    w, x = du.weight(g, 520, 4096, 128, True), du.bf16(g, (T, 4096))
    a, _ = du.linear(w, x)
    for _ in range(5):
        assert torch.equal(du.linear(w, x)[0], a)
    x[T // 2] = 0
    b, _ = du.linear(w, x)
    b[T // 2] = a[T // 2]
    assert torch.equal(a, b), "a token's result depends on its neighbours"


@pytest.mark.gpu
def test_overlaps_host_memory_and_bad_alignment_are_refused():
    L, g = capi.lib(), du.gen(0)
    w, x = du.weight(g, 64, 256, 64, True), du.bf16(g, (4, 256))
    out, ws = du.linear(w, x)
    m = capi.make_w4(w)

    def call(m=m, x=x, out=out, ws=ws, n=None):
        return L.xs_moe_linear_w4(C.byref(m), capi.ptr(x), 4, capi.ptr(out), capi.ptr(ws), ws.numel() if n is None else n, du.stream_ptr())

    def with_(**kw):
        return capi.make_w4(dict(w, **kw))

    assert call() == 0
    assert call(out=x) == -1 and b"overlap" in L.xs_moe_last_error()
    assert call(out=w["s"]) == -1 and b"a weight overlaps" in L.xs_moe_last_error()
    assert call(ws=w["q"].view(-1)) == -1 and b"a weight overlaps" in L.xs_moe_last_error()
    assert call(x=torch.empty(4 * 256 + 8, dtype=torch.bfloat16, device="cuda")[1:]) == -1
    assert call(out=torch.empty(4 * 64 * 2 + 8, dtype=torch.uint8, device="cuda")[1:]) == -1
    for bad in (dict(x=x.cpu()), dict(out=out.cpu()), dict(m=with_(q=w["q"].cpu())), dict(m=with_(s=w["s"].cpu())), dict(m=with_(z=w["z"].cpu()))):
        assert call(**bad) == -1 and b"device mismatch" in L.xs_moe_last_error()
    q = torch.empty(w["q"].numel() + 16, dtype=torch.uint8, device="cuda")[8: 8 + w["q"].numel()].view_as(w["q"])
    assert call(m=with_(q=q)) == -1 and b"aligned" in L.xs_moe_last_error()
    assert call(ws=ws[:128], n=128) == -3


# ---- the gated MLP ----------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("H, I, group, zeros", [(64, 32, 32, True), (128, 320, 64, False), (1056, 96, 32, False), (512, 1024, 128, True), (640, 1408, 128, False)])
def test_mlp_and_its_first_half_match_their_definitions(H, I, group, zeros, act):
    g = du.gen(H + I)
    gu, dn = du.weight(g, 2 * I, H, group, zeros, std=H**-0.5), du.weight(g, H, I, group, zeros, std=I**-0.5)
    for T in (1, 3, 8, 16, 17, 47, 64, 130, 260, 530):
        x = du.bf16(g, (T, H), std=1.5)
        h, ws = du.gated(gu, x, act)
        du.flags(ws)
        ref, tol = du.gated_reference(gu, x, act)
        du.assert_close(h, ref, tol)
        assert du.rel_l2(h, ref) < L2
        buf = torch.full((T * H + 64,), 77.0, dtype=torch.bfloat16, device="cuda")
        out, ws = du.mlp(gu, dn, x, act, out=buf[: T * H].view(T, H))
        du.flags(ws)
        ref, tol = du.mlp_reference(gu, dn, x, act)
        du.assert_close(out, ref, tol)
        # a rounding to bf16 is off by 2^-7 / sqrt(12) of the leading bit's value on average; h handed on in bf16 would double its square
        assert du.rel_l2(out, ref) < 1.05 * 2.0**-7 / 12**0.5
        assert (buf[T * H:] == 77.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40, 300])
def test_mlp_with_tokens_of_very_different_size(T):
    g = du.gen(35)
    H, I = 512, 640
    gu, dn = du.weight(g, 2 * I, H, 64, True, std=H**-0.5), du.weight(g, H, I, 64, False, std=I**-0.5)
    gu["s"][7] *= 64.0  # a row, and its partner, much larger than the others
    gu["s"][I + 7] *= 64.0
    x = (du.bf16(g, (T, H)).float() * 2.0 ** torch.randint(-12, 7, (T, 1), generator=g, device="cuda")).to(torch.bfloat16)
    x[1] = 0.0
    for act in ("silu", "gelu"):
        out, ws = du.mlp(gu, dn, x, act)
        du.flags(ws)
        ref, tol = du.mlp_reference(gu, dn, x, act)
        du.assert_close(out, ref, tol)
        assert (out[1] == 0).all()
        for t in range(0, T, 7):
            if t != 1:
                assert du.rel_l2(out[t], ref[t]) < L2, t


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 40])
def test_mlp_keeps_infinities_and_nans_in_their_rows(T):
    g = du.gen(36)
    H, I = 256, 384
    gu, dn = du.weight(g, 2 * I, H, 128, True, std=H**-0.5), du.weight(g, H, I, 128, True, std=I**-0.5)
    x = du.bf16(g, (T, H))
    clean, _ = du.mlp(gu, dn, x, "silu")
    x[0, 9], x[1, 200] = float("nan"), float("inf")
    out, _ = du.mlp(gu, dn, x, "silu")
    assert out[0].isnan().all() and not out[1].isfinite().any()
    assert torch.equal(out[2:], clean[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T", [2, 40])
def test_activation_far_from_zero(act, T):
    K, I = 64, 32
    w = du.weight(du.gen(1), 2 * I, K, 32, False)
    w["q"].fill_(0x99)  # every weight is the scale
    w["s"].fill_(1.0)
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    values = torch.tensor([-3e38, -1e20, -200.0, -90.0, -20.0, -1.0, 0.0, 1.0, 20.0, 90.0, 1e18], device="cuda")
    for v in values:
        x[:, 3] = v.to(torch.bfloat16)
        h, _ = du.gated(w, x, act)
        gate = x[0, 3].to(du.F)
        want = (du.activation(gate, act) * gate).item()
        assert abs(h.to(du.F) - want).max().item() <= (du.HALF + 2.0**-18) * abs(want) + 1e-30, (v, h[0, 0], want)


# ---- the step between two blocks --------------------------------------------------------------------------------------
def _norm_case(g, T, H, post, kind, nxt, offset):
    y, r = du.bf16(g, (T, H), 0.7), du.bf16(g, (T, H), 2.0)
    weight = lambda: du.bf16(g, (H,), 0.1, 1.0 - offset)
    gate = {"none": None, "channel": (H,), "row": (T, 1), "full": (T, H)}[kind]
    return y, r, weight() if post else None, None if gate is None else du.bf16(g, gate), weight() if nxt else None


# f32: sums of H squares (relative error H * 2^-24 at the worst, half of it after the square root), a handful of products and
# one addition, whose result may be much smaller than its terms
def _norm_tol(ref, magnitude, H):
    return du.HALF * ref.abs() + (H + 32) * 2.0**-24 * magnitude + 1e-37


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("H", [1, 3, 8, 64, 100, 512, 1000, 1032, 2885, 4096, 8192, 11000, 16384, 20000])
def test_norm_residual_matches_its_definition(H, kind):
    g = du.gen(H)
    for T, post, nxt, scale, offset, eps in [(1, True, True, 1.0, 0.0, 1e-6), (2, False, True, 0.22, 1.0, 1e-5), (9, True, False, -1.5, 1.0, 1e-3),
                                             (150, True, True, 0.22, 1.0, 1e-6), (3, False, False, 1.0, 0.0, 1e-6)]:
        y, r, post_w, gate, next_w = _norm_case(g, T, H, post, kind, nxt, offset)
        buf = torch.full((2, T * H + 64), 77.0, dtype=torch.bfloat16, device="cuda")
        out, n = buf[0, : T * H].view(T, H), buf[1, : T * H].view(T, H) if nxt else None
        du.norm_residual(du.norm_args(y, r, post_w, gate, kind, next_w, out, n, eps, scale, offset))
        gate_ref = gate if kind != "row" else gate.expand(T, H)
        ref, nref = du.ref_norm_residual(y, r, post_w, gate_ref, next_w, eps, scale, offset)
        magnitude = r.to(du.F).abs() + (ref - r.to(du.F)).abs()
        du.assert_close(out, ref, _norm_tol(ref, magnitude, H))
        if nxt:
            # an error e of r' moves n by e / rms, and the sum of squares is off by as much as its terms are
            unit = (next_w.to(du.F) + offset).abs() / torch.sqrt((ref * ref).mean(-1, keepdim=True) + eps)
            spread = magnitude * unit + nref.abs() * (magnitude.pow(2).mean(-1, keepdim=True).sqrt() / torch.sqrt((ref * ref).mean(-1, keepdim=True) + eps))
            du.assert_close(n, nref, _norm_tol(nref, spread, H))
        assert (buf[:, T * H:] == 77.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [7, 512, 2885, 4096, 16384])
def test_norm_residual_first_norm_in_place_and_unaligned(H):
    g = du.gen(H + 1)
    T = 33
    y, r, post_w, gate, next_w = _norm_case(g, T, H, True, "full", True, 0.0)
    out, n = torch.empty_like(r), torch.empty_like(r)
    du.norm_residual(du.norm_args(y, r, post_w, gate, "full", next_w, out, n))
    # the first norm of a block alone
    first = torch.empty_like(r)
    du.norm_residual(du.norm_args(None, r, nxt=next_w, next_out=first))
    ref = du.rms(r.to(du.F), next_w, 1e-6, 0.0)
    du.assert_close(first, ref, _norm_tol(ref, ref.abs(), H))
    # over the inputs
    for swap in (False, True):
        y2, r2 = y.clone(), r.clone()
        a, b = (y2, r2) if swap else (r2, y2)
        du.norm_residual(du.norm_args(y2, r2, post_w, gate, "full", next_w, a, b))
        assert torch.equal(a, out) and torch.equal(b, n)
    # from and to addresses that no vector load may use
    odd = lambda t: torch.empty(t.numel() + 8, dtype=t.dtype, device="cuda")[3: 3 + t.numel()].view_as(t).copy_(t)
    out2, n2 = odd(out.zero_().clone()), odd(n)
    du.norm_residual(du.norm_args(odd(y), odd(r), odd(post_w), odd(gate), "full", odd(next_w), out2, n2))
    du.norm_residual(du.norm_args(y, r, post_w, gate, "full", next_w, out, n))
    assert du.rel_l2(out2, out.to(du.F)) < 2.0**-8 and du.rel_l2(n2, n.to(du.F)) < 2.0**-8


@pytest.mark.gpu
def test_norm_residual_zero_rows_nan_rows_and_refused_overlaps():
    g, L = du.gen(2), capi.lib()
    T, H = 6, 512
    y, r, post_w, gate, next_w = _norm_case(g, T, H, True, "row", True, 0.0)
    out, n = torch.empty_like(r), torch.empty_like(r)
    y[1], r[1] = 0, 0
    y[3, 5], r[4, 7] = float("nan"), float("inf")
    du.norm_residual(du.norm_args(y, r, post_w, gate, "row", next_w, out, n))
    assert (out[1] == 0).all() and (n[1] == 0).all()
    assert out[3].isnan().all() and n[3].isnan().all()
    assert out[4, 7].isposinf() and out[4].isinf().sum() == 1
    ref, _ = du.ref_norm_residual(y, r, post_w, gate.expand(T, H), next_w)
    for t in (0, 2, 5):
        assert du.rel_l2(out[t], ref[t]) < 2.0**-8
    a = du.norm_args(y, r, post_w, gate, "row", next_w, out, n)
    for field, value in (("residual_out_dev", n), ("next_out_dev", out), ("next_out_dev", post_w), ("residual_out_dev", next_w), ("next_out_dev", gate)):
        b = capi.XsMoeNormResidual.from_buffer_copy(a)
        setattr(b, field, capi.ptr(value))
        assert L.xs_moe_norm_residual(C.byref(b), du.stream_ptr()) == -1 and b"overlaps" in L.xs_moe_last_error()
    b = capi.XsMoeNormResidual.from_buffer_copy(a)
    b.residual_out_dev = capi.ptr(r.view(-1)[8:])
    assert L.xs_moe_norm_residual(C.byref(b), du.stream_ptr()) == -1
    b = capi.XsMoeNormResidual.from_buffer_copy(a)
    b.gate_dev = C.c_void_p(gate.cpu().data_ptr())
    assert L.xs_moe_norm_residual(C.byref(b), du.stream_ptr()) == -1 and b"device mismatch" in L.xs_moe_last_error()
