"""What is measured of the 4-bit dense operators and of the norms around a block.

Three operators and their composition:
  linear_w4      out = x W^T with W held as 4-bit codes, bf16 group scales and optional zero points
  mlp_w4         out = (act(x Wg^T) * (x Wu^T)) Wd^T with all three matrices in that form
  norm_residual  r' = r + c * gate * norm(y), and norm(r') for the next block
  mlp_w4_block   x + c * gate * norm(mlp_w4(norm(x))): the three together, as a layer calls them

Weights: q (rows, cols / 2) bytes, the even column in the low nibble; scale (rows, cols / group) bf16;
zero (rows, cols / group) bytes 0..15, 8 where there are none; W = (q - zero) * scale.
"""
import math
import os
import sys

import torch

own = False


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through an attention-sized projection: launch and memory latency count
        dict(name="linear_one_token", op="linear", T=1, K=4096, N=4096, group=128, zeros=False),
        # a few sequences decoding together into a vocabulary-sized projection with an odd number of rows
        dict(name="linear_vocabulary", op="linear", T=7, K=4096, N=32003, group=64, zeros=True),
        # a decode batch that no longer fits one small tile, long inner dimension
        dict(name="linear_batch", op="linear", T=83, K=11264, N=4096, group=32, zeros=True),
        # a prompt
        dict(name="linear_prompt", op="linear", T=4096, K=4096, N=8192, group=128, zeros=False),
        # one token through a feed-forward layer of the benchmark's expert size
        dict(name="mlp_one_token", op="mlp", T=1, H=4096, I=2048, group=128, zeros=False, act="silu"),
        # a decode batch through a wide dense layer
        dict(name="mlp_batch", op="mlp", T=45, H=4096, I=10240, group=32, zeros=True, act="gelu"),
        # a long prompt through a dense layer
        dict(name="mlp_prompt", op="mlp", T=8192, H=4096, I=12288, group=128, zeros=False, act="silu"),
        # tail of one token's block together with the next block's first norm
        dict(name="norm_one_token", op="norm", T=1, H=4096, post=True, gate="none", next=True, scale=1.0, offset=0.0),
        # ragged batch, a width that no vector load divides, per-row gate
        dict(name="norm_odd", op="norm", T=777, H=2885, post=True, gate="row", next=True, scale=0.22, offset=1.0),
        # a prompt, gate for every element
        dict(name="norm_prompt", op="norm", T=8192, H=4096, post=True, gate="full", next=True, scale=1.0, offset=0.0),
        # the feed-forward half of a block, decoding four sequences
        dict(name="block_decode", op="block", T=4, H=4096, I=2048, group=128, zeros=False, act="silu", gate="channel", scale=1.0, offset=0.0),
        # the same for a prompt of odd length
        dict(name="block_prompt", op="block", T=1237, H=4096, I=2048, group=64, zeros=True, act="silu", gate="none", scale=0.5, offset=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "mlp", "mlp", "norm", "block"])
    T = _log(rng, 1, 8192)
    group = rng.choice([32, 64, 128])
    zeros = rng.random() < 0.5
    if op == "linear":
        return dict(op=op, T=T, K=group * max(1, _log(rng, 256, 16384) // group), N=_log(rng, 200, 33000 if T < 2048 else 12000), group=group, zeros=zeros)
    if op == "norm":
        H = _log(rng, 128, 16384)
        if rng.random() < 0.7:
            H = max(8, H // 8 * 8)
        return dict(op=op, T=T, H=H, post=rng.random() < 0.8, gate=rng.choice(["none", "channel", "row", "full"]), next=rng.random() < 0.8,
                    scale=rng.choice([1.0, 0.22, 0.5]), offset=rng.choice([0.0, 1.0]))
    H = group * max(1, _log(rng, 512, 6144) // group)
    I = group * max(1, _log(rng, 512, 12288) // group)
    c = dict(op=op, T=T, H=H, I=I, group=group, zeros=zeros, act=rng.choice(["silu", "gelu"]))
    while T * H * I > 8192 * 4096 * 12288:
        c["T"] = T = T // 2
    if op == "block":
        c.update(gate=rng.choice(["none", "channel", "row", "full"]), scale=rng.choice([1.0, 0.22]), offset=rng.choice([0.0, 1.0]))
    return c


def _w4_bytes(c, rows, cols):
    groups = rows * cols // c["group"]
    return rows * cols // 2 + 2 * groups + (groups if c["zeros"] else 0)


def _gate_count(c):
    return {"none": 0, "channel": c["H"], "row": c["T"], "full": c["T"] * c["H"]}[c["gate"]]


def work(case):
    c = case
    if c["op"] == "linear":
        return dict(bytes=_w4_bytes(c, c["N"], c["K"]) + 2 * c["T"] * (c["K"] + c["N"]), flops=2 * c["T"] * c["N"] * c["K"])
    if c["op"] == "norm":
        n = c["T"] * c["H"]
        weights = c["H"] * (int(c["post"]) + int(c["next"]))
        return dict(bytes=2 * (n * (3 + int(c["next"])) + weights + _gate_count(c)), flops=n * (4 + 4 * int(c["post"]) + 4 * int(c["next"])))
    H, I, T = c["H"], c["I"], c["T"]
    w = dict(bytes=_w4_bytes(c, 2 * I, H) + _w4_bytes(c, H, I) + 4 * T * H, flops=6 * T * H * I)
    if c["op"] == "block":
        w["bytes"] += 2 * (2 * H + _gate_count(c))
        w["flops"] += 12 * T * H
    return w


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _w4(gen, c, rows, cols):
    """Weights N(0, 0.02) brought to 4 bits a group at a time, the way a checkpoint of this form is made."""
    g = c["group"]
    q = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    s = torch.empty(rows, cols // g, dtype=torch.bfloat16, device="cuda")
    z = torch.empty(rows, cols // g, dtype=torch.uint8, device="cuda") if c["zeros"] else None
    step = max(1, (1 << 26) // cols)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        w = (torch.randn(b - a, cols // g, g, generator=gen, device="cuda") * 0.02)
        if c["zeros"]:
            lo, hi = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
            sc = ((hi - lo) / 15).to(torch.bfloat16)
            zp = torch.round(-lo / sc.float()).clamp(0, 15)
            z[a:b] = zp.to(torch.uint8)
        else:
            sc = (w.abs().amax(-1) / 7).to(torch.bfloat16)
            zp = torch.full_like(sc, 8, dtype=torch.float32)
        s[a:b] = sc
        codes = (torch.round(w / sc.float().unsqueeze(-1)) + zp.unsqueeze(-1)).clamp(0, 15).to(torch.uint8).view(b - a, cols)
        q[a:b] = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return dict(q=q, s=s, z=z)


def _bf16(gen, shape, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(torch.bfloat16)


def _norm_inputs(gen, c, d):
    H, T = c["H"], c["T"]
    centre = 1.0 - c["offset"]
    d["post_w"] = _bf16(gen, (H,), 0.1, centre) if c.get("post", True) else None
    d["next_w"] = _bf16(gen, (H,), 0.1, centre) if c.get("next", True) else None
    shape = {"none": None, "channel": (H,), "row": (T, 1), "full": (T, H)}[c["gate"]]
    d["gate"] = None if shape is None else torch.sigmoid(torch.randn(shape, generator=gen, device="cuda")).to(torch.bfloat16)


def _inputs(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    d = {}
    if c["op"] == "linear":
        d["x"] = _bf16(gen, (c["T"], c["K"]))
        d["w"] = _w4(gen, c, c["N"], c["K"])
    elif c["op"] == "norm":
        d["y"] = _bf16(gen, (c["T"], c["H"]), 0.7)
        d["r"] = _bf16(gen, (c["T"], c["H"]), 2.0)
        _norm_inputs(gen, c, d)
    else:
        d["x"] = _bf16(gen, (c["T"], c["H"]))
        d["gu"] = _w4(gen, c, 2 * c["I"], c["H"])
        d["dn"] = _w4(gen, c, c["H"], c["I"])
        if c["op"] == "block":
            _norm_inputs(gen, c, d)
            d["pre_w"] = d.pop("next_w")
    return d


EPS = 1e-6


def prepare(case, seed):
    st = dict(case=dict(case), data=_inputs(case, seed))
    if own:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        path = os.path.join(root, "xstar-infer_b200", "xstar_cpp_py")
        if path not in sys.path:
            sys.path.insert(0, path)
        import xstar_cpp as xs

        kinds = {torch.bfloat16: xs.DType.BFloat16}

        def view(t, kind=None):
            return None if t is None else xs.from_device_ptr(t.data_ptr(), list(t.shape), kinds[t.dtype] if kind is None else kind)

        v = {}
        for k, t in st["data"].items():
            if isinstance(t, dict):
                v[k] = (view(t["q"], xs.DType.UInt4x2), view(t["s"]), view(t["z"], xs.DType.UInt8))
            else:
                v[k] = view(t)
        d = st["data"]
        if case["op"] == "linear":
            out = torch.empty(case["T"], case["N"], dtype=torch.bfloat16, device="cuda")
        else:
            out = torch.empty(case["T"], case["H"], dtype=torch.bfloat16, device="cuda")
        st["out"] = out
        st["next_out"] = torch.empty_like(out) if case["op"] == "norm" and d["next_w"] is not None else None
        st["xs"], st["view"], st["scratch"] = xs, v, xs.MoEScratch()
        st["out_view"], st["next_view"] = view(out), view(st["next_out"])
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------
def _dequant(w, group):
    q = w["q"]
    codes = torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1, group).float()
    zero = 8.0 if w["z"] is None else w["z"].float().unsqueeze(-1)
    return ((codes - zero) * w["s"].float().unsqueeze(-1)).view(q.shape[0], -1)


def _act(v, name):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))


def _norm(v, w, offset):
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * (w.float() + offset)


def _mlp(x, gu, dn, c):
    gate, up = (x @ _dequant(gu, c["group"]).t()).chunk(2, -1)
    return (_act(gate, c["act"]) * up) @ _dequant(dn, c["group"]).t()


def _plain(c, d):
    if c["op"] == "linear":
        return (d["x"].float() @ _dequant(d["w"], c["group"]).t()).to(torch.bfloat16)
    if c["op"] == "mlp":
        return _mlp(d["x"].float(), d["gu"], d["dn"], c).to(torch.bfloat16)
    if c["op"] == "block":
        r = d["x"].float()
        y = _mlp(_norm(r, d["pre_w"], c["offset"]), d["gu"], d["dn"], c)
    else:
        r, y = d["r"].float(), d["y"].float()
    if d["post_w"] is not None:
        y = _norm(y, d["post_w"], c["offset"])
    if d["gate"] is not None:
        y = y * d["gate"].float()
    r = r + c["scale"] * y
    out = [r.to(torch.bfloat16)]
    if d.get("next_w") is not None:
        out.append(_norm(r, d["next_w"], c["offset"]).to(torch.bfloat16))
    return out


def _own(st):
    c, xs, v = st["case"], st["xs"], st["view"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "linear":
        q, s, z = v["w"]
        xs.linear_w4_into(v["x"], q, s, st["out_view"], st["scratch"], stream, zeros=z)
        return st["out"]
    if c["op"] == "norm":
        xs.norm_residual_into(v["y"], v["r"], st["out_view"], stream, eps=EPS, post_norm_weight=v["post_w"], gate=v["gate"],
                              residual_scale=c["scale"], weight_offset=c["offset"], next_norm_weight=v["next_w"], next_out=st["next_view"])
        return [st["out"]] + ([] if st["next_out"] is None else [st["next_out"]])
    (gq, gs, gz), (dq, ds, dz) = v["gu"], v["dn"]
    if c["op"] == "mlp":
        xs.mlp_w4_into(v["x"], gq, gs, dq, ds, st["out_view"], st["scratch"], stream, gate_up_zeros=gz, down_zeros=dz, activation=c["act"])
        return st["out"]
    xs.mlp_w4_block_into(v["x"], v["pre_w"], gq, gs, dq, ds, st["out_view"], st["scratch"], stream, eps=EPS, gate_up_zeros=gz, down_zeros=dz,
                         activation=c["act"], post_norm_weight=v["post_w"], gate=v["gate"], residual_scale=c["scale"], weight_offset=c["offset"])
    return [st["out"]]


def run(state):
    return _own(state) if own else _plain(state["case"], state["data"])


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    c, d = case, _inputs(case, seed)
    f = torch.float64

    def matrix(w):
        low, high = torch.bitwise_and(w["q"], 0x0F), torch.bitwise_right_shift(w["q"], 4)
        m = torch.empty(w["q"].shape[0], 2 * w["q"].shape[1], dtype=f, device="cuda")
        m[:, 0::2], m[:, 1::2] = low.to(f), high.to(f)
        m -= 8 if w["z"] is None else w["z"].to(f).repeat_interleave(c["group"], 1)
        return m.mul_(w["s"].to(f).repeat_interleave(c["group"], 1))

    def rms(v, w):
        scale = 1 / torch.sqrt(v.square().sum(-1, keepdim=True) / v.shape[-1] + EPS)
        return scale * v * (c["offset"] + w.to(f))

    def feed_forward(x):
        w, I = matrix(d["gu"]), c["I"]
        g, u = x @ w[:I].T, x @ w[I:].T
        del w
        if c["act"] == "silu":
            h = g * torch.sigmoid(g) * u
        else:
            h = g * u / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * g * (1 + 0.044715 * g.square())))
        del g, u
        return h @ matrix(d["dn"]).T

    if c["op"] == "linear":
        return d["x"].to(f) @ matrix(d["w"]).T
    if c["op"] == "mlp":
        return feed_forward(d["x"].to(f))
    if c["op"] == "block":
        base = d["x"].to(f)
        branch = feed_forward(rms(base, d["pre_w"]))
    else:
        base, branch = d["r"].to(f), d["y"].to(f)
    if d["post_w"] is not None:
        branch = rms(branch, d["post_w"])
    if d["gate"] is not None:
        branch = branch * d["gate"].to(f)
    base = base + c["scale"] * branch
    return [base] if d.get("next_w") is None else [base, rms(base, d["next_w"])]
