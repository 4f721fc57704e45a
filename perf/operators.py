"""Operators for a step of several drafted tokens through a layer whose fp8 weights carry block scales.

A case is a dict of plain values; its "op" names the operator:

  gemm      fp8 x fp8 product with one scale per row and 128 k of the activation, per 128 x 128 block of the weight
  quantize  codes and scales of those operands: 128 x 128 blocks of a weight, 1 x 128 groups of an activation
  norm      the norm after a branch, its gate, the scaled residual add and the norm before the next branch, with
            bf16 output or fp8 codes and 1 x 128 scales
  tree      attention of a tree (or chain) of drafted tokens over a key/value cache that ends with their rows

`run` computes the plain form in 32 bits, or with `own` calls the framework (reng_hip). `exact` is the operator's
definition in 64 bits. Sizes are those of the Llama-3.1-8B, Qwen2.5-7B, Qwen2.5-32B and SmolLM2-135M layers that the
rest of the framework is measured on, and in draw() of the ranges around them. Weights are N(0, 0.02) with a few
outlier columns, as trained projections are; activations N(0, 1) with outlier channels.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 128
MAX_FINITE = {"e4m3": 240.0, "e5m2": 57344.0}
TORCH_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
EPS = 1e-5


def _framework():
    at = os.path.join(os.getcwd(), "reciprocating-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import reng_hip

    return reng_hip


def listed():
    return [
        # One token through Llama-3.1-8B's gate projection: the weight's bytes are the time.
        dict(name="gemm_m1_gate_llama8b", op="gemm", m=1, n=14336, k=4096, afmt="e4m3", bfmt="e4m3"),
        # A tree of 24 drafted tokens through Qwen2.5-7B's down projection.
        dict(name="gemm_m24_down_qwen7b", op="gemm", m=24, n=3584, k=18944, afmt="e4m3", bfmt="e4m3"),
        # A short prompt through SmolLM2-135M's gate projection: k ends inside a block of 128, m inside every tile.
        dict(name="gemm_m333_gate_smol", op="gemm", m=333, n=1536, k=576, afmt="e4m3", bfmt="e4m3"),
        # A prompt of 1024 tokens through Qwen2.5-32B's gate projection.
        dict(name="gemm_m1024_gate_qwen32b", op="gemm", m=1024, n=27648, k=5120, afmt="e4m3", bfmt="e4m3"),
        # Model load: Llama-3.1-8B's gate projection in 128 x 128 blocks.
        dict(name="quantize_gate_llama8b", op="quantize", rows=14336, cols=4096, block_rows=128, dtype="bf16", fmt="e4m3"),
        # The activation of 24 drafted tokens before Qwen2.5-7B's down projection: latency counts.
        dict(name="quantize_24_rows_qwen7b", op="quantize", rows=24, cols=18944, block_rows=1, dtype="bf16", fmt="e4m3"),
        # One token between Llama-3.1-8B's sublayers, both norms, bf16 for a bf16 consumer: latency counts.
        dict(name="norm_1_row_llama8b", op="norm", rows=1, cols=4096, out="bf16", post=True, gate="none", rs=1.0),
        # A prompt of 1024 tokens between Qwen2.5-32B's sublayers, gated per token, straight to the next product's operand.
        dict(name="norm_1024_rows_qwen32b", op="norm", rows=1024, cols=5120, out="e4m3", post=True, gate="rows", rs=0.22),
        # A tree of 16 drafted tokens early in a reply (Llama-3.1-8B heads): latency counts.
        dict(name="tree_16_after_500", op="tree", tokens=16, length=500, heads=32, kv=8, hd=128, mask="tree"),
        # A tree of 63 drafted tokens over a long context.
        dict(name="tree_63_after_32k", op="tree", tokens=63, length=32768, heads=32, kv=8, hd=128, mask="tree"),
        # A wide tree over a context that ends inside a tile (Qwen2.5-7B heads: 28 on 4).
        dict(name="tree_255_after_8191", op="tree", tokens=255, length=8191, heads=28, kv=4, hd=128, mask="tree"),
        # A chain of 1024 tokens, one chunk of a long prompt (Qwen2.5-32B heads).
        dict(name="chain_1024_after_16k", op="tree", tokens=1024, length=16384, heads=40, kv=8, hd=128, mask="chain"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(v, of):
    return max(of, v // of * of)


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "quantize", "norm", "tree", "tree", "tree"])
    fmt = "e4m3" if rng.random() < 0.75 else "e5m2"
    if op == "gemm":
        m = _log(rng, 1, 2048)
        k = _mult(_log(rng, 256, 18944), rng.choice([16, 128, 128, 256]))
        n = _mult(_log(rng, 128, 27648), rng.choice([1, 8, 128]))
        n = max(16, min(n, int(2.8e11 / (2.0 * m * k)), (128 << 20) // k))
        return dict(op=op, m=m, n=n, k=k, afmt=rng.choice(["e4m3", "e4m3", "e5m2"]), bfmt=fmt)
    if op == "quantize":
        block_rows = rng.choice([1, 128])
        cols = _log(rng, 64, 18944)
        cols = cols if rng.random() < 0.3 else _mult(cols, rng.choice([8, 128]))
        rows = min(_log(rng, 1, 16384) if block_rows == 1 else _log(rng, 64, 16384), (48 << 20) // cols)
        return dict(op=op, rows=rows, cols=cols, block_rows=block_rows, dtype=rng.choice(["bf16", "bf16", "f32"]), fmt=fmt)
    if op == "norm":
        cols = _log(rng, 256, 16384)
        cols = cols if rng.random() < 0.3 else _mult(cols, rng.choice([4, 128]))
        return dict(op=op, rows=min(_log(rng, 1, 4096), (5 << 20) // cols), cols=cols, out=rng.choice(["bf16", fmt, fmt]),
                    post=rng.random() < 0.7, gate=rng.choice(["none", "one", "rows"]), rs=rng.choice([1.0, 0.22]))
    hd = rng.choice([64, 128, 128, 256, 96])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 7, 8] if kv < 8 else [1, 2, 4, 5])
    tokens = _log(rng, 1, 1024)
    length = _log(rng, 16, 65536) if rng.random() < 0.9 else 0
    length = min(length, int(6.6e7 / (tokens * max(1, heads * hd // 1024)) / 8))   # scores the plain form holds
    return dict(op=op, tokens=tokens, length=length, heads=heads, kv=kv, hd=hd, mask=rng.choice(["tree", "tree", "chain"]))


# ------------------------------------------------------------------ plain forms

def _blocks(x, br):
    """x [rows, cols] padded with zeros to whole blocks, as [row blocks, br, column blocks, 128]."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % br))
    return x.view(x.shape[0] // br, br, x.shape[1] // BLOCK, BLOCK)


def _plain_quantize(x, br, fmt):
    """x f32 [rows, cols] -> the codes' values as float8 [rows, cols], scales f32 [row blocks, column blocks]."""
    rows, cols = x.shape
    b = _blocks(x, br)
    m = b.abs().amax(dim=(1, 3))
    s = torch.where(m > 0, m / MAX_FINITE[fmt], torch.ones_like(m))
    q = (b / s[:, None, :, None]).clamp(-MAX_FINITE[fmt], MAX_FINITE[fmt])
    q = q.reshape(q.shape[0] * br, -1)[:rows, :cols].contiguous()
    return q.to(TORCH_FP8[fmt]), s


def _expand(v, s, br):
    """Values [rows, cols] times their blocks' scales."""
    rows, cols = v.shape
    return (_blocks(v, br) * s[:, None, :, None]).reshape(-1, s.shape[1] * BLOCK)[:rows, :cols]


def _plain_gemm(st):
    c = st["case"]
    a = _expand(st["a"].view(TORCH_FP8[c["afmt"]]).view(c["m"], c["k"]).float(), st["sa"], 1)
    b = _expand(st["b"].view(TORCH_FP8[c["bfmt"]]).view(c["n"], c["k"]).float(), st["sb"], BLOCK)
    return (a @ b.T).bfloat16()


def _rms(x, gamma):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * gamma


def _plain_norm(st):
    c = st["case"]
    b = st["d"].float()
    if c["post"]:
        b = _rms(b, st["post_gamma"])
    if st["gate"] is not None:
        b = b * st["gate"].float()
    h = st["x"] + c["rs"] * b
    n = _rms(h, st["gamma"])
    if c["out"] == "bf16":
        return h, n.bfloat16()
    return (h, *_plain_quantize(n, 1, c["out"]))


def _visible(st):
    """[tokens, length + tokens] truth values."""
    c = st["case"]
    t = c["tokens"]
    i = torch.arange(t, device="cuda")
    if st["mask"] is None:
        drafted = i[:, None] >= i[None, :]
    else:
        drafted = (st["mask"][:, i // 32] >> (i % 32)) & 1 == 1
    return torch.cat([torch.ones(t, c["length"], dtype=torch.bool, device="cuda"), drafted], dim=1)


def _attend(st, dtype):
    """softmax(scale q k^T) v over the visible rows, heads of one key/value head together."""
    c = st["case"]
    t, h, g, hd = c["tokens"], c["heads"], c["kv"], c["hd"]
    per = h // g
    rows = c["length"] + t
    q = st["q"].view(t, g, per, hd).to(dtype).permute(1, 2, 0, 3).reshape(g, per * t, hd).contiguous()
    k = st["k"][:rows * g * hd].view(rows, g, hd).to(dtype).permute(1, 2, 0).contiguous()
    v = st["v"][:rows * g * hd].view(rows, g, hd).to(dtype).permute(1, 0, 2).contiguous()
    s = torch.bmm(q, k).view(g, per, t, rows) * c["scale"]
    s = s.masked_fill(~_visible(st), -math.inf)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = torch.bmm(p.view(g, per * t, rows), v)
    return o.view(g, per, t, hd).permute(2, 0, 1, 3).reshape(t, h * hd)


# ------------------------------------------------------------------ the cases' data

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _weight(g, rows, cols):
    w = _randn(g, rows, cols) * 0.02
    at = torch.randint(0, cols, (max(1, cols // 256),), generator=g, device="cuda")
    w[:, at] *= 8.0
    return w


def _activation(g, rows, cols):
    x = _randn(g, rows, cols)
    at = torch.randint(0, cols, (max(1, cols // 256),), generator=g, device="cuda")
    x[:, at] *= 16.0
    return x


def _tree(seed, t):
    """Ancestor bits of a random tree, int32 [t, ceil(t / 32)]: parents among the last few tokens, or a new root."""
    rng = np.random.default_rng(seed)
    vis = np.zeros((t, (t + 31) // 32 * 32), dtype=bool)
    for i in range(t):
        back = int(rng.integers(0, min(i, 12) + 1))
        if back:
            vis[i] = vis[i - back]
        vis[i, i] = True
    words = np.packbits(vis, axis=1, bitorder="little").view(np.int32)
    return torch.from_numpy(words.copy()).cuda()


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "gemm":
        a, sa = _plain_quantize(_activation(g, c["m"], c["k"]), 1, c["afmt"])
        b, sb = _plain_quantize(_weight(g, c["n"], c["k"]), BLOCK, c["bfmt"])
        return dict(case=c, a=a.view(torch.uint8), sa=sa, b=b.view(torch.uint8), sb=sb)
    if c["op"] == "quantize":
        w = _weight(g, c["rows"], c["cols"]) if c["block_rows"] == BLOCK else _activation(g, c["rows"], c["cols"])
        return dict(case=c, w=w if c["dtype"] == "f32" else w.bfloat16())
    if c["op"] == "norm":
        rows, cols = c["rows"], c["cols"]
        gate = None if c["gate"] == "none" else (1 + 0.2 * _randn(g, 1 if c["gate"] == "one" else rows, cols)).bfloat16()
        return dict(case=c, x=_activation(g, rows, cols), d=_randn(g, rows, cols).bfloat16(), gate=gate,
                    post_gamma=1 + 0.1 * _randn(g, cols) if c["post"] else None, gamma=1 + 0.1 * _randn(g, cols))
    c["scale"] = 1.0 / math.sqrt(c["hd"])
    rows = c["length"] + c["tokens"]
    cache = lambda: _randn(g, rows * c["kv"] * c["hd"]).bfloat16()  # noqa: E731
    return dict(case=c, q=_randn(g, c["tokens"] * c["heads"] * c["hd"]).bfloat16() * 1.5, k=cache(), v=cache(),
                mask=_tree(seed, c["tokens"]) if c["mask"] == "tree" else None)


def run(state):
    c = state["case"]
    if not own:
        if c["op"] == "gemm":
            return _plain_gemm(state)
        if c["op"] == "quantize":
            return _plain_quantize(state["w"].float(), c["block_rows"], c["fmt"])
        if c["op"] == "norm":
            return _plain_norm(state)
        return _attend(state, torch.float32).bfloat16()
    R = _framework()
    if c["op"] == "gemm":
        return R.gemm_fp8_blocks(state["a"], c["afmt"], state["sa"], state["b"], c["bfmt"], state["sb"], c["m"], c["n"],
                                 c["k"]).view(c["m"], c["n"])
    if c["op"] == "quantize":
        codes, scales = R.quantize_blocks(state["w"], c["rows"], c["cols"], c["fmt"], c["block_rows"])
        return codes.view(TORCH_FP8[c["fmt"]]).view(c["rows"], c["cols"]), scales.view(-1, -(-c["cols"] // BLOCK))
    if c["op"] == "norm":
        args = (state["x"], state["d"], state["gamma"], c["rows"], c["cols"], EPS)
        more = dict(post_gamma=state["post_gamma"], gate=state["gate"], residual_scale=c["rs"])
        if c["out"] == "bf16":
            h, n = R.residual_norm_bf16(*args, **more)
            return h.view(c["rows"], c["cols"]), n.view(c["rows"], c["cols"])
        h, codes, scales = R.residual_norm_fp8(*args, c["out"], **more)
        return (h.view(c["rows"], c["cols"]), codes.view(TORCH_FP8[c["out"]]).view(c["rows"], c["cols"]),
                scales.view(c["rows"], -1))
    return R.attention_tree(state["q"], state["k"], state["v"], c["heads"], c["kv"], c["hd"], c["length"], c["tokens"],
                            c["scale"], mask=state["mask"]).view(c["tokens"], -1)


def work(case):
    c = case
    if c["op"] == "gemm":
        kb = -(-c["k"] // BLOCK)
        scales = 4 * kb * (c["m"] + -(-c["n"] // BLOCK))
        return {"bytes": c["k"] * (c["m"] + c["n"]) + scales + 2 * c["m"] * c["n"], "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        blocks = -(-c["rows"] // c["block_rows"]) * -(-c["cols"] // BLOCK)
        return {"bytes": n * (3 if c["dtype"] == "bf16" else 5) + 4 * blocks, "flops": 2 * n}
    if c["op"] == "norm":
        n = c["rows"] * c["cols"]
        gate = {"none": 0, "one": 2 * c["cols"], "rows": 2 * n}[c["gate"]]
        out = 2 * n if c["out"] == "bf16" else n + 4 * c["rows"] * -(-c["cols"] // BLOCK)
        return {"bytes": n * 10 + gate + out + 4 * c["cols"] * (2 if c["post"] else 1), "flops": 12 * n}
    t, h, rows = c["tokens"], c["heads"], c["length"] + c["tokens"]
    seen = t * c["length"] + (t * (t + 1) // 2 if c["mask"] == "chain" else 8 * t)
    mask = 4 * t * ((t + 31) // 32) if c["mask"] == "tree" else 0
    return {"bytes": 4 * rows * c["kv"] * c["hd"] + 4 * t * h * c["hd"] + mask, "flops": 4 * seen * h * c["hd"]}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_codes(x, br, fmt):
    """Blocks of f64 x: the nearest fp8 value of x / s (ties to even, saturated), and s."""
    mant, emin = (3, -6) if fmt == "e4m3" else (2, -14)
    rows, cols = x.shape
    kb, rb = -(-cols // BLOCK), -(-rows // br)
    full = torch.zeros(rb * br, kb * BLOCK, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    m = full.abs().view(rb, br, kb, BLOCK).permute(0, 2, 1, 3).reshape(rb, kb, -1).max(dim=2).values
    s = m / MAX_FINITE[fmt]
    s[m == 0] = 1.0
    q = x / s.repeat_interleave(br, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    step = torch.exp2((torch.frexp(q).exponent - 1).clamp(min=emin).double() - mant)
    return (torch.round(q / step) * step).clamp(-MAX_FINITE[fmt], MAX_FINITE[fmt]), s


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "gemm":
        sa = st["sa"].double().repeat_interleave(BLOCK, 1)[:, :c["k"]]
        sb = st["sb"].double().repeat_interleave(BLOCK, 0)[:c["n"]].repeat_interleave(BLOCK, 1)[:, :c["k"]]
        a = st["a"].view(TORCH_FP8[c["afmt"]]).double().view(c["m"], c["k"]) * sa
        b = st["b"].view(TORCH_FP8[c["bfmt"]]).double().view(c["n"], c["k"]) * sb
        return torch.matmul(a, b.t())
    if c["op"] == "quantize":
        return _exact_codes(st["w"].double(), c["block_rows"], c["fmt"])
    if c["op"] == "norm":
        b = st["d"].double()
        if c["post"]:
            b = b / torch.sqrt(b.pow(2).sum(1, keepdim=True) / c["cols"] + EPS) * st["post_gamma"].double()
        if st["gate"] is not None:
            b = b * st["gate"].double()
        h = st["x"].double() + c["rs"] * b
        n = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / c["cols"] + EPS) * st["gamma"].double()
        return (h, n) if c["out"] == "bf16" else (h, *_exact_codes(n, 1, c["out"]))
    # One head at a time: its queries, its key/value head's rows, the rows each token sees.
    t, hd, rows = c["tokens"], c["hd"], c["length"] + c["tokens"]
    q = st["q"].view(t, c["heads"], hd)
    k, v = st["k"].view(rows, c["kv"], hd), st["v"].view(rows, c["kv"], hd)
    hidden = torch.zeros(t, rows, dtype=torch.bool, device="cuda")
    if st["mask"] is None:
        hidden[:, c["length"]:] = torch.ones(t, t, dtype=torch.bool, device="cuda").triu(1)
    else:
        bits = np.unpackbits(st["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :t]
        hidden[:, c["length"]:] = torch.from_numpy(bits == 0).cuda()
    out = torch.empty(t, c["heads"], hd, dtype=torch.float64, device="cuda")
    for h in range(c["heads"]):
        g = h * c["kv"] // c["heads"]
        s = torch.matmul(q[:, h].double(), k[:, g].double().t()) * c["scale"]
        out[:, h] = torch.matmul(torch.softmax(s.masked_fill(hidden, -math.inf), 1), v[:, g].double())
    return out.view(t, -1)
