"""Operators for a layer whose weights and key/value cache are held in 4 bits (e2m1 codes, one power-of-two scale per 32).

A case is a dict of plain values; its "op" names the operator:

  quantize   codes and scales of a matrix, and the values they stand for
  gemm       the product of two such matrices
  heads      norms of queries and keys per head and the rotation of their positions (one axis or several) in one pass;
             keys and values as bf16 rows, or quantized into the 4-bit cache and read back
  cache      a cache quantized as it is written: rows appended to it, and all of it read back
  attention  attention of a chain or tree of tokens over that cache

`run` computes the plain form in 32 bits, or with `own` calls the framework (reng_hip). `exact` is the operator's
definition in 64 bits. Sizes are those of the Llama-3.1-8B, Qwen2.5-7B, Qwen2.5-32B and SmolLM2-135M layers that the
rest of the framework is measured on, and in draw() of the ranges around them. Weights are N(0, 0.02) with a few
outlier columns, as trained projections are; activations N(0, 1) with outlier channels.

Layouts: codes [rows, cols / 2], the even column in the low half of a byte; scales [rows, 4 ceil(cols / 128)], byte b of
a row for its columns 32 b .. 32 b + 31, 2^(byte - 127). A cache has [kv heads, capacity] rows of head_dim columns.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
EPS = 1e-6


def _framework():
    at = os.path.join(os.getcwd(), "reciprocating-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import reng_hip

    return reng_hip


def listed():
    return [
        # Model load: Llama-3.1-8B's gate projection to 4 bits, and its values for the error report.
        dict(name="quantize_gate_llama8b", op="quantize", rows=14336, cols=4096, dtype="bf16"),
        # The activation of 24 drafted tokens before Qwen2.5-7B's down projection: latency counts.
        dict(name="quantize_24_rows_qwen7b", op="quantize", rows=24, cols=18944, dtype="bf16"),
        # One token through Llama-3.1-8B's gate projection: the weight's bytes are the time.
        dict(name="gemm_m1_gate_llama8b", op="gemm", m=1, n=14336, k=4096),
        # A tree of 24 drafted tokens through Qwen2.5-7B's down projection.
        dict(name="gemm_m24_down_qwen7b", op="gemm", m=24, n=3584, k=18944),
        # A prompt of 1024 tokens through Qwen2.5-32B's gate projection.
        dict(name="gemm_m1024_gate_qwen32b", op="gemm", m=1024, n=27648, k=5120),
        # One token's heads into the 4-bit cache (Llama-3.1-8B heads), norms and rotation on the way: latency counts.
        dict(name="heads_1_token", op="heads", tokens=1, heads=32, kv=8, hd=128, rot=128, axes=1, norm=True, into="mxfp4"),
        # A prompt of 1024 tokens of text and images (time, height and width) into a bf16 cache (Qwen2.5-32B heads).
        dict(name="heads_1024_tokens_3_axes", op="heads", tokens=1024, heads=40, kv=8, hd=128, rot=128, axes=3, norm=True,
             into="bf16"),
        # One token appended to a short SmolLM2-135M cache, which is then read back: latency counts.
        dict(name="cache_1_after_499_smol", op="cache", tokens=1, length=499, kv=3, hd=64),
        # A chunk of 1024 tokens appended to a long cache, which a consumer of bf16 then reads.
        dict(name="cache_1024_after_31k", op="cache", tokens=1024, length=31744, kv=8, hd=128),
        # One token over a long context: the cache's bytes are the time.
        dict(name="attention_1_after_32k", op="attention", tokens=1, length=32768, heads=32, kv=8, hd=128, mask="chain"),
        # A tree of 63 drafted tokens over a context that ends inside a tile (Qwen2.5-7B heads: 28 on 4).
        dict(name="attention_tree_63_after_8191", op="attention", tokens=63, length=8191, heads=28, kv=4, hd=128, mask="tree"),
        # A chain of 1024 tokens, one chunk of a long prompt (Qwen2.5-32B heads).
        dict(name="attention_chain_1024_after_16k", op="attention", tokens=1024, length=16384, heads=40, kv=8, hd=128,
             mask="chain"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(v, of):
    return max(of, v // of * of)


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "heads", "cache", "attention", "attention", "attention"])
    if op == "quantize":
        cols = _log(rng, 32, 18944)
        cols = cols if rng.random() < 0.3 else _mult(cols, rng.choice([8, 32, 128]))
        return dict(op=op, rows=min(_log(rng, 1, 16384), (48 << 20) // cols), cols=cols, dtype=rng.choice(["bf16", "bf16", "f32"]))
    if op == "gemm":
        m = _log(rng, 1, 2048)
        k = _mult(_log(rng, 256, 18944), rng.choice([32, 128, 256]))
        n = _mult(_log(rng, 128, 27648), rng.choice([1, 8, 128]))
        return dict(op=op, m=m, n=max(16, min(n, int(2.8e11 / (2.0 * m * k)), (128 << 20) // k)), k=k)
    hd = rng.choice([32, 64, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 7, 8] if kv < 8 else [1, 2, 4, 5])
    if op == "heads":
        into = rng.choice(["bf16", "mxfp4"])
        rot = rng.choice([hd, hd, hd // 2])
        return dict(op=op, tokens=_log(rng, 1, 2048 if into == "bf16" else 48), heads=heads, kv=kv, hd=hd, rot=rot,
                    axes=rng.choice([1, 1, 2, 3]), norm=rng.random() < 0.7, into=into)
    if op == "cache":
        return dict(op=op, tokens=_log(rng, 1, 1024), length=_log(rng, 16, 32768), kv=kv, hd=hd)
    tokens = _log(rng, 1, 1024)
    length = _log(rng, 16, 65536) if rng.random() < 0.9 else 0
    length = min(length, int(6.6e7 / (tokens * max(1, heads * hd // 1024)) / 8))   # scores the plain form holds
    return dict(op=op, tokens=tokens, length=length, heads=heads, kv=kv, hd=hd, mask=rng.choice(["tree", "chain", "chain"]))


# ------------------------------------------------------------------ plain forms

def _pitch(cols):
    return 4 * -(-cols // 128)


def _pow2(e):
    """2^e of whole numbers, in f32 (ldexp's own powers are off by a bit on the GPU, exp2 in f64 is exact)."""
    return torch.exp2(e.double()).float()


def _plain_quantize(x):
    """x f32 [rows, cols] -> signed levels (indices 0 .. 15) [rows, cols], exponents [rows, ceil(cols / 32)]."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    f, e = torch.frexp(b.abs().amax(dim=2))
    # The largest magnitude is f 2^e, f in [0.5, 1): below 7 of the scale.
    e = torch.where(f > 0, e + (f >= 0.875).int() - 3, torch.zeros_like(e)).clamp(min=-127)
    q = b * _pow2(-e)[:, :, None]
    a = q.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte())
    code = code + 8 * torch.signbit(q).byte()
    return code.view(rows, -1)[:, :cols], e


def _values(code, e):
    """f32 values of levels [rows, cols] and exponents [rows, blocks]."""
    rows, cols = code.shape
    mag = (code & 7).int()   # 0, 0.5, then 1 or 1.5 times a power of two
    v = torch.where(mag < 2, 0.5 * mag, (1 + 0.5 * (mag & 1)) * _pow2((mag >> 1) - 1))
    v = torch.where(code >= 8, -v, v)
    v = torch.nn.functional.pad(v, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    return (v * _pow2(e)[:, :, None]).view(rows, -1)[:, :cols]


def _unpack(codes, scales, cols):
    """The same values from codes [rows, cols / 2] and scales [rows, 4 ceil(cols / 128)]."""
    code = torch.stack([codes & 15, codes >> 4], dim=2).view(codes.shape[0], -1)
    return _values(code, scales[:, :-(-cols // BLOCK)].int() - 127)


def _plain_heads(x, gamma, st):
    """x f32 [tokens, heads, hd]: the norm of each head, the rotation of its first `rot` values."""
    c = st["case"]
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * gamma
    half = c["rot"] // 2
    at = st["positions"].long()[st["pair_axis"], :].T                   # [tokens, half]: the row of each pair
    pair = torch.arange(half, device="cuda")
    sin, cos = st["sin"], st["cos"]
    lo, hi, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c0, s0, c1, s1 = (t[at, pair + o][:, None] for o in (0, half) for t in (cos, sin))
    return torch.cat([lo * c0 - hi * s0, hi * c1 + lo * s1, rest], dim=-1)


def _split_heads(st):
    """Queries, keys and values of a product's output row [q | k | v], as f32 [tokens, heads, hd]."""
    c = st["case"]
    nq, nk = c["heads"] * c["hd"], c["kv"] * c["hd"]
    t = st["qkv"].float()
    return [t[:, a:b].reshape(c["tokens"], -1, c["hd"]) for a, b in ((0, nq), (nq, nq + nk), (nq + nk, nq + 2 * nk))]


def _plain_read(st, rows):
    """The cache's first rows as f32 [rows, kv, hd], keys and values."""
    c = st["case"]
    take = lambda t: t[:, :rows].reshape(c["kv"] * rows, -1)  # noqa: E731
    return [_unpack(take(st[n + "_codes"]), take(st[n + "_scales"]), c["hd"]).view(c["kv"], rows, c["hd"]).transpose(0, 1)
            for n in ("k", "v")]


def _visible(st):
    """[tokens, length + tokens] truth values."""
    c = st["case"]
    t = c["tokens"]
    i = torch.arange(t, device="cuda")
    if st["mask"] is None:
        own_rows = i[:, None] >= i[None, :]
    else:
        own_rows = (st["mask"][:, i // 32] >> (i % 32)) & 1 == 1
    return torch.cat([torch.ones(t, c["length"], dtype=torch.bool, device="cuda"), own_rows], dim=1)


def _plain_attention(st):
    """softmax(scale q k^T) v over the visible rows, heads of one key/value head together."""
    c = st["case"]
    t, h, g, hd = c["tokens"], c["heads"], c["kv"], c["hd"]
    per, rows = h // g, c["length"] + t
    k, v = _plain_read(st, rows)
    q = st["q"].view(t, g, per, hd).float().permute(1, 2, 0, 3).reshape(g, per * t, hd).contiguous()
    s = torch.bmm(q, k.permute(1, 2, 0).contiguous()).view(g, per, t, rows) * c["scale"]
    s = s.masked_fill(~_visible(st), -math.inf)
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = torch.bmm(p.view(g, per * t, rows), v.transpose(0, 1).contiguous())
    return o.view(g, per, t, hd).permute(2, 0, 1, 3).reshape(t, h * hd).bfloat16()


# ------------------------------------------------------------------ the cases' data

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _outliers(g, x, by):
    """A few columns larger than the others."""
    at = torch.randint(0, x.shape[1], (max(1, x.shape[1] // 256),), generator=g, device="cuda")
    x[:, at] *= by
    return x


def _weight(g, rows, cols):
    return _outliers(g, _randn(g, rows, cols) * 0.02, 8.0)


def _activation(g, rows, cols):
    return _outliers(g, _randn(g, rows, cols), 16.0)


def _packed(x):
    """f32 x [rows, cols], cols even: its codes and scales."""
    code, e = _plain_quantize(x)
    scales = torch.full((x.shape[0], _pitch(x.shape[1])), 127, dtype=torch.uint8, device="cuda")
    scales[:, :e.shape[1]] = (e + 127).byte()
    return (code[:, ::2] | code[:, 1::2] << 4).contiguous(), scales


def _cache(g, c, rows, capacity):
    """A cache of `capacity` rows, the first `rows` written; the others hold what was there."""
    st = {}
    for n in ("k", "v"):
        for name, pitch in (("codes", c["hd"] // 2), ("scales", _pitch(c["hd"]))):
            st["%s_%s" % (n, name)] = torch.full((c["kv"], capacity, pitch), 0x77, dtype=torch.uint8, device="cuda")
        if rows:
            codes, scales = _packed(_randn(g, c["kv"] * rows, c["hd"]).bfloat16().float())
            st[n + "_codes"][:, :rows] = codes.view(c["kv"], rows, -1)
            st[n + "_scales"][:, :rows] = scales.view(c["kv"], rows, -1)
    return st


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


def _sections(half, axes):
    """Rotated pairs of each axis: a quarter for the first of three, as time has beside height and width."""
    if axes == 3:
        first = half // 4
        return (first, (half - first) // 2, half - first - (half - first) // 2)
    return tuple(half // axes + (1 if a < half % axes else 0) for a in range(axes))


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "quantize":
        w = (_weight if c["rows"] > 64 else _activation)(g, c["rows"], c["cols"])
        return dict(case=c, w=w if c["dtype"] == "f32" else w.bfloat16())
    if c["op"] == "gemm":
        a, sa = _packed(_activation(g, c["m"], c["k"]))
        b, sb = _packed(_weight(g, c["n"], c["k"]))
        return dict(case=c, a=a, sa=sa, b=b, sb=sb)
    t, hd = c["tokens"], c["hd"]
    if c["op"] == "heads":
        half = c["rot"] // 2
        sections = _sections(half, c["axes"])
        # Positions of a prompt's tokens: the time axis counts on, the others go over an image's rows and columns.
        far = 4 * t + 256
        first = int(np.random.default_rng(seed).integers(0, 256))
        i = torch.arange(t, device="cuda")
        positions = torch.stack([first + i, first + i // 16 % 64, first + i % 16][:c["axes"]]).int()
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = (torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * freq).repeat(1, 2)
        width = (c["heads"] + 2 * c["kv"]) * hd
        st = dict(case=c, qkv=_activation(g, t, width).bfloat16(), sections=sections, positions=positions.contiguous(),
                  pair_axis=torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(sections)).cuda(),
                  sin=angle.sin().float().contiguous(), cos=angle.cos().float().contiguous(),
                  q_gamma=1 + 0.1 * _randn(g, hd) if c["norm"] else None, k_gamma=1 + 0.1 * _randn(g, hd) if c["norm"] else None)
        return {**st, **_cache(g, c, 0, t)} if c["into"] == "mxfp4" else st
    if c["op"] == "cache":
        return dict(case=c, kv_rows=_randn(g, t, 2 * c["kv"] * hd).bfloat16(), **_cache(g, c, c["length"], c["length"] + t + 13))
    c["scale"] = 1.0 / math.sqrt(hd)
    rows = c["length"] + t
    return dict(case=c, q=_randn(g, t * c["heads"] * hd).bfloat16() * 1.5, mask=_tree(seed, t) if c["mask"] == "tree" else None,
                **_cache(g, c, rows, rows + 13))


def _own_cache(R, st):
    """The program's handle of its cache."""
    if "handle" not in st:
        st["handle"] = R.MxCache(st["case"]["kv"], st["case"]["hd"], st["k_codes"].shape[1],
                                 tensors=(st["k_codes"], st["k_scales"], st["v_codes"], st["v_scales"]))
    return st["handle"]


def _own_rope(R, st):
    """The program's handle of its rotation tables."""
    if "rope" not in st:
        st["rope"] = R.Rope(st["sin"], st["cos"], sections=st["sections"])
    return st["rope"]


def run(state):
    c = state["case"]
    if own:
        return _run_own(state)
    if c["op"] == "quantize":
        return _values(*_plain_quantize(state["w"].float())).bfloat16()
    if c["op"] == "gemm":
        return (_unpack(state["a"], state["sa"], c["k"]) @ _unpack(state["b"], state["sb"], c["k"]).T).bfloat16()
    if c["op"] == "heads":
        q, k, v = _split_heads(state)
        q, k = _plain_heads(q, state["q_gamma"], state), _plain_heads(k, state["k_gamma"], state)
        if c["into"] == "mxfp4":
            k, v = (_values(*_plain_quantize(t.reshape(-1, c["hd"]))) for t in (k, v))
        return [t.reshape(c["tokens"], -1).bfloat16() for t in (q, k, v)]
    if c["op"] == "cache":
        old = [t[:c["length"]] for t in _plain_read(state, c["length"])]
        new = [t.reshape(-1, c["hd"]) for t in state["kv_rows"].float().chunk(2, dim=1)]
        new = [_values(*_plain_quantize(t)).view(c["tokens"], c["kv"], c["hd"]) for t in new]
        return [torch.cat(t).reshape(c["length"] + c["tokens"], -1).bfloat16() for t in zip(old, new)]
    return _plain_attention(state)


def _run_own(state):
    R, c = _framework(), state["case"]
    if c["op"] == "quantize":
        codes, scales = R.quantize_mxfp4(state["w"], c["rows"], c["cols"])
        return R.dequantize_mxfp4(codes, scales, c["rows"], c["cols"]).view(c["rows"], c["cols"])
    if c["op"] == "gemm":
        return R.gemm_mxfp4(state["a"], state["sa"], state["b"], state["sb"], c["m"], c["n"], c["k"]).view(c["m"], c["n"])
    if c["op"] == "heads":
        nq, nk = c["heads"] * c["hd"], c["kv"] * c["hd"]
        q, k, v = (state["qkv"][:, a:b] for a, b in ((0, nq), (nq, nq + nk), (nq + nk, nq + 2 * nk)))
        args = dict(rope=_own_rope(R, state), positions=state["positions"], q_gamma=state["q_gamma"], k_gamma=state["k_gamma"],
                    eps=EPS)
        if c["into"] == "bf16":
            q, k, v = R.head_norm_rope_bf16(q, k, v, c["tokens"], c["heads"], c["kv"], c["hd"], **args)
        else:
            cache = _own_cache(R, state)
            q = R.head_norm_rope_mxfp4(q, k, v, c["tokens"], c["heads"], cache, 0, **args)
            k, v = cache.read(0, c["tokens"])
        return [t.view(c["tokens"], -1) for t in (q, k, v)]
    cache = _own_cache(R, state)
    if c["op"] == "cache":
        nk = c["kv"] * c["hd"]
        cache.write(state["kv_rows"][:, :nk], state["kv_rows"][:, nk:], c["length"], c["tokens"])
        return [t.view(c["length"] + c["tokens"], -1) for t in cache.read(0, c["length"] + c["tokens"])]
    return R.attention_mxfp4(state["q"], cache, c["heads"], c["length"], c["tokens"], c["scale"],
                             mask=state["mask"]).view(c["tokens"], -1)


def work(case):
    c = case
    held = lambda rows, cols: rows * (cols / 2 + cols / BLOCK)  # noqa: E731
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (4 if c["dtype"] == "bf16" else 6) + held(c["rows"], c["cols"]), "flops": 2 * n}
    if c["op"] == "gemm":
        return {"bytes": held(c["m"] + c["n"], c["k"]) + 2 * c["m"] * c["n"], "flops": 2 * c["m"] * c["n"] * c["k"]}
    t, kv, hd = c["tokens"], c["kv"], c["hd"]
    if c["op"] == "heads":
        n = t * (c["heads"] + 2 * kv) * hd
        cache = held(2 * t * kv, hd) if c["into"] == "mxfp4" else 0
        return {"bytes": 4 * n + cache + 8 * t * c["rot"] * (2 if c["axes"] > 1 else 1), "flops": 8 * n}
    if c["op"] == "cache":
        rows = c["length"] + t
        return {"bytes": 2 * held(rows * kv, hd) + 4 * rows * kv * hd + 4 * t * kv * hd, "flops": 2 * rows * kv * hd}
    rows = c["length"] + t
    seen = t * c["length"] + (t * (t + 1) // 2 if c["mask"] == "chain" else 8 * t)
    mask = 4 * t * ((t + 31) // 32) if c["mask"] == "tree" else 0
    return {"bytes": 2 * held(rows * kv, hd) + 4 * t * c["heads"] * hd + mask, "flops": 4 * seen * c["heads"] * hd}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_values(x):
    """f64 x [rows, cols]: each value as the nearest of the 15 levels times its block's scale, ties to the even level."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    full = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :cols] = x
    m = full.abs().view(rows, blocks, BLOCK).max(dim=2).values
    s = torch.ones_like(m)
    at = m > 0
    # The smallest power of two under which the largest magnitude is less than 7.
    e = torch.floor(torch.log2(m[at] / 7.0)) + 1
    e = torch.where(m[at] / torch.exp2(e - 1) < 7.0, e - 1, e)
    e = torch.where(m[at] / torch.exp2(e) < 7.0, e, e + 1)
    s[at] = torch.exp2(e.clamp(min=-127))
    s = s.repeat_interleave(BLOCK, 1)[:, :cols]
    q = x / s
    step = torch.exp2((torch.frexp(q).exponent - 1).clamp(min=0).double() - 1)
    return (torch.round(q / step) * step).clamp(-6.0, 6.0) * s


def _exact_unpack(codes, scales, cols):
    b = codes.long()
    nibble = torch.empty(b.shape[0], 2 * b.shape[1], dtype=torch.int64, device=b.device)
    nibble[:, 0::2], nibble[:, 1::2] = b % 16, b // 16
    mag, sign = nibble % 8, 1.0 - 2.0 * (nibble // 8)
    e, f = (mag // 2).double(), (mag % 2).double()
    v = sign * torch.where(mag < 2, f / 2, torch.exp2(e - 1) * (1 + f / 2))
    s = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1)
    return v[:, :cols] * s[:, :cols]


def _exact_head(x, gamma, st):
    """One head's rows x f64 [tokens, hd]."""
    c = st["case"]
    if gamma is not None:
        x = x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / c["hd"] + EPS) * gamma.double()
    half = c["rot"] // 2
    out = x.clone()
    for pair in range(half):
        at = st["positions"][int(st["pair_axis"][pair])].long()
        a, b = x[:, pair], x[:, pair + half]
        out[:, pair] = a * st["cos"][at, pair].double() - b * st["sin"][at, pair].double()
        out[:, pair + half] = b * st["cos"][at, pair + half].double() + a * st["sin"][at, pair + half].double()
    return out


def _exact_rows(st, name, rows):
    """[kv, rows, hd] of the cache."""
    kv, hd = st["case"]["kv"], st["case"]["hd"]
    return torch.stack([_exact_unpack(st[name + "_codes"][g, :rows], st[name + "_scales"][g, :rows], hd) for g in range(kv)])


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "quantize":
        return _exact_values(st["w"].double())
    if c["op"] == "gemm":
        return torch.matmul(_exact_unpack(st["a"], st["sa"], c["k"]), _exact_unpack(st["b"], st["sb"], c["k"]).t())
    hd = c["hd"]
    if c["op"] == "heads":
        t = st["qkv"].double().view(c["tokens"], -1, hd)
        h, kv = c["heads"], c["kv"]
        q = torch.stack([_exact_head(t[:, i], st["q_gamma"], st) for i in range(h)], 1)
        k = torch.stack([_exact_head(t[:, h + i], st["k_gamma"], st) for i in range(kv)], 1)
        v = t[:, h + kv:]
        if c["into"] == "mxfp4":
            k, v = (_exact_values(x.reshape(-1, hd)) for x in (k, v))
        return [x.reshape(c["tokens"], -1) for x in (q, k, v)]
    rows = c["length"] + c["tokens"]
    if c["op"] == "cache":
        out = []
        for i, n in enumerate(("k", "v")):
            new = st["kv_rows"][:, i * c["kv"] * hd:(i + 1) * c["kv"] * hd].double()
            old = _exact_rows(st, n, c["length"]).transpose(0, 1).reshape(c["length"], -1)
            out.append(torch.vstack([old, _exact_values(new)]))
        return out
    # One head at a time: its queries, its key/value head's rows, the rows each token sees.
    q = st["q"].view(c["tokens"], c["heads"], hd)
    k, v = _exact_rows(st, "k", rows), _exact_rows(st, "v", rows)
    hidden = torch.zeros(c["tokens"], rows, dtype=torch.bool, device="cuda")
    if st["mask"] is None:
        hidden[:, c["length"]:] = torch.ones(c["tokens"], c["tokens"], dtype=torch.bool, device="cuda").triu(1)
    else:
        bits = np.unpackbits(st["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :c["tokens"]]
        hidden[:, c["length"]:] = torch.from_numpy(bits == 0).cuda()
    out = torch.empty(c["tokens"], c["heads"], hd, dtype=torch.float64, device="cuda")
    for h in range(c["heads"]):
        g = h * c["kv"] // c["heads"]
        s = torch.matmul(q[:, h].double(), k[g].t()) * c["scale"]
        out[:, h] = torch.matmul(torch.softmax(s.masked_fill(hidden, -math.inf), 1), v[g])
    return out.view(c["tokens"], -1)
