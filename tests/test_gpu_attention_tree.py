"""Attention of a tree of drafted tokens over a cache, against float64.

Tolerance, per token, head and dimension, with p the exact weights and A = sum_j
p_j |v_j|:

    |got - want| <= 2^-8 |want| + (2^-8 + 2 delta + 64 2^-24) A

2^-8 |want|: the output's rounding to bf16. 2^-8 A: the weights are rounded to
bf16 where they meet the values on the matrix cores (each at most 2^-8 of
itself). delta bounds a score's error, which a weight takes on relatively (twice,
through the sum): products of bf16 values are exact in f32, their sum over
head_dim <= 1024 is off by at most head_dim 2^-24 sum |q k| scale, the scale,
the change of base and the exponential by 2^-21 (1 + |s|). 64 2^-24: the sums
over tiles, waves and splits.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def tree_mask(t, seed, empty=()):
    """Ancestor truth values of a random tree; the tokens in `empty` see no drafted row."""
    rng = np.random.default_rng(seed)
    vis = np.zeros((t, t), dtype=bool)
    for i in range(t):
        back = int(rng.integers(0, min(i, 9) + 1))
        if back:
            vis[i] = vis[i - back]
        vis[i, i] = True
    for i in empty:
        vis[i] = False
    return vis


def pack(vis, junk=True):
    """Words of the truth values; the bits past the last token are set, which says nothing."""
    t = vis.shape[0]
    full = np.full((t, -(-t // 32) * 32), junk)
    full[:, :t] = vis
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def inputs(heads, kv, hd, length, tokens, seed, spare=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda n: torch.randn(n, generator=g, device="cuda").bfloat16()  # noqa: E731
    q = rn(tokens * heads * hd) * 1.5
    k, v = rn((length + tokens + spare) * kv * hd), rn((length + tokens + spare) * kv * hd)
    # Rows behind the last token hold nothing that may be read into a result.
    k[(length + tokens) * kv * hd:] = float("nan")
    v[(length + tokens) * kv * hd:] = float("nan")
    return q, k, v


def reference(q, k, v, heads, kv, hd, length, tokens, vis, scale):
    """(want, bound without the output's rounding) [tokens, heads, hd] in float64."""
    rows = length + tokens
    q = q.view(tokens, heads, hd).double()
    k, v = k[:rows * kv * hd].view(rows, kv, hd).double(), v[:rows * kv * hd].view(rows, kv, hd).double()
    see = torch.ones(tokens, rows, dtype=torch.bool, device="cuda")
    see[:, length:] = torch.from_numpy(vis).cuda()
    want, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(heads):
        g = h // (heads // kv)
        s = (q[:, h] @ k[:, g].T * scale).masked_fill(~see, -float("inf"))
        mag = (q[:, h].abs() @ k[:, g].abs().T * abs(scale)).masked_fill(~see, 0)
        p = torch.softmax(s, 1).masked_fill(~see, 0)   # a row without any seen gives zeros
        delta = (hd * 2.0**-24 * mag + 2.0**-21 * (1 + mag)).amax(1, keepdim=True)
        want[:, h] = p @ v[:, g]
        bound[:, h] = (2.0**-8 + 2 * delta + 64 * 2.0**-24) * (p @ v[:, g].abs())
    return want, bound


def check(R, heads, kv, hd, length, tokens, vis=None, seed=0, scale=None):
    scale = hd**-0.5 if scale is None else scale
    q, k, v = inputs(heads, kv, hd, length, tokens, seed)
    mask = None
    if vis is None:
        vis = np.tril(np.ones((tokens, tokens), dtype=bool))
    else:
        mask = pack(vis)
    want, bound = reference(q, k, v, heads, kv, hd, length, tokens, vis, scale)
    out = torch.full((tokens * heads * hd + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
    n = R.attention_tree_workspace_bytes(heads, kv, hd, length, tokens)
    ws = torch.full((n + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    R.attention_tree(q, k, v, heads, kv, hd, length, tokens, scale, mask, ws[:n] if n else None, out)
    assert (out[tokens * heads * hd:] == 9.0).all(), "written past the output"
    assert (ws[n:] == 0x5A).all(), "written past the workspace"
    got = out[:tokens * heads * hd].view(tokens, heads, hd).double()
    limit = bound + 2.0**-8 * want.abs()
    bad = ~((got - want).abs() <= limit)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), ((got - want).abs() / limit).max().item())
    assert not torch.isnan(got).any()
    return out[:tokens * heads * hd]


CASES = [  # heads, kv, hd, length, tokens
    (1, 1, 128, 0, 1), (4, 4, 64, 1, 1), (8, 2, 128, 31, 2), (32, 8, 128, 500, 16), (28, 4, 128, 63, 33),
    (28, 4, 128, 1000, 7), (8, 8, 128, 4095, 1), (32, 8, 128, 4096, 1), (40, 8, 128, 5000, 5), (8, 1, 64, 700, 9),
    (16, 2, 64, 9000, 12), (9, 3, 64, 257, 65), (4, 2, 256, 300, 20), (2, 1, 256, 2600, 70), (6, 2, 96, 777, 31),
    (10, 5, 96, 64, 129), (5, 1, 128, 129, 255), (28, 4, 128, 2047, 200), (3, 3, 128, 0, 300), (8, 2, 128, 100, 1024),
    (7, 1, 128, 20000, 3), (64, 1, 64, 40, 4), (2, 2, 80, 100, 10), (4, 2, 2, 50, 5), (3, 1, 1024, 60, 4),
    (4, 4, 320, 130, 6), (4, 1, 34, 200, 40),
]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,length,tokens", CASES)
def test_attention_tree_against_float64(R, heads, kv, hd, length, tokens):
    check(R, heads, kv, hd, length, tokens, tree_mask(tokens, length + tokens), seed=hd + length)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,length,tokens", CASES)
def test_attention_chain_against_float64(R, heads, kv, hd, length, tokens):
    check(R, heads, kv, hd, length, tokens, None, seed=hd + length + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
def test_tokens_that_see_nothing_give_zeros(R, hd):
    vis = tree_mask(40, 3, empty=(0, 17, 39))
    out = check(R, 8, 2, hd, 0, 40, vis).view(40, -1)
    assert (out[[0, 17, 39]] == 0).all()
    check(R, 8, 2, hd, 3, 40, vis)           # with context they see that


@pytest.mark.gpu
@pytest.mark.parametrize("length", [0, 37, 2000])
@pytest.mark.parametrize("hd", [64, 96, 128, 256, 80])
def test_rows_not_seen_may_hold_anything(R, hd, length):
    """NaN and infinities in drafted rows reach the tokens that see them and no others."""
    heads, kv, tokens = 8, 2, 70
    vis = tree_mask(tokens, 5)
    bad = {11: float("nan"), 30: float("inf"), 64: -float("inf")}
    for j in bad:
        vis[:, j] = False
        vis[j, j] = True
    q, k, v = inputs(heads, kv, hd, length, tokens, 9)
    scale = hd**-0.5
    want = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, scale, pack(vis)).view(tokens, -1)
    k2, v2 = k.view(-1, kv * hd).clone(), v.view(-1, kv * hd).clone()
    for j, x in bad.items():
        v2[length + j] = x
        k2[length + j] = x
    got = R.attention_tree(q, k2, v2, heads, kv, hd, length, tokens, scale, pack(vis)).view(tokens, -1)
    others = [i for i in range(tokens) if i not in bad]
    assert torch.equal(got[others].view(torch.int16), want[others].view(torch.int16))
    assert torch.isnan(got[11]).all()
    # Infinities in the values alone: those who see them get them, by their weight's sign.
    v3 = v.view(-1, kv * hd).clone()
    v3[length + 30] = float("inf")
    got = R.attention_tree(q, k, v3, heads, kv, hd, length, tokens, scale, pack(vis)).view(tokens, -1)
    others = [i for i in range(tokens) if i != 30]
    assert torch.equal(got[others].view(torch.int16), want[others].view(torch.int16))
    assert (got[30] == float("inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,length", [(128, 100), (128, 3000), (64, 10), (80, 40)])
def test_scores_of_minus_infinity_and_nan(R, hd, length):
    """A score of -inf among others has no weight; scores that are all -inf, or one NaN, give NaN."""
    heads, kv, tokens = 4, 1, 6
    q, k, v = inputs(heads, kv, hd, length, tokens, 2)
    q, k = q.view(tokens, heads, hd), k.view(-1, hd)
    q[:, :, 0] = 1.0
    k[:, 0] = 0.0
    base = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).view(tokens, -1)
    k[5, 0] = -float("inf")                  # one context row no token can weigh
    v0 = v.view(-1, hd).clone()
    got = R.attention_tree(q, k, v0, heads, kv, hd, length, tokens, 0.1).view(tokens, -1)
    assert torch.isfinite(got).all() and not torch.equal(got, base)
    k[:, 0] = -float("inf")
    got = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1)
    assert torch.isnan(got).all()
    k[:, 0] = 0.0
    k[length + 2, 3] = float("nan")          # seen by tokens 2 .. 5 of the chain
    got = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).view(tokens, -1)
    assert torch.equal(got[:2].view(torch.int16), base[:2].view(torch.int16)) and torch.isnan(got[2:]).all()


@pytest.mark.gpu
def test_large_scores_and_scales(R):
    check(R, 8, 2, 128, 900, 20, tree_mask(20, 1), scale=2.0)      # one row takes nearly all the weight
    check(R, 8, 2, 128, 900, 20, tree_mask(20, 1), scale=0.0)      # all rows weigh the same
    check(R, 8, 2, 128, 900, 20, tree_mask(20, 1), scale=-0.3)


@pytest.mark.gpu
def test_one_token_is_the_decode_attention(R):
    """A single token that sees itself: attention_decode_split over len + 1 rows, within both roundings."""
    for heads, kv, hd, length in [(32, 8, 128, 600), (8, 2, 64, 5000), (4, 4, 80, 40)]:
        q, k, v = inputs(heads, kv, hd, length, 1, 4)
        a = R.attention_decode_split(q, k, v, heads, kv, hd, length + 1, hd**-0.5).double()
        b = R.attention_tree(q, k, v, heads, kv, hd, length, 1, hd**-0.5).double()
        assert (a - b).norm() <= 2.0**-7 * a.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [4, 8])
def test_unaligned_caches(R, offset):
    """Caches, queries and outputs on 4- and 8-byte boundaries."""
    heads, kv, hd, length, tokens = 8, 2, 128, 300, 10
    q, k, v = inputs(heads, kv, hd, length, tokens, 6)
    want = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).double()

    def moved(t):
        buf = torch.empty(t.numel() + offset // 2, dtype=t.dtype, device="cuda")
        buf[offset // 2:] = t
        return buf[offset // 2:]

    for args in [(moved(q), k, v), (q, moved(k), v), (q, k, moved(v))]:
        got = R.attention_tree(*args, heads, kv, hd, length, tokens, 0.1).double()
        assert (got - want).norm() <= 2.0**-7 * want.norm()
    out = moved(torch.empty_like(q))
    R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1, out=out)
    assert (out.double() - want).norm() <= 2.0**-7 * want.norm()


@pytest.mark.gpu
def test_attention_tree_streams_graphs_and_workspaces(R):
    """On a side stream, captured and replayed over a cache that changes; a workspace larger than needed, dirty
    from another call."""
    heads, kv, hd, length, tokens = 32, 8, 128, 3000, 12
    q, k, v = inputs(heads, kv, hd, length, tokens, 7)
    mask = pack(tree_mask(tokens, 2))
    n = R.attention_tree_workspace_bytes(heads, kv, hd, 8000, 64)
    assert n >= R.attention_tree_workspace_bytes(heads, kv, hd, length, tokens)
    ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)

    def step():
        R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.08, mask, ws, out)

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step()
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    for i in range(4):
        k.view(-1, kv * hd)[:length + tokens].mul_(-0.9)
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), out.view(torch.int16))
        fresh = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.08, mask)
        assert torch.equal(fresh.view(torch.int16), out.view(torch.int16))


def test_tree_workspace_grows_with_the_call():
    import reng_hip as R

    R.lib()
    f = R.attention_tree_workspace_bytes
    for heads, kv, hd in [(32, 8, 128), (8, 1, 64), (28, 4, 128), (4, 4, 256), (6, 2, 96), (4, 4, 80)]:
        for length, tokens in [(0, 1), (100, 1), (1000, 16), (5000, 3), (32768, 63), (130000, 1000)]:
            most = f(heads, kv, hd, length, tokens)
            rng = np.random.default_rng(length + tokens)
            for _ in range(200):
                a, b = int(rng.integers(0, length + 1)), int(rng.integers(1, tokens + 1))
                assert f(heads, kv, hd, a, b) <= most, (heads, kv, hd, length, tokens, a, b)


def test_attention_tree_refusals():
    import ctypes

    import reng_hip as R

    L = R.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)

    def refused(words, q=p, k=p, v=p, heads=8, kv=2, hd=128, length=100, tokens=4, mask=p, ws=p, wb=1 << 30, out=p):
        rc = L.reng_hip_attention_tree(q, k, v, heads, kv, hd, length, tokens, mask, 0.1, ws, wb, out, None)
        msg = L.reng_hip_last_error().decode()
        assert rc == R.EINVAL and words in msg, msg

    refused("not a multiple", heads=7)
    refused("not a multiple", heads=0)
    refused("not a multiple", kv=0)
    refused("head_dim 0", hd=0)
    refused("head_dim 63", hd=63)
    refused("head_dim 1026", hd=1026)
    refused("0 tokens", tokens=0)
    refused("1025 tokens", tokens=1025)
    refused("at most 131072", length=131072)
    refused("at most 131072", length=(1 << 64) - 1)
    refused("at most 4096", heads=8192)
    for name in ("q", "k", "v", "out"):
        refused("null", **{name: None})
    for name in ("q", "k", "v", "out", "mask"):
        refused("aligned", **{name: odd})
    refused("aligned", ws=ctypes.c_void_p(4104))
    need = R.attention_tree_workspace_bytes(8, 2, 128, 100000, 4)
    if need:
        refused("workspace", length=100000, wb=need - 1)
        refused("null workspace", length=100000, ws=None)


def test_the_binding_refuses_wrong_tree_operands():
    from test_abi import _FakeDev as Fake

    import reng_hip as R

    bf = torch.bfloat16
    heads, kv, hd, length, tokens = 4, 2, 64, 10, 33
    nq, nc = tokens * heads * hd, (length + tokens) * kv * hd
    good = dict(q=Fake(2 * nq, bf), k=Fake(2 * nc, bf), v=Fake(2 * nc, bf), mask=Fake(4 * tokens * 2, torch.int32),
                out=Fake(2 * nq, bf))
    for name, bad, what in [("q", Fake(2 * nq - 2, bf), "q length"), ("k", Fake(2 * nc - 2, bf), "k_cache length"),
                            ("v", Fake(2 * nc - 2, bf), "v_cache length"), ("out", Fake(2 * nq - 2, bf), "out length"),
                            ("mask", Fake(4 * tokens, torch.int32), "mask length"),
                            ("mask", Fake(4 * tokens * 2, torch.uint8), "32-bit words"),
                            ("q", Fake(4 * nq, torch.float32), "q must be bf16")]:
        a = {**good, name: bad}
        with pytest.raises(ValueError, match=what):
            R.attention_tree(a["q"], a["k"], a["v"], heads, kv, hd, length, tokens, 0.1, a["mask"],
                             Fake(1 << 24), a["out"])
