"""Attention over a cache held in 4 bits, against float64 over the values its codes stand for.

The tolerance is that of the tree attention (test_gpu_attention_tree.py): those values are bf16 exactly, so the products
are the same. Beside it 2^-125 sum |v| over the rows: a weight is held against a maximum whose own weight is 1 to 2^8, so
the sum it is divided by is 1 or more, and f32 and bf16 flush weights below 2^-126, where float64 does not (at a
scale of 3 the exact outputs go down to 2^-800).
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mx_plans as D  # noqa: E402
import mx_reference as X  # noqa: E402
from test_gpu_attention_tree import pack, reference, tree_mask  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def make(R, heads, kv, hd, length, tokens, seed, spare=5):
    """(q, cache, k, v): a cache of random rows, NaN behind them, and its values [rows * kv * hd]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rows = length + tokens
    cache = R.MxCache(kv, hd, rows + spare)
    vals = []
    for i in range(2):
        x = rn(kv * rows, hd) * torch.exp2(rn(kv * rows, 1))
        code, byte = X.quantize(x.double())
        full = [t.view(kv, rows + spare, -1) for t in cache.tensors[2 * i:2 * i + 2]]
        for t, part in zip(full, X.pack(code, byte)):
            t.fill_(255)
            t[:, :rows] = part.view(kv, rows, -1)
        vals.append(X.values(code, byte).view(kv, rows, hd).transpose(0, 1).reshape(-1))
    return (rn(tokens * heads * hd) * 1.5).bfloat16(), cache, vals[0], vals[1]


def check(R, heads, kv, hd, length, tokens, vis=None, seed=0, scale=None):
    scale = hd**-0.5 if scale is None else scale
    q, cache, k, v = make(R, heads, kv, hd, length, tokens, seed)
    mask = None if vis is None else pack(vis)
    vis = np.tril(np.ones((tokens, tokens), dtype=bool)) if vis is None else vis
    want, bound = reference(q, k, v, heads, kv, hd, length, tokens, vis, scale)
    n = R.attention_mxfp4_workspace_bytes(heads, kv, hd, length, tokens)
    out = torch.full((tokens * heads * hd + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((n + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    R.attention_mxfp4(q, cache, heads, length, tokens, scale, mask, ws[:n] if n else None, out)
    assert (out[tokens * heads * hd:] == 9.0).all(), "written past the output"
    assert (ws[n:] == 0x5A).all(), "written past the workspace"
    got = out[:tokens * heads * hd].view(tokens, heads, hd).double()
    lost = 2.0**-125 * v.abs().view(-1, kv, hd).sum(0).repeat_interleave(heads // kv, 0)
    limit = bound + 2.0**-8 * want.abs() + lost
    bad = ~((got - want).abs() <= limit)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), ((got - want).abs() / limit).max().item())
    return out[:tokens * heads * hd]


CASES = [  # heads, kv, hd, length, tokens
    (1, 1, 128, 0, 1), (4, 4, 64, 1, 1), (8, 2, 128, 31, 2), (32, 8, 128, 500, 16), (28, 4, 128, 63, 33),
    (28, 4, 128, 1000, 7), (8, 8, 128, 4095, 1), (32, 8, 128, 4096, 1), (40, 8, 128, 5000, 5), (8, 1, 64, 700, 9),
    (16, 2, 64, 9000, 12), (9, 3, 64, 257, 65), (4, 2, 256, 300, 20), (2, 1, 256, 2600, 70), (6, 2, 96, 777, 31),
    (10, 5, 96, 64, 129), (5, 1, 128, 129, 255), (28, 4, 128, 2047, 200), (3, 3, 128, 0, 300), (8, 2, 128, 100, 1024),
    (7, 1, 128, 20000, 3), (64, 1, 64, 40, 4), (2, 2, 32, 100, 10), (4, 2, 160, 50, 5), (3, 1, 224, 3000, 4),
    (4, 4, 192, 130, 6), (16, 2, 256, 4000, 1), (24, 24, 32, 1, 3), (32, 8, 128, 131071, 1),
]


@pytest.mark.parametrize("heads,kv,hd,length,tokens", CASES)
def test_tree_against_float64(R, heads, kv, hd, length, tokens):
    check(R, heads, kv, hd, length, tokens, tree_mask(tokens, length + tokens), seed=hd + length)


@pytest.mark.parametrize("heads,kv,hd,length,tokens", CASES)
def test_chain_against_float64(R, heads, kv, hd, length, tokens):
    check(R, heads, kv, hd, length, tokens, None, seed=hd + length + 1)


@pytest.mark.parametrize("heads,kv,hd,length,tokens", D.ATTENTION_SHAPES)
def test_every_kernel(R, heads, kv, hd, length, tokens):
    check(R, heads, kv, hd, length, tokens, None, seed=length + tokens)
    vis = tree_mask(tokens, length, empty=(0, tokens // 2, tokens - 1))
    out = check(R, heads, kv, hd, length, tokens, vis, seed=length + tokens + 1).view(tokens, -1)
    if length == 0:
        assert (out[[0, tokens // 2, tokens - 1]] == 0).all()


@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 511, 1023, 2049])
def test_lengths(R, length):
    check(R, 8, 2, 128, length, 1, seed=length)
    check(R, 8, 2, 64, length, 9, tree_mask(9, length), seed=length)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_tokens_that_see_nothing_give_zeros(R, hd):
    vis = tree_mask(40, 3, empty=(0, 17, 39))
    out = check(R, 8, 2, hd, 0, 40, vis).view(40, -1)
    assert (out[[0, 17, 39]] == 0).all()
    check(R, 8, 2, hd, 3, 40, vis)           # with context they see that


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-30, 3.0])
def test_scales(R, scale):
    check(R, 8, 2, 128, 300, 5, tree_mask(5, 1), scale=scale)
    check(R, 8, 2, 64, 3000, 1, scale=scale)


@pytest.mark.parametrize("length,tokens", [(0, 40), (37, 40), (2000, 5), (5000, 70), (100, 600), (0, 200)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_that_are_not_seen_take_no_part(R, hd, length, tokens):
    """Rows of NaN scales and the largest values that a token does not see change none of its bits; those that it sees make it NaN."""
    heads, kv = 8, 2
    vis = tree_mask(tokens, 7)
    vis[:, 1] = False
    vis[1] = False
    vis[1, 1] = True
    q, cache, _, _ = make(R, heads, kv, hd, length, tokens, 11)
    mask = pack(vis)
    clean = R.attention_mxfp4(q, cache, heads, length, tokens, hd**-0.5, mask).view(tokens, -1).clone()
    for which, byte, block in ((1, 255, 0), (3, 255, hd // 32 - 1), (3, 253, 0), (1, 254, 0)):
        scales = cache.tensors[which].view(kv, -1, X.pitch(hd))
        old = scales[:, length + 1].clone()
        scales[:, length + 1, block] = byte
        got = R.attention_mxfp4(q, cache, heads, length, tokens, hd**-0.5, mask).view(tokens, -1)
        others = [i for i in range(tokens) if i != 1]
        assert torch.equal(got[others].view(torch.int16), clean[others].view(torch.int16)), (which, byte)
        assert torch.isnan(got[1]).all()
        scales[:, length + 1] = old


def test_large_finite_values(R):
    """Values of 2^100 overflow no sum, and weights of 0 take nothing from them."""
    heads, kv, hd, length = 4, 1, 128, 700
    q, cache, k, v = make(R, heads, kv, hd, length, 1, 12)
    cache.tensors[3].view(-1, 4)[:length + 1] = 127 + 98
    cache.tensors[2].view(-1, 64)[:length + 1] = 0x66   # 4
    out = R.attention_mxfp4(q, cache, heads, length, 1, hd**-0.5).double()
    assert ((out - 2.0**100).abs() <= 2.0**92).all()


def test_infinite_and_nan_queries(R):
    heads, kv, hd, length, tokens = 4, 2, 128, 100, 3
    q, cache, _, _ = make(R, heads, kv, hd, length, tokens, 13)
    want = R.attention_mxfp4(q, cache, heads, length, tokens, 0.1).view(tokens, heads, hd)
    bad = q.clone().view(tokens, heads, hd)
    bad[1, 0, 3], bad[2, 3, 9] = float("nan"), float("inf")
    got = R.attention_mxfp4(bad.view(-1), cache, heads, length, tokens, 0.1).view(tokens, heads, hd)
    assert torch.isnan(got[1, 0]).all() and torch.isnan(got[2, 3]).all()
    keep = torch.ones(tokens, heads, dtype=torch.bool, device="cuda")
    keep[1, 0] = keep[2, 3] = False
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("heads,kv,hd,length,tokens", [(32, 8, 128, 4096, 1), (28, 4, 128, 1000, 40), (4, 2, 256, 3000, 3)])
def test_captured_calls_replay(R, heads, kv, hd, length, tokens):
    """A step captured into a graph (write, then attention) and replayed with eager work between: every replay is the eager result."""
    q, cache, _, _ = make(R, heads, kv, hd, length, tokens, 14)
    n = R.attention_mxfp4_workspace_bytes(heads, kv, hd, length, tokens)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    kv_rows = torch.empty(2, tokens, kv * hd, dtype=torch.bfloat16, device="cuda")

    def step():
        cache.write(kv_rows[0], kv_rows[1], length, tokens)
        R.attention_mxfp4(q, cache, heads, length, tokens, hd**-0.5, None, ws, out)

    g = torch.Generator(device="cuda").manual_seed(3)
    kv_rows.copy_(torch.randn(kv_rows.shape, generator=g, device="cuda"))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(3):
        kv_rows.copy_(torch.randn(kv_rows.shape, generator=g, device="cuda"))
        step()
        want = out.clone()
        out.zero_()
        ws.fill_(0xA5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)), rep


def test_two_streams_with_workspaces_of_their_own(R):
    heads, kv, hd, length, tokens = 16, 4, 128, 4000, 6
    made = [make(R, heads, kv, hd, length, tokens, 20 + i) for i in range(2)]
    alone = [R.attention_mxfp4(m[0], m[1], heads, length, tokens, 0.1) for m in made]
    n = R.attention_mxfp4_workspace_bytes(heads, kv, hd, length, tokens)
    assert n > 0
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = [torch.empty_like(alone[0]) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                R.attention_mxfp4(made[i][0], made[i][1], heads, length, tokens, 0.1, None, ws[i], out[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i].view(torch.int16), alone[i].view(torch.int16))
