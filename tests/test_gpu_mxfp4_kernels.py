"""Kernels of the 4-bit operators that few calls choose: the product of one row over split k, and head norms and writes of
unaligned rows for every number of lanes a head.

Tolerances are those of test_gpu_mxfp4.py; unaligned rows give the bits of aligned ones.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_plans as D  # noqa: E402
from test_gpu_heads import Case, near  # noqa: E402
from test_gpu_mxfp4 import check_product  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


@pytest.mark.parametrize("N,K", D.ROW_SHAPES)
def test_one_row(R, N, K):
    check_product(R, 1, N, K, N)


# Heads, their size, rotation and axes, and where rows start; of 1100 tokens some take four heads a group of lanes.
ROWS = [
    (4, 2, 32, 32, 1, 1), (140, 3, 32, 16, 2, 3), (5, 1, 64, 64, 3, 1), (60, 7, 64, 32, 1, 5), (3, 1, 96, 96, 1, 2),
    (31, 3, 128, 128, 3, 7), (4, 2, 160, 80, 4, 1), (9, 5, 160, 160, 2, 3), (6, 1, 256, 256, 1, 4), (19, 2, 256, 64, 3, 1),
    (2, 2, 224, None, 1, 1),
]


@pytest.mark.parametrize("tokens", [13, 1100])
@pytest.mark.parametrize("heads,kv,hd,rot,axes,off", ROWS)
def test_unaligned_rows(R, heads, kv, hd, rot, axes, off, tokens):
    """Rows that start anywhere, of an odd pitch: against 64 bits, and the bits of aligned rows, as rows and in the cache."""
    c = Case(tokens, heads, kv, hd, rot, axes, True, seed=hd + off)
    nq, nk, n = heads * hd, kv * hd, c.qkv.shape[1]
    wide = torch.zeros(tokens, n + off + 9, dtype=torch.bfloat16, device="cuda")
    wide[:, off:off + n] = c.qkv
    q, k, v = (wide[:, off + a:off + b] for a, b in ((0, nq), (nq, nq + nk), (nq + nk, n)))
    flat = [t.contiguous() for t in (c.q, c.k, c.v)]
    want = R.head_norm_rope_bf16(*flat, tokens, heads, kv, hd, **c.args(R))
    near(want[0], *c.exact(c.q, c.gq), "q")
    near(want[1], *c.exact(c.k, c.gk), "k")
    # Outputs that start anywhere, too.
    outs = [torch.full((t.numel() + off + 64,), 7.0, dtype=torch.bfloat16, device="cuda") for t in want]
    at = [o[off:off + w.numel()] for o, w in zip(outs, want)]
    R.head_norm_rope_bf16(q, k, v, tokens, heads, kv, hd, **c.args(R), q_out=at[0], k_rows=at[1], v_rows=at[2])
    for o, g, w in zip(outs, at, want):
        assert torch.equal(g.view(torch.int16), w.view(torch.int16))
        assert (o[:off] == 7.0).all() and (o[off + w.numel():] == 7.0).all(), "written beside the output"
    caches = [R.MxCache(kv, hd, tokens + 5) for _ in range(2)]
    for cache, rows in zip(caches, (flat, (q, k, v))):
        for t in cache.tensors:
            t.fill_(0x5A)
        got = R.head_norm_rope_mxfp4(*rows, tokens, heads, cache, 3, **c.args(R))
        assert torch.equal(got.view(torch.int16), want[0].view(torch.int16))
    for g, w in zip(caches[0].tensors, caches[1].tensors):
        assert torch.equal(g, w)
