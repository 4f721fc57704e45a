"""The 4-bit operators where an operand passes 2^32 bytes or elements.

What lies behind that border decides the values compared: a wrapped offset reads other rows (the patterns' period
of 1001 rows divides no power of two) or writes elsewhere.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_reference as X  # noqa: E402
from test_gpu_long_offsets import PERIOD, R, randn, repeated  # noqa: E402, F401
from test_gpu_mxfp4 import operand  # noqa: E402

pytestmark = pytest.mark.gpu
ROWS, COLS = 528128, 16384   # 2^33 + 60 * 2^20 codes


def test_quantize_and_back(R):  # noqa: F811
    w = repeated(randn(0, PERIOD, COLS).bfloat16(), ROWS)
    codes, scales = R.quantize_mxfp4(w, ROWS, COLS)
    last = w[-1024:].contiguous()
    del w
    want = R.quantize_mxfp4(last, 1024, COLS)
    assert codes.numel() > 2**32
    assert torch.equal(codes[-want[0].numel():], want[0]) and torch.equal(scales[-want[1].numel():], want[1])
    got = R.dequantize_mxfp4(codes, scales, ROWS, COLS)
    assert torch.equal(got[-1024 * COLS:], R.dequantize_mxfp4(*want, 1024, COLS))


@pytest.mark.parametrize("M", [1, 24, 80, 300])
def test_product_of_long_weights(R, M):  # noqa: F811
    a, base = operand(M, COLS, M), operand(PERIOD, COLS, 3)
    pa, pb = X.pack(*a), X.pack(*base)
    out = R.gemm_mxfp4(*pa, *(repeated(t, ROWS) for t in pb), M, ROWS, COLS).view(M, ROWS)[:, -256:]
    va, vb = X.values(*a), X.values(*base)[torch.arange(ROWS - 256, ROWS, device="cuda") % PERIOD]
    want, t = va @ vb.T.contiguous(), va.abs() @ vb.abs().T.contiguous()
    bound = 2.0**-8 * want.abs() + (2.0**-12 + (COLS // 128 + 24) * 2.0**-23) * t
    assert ((out.double() - want).abs() <= bound).all()


def test_product_of_many_outputs(R):  # noqa: F811
    M, N, K = 66048, 65536, 160
    a, b = operand(M, K, 5), operand(N, K, 6)
    out = R.gemm_mxfp4(*X.pack(*a), *X.pack(*b), M, N, K).view(M, N)[-256:]
    va, vb = X.values(a[0][-256:], a[1][-256:]), X.values(*b)
    want, t = va @ vb.T.contiguous(), va.abs() @ vb.abs().T.contiguous()
    assert ((out.double() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-12 + 26 * 2.0**-23) * t).all()


def test_a_long_cache(R):  # noqa: F811
    kv, hd, capacity, length, tokens = 66, 256, 2**19, 2000, 3
    large, small = R.MxCache(kv, hd, capacity), R.MxCache(kv, hd, length + tokens)
    assert large.tensors[0].numel() - capacity * hd // 2 > 2**32   # the last head starts behind the border
    k, v = (randn(i, length + tokens, kv * hd).bfloat16() for i in range(2))
    q = randn(3, tokens * kv * hd).bfloat16()
    for c in (large, small):
        c.write(k, v, 0, length + tokens)
    out = [R.attention_mxfp4(q, c, kv, length, tokens, hd**-0.5) for c in (large, small)]
    assert torch.equal(out[0], out[1])
    for first in (0, capacity - 1001):
        large.write(k, v, first, 1001)
        for g, w in zip(large.read(first, 1001), small.read(0, 1001)):
            assert torch.equal(g, w)


def test_long_rows_of_heads(R):  # noqa: F811
    tokens, ld = 5000, 2**20
    qkv = torch.zeros(tokens, ld, dtype=torch.bfloat16, device="cuda")
    qkv[-64:, -1536:] = randn(5, 64, 1536).bfloat16()
    q, k, v = qkv[:, -1536:-512], qkv[:, -512:-256], qkv[:, -256:]
    ang = randn(6, 50, 128) * 3
    args = dict(q_gamma=1 + 0.1 * randn(7, 128), k_gamma=1 + 0.1 * randn(8, 128), rope=R.Rope(ang.sin(), ang.cos()))
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32) % 50
    got = R.head_norm_rope_bf16(q, k, v, tokens, 8, 2, 128, positions=pos, **args)
    want = R.head_norm_rope_bf16(q[-64:], k[-64:], v[-64:], 64, 8, 2, 128, positions=pos[-64:].contiguous(), **args)
    for g, w in zip(got, want):
        assert torch.equal(g[-w.numel():], w) and w.abs().sum() > 0
