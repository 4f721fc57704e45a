"""The 4-bit operators without a GPU: refusals, which come before any device work, and the attention's plans."""
import ctypes
import random

import pytest

import mx_plans as D
import reng_hip as R

P = ctypes.c_void_p(64)   # never dereferenced: the checks come first


def refused(rc, text):
    assert rc == R.EINVAL and text in R.lib().reng_hip_last_error().decode(), R.lib().reng_hip_last_error()


def cache(kc=64, ks=64, vc=64, vs=64, kv=2, hd=128, cap=100):
    return R._MxCache(kc, ks, vc, vs, kv, hd, cap)


def rope(sin=64, cos=64, rows=10, rot=128, axes=1, pairs=None):
    return R._Rope(sin, cos, rows, rot, axes, pairs)


def test_quantizer_refusals():
    q, d = R.lib().reng_hip_quantize_mxfp4, R.lib().reng_hip_dequantize_mxfp4
    refused(q(P, R.BF16, 0, 32, 32, P, P, None), "empty shape 0 x 32")
    refused(q(P, R.BF16, 1, 0, 32, P, P, None), "empty shape")
    refused(q(P, 5, 1, 32, 32, P, P, None), "unknown dtype")
    refused(q(P, R.BF16, 1, 32, 31, P, P, None), "row pitch 31")
    refused(q(P, R.BF16, 1, 2**31, 2**31, P, P, None), "too large")
    refused(q(None, R.BF16, 1, 32, 32, P, P, None), "null")
    refused(q(P, R.BF16, 1, 32, 32, P, ctypes.c_void_p(66), None), "4 bytes")
    refused(q(ctypes.c_void_p(65), R.BF16, 1, 32, 32, P, P, None), "aligned")
    refused(q(ctypes.c_void_p(66), R.F32, 1, 32, 32, P, P, None), "aligned")
    refused(d(P, P, 1, 0, R.BF16, P, None), "empty shape")
    refused(d(P, P, 1, 32, 7, P, None), "unknown dtype")
    refused(d(P, None, 1, 32, R.F32, P, None), "null")
    refused(d(P, P, 1, 32, R.F32, ctypes.c_void_p(66), None), "aligned")
    refused(d(P, ctypes.c_void_p(65), 1, 32, R.BF16, P, None), "4 bytes")


def test_product_refusals():
    g = R.lib().reng_hip_gemm_mxfp4
    refused(g(P, P, P, P, 0, 8, 64, P, None), "empty product")
    refused(g(P, P, P, P, 4, 8, 48, P, None), "multiple of 32")
    refused(g(P, P, P, P, 4, 8, (1 << 22) + 32, P, None), "too large")
    refused(g(P, P, P, P, 2**31, 8, 32, P, None), "too large")
    refused(g(P, P, P, P, 2**31 - 1, 2**31 - 1, 32, P, None), "too many for a launch")
    refused(g(P, P, P, P, 1, 2**31 - 1, 32, P, None), "too many for a launch")
    refused(g(P, P, P, P, 16, 2**31 - 1, 32, P, None), "too many for a launch")
    refused(g(P, None, P, P, 4, 8, 64, P, None), "null")
    refused(g(P, P, ctypes.c_void_p(72), P, 4, 8, 64, P, None), "16-byte")
    refused(g(P, P, P, ctypes.c_void_p(65), 4, 8, 64, P, None), "4-byte")
    refused(g(P, P, P, P, 4, 8, 64, ctypes.c_void_p(65), None), "aligned")


@pytest.mark.parametrize("bad,text", [
    (dict(kv=0), "key/value heads"), (dict(kv=4097), "key/value heads"), (dict(hd=48), "multiple of 32"),
    (dict(hd=288), "multiple of 32"), (dict(hd=0), "multiple of 32"), (dict(cap=0), "capacity"), (dict(cap=2**31), "capacity"),
    (dict(kc=None), "null"), (dict(vs=None), "null"), (dict(vc=72), "16-byte"), (dict(ks=66), "aligned")])
def test_every_call_refuses_a_bad_cache(bad, text):
    L, c = R.lib(), cache(**bad)
    ref = ctypes.byref(c)
    refused(L.reng_hip_cache_read_mxfp4(ref, 0, 1, P, P, None), text)
    refused(L.reng_hip_head_norm_rope_mxfp4(P, 4096, P, P, 4096, 1, 1, None, None, 1e-6, None, None, P, ref, 0, None), text)
    refused(L.reng_hip_attention_mxfp4(P, ref, 4, 10, 1, None, 0.1, P, 1 << 30, P, None), text)


def test_no_cache():
    refused(R.lib().reng_hip_cache_read_mxfp4(None, 0, 1, P, P, None), "null cache")


def test_cache_read_refusals():
    f, c = R.lib().reng_hip_cache_read_mxfp4, ctypes.byref(cache())
    refused(f(c, 0, 0, P, P, None), "no rows")
    refused(f(c, 0, 101, P, P, None), "rows 0 .. 101")
    refused(f(c, 100, 1, P, P, None), "rows 100")
    refused(f(c, 2**64 - 1, 2, P, P, None), "of a cache of 100")
    refused(f(c, 0, 1, None, None, None), "null")
    refused(f(c, 0, 1, ctypes.c_void_p(72), P, None), "16-byte")


def heads(q=P, q_ld=512, k=P, v=P, kv_ld=256, tokens=3, nh=4, nkv=2, hd=128, gq=None, gk=None, eps=1e-6, rp=None, pos=None,
          q_out=P, k_rows=P, v_rows=P):
    return R.lib().reng_hip_head_norm_rope_bf16(q, q_ld, k, v, kv_ld, tokens, nh, nkv, hd, gq, gk, eps, rp, pos, q_out, k_rows,
                                                v_rows, None)


@pytest.mark.parametrize("bad,text", [
    (dict(tokens=0), "tokens"), (dict(tokens=1 << 22), "tokens"), (dict(nh=4097, q_ld=2**20), "heads"), (dict(nkv=0), "heads"),
    (dict(hd=40), "multiple of 32"), (dict(hd=288, q_ld=2000, kv_ld=2000), "multiple of 32"), (dict(q=None), "null"),
    (dict(q_out=None), "null"), (dict(nh=0), "0 query heads"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(v_rows=None), "null"), (dict(k_rows=None), "null"), (dict(q_ld=511), "query row pitch 511"),
    (dict(kv_ld=255), "key/value row pitch"), (dict(kv_ld=2**31), "too large"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(q=ctypes.c_void_p(65)), "aligned"), (dict(gq=ctypes.c_void_p(66)), "aligned"),
    (dict(k_rows=ctypes.c_void_p(65)), "aligned"), (dict(tokens=2**22 - 1, nh=4096, nkv=4096, q_ld=2**20, kv_ld=2**20), "too many"),
    (dict(rp=dict(rot=24), pos=P), "rot_dim 24"), (dict(rp=dict(rot=144), pos=P), "rot_dim 144"), (dict(rp=dict(rot=0), pos=P), "rot_dim 0"),
    (dict(rp=dict(axes=0), pos=P), "0 axes"), (dict(rp=dict(axes=5), pos=P), "5 axes"), (dict(rp=dict(rows=0), pos=P), "0 rows"),
    (dict(rp=dict(rows=2**31), pos=P), "rows"), (dict(rp=dict(sin=None), pos=P), "null"), (dict(rp=dict()), "null"),
    (dict(rp=dict(cos=72), pos=P), "16-byte"), (dict(rp=dict(), pos=ctypes.c_void_p(66)), "aligned"),
    (dict(rp=dict(axes=2, pairs=bytes([1] * 63 + [2])), pos=P), "pair 63 has axis 2 of 2")])
def test_heads_refusals(bad, text):
    if "rp" in bad:
        bad = dict(bad, rp=ctypes.byref(rope(**bad["rp"])))
    refused(heads(**bad), text)


def test_heads_into_a_cache_refusals():
    f, c = R.lib().reng_hip_head_norm_rope_mxfp4, cache()

    def call(first=0, tokens=3, v=P, nh=4):
        return f(P, 512, P, v, 256, tokens, nh, None, None, 1e-6, None, None, P, ctypes.byref(c), first, None)
    refused(call(first=98), "rows 98 .. 101 of a cache of 100")
    refused(call(first=2**64 - 2), "of a cache of 100")
    refused(call(tokens=101), "of a cache of 100")
    refused(call(v=None), "null")
    refused(call(nh=0), "0 query heads")


def attention(c=None, q=P, nh=4, length=10, tokens=1, mask=None, scale=0.1, ws=P, nb=1 << 30, out=P):
    c = cache() if c is None else c
    return R.lib().reng_hip_attention_mxfp4(q, ctypes.byref(c), nh, length, tokens, mask, scale, ws, nb, out, None)


def test_attention_refusals():
    refused(attention(nh=3), "not a multiple")
    refused(attention(nh=0), "not a multiple")
    refused(attention(nh=4098), "at most 4096")
    refused(attention(tokens=0), "0 tokens")
    refused(attention(tokens=1025), "1025 tokens")
    refused(attention(length=100), "in a cache of 100")
    refused(attention(cache(cap=2**20), length=131072), "at most 131072 rows")
    refused(attention(cache(cap=2**20), length=2**64 - 1), "at most 131072 rows")
    refused(attention(scale=float("nan")), "scale")
    refused(attention(scale=float("inf")), "scale")
    refused(attention(q=None), "null")
    refused(attention(q=ctypes.c_void_p(72)), "16-byte")
    refused(attention(out=ctypes.c_void_p(68)), "16-byte")
    refused(attention(mask=ctypes.c_void_p(66)), "4-byte")


def test_the_binding_refuses_rows_that_are_too_short():
    import torch

    class Dev(torch.Tensor):
        is_cuda = property(lambda self: True)

    def dev(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype).as_subclass(Dev)

    R._torch()
    assert R._rows16(dev(4, 100)[:, 20:70], "k", 4, 50)[1] == 100
    for t, tokens, width in ((dev(2, 100), 4, 50), (dev(4, 100), 4, 101), (dev(4, 100).t(), 4, 4), (dev(199), 4, 50),
                             (dev(4, 50, dtype=torch.float32), 4, 50)):
        with pytest.raises(ValueError):
            R._rows16(t, "k", tokens, width)
    with pytest.raises(ValueError, match="32 pairs|pairs"):
        R.Rope(torch.zeros(4, 64), torch.zeros(4, 64), sections=(16, 17))
    with pytest.raises(ValueError, match="pitch"):
        R._heads_args(R._T, dev(4, 64), dev(4, 64)[:, :32], dev(4, 32), 4, 2, 1, 32, None, None, None, None)
    with pytest.raises(ValueError, match="shapes"):
        R.Rope(torch.zeros(4, 64), torch.zeros(4, 32))


def test_plans_cover_the_cache_within_the_workspace():
    rng = random.Random(1)
    seen = set()
    for _ in range(20000):
        kv = rng.choice([1, 2, 3, 4, 8, 16, 64])
        heads = kv * rng.choice([1, 2, 4, 5, 7, 8, 16])
        hd = 32 * rng.randint(1, 8)
        tokens = int(2 ** rng.uniform(0, 10))
        length = min(int(2 ** rng.uniform(0, 17)) - 1, 131072 - tokens)
        p = D.mx_attention_plan(heads, kv, hd, length, tokens)
        rows, cache_rows = tokens * heads // kv, length + tokens
        assert p["hdp"] >= hd and p["hdp"] in (64, 128, 256)
        block, tile = D.shape(p["hdp"], p["form"])
        assert block > 0 and (p["row_blocks"] - 1) * block < rows <= p["row_blocks"] * block
        assert p["tiles"] * tile >= cache_rows > (p["tiles"] - 1) * tile
        assert 1 <= p["splits"] <= 64 and p["splits"] <= p["tiles"]
        need = R.attention_mxfp4_workspace_bytes(heads, kv, hd, length, tokens)
        assert p["bytes"] <= need <= 2**17 * 4 * (p["hdp"] + 2), (p, need)
        # A workspace for the longest call serves the shorter ones.
        less = D.mx_attention_plan(heads, kv, hd, rng.randint(0, length), rng.randint(1, tokens))
        assert less["bytes"] <= need
        seen.add((p["hdp"], p["form"], p["splits"] > 1))
    assert seen == {(64, f, s) for f in range(4) for s in (False, True)} | {(128, f, s) for f in range(4) for s in (False, True)} | {
        (256, f, s) for f in range(3) for s in (False, True)}   # every kernel, with and without a merge


def test_every_form_of_the_product_is_chosen():
    """No form is left that no product reaches, and none wastes three quarters of its rows."""
    rng = random.Random(2)
    seen = set()
    for _ in range(20000):
        M, N, K = int(2 ** rng.uniform(1, 13)), int(2 ** rng.uniform(4, 15)), 32 * int(2 ** rng.uniform(0, 10))
        form, (bm, _) = D.mx_form(M, N, K)
        assert bm == 16 or bm < 4 * M
        seen.add(form)
    assert seen == set(range(D.mx_forms()))


def test_the_shapes_of_the_gpu_tests_reach_every_kernel():
    from test_gpu_attention_mxfp4 import CASES

    plans = [D.mx_attention_plan(*c) for c in CASES + D.ATTENTION_SHAPES]
    assert {(p["hdp"], p["form"], p["splits"] > 1) for p in plans} == {
        (h, f, s) for h, forms in ((64, 4), (128, 4), (256, 3)) for f in range(forms) for s in (False, True)}
    assert {p["splits"] > 16 for p in plans} == {False, True}   # both merges
    assert {D.mx_form(*c)[0] for c in D.PRODUCT_SHAPES} == set(range(D.mx_forms()))
