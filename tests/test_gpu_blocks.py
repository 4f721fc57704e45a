"""Block scales: the quantizer (one scale per 128 x 128 block or 1 x 128 group)
and the product that reads its codes.

The quantizer is held bit-exact to the oracle: a block is a row of the oracle's
per-channel scheme (zeros pad a block at an edge and change neither its absmax
nor its codes).

The product is held to float64 over the decoded codes. Per output, with T =
sum_kb sa sb sum_k |a b| and KB = ceil(K / 128) blocks:

    |got - want| <= 2^-8 |want| + (2^-12 + (KB + 24) 2^-23) T

2^-8: the output's rounding to bf16, half a step. 2^-12: a matrix instruction's
own sum of fp8 products (below 2^-13.2 of the sum of magnitudes on this
hardware, as for the per-channel product). Per block one rounding of sa sb, one
of the multiply-add and, over the waves or splits that share a row, fewer than
16 sums: each at most 2^-24 of a partial sum that T bounds.
"""
import numpy as np
import pytest

import oracle as O
from helpers import bf16_bits

torch = pytest.importorskip("torch")

from test_block_forms import FORM_SHAPES  # noqa: E402

FMTS = ["e4m3", "e5m2"]
TORCH_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def blocks_of(x, br):
    """[rows, cols] padded with zeros to whole br x 128 blocks, a block a row."""
    rows, cols = x.shape
    p = np.zeros((-(-rows // br) * br, -(-cols // 128) * 128), x.dtype)
    p[:rows, :cols] = x
    rb, cb = p.shape[0] // br, p.shape[1] // 128
    return np.ascontiguousarray(p.reshape(rb, br, cb, 128).transpose(0, 2, 1, 3)).reshape(rb * cb, br * 128)


def unblock(codes, rows, cols, br):
    rb, cb = -(-rows // br), -(-cols // 128)
    return codes.reshape(rb, cb, br, 128).transpose(0, 2, 1, 3).reshape(rb * br, cb * 128)[:rows, :cols]


def values(rng, rows, cols, special):
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 7, (rows, 1)))).astype(np.float32)
    if special:
        flat = x.reshape(-1)
        at = rng.permutation(flat.size)
        for i, v in enumerate([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-40, -3e-45, 3e38, 240.0, 248.0]):
            flat[at[i::max(11, flat.size // 3)]] = v
        x[rows // 2] = 0.0                       # a row of zeros
        x[0, :min(cols, 128)] *= np.float32(1e-38)   # a subnormal scale
    return x


def check_quantize(R, x, dtype, fmt, br, backoff=1.0, ld=None, shift=0):
    rows, cols = x.shape
    ld = cols if ld is None else ld
    src = bf16_bits(x).reshape(rows, cols) if dtype == "bf16" else x
    buf = np.zeros(rows * ld + shift, src.dtype)
    buf[shift:].reshape(rows, ld)[:, :cols] = src
    dev = torch.from_numpy(buf.view(np.int16) if dtype == "bf16" else buf).cuda()[shift:]
    codes, scales = R.quantize_blocks(dev, rows, cols, fmt, br, backoff, ld)
    b = blocks_of(src, br)
    if dtype == "bf16":
        want = O.quantize_with(b.ravel(), b.shape[0], b.shape[1], fmt, "pcs", backoff)
        wcodes, wscales = want.codes, want.scales
    else:
        wcodes, wscales = quantize_f32(b, fmt, backoff)
    assert np.array_equal(scales.cpu().numpy().view(np.uint32), np.asarray(wscales).view(np.uint32))
    want = unblock(np.asarray(wcodes).reshape(b.shape), rows, cols, br)
    got = codes.cpu().numpy().reshape(rows, cols)
    assert np.array_equal(got, want), np.argwhere(got != want)[:4]


def quantize_f32(b, fmt, backoff):
    """The oracle's encoder over IEEE f32 quotients, block by block."""
    full = np.float32(np.float32(240.0 if fmt == "e4m3" else 57344.0) * np.float32(backoff))
    a = np.abs(b)
    m = np.where(np.isnan(a), np.float32(0), a).max(axis=1)
    with np.errstate(all="ignore"):
        s = np.where(m > 0, m / full, np.float32(1)).astype(np.float32)
        q = (b / s[:, None]).astype(np.float32)
    # x86: a NaN dividend keeps its sign, an invalid quotient is the negative default NaN.
    bits = q.view(np.uint32).copy()
    bad = np.isnan(q) & ~np.isnan(b)
    bits[bad] = 0xFFC00000
    keep = np.isnan(b)
    bits[keep] = b.view(np.uint32)[keep]
    return O.encode_array(bits.view(np.float32).ravel(), fmt), s


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 200), (128, 128), (129, 257), (7, 1000), (300, 576),
                                       (64, 4001), (130, 2048)])
def test_quantize_blocks_is_the_oracle(R, rows, cols, dtype, br, fmt):
    rng = np.random.default_rng(rows * 7919 + cols)
    check_quantize(R, values(rng, rows, cols, rows * cols > 500), dtype, fmt, br)


@pytest.mark.gpu
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_blocks_pitch_alignment_backoff(R, dtype, br):
    rng = np.random.default_rng(5)
    x = values(rng, 200, 384, False)
    check_quantize(R, x, dtype, "e4m3", br, ld=512)           # a window of wider rows
    check_quantize(R, x, dtype, "e4m3", br, ld=385)           # rows off 16 bytes
    check_quantize(R, x, dtype, "e5m2", br, shift=1)          # the tensor off 16 bytes
    check_quantize(R, x, dtype, "e4m3", br, backoff=0.5)
    check_quantize(R, x, dtype, "e4m3", br, backoff=3.0)      # quotients past the range saturate


def operands(M, N, K, afmt, bfmt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kb = -(-K // 128)

    def codes(rows, fmt):
        x = torch.randn(rows, K, generator=g, device="cuda") * 40
        return x.clamp(-240, 240).to(TORCH_FP8[fmt])

    def scales(*shape):
        return torch.exp2(torch.rand(*shape, generator=g, device="cuda") * 8 - 4)

    return codes(M, afmt), scales(M, kb), codes(N, bfmt), scales(-(-N // 128), kb)


def exact_product(a, sa, b, sb):
    """(want, T) in float64."""
    M, K = a.shape
    N = b.shape[0]
    ea = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    eb = b.double() * sb.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return ea @ eb.T, ea.abs() @ eb.abs().T


def check_product(R, M, N, K, afmt="e4m3", bfmt="e4m3", seed=0):
    a, sa, b, sb = operands(M, N, K, afmt, bfmt, seed)
    out = torch.full((M * N + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    R.gemm_fp8_blocks(a.view(torch.uint8), afmt, sa, b.view(torch.uint8), bfmt, sb, M, N, K, out)
    assert (out[M * N:] == 7.0).all(), "written past the output"
    want, t = exact_product(a, sa, b, sb)
    kb = -(-K // 128)
    bound = 2.0**-8 * want.abs() + (2.0**-12 + (kb + 24) * 2.0**-23) * t
    err = (out[:M * N].view(M, N).double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (err / bound).max().item())


SHAPES = [(1, 1, 16), (1, 16, 128), (1, 129, 144), (1, 4096, 4096), (1, 577, 18944), (1, 300, 37888), (2, 17, 144),
          (3, 1000, 2048), (4, 576, 1536), (4, 130, 4112), (5, 100, 576), (8, 1024, 5120), (15, 33, 256),
          (16, 130, 4096), (17, 129, 272), (24, 3584, 2048), (32, 64, 128), (33, 257, 1040), (48, 520, 896),
          (64, 512, 3584), (65, 300, 2048), (100, 128, 16), (128, 1024, 512), (130, 1000, 1040), (255, 129, 400),
          (257, 520, 640), (300, 4096, 256), (512, 777, 576), (1000, 2056, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_fp8_blocks_against_float64(R, M, N, K):
    check_product(R, M, N, K, seed=M + N + K)


@pytest.mark.gpu
@pytest.mark.parametrize("form,M,N,K", FORM_SHAPES)
def test_gemm_fp8_blocks_every_form(R, form, M, N, K):
    """Every form, at ragged sizes, block counts of 1 to 9 (scales go four blocks at a time) and a short last block."""
    check_product(R, M, N, K, seed=M + N + K)
    check_product(R, M, N, K, "e5m2", "e4m3", seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("afmt,bfmt", [("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("M,N,K", [(1, 1000, 4096), (3, 65, 528), (24, 257, 1040), (64, 300, 512), (200, 520, 640),
                                   (512, 1024, 1040)])
def test_gemm_fp8_blocks_formats(R, M, N, K, afmt, bfmt):
    check_product(R, M, N, K, afmt, bfmt, seed=11)


@pytest.mark.gpu
def test_gemm_fp8_blocks_reads_every_block_scale(R):
    """One code of 1 in one k: the output is that block's two scales and nothing else's."""
    M, N, K = 70, 300, 640
    for m, n, k in [(0, 0, 0), (69, 299, 639), (33, 127, 128), (64, 128, 511), (1, 256, 255)]:
        a = torch.zeros(M, K, dtype=torch.uint8, device="cuda")
        b = torch.zeros(N, K, dtype=torch.uint8, device="cuda")
        a[m, k] = 0x38   # 1.0
        b[n, k] = 0x38
        sa = torch.arange(1, M * 5 + 1, dtype=torch.float32, device="cuda").view(M, 5) / 64
        sb = torch.arange(1, 3 * 5 + 1, dtype=torch.float32, device="cuda").view(3, 5)
        out = R.gemm_fp8_blocks(a, "e4m3", sa, b, "e4m3", sb, M, N, K).view(M, N)
        want = torch.zeros(M, N, device="cuda")
        want[m, n] = sa[m, k // 128] * sb[n // 128, k // 128]
        assert torch.equal(out, want.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 500, 2064), (24, 500, 2064), (150, 520, 1040), (520, 1032, 528)])
def test_gemm_fp8_blocks_ends_where_its_operands_end(R, M, N, K):
    """Codes that stand for no number right behind either operand, and behind every short row's last block,
    are not read as part of it; the call gives the same bits again."""
    a, sa, b, sb = operands(M, N, K, "e4m3", "e4m3", 3)

    def fenced(t):
        buf = torch.full((t.numel() + 4096,), 0x7F, dtype=torch.uint8, device="cuda")
        buf[:t.numel()] = t.reshape(-1).view(torch.uint8)
        return buf

    one = R.gemm_fp8_blocks(fenced(a), "e4m3", sa, fenced(b), "e4m3", sb, M, N, K)
    want, t = exact_product(a, sa, b, sb)
    assert ((one.view(M, N).double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-11 * t).all()
    two = R.gemm_fp8_blocks(a.view(torch.uint8), "e4m3", sa, b.view(torch.uint8), "e4m3", sb, M, N, K)
    assert torch.equal(one.view(torch.int16), two.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 24, 200, 600])
def test_quantize_and_product_together_in_a_graph(R, M):
    """Activation rows quantized and multiplied on a side stream, then captured and replayed on new values."""
    N, K = 1024, 1536
    rng = np.random.default_rng(M)
    w = torch.from_numpy((rng.standard_normal((N, K)) * 0.02).astype(np.float32)).cuda()
    wc, ws = R.quantize_blocks(w, N, K, "e4m3", 128)
    x = torch.empty(M * K, dtype=torch.bfloat16, device="cuda")
    codes = torch.empty(M * K, dtype=torch.uint8, device="cuda")
    scales = torch.empty(M * (K // 128), dtype=torch.float32, device="cuda")
    out = torch.empty(M * N, dtype=torch.bfloat16, device="cuda")

    def step():
        R.quantize_blocks_into(x, M, K, "e4m3", 1, 1.0, codes, scales)
        R.gemm_fp8_blocks(codes, "e4m3", scales, wc, "e4m3", ws, M, N, K, out)

    def fill(seed):
        x.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal(M * K).astype(np.float32)))

    st = torch.cuda.Stream()
    fill(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step()
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    for seed in range(1, 5):
        fill(seed)
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(replayed.view(torch.int16), out.view(torch.int16))
        want = x.view(M, K).double() @ w.double().T
        rel = (out.view(M, N).double() - want).norm() / want.norm()
        # Two e4m3 roundings of at most 2^-4 of a value each, independent over K = 1536 products.
        assert rel < 2.0**-4, rel


def test_block_refusals():
    import ctypes

    import reng_hip as R

    L = R.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)

    def refused(rc, *words):
        msg = L.reng_hip_last_error().decode()
        assert rc == R.EINVAL, msg
        for w in words:
            assert w in msg, msg

    def q(w=p, dtype=R.BF16, rows=4, cols=256, ld=256, fmt=R.E4M3, br=128, backoff=1.0, codes=p, scales=p):
        return L.reng_hip_quantize_blocks(w, dtype, rows, cols, ld, fmt, br, backoff, codes, scales, None)

    refused(q(dtype=5), "element type")
    refused(q(fmt=2), "format")
    refused(q(rows=0), "empty shape 0 x 256")
    refused(q(cols=0), "empty shape 4 x 0")
    refused(q(ld=255), "row pitch 255")
    refused(q(br=64), "blocks of 64 rows")
    refused(q(br=0), "blocks of 0 rows")
    for bad in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        refused(q(backoff=bad), "not positive and finite")
    refused(q(w=None), "null")
    refused(q(codes=None), "null")
    refused(q(scales=None), "null")
    refused(q(w=odd), "aligned")
    refused(q(scales=odd), "aligned")
    refused(q(rows=1 << 31), "too large")

    def g(a=p, fa=0, sa=p, b=p, fb=0, sb=p, M=4, N=8, K=128, out=p):
        return L.reng_hip_gemm_fp8_blocks(a, fa, sa, b, fb, sb, M, N, K, out, None)

    refused(g(fa=2), "format")
    refused(g(fb=-1), "format")
    refused(g(M=0), "empty product")
    refused(g(N=0), "empty product")
    refused(g(K=0), "empty product")
    refused(g(K=136), "multiple of 16")
    refused(g(M=1 << 31), "too large")
    for name in ("a", "sa", "b", "sb", "out"):
        refused(g(**{name: None}), "null")
        refused(g(**{name: odd}), "aligned")
    refused(g(a=ctypes.c_void_p(4104)), "16-byte aligned")


def test_the_binding_refuses_wrong_block_operands():
    from test_abi import _FakeDev as Fake

    import reng_hip as R

    bf, f32 = torch.bfloat16, torch.float32
    rows, cols = 8, 256
    w, codes, scales = Fake(2 * rows * cols, bf), Fake(rows * cols), Fake(4 * 2, f32)
    with pytest.raises(ValueError, match="weight length"):
        R.quantize_blocks_into(Fake(2 * rows * cols - 2, bf), rows, cols, "e4m3", 128, 1.0, codes, scales)
    with pytest.raises(ValueError, match="codes length"):
        R.quantize_blocks_into(w, rows, cols, "e4m3", 128, 1.0, Fake(rows * cols - 1), scales)
    with pytest.raises(ValueError, match="scales length"):
        R.quantize_blocks_into(w, rows, cols, "e4m3", 1, 1.0, codes, scales)
    with pytest.raises(ValueError, match="scales must be f32"):
        R.quantize_blocks_into(w, rows, cols, "e4m3", 128, 1.0, codes, Fake(64, bf))
    with pytest.raises(ValueError, match="blocks of 7 rows"):
        R.quantize_blocks_into(w, rows, cols, "e4m3", 7, 1.0, codes, scales)
    M, N, K = 4, 32, 256
    a, sa, b, sb, out = Fake(M * K), Fake(4 * M * 2, f32), Fake(N * K), Fake(4 * 2, f32), Fake(2 * M * N, bf)
    for i, short, what in [(0, Fake(M * K - 1), "a length"), (2, Fake(4 * M * 2 - 4, f32), "scale_a length"),
                           (3, Fake(N * K - 1), "b length"), (5, Fake(4, f32), "scale_b length"),
                           (9, Fake(2 * M * N - 2, bf), "out length"), (0, Fake(2 * M * K, bf), "one code per byte")]:
        args = [a, "e4m3", sa, b, "e4m3", sb, M, N, K, out]
        args[i] = short
        with pytest.raises(ValueError, match=what):
            R.gemm_fp8_blocks(*args)
