"""Block-scaled, norm and tree operators where an operand passes 2^32 bytes or elements.

What lies behind that border decides the values compared: a wrapped offset reads
other rows (the patterns' period of 1001 rows divides no power of two) or writes
elsewhere.
"""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention_tree import inputs, pack, reference, tree_mask  # noqa: E402
from test_gpu_blocks import exact_product, operands  # noqa: E402

pytestmark = pytest.mark.gpu
ROWS, COLS, PERIOD = 264064, 16384, 1001   # 2^32 + 30 * 2^20 elements, whole 128-row blocks


@pytest.fixture()
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GiB of device memory")
    reng_hip.lib()
    yield reng_hip
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def repeated(base, rows):
    """base's rows again and again, [rows, cols]."""
    return base[torch.arange(rows, device="cuda") % base.shape[0]]


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("br", [1, 128])
def test_quantize(R, br):
    w = repeated(randn(0, PERIOD, COLS).bfloat16(), ROWS)
    codes, scales = R.quantize_blocks(w, ROWS, COLS, "e4m3", br)
    last = w[-1024:].contiguous()
    wcodes, wscales = R.quantize_blocks(last, 1024, COLS, "e4m3", br)
    assert torch.equal(codes[-1024 * COLS:], wcodes)
    assert torch.equal(scales[-wscales.numel():], wscales)


@pytest.mark.parametrize("fp8", [False, True])
def test_residual_norm(R, fp8):
    x = repeated(randn(1, PERIOD, COLS), ROWS)
    d = repeated(randn(2, PERIOD, COLS).bfloat16(), ROWS)
    gamma = 1 + 0.2 * randn(3, COLS)
    # 1024 rows take the same kernel as all of them: the same bits.
    lx, ld = x[-1024:].clone(), d[-1024:].clone()

    def call(x, d, rows):
        if fp8:
            return R.residual_norm_fp8(x, d, gamma, rows, COLS, 1e-5, "e4m3", gamma, d, 0.3, h=x)
        return R.residual_norm_bf16(x, d, gamma, rows, COLS, 1e-5, gamma, d, 0.3, h=x)

    got, want = call(x, d, ROWS), call(lx, ld, 1024)
    for g, w in zip(got, want):
        assert torch.equal(g.reshape(-1)[-w.numel():], w.reshape(-1))


def product_bound(want, t, kb):
    return 2.0**-8 * want.abs() + (2.0**-12 + (kb + 24) * 2.0**-23) * t   # test_gpu_blocks.py


@pytest.mark.parametrize("M", [1, 24, 80])
def test_product_of_long_weights(R, M):
    a, sa, base, _ = operands(M, PERIOD, COLS, "e4m3", "e4m3", M)
    b = repeated(base.view(torch.uint8), ROWS)
    sb = torch.exp2(randn(4, ROWS // 128, COLS // 128))
    out = R.gemm_fp8_blocks(a.view(torch.uint8), "e4m3", sa, b, "e4m3", sb, M, ROWS, COLS).view(M, ROWS)
    want, t = exact_product(a, sa, b[-256:].view(base.dtype), sb[-2:])
    assert ((out[:, -256:].double() - want).abs() <= product_bound(want, t, COLS // 128)).all()


def test_product_of_many_outputs(R):
    M, N, K = 66048, 65536, 144
    a, sa, b, sb = operands(M, N, K, "e4m3", "e4m3", 5)
    out = R.gemm_fp8_blocks(a.view(torch.uint8), "e4m3", sa, b.view(torch.uint8), "e4m3", sb, M, N, K).view(M, N)
    want, t = exact_product(a[-256:], sa[-256:], b, sb)
    assert ((out[-256:].double() - want).abs() <= product_bound(want, t, 2)).all()


def test_long_caches(R):
    heads, hd, tokens = 66, 256, 3
    length = 131072 - tokens
    q, k, v = inputs(heads, heads, hd, length, tokens, 6)
    at = 130000   # its rows' keys are a token's queries: nearly all of the weight
    assert at * heads * hd * 2 > 2**32
    k.view(-1, heads * hd)[at:at + tokens] = q.view(tokens, heads * hd)
    vis = tree_mask(tokens, 1)
    want, bound = reference(q, k, v, heads, heads, hd, length, tokens, vis, hd**-0.5)
    got = R.attention_tree(q, k, v, heads, heads, hd, length, tokens, hd**-0.5, pack(vis))
    # bound holds 64 roundings of the sums and 2^-8 p |v|. Up to 2048 rows of a split are summed
    # here, in chains of fewer than 512: at most 512 2^-24 p |v| <= 2^-7 bound more.
    limit = bound * (1 + 2.0**-7) + 2.0**-8 * want.abs()
    assert ((got.view(tokens, heads, hd).double() - want).abs() <= limit).all()
    # The planted rows decide: without them the outputs are means of thousands of values of
    # variance 1, and a distance of 1 to a planted row of such values is usual.
    planted = v.view(-1, heads, hd)[at:at + tokens].double()
    assert (want - planted).abs().median() < 0.25
