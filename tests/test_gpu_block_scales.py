"""Blocks whose largest magnitude over max_finite is 0 in f32 (below half of its
smallest subnormal, 2^-150): their scale is 1 and their codes are zeros, as in a
block of zeros. A scale of 0 would give 0 / 0 = NaN for the zeros among them."""
import pytest

torch = pytest.importorskip("torch")

FULL = {"e4m3": 240.0, "e5m2": 57344.0}
TINY = 2.0**-149   # f32's smallest subnormal


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def tiny_rows(rows, cols, top, seed):
    """Whole multiples of the smallest subnormal up to `top` of them in magnitude, zeros among them."""
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(-top, top + 1, (rows, cols), generator=g, dtype=torch.int32)
    n[:, ::3] = 0
    n[0, 1] = top
    return torch.where(n < 0, n.abs() | -(2**31), n).to(torch.int32).view(torch.float32).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 128), (5, 384), (130, 257), (200, 1024)])
def test_blocks_of_the_smallest_subnormals(R, rows, cols, br, fmt):
    x = tiny_rows(rows, cols, int(FULL[fmt]) // 2, rows)
    codes, scales = R.quantize_blocks(x, rows, cols, fmt, br)
    assert (scales == 1).all()
    assert (codes.view(rows, cols) & 0x7F == 0).all()
    # Behind that border the scale is a subnormal and codes are numbers.
    codes, scales = R.quantize_blocks(tiny_rows(rows, cols, int(FULL[fmt]) * 3, rows), rows, cols, fmt, br)
    assert (scales[0] > 0) and (codes & 0x7F < 0x78 if fmt == "e4m3" else codes & 0x7F < 0x7C).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("cols", [512, 1001])
def test_norms_that_leave_the_smallest_subnormals(R, cols, fmt):
    rows = 3
    x = torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x[:, ::3] = 0
    gamma = torch.full((cols,), 4 * TINY, device="cuda")
    _, codes, scales = R.residual_norm_fp8(x, None, gamma, rows, cols, 1e-5, fmt)
    assert (scales == 1).all() and (codes & 0x7F == 0).all()


@pytest.mark.gpu
def test_a_product_over_such_blocks_is_zero(R):
    M, N, K = 3, 32, 256
    x = tiny_rows(M, K, 100, 2)
    w = torch.randn(N, K, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    a, sa = R.quantize_blocks(x, M, K, "e4m3", 1)
    b, sb = R.quantize_blocks(w, N, K, "e4m3")
    assert (R.gemm_fp8_blocks(a, "e4m3", sa, b, "e4m3", sb, M, N, K) == 0).all()
