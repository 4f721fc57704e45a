"""MXFP4 matrices: quantizer, values and product, against 64 bits.

Codes, scales and values are exact. The product, per output, with T = sum_k |a b| and
KB = ceil(K / 128):

    |got - want| <= 2^-8 |want| + (2^-12 + (KB + 24) 2^-23) T

2^-8: the output's rounding to bf16. 2^-12: a matrix instruction's own sum of 128
products, as for the fp8 product. Per instruction one rounding of the running sum and,
over the waves that share a row, fewer than 16 sums, each at most 2^-24 of a partial sum that T bounds.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_plans as D  # noqa: E402
import mx_reference as X  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def check_quantize(R, w, rows, cols, ld=None):
    x = w.view(-1)
    ld = cols if ld is None else ld
    x = torch.as_strided(x, (rows, cols), (ld, 1))
    n, ns = rows * -(-cols // 2), rows * X.pitch(cols)
    codes, scales = (torch.full((m + 64,), 0xA5, dtype=torch.uint8, device="cuda") for m in (n, ns))
    R.quantize_mxfp4_into(w, rows, cols, codes, scales, ld)
    want = X.pack(*X.quantize(x.double()))
    assert torch.equal(scales[:ns].view(rows, -1), want[1])
    assert torch.equal(codes[:n].view(rows, -1), want[0])
    assert (codes[n:] == 0xA5).all() and (scales[ns:] == 0xA5).all(), "written past the end"
    return codes[:n], scales[:ns]


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (7, 64), (2, 127), (4, 128), (4, 129), (17, 136), (9, 4104), (300, 576),
          (24, 18944), (33, 5118), (1000, 40), (2, 131072)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(R, rows, cols, dtype):
    w = randn(rows + cols, rows, cols)
    w[:, ::7] *= torch.exp2(4 * randn(1, rows, -(-cols // 7)))
    check_quantize(R, w.to(dtype), rows, cols)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ld,off", [(200, 0), (168, 8), (160, 1), (163, 0)])
def test_quantize_windows(R, ld, off, dtype):
    w = randn(ld, 21 * ld + off).to(dtype)[off:]
    check_quantize(R, w[:20 * ld + 160].contiguous() if off == 0 else w, 21, 160, ld)


def test_quantize_every_bf16_value(R):
    """Each finite bf16 value under the largest magnitude 1, 1.75 and its own power's neighbours, NaN and infinities too."""
    bits = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    w = torch.zeros(65536, 32, dtype=torch.bfloat16, device="cuda")
    w[:, 3] = bits
    check_quantize(R, w, 65536, 32)
    for top in (1.0, 1.7421875, 1.75, -6.0, 2.0**-126, 3e38):
        w[:, 9] = top
        check_quantize(R, w, 65536, 32)


def test_quantize_f32_edges(R):
    tiny, big = 2.0**-149, 3.4028235e38
    x = torch.zeros(16, 96, device="cuda")
    x[0, :4] = torch.tensor([tiny, -tiny, 0.0, -0.0])
    x[1, 0], x[1, 1] = 2.0**-126, 2.0**-128
    x[2, 0], x[2, 33], x[2, 70] = float("inf"), float("nan"), -float("inf")
    x[3, :3] = torch.tensor([big, -big, 1.0])
    x[4] = -0.0
    x[5, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])        # ties
    x[6, :8] = -torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    one = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    x[7, 0], x[7, 1:8] = 6.0, torch.nextafter(one, one * 0)
    x[8, 0], x[8, 1:8] = 6.0, torch.nextafter(one, one * 9)
    x[9, 0] = torch.nextafter(torch.tensor(7.0), torch.tensor(0.0))
    x[10, 0] = 7.0
    x[11, :2] = torch.tensor([1.75 * 2.0**-125, 2.0**-127])
    x[12, :2] = torch.tensor([2.0**-125, 3 * 2.0**-129])
    check_quantize(R, x, 16, 96)


@pytest.mark.parametrize("f32", [False, True])
def test_values_of_every_code_and_scale(R, f32):
    code = torch.arange(16, device="cuda", dtype=torch.uint8).repeat(2)
    codes = (code[::2] | (code[1::2] << 4)).repeat(256, 1).contiguous()
    scales = torch.full((256, 4), 127, dtype=torch.uint8, device="cuda")
    scales[:, 0] = torch.arange(256, device="cuda")
    out = torch.empty(256 * 32, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    R.dequantize_mxfp4(codes, scales, 256, 32, out)
    want = X.values(code.repeat(256, 1), scales[:, :1])
    want = torch.where(want.abs() >= 2.0**128, want * float("inf"), want)
    assert torch.equal(torch.nan_to_num(out.view(256, 32).double(), 1.5), torch.nan_to_num(want, 1.5))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES[:-1])
def test_dequantize(R, rows, cols, f32):
    code, byte = X.quantize(randn(cols, rows, cols).double())
    codes, scales = X.pack(code, byte)
    out = torch.full((rows * cols + 8,), 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    R.dequantize_mxfp4(codes, scales, rows, cols, out)
    assert torch.equal(out[:rows * cols].view(rows, cols).double(), X.values(code, byte))
    assert (out[rows * cols:] == 7.0).all(), "written past the end"


def operand(rows, cols, seed):
    """Codes with scales of their own range, some blocks all zeros."""
    x = randn(seed, rows, cols) * torch.exp2(2 * randn(seed + 1, rows, 1))
    x[:, ::37] *= 16
    x[:, :32] *= (torch.arange(rows, device="cuda") % 5 != 0)[:, None]
    return X.quantize(x.double())


def check_product(R, M, N, K, seed=0, off=0):
    a, b = operand(M, K, seed), operand(N, K, seed + 7)
    pa, pb = X.pack(*a), X.pack(*b)
    out = torch.full((M * N + 64 + off,), 7.0, dtype=torch.bfloat16, device="cuda")[off:]
    R.gemm_mxfp4(*pa, *pb, M, N, K, out)
    assert (out[M * N:] == 7.0).all(), "written past the output"
    va, vb = X.values(*a), X.values(*b)
    want, t = va @ vb.T.contiguous(), va.abs() @ vb.abs().T.contiguous()
    bound = 2.0**-8 * want.abs() + (2.0**-12 + (-(-K // 128) + 24) * 2.0**-23) * t
    err = (out[:M * N].view(M, N).double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (err / bound).max().item())


@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 24, 32, 33, 64, 65, 100, 128, 200, 256, 257, 333])
@pytest.mark.parametrize("N,K", [(16, 32), (129, 96), (576, 576), (250, 1024), (1536, 2080)])
def test_product(R, M, N, K):
    check_product(R, M, N, K, M)


@pytest.mark.parametrize("M,N,K", [(1, 14336, 4096), (1, 4096, 14336), (1, 1, 32), (3, 7, 18944), (24, 3584, 18944), (130, 3584, 18944),
                                   (1024, 1030, 5120), (512, 4096, 4096), (2048, 2047, 160), (700, 5120, 5120)])
def test_larger_products(R, M, N, K):
    check_product(R, M, N, K, K)


@pytest.mark.parametrize("M,N,K", D.PRODUCT_SHAPES)
def test_every_form(R, M, N, K):
    check_product(R, M, N, K, K + 1)


def test_product_to_an_odd_address(R):
    check_product(R, 33, 640, 256, off=1)
    check_product(R, 300, 640, 256, off=3)


@pytest.mark.parametrize("M,N,K", [(2, 100, 4096), (70, 333, 1056), (300, 600, 288), (138, 11009, 2112),
                                   (1451, 8248, 1312)])
def test_a_nan_block_is_its_rows_alone(R, M, N, K):
    """A NaN scale reaches its row's outputs and no others, also in the last block of a row that ends inside a tile."""
    a, b = operand(M, K, 1), operand(N, K, 2)
    a[1][1, -1], b[1][7, 0], b[1][N - 1, -1] = 255, 255, 255
    out = R.gemm_mxfp4(*X.pack(*a), *X.pack(*b), M, N, K).view(M, N)
    want = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    want[1], want[:, 7], want[:, N - 1] = True, True, True
    assert torch.equal(torch.isnan(out), want)


@pytest.mark.parametrize("N,K", [(101, 4096), (33, 1056), (7, 18944)])
def test_nan_blocks_of_one_row(R, N, K):
    """With one row of activations, NaN weights are their outputs alone, a NaN activation is all of them."""
    a, b = operand(1, K, 3), operand(N, K, 4)
    b[1][5, 0], b[1][N - 1, -1] = 255, 255
    out = R.gemm_mxfp4(*X.pack(*a), *X.pack(*b), 1, N, K)
    want = torch.zeros(N, dtype=torch.bool, device="cuda")
    want[5] = want[N - 1] = True
    assert torch.equal(torch.isnan(out), want)
    a[1][0, K // 64] = 255
    assert torch.isnan(R.gemm_mxfp4(*X.pack(*a), *X.pack(*b), 1, N, K)).all()


def test_scales_of_both_ends(R):
    """Scales whose product is far from 1: 2^-126 by 2^100, and products that leave f32."""
    M, N, K = 4, 32, 256
    code = torch.full((N, K), 2, dtype=torch.uint8, device="cuda")
    def run(ea, eb):
        a = torch.full((M, K // 32), ea + 127, dtype=torch.uint8, device="cuda")
        b = torch.full((N, K // 32), eb + 127, dtype=torch.uint8, device="cuda")
        return R.gemm_mxfp4(*X.pack(code[:M], a), *X.pack(code, b), M, N, K).double()
    assert (run(-126, 100) == 256 * 2.0**-26).all()
    assert (run(60, 50) == 256 * 2.0**110).all()
    assert torch.isinf(run(100, 100)).all()
