"""Kernels of the 4-bit operators that few calls choose: the product of one row over split k.

Tolerances are those of test_gpu_mxfp4.py.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_plans as D  # noqa: E402
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
