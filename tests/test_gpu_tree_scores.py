"""Scores near the end of f32's range in the tree attention, on every kernel."""
import pytest

torch = pytest.importorskip("torch")

from test_tree_forms import TREE_FORM_SHAPES  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


@pytest.mark.parametrize("heads,kv,hd,length,tokens", TREE_FORM_SHAPES.values())
def test_scores_near_the_lowest_value_weigh_nothing(R, heads, kv, hd, length, tokens):
    """Whole tiles of rows with scores of -1.75 2^127, which times log2 e lie below f32's range, and rows of score 0
    behind them: the outputs are the mean of the latter's values, 1, exactly."""
    k = torch.zeros(length + tokens, kv, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.ones_like(k)
    k[:64, :, 0], v[:64] = -2.0**27, 6
    q = torch.zeros(tokens * heads, hd, dtype=torch.bfloat16, device="cuda")
    q[:, 0] = 1.75 * 2.0**100
    out = R.attention_tree(q.view(-1), k.view(-1), v.view(-1), heads, kv, hd, length, tokens, 1.0)
    assert (out == 1.0).all(), out[out != 1.0][:4]
