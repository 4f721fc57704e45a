"""Every kernel of the tree attention (test_tree_forms.py names them by shape)
against float64, as a tree and as a chain, and with rows that hold no numbers, by
test_gpu_attention_tree.py's tolerance."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention_tree import check, inputs, pack, tree_mask  # noqa: E402
from test_tree_forms import TREE_EDGE_SHAPES, TREE_FORM_SHAPES  # noqa: E402

pytestmark = pytest.mark.gpu
SHAPES = [(*k, *s) for k, s in TREE_FORM_SHAPES.items()]


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


@pytest.mark.parametrize("size,form,merge,heads,kv,hd,length,tokens", SHAPES)
def test_every_kernel_against_float64(R, size, form, merge, heads, kv, hd, length, tokens):
    empty = (0, tokens // 2, tokens - 1)   # see the context alone
    check(R, heads, kv, hd, length, tokens, tree_mask(tokens, length, empty), seed=length)
    check(R, heads, kv, hd, length, tokens, None, seed=tokens)


@pytest.mark.parametrize("size,form,heads,kv,hd,length,tokens", TREE_EDGE_SHAPES)
def test_the_eight_wave_form_at_its_borders(R, size, form, heads, kv, hd, length, tokens):
    out = check(R, heads, kv, hd, length, tokens, tree_mask(tokens, length, (0, 33, tokens - 1)), seed=length)
    if length == 0:
        assert (out.view(tokens, -1)[[0, 33, tokens - 1]] == 0).all()
    check(R, heads, kv, hd, length, tokens, None, seed=tokens)


@pytest.mark.parametrize("size,form,merge,heads,kv,hd,length,tokens", SHAPES)
def test_rows_not_seen_may_hold_anything_on_every_kernel(R, size, form, merge, heads, kv, hd, length, tokens):
    """NaN and infinities in drafted rows that only their own tokens see, as a tree; as a chain, in the last ones."""
    scale = hd**-0.5
    q, k, v = inputs(heads, kv, hd, length, tokens, 9)
    vis = tree_mask(tokens, 5)
    bad = {j: x for j, x in [(tokens - 1, float("nan")), (tokens // 2, float("inf")), (tokens // 3, -float("inf"))]}
    for j in bad:
        vis[:, j] = False
        vis[j, j] = True
    k2, v2 = k.view(-1, kv * hd).clone(), v.view(-1, kv * hd).clone()
    for j, x in bad.items():
        k2[length + j], v2[length + j] = x, x
    others = [i for i in range(tokens) if i not in bad]
    want, got = (R.attention_tree(q, *c, heads, kv, hd, length, tokens, scale, pack(vis)).view(tokens, -1)
                 for c in ((k, v), (k2, v2)))
    assert torch.equal(got[others].view(torch.int16), want[others].view(torch.int16))
    assert torch.isnan(got[tokens - 1]).all()
    last = -(-tokens * 3 // 4) - 1
    k3, v3 = k.view(-1, kv * hd).clone(), v.view(-1, kv * hd).clone()
    k3[length + last + 1:], v3[length + last + 1:] = float("nan"), float("inf")
    want, got = (R.attention_tree(q, *c, heads, kv, hd, length, tokens, scale).view(tokens, -1) for c in ((k, v), (k3, v3)))
    assert torch.equal(got[:last + 1].view(torch.int16), want[:last + 1].view(torch.int16))
    assert torch.isnan(got[last + 1:]).all()


@pytest.mark.parametrize("size,form,merge,heads,kv,hd,length,tokens", SHAPES)
def test_scores_of_minus_infinity_and_nan_on_every_kernel(R, size, form, merge, heads, kv, hd, length, tokens):
    q, k, v = inputs(heads, kv, hd, length, tokens, 2)
    q.view(tokens, heads, hd)[:, :, 0] = 1.0
    k = k.view(-1, kv, hd)
    k[:length + tokens, :, 0] = 0.0
    base = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).view(tokens, -1)
    k[[5, length // 2, length - 1], :, 0] = -float("inf")   # context rows that no token can weigh
    got = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).view(tokens, -1)
    assert torch.isfinite(got).all() and not torch.equal(got, base)
    k[:length + tokens, :, 0] = -float("inf")
    assert torch.isnan(R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1)).all()
    k[:length + tokens, :, 0] = 0.0
    at = tokens // 2
    k[length + at, :, 3] = float("nan")                      # seen by tokens `at` on
    got = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).view(tokens, -1)
    assert torch.equal(got[:at].view(torch.int16), base[:at].view(torch.int16)) and torch.isnan(got[at:]).all()


@pytest.mark.parametrize("size,form,merge", [(64, 3, 0), (96, 3, 1), (128, 3, 4), (128, 1, 4), (256, 2, 1)])
def test_the_same_call_gives_the_same_bits(R, size, form, merge):
    """Again and again, on two streams at once with workspaces of their own, and with a workspace full of junk."""
    heads, kv, hd, length, tokens = TREE_FORM_SHAPES[size, form, merge]
    q, k, v = inputs(heads, kv, hd, length, tokens, 7)
    mask = pack(tree_mask(tokens, 2))
    n = max(16, R.attention_tree_workspace_bytes(heads, kv, hd, length, tokens))
    ws = [torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    want = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.08, mask)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(4)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(4):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.08, mask, ws[s], outs[s][i])
    torch.cuda.synchronize()
    for got in outs[0] + outs[1]:
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
