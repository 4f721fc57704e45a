"""Which outputs of the attention over a 4-bit cache a row reaches, and scores near the end of f32's range."""
import pytest

torch = pytest.importorskip("torch")

import mx_reference as X  # noqa: E402
from test_gpu_attention_mxfp4 import make, pack, reference, tree_mask  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


# (heads, kv, hd, length, tokens): every form of 64, 128 and 256 dimensions, with and without a merge.
SHAPES = [
    (2, 2, 64, 64, 1), (2, 2, 64, 3000, 1), (14, 2, 64, 64, 74), (14, 2, 64, 1000, 74), (14, 2, 64, 64, 293), (8, 2, 64, 200, 707),
    (14, 2, 64, 65, 596), (14, 2, 64, 200, 677), (2, 2, 96, 64, 1), (2, 2, 96, 3000, 1), (14, 2, 96, 64, 154), (6, 3, 96, 1000, 285),
    (14, 2, 96, 65, 295), (6, 3, 96, 1000, 530), (14, 2, 96, 64, 586), (14, 2, 96, 200, 592), (2, 2, 160, 64, 1), (2, 2, 160, 1000, 1),
    (14, 2, 160, 64, 74), (2, 2, 160, 64, 523), (14, 2, 160, 65, 293), (14, 2, 160, 100, 322),
]


@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES)
def test_a_nan_row_reaches_its_own_heads_alone(R, heads, kv, hd, length, tokens):
    """A NaN block of one key/value head makes the query heads that share it NaN, of the tokens that see its row;
    the other heads' bits stay."""
    q, cache, _, _ = make(R, heads, kv, hd, length, tokens, 31)
    vis = tree_mask(tokens, 4)
    mask = pack(vis)
    clean = R.attention_mxfp4(q, cache, heads, length, tokens, hd**-0.5, mask).view(tokens, kv, -1).clone()
    assert not torch.isnan(clean).any()
    see = torch.from_numpy(vis[:, tokens - 1]).cuda()
    for which, byte in ((1, 255), (3, 253)):
        for g in range(kv):
            scales = cache.tensors[which].view(kv, -1, X.pitch(hd))
            old = scales[g, length + tokens - 1].clone()
            scales[g, length + tokens - 1, hd // 32 - 1] = byte
            got = R.attention_mxfp4(q, cache, heads, length, tokens, hd**-0.5, mask).view(tokens, kv, -1)
            want = clean.clone()
            want[see, g] = float("nan")
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (which, g)
            keep = ~torch.isnan(want)
            assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16)), (which, g)
            scales[g, length + tokens - 1] = old


@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES)
def test_scores_near_the_lowest_value_weigh_nothing(R, heads, kv, hd, length, tokens):
    """Whole tiles of rows with scores of -1.75 2^127, which times log2 e lie below f32's range, and rows of score 0
    behind them: the outputs are the mean of the latter's values, 1, exactly."""
    cache = R.MxCache(kv, hd, length + tokens)
    for t, byte in zip(cache.tensors, (0, 127, 0x22, 127)):   # keys 0, values 1
        t.fill_(byte)
    bad = 64
    codes, scales = (t.view(kv, length + tokens, -1) for t in cache.tensors[:2])
    codes[:, :bad, 0], scales[:, :bad, 0] = 0x0A, 127 + 27    # -1 times 2^27 on dimension 0
    cache.tensors[2].view(kv, length + tokens, -1)[:, :bad] = 0x77   # values of 6
    q = torch.zeros(tokens * heads, hd, dtype=torch.bfloat16, device="cuda")
    q[:, 0] = 1.75 * 2.0**100
    out = R.attention_mxfp4(q.view(-1), cache, heads, length, tokens, 1.0)
    assert (out == 1.0).all(), out[out != 1.0][:4]


@pytest.mark.parametrize("scale", [2.0**127, -2.0**127])
@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES[::3])
def test_the_largest_scale(R, heads, kv, hd, length, tokens, scale):
    """Products of 0 are scores of 0 under it: the mean of equal values."""
    cache = R.MxCache(kv, hd, length + tokens)
    for t, byte in zip(cache.tensors, (0x22, 127, 0x33, 127)):   # keys 1, values 1.5
        t.fill_(byte)
    q = torch.zeros(tokens * heads * hd, dtype=torch.bfloat16, device="cuda")
    assert (R.attention_mxfp4(q, cache, heads, length, tokens, scale) == 1.5).all()


@pytest.mark.parametrize("scale", [1.0, -3.0])
@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES)
def test_weights_that_vanish(R, heads, kv, hd, length, tokens, scale):
    """Scores hundreds apart, within the tolerance of test_gpu_attention_tree.py and what may vanish: the sums of waves and
    splits are each held against a maximum of their own, which their largest weight passes by up to 2^8, and meet
    under a factor that f32 ends at 2^-126. So a weight below 2^-118 of the token's largest may be lost, sum |v| of them at most."""
    for seed in range(3):
        q, cache, k, v = make(R, heads, kv, hd, length, tokens, seed)
        vis = tree_mask(tokens, seed)
        want, bound = reference(q, k, v, heads, kv, hd, length, tokens, vis, scale)
        got = R.attention_mxfp4(q, cache, heads, length, tokens, scale, pack(vis)).view(tokens, heads, hd).double()
        lost = 2.0**-118 * v.abs().view(-1, kv, hd).sum(0).repeat_interleave(heads // kv, 0)
        assert ((got - want).abs() <= bound + 2.0**-8 * want.abs() + lost).all()
