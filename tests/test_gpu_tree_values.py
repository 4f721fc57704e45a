"""Infinite and NaN values in rows that tokens of the tree attention see.

The definition over the rows seen, in float64: sum_j p_j v_j, where a row of any
finite score has a weight above 0, however small, and a row whose score is -inf
(its key holds an infinity) has weight 0. So an infinite value gives an infinity
of its sign; one under a weight of 0, two of different signs, or a NaN give NaN.
That must hold wherever the row lies (a tile of context rows alone, the tile in
which the context ends, the drafted rows), on every form, and where the row's
weight underflows f32 against its tile, against a later tile, or against another
split. The dimensions that no such value reaches keep test_gpu_attention_tree's
tolerance.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention_tree import inputs, pack, tree_mask  # noqa: E402

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def definition(q, k, v, heads, kv, hd, length, tokens, vis, scale):
    """(want, bound of its finite values) [tokens, heads, hd] in float64."""
    rows = length + tokens
    q = q.view(tokens, heads, hd).double()
    k, v = k.view(-1, kv, hd)[:rows].double(), v.view(-1, kv, hd)[:rows].double()
    see = torch.ones(tokens, rows, dtype=torch.bool, device=q.device)
    see[:, length:] = torch.from_numpy(vis).to(q.device)
    want, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(heads):
        g = h // (heads // kv)
        kg, vg = k[:, g], v[:, g]
        weighs = see & ~torch.isinf(kg).any(1)
        kf, vf = torch.where(torch.isinf(kg), 0.0, kg), torch.where(torch.isfinite(vg), vg, 0.0)
        s = (q[:, h] @ kf.T * scale).masked_fill(~weighs, -INF)
        mag = (q[:, h].abs() @ kf.abs().T * abs(scale)).masked_fill(~weighs, 0)
        p = torch.softmax(s, 1)
        o = p @ vf
        plus = weighs.double() @ (vg == INF).double() > 0
        minus = weighs.double() @ (vg == -INF).double() > 0
        nan = (see.double() @ torch.isnan(vg).double() > 0) | ((see & ~weighs).double() @ torch.isinf(vg).double() > 0)
        o = torch.where(plus, INF, torch.where(minus, -INF, o))
        want[:, h] = torch.where(nan | (plus & minus), NAN, o)
        delta = (hd * 2.0**-24 * mag + 2.0**-21 * (1 + mag)).amax(1, keepdim=True)
        bound[:, h] = (2.0**-8 + 2 * delta + 64 * 2.0**-24) * (p @ vf.abs()) + 2.0**-8 * o.abs()
    return want, bound


def check(R, q, k, v, heads, kv, hd, length, tokens, vis, masked, scale):
    want, bound = definition(q, k, v, heads, kv, hd, length, tokens, vis, scale)
    got = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, scale, pack(vis) if masked else None)
    got = got.view(tokens, heads, hd).double()
    differ = (torch.isnan(got) != torch.isnan(want)).nonzero()
    assert not len(differ), (len(differ), differ[:4].tolist())
    inf, fin = torch.isinf(want) | torch.isinf(got), torch.isfinite(want)
    assert (got[inf] == want[inf]).all()
    bad = ~((got - want).abs() <= bound) & fin
    assert not bad.any(), (bad.nonzero()[:4].tolist(), ((got - want).abs() / bound)[fin].max().item())
    return want


# heads, kv, hd, length, tokens: each head size of the tiled form with one split and with several, its eight-wave form,
# and heads that only the general form takes. Contexts end inside a tile.
SHAPES = [(8, 2, 128, 77, 20), (8, 2, 128, 1500, 20), (28, 4, 128, 4111, 255), (4, 1, 64, 3001, 6), (28, 4, 64, 13715, 120),
          (6, 2, 96, 777, 31), (32, 8, 96, 3444, 671), (4, 4, 256, 301, 20), (5, 1, 256, 937, 638), (4, 4, 320, 130, 6),
          (4, 1, 34, 700, 40)]


def planted(heads, kv, hd, length, tokens, seed):
    """Inputs whose scores are moved by 0.1 k[row, :, 0] alone where dimension 0 is set; the rows to plant values in:
    one in the first tile, in the last whole tile, in the tile where the context ends, and drafted ones."""
    q, k, v = inputs(heads, kv, hd, length, tokens, seed)
    q.view(tokens, heads, hd)[:, :, 0] = 1.0
    k.view(-1, kv, hd)[:length + tokens, :, 0] = 0.0
    vis = tree_mask(tokens, length)
    return q, k, v, vis, [3, length // 64 * 64 - 5, length - 1, length + 1, length + tokens - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES)
@pytest.mark.parametrize("score", ["usual", "underflows", "-inf"])
def test_infinite_values_wherever_their_row_lies(R, heads, kv, hd, length, tokens, score, masked):
    q, k, v, vis, rows = planted(heads, kv, hd, length, tokens, 3)
    if not masked:
        vis = np.tril(np.ones((tokens, tokens), dtype=bool))
    for i, row in enumerate(rows):
        k1, v1 = k.view(-1, kv, hd).clone(), v.view(-1, kv, hd).clone()
        if score != "usual":
            k1[row, :, 0] = -INF if score == "-inf" else -4000.0   # a weight of 0, of e^-400
        v1[row, :, hd // 2] = INF if i % 2 else -INF
        v1[row, 0, hd - 1] = NAN
        want = check(R, q, k1, v1, heads, kv, hd, length, tokens, vis, masked, 0.1)
        hit = want[:, 0, hd // 2]
        assert (torch.isnan(hit) if score == "-inf" else torch.isinf(hit)).any()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES)
def test_infinities_whose_weight_underflows_later(R, heads, kv, hd, length, tokens):
    """Rows that weigh when their tile is summed, and e^-400 of the final maximum."""
    q, k, v, vis, rows = planted(heads, kv, hd, length, tokens, 4)
    k.view(-1, kv, hd)[length // 2:length + tokens, :, 0] = 4000.0
    v = v.view(-1, kv, hd)
    v[rows[0], :, 1] = INF
    v[rows[0] + 1, :, hd - 2] = -INF
    v[rows[2], :, 2] = INF
    v[rows[0], :, 3], v[rows[2], :, 3] = INF, -INF   # both signs: NaN
    want = check(R, q, k, v, heads, kv, hd, length, tokens, vis, True, 0.1)
    assert (want[:, :, 1] == INF).all() and (want[:, :, hd - 2] == -INF).all() and torch.isnan(want[:, :, 3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,length,tokens", SHAPES + [(32, 8, 128, 60000, 2)])
def test_the_largest_values_do_not_overflow(R, heads, kv, hd, length, tokens):
    """Values of up to 2^102, over weights that reach 2^8 before they are normalised: the first half of the rows scores
    5.5 below the rest (2^7.9), where a maximum does not move."""
    q, k, v, vis, _ = planted(heads, kv, hd, length, tokens, 6)
    k.view(-1, kv, hd)[:, :, 1:] = 0.0
    k.view(-1, kv, hd)[length // 2:length + tokens, :, 0] = 55.0
    v = torch.where(v.view(-1, kv, hd) < 0, -1.0, 1.0).to(v.dtype) * 2.0**102
    v[:, :, 0] = 2.0**102
    want = check(R, q, k, v, heads, kv, hd, length, tokens, vis, True, 0.1)
    assert torch.isfinite(want).all()   # and check held every output to it


@pytest.mark.gpu
@pytest.mark.parametrize("hd,length", [(128, 130), (128, 5000), (34, 130)])
def test_a_dimension_of_infinities(R, hd, length):
    """Every row infinite in one dimension (every row but the last underflows), and a key of -inf among them."""
    heads, kv, tokens = 4, 2, 9
    q, k, v, vis, rows = planted(heads, kv, hd, length, tokens, 5)
    vis[:, 0] = True
    k.view(-1, kv, hd)[length, :, 0] = 4000.0
    v.view(-1, kv, hd)[:, :, 4] = INF
    want = check(R, q, k, v, heads, kv, hd, length, tokens, vis, True, 0.1)
    assert (want[:, :, 4] == INF).all()
    k.view(-1, kv, hd)[rows[1], 1, 0] = -INF
    want = check(R, q, k, v, heads, kv, hd, length, tokens, vis, True, 0.1)
    assert (want[:, :2, 4] == INF).all() and torch.isnan(want[:, 2:, 4]).all()
