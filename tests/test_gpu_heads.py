"""Head norms, rotation and the 4-bit cache, against 64 bits.

Per value, with y the normalised head, (c, s) its cosine and sine and E = |y| |c| + |y'| |s| (|y| where nothing
rotates):

    |got - want| <= 2^-8 |want| + (head_dim + 16) 2^-23 E

2^-8: the rounding to bf16. A sum of head_dim squares is off by at most head_dim 2^-24 of itself, its root by half of
that; the mean, eps, root, reciprocal, two products and the rotation's three roundings by 2^-24 each. In the cache a
value is the rounding of one within the second term of the exact one: rounding keeps order, so the code lies between
those of the two ends, and the scale is one that either end of the largest magnitude has.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_reference as X  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def sections_of(half, axes):
    first = [half // axes - (1 if a == 0 and axes > 1 else 0) for a in range(axes)]
    first[-1] += half - sum(first)
    return first


class Case:
    def __init__(self, tokens, heads, kv, hd, rot=None, axes=1, norm=True, seed=0, rows=300, pair_axis=None):
        self.tokens, self.heads, self.kv, self.hd = tokens, heads, kv, hd
        nq, nk = heads * hd, kv * hd
        self.qkv = (randn(seed, tokens, nq + 2 * nk) * torch.exp2(randn(seed + 1, tokens, 1))).bfloat16()
        self.q, self.k, self.v = self.qkv[:, :nq], self.qkv[:, nq:nq + nk], self.qkv[:, nq + nk:]
        self.gq, self.gk = (1 + 0.2 * randn(seed + 2, hd), 1 + 0.2 * randn(seed + 3, hd)) if norm else (None, None)
        self.rot, self.axes = rot, axes
        if rot:
            half = rot // 2
            # Halves with angles of their own, as scaled tables have them.
            ang = randn(seed + 4, rows, rot).double() * 3
            self.sin, self.cos = ang.sin().float().contiguous(), ang.cos().float().contiguous()
            g = torch.Generator(device="cuda").manual_seed(seed + 5)
            self.positions = torch.randint(0, rows, (axes, tokens), generator=g, device="cuda").int()
            if pair_axis is None:
                self.sections = sections_of(half, axes)
                self.pair_axis = torch.repeat_interleave(torch.arange(axes), torch.tensor(self.sections)).cuda()
            else:
                self.sections, self.pair_axis = None, torch.tensor(pair_axis).cuda()

    def rope(self, R):
        if not self.rot:
            return None
        if self.sections is None:
            return R.Rope(self.sin, self.cos, pair_axis=self.pair_axis.tolist())
        return R.Rope(self.sin, self.cos, sections=self.sections if self.axes > 1 else None)

    def args(self, R):
        return dict(q_gamma=self.gq, k_gamma=self.gk, eps=EPS, rope=self.rope(R), positions=self.positions if self.rot else None)

    def exact(self, x, gamma):
        """(want, error bound without the rounding) [tokens, heads, hd] of rows x."""
        x = x.double().reshape(self.tokens, -1, self.hd)
        y = x
        if gamma is not None:
            y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * gamma.double()
        e = y.abs()
        if self.rot:
            half = self.rot // 2
            row = self.positions.long()[self.pair_axis].T          # [tokens, half]
            d = torch.arange(half, device="cuda")
            t = lambda table, o: table.double()[row, d + o][:, None]  # noqa: E731
            a, b = y[..., :half], y[..., half:self.rot]
            c0, s0, c1, s1 = t(self.cos, 0), t(self.sin, 0), t(self.cos, half), t(self.sin, half)
            e = torch.cat([a.abs() * c0.abs() + b.abs() * s0.abs(), b.abs() * c1.abs() + a.abs() * s1.abs(), e[..., self.rot:]], -1)
            y = torch.cat([a * c0 - b * s0, b * c1 + a * s1, y[..., self.rot:]], -1)
        exact = gamma is None and not self.rot
        return y, (0 if exact else (self.hd + 16) * 2.0**-23) * e


def near(got, want, err, what):
    bound = 2.0**-8 * want.abs() + err
    off = (got.view(want.shape).double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, bad.nonzero()[:4].tolist(), (off / bound).nan_to_num(0).max().item())


def check_codes(codes, scales, want, err, what):
    """A cache's rows [n, hd / 2] and [n, pitch] against f64 want, err [n, hd]."""
    n, hd = want.shape
    low, high = want.abs() - err, want.abs() + err
    top = lambda t: t.clamp(min=0).view(n, -1, 32).amax(-1)  # noqa: E731
    byte = scales[:, :hd // 32]
    assert (scales[:, hd // 32:] == 127).all(), what
    blo, bhi = (X.quantize(top(t).repeat_interleave(32, 1))[1] for t in (low, high))
    assert ((byte == blo) | (byte == bhi)).all(), what
    s = torch.exp2(byte.double() - 127).repeat_interleave(32, 1)
    clamp = lambda q: q.clamp(-6.9, 6.9)  # noqa: E731  (an end may lie past the largest)
    lo, hi = (X.level(X.nearest(clamp((want + z * err) / s))) for z in (-1, 1))
    got = X.level(X.unpack(codes, hd))
    assert ((got >= lo) & (got <= hi)).all(), (what, ((got < lo) | (got > hi)).nonzero()[:4].tolist())


def guarded_cache(R, kv, hd, capacity):
    """A cache whose tensors lie between guards."""
    parts, full = [], []
    for n in (hd // 2, X.pitch(hd)) * 2:
        t = torch.full((kv * capacity * n + 128,), 0x5A, dtype=torch.uint8, device="cuda")
        full.append(t)
        parts.append(t[64:64 + kv * capacity * n])
    return R.MxCache(kv, hd, capacity, tensors=parts), full


CASES = [  # tokens, heads, kv, hd, rot, axes, norm
    (1, 32, 8, 128, 128, 1, True), (1, 1, 1, 32, 32, 1, True), (3, 9, 3, 64, 64, 1, False), (17, 28, 4, 128, 128, 3, True),
    (5, 4, 2, 96, 96, 1, True), (7, 6, 2, 256, 256, 2, True), (33, 8, 8, 64, 32, 1, True), (2, 5, 5, 160, 80, 4, True),
    (64, 40, 8, 128, 64, 3, True), (9, 3, 1, 32, 16, 1, True), (6, 4, 4, 224, None, 1, True), (11, 2, 1, 128, 128, 4, False),
    (300, 8, 2, 128, 128, 1, True), (1, 4, 4, 192, 192, 3, True),
]


@pytest.mark.parametrize("tokens,heads,kv,hd,rot,axes,norm", CASES)
def test_bf16_rows(R, tokens, heads, kv, hd, rot, axes, norm):
    c = Case(tokens, heads, kv, hd, rot, axes, norm, seed=tokens + hd)
    guard = lambda n: torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    outs = [guard(tokens * h * hd) for h in (heads, kv, kv)]
    R.head_norm_rope_bf16(c.q, c.k, c.v, tokens, heads, kv, hd, **c.args(R), q_out=outs[0], k_rows=outs[1], v_rows=outs[2])
    for out, h in zip(outs, (heads, kv, kv)):
        assert (out[tokens * h * hd:] == 7.0).all(), "written past the end"
    near(outs[0][:tokens * heads * hd], *c.exact(c.q, c.gq), "q")
    near(outs[1][:tokens * kv * hd], *c.exact(c.k, c.gk), "k")
    assert torch.equal(outs[2][:tokens * kv * hd].view(tokens, -1), c.v)


@pytest.mark.parametrize("tokens,heads,kv,hd,rot,axes,norm", CASES)
@pytest.mark.parametrize("first,spare", [(0, 0), (13, 5)])
def test_cache_rows(R, tokens, heads, kv, hd, rot, axes, norm, first, spare):
    c = Case(tokens, heads, kv, hd, rot, axes, norm, seed=tokens + hd + 1)
    capacity = first + tokens + spare
    cache, full = guarded_cache(R, kv, hd, capacity)
    q = R.head_norm_rope_mxfp4(c.q, c.k, c.v, tokens, heads, cache, first, **c.args(R))
    near(q, *c.exact(c.q, c.gq), "q")
    for t in full:
        assert (t[:64] == 0x5A).all() and (t[-64:] == 0x5A).all(), "written past the cache"
    exact = dict(k=c.exact(c.k, c.gk), v=(c.v.double().reshape(tokens, kv, hd), torch.zeros((), device="cuda")))
    for i, n in enumerate("kv"):
        codes, scales = (t.view(kv, capacity, -1) for t in cache.tensors[2 * i:2 * i + 2])
        for t in (codes, scales):
            assert (t[:, :first] == 0x5A).all() and (t[:, first + tokens:] == 0x5A).all(), "other rows were written"
        rows = slice(first, first + tokens)
        want, err = (torch.broadcast_to(t, (tokens, kv, hd)).transpose(0, 1).reshape(-1, hd) for t in exact[n])
        check_codes(codes[:, rows].reshape(-1, hd // 2), scales[:, rows].reshape(kv * tokens, -1), want, err, n)
    # What is read back are those codes' values.
    k, v = cache.read(first, tokens)
    for i, t in enumerate((k, v)):
        codes, scales = (x.view(kv, capacity, -1)[:, first:first + tokens] for x in cache.tensors[2 * i:2 * i + 2])
        want = X.values(X.unpack(codes.reshape(-1, hd // 2), hd), scales.reshape(kv * tokens, -1)[:, :hd // 32])
        assert torch.equal(t.view(tokens, kv, hd).double(), want.view(kv, tokens, hd).transpose(0, 1))


@pytest.mark.parametrize("heads,kv,hd,rot,axes,off", [(140, 3, 32, 32, 1, 0), (60, 7, 64, 32, 3, 0), (28, 4, 128, 128, 3, 0),
                                                      (9, 5, 160, 160, 2, 0), (31, 2, 96, 96, 1, 1), (40, 8, 128, 128, 1, 3)])
def test_many_tokens_are_the_same_as_few(R, heads, kv, hd, rot, axes, off):
    """Many tokens, of which a group of lanes takes several heads: the bits of calls of a few, rows and cache, in place too."""
    tokens = 1100
    c = Case(tokens, heads, kv, hd, rot, axes, True, seed=hd)
    n, nq, nk = c.qkv.shape[1], heads * hd, kv * hd
    wide = torch.zeros(tokens, n + off, dtype=torch.bfloat16, device="cuda")
    wide[:, off:] = c.qkv
    q, k, v = wide[:, off:off + nq], wide[:, off + nq:off + nq + nk], wide[:, off + nq + nk:]
    got = R.head_norm_rope_bf16(q, k, v, tokens, heads, kv, hd, **c.args(R))
    caches = [R.MxCache(kv, hd, tokens + 9) for _ in range(2)]
    for t in caches[0].tensors + caches[1].tensors:
        t.fill_(0x5A)
    q4 = R.head_norm_rope_mxfp4(q, k, v, tokens, heads, caches[0], 4, **c.args(R))
    for a in range(0, tokens, 50):
        b = a + 50
        args = dict(c.args(R), positions=c.positions[:, a:b].contiguous())
        want = R.head_norm_rope_bf16(q[a:b], k[a:b], v[a:b], 50, heads, kv, hd, **args)
        for g, w, h in zip(got, want, (heads, kv, kv)):
            assert torch.equal(g.view(tokens, -1)[a:b].reshape(-1), w), a
        R.head_norm_rope_mxfp4(q[a:b], k[a:b], v[a:b], 50, heads, caches[1], 4 + a, **args)
    assert torch.equal(q4, got[0])
    for g, w in zip(caches[0].tensors, caches[1].tensors):
        assert torch.equal(g, w)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    R.head_norm_rope_bf16(q, k, v, tokens, heads, kv, hd, **c.args(R), q_out=q, k_rows=k, v_rows=v)
    for g, w in zip((q, k, v), got):
        assert torch.equal(g.view(-1), w)


@pytest.mark.parametrize("hd,kv", [(32, 1), (64, 3), (128, 8), (256, 2), (96, 5)])
def test_a_plain_write_is_the_quantizer(R, hd, kv):
    """Without gammas and rotation the cache holds the quantizer's codes and scales of each head's rows."""
    tokens = 37
    k, v = (randn(i + hd, tokens, kv * hd).bfloat16() for i in range(2))
    cache = R.MxCache(kv, hd, 50)
    cache.write(k, v, 9, tokens)
    for i, t in enumerate((k, v)):
        rows = t.view(tokens, kv, hd).transpose(0, 1).contiguous()
        codes, scales = R.quantize_mxfp4(rows, kv * tokens, hd)
        got = [x.view(kv, 50, -1)[:, 9:9 + tokens].reshape(-1) for x in cache.tensors[2 * i:2 * i + 2]]
        assert torch.equal(got[0], codes) and torch.equal(got[1], scales)


def test_rows_written_again(R):
    """The last write of a row counts, also with other rows written between."""
    cache = R.MxCache(2, 64, 8)
    a, b = (randn(i, 3, 128).bfloat16() for i in range(2))
    cache.write(a, a, 2, 3)
    cache.write(b, b, 3, 3)
    cache.write(a, a, 4, 1)
    k, _ = cache.read(2, 4)
    want = torch.stack([a[0], b[0], a[0], b[2]])
    codes, scales = R.quantize_mxfp4(want, 8, 64)
    assert torch.equal(k, R.dequantize_mxfp4(codes, scales, 8, 64))


def test_axes_of_pairs_in_turn(R):
    """An axis for each pair, interleaved, and two positions equal."""
    pair_axis = [d % 3 for d in range(64)]
    c = Case(21, 4, 2, 128, 128, 3, True, seed=5, pair_axis=pair_axis)
    q, k, _ = R.head_norm_rope_bf16(c.q, c.k, c.v, 21, 4, 2, 128, **c.args(R))
    near(q, *c.exact(c.q, c.gq), "q")
    near(k, *c.exact(c.k, c.gk), "k")


def test_in_place_and_without_values_or_queries(R):
    c = Case(19, 8, 2, 64, 64, 1, True, seed=6)
    q, k = c.q.contiguous(), c.k.contiguous()
    want = R.head_norm_rope_bf16(q, k, None, 19, 8, 2, 64, **c.args(R))
    assert want[2] is None
    R.head_norm_rope_bf16(q, k, None, 19, 8, 2, 64, **c.args(R), q_out=q, k_rows=k)
    assert torch.equal(q.view(-1), want[0]) and torch.equal(k.view(-1), want[1])
    only = R.head_norm_rope_bf16(None, c.k, None, 19, 0, 2, 64, **c.args(R))
    assert only[0] is None and torch.equal(only[1], want[1])


@pytest.mark.parametrize("off", [1, 4])
def test_unaligned_rows(R, off):
    """Rows that start anywhere, of an odd pitch: the same bits as aligned ones."""
    tokens, heads, kv, hd = 13, 4, 2, 96
    c = Case(tokens, heads, kv, hd, 96, 1, True, seed=8)
    want = R.head_norm_rope_bf16(c.q, c.k, c.v, tokens, heads, kv, hd, **c.args(R))
    width = c.qkv.shape[1] + 7
    wide = torch.zeros(tokens, width, dtype=torch.bfloat16, device="cuda")
    wide[:, off:off + c.qkv.shape[1]] = c.qkv
    nq, nk = heads * hd, kv * hd
    q, k, v = wide[:, off:off + nq], wide[:, off + nq:off + nq + nk], wide[:, off + nq + nk:off + nq + 2 * nk]
    got = R.head_norm_rope_bf16(q, k, v, tokens, heads, kv, hd, **c.args(R))
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    caches = [R.MxCache(kv, hd, 20) for _ in range(2)]
    for cache, (a, b, d) in zip(caches, ((c.q, c.k, c.v), (q, k, v))):
        for t in cache.tensors:
            t.zero_()
        R.head_norm_rope_mxfp4(a, b, d, tokens, heads, cache, 3, **c.args(R))
    for g, w in zip(caches[0].tensors, caches[1].tensors):
        assert torch.equal(g, w)


@pytest.mark.parametrize("bad", [-1, 300, 2**31 - 1, -2**31])
def test_a_position_outside_the_tables_is_nan(R, bad):
    c = Case(5, 2, 2, 128, 64, 2, True, seed=9)
    c.positions[1, 2] = bad
    q, k, v = R.head_norm_rope_bf16(c.q, c.k, c.v, 5, 2, 2, 128, **c.args(R))
    nan = torch.zeros(5, 2, 128, dtype=torch.bool, device="cuda")
    pairs = (c.pair_axis == 1).nonzero().view(-1)
    nan[2, :, pairs] = True
    nan[2, :, pairs + 32] = True
    assert torch.equal(torch.isnan(q.view(5, 2, 128)), nan) and torch.equal(torch.isnan(k.view(5, 2, 128)), nan)
    cache = R.MxCache(2, 128, 5)
    R.head_norm_rope_mxfp4(None, c.k, c.v, 5, 0, cache, 0, **c.args(R))
    k, v = (t.view(5, 2, 4, 32) for t in cache.read(0, 5))
    assert torch.equal(torch.isnan(k).all(-1), nan.view(5, 2, 4, 32).any(-1)) and not torch.isnan(v).any()


def test_zeros_infinities_and_nan(R):
    """A head of zeros stays zeros; one with NaN is NaN, and its neighbours are as they were."""
    c = Case(6, 2, 2, 64, 64, 1, True, seed=10)
    want = R.head_norm_rope_bf16(c.q, c.k, c.v, 6, 2, 2, 64, **c.args(R))
    q = c.q.clone()
    q[1, :64], q[2, 5], q[3, 70] = 0, float("nan"), float("inf")
    got = R.head_norm_rope_bf16(q, c.k, c.v, 6, 2, 2, 64, **c.args(R))[0].view(6, 2, 64)
    assert (got[1, 0] == 0).all() and torch.isnan(got[2, 0]).all() and torch.isnan(got[3, 1]).any()
    keep = torch.ones(6, 2, dtype=torch.bool, device="cuda")
    keep[1, 0] = keep[2, 0] = keep[3, 1] = False
    assert torch.equal(got[keep], want[0].view(6, 2, 64)[keep])


def test_read_one_of_both(R):
    cache = R.MxCache(3, 64, 7)
    k, v = (randn(i, 7, 192).bfloat16() for i in range(2))
    cache.write(k, v, 0, 7)
    both = cache.read(2, 4)
    L, T = R.lib(), R._torch()
    out = torch.empty_like(both[0])
    for i in range(2):
        args = (None, out.data_ptr()) if i else (out.data_ptr(), None)
        assert L.reng_hip_cache_read_mxfp4(cache._ref, 2, 4, *args, T.stream()) == 0
        assert torch.equal(out, both[i])


def test_positions_of_another_number_of_tokens_are_refused(R):
    """With several axes an axis' positions start where the one before it ends: more of them than tokens would shift them."""
    c = Case(6, 2, 2, 64, 64, 2, True, seed=12)
    for tokens, positions in ((5, c.positions), (6, c.positions[:1]), (6, c.positions.long()), (6, None)):
        with pytest.raises(ValueError, match="positions"):
            R.head_norm_rope_bf16(c.q, c.k, c.v, tokens, 2, 2, 64, **dict(c.args(R), positions=positions))
