"""The steps between two branches in one pass (post-norm, gate, scaled residual
add, pre-norm), with bf16 rows or fp8 codes and a scale for each 128 columns,
against float64.

u = 2^-24 is f32's half step. A block sum of up to 32768 squares, added over at
most 32 values a thread, 6 steps across a wave and 16 waves, and the division
and square root behind it leave 1 / rms off by at most 32 u relative; a
product chain of three more factors gives 36 u, bounded by 40 u below. So
    |h - want| <= u |want| + 40 u |rs b|
    |n - want| <= 2^-8 |want| (bf16) + 40 u |want| + |g / rms| (u |h| + 40 u |rs b|) + 40 u |want|
the second norm's own 40 u and what the error of h does to the row's mean
square (at most its largest relative share, within the last term).
An fp8 value is off by half a step of its code: 2^-4 (e4m3) or 2^-3 (e5m2) of
itself, or half the smallest code times the scale below the normal range.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

TORCH_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FULL = {"e4m3": 240.0, "e5m2": 57344.0}
HALF_STEP = {"e4m3": 2.0**-4, "e5m2": 2.0**-3}
HALF_TINY = {"e4m3": 2.0**-10, "e5m2": 2.0**-17}
U = 2.0**-24
EPS = 1e-5


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def inputs(rows, cols, post, gate, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(x=rn(rows, cols) * 3, d=rn(rows, cols).bfloat16(), gamma=1 + 0.2 * rn(cols),
                post_gamma=1 + 0.2 * rn(cols) if post else None,
                gate=None if gate == "none" else rn(1 if gate == "one" else rows, cols).bfloat16())


def reference(t, rs):
    """(h, bound of h, n, bound of n before any rounding of the output) in float64."""
    x, d, cols = t["x"].double(), t["d"], t["x"].shape[1]
    b = torch.zeros_like(x) if d is None else d.double()
    if t["post_gamma"] is not None:
        b = b / torch.sqrt(b.pow(2).mean(1, keepdim=True) + EPS) * t["post_gamma"].double()
    if t["gate"] is not None:
        b = b * t["gate"].double()
    b = rs * b
    h = x + b
    dh = U * h.abs() + 40 * U * b.abs()
    g = t["gamma"].double() / torch.sqrt(h.pow(2).mean(1, keepdim=True) + EPS)
    n = h * g
    dn = 80 * U * n.abs() + g.abs() * dh
    return h, dh, n, dn


def check(R, t, rs, out, inplace=False):
    rows, cols = t["x"].shape
    h, dh, n, dn = reference(t, rs)
    x = t["x"].clone()
    kw = dict(post_gamma=t["post_gamma"], gate=t["gate"], residual_scale=rs, h=x if inplace else None)
    if out == "bf16":
        gh, gn = R.residual_norm_bf16(x, t["d"], t["gamma"], rows, cols, EPS, **kw)
        err = (gn.view(rows, cols).double() - n).abs()
        assert (err <= dn + 2.0**-8 * n.abs()).all(), (err / (dn + 2.0**-8 * n.abs())).max()
    else:
        gh, codes, scales = R.residual_norm_fp8(x, t["d"], t["gamma"], rows, cols, EPS, out, **kw)
        kb = -(-cols // 128)
        pad = torch.nn.functional.pad(n.abs(), (0, kb * 128 - cols)).view(rows, kb, 128)
        dpad = torch.nn.functional.pad(dn, (0, kb * 128 - cols)).view(rows, kb, 128)
        m, dm = pad.amax(2), dpad.amax(2)
        s = scales.view(rows, kb).double()
        want = torch.where(m > 0, m / FULL[out], torch.ones_like(m))
        assert ((s - want).abs() <= dm / FULL[out] + 2 * U * want).all()
        se = s.repeat_interleave(128, 1)[:, :cols]
        v = codes.view(TORCH_FP8[out]).view(rows, cols).double() * se
        bound = (n.abs() + dn) * HALF_STEP[out] + dn * 2 + HALF_TINY[out] * se
        assert ((v - n).abs() <= bound).all(), ((v - n).abs() / bound).max()
        assert (codes.view(TORCH_FP8[out]).float().abs() <= FULL[out]).all()
    if t["d"] is not None:
        assert ((gh.view(rows, cols).double() - h).abs() <= dh).all()
        if inplace:
            assert gh.data_ptr() == x.data_ptr()
        else:
            assert torch.equal(x, t["x"]), "an input changed"


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["bf16", "e4m3", "e5m2"])
@pytest.mark.parametrize("post,gate,rs", [(True, "rows", 0.22), (True, "none", 1.0), (False, "one", -1.5),
                                          (False, "none", 1.0)])
@pytest.mark.parametrize("rows,cols", [(1, 4), (2, 1), (3, 127), (1, 128), (5, 132), (2, 576), (33, 1000), (2, 1001),
                                       (1, 4096), (24, 5120), (3, 8196), (2, 16384), (1, 32768), (1, 40000),
                                       (700, 256)])
def test_residual_norm_against_float64(R, rows, cols, post, gate, rs, out):
    check(R, inputs(rows, cols, post, gate, rows * 131 + cols), rs, out)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
@pytest.mark.parametrize("cols", [576, 1001, 40000])
def test_residual_norm_in_place_and_without_a_branch(R, cols, out):
    t = inputs(9, cols, True, "rows", 3)
    check(R, t, 0.5, out, inplace=True)
    t["d"] = t["post_gamma"] = t["gate"] = None
    check(R, t, 0.5, out)
    x = t["x"].clone()
    h = torch.empty_like(x)
    fn = (lambda **k: R.residual_norm_bf16(x, None, t["gamma"], 9, cols, EPS, **k)) if out == "bf16" else (
        lambda **k: R.residual_norm_fp8(x, None, t["gamma"], 9, cols, EPS, out, **k))
    assert fn()[0] is None
    assert fn(h=h)[0] is h and torch.equal(h, x)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_residual_norm_unaligned(R, out):
    """Tensors that begin off 16 bytes take the general form and give the same values."""
    rows, cols = 4, 1024
    t = inputs(rows, cols, True, "rows", 8)
    for name in ("x", "d", "gamma", "post_gamma", "gate"):
        u = dict(t)
        buf = torch.empty(t[name].numel() + 1, dtype=t[name].dtype, device="cuda")
        buf[1:] = t[name].reshape(-1)
        u[name] = buf[1:].view(t[name].shape)
        check(R, u, 0.7, out)


@pytest.mark.gpu
def test_residual_norm_plain_case_is_add_rms_norm(R):
    """No post-norm, no gate, scale 1: the existing add + norm, to its own last bits."""
    t = inputs(17, 2048, False, "none", 4)
    h0, n0 = R.add_rms_norm_bf16(t["x"], t["d"], t["gamma"], 17, 2048, EPS)
    h1, n1 = R.residual_norm_bf16(t["x"], t["d"], t["gamma"], 17, 2048, EPS)
    assert torch.equal(h0, h1)
    # The sums of squares differ in order alone: at most one bf16 step apart.
    assert ((n0.double() - n1.double()).abs() <= 2.0**-7 * n0.double().abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [512, 1001])
def test_residual_norm_special_rows(R, cols):
    """Zero rows stay zero with scale 1; a row with a NaN or an infinity touches no other row."""
    t = inputs(6, cols, False, "none", 5)
    t["x"][1] = 0
    t["d"][1] = 0
    t["x"][2, 7] = float("nan")
    t["x"][4, 3] = float("inf")
    h, codes, scales = R.residual_norm_fp8(t["x"], t["d"], t["gamma"], 6, cols, EPS, "e4m3")
    codes, scales = codes.view(6, cols), scales.view(6, -1)
    assert (codes[1] & 0x7F == 0).all() and (scales[1] == 1).all()
    assert (codes[2] & 0x7F == 0x7F).all()              # every value of that row is NaN
    v = codes.view(torch.float8_e4m3fn).float()
    assert torch.isnan(v[4, 3]) and (v[4, :3] == 0).all()   # inf / inf, and finite / inf
    fine = [0, 3, 5]
    sub = {k: (a[fine].contiguous() if k in ("x", "d") else a) for k, a in t.items()}
    check(R, sub, 1.0, "e4m3")
    h3, c3, s3 = R.residual_norm_fp8(sub["x"], sub["d"], t["gamma"], 3, cols, EPS, "e4m3")
    assert torch.equal(c3.view(3, cols), codes[fine]) and torch.equal(s3.view(3, -1), scales[fine])


@pytest.mark.gpu
def test_residual_norm_in_a_graph(R):
    rows, cols = 24, 1536
    t = inputs(rows, cols, True, "rows", 6)
    h = torch.empty(rows * cols, device="cuda")
    codes = torch.empty(rows * cols, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows * 12, device="cuda")

    def step():
        R.residual_norm_fp8(t["x"], t["d"], t["gamma"], rows, cols, EPS, "e4m3", t["post_gamma"], t["gate"], 0.3, 1.0,
                            h, codes, scales)

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    for k in range(3):
        t["x"].mul_(-0.5).add_(k)
        codes.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = codes.clone(), scales.clone(), h.clone()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (codes, scales, h)))


def test_residual_norm_refusals():
    import ctypes

    import reng_hip as R

    L = R.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    base = dict(x=p, d=p, post_gamma=p, gate=p, gate_ld=256, rs=1.0, gamma=p, rows=4, cols=256, eps=1e-5)

    def refused(words, fp8=None, h=p, out=p, scales=p, **kw):
        a = list({**base, **kw}.values())
        for as_fp8 in ([False, True] if fp8 is None else [fp8]):
            rc = (L.reng_hip_residual_norm_fp8(*a, kw.get("fmt", 0), kw.get("backoff", 1.0), h, out, scales, None) if as_fp8
                  else L.reng_hip_residual_norm_bf16(*a, h, out, None))
            msg = L.reng_hip_last_error().decode()
            assert rc == R.EINVAL and words in msg, msg

    refused("empty shape", rows=0)
    refused("empty shape", cols=0, gate_ld=0)
    refused("too large", rows=1 << 22)
    refused("too large", cols=1 << 31, gate_ld=0)
    refused("null", x=None)
    refused("null", gamma=None)
    refused("null", out=None)
    refused("without a branch", d=None)
    refused("without a branch", d=None, gate=None, gate_ld=0)
    refused("without h", h=None)
    refused("gate pitch 255", gate_ld=255)
    refused("gate pitch 256", gate=None)
    refused("negative", eps=-1.0)
    refused("negative", eps=float("nan"))
    for name in ("x", "post_gamma", "gamma", "d", "gate"):
        refused("aligned", **{name: odd})
    refused("aligned", h=odd)
    refused("aligned", fp8=False, out=odd)
    refused("null", fp8=True, scales=None)
    refused("aligned", fp8=True, scales=odd)
    args = [p, p, None, None, 0, 1.0, p, 4, 256, 1e-5]
    assert L.reng_hip_residual_norm_fp8(*args, 3, 1.0, p, p, p, None) == R.EINVAL
    for bad in (0.0, float("nan"), float("inf"), 3e38):
        assert L.reng_hip_residual_norm_fp8(*args, 0, bad, p, p, p, None) == R.EINVAL


def test_the_binding_refuses_wrong_norm_operands():
    from test_abi import _FakeDev as Fake

    import reng_hip as R

    bf, f32 = torch.bfloat16, torch.float32
    n, cols = 4 * 256, 256
    x, d, g, out = Fake(4 * n, f32), Fake(2 * n, bf), Fake(4 * cols, f32), Fake(2 * n, bf)
    ok = dict(h=Fake(4 * n, f32), out=out)
    for bad, what in [(dict(x=Fake(4 * n - 4, f32)), "x length"), (dict(d=Fake(2 * n - 2, bf)), "d length"),
                      (dict(gamma=Fake(4 * cols - 4, f32)), "gamma length"), (dict(x=Fake(4 * n, bf)), "x must be f32"),
                      (dict(gamma=Fake(2 * cols, bf)), "gamma must be f32")]:
        a = {**dict(x=x, d=d, gamma=g), **bad}
        with pytest.raises(ValueError, match=what):
            R.residual_norm_bf16(a["x"], a["d"], a["gamma"], 4, 256, 1e-5, **ok)
    with pytest.raises(ValueError, match="gate length"):
        R.residual_norm_bf16(x, d, g, 4, 256, 1e-5, gate=Fake(2 * n - 2, bf), **ok)
    with pytest.raises(ValueError, match="post_gamma length"):
        R.residual_norm_bf16(x, d, g, 4, 256, 1e-5, post_gamma=Fake(4, f32), **ok)
    with pytest.raises(ValueError, match="h length"):
        R.residual_norm_bf16(x, d, g, 4, 256, 1e-5, h=Fake(4 * n - 4, f32), out=out)
    with pytest.raises(ValueError, match="scales length"):
        R.residual_norm_fp8(x, d, g, 4, 256, 1e-5, "e4m3", h=Fake(4 * n, f32), codes=Fake(n), scales=Fake(4 * 7, f32))
