"""A layer held in 4 bits, as its operators are used together: norm, quantize, q/k/v products, head norms with
rotation into the 4-bit cache, attention, quantize, o product, residual norm, quantize, gate and up products, SiLU,
quantize, down product; a prompt, then a tree of drafted tokens, then single tokens over the same cache.

Each operator is held against 64 bits over what the one before it left, with the bounds of its own tests: codes
are the quantizer's exactly, products, queries, cache rows and attention within theirs.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mx_reference as X  # noqa: E402
from test_gpu_attention_tree import pack, reference, tree_mask  # noqa: E402
from test_gpu_heads import check_codes, near  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


class Layer:
    def __init__(self, R, hidden, heads, kv, hd, inter, capacity, axes=1):
        g = torch.Generator(device="cuda").manual_seed(hidden + hd)
        self.rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.R, self.hidden, self.heads, self.kv, self.hd, self.inter = R, hidden, heads, kv, hd, inter
        shapes = dict(qkv=((heads + 2 * kv) * hd, hidden), o=(hidden, heads * hd), gate=(inter, hidden), up=(inter, hidden),
                      down=(hidden, inter))
        self.shapes = shapes
        self.w = {n: R.quantize_mxfp4(self.rn(*s) / s[1]**0.5, *s) for n, s in shapes.items()}
        self.g1, self.g2 = (1 + 0.1 * self.rn(hidden) for _ in range(2))
        self.gq, self.gk = (1 + 0.1 * self.rn(hd) for _ in range(2))
        ang = torch.arange(capacity, device="cuda")[:, None].double() / 100.0 ** (torch.arange(hd // 2, device="cuda") / (hd // 2))
        ang = torch.cat([ang, ang], 1)
        first = hd // 2 // axes
        self.rope = R.Rope(ang.sin().float(), ang.cos().float(), sections=[first] * (axes - 1) + [hd // 2 - first * (axes - 1)])
        self.ang, self.axes = ang.double(), axes
        self.pair_axis = torch.tensor([min(d // first, axes - 1) for d in range(hd // 2)], device="cuda")
        self.cache = R.MxCache(kv, hd, capacity)
        for t in self.cache.tensors:
            t.fill_(255)

    def linear(self, seen, name, x, m):
        n, k = self.shapes[name]
        codes, scales = self.R.quantize_mxfp4(x, m, k)
        out = self.R.gemm_mxfp4(codes, scales, *self.w[name], m, n, k)
        seen.append(("linear", name, x, codes, scales, out))
        return out

    def forward(self, x, positions, length, mask):
        """x f32 [tokens, hidden] to the layer's output; also what every operator took and left."""
        R, seen, m = self.R, [], x.shape[0]
        nq, nk = self.heads * self.hd, self.kv * self.hd
        _, a = R.residual_norm_bf16(x, None, self.g1, m, self.hidden, EPS)
        qkv = self.linear(seen, "qkv", a, m).view(m, -1)
        q = R.head_norm_rope_mxfp4(qkv[:, :nq], qkv[:, nq:nq + nk], qkv[:, nq + nk:], m, self.heads, self.cache, length,
                                   self.gq, self.gk, EPS, self.rope, positions)
        att = R.attention_mxfp4(q, self.cache, self.heads, length, m, self.hd**-0.5, mask)
        seen.append(("attention", qkv, q, att))
        h, a = R.residual_norm_bf16(x, self.linear(seen, "o", att, m), self.g2, m, self.hidden, EPS)
        gate, up = self.linear(seen, "gate", a, m), self.linear(seen, "up", a, m)
        act = R.silu_mul_bf16(gate, up, m * self.inter)
        return R.add_bf16_f32(h, self.linear(seen, "down", act, m), m * self.hidden).view(m, -1), seen

    def rotated(self, x, gamma, positions):
        """(want, error) [tokens, heads, hd] as in the head norms' own tests."""
        y = x.double().reshape(x.shape[0], -1, self.hd)
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * gamma.double()
        half = self.hd // 2
        row = positions.view(self.axes, -1).long()[self.pair_axis].T
        ang = self.ang[row, torch.arange(half, device="cuda")][:, None]
        c, s = ang.cos().float().double(), ang.sin().float().double()
        a, b = y[..., :half], y[..., half:]
        e = torch.cat([a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs()], -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1), (self.hd + 16) * 2.0**-23 * e

    def check(self, seen, positions, length, vis):
        m = positions.numel() // self.axes
        for kind, *rest in seen:
            if kind == "linear":
                name, x, codes, scales, out = rest
                n, k = self.shapes[name]
                want = X.pack(*X.quantize(x.double().view(m, k)))
                assert torch.equal(codes.view(m, -1), want[0]) and torch.equal(scales.view(m, -1), want[1]), name
                a, b = (X.values(X.unpack(c.view(r, -1), k), s.view(r, -1)[:, :k // 32])
                        for c, s, r in ((codes, scales, m), (*self.w[name], n)))
                exact, t = a @ b.T.contiguous(), a.abs() @ b.abs().T.contiguous()
                bound = 2.0**-8 * exact.abs() + (2.0**-12 + (-(-k // 128) + 24) * 2.0**-23) * t
                assert ((out.view(m, n).double() - exact).abs() <= bound).all(), name
                continue
            qkv, q, att = rest
            nq, nk = self.heads * self.hd, self.kv * self.hd
            near(q, *self.rotated(qkv[:, :nq], self.gq, positions), "q")
            parts = [self.rotated(qkv[:, nq:nq + nk], self.gk, positions),
                     (qkv[:, nq + nk:].double().reshape(m, self.kv, self.hd), torch.zeros(m, self.kv, self.hd, device="cuda"))]
            vals = []
            for i, part in enumerate(parts):
                codes, scales = (t.view(self.kv, self.cache.capacity, -1) for t in self.cache.tensors[2 * i:2 * i + 2])
                want, err = (t.transpose(0, 1).reshape(-1, self.hd) for t in part)
                new = slice(length, length + m)
                check_codes(codes[:, new].reshape(-1, self.hd // 2), scales[:, new].reshape(self.kv * m, -1), want, err, "kv"[i])
                rows = slice(0, length + m)
                v = X.values(X.unpack(codes[:, rows].reshape(-1, self.hd // 2), self.hd),
                             scales[:, rows].reshape(self.kv * (length + m), -1)[:, :self.hd // 32])
                vals.append(v.view(self.kv, length + m, self.hd).transpose(0, 1).reshape(-1))
            want, bound = reference(q, *vals, self.heads, self.kv, self.hd, length, m, vis, self.hd**-0.5)
            lost = 2.0**-125 * vals[1].abs().view(-1, self.kv, self.hd).sum(0).repeat_interleave(self.heads // self.kv, 0)
            got = att.view(m, self.heads, self.hd).double()
            assert ((got - want).abs() <= bound + 2.0**-8 * want.abs() + lost).all()


@pytest.mark.parametrize("hidden,heads,kv,hd,inter,axes", [(512, 8, 2, 64, 1024, 1), (576, 9, 3, 64, 1536, 1),
                                                           (1024, 4, 4, 128, 1536, 3), (480, 3, 1, 96, 416, 2)])
def test_prompt_tree_and_single_tokens(R, hidden, heads, kv, hd, inter, axes):
    layer = Layer(R, hidden, heads, kv, hd, inter, 400, axes)
    length = 0
    for tokens, tree in ((150, False), (33, True), (1, False), (2, False), (1, False)):
        vis = tree_mask(tokens, 5) if tree else np.tril(np.ones((tokens, tokens), dtype=bool))
        depth = torch.from_numpy(vis.sum(1) - 1).cuda()
        positions = (length + depth + torch.arange(axes, device="cuda")[:, None]).int().contiguous()
        x = layer.rn(tokens, hidden)
        out, seen = layer.forward(x, positions, length, pack(vis) if tree else None)
        assert torch.isfinite(out).all()
        layer.check(seen, positions, length, vis)
        length += tokens if not tree else 4   # a few of the drafted tokens stay


def test_a_captured_step_replays(R):
    """A whole single-token step as one graph, replayed with other inputs and eager work between: each replay gives the
    eager step's bits."""
    layer = Layer(R, 512, 8, 2, 64, 1024, 300)
    length = 200
    layer.forward(layer.rn(length, 512), torch.arange(length, device="cuda").int(), 0, None)
    x, positions = layer.rn(1, 512), torch.tensor([length], dtype=torch.int32, device="cuda")
    layer.forward(x, positions, length, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = layer.forward(x, positions, length, None)
    for rep in range(4):
        x.copy_(layer.rn(1, 512))
        positions.fill_(length + rep)
        want = layer.forward(x, positions, length, None)[0].clone()
        out.zero_()
        layer.cache.write(*(layer.rn(1, 128).bfloat16() for _ in range(2)), length, 1)   # the step writes its row anew
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep


def test_steps_on_two_streams(R):
    """Two layers at once, each on a stream of its own, give what each gives alone."""
    layers = [Layer(R, 512, 8, 2, 64, 1024, 300), Layer(R, 576, 9, 3, 64, 1536, 300)]
    xs = [x.rn(n, x.hidden) for x, n in zip(layers, (70, 70))]
    pos = torch.arange(70, device="cuda").int()
    alone = [m.forward(x, pos, 0, None)[0].clone() for m, x in zip(layers, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(5):
        got = []
        for s, m, x in zip(streams, layers, xs):
            with torch.cuda.stream(s):
                got.append(m.forward(x, pos, 0, None))
        torch.cuda.synchronize()
        for g, w in zip(got, alone):
            assert torch.equal(g[0], w)
