"""A step of several drafted tokens through a layer whose weights carry block
scales, as the operators are used together: norm to fp8, q/k/v product, RoPE and
cache rows per token, tree attention, quantize, o product, gated residual norm to
fp8, gate/up product, SiLU, quantize, down product, the next norm in bf16.

Against the same layer in float64 over the dequantized weights. What differs is
the rounding of activations: four of them pass through e4m3, whose step leaves a
value off by at most 2^-4 of itself, uniformly 2^-4 / sqrt(3) = 3.6% in the root
mean square, and a product's output takes over that share of its operand's. Added
up without any cancelling, four times 3.6% is 15% of a branch's output; bf16's
2^-8 and the rest are within the 0.6% to 16%.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

EPS = 1e-5


@pytest.fixture(scope="module")
def R():
    import reng_hip

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    reng_hip.lib()
    return reng_hip


def tree(t, seed):
    """(parent truth values, depths) of a random tree."""
    rng = np.random.default_rng(seed)
    vis, depth = np.zeros((t, t), dtype=bool), np.zeros(t, dtype=int)
    for i in range(t):
        back = int(rng.integers(0, min(i, 4) + 1))
        if back:
            vis[i], depth[i] = vis[i - back], depth[i - back] + 1
        vis[i, i] = True
    return vis, depth


def words(vis):
    t = vis.shape[0]
    full = np.zeros((t, -(-t // 32) * 32), dtype=bool)
    full[:, :t] = vis
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def rms(x, g):
    return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * g


def rotate(x, sin, cos):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]], -1)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,length,hidden,heads,kv,hd,inter", [(9, 70, 512, 8, 2, 64, 1024), (1, 300, 576, 9, 3, 64, 1536),
                                                                    (33, 0, 640, 5, 1, 128, 1008), (70, 130, 512, 4, 4, 128, 784)])
def test_step_of_drafted_tokens(R, tokens, length, hidden, heads, kv, hd, inter):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731

    def weight(n, k):
        w = rn(n, k) / k**0.5
        codes, scales = R.quantize_blocks(w, n, k, "e4m3", 128)
        v = codes.view(torch.float8_e4m3fn).view(n, k).double()
        kb = -(-k // 128)
        s = scales.view(-1, kb).double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        return codes, scales, v * s

    def product(a, sa, w, m, n, k):
        return R.gemm_fp8_blocks(a, "e4m3", sa, w[0], "e4m3", w[1], m, n, k).view(m, n)

    nq, nk = heads * hd, kv * hd
    wqkv, wo, wgu, wd = weight(nq + 2 * nk, hidden), weight(hidden, nq), weight(2 * inter, hidden), weight(hidden, inter)
    g1, g2, g3, pg = (1 + 0.1 * rn(hidden) for _ in range(4))
    gate = (1 + 0.2 * rn(tokens, hidden)).bfloat16()
    x = rn(tokens, hidden)
    kc, vc = rn(length + tokens, nk).bfloat16(), rn(length + tokens, nk).bfloat16()
    kr, vr = kc.double(), vc.double()
    vis, depth = tree(tokens, 3)
    pos = torch.from_numpy(length + depth).cuda()
    ang = pos[:, None].float() * (10000.0 ** (-torch.arange(hd // 2, device="cuda").float() * 2 / hd)).repeat(2)[None]
    sin, cos = ang.sin().contiguous(), ang.cos().contiguous()
    scale, rs = hd**-0.5, 0.6

    # The operators, as a program strings them together.
    _, a, sa = R.residual_norm_fp8(x, None, g1, tokens, hidden, EPS, "e4m3")
    qkv = product(a, sa, wqkv, tokens, nq + 2 * nk, hidden)
    q = qkv[:, :nq].contiguous()
    for i in range(tokens):
        R.rope_append(q[i], qkv[i, nq:nq + nk].contiguous(), qkv[i, nq + nk:].contiguous(), heads, kv, hd, sin[i], cos[i],
                      kc[length + i], vc[length + i])
    att = R.attention_tree(q, kc, vc, heads, kv, hd, length, tokens, scale, words(vis))
    a, sa = R.quantize_blocks(att, tokens, nq, "e4m3", 1)
    d1 = product(a, sa, wo, tokens, hidden, nq)
    h1, a, sa = R.residual_norm_fp8(x, d1, g2, tokens, hidden, EPS, "e4m3", pg, gate, rs)
    gu = product(a, sa, wgu, tokens, 2 * inter, hidden)
    act = R.silu_mul_bf16(gu[:, :inter].contiguous(), gu[:, inter:].contiguous(), tokens * inter)
    a, sa = R.quantize_blocks(act, tokens, inter, "e4m3", 1)
    d2 = product(a, sa, wd, tokens, hidden, inter)
    h2, n = R.residual_norm_bf16(h1, d2, g3, tokens, hidden, EPS)

    # The layer in float64.
    X = x.double()
    y = rms(X, g1.double()) @ wqkv[2].T
    s64, c64 = sin.double()[:, None], cos.double()[:, None]
    Q = rotate(y[:, :nq].view(tokens, heads, hd), s64, c64)
    kr[length:] = rotate(y[:, nq:nq + nk].view(tokens, kv, hd), s64, c64).reshape(tokens, nk)
    vr[length:] = y[:, nq + nk:]
    see = torch.ones(tokens, length + tokens, dtype=torch.bool, device="cuda")
    see[:, length:] = torch.from_numpy(vis).cuda()
    A = torch.empty(tokens, heads, hd, dtype=torch.float64, device="cuda")
    for h in range(heads):
        lo = h // (heads // kv) * hd
        s = (Q[:, h] @ kr[:, lo:lo + hd].T * scale).masked_fill(~see, -float("inf"))
        A[:, h] = torch.softmax(s, 1) @ vr[:, lo:lo + hd]
    D1 = A.view(tokens, nq) @ wo[2].T
    H1 = X + rs * gate.double() * rms(D1, pg.double())
    u = rms(H1, g2.double()) @ wgu[2].T
    D2 = (u[:, :inter] * torch.sigmoid(u[:, :inter]) * u[:, inter:]) @ wd[2].T
    H2 = H1 + D2
    N = rms(H2, g3.double())
    for name, got, want in (("o", d1, D1), ("down", d2, D2)):
        rel = (got.double() - want).norm() / want.norm()
        assert rel < 0.16, (name, rel.item())
    rel = (n.view(tokens, hidden).double() - N).norm() / N.norm()
    assert rel < 0.16, rel.item()
    assert torch.isfinite(h2).all()


@pytest.mark.gpu
def test_a_chain_is_its_tokens_one_by_one(R):
    """A chain of tokens in one call and the same tokens decoded one at a time, within both roundings."""
    heads, kv, hd, length, tokens = 8, 2, 128, 200, 37
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(tokens * heads * hd, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn((length + tokens) * kv * hd, generator=g, device="cuda").bfloat16() for _ in range(2))
    whole = R.attention_tree(q, k, v, heads, kv, hd, length, tokens, 0.1).view(tokens, -1).double()
    for i in range(tokens):
        one = R.attention_tree(q.view(tokens, -1)[i], k, v, heads, kv, hd, length + i, 1, 0.1).double()
        assert (one - whole[i]).norm() <= 2.0**-7 * whole[i].norm()


@pytest.mark.gpu
def test_two_streams_with_workspaces_of_their_own(R):
    """Two attention calls at once on two streams, each with its own workspace, give what they give alone."""
    heads, kv, hd, length, tokens = 16, 4, 128, 4000, 6
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(2, tokens * heads * hd, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(2, (length + tokens) * kv * hd, generator=g, device="cuda").bfloat16() for _ in range(2))
    alone = [R.attention_tree(q[i], k[i], v[i], heads, kv, hd, length, tokens, 0.1) for i in range(2)]
    n = R.attention_tree_workspace_bytes(heads, kv, hd, length, tokens)
    assert n > 0
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = [torch.empty_like(alone[0]) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                R.attention_tree(q[i], k[i], v[i], heads, kv, hd, length, tokens, 0.1, None, ws[i], out[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i].view(torch.int16), alone[i].view(torch.int16))
