"""The rules of the 4-bit operators' launchers, on the host, and what they refuse."""
import ctypes

import pytest

import mx_plans as D


def test_the_shapes_of_one_row_reach_every_number_of_waves():
    """One, two and four waves an output, and no more waves than pieces of k: a wave without any leaves zeros, which is
    right but idle."""
    seen = {}
    for N, K in D.ROW_SHAPES:
        ks = D.mx_row_waves(N, K)
        assert ks <= max(1, -(-K // 2048))
        seen.setdefault(ks, set()).add((N % 2, K % 2048 != 0))
    assert set(seen) == {1, 2, 4}
    for ks, kinds in seen.items():
        assert kinds == {(a, b) for a in (0, 1) for b in (False, True)}, (ks, kinds)


def test_the_shapes_of_the_seen_rows_reach_every_attention_kernel():
    from test_gpu_mxfp4_seen import SHAPES

    plans = [D.mx_attention_plan(*c) for c in SHAPES]
    assert {(p["hdp"], p["form"], p["splits"] > 1) for p in plans} == {
        (h, f, s) for h, forms in ((64, 4), (128, 4), (256, 3)) for f in range(forms) for s in (False, True)}


@pytest.mark.parametrize("scale", [1.01 * 2.0**127, -3e38])
def test_a_scale_that_base_2_cannot_hold_is_refused(scale):
    """Times log2 e it is an infinity, which made NaN of a score of 0."""
    import reng_hip as R

    c, p = R._MxCache(64, 64, 64, 64, 2, 128, 100), ctypes.c_void_p(64)
    assert R.lib().reng_hip_attention_mxfp4(p, ctypes.byref(c), 4, 10, 1, None, scale, p, 1 << 30, p, None) == R.EINVAL
    assert "above 2^127" in R.lib().reng_hip_last_error().decode()


def test_heads_are_refused_where_the_header_says():
    """tokens * ceil(heads D / 8192) of 2^24 and more, for D of 32, 64, 128 and 256."""
    import reng_hip as R

    p = ctypes.c_void_p(64)   # never dereferenced: refused before any device work
    for hd in range(32, 257, 32):
        D = next(d for d in (32, 64, 128, 256) if d >= hd)
        for nh, nkv in ((4096, 4096), (4000, 7), (16 * 256 // D * 32, 1), (16 * 256 // D * 32 - 2, 1)):
            parts = -(-(nh + 2 * nkv) * D // 8192)
            if nh > 4096 or parts * (2**22 - 1) < 2**24:
                continue
            least = -(-2**24 // parts)
            for tokens in (least, 2**22 - 1):
                rc = R.lib().reng_hip_head_norm_rope_bf16(p, nh * hd, p, p, nkv * hd, tokens, nh, nkv, hd, None, None, 1e-6,
                                                          None, None, p, p, p, None)
                assert rc == R.EINVAL and "too many for a launch" in R.lib().reng_hip_last_error().decode(), (hd, nh, nkv, tokens)


def test_axes_of_pairs_come_in_any_sequence():
    """A list, an array of any whole type or a tensor name the same axes; what is no axis is refused."""
    import numpy as np
    import torch

    import reng_hip as R

    class Dev(torch.Tensor):
        is_cuda = property(lambda self: True)

    tables = [torch.zeros(4, 32).as_subclass(Dev) for _ in range(2)]
    axes = [0, 1, 2, 3] * 4
    for pairs in (axes, tuple(axes), np.array(axes), np.array(axes, dtype=np.int32), np.array(axes, dtype=np.uint8), torch.tensor(axes)):
        rope = R.Rope(*tables, pair_axis=pairs)
        assert rope.axes == 4 and rope._struct.axes == 4
        at = ctypes.c_void_p.from_buffer(rope._struct, R._Rope.pair_axis.offset).value
        assert list(ctypes.string_at(at, 16)) == axes
    assert R.Rope(*tables, pair_axis=[0] * 16).axes == 1
    assert R.Rope(*tables, sections=np.array([4, 5, 7])).axes == 3
    for pairs in ([0] * 15 + [-1], [0] * 15 + [4], [0, 300] * 8, [0.5] * 16):
        with pytest.raises((ValueError, TypeError)):
            R.Rope(*tables, pair_axis=pairs)
    for sections in ((16, -3), (20, -4), (4, 4, 4, 2, 2), ()):
        with pytest.raises(ValueError):
            R.Rope(*tables, sections=sections)


def test_the_heads_rule():
    """Few tokens take one head a group of lanes, many four where that wastes few groups, and where one would not fit a launch;
    the GPU tests' shapes reach both for every number of lanes."""
    four = D.heads_by_four
    assert [four(t, 56, 128) for t in (1, 300, 639, 640, 1024, 4096)] == [False, False, False, True, True, True]
    assert [four(t, 56, 128, mixed=True) for t in (1, 383, 384, 640)] == [False, False, True, True]
    assert not four(4000, 80, 128) and four(4000, 80, 128, mixed=True) and not four(4000, 16, 128) and not four(4000, 36, 128, rotates=False)
    assert four(2**22 - 1, 80, 128) and not four(2**20, 80, 128)
    from test_gpu_mxfp4_kernels import ROWS

    seen = {(D.head_lanes(hd), four(t, h + 2 * kv, hd, bool(rot), axes > 1)) for h, kv, hd, rot, axes, _ in ROWS for t in (13, 1100)}
    assert seen == {(n, f) for n in (4, 8, 16, 32) for f in (False, True)}
