"""The rules of the 4-bit operators' launchers, on the host."""
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
