"""The sizes that the GPU tests of the scan's and the 8-bit product's layouts
run take the layouts that they are there for (no GPU)."""

from __future__ import annotations

from . import plans


def test_scan_layouts():
    got = plans.scan_plans([c[:3] for c in plans.SCAN_LAYOUTS])
    wrong = [(c, g) for c, g in zip(plans.SCAN_LAYOUTS, got) if c[3] != g]
    assert not wrong, wrong
    for bf16 in (True, False):
        mine = [c for c in plans.SCAN_LAYOUTS if c[0] == bf16]
        assert {c[3][:2] for c in mine} == {(1, 4), (2, 4), (1, 8), (2, 8)}
        # wide workgroups with each width of state that a kernel is built for, in segments
        assert {max(32, 1 << (c[2][3] - 1).bit_length()) for c in mine if c[3][1] == 8 and c[3][2]} == {32, 64, 128, 256}
        assert any(len(c[1]) > 64 and c[3][2] for c in mine) and any(c[2][1] % 64 for c in mine if c[3][1] == 8)


def test_fp8_layouts():
    got = plans.fp8_plans([c[:4] for c in plans.FP8_LAYOUTS])
    wrong = [(c, g) for c, g in zip(plans.FP8_LAYOUTS, got) if c[4] != g]
    assert not wrong, wrong
    tiles = lambda exact: {launch.split(":")[1].split("/")[0] for c in plans.FP8_LAYOUTS if c[0] == exact for launch in c[4]}
    assert tiles(False) == {"64x32", "64x64", "128x256", "256x256"} and tiles(True) == {"64x32", "64x64", "128x128"}


def test_every_product_has_a_grid():
    """Large products leave tiles whose grid would hold 2^32 threads and more."""
    for exact, sizes in ((False, ((1 << 28, 129, 16), (1 << 28, 256, 128), (1, 1 << 30, 16))),
                         (True, ((1 << 28, 193, 16), (1 << 27, 500, 128)))):
        for M, N, K in sizes:
            (plan,) = plans.fp8_plans([(exact, M, N, K)])
            if plan == ["skinny"]:
                continue
            for launch in plan:
                cols, tile = launch.split(":")
                tn, tm = map(int, tile.split("/")[0].split("x"))
                threads = -(-int(cols) // tn) * -(-M // tm) * (512 if tm == 256 else 256)
                assert threads < 1 << 32, (exact, M, N, K, plan)
