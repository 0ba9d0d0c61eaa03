"""Calls of more threads than a grid dimension holds are refused where the
kernel has one row of workgroups only (no GPU: nothing is launched)."""

from __future__ import annotations

import ctypes

from mlx_lean_moe_amd import _lib


def _p(i):
    return ctypes.c_void_p(1 << (20 + i))


def _refused(rc, who):
    err = _lib.load().gdn_last_error().decode()
    assert rc == _lib.GDN_EINVAL and who in err and "exceed" in err, (rc, err)


def test_scans_refuse_more_workgroups_than_a_grid_row():
    """8 rows of 2^24 heads (one workgroup of 256 threads each), and 2^32 rows."""
    scan = lambda f, N, Dv: f(_p(0), _p(1), 0, _p(2), 0, _p(3), 0, _p(4), 0, _p(5), _p(6), 0, _p(7), 0, None, N, N, 1, 64,
                              32, Dv, None)
    _refused(scan(_lib.load().gdn_scan, 1 << 18, 8), "gdn_scan")
    _refused(scan(_lib.load().gdn_scan_reference, 1 << 23, 8), "gdn_scan_reference")


def test_frontend_refuses_more_tokens_than_a_grid_row():
    rc = _lib.load().gdn_frontend(_p(0), 24, _p(10), _p(17), 0, _p(3), None, 1, 1 << 24, _p(4), _p(5), _p(6), 1, 1, 8, 8,
                                  4, 0, None)
    _refused(rc, "gdn_frontend")
