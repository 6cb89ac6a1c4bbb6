"""Refusals of the gated linear recurrence's entry points: wrong arguments raise before anything is launched."""
import pytest
import torch


def test_gated_scan_refuses():
    from cpcsv import functional as F
    p, h = torch.zeros(2, 5, 12), torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        F.gated_scan(p, h)
    with pytest.raises(ValueError, match="dimensions"):
        F.gated_scan(p[0], h)
    with pytest.raises(ValueError, match="column blocks"):
        F.gated_scan(torch.zeros(2, 5, 13), h)
    with pytest.raises(ValueError, match="column blocks"):
        F.gated_scan(torch.zeros(2, 5, 0))
    with pytest.raises(ValueError, match="column blocks"):
        F.gated_scan(torch.zeros(2, 5, 9), out_gate=False)
    with pytest.raises(TypeError, match="unsupported dtype"):
        F.gated_scan(p.half(), h)
    with pytest.raises(TypeError, match="float32"):
        F.gated_scan(p, h.bfloat16())
    with pytest.raises(ValueError, match="state must have shape"):
        F.gated_scan(p, torch.zeros(2, 5))
    with pytest.raises(ValueError, match="state must have shape"):
        F.gated_scan(p, torch.zeros(3, 4))
    with pytest.raises(TypeError, match="int32"):
        F.gated_scan(p, h, lengths=torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="lengths"):
        F.gated_scan(p, h, lengths=torch.zeros(3, dtype=torch.int32))


def test_gated_scan_step_refuses():
    from cpcsv import functional as F
    p, h = torch.zeros(2, 12), torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        F.gated_scan_step(p, h)
    with pytest.raises(ValueError, match="dimensions"):
        F.gated_scan_step(p.view(2, 1, 12), h)
    with pytest.raises(ValueError, match="state must have shape"):
        F.gated_scan_step(p, torch.zeros(2, 6))
    assert F.L.SCAN_MAX_T == 1 << 28


def test_scan_entry_points_reject_bad_arguments():
    """The C entry points answer with an error code, without a launch: unknown type, sizes, missing workspaces."""
    import os
    import re
    from cpcsv import _lib
    lib = _lib.load()
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cpcsv_hip.h")).read()
    assert int(re.search(r"#define CPCSV_SCAN_MAX_T (\d+)", header).group(1)) == _lib.SCAN_MAX_T
    assert [lib.cpcsv_scan_states(t) for t in (0, 1, 32, 33, 48, 49, _lib.SCAN_MAX_T + 1)] == [0, 0, 0, 3, 3, 4, 0]
    assert lib.cpcsv_scan_workspace(2, 32, 8, 0) == 0 and lib.cpcsv_scan_workspace(0, 64, 8, 0) == 0
    for back in (0, 1):
        n = lib.cpcsv_scan_workspace(2, 5000, 9, back)
        assert n > 2 * 9 * 8 * 5000 // 128 and n % 16 == 0
    one, odd = 0x1000, 0x1008
    fwd = lambda p=one, dt=0, y=one, ws=None, B=1, T=1: lib.cpcsv_scan_fwd(p, dt, 1, 1, None, None, y, None, None, ws, B, T, 1, 1, None)
    assert fwd(dt=7) == -1001 and fwd(B=0) == -1001 and fwd(T=0) == -1001 and fwd(T=_lib.SCAN_MAX_T + 1) == -1001
    assert fwd(p=None) == -1003 and fwd(y=None) == -1003 and fwd(T=64) == -1003 and fwd(T=64, ws=odd) == -1003
    bwd = lambda hin=one, dy=one, dp=one, ws=one, T=64: lib.cpcsv_scan_bwd(one, 0, 1, 1, None, None, hin, dy, None, dp, None, ws, 1, T, 1, 1, None)
    assert bwd(hin=None) == -1003 and bwd(ws=None) == -1003 and bwd(ws=odd) == -1003 and bwd(dy=None) == -1003 and bwd(dp=None, T=1) == -1003


def test_launches_beyond_the_grid_are_refused():
    """(2^32 threads a launch: refused before anything is started, whatever the runtime would do with them)"""
    from cpcsv import _lib
    lib = _lib.load()
    one = 0x1000
    for B, T, H in ((1 << 30, 1, 8), (1 << 22, 32, 1024), (1 << 24, 33, 1), (16, 1 << 28, 1), (1, 1 << 28, 1024)):
        assert lib.cpcsv_scan_fwd(one, 0, 1, 1, None, None, one, None, None, one, B, T, H, 1, None) == -1002, (B, T, H)
        assert lib.cpcsv_scan_bwd(one, 0, 1, 1, None, None, one, one, None, one, None, one, B, T, H, 1, None) == -1002, (B, T, H)
