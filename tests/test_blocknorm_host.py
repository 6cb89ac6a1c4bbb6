"""Refusals of the block norms' entry points: wrong arguments raise before anything is launched."""
import pytest
import torch


def test_norm_residual_refuses():
    from cpcsv import functional as F
    x, w = torch.zeros(2, 5, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU only"):
        F.norm_residual(x, x, w)
    with pytest.raises(TypeError, match="unsupported dtype"):
        F.norm_residual(x.half(), x.half(), w)
    with pytest.raises(TypeError, match="bfloat16 residual stream"):
        F.norm_residual(x.bfloat16(), x, w)
    with pytest.raises(ValueError, match="x's shape"):
        F.norm_residual(x, x[:1], w)
    with pytest.raises(TypeError, match="w_post must be float32"):
        F.norm_residual(x, x, w.bfloat16())
    with pytest.raises(TypeError, match="w_post must be given"):
        F.norm_residual(x, x, None)
    for bad in (dict(w_post=torch.ones(7)), dict(w_post=w, scale=torch.ones(1)), dict(w_post=w, w_next=torch.ones(1, 8))):
        with pytest.raises(ValueError, match="must have shape"):
            F.norm_residual(x, x, **bad)
    with pytest.raises(TypeError, match="gate must have"):
        F.norm_residual(x, x, w, gate=x.bfloat16())
    for shape in ((2, 5, 1), (2, 1, 1), (5, 8), (1, 5, 8), (8,)):
        with pytest.raises(ValueError, match="gate must have"):
            F.norm_residual(x, x, w, gate=torch.zeros(shape))
    with pytest.raises(ValueError, match="two dimensions"):
        F.norm_residual(x[0, 0], x[0, 0], w, gate=x[0, 0])
    with pytest.raises(ValueError, match="rows of"):
        F.norm_residual(torch.zeros(2, 0), torch.zeros(2, 0), torch.ones(0))
    with pytest.raises(ValueError, match="rows of"):
        F.norm_residual(torch.zeros(1, 16385), torch.zeros(1, 16385), torch.ones(16385))


def test_rms_norm_refuses():
    from cpcsv import functional as F
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU only"):
        F.rms_norm(x, w)
    with pytest.raises(TypeError, match="out_dtype"):
        F.rms_norm(x.bfloat16(), w, out_dtype=torch.float32)
    with pytest.raises(TypeError, match="out_dtype"):
        F.rms_norm(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="must have shape"):
        F.rms_norm(x, torch.ones(9))
    with pytest.raises(ValueError, match="rows of"):
        F.rms_norm(torch.zeros(()), w)


def test_entry_points_reject_bad_arguments():
    """Error codes of the C entry points, without a launch."""
    import os
    import re
    from cpcsv import _lib
    lib = _lib.load()
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cpcsv_hip.h")).read()
    assert int(re.search(r"#define CPCSV_NORM_MAX_D (\d+)", header).group(1)) == _lib.NORM_MAX_D
    p = 0x1000
    fwd = lambda x=p, u=p, gate=None, wp=p, wn=p, rows=4, d=8, xdt=0, udt=0, mode=0, t=1, xo=p, z=p: lib.cpcsv_norm_residual_fwd(
        x, u, gate, None, wp, wn, xo, z, p, p, rows, d, xdt, udt, mode, t, 1e-6, None)
    assert fwd(xdt=1, udt=0) == -1001 and fwd(udt=5) == -1001
    assert fwd(rows=0) == -1002 and fwd(d=0) == -1002 and fwd(d=16385) == -1002 and fwd(mode=3) == -1002
    assert fwd(mode=2, gate=p, rows=(1 << 30) + 1) == -1002
    assert fwd(mode=2, gate=p, t=3) == -1002 and fwd(mode=2, gate=p, t=0) == -1002
    assert fwd(x=None) == -1003 and fwd(wp=None) == -1003 and fwd(mode=1) == -1003 and fwd(u=None, wn=None) == -1003 and fwd(xo=None) == -1003 and fwd(z=None) == -1003
    bwd = lambda dx=p, part=p, dz=p, rx=p: lib.cpcsv_norm_residual_bwd(p, p, None, None, p, p, p, rx, p, dz, dx, p, None, None, p, p, part,
                                                                       4, 8, 0, 0, 0, 1, None)
    assert bwd(dx=None) == -1003 and bwd(part=None) == -1003 and bwd(rx=None) == -1003
    assert lib.cpcsv_norm_residual_part(0, 8, 0, 1) == 0 and lib.cpcsv_norm_residual_part(100, 8, 2, 10) >= 10 * 8
