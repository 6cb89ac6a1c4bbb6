"""Refusals of the orthogonalised update's entry points: wrong arguments raise before anything is launched."""
import ctypes as C

import pytest
import torch


def test_orthogonalize_refuses():
    from cpcsv.optim import orthogonalize
    g = torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="GPU only"):
        orthogonalize(g)
    with pytest.raises(ValueError, match="expects"):
        orthogonalize(g[0])
    with pytest.raises(ValueError, match="expects"):
        orthogonalize(g.view(1, 1, 4, 6))
    with pytest.raises(TypeError, match="unsupported dtype"):
        orthogonalize(g.half())
    for steps in (0, -1, 2.5):
        with pytest.raises(ValueError, match="steps"):
            orthogonalize(g, steps=steps)
    for eps in (-1e-9, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            orthogonalize(g, eps=eps)
    with pytest.raises(ValueError, match="sides of"):
        orthogonalize(torch.zeros(0, 4))
    with pytest.raises(ValueError, match="sides of"):
        orthogonalize(torch.zeros(1, 131073))
    with pytest.raises(ValueError, match="sides of"):
        orthogonalize(torch.zeros(1, 1).expand(16385, 16385))


def test_muon_refuses():
    from cpcsv.optim import FusedMuon
    w = torch.nn.Parameter(torch.zeros(4, 6))
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(eps=-1.0), dict(steps=0), dict(steps=1.5),
                dict(lr=float("nan"))):
        with pytest.raises(ValueError, match="FusedMuon"):
            FusedMuon([w], **bad)
    with pytest.raises(ValueError, match="vectors to FusedAdam"):
        FusedMuon([w, torch.nn.Parameter(torch.zeros(6))])
    with pytest.raises(ValueError, match="sides of"):
        FusedMuon([torch.nn.Parameter(torch.zeros(0, 6))])
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="twice"):
        FusedMuon([w, w])
    w.grad = torch.zeros_like(w)
    with pytest.raises(RuntimeError, match="contiguous fp32 GPU"):
        FusedMuon([w]).step()


def test_entry_points_reject_bad_arguments():
    """Error codes of the C entry points, without a launch; the constants of the header."""
    import os
    import re
    from cpcsv import _lib
    lib = _lib.load()
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "cpcsv_hip.h")).read()
    val = lambda n: int(re.search(r"#define %s (\d+)" % n, header).group(1))
    assert (val("CPCSV_ORTH_JOBS"), val("CPCSV_ORTH_MAX_SIDE"), val("CPCSV_ORTH_MAX_MIN")) == (_lib.ORTH_JOBS, _lib.ORTH_MAX_SIDE, _lib.ORTH_MAX_MIN)
    dims = lambda *v: (C.c_long * len(v))(*v)
    assert lib.cpcsv_orth_workspace(dims(3, 5), 0) == -1001 and lib.cpcsv_orth_workspace(dims(3, 5), 17) == -1001
    assert lib.cpcsv_orth_workspace(dims(0, 5), 1) == -1002 and lib.cpcsv_orth_workspace(dims(3, 131073), 1) == -1002
    assert lib.cpcsv_orth_workspace(dims(16385, 16385), 1) == -1002
    assert lib.cpcsv_orth_workspace(dims(3, 5, 300, 200), 2) > lib.cpcsv_orth_workspace(dims(300, 200), 1) > 0
    ptrs = (C.c_void_p * 1)(0x1000)
    none = (C.c_void_p * 1)(None)
    assert lib.cpcsv_orthogonalize(ptrs, ptrs, dims(3, 5), 1, 9, 5, 0.0, 0x1000, None) == -1001
    assert lib.cpcsv_orthogonalize(ptrs, ptrs, dims(3, 5), 1, 0, 0, 0.0, 0x1000, None) == -1001
    assert lib.cpcsv_orthogonalize(ptrs, none, dims(3, 5), 1, 0, 5, 0.0, 0x1000, None) == -1003
    assert lib.cpcsv_orthogonalize(ptrs, ptrs, dims(3, 5), 1, 0, 5, 0.0, None, None) == -1003
    assert lib.cpcsv_muon_step(ptrs, ptrs, none, dims(3, 5), 1, 0x1000, 0.9, 1, 0.0, 5, 0.0, 0x1000, None) == -1003
    assert lib.cpcsv_muon_step(ptrs, ptrs, ptrs, dims(3, 5), 1, None, 0.9, 1, 0.0, 5, 0.0, 0x1000, None) == -1003
