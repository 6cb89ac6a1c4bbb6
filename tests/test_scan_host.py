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


def test_scan_entry_points_reject_bad_arguments():
    """The C entry points answer with an error code, without a launch: unknown type, sizes, missing workspaces."""
    from cpcsv import _lib
    lib = _lib.load()
    assert [lib.cpcsv_scan_chunks(t) for t in (0, 1, 32, 33, 64, 65)] == [0, 1, 1, 2, 2, 3]
    one = 0x1000
    assert lib.cpcsv_scan_fwd(one, 7, 1, 1, None, None, one, None, None, None, 1, 1, 1, 1, None) == -1001
    assert lib.cpcsv_scan_fwd(one, 0, 1, 1, None, None, one, None, None, None, 0, 1, 1, 1, None) == -1001
    assert lib.cpcsv_scan_fwd(None, 0, 1, 1, None, None, one, None, None, None, 1, 1, 1, 1, None) == -1003
    assert lib.cpcsv_scan_fwd(one, 0, 1, 1, None, None, one, None, None, None, 1, 64, 1, 1, None) == -1003
    assert lib.cpcsv_scan_bwd(one, 0, 1, 1, None, None, None, one, None, one, None, None, None, 1, 64, 1, 1, None) == -1003
    assert lib.cpcsv_scan_bwd(one, 0, 1, 1, None, None, None, None, None, one, None, None, None, 1, 1, 1, 1, None) == -1003
