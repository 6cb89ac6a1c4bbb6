"""Refusals of the orthogonalised optimiser beside the ordinary ones: what they leave behind, and what they name. No GPU."""
import pytest
import torch


def test_a_refused_group_is_not_kept():
    from cpcsv.optim import FusedMuon
    w, other = torch.nn.Parameter(torch.zeros(4, 6)), torch.nn.Parameter(torch.zeros(3, 5))
    opt = FusedMuon([w])
    for bad in ([torch.nn.Parameter(torch.zeros(6))], [other, torch.nn.Parameter(torch.zeros(2, 0))], [torch.nn.Parameter(torch.zeros(131073, 1))]):
        with pytest.raises(ValueError):
            opt.add_param_group({"params": bad})
        assert len(opt.param_groups) == 1 and opt.param_groups[0]["params"] == [w]
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="twice"):
        opt.add_param_group({"params": [other, other]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [other], "lr": 0.1})              # (free to join: the refused groups left no trace)
    assert len(opt.param_groups) == 2 and opt.state_dict()["param_groups"][1]["lr"] == 0.1


def test_weights_of_a_deferred_update_are_named():
    """GANTrainer's larger weights have no gradient of their own (FusedAdam.attach_layer: it stays in the layer's accumulator)."""
    from cpcsv.dist import GradBucket
    from cpcsv.optim import FusedMuon
    w = torch.nn.Parameter(torch.zeros(4, 6))
    GradBucket([w, torch.nn.Parameter(torch.zeros(3))]).adopt(retired=[w])
    with pytest.raises(RuntimeError, match="deferred update"):
        FusedMuon([w]).step()


def test_weights_that_share_memory_are_refused():
    """Matrices of a group are updated at once: two that overlap (a tied weight held twice, a slice of another) would race. Neighbours in
    one buffer do not overlap."""
    from cpcsv.optim import FusedMuon
    base = torch.zeros(10, 6)
    held = lambda *views: [torch.nn.Parameter(v) for v in views]
    for params in (held(base, base), held(base, base[3:5]), held(base[4:], base[:5])):
        for p in params:
            p.grad = torch.zeros_like(p)
        with pytest.raises(RuntimeError, match="share memory"):
            FusedMuon(params).step()
        params[1].grad = None                                        # (only one of them moves)
        with pytest.raises(RuntimeError, match="contiguous fp32 GPU"):
            FusedMuon(params).step()
    apart = held(base[5:], base[:5])
    for p in apart:
        p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="contiguous fp32 GPU"):
        FusedMuon(apart).step()
