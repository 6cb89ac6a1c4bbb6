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
