"""States that snws.optim.FlatMuon refuses, with nothing changed."""
import copy

import pytest
import torch

from snws.optim import FlatMuon

DEV = "cuda:0"
gpu = pytest.mark.gpu


@gpu
def test_state_without_a_step_count_changes_nothing():
    params = [torch.nn.Parameter(torch.full(s, 0.5, device=DEV)) for s in ((4, 6), (7,))]
    opt = FlatMuon(params, lr=0.02)
    for _ in range(2):
        opt.zero_grad()
        sum((p * p).sum() for p in params).backward()
        opt.step()
    kept = [t.clone() for t in (opt.exp_avg, opt.exp_avg_sq)] + [list(opt.steps)]
    sd = copy.deepcopy(opt.state_dict())
    sd["param_groups"][0]["lr"] = 9.0
    sd["state"][0]["momentum_buffer"].fill_(3.0)
    del sd["state"][1]["step"]
    with pytest.raises(ValueError, match="step"):
        opt.load_state_dict(sd)
    assert torch.equal(opt.exp_avg, kept[0]) and torch.equal(opt.exp_avg_sq, kept[1]) and opt.steps == kept[2]
    assert opt.param_groups[0]["lr"] == 0.02
