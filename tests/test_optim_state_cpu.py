"""Loading state into the multi-tensor AdamW: what is refused on the CPU, and that nothing has changed then."""
import pytest
import torch


def test_state_for_parameters_on_the_cpu_is_refused_before_anything_changes():
    from nvfp4_sm120_b200._lib import NVFP4Error
    from nvfp4_sm120_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    other = torch.optim.AdamW([p], lr=0.5)
    other.step()
    opt = AdamW([p], lr=0.1)
    with pytest.raises(NVFP4Error, match="CUDA"):
        opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] == 0.1 and not opt.state
    opt.load_state_dict({"state": {}, "param_groups": other.state_dict()["param_groups"]})      # nothing to place
    assert opt.param_groups[0]["lr"] == 0.5


def test_groups_that_do_not_match_are_refused_before_anything_changes():
    from nvfp4_sm120_b200.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(4)) for _ in range(2))
    opt = AdamW([p], lr=0.1)
    for other in (torch.optim.AdamW([p, q], lr=0.5), torch.optim.AdamW([{"params": [p]}, {"params": [q]}], lr=0.5)):
        with pytest.raises(ValueError):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 0.1 and not opt.state
