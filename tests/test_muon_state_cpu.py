"""What the Muon optimizer takes for a saved state, without a device."""
import copy

import pytest
import torch

from paralleltnnlayers_amd import optim


def params(dtype=torch.float32):
    return [torch.nn.Parameter(torch.randn(4, 6, generator=torch.Generator().manual_seed(i)).to(dtype)) for i in range(2)]


def state(lr=0.5):
    opt = optim.Muon(params(), lr=lr)
    for p in opt.param_groups[0]["params"]:
        opt.state[p]["momentum_buffer"] = torch.ones(4, 6)
    return copy.deepcopy(opt.state_dict())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_states_keep_their_type(dtype):
    opt = optim.Muon(params(dtype))
    opt.load_state_dict(state())
    assert opt.param_groups[0]["lr"] == 0.5
    for p in opt.param_groups[0]["params"]:
        assert opt.state[p]["momentum_buffer"].dtype == torch.float32 and (opt.state[p]["momentum_buffer"] == 1).all()
        assert ("master" in opt.state[p]) == (dtype != torch.float32)


def test_refused_states_leave_the_optimizer_as_it_is():
    def without_momentum(s):
        del s["state"][1]["momentum_buffer"]
        s["state"][1]["exp_avg"] = torch.zeros(4, 6)

    def of_none(s):
        s["state"][0]["momentum_buffer"] = None

    def of_no_group(s):
        s["state"][9] = {"exp_avg": torch.zeros(4, 6)}

    def without_settings(s):
        del s["param_groups"][0]["steps"]
    for change in (without_momentum, of_none, of_no_group, without_settings):
        opt, bad = optim.Muon(params(), lr=0.1), state()
        opt.state[opt.param_groups[0]["params"][0]]["momentum_buffer"] = torch.full((4, 6), 3.0)
        change(bad)
        with pytest.raises(ValueError, match="Muon"):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == 0.1 and len(opt.state) == 1
        assert (opt.state[opt.param_groups[0]["params"][0]]["momentum_buffer"] == 3).all()
