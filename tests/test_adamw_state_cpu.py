"""What the AdamW optimizer makes of saved states, without a device (a state is tensors wherever they lie)."""
import copy
import io

import pytest
import torch

from paralleltnnlayers_amd import optim


def params(*sizes, dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    return [torch.nn.Parameter(torch.randn(n, generator=gen).to(dtype)) for n in sizes]


def torch_state(P, have, **kw):
    """A state of torch's AdamW in which parameter i has stepped have[i] times."""
    opt = torch.optim.AdamW(P, lr=1e-3, **kw)
    for t in range(max(have)):
        for p, n in zip(P, have):
            p.grad = torch.ones_like(p) if t < n else None
        opt.step()
    return opt.state_dict()


def test_a_state_of_torchs_optimizer():
    P = params(5, 6, 7)
    state = torch_state(P, (4, 4, 2))
    opt = optim.AdamW(P)
    opt.load_state_dict(state)
    for p, n in zip(P, (4, 4, 2)):
        s = opt.state[p]
        assert set(s) == {"exp_avg", "exp_avg_sq", "counter"}
        assert s["counter"].dtype == torch.float64
        assert s["counter"].tolist() == [n, 0.9 ** n, 0.999 ** n, 0.0]
    a, b, c = (opt.state[p]["counter"] for p in P)
    assert a is b and a is not c                                     # (one launch for those that go on together)


def test_a_16_bit_state_of_torchs_optimizer():
    P = params(5, dtype=torch.bfloat16)
    state = torch_state(P, (3,))
    assert state["state"][0]["exp_avg"].dtype == torch.bfloat16
    for masters in (True, False):
        opt = optim.AdamW(P, masters=masters)
        opt.load_state_dict(state)
        s = opt.state[P[0]]
        assert s["exp_avg"].dtype == s["exp_avg_sq"].dtype == torch.float32
        assert ("master" in s) == masters
        if masters:
            assert torch.equal(s["master"], P[0].detach().float())


def our_state(P, counts, bits=32):
    """A state of this optimizer: parameter i with counts[i] (the same object: stepped together so far)."""
    opt = optim.AdamW(P, state_bits=bits, min_8bit_size=1)
    for p, c in zip(P, counts):
        opt._state(p)["counter"] = c
    return opt


@pytest.mark.parametrize("how", ["as it is", "deepcopy", "file"])
@pytest.mark.parametrize("bits", [32, 8])
def test_counts_that_are_shared_stay_shared(bits, how):
    P = params(5, 300, 7)
    two, one = (torch.tensor([n, 0.9 ** n, 0.999 ** n, 0.0], dtype=torch.float64) for n in (2, 1))
    state = our_state(P, (two, two, one), bits).state_dict()
    if how == "deepcopy":
        state = copy.deepcopy(state)
    elif how == "file":
        room = io.BytesIO()
        torch.save(state, room)
        room.seek(0)
        state = torch.load(room, weights_only=True)
    Q = params(5, 300, 7)
    opt = optim.AdamW(Q, state_bits=bits, min_8bit_size=1)
    opt.load_state_dict(state)
    a, b, c = (opt.state[q]["counter"] for q in Q)
    assert a is b and a is not c and a is not two
    assert a.tolist() == two.tolist() and c.tolist() == one.tolist()
    assert opt.state[Q[1]]["exp_avg"].dtype == (torch.int8 if bits == 8 else torch.float32)


def test_a_state_with_a_count_for_each_group():
    """As they were saved before parameters had counts of their own."""
    P = params(5, 6)
    count = torch.tensor([7, 0.9 ** 7, 0.999 ** 7, 0.0], dtype=torch.float64)
    state = our_state(P, (count, count)).state_dict()
    for s in state["state"].values():
        del s["counter"]
    state["param_groups"][0]["counter"] = count
    opt = optim.AdamW(params(5, 6))
    opt.load_state_dict(state)
    (group,) = opt.param_groups
    a, b = (opt.state[p]["counter"] for p in group["params"])
    assert a is b and a.tolist() == count.tolist() and "counter" not in group


def test_states_that_are_refused():
    P = params(5, 6)
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError, match="amsgrad or maximize"):
            optim.AdamW(P).load_state_dict(torch_state(P, (1, 1), **kw))
    opt = optim.AdamW(P)
    bare = torch_state(P, (1, 1))
    for s in bare["state"].values():
        del s["step"]
    with pytest.raises(ValueError, match="without a count"):
        opt.load_state_dict(bare)
    assert not opt.state                                             # (refused before anything is taken)


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_copies_of_the_optimizer(how):
    """A copy has the optimizer's settings and its state, counts still shared."""
    import pickle
    P = params(5, 300)
    count = torch.tensor([2, 0.9 ** 2, 0.999 ** 2, 0.0], dtype=torch.float64)
    opt = our_state(P, (count, count), bits=8)
    opt.max_norm, opt.masters = 2.0, False
    new = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    assert (new.state_bits, new.min_8bit_size, new.masters, new.max_norm, new.last_norm) == (8, 1, False, 2.0, None)
    a, b = (new.state[p]["counter"] for p in new.param_groups[0]["params"])
    assert a is b and a is not count and a.tolist() == count.tolist()
    assert callable(new.step) and new.state_dict()["param_groups"] == opt.state_dict()["param_groups"]


def test_a_state_of_no_group():
    """One that belongs to no parameter of a group, and has no count: refused like any other."""
    P = params(5)
    state = our_state(P, (torch.zeros(4, dtype=torch.float64),)).state_dict()
    state["state"][9] = {"exp_avg": torch.zeros(5), "exp_avg_sq": torch.zeros(5)}
    with pytest.raises(ValueError, match="without a count"):
        optim.AdamW(params(5)).load_state_dict(state)
