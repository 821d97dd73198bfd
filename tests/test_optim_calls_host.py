"""Host side of calls of the optimiser (no GPU): checks without a step."""
import ctypes

import pytest
import torch

import flexsae_amd as flex
from flexsae_amd import _lib
from tests.test_optim_host import FAKE, _config, _step, _tensor


@pytest.mark.parametrize("tensor,config", [
    (dict(rows=-1), {}), (dict(lr=-1.0), {}), (dict(param=None), {}), (dict(rows=1 << 30, cols=1 << 30), {}), (dict(grad=FAKE + 2), {}),
    ({}, dict(beta1=1.0)), ({}, dict(state_bits=16)), ({}, dict(max_norm=1.0)), ({}, dict(flags=2)), ({}, dict(counter=FAKE + 4)),
    (dict(state1=FAKE + 4), dict(state_bits=8))])
def test_a_check_refuses_what_a_step_does(tensor, config):
    lib = _lib.load()
    tensors, config = [_tensor(), _tensor(**tensor)], _config(**config)
    table = (_lib.AdamwTensor * 2)(*tensors)
    status = lib.flexsae_adamw_check(table, 2, ctypes.byref(config))
    assert status != _lib.OK and status == _step(tensors, config)


def test_a_check_launches_nothing():
    """(the addresses are none)"""
    lib = _lib.load()
    for bits, flags in ((32, 0), (8, 0), (32, _lib.ADAMW_UNIT_ROWS), (8, _lib.ADAMW_UNIT_ROWS)):
        table = (_lib.AdamwTensor * 2)(_tensor(), _tensor(rows=0, param=None))
        assert lib.flexsae_adamw_check(table, 2, ctypes.byref(_config(state_bits=bits, flags=flags))) == _lib.OK
    assert lib.flexsae_adamw_check(None, 0, ctypes.byref(_config())) == _lib.OK
    assert lib.flexsae_adamw_check(None, 1, ctypes.byref(_config())) == _lib.ERR_INVALID_ARGUMENT


def test_asking_for_moments_before_a_step_begins_no_state():
    p = torch.nn.Parameter(torch.ones(3))
    opt = flex.AdamW([p])
    with pytest.raises(KeyError, match="not been stepped"):
        opt.moments(p)
    assert not opt.state
    opt.load_state_dict(opt.state_dict())


def _stepped(dtype=torch.bfloat16):
    """An optimizer as after a step (no GPU)."""
    params = [torch.nn.Parameter(torch.ones(n, 4, dtype=dtype)) for n in (2, 3)]
    opt = flex.AdamW(params)
    counter = torch.tensor([5, 0])
    for i, p in enumerate(params):
        opt.state[p] = opt._new_state(p, opt.param_groups[0], counter)
        opt.state[p]["exp_avg"].fill_(1.0 + 2.0 ** -20 + i)
    return opt


def test_hooks_of_loading_states():
    one, two = _stepped(), _stepped()
    seen = []

    def before(opt, state_dict):
        seen.append("before")
        state = {k: {**s, "exp_avg": s["exp_avg"] * 2} for k, s in state_dict["state"].items()}
        return {**state_dict, "state": state}

    def after(opt):
        seen.append(float(opt.state[opt.param_groups[0]["params"][1]]["exp_avg"][0, 0]))

    two.register_load_state_dict_pre_hook(before)
    two.register_load_state_dict_post_hook(after)
    for _ in range(2):
        two.load_state_dict(one.state_dict())
    assert seen == ["before", 2 * (2 + 2.0 ** -20)] * 2
    first, second = two.param_groups[0]["params"]
    assert float(two.state[first]["exp_avg"][0, 0]) == 2 * (1 + 2.0 ** -20)
    assert two.state[first]["exp_avg"].dtype == torch.float32 and two.state[first]["master"].dtype == torch.float32
    assert two.state[first]["counter"] is two.state[second]["counter"] and two.state[first]["counter"].tolist() == [5, 0]


def test_a_refused_load_leaves_the_states():
    one, its = _stepped(), torch.optim.AdamW([torch.nn.Parameter(torch.ones(n, 4)) for n in (2, 3)])
    for p in its.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    its.step()
    state, groups = dict(one.state), [dict(g) for g in one.param_groups]
    with pytest.raises(ValueError, match="not those of this optimizer"):
        one.load_state_dict(its.state_dict())
    assert dict(one.state) == state and [dict(g) for g in one.param_groups] == groups
    one.load_state_dict(_stepped().state_dict())  # (and the next one is loaded)
    assert one.state[one.param_groups[0]["params"][0]]["counter"].tolist() == [5, 0]


def test_options_of_another_optimizer_are_refused():
    """Its states are none yet: its groups would leave this one without options."""
    its = torch.optim.AdamW([torch.nn.Parameter(torch.ones(n, 4)) for n in (2, 3)])
    one = _stepped()
    state, groups = dict(one.state), [dict(g) for g in one.param_groups]
    with pytest.raises(ValueError, match="not those of this optimizer"):
        one.load_state_dict(its.state_dict())
    assert dict(one.state) == state and [dict(g) for g in one.param_groups] == groups
    fresh = flex.AdamW([torch.nn.Parameter(torch.ones(n, 4)) for n in (2, 3)], lr=0.5, state_bits=8)
    one.load_state_dict(fresh.state_dict())
    assert one.param_groups[0]["state_bits"] == 8 and one.param_groups[0]["lr"] == 0.5 and not one.state


def test_a_parameter_twice_in_a_group_is_refused():
    """(Between groups torch refuses it.)"""
    p, q = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning):
        flex.AdamW([p, q, p])
    opt = flex.AdamW([q])
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning):
        opt.add_param_group({"params": [p, p]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [p]})
