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
