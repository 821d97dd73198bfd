"""Host side of the optimiser (no GPU): refusals of the C ABI and of the Python layer, options of the optimizer."""
import copy
import ctypes
import pickle

import pytest
import torch

import flexsae_amd as flex
from flexsae_amd import _lib, optim

FAKE = 0x10000  # never dereferenced: validation fails first


def _tensor(**kw):
    fields = dict(param=FAKE, grad=FAKE, master=None, state0=FAKE, state1=FAKE, rows=4, cols=8, lr=1e-3, weight_decay=0.0, dtype=0)
    return _lib.AdamwTensor(**{**fields, **kw})


def _config(**kw):
    fields = dict(beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, max_norm=0.0, grad_norm=None, lr=None, counter=FAKE,
                  state_bits=32, flags=0)
    return _lib.AdamwConfig(**{**fields, **kw})


def _step(tensors, config, count=None):
    table = (_lib.AdamwTensor * max(1, len(tensors)))(*tensors)
    return _lib.load().flexsae_adamw_step(table, len(tensors) if count is None else count, ctypes.byref(config), None)


@pytest.mark.parametrize("change,want", [
    (dict(rows=-1), _lib.ERR_INVALID_ARGUMENT), (dict(cols=-1), _lib.ERR_INVALID_ARGUMENT), (dict(dtype=3), _lib.ERR_INVALID_ARGUMENT),
    (dict(lr=-1.0), _lib.ERR_INVALID_ARGUMENT), (dict(lr=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    (dict(weight_decay=-1.0), _lib.ERR_INVALID_ARGUMENT), (dict(param=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(grad=None), _lib.ERR_INVALID_ARGUMENT), (dict(state0=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(state1=None), _lib.ERR_INVALID_ARGUMENT), (dict(master=FAKE), _lib.ERR_INVALID_ARGUMENT),
    (dict(rows=1 << 30, cols=1 << 30), _lib.ERR_UNSUPPORTED), (dict(param=FAKE + 2), _lib.ERR_ALIGNMENT),
    (dict(grad=FAKE + 1, dtype=1), _lib.ERR_ALIGNMENT), (dict(state0=FAKE + 2), _lib.ERR_ALIGNMENT)])
def test_step_refuses_a_tensor(change, want):
    assert _step([_tensor(), _tensor(**change)], _config()) == want


@pytest.mark.parametrize("change,want", [
    (dict(counter=None), _lib.ERR_INVALID_ARGUMENT), (dict(state_bits=16), _lib.ERR_INVALID_ARGUMENT),
    (dict(beta1=1.0), _lib.ERR_INVALID_ARGUMENT), (dict(beta2=-0.5), _lib.ERR_INVALID_ARGUMENT),
    (dict(beta2=float("nan")), _lib.ERR_INVALID_ARGUMENT), (dict(eps=-1.0), _lib.ERR_INVALID_ARGUMENT),
    (dict(grad_scale=0.0), _lib.ERR_INVALID_ARGUMENT), (dict(grad_scale=float("inf")), _lib.ERR_INVALID_ARGUMENT),
    (dict(grad_scale=1e-45), _lib.ERR_INVALID_ARGUMENT), (dict(max_norm=-1.0), _lib.ERR_INVALID_ARGUMENT),
    (dict(max_norm=1.0), _lib.ERR_INVALID_ARGUMENT), (dict(flags=2), _lib.ERR_INVALID_ARGUMENT),
    (dict(counter=FAKE + 4), _lib.ERR_ALIGNMENT), (dict(lr=FAKE + 2), _lib.ERR_ALIGNMENT),
    (dict(grad_norm=FAKE + 1), _lib.ERR_ALIGNMENT)])
def test_step_refuses_a_configuration(change, want):
    assert _step([_tensor()], _config(**change)) == want


def test_step_refuses_states_of_8_bits_out_of_place():
    for change in (dict(state0=FAKE + 1), dict(state1=FAKE + 4)):
        assert _step([_tensor(**change)], _config(state_bits=8)) == _lib.ERR_ALIGNMENT
    assert _step([], _config(), count=-1) == _lib.ERR_INVALID_ARGUMENT
    assert _lib.load().flexsae_adamw_step(None, 1, ctypes.byref(_config()), None) == _lib.ERR_INVALID_ARGUMENT
    assert _lib.load().flexsae_adamw_step((_lib.AdamwTensor * 1)(_tensor()), 1, None, None) == _lib.ERR_INVALID_ARGUMENT


def test_norm_and_moments_refuse():
    lib = _lib.load()
    p = ctypes.c_void_p
    assert lib.flexsae_grad_norm_workspace_bytes(-1) == 0
    need = lib.flexsae_grad_norm_workspace_bytes(1)
    assert 0 < need <= lib.flexsae_grad_norm_workspace_bytes(1000)

    def norm(grad=FAKE, n=4, dtype=0, out=FAKE, ws=FAKE, nbytes=need, count=1):
        return lib.flexsae_grad_norm((_lib.Grad * 1)((grad, n, dtype)), count, p(out), p(ws), nbytes, None)

    assert norm(grad=None) == norm(n=-1) == norm(dtype=9) == norm(out=0) == norm(count=-1) == _lib.ERR_INVALID_ARGUMENT
    assert norm(grad=FAKE + 2) == norm(out=FAKE + 2) == _lib.ERR_ALIGNMENT
    assert norm(ws=0) == norm(ws=FAKE + 16) == norm(nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert norm(n=1 << 41) == _lib.ERR_UNSUPPORTED

    def moments(dtype=0, count=1, **kw):
        fields = dict(codes=FAKE, absmax=FAKE, exp_avg=FAKE, exp_avg_sq=FAKE, rows=1, cols=8)
        return lib.flexsae_adamw8_moments((_lib.Adamw8State * 1)(_lib.Adamw8State(**{**fields, **kw})), count, dtype, None)

    assert moments(dtype=4) == moments(rows=-1) == moments(codes=None) == moments(exp_avg=None) == _lib.ERR_INVALID_ARGUMENT
    assert moments(codes=FAKE + 1) == moments(absmax=FAKE + 4) == moments(exp_avg_sq=FAKE + 2) == _lib.ERR_ALIGNMENT
    assert moments(count=0) == _lib.OK


def test_tensors_on_the_cpu_are_refused():
    p, g = torch.ones(4, 8), torch.ones(4, 8)
    m, v = torch.zeros(4, 8), torch.zeros(4, 8)
    counter = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        flex.adamw_step([p], [g], [m], [v], counter)
    codes, absmax = flex.adamw8_state(p)
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        flex.adamw8_step([p], [g], [codes], [absmax], counter)
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        flex.grad_norm([g])
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        flex.adamw8_moments([codes], [absmax])
    opt = flex.AdamW([torch.nn.Parameter(p)])
    opt.param_groups[0]["params"][0].grad = g
    with pytest.raises(RuntimeError, match="AMD GPU only"):
        opt.state[opt.param_groups[0]["params"][0]] = {"counter": counter, "exp_avg": m, "exp_avg_sq": v}
        opt.step()


@pytest.mark.parametrize("shape,unit,want", [((4, 600), False, (1, 10, 2)), ((4, 600), True, (4, 3, 2)), ((5,), False, (1, 1, 2)),
                                             ((2, 3, 256), True, (6, 1, 2)), ((0, 7), True, (0, 1, 2)), ((3, 0), True, (0, 0, 2))])
def test_new_states_of_8_bits(shape, unit, want):
    codes, absmax = flex.adamw8_state(torch.zeros(shape, dtype=torch.bfloat16), unit)
    assert codes.shape == (*shape, 2) and codes.dtype == torch.uint8 and tuple(absmax.shape) == want and not absmax.any()


@pytest.mark.parametrize("kw", [dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(lr=-1.0),
                                dict(max_norm=0.0), dict(unit_rows=True)])
def test_options_that_are_refused(kw):
    with pytest.raises(ValueError):
        flex.AdamW([torch.nn.Parameter(torch.ones(3))], **kw)


def test_copies_keep_the_options_and_states_of_others_are_refused():
    p = torch.nn.Parameter(torch.ones(3, 4))
    opt = flex.AdamW([p], lr=0.5, state_bits=8, max_norm=2.0, skip_nonfinite=True)
    for again in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert again.max_norm == 2.0 and again.skip_nonfinite and again.grad_norm is None
        assert again.param_groups[0]["state_bits"] == 8 and again.param_groups[0]["lr"] == 0.5
    its = torch.optim.AdamW([p])
    p.grad = torch.ones(3, 4)
    its.step()
    with pytest.raises(ValueError, match="not those of this optimizer"):
        opt.load_state_dict(its.state_dict())


def test_masters_follow_parameters_that_were_changed_from_outside():
    p = torch.nn.Parameter(torch.ones(3, 4, dtype=torch.bfloat16))
    opt = flex.AdamW([p])
    opt.state[p] = opt._new_state(p, opt.param_groups[0], torch.zeros(2, dtype=torch.int64))
    with torch.no_grad():
        p.mul_(3.0)
    opt.reset_masters()
    assert torch.equal(opt.state[p]["master"], torch.full((3, 4), 3.0))


def test_fake_kernels():
    meta = lambda *s, dt=torch.float32: torch.empty(*s, dtype=dt, device="meta")
    assert optim._grad_norm_op([meta(3, dt=torch.bfloat16)]).shape == ()
    m, v = optim._moments_op([meta(3, 5, 2, dt=torch.uint8)], [meta(1, 1, 2)], torch.bfloat16)
    assert m.shape == v.shape == (3, 5) and m.dtype == torch.bfloat16
