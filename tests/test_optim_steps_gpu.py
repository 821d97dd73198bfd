"""Steps of the optimiser as programs make them."""
import pytest
import torch

import flexsae_amd as flex
from tests.test_optim_gpu import BF16, DEV, F16, F32, Problem, _model, _set_grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtypes", [[F32, F32], [BF16, F32, F16, F32], [F16, BF16]], ids=str)
@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_a_compiled_step_with_masters_of_fp32_parameters(bits, dtypes, backend):
    """The entry of an fp32 parameter is ignored, the parameter itself in that place too."""
    torch._dynamo.reset()  # (compilations of other cases count)
    a, b = (Problem([(30, 40 + i) for i in range(len(dtypes))], dtypes, bits, seed=21) for _ in range(2))

    @torch.compile(fullgraph=True, backend=backend)
    def compiled(params, grads, s0, s1, masters, counter):
        (flex.adamw_step if bits == 32 else flex.adamw8_step)(params, grads, s0, s1, counter, masters=masters, lr=1e-2)

    for p in (a, b):
        p.master = True
        p.masters = [w if w.dtype == F32 else m for w, m in zip(p.params, p.masters)]
    start = [w.clone() for w in a.params]
    for _ in range(2):
        a.step(lr=1e-2)
        compiled(b.params, b.grads, b.s0, b.s1, b.masters, b.counter)
        for x, y in zip(a.tensors(), b.tensors()):
            assert torch.equal(x, y)
    assert not any(torch.equal(x, y) for x, y in zip(start, b.params))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtypes", [[F32] * 4, [BF16, F32, F32, BF16]], ids=str)
def test_a_compiled_step_of_the_optimizer(bits, dtypes):
    torch._dynamo.reset()
    models = [[torch.nn.Parameter(p.detach().to(d)) for p, d in zip(_model(), dtypes)] for _ in range(2)]
    opts = [flex.AdamW([{"params": m[:1], "unit_rows": True}, {"params": m[1:]}], lr=1e-2, state_bits=bits, max_norm=0.1) for m in models]
    compiled = torch.compile(opts[1].step, backend="aot_eager")
    for i in range(3):
        for m in models:
            _set_grads(m, i)
        opts[0].step()
        compiled()
        for x, y in zip(*models):
            assert torch.equal(x, y)
            for k, s in opts[0].state[x].items():
                assert torch.equal(s, opts[1].state[y][k]), k


def test_a_step_within_a_compiled_function():
    """... with its closure, hooks that run once, and the norm for the caller."""
    torch._dynamo.reset()
    a, b = _model(), _model()
    mine, its = flex.AdamW(a, lr=1e-2, max_norm=0.5), flex.AdamW(b, lr=1e-2, max_norm=0.5)

    def one(opt, params):
        def loss():
            opt.zero_grad()
            total = sum((p * p).sum() for p in params)
            total.backward()
            return total.detach()
        return opt.step(loss, grad_scale=2.0) + opt.grad_norm

    ran = []
    its.register_step_pre_hook(lambda *_: ran.append("before"))
    its.register_step_post_hook(lambda *_: ran.append("after"))
    compiled = torch.compile(one, backend="aot_eager")
    for _ in range(3):
        # (the loss and its gradients may be summed in another order)
        assert torch.allclose(one(mine, a), compiled(its, b), rtol=1e-5)
        for x, y in zip(a, b):
            assert torch.allclose(x, y, rtol=1e-4, atol=1e-5)
    assert ran == ["before", "after"] * 3


@pytest.mark.parametrize("bits", [32, 8])
def test_the_ops_with_masters_pass_torchs_own_checks(bits):
    p = Problem([(20, 30), (30,), (7, 9)], [F16, F32, BF16], bits, master=True)
    op = torch.ops.flexsae_amd.adamw_step_ if bits == 32 else torch.ops.flexsae_amd.adamw8_step_
    torch.library.opcheck(op.default, (p.params, p.grads, p.s0, p.s1, [p.masters[0], p.masters[2]], p.counter, [1e-3] * 3, [0.0] * 3, None,
                                       None, 0.9, 0.999, 1e-8, 1.0, 0.0, False))


def test_the_op_takes_masters_of_16_bit_parameters_alone():
    p = Problem([(20, 30), (30,)], [F16, F32], 32, master=True)
    for masters in (p.masters, [p.masters[1]]):
        with pytest.raises(ValueError, match="master"):
            torch.ops.flexsae_amd.adamw_step_(p.params, p.grads, p.s0, p.s1, masters, p.counter, [1e-3] * 2, [0.0] * 2, None, None, 0.9, 0.999,
                                              1e-8, 1.0, 0.0, False)


# ---- numbers whose reading runs Python code ------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_numbers_that_change_the_lists_as_they_are_read(bits):
    for where in ("lr", "weight_decay"):
        p = Problem([(20, 30), (30,)], F32, bits)
        kept = [*p.params, *p.s0, *p.s1]
        before = [x.clone() for x in (*kept, p.counter)]

        class Clearing:
            def __float__(self):
                for x in (p.params, p.grads, p.s0, p.s1):
                    x.clear()
                return 1e-3

        numbers = [Clearing(), 1e-3]
        with pytest.raises(ValueError, match="at least one parameter"):
            p.step(**{where: numbers})

        class Shortening:
            def __float__(self):
                del numbers[1:]
                return 1e-3

        p.params, p.s0, p.s1 = kept[:2], kept[2:4], kept[4:]
        p.grads = [torch.ones_like(x) for x in p.params]
        numbers[:] = [Shortening(), 1e-3]
        with pytest.raises(ValueError):
            p.step(**{where: numbers})
        assert all(torch.equal(x, y) for x, y in zip(before, (*kept, p.counter)))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_list_of_numbers_on_the_device(bits):
    a, b = (Problem([(20, 30), (30,)], F32, bits, seed=8) for _ in range(2))
    a.step(lr=[0.5, 0.25], weight_decay=(0.0, 0.125))
    b.step(lr=[torch.tensor(0.5, device=DEV), 0.25], weight_decay=(0, torch.tensor(0.125, device=DEV)))
    for x, y in zip(a.tensors(), b.tensors()):
        assert torch.equal(x, y)


# ---- capture -------------------------------------------------------------------------------


def _capture(opt):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    return graph


@pytest.mark.parametrize("bits", [32, 8])
def test_a_capture_in_which_states_would_begin_is_refused(bits):
    """Its replays would clear the states each time."""
    m = _model()
    opt = flex.AdamW(m, state_bits=bits)
    _set_grads(m, 0)
    with pytest.raises(RuntimeError, match="captur"):
        _capture(opt)
    assert not opt.state
    before = [p.detach().clone() for p in m]
    opt.step()
    graph = _capture(opt)
    graph.replay()
    torch.cuda.synchronize()
    assert int(opt.state[m[0]]["counter"][0]) == 2 and not any(torch.equal(x, y) for x, y in zip(before, m))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_capture_that_leaves_a_parameter_behind(bits):
    """The count of a parameter without a gradient stays what it was over all replays."""
    a, b = _model(), _model()
    opts = [flex.AdamW(x, lr=1e-2, state_bits=bits) for x in (a, b)]
    for x, opt in zip((a, b), opts):
        _set_grads(x, 0)
        opt.step()
        _set_grads(x, 1, but=(2,))
    with pytest.raises(RuntimeError, match="captur"):
        _capture(opts[1])
    for opt in opts:
        opt.step()
    graph = _capture(opts[1])
    for _ in range(3):
        opts[0].step()
        graph.replay()
        torch.cuda.synchronize()
    assert [int(opts[1].state[p]["counter"][0]) for p in b] == [5, 5, 1, 5]
    for x, opt in zip((a, b), opts):
        _set_grads(x, 2)
        opt.step()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
        assert int(opts[0].state[x]["counter"][0]) == int(opts[1].state[y]["counter"][0])


# ---- groups --------------------------------------------------------------------------------


def _break(opt, how):
    group = opt.param_groups[1]
    if how == "lr":
        group["lr"] = -1.0
    elif how == "lr on the device":
        group["lr"] = torch.ones((), dtype=torch.float64, device=DEV)
    elif how == "betas":
        group["betas"] = (0.9, 1.0)
    elif how == "state":
        s = opt.state[group["params"][1]]
        key = "exp_avg" if "exp_avg" in s else "codes"
        s[key] = s[key][:1]
    elif how == "unit rows":
        group["unit_rows"] = True


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["lr", "lr on the device", "betas", "state", "unit rows"])
def test_a_group_that_is_refused_leaves_the_others_unstepped(bits, how):
    m = _model()
    opt = flex.AdamW([{"params": m[:2]}, {"params": m[2:]}], state_bits=bits)
    _set_grads(m, 0)
    opt.step()
    _break(opt, how)
    before = [p.detach().clone() for p in m]
    states = [{k: t.clone() for k, t in opt.state[p].items()} for p in m]
    with pytest.raises(ValueError):
        opt.step()
    for p, x, s in zip(m, before, states):
        assert torch.equal(p, x)
        assert all(torch.equal(t, opt.state[p][k]) for k, t in s.items())


# ---- masters of fp32 parameters ------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_an_ignored_master_is_left_alone(bits):
    """... its version too, and whatever stands there: one of inference mode has none."""
    p = Problem([(20, 30), (30,), (40,)], [F32, F16, F32], bits, master=True)
    with torch.inference_mode():
        p.masters[2] = torch.ones(7, device=DEV)
    first, version = p.masters[0].clone(), p.masters[0]._version
    versions = [p.masters[1]._version, *(x._version for x in p.params)]
    p.step()
    assert p.masters[0]._version == version and torch.equal(p.masters[0], first)
    assert bool((p.masters[2] == 1).all())
    assert all(x._version > v for x, v in zip([p.masters[1], *p.params], versions))
    assert int(p.counter[0]) == 8


# ---- refusals ------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_expanded_tensors_are_refused_before_the_step(bits):
    for which in ("params", "s0", "s1", "masters"):
        p = Problem([(4, 600), (7,)], F16, bits, master=True)
        x = getattr(p, which)[0]
        getattr(p, which)[0] = x[..., :1].expand(x.shape)
        before = [t.clone() for t in p.tensors()]
        with pytest.raises(ValueError, match="one memory"):
            p.step()
        assert all(torch.equal(x, y) for x, y in zip(before, p.tensors())), which
    # (gradients are read alone: that of a sum is one number)
    a, b = (Problem([(4, 600)], F32, bits, seed=3) for _ in range(2))
    a.grads = [torch.ones((), device=DEV).expand(4, 600)]
    b.grads = [torch.ones(4, 600, device=DEV)]
    assert torch.equal(flex.grad_norm(a.grads), flex.grad_norm(b.grads))
    for p in (a, b):
        p.step()
    for x, y in zip(a.tensors(), b.tensors()):
        assert torch.equal(x, y)
