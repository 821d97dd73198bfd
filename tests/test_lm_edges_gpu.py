"""Layer norm, lookup and distillation where calls, values and captures are out of the ordinary (bounds of tests/lm_reference.py)."""
import math

import pytest
import torch

import flexsae_amd as flex
from tests import lm_reference as ref
from tests.test_lm_gpu import DEV, DTYPES, NAMES, _check_distill, _check_lookup, _distill_inputs, _gen, _lookup_inputs

pytestmark = pytest.mark.gpu


# ---- distillation in graphs ----------------------------------------------------------------


def _captured(stream, fn):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = fn()
    return graph, out


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_a_captured_backward_of_an_eager_forward(dtype):
    """Every replay makes the gradient for the upstream gradient of its time, whatever became of the one before."""
    z, top, index = _distill_inputs(40, 3001, 16, dtype, seed=40)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaf = z.clone().requires_grad_()
        g = torch.ones((), device=DEV)
        torch.autograd.grad(flex.distillation_loss(leaf, top, index), leaf, g)
        loss = flex.distillation_loss(leaf, top, index)
    graph, (dz,) = _captured(stream, lambda: torch.autograd.grad(loss, leaf, g))
    for value in (1.0, 64.0, 1.0, 0.5, 1.0, 1.0):
        g.fill_(value)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, tol = ref.distill(z, top, index, None, 1.0, False, g)
        ref.within(dz, want["dz"], ref.rounded(want["dz"], dtype, tol["dz"]), f"upstream gradient {value}")
        dz.fill_(7.0)
        torch.cuda.synchronize()
    del graph


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_an_eager_backward_of_a_captured_forward(dtype):
    """Its gradient is no memory that a replay writes."""
    z, top, index = _distill_inputs(40, 3001, 16, dtype, seed=41)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaf = z.clone().requires_grad_()
        flex.distillation_loss(leaf, top, index)
    graph, loss = _captured(stream, lambda: flex.distillation_loss(leaf, top, index))
    graph.replay()
    torch.cuda.synchronize()
    dz, = torch.autograd.grad(loss, leaf, torch.ones((), device=DEV))
    torch.cuda.synchronize()
    first = dz.clone()
    with torch.no_grad():
        leaf.mul_(2.0)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dz, first)
    want, tol = ref.distill(z, top, index, None, 1.0, False, torch.ones(()))
    ref.within(dz, want["dz"], ref.rounded(want["dz"], dtype, tol["dz"]), "dz")
    del graph
