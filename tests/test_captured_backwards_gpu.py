"""A hierarchical step of which the forward is captured and the backward not, or the other way round, or each into a graph of its own:
every backward makes the gradients for the upstream gradient of its time."""
import pytest
import torch

import flexsae_amd as flex
from flexsae_amd import ops
from tests.helpers import make_inputs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _by_op(idx, W, v, b, t):
    return ops.hier_train_sliced(idx, W, v, b, t, True, False, False)[0]


def _by_functions(idx, W, v, b, t):
    return ops._HierTrainSliced.apply(idx, W, v, b, t, True, False, False)


@pytest.mark.parametrize("fn", [flex.triton_hierarchical_sae_loss, _by_functions, _by_op], ids=["eager", "functions", "op"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_a_captured_backward_of_an_eager_step(fn, dtype, monkeypatch):
    monkeypatch.setattr(ops, "_late_step", lambda *_: False)
    idx, W, v, b, t = (x.to(DEV) for x in make_inputs(40, 16, 411, 256, dtype, seed=6))
    leaves = [x.clone().requires_grad_() for x in (W, v, b)]
    up = torch.tensor(2.0, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = {}
        for value in (2.0, 0.5, 1.0):
            up.fill_(value)
            want[value] = torch.autograd.grad(fn(idx, *leaves, t), leaves, up)
        loss = fn(idx, *leaves, t)
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad(loss, leaves, up, retain_graph=True)
    for value in (2.0, 2.0, 0.5, 1.0, 2.0):
        up.fill_(value)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, want[value]):
            assert torch.equal(a, c), value
    del graph
    # an eager backward of the same step, whose gradients no replay changes
    up.fill_(0.5)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        left = torch.autograd.grad(loss, leaves, up)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(left, want[0.5]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
def test_backwards_of_a_captured_step(dtype, monkeypatch):
    monkeypatch.setattr(ops, "_late_step", lambda *_: False)
    inputs = [[x.to(DEV) for x in make_inputs(40, 16, 411, 256, dtype, seed=seed)] for seed in (6, 7)]
    up = torch.tensor(2.0, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    idx, W, v, b, t = (x.clone() for x in inputs[0])
    leaves = [x.requires_grad_() for x in (W, v, b)]
    want = {}
    with torch.cuda.stream(stream):
        for which, (i, w, a, c, y) in enumerate(inputs):
            for value in (2.0, 0.5, 1.0):
                up.fill_(value)
                own = [x.clone().requires_grad_() for x in (w, a, c)]
                want[which, value] = torch.autograd.grad(flex.triton_hierarchical_sae_loss(i, *own, y), own, up)
        torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=stream):
        loss = flex.triton_hierarchical_sae_loss(idx, *leaves, t)
    with torch.cuda.graph(backward, stream=stream, pool=forward.pool()):
        got = torch.autograd.grad(loss, leaves, up, retain_graph=True)
    for which in (0, 1, 0):
        for to, x in zip((idx, *leaves, t), inputs[which]):
            to.data.copy_(x)  # (the values alone: what autograd has saved is these very tensors)
        torch.cuda.synchronize()
        forward.replay()
        for value in (2.0, 0.5, 1.0, 0.5):
            up.fill_(value)
            torch.cuda.synchronize()
            backward.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(got, want[which, value])), (which, value)
        with torch.cuda.stream(stream):  # (and an eager one)
            eager = torch.autograd.grad(loss, leaves, up, retain_graph=True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(eager, want[which, 0.5]))
    del forward, backward
