"""Layer norm, lookup and distillation at sizes where a group of lanes has several rows one after another, as in training batches:
rows are the bits of calls on slices, whose groups have one row each, and sums over rows are within the bounds of
tests/lm_reference.py."""
import pytest
import torch

import flexsae_amd as flex
from tests import lm_reference as ref
from tests.test_lm_gpu import DEV, DTYPES, NAMES, _check_distill, _check_lookup, _check_norm, _lookup_inputs, _norm_inputs

pytestmark = pytest.mark.gpu


def _gpu_gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


# ---- layer norm ----------------------------------------------------------------------------


@pytest.mark.parametrize("n,d,slice_rows", [(65541, 1025, 1000), (524299, 16, 4000), (300007, 130, 4000), (41003, 2304, 700),
                                            (8195, 16384, 500), (100003, 3, 8000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_norm_forward_of_many_rows(n, d, slice_rows, dtype):
    g = _gpu_gen(n)
    x = torch.empty(n, d, dtype=dtype, device=DEV)
    for piece in x.split(1 << 26):
        piece.copy_(torch.randn(piece.shape, generator=g, device=DEV) + 0.3)
    x *= torch.linspace(0.5, 3.0, n, device=DEV).to(dtype)[:, None]  # (rows that differ in their statistics)
    w, b = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype), (0.2 * torch.randn(d, generator=g, device=DEV)).to(dtype)
    y, mean, rstd = flex.layer_norm_stats(x, w, b)
    for first in (0, n // 3, n - slice_rows):
        rows = slice(first, first + slice_rows)
        y2, mean2, rstd2 = flex.layer_norm_stats(x[rows], w, b)
        assert torch.equal(y[rows], y2) and torch.equal(mean[rows], mean2) and torch.equal(rstd[rows], rstd2)
        few = slice(first, first + 40)
        want, tol = ref.layer_norm(x[few], w, b, 1e-5)
        ref.within(y[few], want["y"], ref.rounded(want["y"], dtype, tol["y"]), "y")
    want, tol = ref.layer_norm(x[n // 2:n // 2 + 40], w, b, 1e-5)
    ref.within(mean[n // 2:n // 2 + 40], want["mean"], ref.rounded(want["mean"], torch.float32, tol["mean"]), "mean")


@pytest.mark.parametrize("n,d", [(20011, 64), (20011, 5), (9001, 130), (6007, 300), (3001, 1025), (3001, 1538), (2777, 2304), (1501, 4099),
                                 (1031, 8192), (701, 16384), (203, 17001)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_norm_backward_of_many_rows(n, d, dtype):
    x, w, b, dy = _norm_inputs(n, d, dtype, seed=n + d)
    x *= torch.linspace(0.5, 3.0, n, device=DEV).to(dtype)[:, None]
    _, (dx, _, _) = _check_norm(x, w, b, dy)
    for first in (0, n // 2, n - 50):  # (a slice's groups have one row each)
        rows = slice(first, first + 50)
        leaf = x[rows].clone().requires_grad_()
        flex.layer_norm(leaf, w, b).backward(dy[rows])
        assert torch.equal(leaf.grad, dx[rows])


# ---- lookup --------------------------------------------------------------------------------


@pytest.mark.parametrize("n,v,d", [(33003, 33005, 500), (17003, 17001, 900), (131075, 131077, 100), (262147, 140001, 12), (262147, 262147, 3)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_lookup_of_many_rows(n, v, d, dtype):
    """Numbers of tokens and rows that four does not divide; with and without gates, padding and frequent tokens."""
    tokens, w, scale, dout = _lookup_inputs(n, v, d, dtype, seed=n + d, hot=0.02)
    tokens[-2:] = torch.tensor([0, v - 1], device=DEV)
    _, (dw, _) = _check_lookup(tokens, w, scale, dout)
    _check_lookup(tokens, w, None, dout)
    few = tokens[:4000]
    out, (dw, ds) = _check_lookup(few, w, scale[:4000], dout[:4000])  # (few tokens, all rows of the table)
    assert torch.equal(flex.embedding_lookup(tokens, w, scale)[:4000], out)
    every = tokens.clamp(0, 99)
    _check_lookup(every, w[:100], scale, dout)  # (the other way round: all of them frequent)


# ---- distillation --------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_distill_rows_are_those_of_slices(dtype):
    """The losses of rows do not depend on what else is in the call, where a row is split alike."""
    g = _gpu_gen(7)
    n, v, k = 4100, 3001, 20
    z = (1.5 * torch.randn(n, v, generator=g, device=DEV)).to(dtype)
    index = torch.randint(0, v, (n, k), generator=g, device=DEV)
    top = torch.randn(n, k, generator=g, device=DEV) + 3.0
    leaf = z.clone().requires_grad_()
    loss = flex.distillation_loss(leaf, top, index, reduction="none")
    grad = torch.linspace(0.5, 2.0, n, device=DEV)
    loss.backward(grad)
    rows = slice(4000, 4100)
    loss2, dz2 = _check_distill(z[rows], top[rows], index[rows], by_row=True)
    assert torch.equal(loss[rows].detach(), loss2)
    leaf2 = z[rows].clone().requires_grad_()
    flex.distillation_loss(leaf2, top[rows], index[rows], reduction="none").backward(grad[rows])
    assert torch.equal(leaf.grad[rows], leaf2.grad)
