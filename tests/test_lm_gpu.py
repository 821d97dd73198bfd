"""Layer norm, lookup by token and distillation from top logits against their formulas in 64 bits (tests/lm_reference.py, which
derives the bounds)."""
import math

import pytest
import torch

import flexsae_amd as flex
from tests import lm_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ["fp32", "bf16", "fp16"]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _strided(t, pad, first=0):
    """The same rows, `pad` elements apart, the first at an offset."""
    n, d = t.shape
    flat = torch.full((first + n * (d + pad),), 7.0, dtype=t.dtype, device=t.device)
    view = flat[first:].view(n, d + pad)[:, :d]
    view.copy_(t)
    return view


# ---- layer norm ----------------------------------------------------------------------------


def _norm_inputs(n, d, dtype, seed, mean=0.3):
    g = _gen(seed)
    x = (torch.randn(n, d, generator=g) * torch.randn(d, generator=g).exp() + mean).to(dtype).to(DEV)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype).to(DEV)
    b = (0.2 * torch.randn(d, generator=g)).to(dtype).to(DEV)
    dy = torch.randn(n, d, generator=g).to(dtype).to(DEV)
    return x, w, b, dy


def _check_norm(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    x_, w_, b_ = (next(it) if t is not None else None for t in (x, w, b))
    y = flex.layer_norm(x_, w_, b_, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    want, tol = ref.layer_norm(x, w, b, eps, dy)
    ref.within(y, want["y"], ref.rounded(want["y"], x.dtype, tol["y"]), "y")
    got = iter(grads)
    dx = next(got)
    ref.within(dx, want["dx"], ref.rounded(want["dx"], x.dtype, tol["dx"]), "dx")
    for name, t in (("dw", w), ("db", b)):
        if t is not None:
            d = next(got)
            assert d.dtype == t.dtype
            ref.within(d, want[name], ref.rounded(want[name], t.dtype, tol[name]), name)
    return y, grads


@pytest.mark.parametrize("n,d", [(1, 1), (2, 2), (5, 7), (3, 48), (70, 64), (33, 65), (64, 128), (9, 129), (31, 256), (300, 257),
                                 (17, 512), (6, 515), (9, 1024), (7, 1025), (600, 1538), (5, 2304), (3, 4096), (3, 4099),
                                 (2, 8192), (2, 9001), (3, 16384), (2, 16385), (3, 33001), (2100, 67)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_norm(n, d, dtype):
    _check_norm(*_norm_inputs(n, d, dtype, seed=n * 7 + d))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_norm_without_weight_or_bias(dtype, weight, bias):
    for n, d in ((37, 200), (5, 1500), (2, 20001)):
        x, w, b, dy = _norm_inputs(n, d, dtype, seed=d)
        _check_norm(x, w if weight else None, b if bias else None, dy)


def test_norm_weights_of_other_types():
    x, w, b, dy = _norm_inputs(41, 1301, torch.bfloat16, seed=3)
    _check_norm(x, w.float(), b.half(), dy)
    x, w, b, dy = _norm_inputs(41, 131, torch.float32, seed=4)
    _check_norm(x, w.bfloat16(), b.half(), dy)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("d", [67, 256, 1027, 17001])
def test_norm_of_rows_apart_and_at_odd_addresses(d, dtype):
    x, w, b, dy = _norm_inputs(13, d, dtype, seed=d)
    y, grads = _check_norm(x, w, b, dy)
    for pad, first in ((0, 1), (3, 0), (5, 1)):
        y2, grads2 = _check_norm(_strided(x, pad, first), w, b, _strided(dy, pad + 1, first))
        assert torch.equal(y, y2) and all(torch.equal(a, c) for a, c in zip(grads, grads2))
    odd = torch.cat([w[:1], w])[1:], torch.cat([b[:1], b])[1:]
    assert torch.equal(flex.layer_norm(x, *odd), y)


def test_norm_of_other_layouts():
    x, w, b, dy = _norm_inputs(24, 80, torch.float32, seed=5)
    y = flex.layer_norm(x, w, b)
    assert torch.equal(flex.layer_norm(x.view(2, 3, 4, 80), w, b).view(24, 80), y)
    assert torch.equal(flex.layer_norm(x.view(4, 6, 80).transpose(0, 1), w, b).transpose(0, 1).reshape(24, 80), y)
    assert torch.equal(flex.layer_norm(x.t().contiguous().t(), w, b), y)
    assert torch.equal(flex.layer_norm(x[3], w, b), y[3])
    assert torch.equal(flex.layer_norm(x[:1].expand(5, 80), w, b), y[:1].expand(5, 80))
    assert torch.equal(flex.layer_norm(x, w[:1].expand(80), b), flex.layer_norm(x, w[:1].repeat(80), b))
    # a gradient that has one memory for all elements
    a, c = x.clone().requires_grad_(), x.clone().requires_grad_()
    flex.layer_norm(a, w, b).sum().backward()
    flex.layer_norm(c, w, b).backward(torch.ones_like(c))
    assert torch.equal(a.grad, c.grad)


def test_norm_without_rows():
    x = torch.zeros(0, 33, device=DEV, requires_grad=True)
    w, b = torch.ones(33, device=DEV, requires_grad=True), torch.ones(33, device=DEV, requires_grad=True)
    y, mean, rstd = flex.layer_norm_stats(x, w, b)
    assert y.shape == (0, 33) and mean.shape == (0,) and rstd.shape == (0,)
    y.sum().backward()
    assert x.grad.shape == (0, 33) and torch.equal(w.grad, torch.zeros(33, device=DEV)) and torch.equal(b.grad, torch.zeros(33, device=DEV))


@pytest.mark.parametrize("d", [60, 900, 5000, 20000])
def test_norm_of_constant_rows_and_far_from_zero(d):
    """A constant row gives the bias; a large common offset costs what it costs in the input's own digits."""
    x = torch.full((4, d), 3.25, device=DEV)
    w, b = torch.full((d,), 2.0, device=DEV), torch.full((d,), 0.5, device=DEV)
    y = flex.layer_norm(x, w, b)
    assert (y - 0.5).abs().max() <= 80 * ref.U * 3.25 / math.sqrt(1e-5) * 2
    x, w, b, dy = _norm_inputs(6, d, torch.float32, seed=d, mean=5000.0)
    _check_norm(x, w, b, dy)


def test_norm_keeps_nan_and_infinity_to_their_rows():
    x, w, b, _ = _norm_inputs(40, 300, torch.float32, seed=8)
    y = flex.layer_norm(x, w, b)
    x[3, 17], x[5, 0] = math.nan, math.inf
    z = flex.layer_norm(x, w, b)
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 5]] = True
    assert z[bad].isnan().all() and torch.equal(z[~bad], y[~bad])


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_norm_stats(dtype):
    for n, d in ((65, 96), (7, 3001), (2, 18000)):
        x, w, b, _ = _norm_inputs(n, d, dtype, seed=n)
        y, mean, rstd = flex.layer_norm_stats(x, w, b)
        want, tol = ref.layer_norm(x, w, b, 1e-5)
        assert mean.dtype == rstd.dtype == torch.float32
        ref.within(mean, want["mean"], ref.rounded(want["mean"], torch.float32, tol["mean"]), "mean")
        ref.within(rstd, want["rstd"], ref.rounded(want["rstd"], torch.float32, tol["rstd"]), "rstd")
        assert torch.equal(y, flex.layer_norm(x, w, b))
        x.requires_grad_()
        y2, mean2, rstd2 = flex.layer_norm_stats(x, w, b)
        assert y2.requires_grad and not mean2.requires_grad and not rstd2.requires_grad
        assert torch.equal(mean, mean2) and torch.equal(rstd, rstd2) and torch.equal(y, y2)


@pytest.mark.parametrize("d", [100, 3001, 17000])
def test_norm_gradients_of_some_inputs(d):
    x, w, b, dy = _norm_inputs(50, d, torch.float32, seed=d)
    _, every = _check_norm(x, w, b, dy)
    for mask in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        flex.layer_norm(*leaves).backward(dy)
        for t, g in zip(leaves, every):
            assert (t.grad is None) == (not t.requires_grad) and (t.grad is None or torch.equal(t.grad, g))


def test_norm_gradient_by_differences():
    x, w, b, dy = _norm_inputs(6, 40, torch.float32, seed=11)
    _, grads = _check_norm(x, w, b, dy)
    f64 = [t.cpu().double() for t in (x, w, b)]
    value = lambda args: (ref.layer_norm(*args, 1e-5)[0]["y"] * dy.cpu().double()).sum()
    for i, g in enumerate(grads):
        along = torch.randn(f64[i].shape, generator=_gen(i), dtype=torch.float64)
        h = 1e-5
        moved = [[t + s * h * along if k == i else t for k, t in enumerate(f64)] for s in (1, -1)]
        slope = (value(moved[0]) - value(moved[1])) / (2 * h)
        # (differences: h^2 of the third derivative, and 2^-53 / h of the value)
        assert abs((g.cpu().double() * along).sum() - slope) <= 1e-5 * (g.cpu().double() * along).abs().sum()


# ---- lookup --------------------------------------------------------------------------------


def _lookup_inputs(n, v, d, dtype, seed, pad=0.2, hot=0.0):
    g = _gen(seed)
    tokens = torch.randint(0, v, (n,), generator=g)
    tokens[torch.rand(n, generator=g) < hot] = v // 2
    tokens[torch.rand(n, generator=g) < pad] = -1
    w = torch.randn(v, d, generator=g).to(dtype).to(DEV)
    scale = (torch.rand(n, generator=g) + 0.25).to(dtype).to(DEV)
    dout = torch.randn(n, d, generator=g).to(dtype).to(DEV)
    return tokens.to(DEV), w, scale, dout


def _check_lookup(tokens, w, scale, dout):
    factor = scale if isinstance(scale, float) else 1.0
    each = scale if isinstance(scale, torch.Tensor) else None
    w_ = w.detach().requires_grad_()
    s_ = scale if each is None else each.detach().requires_grad_()
    out = flex.embedding_lookup(tokens, w_, s_)
    grads = torch.autograd.grad(out, [w_] if each is None else [w_, s_], dout)
    want, tol = ref.lookup(tokens, w, each, factor, dout)
    ref.within(out, want["out"], ref.rounded(want["out"], w.dtype, tol["out"]), "out")
    ref.within(grads[0], want["dw"], ref.rounded(want["dw"], w.dtype, tol["dw"]), "dw")
    empty = want["dw"].abs().sum(1) == 0
    assert not grads[0][empty.to(DEV)].any()
    if each is not None:
        assert grads[1].dtype == each.dtype
        ref.within(grads[1], want["ds"], ref.rounded(want["ds"], each.dtype, tol["ds"]), "ds")
    return out, grads


@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 5, 3), (31, 50, 64), (64, 7, 48), (65, 1, 130), (257, 2, 257), (1000, 30, 129),
                                   (500, 3000, 515), (129, 40, 2304), (300, 20, 4099), (63, 5000, 33), (4000, 700, 20)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_lookup(n, v, d, dtype):
    for kind in range(3):
        tokens, w, scale, dout = _lookup_inputs(n, v, d, dtype, seed=n + v + d + kind, pad=0.2 * (kind != 1))
        _check_lookup(tokens, w, (scale, 1.75, None)[kind], dout)


@pytest.mark.parametrize("n", [63, 64, 65, 127, 128, 129, 191, 192, 193, 640, 5000])
@pytest.mark.parametrize("d", [40, 700])
def test_lookup_of_frequent_tokens(n, d):
    """Tokens that fill less than, exactly and more than the stretches that are added up apart; several of them in a row."""
    for seed, hot in ((1, 1.0), (2, 0.5), (3, 0.0)):
        tokens, w, scale, dout = _lookup_inputs(n, 3, d, torch.float32, seed=seed, pad=0.0, hot=hot)
        _check_lookup(tokens, w, scale, dout)
    for first in (1, 63, 64, 65, 100):
        tokens = torch.full((n,), 4, device=DEV)
        tokens[:first] = 2
        tokens[-1] = 5
        _check_lookup(tokens, torch.randn(6, d, device=DEV), None, torch.randn(n, d, device=DEV))


def test_lookup_of_padding_is_not_looked_at():
    tokens, w, scale, dout = _lookup_inputs(700, 9, 65, torch.float32, seed=5, pad=0.5)
    _, grads = _check_lookup(tokens, w, scale, dout)
    dout[tokens < 0] = math.nan
    scale = scale.masked_fill(tokens < 0, math.nan)
    out, again = _check_lookup(tokens, w, scale, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)) and out.isfinite().all()
    every = torch.full((200,), -1, device=DEV)
    out, grads = _check_lookup(every, w, None, torch.full((200, 65), math.nan, device=DEV))
    assert not out.any() and not grads[0].any()
    flex.check_index_flag()


def test_lookup_of_tokens_outside_the_table():
    w = torch.randn(10, 24, device=DEV)
    tokens = torch.tensor([3, 10, 0, -2, 2 ** 40, -2 ** 60, 9], device=DEV)
    _check_lookup(tokens, w, None, torch.randn(7, 24, device=DEV))
    with pytest.raises(IndexError, match="token"):
        flex.check_index_flag()
    flex.check_index_flag()
    flex.set_index_checking(True)
    try:
        with pytest.raises(IndexError, match="token"):
            flex.embedding_lookup(tokens, w)
    finally:
        flex.set_index_checking(False)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_lookup_layouts(dtype):
    tokens, w, scale, dout = _lookup_inputs(150, 11, 77, dtype, seed=9)
    out, grads = _check_lookup(tokens, w, scale, dout)
    out2, grads2 = _check_lookup(tokens, _strided(w, 5, 1), scale, _strided(dout, 2, 3))
    assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))
    cube = tokens.view(5, 30)
    assert torch.equal(flex.embedding_lookup(cube, w, scale.view(5, 30)).view(150, 77), out)
    assert torch.equal(flex.embedding_lookup(cube.t(), w, scale.view(5, 30).t()), out.view(5, 30, 77).transpose(0, 1))
    assert torch.equal(flex.embedding_lookup(tokens.int(), w, scale), out)
    assert torch.equal(flex.embedding_lookup(tokens[4], w, scale[4]), out[4])
    assert torch.equal(flex.embedding_lookup(tokens, w.t().contiguous().t(), scale), out)
    assert torch.equal(flex.embedding_lookup(tokens.clamp_min(0), w), w[tokens.clamp_min(0)])


def test_lookup_gradients_of_broadcast_scales():
    tokens, w, _, dout = _lookup_inputs(60, 8, 50, torch.float32, seed=10)
    one = torch.tensor(1.5, device=DEV, requires_grad=True)
    rows = torch.rand(6, 1, device=DEV).requires_grad_()
    flex.embedding_lookup(tokens.view(6, 10), w, one).backward(dout.view(6, 10, 50))
    flex.embedding_lookup(tokens.view(6, 10), w, rows).backward(dout.view(6, 10, 50))
    want, tol = ref.lookup(tokens, w, torch.ones(60), 1.0, dout)
    ref.within(one.grad, want["ds"].sum(), tol["ds"].sum() + 64 * ref.U * want["ds"].abs().sum(), "one")
    ref.within(rows.grad, want["ds"].view(6, 10).sum(1, keepdim=True),
               (tol["ds"] + 16 * ref.U * want["ds"].abs()).view(6, 10).sum(1, keepdim=True) + 16 * ref.U * want["ds"].abs().max(), "rows")


def test_lookup_gradients_of_one_input():
    for n, d in ((400, 60), (400, 1500)):
        tokens, w, scale, dout = _lookup_inputs(n, 12, d, torch.bfloat16, seed=n + d)
        _, (dw, ds) = _check_lookup(tokens, w, scale, dout)
        a = w.clone().requires_grad_()
        flex.embedding_lookup(tokens, a, scale).backward(dout)
        b = scale.clone().requires_grad_()
        flex.embedding_lookup(tokens, w, b).backward(dout)
        assert torch.equal(a.grad, dw)
        want, tol = ref.lookup(tokens, w, scale, 1.0, dout)
        ref.within(b.grad, want["ds"], ref.rounded(want["ds"], b.dtype, tol["ds"]), "ds")


def test_lookup_without_tokens():
    w = torch.randn(5, 6, device=DEV, requires_grad=True)
    scale = torch.rand(0, 3, device=DEV, requires_grad=True)
    out = flex.embedding_lookup(torch.zeros(0, 3, dtype=torch.int64, device=DEV), w, scale)
    assert out.shape == (0, 3, 6)
    out.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and scale.grad.shape == (0, 3)


def test_lookup_gradient_by_differences():
    tokens, w, scale, dout = _lookup_inputs(30, 6, 20, torch.float32, seed=12)
    _, grads = _check_lookup(tokens, w, scale, dout)
    f64 = [w.cpu().double(), scale.cpu().double()]
    value = lambda args: (ref.lookup(tokens, *args, 1.0)[0]["out"] * dout.cpu().double()).sum()
    for i, g in enumerate(grads):
        along = torch.randn(f64[i].shape, generator=_gen(i), dtype=torch.float64)
        moved = [[t + s * 1e-4 * along if k == i else t for k, t in enumerate(f64)] for s in (1, -1)]
        slope = (value(moved[0]) - value(moved[1])) / 2e-4
        assert abs((g.cpu().double() * along).sum() - slope) <= 1e-5 * (g.cpu().double() * along).abs().sum()


# ---- distillation --------------------------------------------------------------------------


def _distill_inputs(n, v, k, dtype, seed, ragged=False, top_dtype=None):
    g = _gen(seed)
    index = torch.randint(0, v, (n, k), generator=g)
    top = 5.0 - 1.5 * torch.arange(k).add(1).log() + 0.5 * torch.randn(n, k, generator=g)
    z = 1.5 * torch.randn(n, v, generator=g)
    z.scatter_(1, index, top + 0.7 * torch.randn(n, k, generator=g))
    if ragged:
        index[torch.rand(n, k, generator=g) < 0.4] = -1
        index[0] = -1
    return z.to(dtype).to(DEV), top.to(top_dtype or dtype).to(DEV), index.to(DEV)


def _check_distill(z, top, index, weights=None, T=1.0, by_row=False, grad=1.0):
    g = torch.as_tensor(grad, dtype=torch.float32, device=DEV)
    if by_row:
        g = g.expand(z.shape[0]).contiguous()
    leaf = z.detach().requires_grad_()
    loss = flex.distillation_loss(leaf, top, index, temperature=T, row_weights=weights, reduction="none" if by_row else "mean")
    dz, = torch.autograd.grad(loss, leaf, g)
    want, tol = ref.distill(z, top, index, weights, T, by_row, g)
    assert loss.dtype == torch.float32 and dz.dtype == z.dtype and dz.is_contiguous()
    ref.within(loss, want["loss"], tol["loss"] + ref.U * want["loss"].abs() + 1e-38, "loss")
    ref.within(dz, want["dz"], ref.rounded(want["dz"], z.dtype, tol["dz"]), "dz")
    alone = flex.distillation_loss(z, top, index, temperature=T, row_weights=weights, reduction="none" if by_row else "mean")
    ref.within(alone, want["loss"], tol["loss"] + ref.U * want["loss"].abs() + 1e-38, "loss alone")
    return loss.detach(), dz


@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 2, 3), (3, 7, 2), (2, 64, 64), (5, 255, 9), (4, 1000, 65), (1, 4097, 5), (7, 5003, 50),
                                   (2, 32000, 32), (3, 50001, 300), (1, 131072, 128), (300, 515, 20), (2100, 130, 8), (520, 9001, 6)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_distill(n, v, k, dtype):
    z, top, index = _distill_inputs(n, v, k, dtype, seed=n + v + k)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    _check_distill(z, top, index, grad=scale)


@pytest.mark.parametrize("n,v,k", [(3, 4, 1), (3, 8, 2), (300, 4097, 256), (5, 8193, 257), (260, 16385, 300), (258, 32771, 9),
                                   (256, 65535, 512), (300, 65536, 40), (257, 131071, 700), (260, 131080, 20), (260, 3000, 1500)])
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_distill_of_rows_in_registers_and_beyond(n, v, k, dtype):
    z, top, index = _distill_inputs(n, v, k, dtype, seed=n + v)
    index[:, k // 2:] = torch.where(torch.rand(n, k - k // 2, generator=_gen(1)).to(DEV) < 0.1, index[:, :1], index[:, k // 2:])
    weights = torch.rand(n, generator=_gen(2)).to(DEV)
    weights[1] = 0.0
    index[2] = -1
    _check_distill(z, top, index, weights, T=0.8, grad=1.0 if dtype != torch.float16 else 4096.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("T", [0.5, 3.0])
def test_distill_options(dtype, by_row, T):
    for n, v, k in ((33, 1003, 12), (3, 20001, 40)):
        z, top, index = _distill_inputs(n, v, k, dtype, seed=n, ragged=True, top_dtype=torch.float32)
        weights = torch.rand(n, generator=_gen(1)).to(DEV)
        weights[1] = 0.0
        grad = torch.linspace(-2.0, 3.0, n) if by_row else 300.0
        _check_distill(z, top, index, weights, T, by_row, grad)
        _check_distill(z, top, index, None, T, by_row, grad)


def test_distill_masks_of_rows():
    z, top, index = _distill_inputs(20, 700, 10, torch.float32, seed=4)
    mask = torch.arange(20, device=DEV) % 3 != 0
    loss, dz = _check_distill(z, top, index, mask.float())
    other = z.detach().clone()
    other[~mask] = math.nan
    leaf = other.requires_grad_()
    for weights in (mask, mask.float(), mask.bfloat16()):
        again = flex.distillation_loss(leaf, top, index, row_weights=weights)
        again.backward()
        assert torch.equal(again.detach(), loss) and torch.equal(leaf.grad, dz) and not leaf.grad[~mask].any()
        leaf.grad = None
    none = flex.distillation_loss(leaf, top, index, row_weights=torch.zeros(20, device=DEV))
    none.backward()
    assert none.item() == 0.0 and not leaf.grad.any()
    # rows without a stored logit, and those whose stored logits are all minus infinity
    index = index.clone()
    index[2] = -1
    top = top.clone()
    top[4] = -math.inf
    top[5, :5] = -math.inf
    z = z.detach().clone()
    z[2], z[4] = math.nan, math.inf
    _check_distill(z, top, index)


def test_distill_masked_logits():
    """Vocabulary entries at minus infinity, at the type's lowest value, and infinite or NaN ones."""
    for dtype in DTYPES:
        z, top, index = _distill_inputs(8, 900, 6, dtype, seed=6)
        away = torch.rand(8, 900, generator=_gen(2)).to(DEV) < 0.5
        away.scatter_(1, index, False)
        _check_distill(z.masked_fill(away, -math.inf), top, index, grad=64.0)
        for low in (torch.finfo(dtype).min, torch.finfo(dtype).min / 2, -1000.0):
            _check_distill(z.masked_fill(away, low), top, index, grad=64.0)
            every = z.clone()
            every[3] = low  # nothing else: even
            _check_distill(every, top, index, T=0.25, grad=64.0)
    z, top, index = _distill_inputs(4, 300, 5, torch.float32, seed=7)
    lost = z.clone()
    lost[1, index[1, 0]] = -math.inf
    loss = flex.distillation_loss(lost, top, index, reduction="none")
    assert loss[1] == math.inf and loss[[0, 2, 3]].isfinite().all()
    z[2, 5], z[3, 7] = math.nan, math.inf
    leaf = z.requires_grad_()
    loss = flex.distillation_loss(leaf, top, index, reduction="none")
    loss.backward(torch.ones(4, device=DEV))
    assert loss[:2].isfinite().all() and loss[2:].isnan().all()
    assert leaf.grad[:2].isfinite().all() and leaf.grad[2:].isnan().all()
    top = top.clone()
    top[0, 1] = math.nan
    assert flex.distillation_loss(z, top, index, reduction="none")[0].isnan()
    top[0] = math.nan
    assert flex.distillation_loss(z, top, index, reduction="none")[0].isnan()


def test_distill_far_logits():
    """Large logits, and a student that equals its teacher."""
    z, top, index = _distill_inputs(6, 2000, 8, torch.float32, seed=8)
    _check_distill(z + 3000.0, top - 5000.0, index)
    _check_distill(z * 40.0, top * 40.0, index)
    z = torch.full((3, 500), -math.inf, device=DEV)
    z.scatter_(1, torch.arange(8, device=DEV).expand(3, 8), top[:3])
    loss, dz = _check_distill(z, top[:3], torch.arange(8, device=DEV).expand(3, 8))
    assert loss.abs() < 1e-6 and dz.abs().max() < 1e-6


def test_distill_entries_stored_twice():
    z, top, index = _distill_inputs(9, 400, 40, torch.float32, seed=9)
    index[:, 20:] = index[:, :20].flip(1)
    index[3] = index[3, 0]
    _check_distill(z, top, index)
    # rows in registers: all places of a row the same, two in turn, and many entries of one thread
    for k in (200, 1000):
        z, top, index = _distill_inputs(260, 9000, k, torch.float32, seed=14)
        index[0], index[1], index[2] = 8999, torch.arange(k, device=DEV) % 2, torch.arange(k, device=DEV) % 4
        index[3] = torch.arange(k, device=DEV) % 8 * 4096 // 4
        top[4:8] = -1e4
        top[4:8, -1] = 1.0
        index[4:8, :-1] = 0  # (places without weight, as of padding)
        first = _check_distill(z, top, index)
        again = _check_distill(z, top, index)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_distill_indices_outside_the_vocabulary():
    z, top, index = _distill_inputs(5, 60, 7, torch.float32, seed=10)
    index[0, 2], index[1, 3], index[2, 0] = 60, -2, 2 ** 33
    _check_distill(z, top, index)
    with pytest.raises(IndexError, match="token"):
        flex.check_index_flag()
    _check_distill(z, top, index.clamp(-1, 59).int())
    flex.check_index_flag()
    weights = torch.ones(5, device=DEV)
    weights[0] = weights[1] = weights[2] = 0.0  # (also of rows that are not used)
    for leaf in (z, z.clone().requires_grad_()):
        flex.distillation_loss(leaf, top, index, row_weights=weights)
        with pytest.raises(IndexError, match="token"):
            flex.check_index_flag()


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_distill_layouts(dtype):
    z, top, index = _distill_inputs(12, 1001, 9, dtype, seed=11)
    loss, dz = _check_distill(z, top, index, grad=8.0)
    loss2, dz2 = _check_distill(_strided(z, 7, 1), top, index, grad=8.0)
    assert torch.equal(loss, loss2) and torch.equal(dz, dz2)
    leaf = z.view(3, 4, 1001).clone().requires_grad_()
    cube = flex.distillation_loss(leaf, top.view(3, 4, 9), index.view(3, 4, 9), reduction="none",
                                  row_weights=torch.ones(3, 4, device=DEV))
    assert cube.shape == (3, 4)
    rows = flex.distillation_loss(z, top, index, reduction="none")
    assert torch.equal(cube.view(12), rows)
    one = flex.distillation_loss(z[5], top[5], index[5], reduction="none")
    assert one.shape == () and one == rows[5]
    cube.sum().backward()
    assert leaf.grad.shape == leaf.shape


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_distill_backward_twice_and_scaled(dtype):
    z, top, index = _distill_inputs(40, 3001, 16, dtype, seed=12)
    for grad in (1.0, 512.0, 0.3):
        leaf = z.clone().requires_grad_()
        loss = flex.distillation_loss(leaf, top, index)
        g = torch.tensor(grad, device=DEV)
        first, = torch.autograd.grad(loss, leaf, g, retain_graph=True)
        second, = torch.autograd.grad(loss, leaf, g)
        assert torch.equal(first, second) and first.data_ptr() != second.data_ptr()
        _, dz = _check_distill(z, top, index, grad=grad)
        assert torch.equal(dz, first)
    leaf = z.clone().requires_grad_()
    loss = flex.distillation_loss(leaf, top, index)
    with torch.no_grad():
        leaf.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_distill_gradient_by_differences():
    z, top, index = _distill_inputs(5, 30, 6, torch.float32, seed=13)
    weights = torch.tensor([1.0, 0.5, 0.0, 2.0, 1.0], device=DEV)
    _, dz = _check_distill(z, top, index, weights, T=1.5)
    along = torch.randn(z.shape, generator=_gen(3), dtype=torch.float64)
    value = lambda s: ref.distill(z.cpu().double() + s * 1e-4 * along, top, index, weights, 1.5, False)[0]["loss"]
    slope = (value(1) - value(-1)) / 2e-4
    assert abs((dz.cpu().double() * along).sum() - slope) <= 1e-5 * (dz.cpu().double() * along).abs().sum()


# ---- together, and around the calls --------------------------------------------------------


def _chain(leaves, tokens, top, index, mask, norm, lookup, distill):
    x, table, gates, w, b, out = leaves
    return distill(norm(x + lookup(tokens, table, gates), w, b) @ out, top, index, mask)


def test_the_three_together():
    """Reconstruction plus rows by token, the model's last norm, its logits, the loss: gradients of everything against autograd in
    64 bits."""
    g = _gen(20)
    n, v, d, k = 96, 301, 72, 10
    leaves = [torch.randn(n, d, generator=g), 0.5 * torch.randn(v, d, generator=g), torch.rand(n, generator=g),
              1 + 0.1 * torch.randn(d, generator=g), 0.1 * torch.randn(d, generator=g), 0.3 * torch.randn(d, v, generator=g)]
    tokens = torch.randint(-1, v, (n,), generator=g)
    _, top, index = _distill_inputs(n, v, k, torch.float32, seed=21)
    mask = torch.rand(n, generator=g) < 0.8
    mine = [t.to(DEV).requires_grad_() for t in leaves]
    loss = _chain(mine, tokens.to(DEV), top, index, mask.to(DEV), flex.layer_norm, flex.embedding_lookup,
                  lambda z, t, i, m: flex.distillation_loss(z, t, i, row_weights=m))
    loss.backward()

    def lookup(tokens, table, gates):
        return torch.where((tokens >= 0)[:, None], table[tokens.clamp_min(0)] * gates[:, None], 0.0)

    def norm(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b

    def distill(z, t, i, m):
        p = torch.softmax(t, 1)
        kl = (p * (p.log() - torch.log_softmax(z, 1).gather(1, i))).sum(1)
        return (kl * m).sum() / m.sum()

    theirs = [t.double().requires_grad_() for t in leaves]
    want = _chain(theirs, tokens, top.cpu().double(), index.cpu(), mask, norm, lookup, distill)
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for a, b in zip(mine, theirs):
        assert (a.grad.cpu().double() - b.grad).norm() <= 1e-5 * b.grad.norm()


def _calls(seed=30):
    """(name, function of leaves, leaves) with all gradients wanted; losses are sums against fixed weights."""
    x, w, b, dy = _norm_inputs(60, 1100, torch.bfloat16, seed)
    tokens, table, scale, dout = _lookup_inputs(900, 50, 300, torch.bfloat16, seed)
    z, top, index = _distill_inputs(30, 5001, 12, torch.bfloat16, seed)
    zh = z.half()
    return [("norm", lambda x, w, b: flex.layer_norm(x, w, b), [x, w, b], dy),
            ("lookup", lambda t, s: flex.embedding_lookup(tokens, t, s), [table, scale], dout),
            ("mean", lambda z: flex.distillation_loss(z, top, index), [z], torch.tensor(1.0, device=DEV)),
            ("scaled", lambda z: flex.distillation_loss(z, top, index), [z], torch.tensor(128.0, device=DEV)),
            ("half", lambda z: flex.distillation_loss(z, top, index, temperature=2.0), [zh], torch.tensor(128.0, device=DEV)),
            ("rows", lambda z: flex.distillation_loss(z, top, index, reduction="none"), [z], torch.full((30,), 0.5, device=DEV))]


def _pass(fn, tensors, grad):
    leaves = [t.detach().requires_grad_() for t in tensors]
    out = fn(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, grad)]


def _same(name, a, b):
    """The ops take the gradient of a mean from other partial sums than the one that is made along with the loss: both within the
    bounds of the formula, so within twice the rounding of each other (and 1e-5 for the sums, of 1e3 terms in a lane at most)."""
    if name not in ("mean", "scaled"):
        return all(torch.equal(p, q) for p, q in zip(a, b))
    return all(bool(((p.double() - q.double()).abs() <= (2 * ref.half(p.dtype) + 1e-5) * q.double().abs()).all()) for p, q in zip(a, b))


def test_the_same_bits_on_every_run_and_through_the_ops():
    for name, fn, tensors, grad in _calls():
        first = _pass(fn, tensors, grad)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, _pass(fn, tensors, grad))), name
        flex.set_index_checking(True)  # (calls then go through the ops)
        try:
            assert _same(name, first, _pass(fn, tensors, grad)), name
        finally:
            flex.set_index_checking(False)


def test_on_another_stream():
    stream = torch.cuda.Stream()
    for name, fn, tensors, grad in _calls(31):
        want = _pass(fn, tensors, grad)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            got = _pass(fn, tensors, grad)
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), name


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed between eager calls with other inputs in the same places."""
    for name, fn, tensors, grad in _calls(32):
        static = [t.clone() for t in tensors]
        leaves = [t.detach().requires_grad_() for t in static]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(fn(*leaves), leaves, grad)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn(*leaves)
            grads = torch.autograd.grad(out, leaves, grad)
        for turn in range(4):
            with torch.no_grad():
                for s, t in zip(static, tensors):
                    s.copy_(t * (1 + 0.125 * turn))
            graph.replay()
            torch.cuda.synchronize()
            want = _pass(fn, [t * (1 + 0.125 * turn) for t in tensors], grad)
            for a, b in zip(want, [out, *grads]):
                assert torch.equal(a, b), (name, turn)
        del graph


def test_two_calls_in_flight():
    """Calls on two streams at once have nothing in common."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    for name, fn, tensors, grad in _calls(33):
        other = [t.flip(0) if t.dim() == 2 else t for t in tensors]
        want = [_pass(fn, t, grad) for t in (tensors, other)]
        torch.cuda.synchronize()
        got = []
        for stream, t in zip(streams, (tensors, other)):
            with torch.cuda.stream(stream):
                got.append(_pass(fn, t, grad))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b)), name


def test_saved_tensors_that_hooks_hand_back():
    pack = lambda t: t.cpu()
    for name, fn, tensors, grad in _calls(34):
        want = _pass(fn, tensors, grad)
        leaves = [t.detach().requires_grad_() for t in tensors]
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(DEV)):
            out = fn(*leaves)
        got = torch.autograd.grad(out, leaves, grad)
        assert all(torch.equal(a, b) for a, b in zip(want[1:], got)), name


def test_gradients_of_gradients_are_refused():
    for name, fn, tensors, grad in _calls(35):
        leaves = [t.detach().requires_grad_() for t in tensors]
        grads = torch.autograd.grad(fn(*leaves), leaves, grad, create_graph=True)
        with pytest.raises(RuntimeError):
            grads[0].float().sum().backward()


def test_compiled_calls():
    for name, fn, tensors, grad in _calls(36):
        want = _pass(fn, tensors, grad)
        compiled = torch.compile(fn, backend="aot_eager", fullgraph=True)
        got = _pass(compiled, tensors, grad)
        assert _same(name, want, got), name


def test_large_offsets():
    """Rows of logits and of a table beyond 2^31 elements from the first."""
    d = 4096
    v = (1 << 31) // d + 5
    w = torch.zeros(v, d, dtype=torch.bfloat16, device=DEV)
    w[-3:] = torch.arange(1, 4, device=DEV, dtype=torch.bfloat16)[:, None]
    w.requires_grad_()
    tokens = torch.tensor([v - 3, v - 1, 0, v - 1], device=DEV)
    out = flex.embedding_lookup(tokens, w)
    assert torch.equal(out[:, 5].float().cpu(), torch.tensor([1.0, 3.0, 0.0, 3.0]))
    out.backward(torch.ones_like(out))
    assert w.grad[v - 1].eq(2).all() and w.grad[v - 3].eq(1).all() and w.grad[0].eq(1).all() and not w.grad[v - 2].any()
    assert w.grad[1:v - 3].count_nonzero() == 0
    del w, out
    torch.cuda.empty_cache()
    n, v = (1 << 31) // 262144 + 3, 262144
    z = torch.zeros(n, v, dtype=torch.bfloat16, device=DEV)
    z[-1] = torch.randn(v, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).bfloat16()
    index = torch.full((n, 3), -1, device=DEV)
    index[-1] = torch.tensor([1, 70000, 262143], device=DEV)
    top = torch.ones(n, 3, device=DEV)
    last, dlast = _check_distill(z[-1:].clone(), top[-1:], index[-1:], by_row=True)
    leaf = z.requires_grad_()
    loss = flex.distillation_loss(leaf, top, index, reduction="none")
    loss.backward(torch.ones(n, device=DEV))
    assert not loss[:-1].any() and not leaf.grad[:-1].any()
    assert abs(loss[-1] - last[0]) <= 1e-5 * last[0]
    assert (leaf.grad[-1].float() - dlast[0].float()).abs().max() <= 2 ** -8 * dlast.float().abs().max()
