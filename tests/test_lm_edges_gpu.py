"""Layer norm, lookup and distillation where calls, values and captures are out of the ordinary (bounds of tests/lm_reference.py)."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

import flexsae_amd as flex
from flexsae_amd import _lib
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
    graph, (dz,) = _captured(stream, lambda: torch.autograd.grad(loss, leaf, g, retain_graph=True))
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


# ---- distillation's values -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=NAMES[:2])  # (the range of fp16 does not hold such gradients)
@pytest.mark.parametrize("n,v,k", [(70, 5000, 12), (260, 9000, 200), (260, 40000, 900), (5, 700, 1500)])
@pytest.mark.parametrize("by_row", [False, True])
def test_entries_stored_twice_with_small_probabilities(n, v, k, dtype, by_row):
    """Places of one entry far below the row's largest add up as others do, and to the same bits on every run; the student's own
    probability of it vanishes, so that they are all of its gradient."""
    z, top, index = _distill_inputs(n, v, k, dtype, seed=n + k, top_dtype=torch.float32)
    index = 18 + index % (v - 18)
    index[:, 0] = 0
    top[:, 0] = 1.0
    for row in range(4):  # below 2^-52 of the largest, about there, and between there and 2^-28
        place = torch.arange(1, 9, device=DEV) * ((k - 1) // 8)
        index[row, place] = 17
        top[row, place] = torch.linspace(-39.0, -40.0, 8, device=DEV) + 8.0 * row
    index[4, 1:] = 17  # all but one
    top[4, 1:] = -45.0 + torch.rand(k - 1, generator=_gen(3)).to(DEV)
    z[:, 17] = -200.0
    first = _check_distill(z, top, index, by_row=by_row)[1]
    assert (first[:5, 17] < 0).all()
    for _ in range(4):
        assert torch.equal(first, _check_distill(z, top, index, by_row=by_row)[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("lost", [math.nan, math.inf])
@pytest.mark.parametrize("by_row", [False, True])
def test_a_teacher_without_a_distribution(lost, by_row, dtype):
    """A stored logit that is NaN or infinite leaves none of the row's stored entries a probability: their gradients are NaN, those of
    the other entries and rows what they are."""
    for n, v, k in ((12, 900, 7), (260, 9000, 300)):
        z, top, index = _distill_inputs(n, v, k, dtype, seed=v)
        index[:, 0] = 5
        top[2, 0], top[7, k - 1] = lost, lost
        loss, dz = _check_distill(z, top, index, by_row=by_row)
        assert dz[2, index[2]].isnan().all() and not dz[3].isnan().any()
        assert loss[[2, 7]].isnan().all() if by_row else loss.isnan()


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("n,v,k", [(3, 9001, 1024), (3, 9001, 2048), (3, 9001, 2049), (520, 6001, 2500), (9, 30000, 30000), (2, 300, 5000)])
def test_many_stored_entries(n, v, k, dtype):
    """Up to the whole vocabulary and beyond it: all different, some more than once, all the same."""
    for top_dtype in DTYPES:
        z, top, index = _distill_inputs(n, v, k, dtype, seed=k, top_dtype=top_dtype)
        index[0] = torch.arange(k, device=DEV) % v
        index[1] = torch.where(torch.rand(k, generator=_gen(n + k)).to(DEV) < 0.5, v - 1, index[1])
        index[-1, k // 3:] = -1
        scale = 1.0 if dtype != torch.float16 else 4096.0
        first = _check_distill(z, top, index, grad=0.5 * scale)  # (not the gradient that is made along with the loss)
        assert all(torch.equal(a, b) for a, b in zip(first, _check_distill(z, top, index, grad=0.5 * scale)))
        _check_distill(z, top, index, by_row=True, grad=torch.full((n,), scale))


@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -130, 2.0 ** 118, 2.0 ** 126])
def test_row_weights_of_any_size(size):
    """Of a mean only the ratios of the weights count, also where their sum, or one over it, is beyond the normal numbers of fp32."""
    n = 600
    weights = (1.0 + torch.randint(0, 2, (n,), generator=_gen(5)) * (torch.arange(n) > 2)).to(DEV)
    weights[3] = 0.0
    for dtype in DTYPES:
        z, top, index = _distill_inputs(n, 700, 9, dtype, seed=50)
        scale = 1.0 if dtype != torch.float16 else 4096.0
        loss, dz = _check_distill(z, top, index, weights, grad=scale)
        again, dz2 = _check_distill(z, top, index, weights * size, grad=scale)
        assert torch.equal(loss, again) and torch.equal(dz, dz2)


# ---- lookup --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_the_gradient_of_a_broadcast_scale_is_rounded_once(dtype):
    """Shares of tokens that nearly cancel, each of which a 16-bit type would round by more than is left of their sum."""
    n = 256
    w = torch.ones(3, 40, device=DEV, dtype=dtype)
    tokens = torch.arange(n, device=DEV) % 3
    dout = torch.zeros(n, 40, device=DEV, dtype=dtype)
    dout[:, 0] = torch.where(torch.arange(n, device=DEV) % 2 == 0, 1.0, -1.0).to(dtype)
    dout[::2, 1] = torch.finfo(dtype).eps * 0.375
    for shape in ((), (1,), (16, 1), (1, 16)):
        cube = tokens if len(shape) < 2 else tokens.view(16, 16)
        scale = torch.full(shape, 1.5, device=DEV, dtype=dtype, requires_grad=True)
        out = flex.embedding_lookup(cube, w, scale)
        assert out.dtype == dtype and out.eq(1.5).all()
        out.backward(dout.view(*cube.shape, 40))
        assert scale.grad.dtype == dtype and scale.grad.shape == scale.shape
        want, _ = ref.lookup(tokens, w, torch.full((n,), 1.5), 1.0, dout)
        shares = want["ds"].view(cube.shape)
        for axis, size in enumerate(shape if len(shape) == 2 else ()):
            if size == 1:
                shares = shares.sum(axis, keepdim=True)
        shares = shares.sum().view(shape) if len(shape) < 2 else shares
        many = n // scale.numel()  # (shares of at most 1 + 2^-8, added up in any order)
        ref.within(scale.grad, shares, ref.rounded(shares, dtype, many * (many + 4) * ref.U), str(shape))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("n,d", [(15, 3), (64, 100), (300, 130), (1000, 40), (700, 1537), (5000, 600)])
def test_tokens_that_are_no_row_among_those_of_row_zero(n, d, dtype):
    """They are filed under row 0: in every order, few and many, alone in a stretch of sorted places and beside it; with a row that
    the gradient is wanted for among them or none."""
    for kind, (rows, none) in enumerate([(1, 0.5), (3, 0.9), (2, 0.02), (1, 0.99), (5, 1.0)]):
        tokens, w, scale, dout = _lookup_inputs(n, rows, d, dtype, seed=n + kind, pad=0.0)
        away = torch.rand(n, generator=_gen(kind)).to(DEV) < none
        away[n // 2:n // 2 + 100] = True
        tokens[away] = torch.where(torch.arange(n, device=DEV) % 3 == 0, -1, -1 - rows)[away]
        dout[away] = math.nan
        scale[away] = math.inf
        _check_lookup(tokens, w, scale, dout)
        _check_lookup(tokens, w, None, dout)
    with pytest.raises(IndexError, match="token"):
        flex.check_index_flag()


def test_rows_of_the_gradient_behind_the_last_token_are_not_needed():
    """A padded batch whose upstream gradient ends with its tokens, by the library's entry point, which promises not to read rows of
    tokens that are none."""
    n, there, d = 1000, 421, 256
    tokens, w, scale, dout = _lookup_inputs(n, 7, d, torch.float32, seed=3, pad=0.1)
    tokens[there:] = -1
    short = dout[:there].clone()
    dweight, dscale = torch.full_like(w, 7.0), torch.full_like(scale, 7.0)
    lib = _lib.load()
    lookup = ctypes.byref(_lib.Lookup(n, 7, d, d, d, 1.0, _lib.F32, _lib.F32))
    nbytes = lib.flexsae_lookup_bwd_workspace_bytes(lookup)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.flexsae_lookup_bwd(lookup, at(tokens), at(w), at(scale), at(short), at(dweight), at(dscale), at(workspace), nbytes,
                                  stream) == _lib.OK
    want, tol = ref.lookup(tokens, w, scale, 1.0, dout)
    ref.within(dweight, want["dw"], ref.rounded(want["dw"], torch.float32, tol["dw"]), "dw")
    ref.within(dscale, want["ds"], ref.rounded(want["ds"], torch.float32, tol["ds"]), "ds")


# ---- the flag ------------------------------------------------------------------------------


def test_the_flag_names_all_that_was_out_of_range():
    w = torch.randn(10, 24, device=DEV)
    flex.embedding_lookup(torch.tensor([3, 10], device=DEV), w)
    flex.triton_topk_sae_loss(torch.tensor([[1, 10]], device=DEV), w, torch.ones(1, 2, device=DEV), torch.zeros(24, device=DEV),
                              torch.zeros(1, 24, device=DEV))
    with pytest.raises(IndexError, match=r"(?s)`indices`.*token"):
        flex.check_index_flag()
    flex.check_index_flag()


# ---- long tables ---------------------------------------------------------------------------


@pytest.mark.parametrize("v", [(1 << 26) - 3, (1 << 26) + 5, (1 << 27) + 11])
def test_the_same_bits_for_long_tables(v):
    """A table's gradient by sorted tokens at its end, where the lists of rows are more than a grid has threads along an axis."""
    n, d = 200_000, 2
    g = torch.Generator(DEV).manual_seed(1)
    w = torch.zeros(v, d, device=DEV, requires_grad=True)
    low = torch.randint(0, 4000, (n,), generator=g, device=DEV)
    dout = torch.randn(n, d, generator=g, device=DEV)
    out = flex.embedding_lookup(low + (v - 4000), w)
    runs = [torch.autograd.grad(out, w, dout, retain_graph=True)[0] for _ in range(3)]
    assert all(torch.equal(runs[0], r) for r in runs[1:])
    few = torch.zeros(4000, d, device=DEV, requires_grad=True)
    want, = torch.autograd.grad(flex.embedding_lookup(low, few), few, dout)
    assert torch.equal(runs[0][-4000:], want) and not runs[0][:-4000].any()


# ---- compiled calls ------------------------------------------------------------------------


@pytest.mark.parametrize("dynamic", [True, None])
def test_compiled_calls_of_changing_sizes_and_numbers(dynamic):
    def chain(x, w, tokens, table, scale, top, index, out, temperature, eps):
        z = flex.layer_norm(x + flex.embedding_lookup(tokens, table, scale), w, eps=eps) @ out
        return flex.distillation_loss(z, top, index, row_weights=tokens >= 0, temperature=temperature) + flex.distillation_loss(z, top, index)

    compiled = torch.compile(chain, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    g = _gen(60)
    for n, scale, temperature, eps in ((7, 1.5, 1.0, 1e-5), (12, 0.5, 2.0, 1e-6), (33, 3, 0.7, 1e-3), (33, 2, 3, 1e-4)):
        x, w, table, out, top = (torch.randn(s, generator=g).to(DEV) for s in ((n, 64), (64,), (9, 64), (64, 70), (n, 4)))
        tokens, index = torch.randint(-1, 9, (n,), generator=g).to(DEV), torch.randint(0, 70, (n, 4), generator=g).to(DEV)
        leaves = [t.requires_grad_() for t in (x, w, table, out)]
        results = []
        for fn in (chain, compiled):
            loss = fn(x, w, tokens, table, scale, top, index, out, temperature, eps)
            results.append([loss, *torch.autograd.grad(loss, leaves)])
        for a, b in zip(*results):  # (the ops take gradients of a mean from other partial sums: rounding errors of sums of 70 terms)
            assert (a - b).norm() <= 200 * ref.U * a.norm()


def test_forward_mode_is_refused():
    x, tokens = torch.randn(6, 40, device=DEV), torch.randint(0, 6, (5,), device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda t: flex.layer_norm(t), lambda t: flex.layer_norm(x, t[0]), lambda t: flex.layer_norm_stats(t),
                     lambda t: flex.embedding_lookup(tokens, t), lambda t: flex.embedding_lookup(tokens, x, t[0, :5]),
                     lambda t: flex.distillation_loss(t, x[:, :3], tokens.new_zeros(6, 3))):
            call(x)
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
