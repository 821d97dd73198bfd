"""AdamW steps, the gradients' norm and 8-bit states against their formulas in 64 bits (optim_reference.py has the bounds)."""
import itertools
import random

import pytest
import torch

import flexsae_amd as flex
from tests import optim_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


class Problem:
    """Tensors of a step over `shapes`; `views`: at odd places of larger buffers."""

    def __init__(self, shapes, dtypes, bits, unit=False, master=False, seed=0, views=False, scale=1.0, g_std=1e-3, fresh=False):
        g = _gen(seed)
        self.bits, self.unit, self.shapes = bits, unit, shapes
        dtypes = dtypes if isinstance(dtypes, list) else [dtypes] * len(shapes)

        def place(x, odd=1):
            if not views or x.numel() == 0:
                return x
            buf = torch.zeros(x.numel() + 16, dtype=x.dtype, device=DEV)
            out = buf[odd:odd + x.numel()].view(x.shape)
            out.copy_(x)
            return out

        def randn(shape):
            return torch.randn(shape, generator=g, device=DEV)

        self.params, self.grads, self.s0, self.s1, self.masters = [], [], [], [], []
        for shape, dt in zip(shapes, dtypes):
            w = randn(shape) * 0.05
            if unit and w.numel():
                w /= w.norm(dim=-1, keepdim=True).clamp_min(1e-20)
            self.masters.append(place(w.clone()))
            self.params.append(place(w.to(dt)))
            std = torch.exp(randn((*shape[:-1], 1)))
            self.grads.append(place((randn(shape) * std * g_std * scale).to(dt), 3))
            if bits == 32:
                m, v = randn(shape) * 0.3 * g_std, (randn(shape) * g_std).square()
                self.s0.append(place(m * (not fresh)))
                self.s1.append(place(v * (not fresh)))
            else:
                codes, absmax = flex.adamw8_state(self.params[-1], unit)
                if not fresh:
                    codes.random_(0, 256, generator=g)
                    codes[..., 0].clamp_(1, 255)
                    absmax.uniform_(0.5, 2.0, generator=g).mul_(torch.tensor([g_std, g_std ** 2], device=DEV))
                codes = place(codes, 2)
                self.s0.append(codes)
                self.s1.append(place(absmax, 2))
        self.master = master
        self.counter = flex.adamw_counter(DEV, 0 if fresh else 7)

    def step(self, **kw):
        fn = flex.adamw_step if self.bits == 32 else flex.adamw8_step
        fn(self.params, self.grads, self.s0, self.s1, self.counter, masters=self.masters if self.master else None,
           unit_rows=self.unit, **kw)

    def tensors(self):
        return [*self.params, *self.s0, *self.s1, *(self.masters if self.master else []), self.counter]

    def moments(self, i):
        shape = ref.layout(self.shapes[i], self.unit)
        if self.bits == 32:
            return self.s0[i].reshape(shape).double(), self.s1[i].reshape(shape).double()
        return ref.decode(self.s0[i], self.s1[i], self.unit)

    def held(self, i):
        return (self.masters if self.master and self.params[i].dtype != F32 else self.params)[i]

    def checked_step(self, c=1.0, lr=1e-3, wd=0.01, betas=(0.9, 0.999), eps=1e-8, lrs=None, wds=None, **kw):
        """A step, each tensor against the formula on the state before it."""
        before = [(self.held(i).reshape(ref.layout(s, self.unit)).double().clone(), *(x.clone() for x in self.moments(i)))
                  for i, s in enumerate(self.shapes)]
        grads = [x.clone() for x in self.grads]
        t = int(self.counter[0]) + 1
        self.step(lr=lrs or lr, weight_decay=wds or wd, beta1=betas[0], beta2=betas[1], eps=eps, **kw)
        assert int(self.counter[0]) == t
        for i, shape in enumerate(self.shapes):
            if self.params[i].numel() == 0:
                continue
            R, C = ref.layout(shape, self.unit)
            w, m, v = before[i]
            a = float(lr) if lrs is None else float(lrs[i])
            w2, m2, v2, dw, dm, dv = ref.step(w, grads[i].reshape(R, C), m, v, t, a, *betas, eps, wd if wds is None else wds[i], c,
                                              self.unit)
            assert torch.equal(grads[i], self.grads[i])
            dt = self.params[i].dtype
            ref.within(self.held(i).reshape(R, C), w2, dw if self.held(i).dtype == F32 else ref.rounded(w2, dw, dt), "weight")
            if self.master and dt != F32:
                assert torch.equal(self.params[i], self.masters[i].to(dt))
            if self.bits == 32:
                ref.within(self.s0[i].reshape(R, C), m2, dm, "m")
                ref.within(self.s1[i].reshape(R, C), v2, dv, "v")
            else:
                # (the reference decodes in 64 bits: the kernels' decoding adds four roundings to m and v)
                ref.check_codes(self.s0[i], self.s1[i], m2, v2, dm + 8 * ref.U * m.abs(), dv + 8 * ref.U * v, self.unit)


SIZES = [(1,), (7,), (8,), (9,), (255,), (256,), (257,), (511,), (2047,), (2048,), (2049,), (3, 5, 7), (33, 129), (131, 1538)]
TYPES = [(F32, False), (BF16, False), (BF16, True), (F16, False), (F16, True)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", TYPES)
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_step_of_one_tensor(shape, dtype, master, bits):
    p = Problem([shape], dtype, bits, master=master, seed=sum(shape))
    for _ in range(2):
        p.checked_step()


@pytest.mark.parametrize("bits", [32, 8])
def test_first_steps_from_nothing(bits):
    p = Problem([(300, 70), (70,)], F32, bits, fresh=True)
    for _ in range(4):
        p.checked_step()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("betas,eps", [((0.0, 0.0), 1e-8), ((0.95, 0.5), 1e-3), ((0.0, 0.9999), 1e-12)])
def test_other_betas(betas, eps, bits):
    p = Problem([(37, 41)], F32, bits)
    p.checked_step(betas=betas, eps=eps)


@pytest.mark.parametrize("steps", [0, 9, 100, 499, 501, 4999, 10 ** 7, 2 ** 40])
def test_bias_corrections_early_and_late(steps):
    """On either side of where the series ends (t log b = -0.5), and where the powers are gone."""
    for bits in (32, 8):
        p = Problem([(33, 70)], F32, bits, seed=steps % 97)
        p.counter = flex.adamw_counter(DEV, steps)
        p.checked_step()
        assert int(p.counter[0]) == steps + 1


@pytest.mark.parametrize("bits", [32, 8])
def test_no_gradient_ever_and_no_eps(bits):
    """0 / 0 moves nothing."""
    p = Problem([(5, 300)], F32, bits, fresh=True)
    p.grads[0][2:] = 0.0
    w = p.params[0].clone()
    p.step(eps=0.0, lr=1e-2)
    assert torch.equal(p.params[0][2:], w[2:])
    moved = (p.params[0][:2] - w[:2]) / (-1e-2 * p.grads[0][:2].sign())
    assert torch.allclose(moved, torch.ones_like(moved), rtol=1e-4)  # the first step is the sign (of weights of 0.05, rounded)


ROWS = [1, 2, 48, 63, 64, 65, 100, 128, 255, 256, 257, 511, 512, 513, 1024, 1025, 1536, 1538, 2304, 2560, 2561, 4096, 4099, 8192,
        8193, 16384, 16390, 20001, 33001]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", TYPES)
@pytest.mark.parametrize("cols", ROWS)
def test_unit_rows(cols, dtype, master, bits):
    # (a row of one column has no direction but its own: nothing is left of the gradient)
    for rows in (1, 5, 67) if cols < 5000 else (1, 6):
        p = Problem([(rows, cols)], dtype, bits, unit=True, master=master, seed=cols)
        p.checked_step()
        if p.held(0).dtype == F32:
            length = p.held(0).double().norm(dim=1)
            assert bool(((length - 1).abs() < 1e-5).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_unit_rows_of_zeros_and_of_other_lengths(bits):
    p = Problem([(6, 300), (2, 3, 129)], F32, bits, unit=True, fresh=True)
    for x in p.params:
        x.view(-1, x.shape[-1])[1] *= 3.0
    p.params[0][2] = 0.0
    p.grads[0][2:4] = 0.0
    p.checked_step(wd=0.0)
    assert bool((p.params[0][2] == 0).all())
    assert abs(float(p.params[1].view(-1, 129)[1].norm()) - 1) < 1e-5


def _many(seed, n=150):
    r = random.Random(seed)
    return [(r.choice([0, 1, 3, 64, 100, 257]), r.choice([1, 2, 67, 256, 300])) for _ in range(n)]


@pytest.mark.parametrize("bits,unit,views", itertools.product([32, 8], [False, True], [False, True]))
def test_many_tensors_of_many_types(bits, unit, views):
    shapes = _many(bits + unit)
    r = random.Random(3)
    p = Problem(shapes, [r.choice([F32, BF16, F16]) for _ in shapes], bits, unit=unit, master=True, views=views)
    n = len(shapes)
    p.checked_step(lrs=[1e-3 * (1 + i % 5) for i in range(n)], wds=[0.01 * (i % 3) for i in range(n)])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("views", [False, True])
def test_more_tiles_than_blocks(bits, views):
    p = Problem([(4099, 1027), (5, 7), (2300, 2304)], [BF16, F32, BF16], bits, master=bits == 32, views=views)
    p.checked_step()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("unit", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_clipping_and_loss_scale(bits, unit, max_norm):
    p = Problem([(123, 200), (40, 300)], F16, bits, unit=unit, master=True, scale=65536.0, g_std=1e-2)
    norm = flex.grad_norm(p.grads)
    want = float(torch.cat([g.double().flatten() for g in p.grads]).norm())
    assert abs(float(norm) / want - 1) < 2 * ref.U
    p.checked_step(c=ref.factor(want, 65536.0, max_norm), grad_norm=norm, max_norm=max_norm, grad_scale=65536.0)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("unit", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_norm_that_is_not_finite_changes_nothing(bits, unit, bad):
    p = Problem([(50, 300), (60, 3000)], BF16, bits, unit=unit, master=True)
    p.grads[1][17, 5] = bad
    norm = flex.grad_norm(p.grads)
    assert not torch.isfinite(norm)
    before = [x.clone() for x in p.tensors()]
    p.step(grad_norm=norm, max_norm=1.0)
    p.step(grad_norm=norm)
    for x, y in zip(before, p.tensors()):
        assert torch.equal(x, y)
    p.grads[1][17, 5] = 1e-3
    p.checked_step()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_infinities_stay_where_they_are(bad):
    """Without a norm: in 32 bits in their element, in 8 bits in their block."""
    p = Problem([(4, 1000)], F32, 32)
    p.grads[0].view(-1)[777] = bad
    p.step()
    for x in (p.s0[0], p.s1[0]):
        assert (~torch.isfinite(x)).view(-1).nonzero().flatten().tolist() == [777]
    assert (~torch.isfinite(p.params[0])).view(-1).nonzero().flatten().tolist() == [777]
    p = Problem([(4, 1000)], F32, 8)
    p.grads[0].view(-1)[777] = bad
    p.step()
    assert (~torch.isfinite(p.params[0])).view(-1).nonzero().flatten().tolist() == [777]
    for x in flex.adamw8_moments(p.s0, p.s1):
        assert torch.isnan(x[0].view(-1)).nonzero().flatten().tolist() == list(range(768, 1024))


def test_values_at_the_ends_of_the_range():
    """Maxima below the smallest normal number are kept as zero; large ones do not overflow on the way."""
    p = Problem([(1024,)], F32, 8, fresh=True)
    p.params[0].zero_()
    p.grads[0].zero_()
    p.grads[0][:256] = 1e-37   # v vanishes, m stays
    p.grads[0][256:512] = 1e18  # v = 1e33
    p.grads[0][512] = 1e-30
    p.step(eps=1e-8)
    m, v = (x[0].double() for x in flex.adamw8_moments(p.s0, p.s1))
    assert torch.allclose(m[:256], torch.full_like(m[:256], 1e-38), rtol=1e-5) or bool((m[:256] == 0).all())
    assert bool((v[:256] == 0).all())
    assert torch.allclose(m[256:512], torch.full_like(m[:256], 1e17), rtol=1e-5)
    assert torch.allclose(v[256:512], torch.full_like(m[:256], 1e33), rtol=1e-5)
    assert abs(float(m[512]) / 1e-31 - 1) < 1e-5 and float(m[513:].abs().max()) == 0
    assert torch.isfinite(p.params[0]).all()


def test_equal_decay_leaves_the_codes():
    p = Problem([(3, 700)], F32, 8)
    p.step()
    p.grads[0].zero_()
    codes = p.s0[0].clone()
    for _ in range(5):
        p.step()
    # the block's largest has the highest code from the first step on, and all others keep their share of it
    assert torch.equal(codes, p.s0[0])


def test_learning_rate_on_the_device_and_lists():
    for bits in (32, 8):
        a, b = (Problem([(70, 90), (90,)], F32, bits, seed=5) for _ in range(2))
        a.step(lr=torch.tensor(2.5e-3, device=DEV), weight_decay=0.1)
        b.step(lr=[2.5e-3, 2.5e-3], weight_decay=(0.1, 0.1))
        for x, y in zip(a.tensors(), b.tensors()):
            assert torch.allclose(x.double(), y.double(), rtol=4 * ref.U, atol=0)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_are_not_contiguous(bits):
    a, b = (Problem([(70, 90), (40, 66)], F32, bits, seed=6) for _ in range(2))
    for x in (b.params, b.grads, b.s0, b.s1):
        for i, t in enumerate(x):
            # every other column of a wider buffer, and a transposed one
            if i == 0:
                wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype, device=DEV)
                y = wide[..., ::2]
            else:
                y = torch.empty(*t.shape[::-1], dtype=t.dtype, device=DEV).permute(*reversed(range(t.dim())))
            x[i] = y.copy_(t)
            assert not x[i].is_contiguous() or t.shape[-1] == 1
    a.step()
    b.step()
    for x, y in zip(a.tensors(), b.tensors()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_same_bits_through_the_op_and_on_another_stream(bits):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    problems = [Problem([(700, 900), (900,)], BF16, bits, master=True, seed=9) for _ in range(3)]
    norms = []
    for how, p in enumerate(problems):
        stream = torch.cuda.Stream() if how == 2 else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            if how == 1:
                with Watch():
                    norms.append(flex.grad_norm(p.grads))
                    p.step(grad_norm=norms[-1], max_norm=0.1)
            else:
                norms.append(flex.grad_norm(p.grads))
                p.step(grad_norm=norms[-1], max_norm=0.1)
        torch.cuda.synchronize()
    assert any("adamw" in s for s in Watch.seen) and any("grad_norm" in s for s in Watch.seen)
    for p, norm in zip(problems[1:], norms[1:]):
        assert torch.equal(norm, norms[0])
        for x, y in zip(problems[0].tensors(), p.tensors()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_of_a_captured_step(bits):
    a, b = (Problem([(300, 400), (400,)], BF16, bits, master=True, seed=11) for _ in range(2))
    lr = torch.tensor(1e-3, device=DEV)

    def one(p):
        norm = flex.grad_norm(p.grads)
        p.step(lr=lr, grad_norm=norm, max_norm=0.1)
        return norm

    one(a)
    one(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = one(b)
    for i in range(4):
        for p in (a, b):
            g = _gen(100 + i)
            for x in p.grads:
                x.copy_(torch.randn(x.shape, generator=g, device=DEV) * (float("inf") if i == 2 else 1e-3))
        lr.fill_(1e-3 / (i + 1))
        want = one(a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, norm) or bool(want.isnan() & norm.isnan())
        for x, y in zip(a.tensors(), b.tensors()):
            assert torch.equal(x, y), i
    assert int(a.counter[0]) == 11  # seven, one, and three of four


def test_versions_move():
    p = Problem([(30, 40)], F32, 32)
    versions = [x._version for x in p.tensors()]
    g = p.grads[0]._version
    p.step()
    assert all(x._version > v for x, v in zip(p.tensors(), versions)) and p.grads[0]._version == g


def test_offsets_beyond_32_bits():
    """2^32 + 555 elements in one tensor: pieces about the places where narrower numbers end, and the end itself."""
    n = 2 ** 32 + 555
    params = [torch.zeros(n, dtype=BF16, device=DEV)]
    grads = [torch.zeros(n, dtype=BF16, device=DEV)]
    codes, absmax = flex.adamw8_state(params[0])
    pieces = [slice(a, min(n, a + 4096)) for a in (0, 2 ** 30 - 2048, 2 ** 31 - 2048, 2 ** 32 - 2048)]
    g = _gen(2)
    for s in pieces:
        params[0][s] = torch.randn(s.stop - s.start, generator=g, device=DEV).to(BF16)
        grads[0][s] = torch.randn(s.stop - s.start, generator=g, device=DEV).to(BF16)
    before = [params[0][s].clone() for s in pieces]
    norm = flex.grad_norm(grads)
    want = float(grads[0][:2 ** 20].double().square().sum() + sum(grads[0][s].double().square().sum() for s in pieces[1:])) ** 0.5
    assert abs(float(norm) / want - 1) < 2 * ref.U
    flex.adamw8_step(params, grads, [codes], [absmax], flex.adamw_counter(DEV), lr=1e-2)
    for s, w in zip(pieces, before):
        k = s.stop - s.start
        zero = torch.zeros(1, k, device=DEV)
        w2, m2, v2, dw, dm, dv = ref.step(w.view(1, k), grads[0][s].view(1, k), zero, zero, 1, 1e-2)
        ref.within(params[0][s].view(1, k), w2, ref.rounded(w2, dw, BF16), s)
        assert s.start % 256 == 0
        ref.check_codes(codes[s], absmax[:, s.start // 256:-(-s.stop // 256)], m2, v2, dm, dv, False)
    m, v = flex.adamw8_moments([codes], [absmax], BF16)
    at = slice(n - 300, n)
    want_m, _ = ref.decode(codes[at.start - at.start % 256:], absmax[:, at.start // 256:], False)
    assert torch.equal(m[0][at.start - at.start % 256:], want_m[0].to(F32).to(BF16)) or torch.allclose(
        m[0][at.start - at.start % 256:].double(), want_m[0], rtol=2.0 ** -8, atol=0)


# ---- the norm ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[1], [0, 5], [2047], [2048, 1, 2049], [3_000_001], [0]], ids=str)
def test_norm(sizes, dtype):
    g = _gen(len(sizes))
    grads = [torch.randn(n, generator=g, device=DEV).to(dtype) for n in sizes]
    want = float(torch.cat([x.double() for x in grads]).norm())
    got = flex.grad_norm(grads)
    assert got.shape == () and got.dtype == F32
    # a sum in 64 bits of exact squares, its root, and one rounding to fp32
    assert abs(float(got) - want) <= 1.01 * ref.U * want
    assert torch.equal(got, flex.grad_norm(grads))


def test_norm_of_many_tensors_of_many_types():
    g = _gen(1)
    r = random.Random(1)
    buf = torch.randn(400_000, generator=g, device=DEV)
    grads = [(torch.randn(n, generator=g, device=DEV) * 10.0 ** r.randint(-3, 1)).to(r.choice([F32, BF16, F16]))
             for n in (r.choice([0, 1, 7, 100, 5000]) for _ in range(300))]
    grads += [buf[1:1001], buf[2000:12000].view(100, 100).t(), buf[::7]]
    want = float(torch.cat([x.double().flatten() for x in grads]).norm())
    assert abs(float(flex.grad_norm(grads)) - want) <= 1.01 * ref.U * want
    assert abs(float(flex.grad_norm(tuple(grads))) - want) <= 1.01 * ref.U * want


def test_norm_of_large_and_small_numbers():
    x = torch.full((10_000,), 1e30, device=DEV)
    assert abs(float(flex.grad_norm([x])) / 1e32 - 1) < 1e-6
    x = torch.full((10_000,), 1e-40, device=DEV)
    assert abs(float(flex.grad_norm([x])) / float(x.double().norm()) - 1) < 1e-3  # (itself below the normal numbers)
    x = torch.full((4,), 3e38, device=DEV)
    assert float(flex.grad_norm([x])) == float("inf")  # 6e38 is none of fp32's numbers
    x = torch.zeros(10_000, device=DEV)
    assert float(flex.grad_norm([x])) == 0
    x[7777] = float("-inf")
    assert float(flex.grad_norm([x])) == float("inf")
    x[1] = float("nan")
    assert flex.grad_norm([x]).isnan()


# ---- the values of 8-bit states ------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("unit", [False, True])
def test_moments(dtype, unit):
    shapes = [(1, 1), (3, 255), (70, 256), (5, 7, 129), (9, 2309), (200, 67), (0, 5), (6, 8200), (33, 264)]
    p = Problem(shapes, F32, 8, unit=unit, g_std=1.0)
    ms, vs = flex.adamw8_moments(p.s0, p.s1, dtype)
    for i, shape in enumerate(shapes):
        assert ms[i].shape == shape and ms[i].dtype == dtype and vs[i].dtype == dtype
        if not ms[i].numel():
            continue
        for got, want in zip((ms[i], vs[i]), ref.decode(p.s0[i], p.s1[i], unit)):
            # five roundings in fp32 and the one to the type
            bound = 6 * ref.U * want.abs()
            ref.within(got.reshape(want.shape), want, bound if dtype == F32 else ref.rounded(want, bound, dtype), shape)


# ---- the optimizer -------------------------------------------------------------------------


def _model(dtype=F32, seed=0):
    g = _gen(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g, device=DEV) * 0.05).to(dtype))
            for s in ((300, 70), (300,), (300, 70), (70,))]


def _set_grads(params, seed, std=1e-3, but=()):
    g = _gen(seed)
    for i, p in enumerate(params):
        x = torch.randn(p.shape, generator=g, device=DEV) * std
        p.grad = None if i in but else x.to(p.dtype)


def test_optimizer_follows_torch():
    a, b = _model(), _model()
    mine = flex.AdamW([{"params": a[:2]}, {"params": a[2:], "lr": 3e-3, "weight_decay": 0.1}], lr=1e-3, max_norm=0.02)
    its = torch.optim.AdamW([{"params": b[:2]}, {"params": b[2:], "lr": 3e-3, "weight_decay": 0.1}], lr=1e-3)
    schedules = [torch.optim.lr_scheduler.StepLR(o, 3) for o in (mine, its)]
    for i in range(10):
        for x in (a, b):
            _set_grads(x, i)
        norm = torch.nn.utils.clip_grad_norm_(b, 0.02)
        loss = mine.step(lambda: torch.ones(()))
        assert loss == 1 and abs(float(mine.grad_norm / norm) - 1) < 1e-5
        its.step()
        for s in schedules:
            s.step()
        for x, y in zip(a, b):
            # ten steps of at most 3e-3, each off by a few roundings of the update
            assert torch.allclose(x, y, rtol=1e-6, atol=3e-7)


@pytest.mark.parametrize("bits,dtype,unit", [(32, F32, False), (8, BF16, False), (8, F32, True), (32, F16, True)])
def test_state_dict_goes_on_where_it_was(bits, dtype, unit, tmp_path):
    def make(params):
        return flex.AdamW([{"params": params[::2], "unit_rows": unit}, {"params": params[1::2]}], state_bits=bits, max_norm=1.0)

    a = _model(dtype)
    one = make(a)
    for i in range(3):
        _set_grads(a, i, but=(1,) if i == 0 else ())
        one.step()
    torch.save(one.state_dict(), tmp_path / "state.pt")
    b = _model(dtype)
    for x, y in zip(a, b):
        y.data.copy_(x.data)
    two = make(b)
    two.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    for i in range(3, 6):
        for x, opt in ((a, one), (b, two)):
            _set_grads(x, i)
            opt.step()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
        for k, s in one.state[x].items():
            assert torch.equal(s, two.state[y][k]) and s.dtype == two.state[y][k].dtype, k
        m, v = two.moments(y)
        assert m.shape == y.shape and m.dtype == F32 and bool((v >= 0).all())
    # counts: one for the parameters of a group that have taken the same steps
    assert int(one.state[a[1]]["counter"][0]) == 5 and int(one.state[a[3]]["counter"][0]) == 6
    assert two.state[b[0]]["counter"] is two.state[b[2]]["counter"]


def test_parameters_without_a_gradient_keep_their_count():
    a, b = _model(), _model()
    mine, its = flex.AdamW(a, lr=1e-2), torch.optim.AdamW(b, lr=1e-2)
    for i, but in enumerate([(), (2,), (0, 2), (), (1,), ()]):
        for x, opt in ((a, mine), (b, its)):
            _set_grads(x, i, but=but)
            opt.step()
        for x, y in zip(a, b):
            assert torch.allclose(x, y, rtol=1e-6, atol=1e-6)
    assert [int(mine.state[p]["counter"][0]) for p in a] == [5, 5, 4, 6]


def test_skipped_steps_and_no_steps():
    a = _model(BF16)
    opt = flex.AdamW(a, skip_nonfinite=True)
    opt.step()  # no gradients: nothing to do
    assert not opt.state
    before = [p.detach().clone() for p in a]
    _set_grads(a, 0)
    a[2].grad[1, 1] = float("nan")
    opt.step()
    assert opt.grad_norm.isnan() and all(torch.equal(x, y) for x, y in zip(before, a))
    _set_grads(a, 0, std=65.536)
    opt.step(grad_scale=65536.0)
    assert int(opt.state[a[0]]["counter"][0]) == 1
    assert all(torch.equal(opt.state[p]["master"].to(BF16), p) for p in a)


def test_gradients_of_the_losses_go_in():
    """The framework's own path: a loss, its backward, the step."""
    torch.manual_seed(0)
    B, K, F, D = 64, 8, 512, 64
    W = torch.nn.Parameter(torch.randn(F, D, device=DEV))
    W.data /= W.data.norm(dim=1, keepdim=True)
    bias = torch.nn.Parameter(torch.zeros(D, device=DEV))
    target = torch.randn(B, D, device=DEV)
    opt = flex.AdamW([{"params": [W], "unit_rows": True}, {"params": [bias]}], lr=1e-2, weight_decay=0.0, max_norm=10.0, state_bits=8)
    losses = []
    for _ in range(30):
        vals, idx = (target @ W.detach().t()).topk(K)
        loss = flex.triton_hierarchical_sae_loss(idx, W, vals, bias, target)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.8 * losses[0]
    assert bool(((W.detach().norm(dim=1) - 1).abs() < 1e-5).all())


def test_ops_pass_torchs_own_checks():
    p = Problem([(20, 30), (30,)], F32, 32)
    torch.library.opcheck(torch.ops.flexsae_amd.grad_norm.default, (p.grads,))
    args = (p.params, p.grads, p.s0, p.s1, [], p.counter, [1e-3] * 2, [0.0] * 2, None, None, 0.9, 0.999, 1e-8, 1.0, 0.0, False)
    torch.library.opcheck(torch.ops.flexsae_amd.adamw_step_.default, args)
    p = Problem([(20, 30), (30,)], F32, 8)
    torch.library.opcheck(torch.ops.flexsae_amd.adamw8_step_.default, (p.params, p.grads, p.s0, p.s1, *args[4:5], p.counter, *args[6:]))
    torch.library.opcheck(torch.ops.flexsae_amd.adamw8_moments.default, (p.s0, p.s1, BF16))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_compiled_step(bits):
    """Traced calls see the ops: no break in the graph, the same bits."""
    a, b = (Problem([(60, 70), (70,)], BF16, bits, master=True, seed=13) for _ in range(2))

    @torch.compile(fullgraph=True)
    def compiled(params, grads, s0, s1, masters, counter):
        norm = flex.grad_norm(grads)
        (flex.adamw_step if bits == 32 else flex.adamw8_step)(params, grads, s0, s1, counter, masters=masters, lr=1e-2, grad_norm=norm,
                                                              max_norm=0.1)
        return norm * 2

    for _ in range(2):
        norm = flex.grad_norm(a.grads)
        a.step(lr=1e-2, grad_norm=norm, max_norm=0.1)
        assert torch.equal(compiled(b.params, b.grads, b.s0, b.s1, b.masters, b.counter), norm * 2)
        for x, y in zip(a.tensors(), b.tensors()):
            assert torch.equal(x, y)


# ---- refusals ------------------------------------------------------------------------------


def test_refusals():
    def problem(bits=32, **kw):
        return Problem([(20, 30), (30,)], kw.pop("dtype", F32), bits, **kw)

    for bits in (32, 8):
        for change, error in (
                (lambda p: p.grads.pop(), ValueError), (lambda p: p.s0.pop(), ValueError),
                (lambda p: p.grads.__setitem__(0, p.grads[0][:19]), ValueError),
                (lambda p: p.grads.__setitem__(0, p.grads[0].half()), ValueError),
                (lambda p: p.s0.__setitem__(0, p.s0[0][:, :29]), ValueError),
                (lambda p: p.s1.__setitem__(1, p.s1[1].double()), ValueError),
                (lambda p: p.params.__setitem__(0, p.params[0].double()), TypeError),
                (lambda p: p.grads.__setitem__(1, p.grads[1].cpu()), RuntimeError),
                (lambda p: setattr(p, "counter", p.counter.int()), ValueError),
                (lambda p: setattr(p, "counter", p.counter[:1]), ValueError),
                (lambda p: (p.params.clear(), p.grads.clear()), ValueError)):
            p = problem(bits)
            change(p)
            before = [x.clone() for x in p.tensors()]
            with pytest.raises(error):
                p.step()
            assert all(torch.equal(x, y) for x, y in zip(before, p.tensors()))
        for kw in ({"beta1": 1.0}, {"beta2": -0.1}, {"eps": -1e-8}, {"eps": float("nan")}, {"lr": -1.0}, {"lr": float("nan")},
                   {"weight_decay": -1.0}, {"grad_scale": 0.0}, {"grad_scale": float("inf")}, {"max_norm": 1.0},
                   {"max_norm": -1.0, "grad_norm": torch.ones((), device=DEV)}, {"lr": [1e-3]},
                   {"lr": torch.ones((), device=DEV, dtype=torch.float64)}, {"grad_norm": torch.ones(2, device=DEV)}):
            p = problem(bits)
            before = [x.clone() for x in p.tensors()]
            with pytest.raises(ValueError):
                p.step(**kw)
            assert all(torch.equal(x, y) for x, y in zip(before, p.tensors())), kw
        p = problem(bits, dtype=BF16)
        p.master, p.masters[0] = True, p.masters[0].half()
        with pytest.raises(ValueError):
            p.step()
        p = problem(bits)
        p.unit = True  # (a vector has no rows)
        with pytest.raises(ValueError):
            p.step()
    with pytest.raises(TypeError):
        flex.grad_norm([torch.ones(3, device=DEV, dtype=torch.float64)])
    with pytest.raises(ValueError):
        flex.grad_norm([])
    p = problem(8)
    for codes, absmax, error in (([p.s0[0]], [], ValueError), ([], [], ValueError), ([p.s0[0][:19]], [p.s1[0][:, :2]], ValueError),
                                 ([p.s0[0].int()], [p.s1[0]], ValueError)):
        with pytest.raises(error):
            flex.adamw8_moments(codes, absmax)
    with pytest.raises(TypeError):
        flex.adamw8_moments([p.s0[0]], [p.s1[0]], torch.float64)


@pytest.mark.parametrize("bits,dtype", [(32, F32), (8, BF16), (8, F16)])
def test_the_example(bits, dtype):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_sae.py")
    spec = importlib.util.spec_from_file_location("train_sae", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, model, opt = example.train(F=512, D=64, K=8, B=128, steps=60, bits=bits, dtype=dtype, lr=3e-3)
    assert losses[-1] < 0.8 * losses[0]
    # (rounding a row of length one to 16 bits moves its length by less than the rounding of a number)
    assert float((model.W_dec.detach().double().norm(dim=1) - 1).abs().max()) < {F32: 1e-5, BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
    assert int(opt.state[model.W_dec]["counter"][0]) == 60
