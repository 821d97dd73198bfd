"""AdamW steps where squares overflow or vanish, and codes of 8-bit states at both ends of the range."""
import pytest
import torch

import flexsae_amd as flex
from tests import optim_reference as ref
from tests.test_optim_gpu import BF16, DEV, F16, F32, Problem

pytestmark = pytest.mark.gpu

# a NaN in v: bits, type, master, columns of a row (0: as stored); four and eight elements a lane, held and walked rows
FORMS = [(32, F32, False, 0), (32, BF16, True, 0), (32, F32, False, 300), (32, F32, False, 40), (32, F32, False, 20001),
         (8, F32, False, 0), (8, BF16, False, 0), (8, BF16, True, 0), (8, F16, False, 0), (8, F32, False, 300), (8, BF16, False, 300),
         (8, BF16, False, 100), (8, BF16, False, 20001)]


@pytest.mark.parametrize("bits,dtype,master,cols", FORMS)
def test_a_v_that_is_nan_reaches_the_weight(bits, dtype, master, cols):
    """... of its element (32 bits), or of its block (8 bits), with an m that is finite."""
    p = Problem([(3, cols)] if cols else [(4, 1000)], dtype, bits, unit=cols > 0, master=master)
    bad = torch.zeros(p.params[0].shape, dtype=torch.bool, device=DEV)
    if bits == 32:
        p.s1[0].view(-1)[37] = float("nan")
        bad.view(-1)[37] = True
    else:
        p.s1[0].view(-1, 2)[0, 1] = float("nan")
        bad.view(-1)[:min(256, cols or 256)] = True
    p.step()
    _, v = p.moments(0)
    assert torch.equal(v.isnan().view(-1), bad.view(-1))
    assert torch.equal(p.held(0).isnan(), bad) and torch.equal(p.params[0].isnan(), bad)


@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, False), (BF16, True)])
def test_a_square_that_overflows(dtype, master):
    """A finite gradient whose square is infinite: v of its block is NaN from then on, m keeps its values, the weights follow in
    the next step."""
    p = Problem([(4, 1000)], dtype, 8, master=master, fresh=True)
    p.grads[0].view(-1)[777] = 1e20
    assert torch.isfinite(flex.grad_norm(p.grads))
    p.step()
    block = torch.zeros(4000, dtype=torch.bool, device=DEV)
    block[768:1024] = True
    for again in range(2):
        m, v = (x[0].view(-1) for x in flex.adamw8_moments(p.s0, p.s1))
        assert torch.equal(v.isnan(), block)
        assert torch.isfinite(m).all()
        assert abs(float(m[777]) / (1e19 * 0.9 ** again) - 1) < 2.0 ** -7  # (1e20 rounded to the type)
        assert torch.equal(p.held(0).view(-1).isnan(), block if again else torch.zeros_like(block))
        p.grads[0].view(-1)[777] = 0.0
        p.step()


@pytest.mark.parametrize("dtype,master,cols", [f[1:] for f in FORMS if f[0] == 8])
def test_m_keeps_its_values_beside_a_v_that_is_nan(dtype, master, cols):
    p = Problem([(3, cols)] if cols else [(4, 1000)], dtype, 8, unit=cols > 0, master=master)
    m, v = p.moments(0)
    m = 0.9 * m
    p.s1[0].view(-1, 2)[0, 1] = float("nan")
    p.grads[0].zero_()
    p.step()
    # equal decay leaves the codes where the largest has the highest one, and moves a code by half at most elsewhere: half a
    # code of c is 1 / 2c of the root, 1 / c and a bit of the value
    got, _ = p.moments(0)
    top = m.abs().amax()
    assert bool(((got - m).abs() <= (m.abs() * top).sqrt() / 127 + top / (4 * 127 ** 2) + 1e-6 * m.abs()).all())


def test_an_m_that_is_nan_does_not_need_a_v():
    for dtype in (F32, BF16):
        p = Problem([(4, 1000)], dtype, 8)
        p.s1[0].view(-1, 2)[1, 0] = float("nan")
        p.step()
        m, v = (x[0].view(-1) for x in flex.adamw8_moments(p.s0, p.s1))
        assert m.isnan().nonzero().flatten().tolist() == list(range(256, 512)) and torch.isfinite(v).all()


WIDTHS = [(F32, False, 0), (BF16, False, 0), (BF16, True, 0), (F32, False, 300), (BF16, False, 300), (BF16, False, 20001)]


def _state_with(dtype, master, cols, top, seed):
    """A state of 8 bits whose maxima of v are `top` times one to two."""
    p = Problem([(3, cols)] if cols else [(2, 700)], dtype, 8, unit=cols > 0, master=master, seed=seed)
    a = p.s1[0]
    a[..., 1] = (torch.rand(a.shape[:-1], generator=torch.Generator(DEV).manual_seed(seed), device=DEV) + 1.0) * top
    p.grads[0].zero_()
    return p


@pytest.mark.parametrize("dtype,master,cols", WIDTHS)
def test_codes_below_a_very_large_maximum(dtype, master, cols):
    """Above 2^126 the inverse of the maximum is no normal number."""
    for top in (2.0 ** 125, 2.0 ** 126, 1.6e38):
        p = _state_with(dtype, master, cols, top, 3)
        p.s0[0][..., 1].view(-1)[::5] = 255
        p.checked_step()
        assert int(p.s0[0][..., 1].max()) >= 254


@pytest.mark.parametrize("dtype,master,cols", WIDTHS)
def test_codes_of_values_below_the_normal_numbers(dtype, master, cols):
    """... beside a maximum that is a normal number: the nearest code, and at least one."""
    for top in (3e-38, 1e-37, 1e-34, 2.0 ** -98, 2.0 ** -97, 2.0 ** -96, 2.0 ** -95, 1e-27):
        p = _state_with(dtype, master, cols, top, 4)
        codes = p.s0[0][..., 1]
        # (from where 32 bits hold a value at all: (c / 255)^4 top is at least 2^-146)
        codes.clamp_(max(1, int(255 * (2.0 ** -146 / top) ** 0.25) + 1))
        codes.view(-1)[::3] = 1 if top > 1e-34 else codes.min()
        p.checked_step()
        assert bool((p.s0[0][..., 1] >= 1).all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,cols", [(F32, 300), (BF16, 40), (F32, 20001)])
def test_rows_of_very_small_and_very_large_lengths(bits, dtype, cols):
    p = Problem([(4, cols)], dtype, bits, unit=True, seed=5)
    w = p.params[0]
    w[1] = (w[1].float() * 1e-16).to(dtype)
    w[2] = (w[2].float() * 1e18).to(dtype)
    p.checked_step(wd=0.0)
    # (rounding a row of length one to 16 bits moves its length by less than the rounding of a number)
    assert float((p.params[0].double().norm(dim=1) - 1).abs().max()) < (1e-5 if dtype == F32 else 2.0 ** -8)
