"""The optimiser's formulas in 64 bits, on the CPU or where the tensors are, and what fp32 arithmetic may differ from them by.

A step is checked from the state that the kernels were given, so that errors do not add up over steps.  With u = 2^-24 (half a
unit in the last place of fp32, relative):

* m = b1 m + (1-b1) g: the constants, the two products and the sum, each within u of the sum of the terms' magnitudes: 4 u of
  |b1 m| + |(1-b1) c g|; the clipping factor c (a quotient of a norm rounded to fp32) adds 4 u of the second.
* v = b2 v + (1-b2) g^2: all terms positive: 12 u of v (c enters squared).
* the update lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps): m's error, and a chain of ten roundings, the exponentials of the two
  bias corrections (2 u each) and the hardware's functions: 32 u of the update that |b1 m| + |(1-b1) c g| in m's place gives.
* the weight: 4 u of |w| beside that, and half a unit of its own type where it is kept in 16 bits.
"""
import torch

U = 2.0 ** -24
HALF = {torch.float32: (U, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25)}
BLOCK = 256
TINY = 2.0 ** -126


def layout(shape, unit):
    n = 1
    for s in shape:
        n *= s
    return (n // shape[-1], shape[-1]) if unit else (1, n)


def per_element(a, R, C):
    """[R, blocks] -> [R, C]"""
    return a.repeat_interleave(BLOCK, 1)[:, :C]


def decode(codes, absmax, unit):
    """-> m, v as [R, C] float64"""
    R, C = layout(codes.shape[:-1], unit)
    c = codes.reshape(R, C, 2).double()
    a = absmax.double()
    q = (c[..., 0] - 128) / 127
    return q * q.abs() * per_element(a[..., 0], R, C), (c[..., 1] / 255) ** 4 * per_element(a[..., 1], R, C)


def factor(norm, scale, max_norm):
    c = 1.0 / scale
    return c * min(1.0, max_norm / (norm * c + 1e-6)) if max_norm else c


def step(w, g, m, v, t, lr, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.0, c=1.0, unit=False):
    """[R, C] tensors in; w, m, v after step t and the bounds of their fp32 errors (before the weight is rounded to 16 bits)."""
    w, g, m, v = (x.double() for x in (w, g, m, v))
    g = c * g
    dg = 4 * U * g.abs()
    if unit:
        ww = w.square().sum(1, keepdim=True)
        along = torch.where(ww > 0, (g * w).sum(1, keepdim=True) / ww, 0.0)
        # sums of n terms: a lane adds at most 8 terms a stretch, the rest is a tree: n / 64 + 20 roundings at most
        k = (w.shape[1] / 64 + 20) * U
        dalong = torch.where(ww > 0, k * (g * w).abs().sum(1, keepdim=True) / ww, 0.0) + (k + 4 * U) * along.abs()
        g = g - along * w
        dg = dg + dalong * w.abs() + 4 * U * ((along * w).abs() + g.abs())
    parts = (beta1 * m).abs() + ((1 - beta1) * g).abs()
    m2 = beta1 * m + (1 - beta1) * g
    v2 = beta2 * v + (1 - beta2) * g * g
    dm = 4 * U * parts + (1 - beta1) * dg + 2.0 ** -148
    dv = 12 * U * v2 + 2 * (1 - beta2) * g.abs() * dg + (1 - beta2) * dg * dg + 2.0 ** -146
    bc1, bc2 = 1 - beta1 ** t, 1 - beta2 ** t
    denom = (v2 / bc2).sqrt() + eps
    # sqrt(v): relative error dv / 2v, and never more than sqrt(dv)
    ddenom = torch.minimum(dv / (2 * v2.clamp_min(1e-300)).sqrt() / v2.clamp_min(1e-300).sqrt() / 1.41, (dv / v2.clamp_min(1e-300)) / 2 + 0 * v2)
    ddenom = torch.minimum(ddenom, dv.sqrt() / v2.sqrt().clamp_min(1e-150)).nan_to_num(0.0, posinf=0.0)
    update = lr / bc1 * m2 / denom
    dupdate = lr / bc1 * (dm + 32 * U * parts) / denom + update.abs() * ddenom
    w2 = (1 - lr * wd) * w - update
    dw = 4 * U * (w.abs() + w2.abs()) + dupdate + lr * wd * 4 * U * w.abs()
    if unit:
        length = w2.square().sum(1, keepdim=True).sqrt()
        dlength = dw.square().sum(1, keepdim=True).sqrt() + k * length
        w3 = torch.where(length > 0, w2 / length.clamp_min(1e-300), w2)
        dw = torch.where(length > 0, (dw + w3.abs() * dlength) / length.clamp_min(1e-300), dw) + 6 * U * w3.abs()
        w2 = w3
    return w2, m2, v2, dw, dm, dv


def within(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() / bound.clamp_min(1e-300)).max()))


def rounded(want, bound, dtype):
    rel, tiny = HALF[dtype]
    return bound + rel * (want.abs() + bound) * (1.001 if dtype != torch.float32 else 0) + (tiny if dtype != torch.float32 else 0)


def check_codes(codes, absmax, m, v, dm, dv, unit):
    """Codes and maxima against m, v in 64 bits: the maxima within their elements' errors, and every code within half a code, and
    what an error of the value moves it by, of its place on the root's scale."""
    R, C = layout(codes.shape[:-1], unit)
    nb = -(-C // BLOCK)
    c = codes.reshape(R, C, 2).double()

    def blocks(x):
        pad = nb * BLOCK - C
        return torch.cat([x, x.new_zeros(R, pad)], 1).view(R, nb, BLOCK) if pad else x.view(R, nb, BLOCK)

    for j, (x, dx, n, root) in enumerate(((m, dm, 127, 2), (v, dv, 255, 4))):
        a, da = blocks(x.abs()).amax(-1), blocks(dx).amax(-1)
        got = absmax[..., j].double()
        live = a > 2 * TINY  # (a maximum about the smallest normal number may be kept or not)
        within(torch.where(live, got, 0.0), torch.where(live, a, 0.0), 2 * U * a + da, f"absmax {j}")
        assert bool((got[a < TINY / 2] == 0).all())
        a_el, live_el = per_element(a, R, C), per_element(live, R, C)
        q = (x.abs() / a_el.clamp_min(1e-300)).clamp_max(1.0)
        dq = dx / a_el.clamp_min(1e-300) + q * per_element(da / a.clamp_min(1e-300), R, C) + 8 * U * q
        at = q ** (1 / root)
        move = n * torch.maximum((q + dq) ** (1 / root) - at, at - (q - dq).clamp_min(0) ** (1 / root)) + n * 8 * U
        place = n * at * (torch.sign(x) if j == 0 else 1.0)
        mine = c[..., j] - (128 if j == 0 else 0)
        near = (mine - place).abs() <= 0.5 + move + 1e-6
        if j == 1:
            near |= (mine == 1) & (place <= 1) & (x > 0)
            assert bool((mine[live_el & (x > 0)] >= 1).all()), "a v above zero became zero"
        assert bool(near[live_el].all()), (j, int((~near & live_el).sum()))
        dead = per_element(got == 0, R, C)
        assert bool((c[..., j][dead] == (128 if j == 0 else 0)).all())
