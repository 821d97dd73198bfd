"""Layer norm, lookup and distillation from their formulas in 64 bits, with bounds on what 32-bit arithmetic and one rounding of
each result may differ by.

Bounds: U = 2^-24 is the rounding of one fp32 operation, half(t) that of a result (half a step), and a sum of n terms of magnitudes
a_i in which no term goes through more than d additions is off by at most d U sum(a_i).  The kernels add at most 32 terms in a lane
one after another (more only where a row is longer than 16384 columns or many rows meet, which `depth` counts), then 6 levels of
lanes and up to 16 wavefronts."""
import torch

U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def least(t):
    """Half a step below the normal numbers."""
    f = torch.finfo(t)
    return f.smallest_normal * f.eps / 2


def rounded(ref, t, arithmetic):
    """Bound on a result of type t that is off by `arithmetic` before it is rounded."""
    return half(t) * ref.abs() + (1 + half(t)) * arithmetic + least(t)


def within(got, ref, bound, what=""):
    got, ref = got.detach().cpu().double(), ref.cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(got.isnan(), ref.isnan()), what
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), what
    ok = ref.isfinite()
    off = (got - ref).abs()[ok]
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand(ref.shape)[ok]
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def layer_norm(x, w, b, eps, dy=None):
    """-> dict of results and of their bounds' arithmetic parts; x of shape [N, D]; w, b may be None."""
    f = torch.float64
    x = x.detach().cpu().to(f)
    N, D = x.shape
    one = torch.ones(D, dtype=f)
    w_, b_ = one if w is None else w.detach().cpu().to(f), 0 * one if b is None else b.detach().cpu().to(f)
    m = x.mean(1, keepdim=True)
    var = (x - m).square().mean(1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    u = (x - m) * r
    c = 80 + D / 1024 * 2  # additions and the few operations around them
    shift = c * U * x.abs().mean(1, keepdim=True) * r  # of u, by the mean
    du_ = shift + 3 * U * u.abs() + c * U * u.abs()    # ... and by its own operations and rstd (whose square's sum is off by c U)
    out = {"y": u * w_ + b_, "mean": m[:, 0], "rstd": r[:, 0]}
    tol = {"y": du_ * w_.abs() + 2 * U * ((u * w_).abs() + b_.abs()), "mean": shift[:, 0] / r[:, 0] + U * m[:, 0].abs(),
           "rstd": c * U * r[:, 0]}
    if dy is not None:
        dy = dy.detach().cpu().to(f)
        g = dy * w_
        c1, c2 = g.mean(1, keepdim=True), (g * u).mean(1, keepdim=True)
        out["dx"] = r * (g - c1 - u * c2)
        c1_off = c * U * g.abs().mean(1, keepdim=True)
        c2_off = c * U * (g * u).abs().mean(1, keepdim=True) + (g.abs() * du_).mean(1, keepdim=True)
        inner = 2 * U * g.abs() + c1_off + du_ * c2.abs() + u.abs() * c2_off + 4 * U * (g.abs() + c1.abs() + (u * c2).abs())
        tol["dx"] = r * inner + c * U * out["dx"].abs()
        deep = 80 + N / 16  # rows of a block, blocks of a wavefront
        out["dw"], out["db"] = (dy * u).sum(0), dy.sum(0)
        tol["dw"] = deep * U * (dy * u).abs().sum(0) + (dy.abs() * du_).sum(0)
        tol["db"] = deep * U * dy.abs().sum(0)
    return out, tol


def lookup(tokens, w, scale, factor, dout=None):
    """tokens [N]; scale [N] or None."""
    f = torch.float64
    tokens, w = tokens.cpu().long(), w.detach().cpu().to(f)
    there = (tokens >= 0) & (tokens < w.shape[0])
    at = torch.where(there, tokens, 0)
    s = torch.full((len(tokens),), factor, dtype=f) if scale is None else scale.detach().cpu().to(f) * factor
    s = torch.where(there, s, 0.0)
    rows = w[at] * there[:, None]
    out = {"out": rows * s[:, None]}
    tol = {"out": 2 * U * out["out"].abs()}
    if dout is not None:
        dout = torch.where(there[:, None], dout.detach().cpu().to(f), 0.0)
        sd = dout * s[:, None]
        out["dw"] = torch.zeros_like(w).index_add_(0, at, sd)
        size = torch.zeros_like(w).index_add_(0, at, sd.abs())
        most = int(torch.bincount(at[there], minlength=1).max()) if there.any() else 0
        tol["dw"] = (min(most, 64) + most / 64 + 4) * U * size
        out["ds"] = factor * (dout * rows).sum(1)
        tol["ds"] = (40 + w.shape[1] / 256) * U * abs(factor) * (dout * rows).abs().sum(1)
    return out, tol


def distill(z, top, index, weights, T, by_row, grad=None):
    """z [N, V]; top, index [N, K]; weights [N] or None; grad: 0-dim or [N]."""
    f = torch.float64
    z, top, index = z.detach().cpu().to(f), top.detach().cpu().to(f), index.cpu().long()
    N, V = z.shape
    a = torch.ones(N, dtype=f) if weights is None else weights.detach().cpu().to(f)
    there = (index >= 0) & (index < V)
    at = torch.where(there, index, 0)
    t = torch.where(there, top / T, -torch.inf)
    used = (t != -torch.inf).any(1) & (a != 0)
    z = torch.where(used[:, None], z, 0.0)
    t = torch.where(used[:, None], t, 0.0)
    total = a.sum()
    part = a if by_row else (a / total if total != 0 else a * 0)
    log_p, log_q = torch.log_softmax(t, 1), torch.log_softmax(z / T, 1)
    p, q = log_p.exp() * used[:, None], log_q.exp() * used[:, None]
    at_q = log_q.gather(1, at)
    terms = torch.where(p != 0, p * (log_p - at_q), 0.0)
    kl = torch.where(used, terms.sum(1), 0.0)
    # exponents are off by a few U of the distance from the maximum, sums of exponentials by their depth
    m = z.amax(1, keepdim=True)
    c = 96 + V / 256
    log_s = torch.log(((z - m) / T).exp().sum(1, keepdim=True))
    spread = torch.where(z.isfinite(), (z - m).abs() / T, 0.0)
    q_off = U * (c + 4 * spread + 4 * log_s.abs())
    t_max = t.amax(1, keepdim=True)
    t_spread = torch.where(t.isfinite(), (t - t_max).abs(), 0.0)
    p_off = U * (c + top.shape[1] + 4 * t_spread)
    near = torch.where(at_q.isfinite(), at_q.abs(), 0.0)
    kl_off = (p * (p_off * torch.where(p != 0, log_p - at_q, 0.0).abs().nan_to_num(posinf=0.0)
                   + U * (c + top.shape[1] + 8 * (t_spread + near + log_s.abs() + spread.gather(1, at))))).sum(1)
    rows, rows_off = T * T * a * kl, T * T * a.abs() * kl_off + 4 * U * (T * T * a * kl).abs()
    part_off = 8 * U
    if by_row:
        out, tol = {"loss": rows}, {"loss": rows_off + U * rows.abs()}
    else:
        out = {"loss": (T * T * part * kl).sum()}
        tol = {"loss": (T * T * part.abs() * kl_off).sum() + part_off * (T * T * part * kl).abs().sum()}
    if grad is not None:
        g = grad.detach().cpu().to(f)
        coef = T * part * g
        push = torch.zeros_like(z).scatter_add_(1, at, p * there)
        out["dz"] = torch.where(used[:, None], coef[:, None] * (q - push), 0.0)
        push_off = torch.zeros_like(z).scatter_add_(1, at, p * p_off * there)
        tol["dz"] = coef.abs()[:, None] * (q * q_off + push_off + (part_off + 2 * U) * (q + push) + 2.0 ** -126)
    return out, tol
