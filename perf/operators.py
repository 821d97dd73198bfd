"""What is measured of the optimiser's operators: the global norm of gradients, and AdamW steps over many tensors with states
in 32 bits and in 8, plain, clipped, under a loss scale, and on decoder rows that are held at length one.

A case is one call (with clipping, two) that a training loop makes after ``backward()``.  Fields:

    op      "norm" (the gradients' global norm), "adamw" (states in 32 bits) or "adamw8" (states in 8 bits; the moments come
            back as the values that they stand for, as of a loop that logs or checkpoints them)
    set     "sae": encoder weight [F, D], encoder bias [F], decoder weight [F, D], decoder bias [D]; "decoder": its weight alone
    L       so many of them at once (a sweep over dictionaries, trained side by side)
    F, D    latents of a dictionary, columns of a row
    dtype   of parameters and gradients; master: 16-bit parameters have 32-bit copies, which the step works on
    clip    the gradients' norm is taken first and held at most 1; scale: the loss scale that the gradients carry
    unit    rows of length one: the gradient's part along the row is left out, and the row is brought back to length one
"""
import itertools
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BLOCK = 256
_TINY = 2.0 ** -126
_LR, _B1, _B2, _EPS, _WD, _MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 0.01, 1.0


def _case(name, op, set_, F, D, dtype, L=1, master=False, clip=False, scale=1.0, unit=False):
    return {"name": name, "op": op, "set": set_, "L": L, "F": F, "D": D, "dtype": dtype, "master": master, "clip": clip,
            "scale": scale, "unit": unit}


def listed():
    return [
        # Gradients of a notebook-sized dictionary (the repository's smallest configuration): launches.
        _case("norm_small", "norm", "sae", 4096, 256, "fp32"),
        # A sweep of small dictionaries trained side by side: many tensors, odd sizes.
        _case("norm_sweep", "norm", "sae", 1021, 67, "bf16", L=48),
        # The widest trained dictionary: one read of 4.3 GB.
        _case("norm_large", "norm", "sae", 262144, 4096, "bf16"),
        # The smallest configuration's step.
        _case("adamw_small", "adamw", "sae", 4096, 256, "fp32"),
        # The sweep: 192 tensors in a step.
        _case("adamw_sweep", "adamw", "sae", 1021, 67, "fp32", L=48),
        # fp16 training: master weights, a loss scale, clipping; ragged sizes.
        _case("adamw_clip_fp16", "adamw", "sae", 24571, 1538, "fp16", master=True, clip=True, scale=65536.0),
        # The headline dictionary in mixed precision.
        _case("adamw_headline", "adamw", "sae", 65536, 2304, "bf16", master=True),
        # Its decoder, rows held at length one.
        _case("adamw_unit", "adamw", "decoder", 65536, 2304, "bf16", master=True, unit=True),
        # The same with states in 8 bits: the smallest, ...
        _case("adamw8_small", "adamw8", "sae", 4096, 256, "fp32"),
        # ... the headline dictionary with nothing but 16-bit weights, ...
        _case("adamw8_headline", "adamw8", "sae", 65536, 2304, "bf16"),
        # ... unit rows whose last block is a short one, clipped, ...
        _case("adamw8_unit_ragged", "adamw8", "decoder", 24571, 1538, "fp32", clip=True, unit=True),
        # ... and the largest: two thousand million parameters, where 32-bit states would take 17 GB.
        _case("adamw8_large", "adamw8", "sae", 262144, 4096, "bf16"),
    ]


def _shapes(case):
    F, D = case["F"], case["D"]
    return ([(F, D), (F,), (F, D), (D,)] if case["set"] == "sae" else [(F, D)]) * case["L"]


def work(case):
    n = sum(math.prod(s) for s in _shapes(case))
    P = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        return {"bytes": n * P + 4, "flops": 2 * n}
    params = 2 * P + (8 + P if case["master"] else P)  # gradient, weight written, weight (or master, which is written too) read
    if case["master"]:
        params -= P  # (a weight with a master is not read)
    states = 16.0 if case["op"] == "adamw" else 4.0 + 16.0 / _BLOCK + 4.0  # read, written; 8 bits: also as values, in bf16
    flops = 16 + (2 if case["clip"] else 0) + (9 if case["unit"] else 0) + (16 if case["op"] == "adamw8" else 0)
    return {"bytes": n * (params + states), "flops": n * flops}


def draw(rng):
    """Every axis over the whole range of the listed cases, sizes over their logarithm, about half of them off round numbers."""
    def size(lo, hi):
        x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return min(hi, max(lo, 1 << round(math.log2(x)) if rng.random() < 0.4 else int(x)))

    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["norm", "adamw", "adamw", "adamw8", "adamw8"])
        dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
        unit = op != "norm" and rng.random() < 0.4
        many = rng.random() < 0.25
        c = {"op": op, "set": "decoder" if unit or rng.random() < 0.2 else "sae", "L": size(2, 64) if many else 1,
             "F": size(256, 4096) if many else size(1024, 262144), "D": size(48, 512) if many else size(64, 8192),
             "dtype": dtype, "master": op != "norm" and dtype != "fp32" and (dtype == "fp16" or rng.random() < 0.5),
             "clip": op != "norm" and rng.random() < 0.4, "scale": 65536.0 if dtype == "fp16" else 1.0, "unit": unit}
        n = sum(math.prod(s) for s in _shapes(c))
        if 100_000 <= n <= 2_200_000_000 and work(c)["bytes"] <= most:
            return c


def _layout(shape, unit):
    """(rows, columns) that blocks of states follow: those of the matrix where rows are held at length one, else one long row."""
    n = math.prod(shape)
    return (n // shape[-1], shape[-1]) if unit else (1, n)


def _blocks(x):
    """[R, C, ...] as [R, blocks, 256, ...], zeros after the end of a row."""
    R, C, rest = x.shape[0], x.shape[1], x.shape[2:]
    short = -C % _BLOCK
    if short:
        x = torch.cat([x, x.new_zeros((R, short, *rest))], 1)
    return x.view(R, -1, _BLOCK, *rest)


def _arena(sizes, dtype):
    """One buffer, and views of it for tensors of these numbers of elements, each starting at a multiple of 64."""
    starts = list(itertools.accumulate((-(-n // 64) * 64 for n in sizes), initial=0))
    buffer = torch.zeros(starts[-1], dtype=dtype, device="cuda")
    return buffer, [buffer[a:a + n] for a, n in zip(starts, sizes)]


def prepare(case, seed):
    dt, dev = _DTYPES[case["dtype"]], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    views = len(shapes) > 4  # many tensors come back as the buffers that they are views of

    def make(dtype):
        if views:
            return _arena(sizes, dtype)
        flat = [torch.zeros(n, dtype=dtype, device=dev) for n in sizes]
        return flat, flat

    s = {"case": dict(case), "shapes": shapes}
    all_params, params = make(dt) if case["op"] != "norm" else (None, [])
    _, grads = make(dt)
    s["grads"] = [x.view(shape) for x, shape in zip(grads, shapes)]
    s["params"] = [x.view(shape) for x, shape in zip(params, shapes)]
    s["out"] = {"params": all_params}
    masters = ms = vs = None
    if case["op"] != "norm":
        if case["master"]:
            s["out"]["masters"], masters = make(torch.float32)
            s["masters"] = [x.view(shape) for x, shape in zip(masters, shapes)]
        if case["op"] == "adamw":
            s["out"]["exp_avgs"], ms = make(torch.float32)
            s["out"]["exp_avg_sqs"], vs = make(torch.float32)
            s["exp_avgs"] = [x.view(shape) for x, shape in zip(ms, shapes)]
            s["exp_avg_sqs"] = [x.view(shape) for x, shape in zip(vs, shapes)]
        else:
            s["codes"], s["absmax"] = [], []
        # steps taken so far, and a word that the step works with
        s["counter"] = torch.tensor([100, 0], dtype=torch.int64, device=dev)
    grad_std = 1e-4 if case["clip"] else 1e-5
    for i, shape in enumerate(shapes):
        # Latents differ in how often they fire: rows of gradients by a factor of some ten, a fifth of them (of a matrix) zero.
        n, cols = sizes[i], shape[-1] if len(shape) == 2 else 1
        rows = n // cols
        row_std = torch.empty(rows, 1, device=dev).normal_(generator=g).exp_().mul_(grad_std)
        if len(shape) == 2:
            row_std *= torch.rand(rows, 1, generator=g, device=dev) >= 0.2
        part = max(1, (1 << 28) // cols)
        for r in range(0, rows, part):
            at = slice(r * cols, min(rows, r + part) * cols)
            std = row_std[r:r + part]
            x = torch.randn(len(std), cols, generator=g, device=dev)
            grads[i][at] = (x * (std * case["scale"])).clamp_(-6e4, 6e4).view(-1)
            if case["op"] == "norm":
                continue
            x.normal_(generator=g).mul_(0.02)
            if case["unit"]:
                x /= x.norm(dim=1, keepdim=True).clamp_min(1e-20)
            params[i][at] = x.view(-1)
            if case["master"]:
                masters[i][at] = x.view(-1)
            if case["op"] == "adamw":
                ms[i][at] = (x.normal_(generator=g).mul_(0.3) * std).view(-1)
                vs[i][at] = (x.uniform_(0.2, 1.5, generator=g).mul_(std)).square_().view(-1)
        if case["op"] == "adamw8":
            R, C = _layout(shape, case["unit"])
            blocks = -(-C // _BLOCK)
            codes = torch.empty(R, C, 2, dtype=torch.uint8, device=dev)
            # codes as steps leave them: the first moment's about its middle, the second's in the upper part
            codes[..., 0].random_(8, 249, generator=g)
            codes[..., 1].random_(96, 256, generator=g)
            absmax = torch.rand(R, blocks, 2, generator=g, device=dev).add_(0.5)
            absmax[..., 0] *= grad_std
            absmax[..., 1] = (absmax[..., 1] * (1.5 * grad_std)).square_()
            s["codes"].append(codes.view(*shape, 2))
            s["absmax"].append(absmax)
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the framework's operators -------------------------------------------------------------


def _run_own(s):
    import flexsae_amd as flex

    c = s["case"]
    if c["op"] == "norm":
        return {"norm": flex.grad_norm(s["grads"])}
    how = {"lr": _LR, "beta1": _B1, "beta2": _B2, "eps": _EPS, "weight_decay": _WD, "grad_scale": c["scale"],
           "unit_rows": c["unit"], "masters": s.get("masters")}
    out = dict(s["out"], steps=s["counter"][:1])
    if c["clip"]:
        out["norm"] = how["grad_norm"] = flex.grad_norm(s["grads"])
        how["max_norm"] = _MAX_NORM
    if c["op"] == "adamw":
        flex.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["counter"], **how)
        return out
    flex.adamw8_step(s["params"], s["grads"], s["codes"], s["absmax"], s["counter"], **how)
    ms, vs = flex.adamw8_moments(s["codes"], s["absmax"], torch.bfloat16)
    return dict(out, exp_avgs=_joined(ms), exp_avg_sqs=_joined(vs))


def _joined(tensors):
    return tensors if len(tensors) <= 4 else torch.cat([t.reshape(-1) for t in tensors])


# ---- the plain form ------------------------------------------------------------------------


def _plain_norm(grads):
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _plain_decode(codes, absmax, R, C):
    c = _blocks(codes.view(R, C, 2)).float()
    m, v = c[..., 0] - 128.0, c[..., 1]
    m = m * m.abs() * (1.0 / 127.0 ** 2) * absmax[..., :1]
    v = (v * v * (1.0 / 255.0 ** 2)).square() * absmax[..., 1:]
    return (x.reshape(R, -1)[:, :C] for x in (m, v))


def _plain_encode(m, v, codes, absmax, R, C):
    m, v = _blocks(m), _blocks(v)
    a = torch.stack([m.abs().amax(-1), v.amax(-1)], -1)
    a = torch.where(a < _TINY, 0.0, torch.where(a.isfinite(), a, math.nan))
    per = torch.where(a > 0, 1.0 / a, 0.0)
    cm = (m.abs() * per[..., :1]).sqrt().mul(127.0).round() * m.sign() + 128.0
    cv = (v * per[..., 1:]).sqrt().sqrt().mul(255.0).round().maximum(((v > 0) & (a[..., 1:] > 0)).float())
    both = torch.stack([cm, cv], -1).nan_to_num(0.0).to(torch.uint8)
    codes.view(R, C, 2).copy_(both.view(R, -1, 2)[:, :C])
    absmax.copy_(a)


def _plain_step(s, i, coef, go, bc1, bc2):
    c = s["case"]
    R, C = _layout(s["shapes"][i], c["unit"])
    held = s["masters"][i] if c["master"] else s["params"][i]
    w = held.view(R, C).float()
    g = s["grads"][i].view(R, C).float() * coef
    if c["op"] == "adamw":
        m, v = s["exp_avgs"][i].view(R, C), s["exp_avg_sqs"][i].view(R, C)
    else:
        m, v = _plain_decode(s["codes"][i], s["absmax"][i], R, C)
    if c["unit"]:
        ww = (w * w).sum(1, keepdim=True)
        g = g - torch.where(ww > 0, (g * w).sum(1, keepdim=True) / ww, 0.0) * w
    m2 = m * _B1 + g * (1.0 - _B1)
    v2 = v * _B2 + g * g * (1.0 - _B2)
    w2 = w * (1.0 - _LR * _WD) - m2 / ((v2 / bc2).sqrt() + _EPS) * (_LR / bc1)
    if c["unit"]:
        length = (w2 * w2).sum(1, keepdim=True).sqrt()
        w2 = w2 / torch.where(length > 0, length, 1.0)
    w2 = torch.where(go, w2, w)
    s["params"][i].view(R, C).copy_(w2)
    if c["master"]:
        held.view(R, C).copy_(w2)
    if c["op"] == "adamw":
        m.copy_(torch.where(go, m2, m))
        v.copy_(torch.where(go, v2, v))
        return m, v
    _plain_encode(torch.where(go, m2, m), torch.where(go, v2, v), s["codes"][i], s["absmax"][i], R, C)
    return [x.to(torch.bfloat16).view(s["shapes"][i]) for x in _plain_decode(s["codes"][i], s["absmax"][i], R, C)]


def _run_plain(s):
    c = s["case"]
    if c["op"] == "norm":
        return {"norm": _plain_norm(s["grads"])}
    out = dict(s["out"], steps=s["counter"][:1])
    coef, go = 1.0 / c["scale"], torch.ones((), dtype=torch.bool, device="cuda")
    if c["clip"]:
        out["norm"] = norm = _plain_norm(s["grads"])
        coef, go = (_MAX_NORM / (norm * coef + 1e-6)).clamp_max(1.0) * coef, norm.isfinite()
    t = (s["counter"][0] + 1).float()
    bc1, bc2 = -torch.expm1(t * math.log(_B1)), -torch.expm1(t * math.log(_B2))
    moments = [_plain_step(s, i, coef, go, bc1, bc2) for i in range(len(s["shapes"]))]
    s["counter"][0] += go
    if c["op"] == "adamw8":
        out["exp_avgs"], out["exp_avg_sqs"] = (_joined(list(x)) for x in zip(*moments))
    return out


# ---- the definition, in 64 bits ------------------------------------------------------------


def exact(case, seed):
    """Rows (of unit length) or stretches of whole blocks at a time, in float64, from the formulas:

        g <- c g, c = min(1, max_norm / (|g| / scale + 1e-6)) / scale;   unit rows: g <- g - (<g, w> / <w, w>) w
        m <- b1 m + (1 - b1) g;   v <- b2 v + (1 - b2) g^2
        w <- (1 - lr wd) w - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps);   unit rows: w <- w / |w|

    8-bit states: the code c of m (-127 ... 127) stands for sign(c) (c / 127)^2 a, that of v (0 ... 255) for (c / 255)^4 a, a the
    block's largest; a new code is the nearest on the root's scale, and at least one for a v above zero."""
    f64 = torch.float64
    s = prepare(case, seed)
    part = 1 << 25
    squares = torch.zeros((), dtype=f64, device="cuda")
    for g in s["grads"]:
        for piece in g.reshape(-1).split(part):
            squares += piece.to(f64).square().sum()
    norm = squares.sqrt()
    if case["op"] == "norm":
        return {"norm": norm}
    c = 1.0 / case["scale"]
    if case["clip"]:
        c = c * min(1.0, _MAX_NORM / (float(norm) * c + 1e-6))
    t = 101
    sizes = [math.prod(shape) for shape in s["shapes"]]

    def room():
        if isinstance(s["out"]["params"], list):
            flat = [torch.zeros(n, dtype=f64, device="cuda") for n in sizes]
            return flat, flat
        return _arena(sizes, f64)

    out, places = {}, {}
    for key in ["params", "exp_avgs", "exp_avg_sqs"] + (["masters"] if case["master"] else []):
        if key in ("exp_avgs", "exp_avg_sqs") and case["op"] == "adamw8":
            places[key] = [torch.zeros(n, dtype=f64, device="cuda") for n in sizes]
            out[key] = [x.view(shape) for x, shape in zip(places[key], s["shapes"])]
        else:
            out[key], places[key] = room()
    for i, shape in enumerate(s["shapes"]):
        cols = shape[-1] if case["unit"] else _BLOCK
        step = max(1, part // cols) * cols
        for a in range(0, sizes[i], step):
            at = slice(a, min(sizes[i], a + step))
            w = (s["masters"] if case["master"] else s["params"])[i].reshape(-1)[at].to(f64)
            g = s["grads"][i].reshape(-1)[at].to(f64) * c
            if case["unit"]:
                w, g = w.view(-1, cols), g.view(-1, cols)
                g = g - (g * w).sum(1, keepdim=True) / w.square().sum(1, keepdim=True) * w
                w, g = w.view(-1), g.view(-1)
            if case["op"] == "adamw":
                m, v = (s[k][i].reshape(-1)[at].to(f64) for k in ("exp_avgs", "exp_avg_sqs"))
            else:
                code = s["codes"][i].reshape(-1, 2)[at].to(f64)
                n, per = at.stop - a, -(-cols // _BLOCK)
                e = torch.arange(n, device="cuda")
                block = e // cols * per + e % cols // _BLOCK  # of this stretch
                count = int(block[-1]) + 1
                top = s["absmax"][i].reshape(-1, 2)[a // cols * per:][:count].to(f64)[block]
                m = torch.sign(code[:, 0] - 128) * ((code[:, 0] - 128) / 127) ** 2 * top[:, 0]
                v = (code[:, 1] / 255) ** 4 * top[:, 1]
            m = _B1 * m + (1 - _B1) * g
            v = _B2 * v + (1 - _B2) * g ** 2
            w = (1 - _LR * _WD) * w - _LR * (m / (1 - _B1 ** t)) / ((v / (1 - _B2 ** t)).sqrt() + _EPS)
            if case["unit"]:
                w = (w.view(-1, cols) / w.view(-1, cols).norm(dim=1, keepdim=True)).view(-1)
            if case["op"] == "adamw8":
                tops = torch.zeros(count, 2, dtype=f64, device="cuda")
                tops.scatter_reduce_(0, block[:, None].expand(-1, 2), torch.stack([m.abs(), v], 1), "amax")
                tops = tops[block]
                cm = torch.round(127 * (m.abs() / tops[:, 0]).sqrt())
                cv = torch.maximum(torch.round(255 * (v / tops[:, 1]) ** 0.25), (v > 0).to(f64))
                m = (torch.sign(m) * (cm / 127) ** 2 * tops[:, 0]).nan_to_num(0.0)  # (a block of zeros)
                v = ((cv / 255) ** 4 * tops[:, 1]).nan_to_num(0.0)
            for key, x in (("params", w), ("masters", w), ("exp_avgs", m), ("exp_avg_sqs", v)):
                if key in places:
                    places[key][i][at] = x
    if case["op"] == "adamw8":
        out["exp_avgs"], out["exp_avg_sqs"] = _joined(out["exp_avgs"]), _joined(out["exp_avg_sqs"])
    out["steps"] = torch.tensor([t], dtype=torch.int64, device="cuda")
    if case["clip"]:
        out["norm"] = norm
    return out
