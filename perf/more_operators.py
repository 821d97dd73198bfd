"""What is measured of the operators around a dictionary that is trained inside a language model: the layer norm of activations,
the lookup of a per-token table whose rows are added to a reconstruction, and the distillation loss that compares the logits of
the model with the dictionary in it to the top logits of the model without.

A case is one pass: the call, and, where it trains, its backward pass for a given gradient.  Fields:

    op      "norm", "lookup" or "distill"
    train   with gradients
    dtype   of activations, tables and logits, and of their gradients
    N, D    rows (tokens) and columns; norm: affine: with weight and bias; stats: mean and 1 / deviation of the rows come back
            too, as for a reconstruction that is scaled back
    V       rows of the table, or logits of a row; lookup: scale: "none", "all" (one number) or "each" (one of every token),
            pad: share of places without a token, which hold -1
    K       top logits of a row; T: temperature; weights: of rows, some of them zero; rows: the loss of every row
            comes back, not their mean; ragged: rows with fewer than K of them,
            the missing places holding -1, some rows with none; scale: the loss scale (the upstream gradient)
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5


def _norm(name, N, D, dtype, train=True, affine=True, stats=False):
    return {"name": name, "op": "norm", "N": N, "D": D, "dtype": dtype, "train": train, "affine": affine, "stats": stats}


def _lookup(name, N, V, D, dtype, train=True, scale="none", pad=0.0):
    return {"name": name, "op": "lookup", "N": N, "V": V, "D": D, "dtype": dtype, "train": train, "scale": scale, "pad": pad}


def _distill(name, N, V, K, dtype, train=True, T=1.0, weights=False, rows=False, ragged=False, scale=1.0):
    return {"name": name, "op": "distill", "N": N, "V": V, "K": K, "dtype": dtype, "train": train, "T": T, "weights": weights,
            "rows": rows, "ragged": ragged, "scale": scale}


def listed():
    return [
        # A training step's norm at the repository's smallest configuration: launches.
        _norm("norm_small", 64, 256, "fp32"),
        # Activations normalised on their way into the widest dictionary, with what scales its reconstruction back.
        _norm("norm_inputs", 16384, 8192, "bf16", train=False, affine=False, stats=True),
        # fp16 training on a short last batch: ragged sizes.
        _norm("norm_ragged", 2999, 1538, "fp16"),
        # The model's last norm, between the reconstruction and the logits: a large batch of the headline width.
        _norm("norm_large", 65536, 2304, "bf16"),
        # Rows for a handful of tokens.
        _lookup("lookup_small", 64, 4096, 256, "fp32", train=False, scale="all"),
        # Padded sequences, one gate a token, odd sizes.
        _lookup("lookup_ragged", 8191, 24571, 1537, "fp16", scale="each", pad=0.2),
        # A batch of the headline width.
        _lookup("lookup_headline", 32768, 65536, 2304, "bf16", scale="each"),
        # A large vocabulary: most of the time goes into a gradient of 2.1 GB.
        _lookup("lookup_large", 131072, 262144, 4096, "bf16"),
        # A few rows: the vocabulary has to be shared out.
        _distill("distill_small", 16, 32000, 32, "fp32"),
        # fp16 with a loss scale, a temperature, padded rows and rows with fewer stored logits; odd sizes.
        _distill("distill_ragged", 1021, 50001, 50, "fp16", T=2.0, weights=True, ragged=True, scale=65536.0),
        # Evaluation: the loss of every token.
        _distill("distill_eval", 2048, 131071, 64, "bf16", train=False, rows=True),
        # A training batch with a large vocabulary: 2.1 GB of logits, and as much of gradients.
        _distill("distill_large", 8192, 131072, 128, "bf16"),
    ]


def _distinct(N, V):
    """Expected number of different ranks among N that are spread evenly over their logarithm in 1 ... V."""
    often = N / math.log(V + 1.0)  # ranks up to about here are all there
    return V if often >= V else max(1.0, min(N, V, often * (1.0 + math.log(V / often)) if often > 1.0 else N))


def work(case):
    P = 4 if case["dtype"] == "fp32" else 2
    N, train = case["N"], case["train"]
    if case["op"] == "norm":
        D = case["D"]
        small = (2 if case["affine"] else 0) * D * P * (2 if train else 1) + (8 * N if case["stats"] else 0)
        return {"bytes": N * D * P * (4 if train else 2) + small, "flops": N * D * (20 if train else 8)}
    if case["op"] == "lookup":
        V, D = case["V"], case["D"]
        there = N * (1.0 - case["pad"])
        each = N * P * (2 if train else 1) if case["scale"] == "each" else 0
        rows = _distinct(there, V) * D + N * D  # read of the table, written
        if train:
            rows += there * D + V * D  # gradients read, the table's gradient written
        return {"bytes": rows * P + 8 * N + each, "flops": there * D * (5 if train else 1)}
    V, K = case["V"], case["K"]
    return {"bytes": N * V * P * (2 if train else 1) + N * K * (8 + P) + (4 * N if case["weights"] else 0) + 4 * (N if case["rows"] else 1),
            "flops": N * V * (7 if train else 4) + 10 * N * K}


def draw(rng):
    """Every axis over the whole range of the listed cases and somewhat beyond, sizes over their logarithm, about half of them off
    round numbers."""
    def size(lo, hi):
        x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return min(hi, max(lo, 1 << round(math.log2(x)) if rng.random() < 0.4 else int(x)))

    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["norm", "lookup", "distill"])
        dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
        train = rng.random() < 0.75
        if op == "norm":
            c = _norm("", size(1, 131072), size(48, 16384), dtype, train, rng.random() < 0.7, not train and rng.random() < 0.5)
        elif op == "lookup":
            c = _lookup("", size(1, 131072), size(1000, 262144), size(48, 8192), dtype, train,
                        rng.choice(["none", "all", "each", "each"]), rng.choice([0.0, 0.0, 0.1, 0.5]))
        else:
            c = _distill("", size(1, 8192), size(1000, 262144), size(1, 256), dtype, train, rng.choice([1.0, 1.0, 2.0, 0.7]),
                         rng.random() < 0.4, rng.random() < 0.2, rng.random() < 0.4, 65536.0 if dtype == "fp16" else rng.choice([1.0, 1.0, 128.0]))
        del c["name"]
        if work(c)["bytes"] <= most:
            return c


def prepare(case, seed):
    dt, dev = _DTYPES[case["dtype"]], "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        """In pieces: 32-bit numbers of a large 16-bit tensor are never there at once."""
        if dtype == torch.float32:
            return torch.randn(*shape, generator=g, device=dev)
        out = torch.empty(*shape, dtype=dtype, device=dev)
        for piece in out.view(-1).split(1 << 28):
            piece.copy_(torch.randn(piece.numel(), generator=g, device=dev))
        return out

    s = {"case": dict(case)}
    N = case["N"]
    if case["op"] == "norm":
        # activations: columns differ in their mean and spread, a few of them are far larger than the rest
        D = case["D"]
        spread = torch.randn(D, generator=g, device=dev).mul_(0.5).exp_()
        spread[torch.randint(0, D, (max(1, D // 512),), generator=g, device=dev)] *= 20.0
        s["x"] = normal(N, D, dtype=dt).mul_(spread.to(dt)).add_(normal(D).mul_(0.3).to(dt))
        if case["affine"]:
            s["weight"], s["bias"] = normal(D).mul_(0.1).add_(1.0).to(dt), normal(D).mul_(0.1).to(dt)
        if case["train"]:
            s["dy"] = normal(N, D, dtype=dt).mul_(0.01)
            for k in ("x", "weight", "bias"):
                if k in s:
                    s[k].requires_grad_()
    elif case["op"] == "lookup":
        # tokens: their frequencies fall as one over their rank, which has nothing to do with their number
        V, D = case["V"], case["D"]
        rank = torch.exp(torch.rand(N, generator=g, device=dev, dtype=torch.float64) * math.log(V + 1.0)).long().sub_(1).clamp_(0, V - 1)
        tokens = torch.randperm(V, generator=g, device=dev)[rank]
        tokens[torch.rand(N, generator=g, device=dev) < case["pad"]] = -1
        s["tokens"] = tokens
        s["weight"] = normal(V, D, dtype=dt).mul_(0.02)
        if case["scale"] == "all":
            s["scale"] = math.sqrt(D)
        elif case["scale"] == "each":
            s["scale"] = torch.rand(N, generator=g, device=dev).add_(0.25).to(dt)
        if case["train"]:
            s["dout"] = normal(N, D, dtype=dt).mul_(0.01)
            s["weight"].requires_grad_()
            if case["scale"] == "each":
                s["scale"].requires_grad_()
    else:
        # the teacher's logits fall from about 12; the student's are near them, among others about zero
        V, K = case["V"], case["K"]
        place = torch.arange(K, device=dev)
        apart = 1 + (torch.rand(N, 1, generator=g, device=dev, dtype=torch.float64) * (V // K)).long().clamp_max(V // K - 1)
        index = (torch.randint(0, V, (N, 1), generator=g, device=dev) + apart * place) % V  # all different
        top = 12.0 - 1.5 * torch.log1p(place) + 0.5 * normal(N, K)
        logits = normal(N, V, dtype=dt).mul_(1.5)
        logits.scatter_(1, index, (top + 0.7 * normal(N, K)).to(dt))
        if case["ragged"]:
            there = (torch.rand(N, 1, generator=g, device=dev) * (K + 1)).floor()
            index = index.masked_fill(place >= there, -1)
        s["logits"], s["top"], s["index"] = logits, top.to(dt), index
        if case["weights"]:
            u = torch.rand(N, generator=g, device=dev)
            s["weights"] = torch.where(u < 0.2, 0.0, u)
            s["weights"][0] = 1.0
        if case["train"]:
            s["logits"].requires_grad_()
            s["grad"] = torch.full((N,) if case["rows"] else (), case["scale"], device=dev)
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the framework's operators -------------------------------------------------------------


def _run_own(s):
    import flexsae_amd as flex

    c = s["case"]
    if c["op"] == "norm":
        if c["stats"]:
            y, mean, rstd = flex.layer_norm_stats(s["x"], s.get("weight"), s.get("bias"), eps=_EPS)
            return {"y": y, "mean": mean, "rstd": rstd}
        y = flex.layer_norm(s["x"], s.get("weight"), s.get("bias"), eps=_EPS)
        if not c["train"]:
            return {"y": y}
        names = ("x", "weight", "bias") if c["affine"] else ("x",)
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return dict({"y": y.detach()}, **{"d" + k: v for k, v in zip(names, grads)})
    if c["op"] == "lookup":
        out = flex.embedding_lookup(s["tokens"], s["weight"], s.get("scale"))
        if not c["train"]:
            return {"out": out}
        names = ("weight", "scale") if c["scale"] == "each" else ("weight",)
        grads = torch.autograd.grad(out, [s[k] for k in names], s["dout"])
        return dict({"out": out.detach()}, **{"d" + k: v for k, v in zip(names, grads)})
    loss = flex.distillation_loss(s["logits"], s["top"], s["index"], temperature=c["T"], row_weights=s.get("weights"),
                                  reduction="none" if c["rows"] else "mean")
    if not c["train"]:
        return {"loss": loss}
    dlogits, = torch.autograd.grad(loss, s["logits"], s["grad"])
    return {"loss": loss.detach(), "dlogits": dlogits}


# ---- the plain form ------------------------------------------------------------------------


def _plain_norm(s):
    c = s["case"]
    dt = _DTYPES[c["dtype"]]
    x = s["x"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = (centred.square().mean(1, keepdim=True) + _EPS).rsqrt()
    unit = centred * rstd
    y = unit * s["weight"].float() + s["bias"].float() if c["affine"] else unit
    out = {"y": y.to(dt)}
    if c["stats"]:
        out["mean"], out["rstd"] = x.mean(1), rstd[:, 0]
    if c["train"]:
        dy = s["dy"].float()
        du = dy * s["weight"].float() if c["affine"] else dy
        out["dx"] = (rstd * (du - du.mean(1, keepdim=True) - unit * (du * unit).mean(1, keepdim=True))).to(dt)
        if c["affine"]:
            out["dweight"], out["dbias"] = (dy * unit).sum(0).to(dt), dy.sum(0).to(dt)
    return out


def _plain_lookup(s):
    c = s["case"]
    dt = _DTYPES[c["dtype"]]
    there = (s["tokens"] >= 0) & (s["tokens"] < c["V"])
    at = torch.where(there, s["tokens"], 0)
    rows = s["weight"][at].float()
    scale = s["scale"].float()[:, None] if c["scale"] == "each" else s.get("scale", 1.0)
    out = {"out": torch.where(there[:, None], rows * scale, 0.0).to(dt)}
    if c["train"]:
        dout = torch.where(there[:, None], s["dout"].float(), 0.0)
        out["dweight"] = torch.zeros(c["V"], c["D"], device="cuda").index_add_(0, at, dout * scale).to(dt)
        if c["scale"] == "each":
            out["dscale"] = (dout * rows).sum(1).to(dt)
    return out


def _plain_distill(s):
    c = s["case"]
    T, there = c["T"], s["index"] >= 0
    at = torch.where(there, s["index"], 0)
    weights = s["weights"] if c["weights"] else torch.ones(c["N"], device="cuda")
    part = weights if c["rows"] else weights / weights.sum()
    any_ = there.any(1)
    t = torch.where(there, s["top"].float() / T, -math.inf)
    t = t - torch.where(any_, t.amax(1), 0.0)[:, None]
    log_p = t - torch.where(any_, t.exp().sum(1), 1.0).log()[:, None]
    p = log_p.exp()
    z = s["logits"].float() / T
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    log_q = z.gather(1, at) - top - total.log()
    kl = torch.where(there, p * (log_p - log_q), 0.0).sum(1)
    losses = T * T * part * kl
    out = {"loss": losses if c["rows"] else losses.sum()}
    if c["train"]:
        d = (e / total * any_[:, None]).scatter_add_(1, at, torch.where(there, -p, 0.0))
        out["dlogits"] = (d * (part * (T * c["scale"]))[:, None]).to(_DTYPES[c["dtype"]])
    return out


def _run_plain(s):
    with torch.no_grad():
        return {"norm": _plain_norm, "lookup": _plain_lookup, "distill": _plain_distill}[s["case"]["op"]](s)


# ---- the definition, in 64 bits ------------------------------------------------------------


def exact(case, seed):
    """From the formulas, in float64, some rows or columns at a time:

        y = (x - m) r w + b,  m the mean of the row, r = 1 / sqrt(mean((x - m)^2) + eps)
        with u = (x - m) r and g = dy w:  dx = r (g - mean(g) - u mean(g u)),  dw = sum over rows of dy u,  db = of dy

        out[n] = scale[n] W[token[n]];  dW[v] = sum over n with token[n] = v of scale[n] dout[n],  dscale[n] = <dout[n], W[token[n]]>

        L[n] = T^2 a[n] sum over k of p[k] (log p[k] - log q[index[k]]),  a the rows' weights (divided by their sum where the
        mean is taken, L = sum of L[n]),  p = softmax(top / T) over the stored places, q = softmax(logits / T);  a row without
        stored places counts as zero;  dL[n] / dlogits[n, v] = T a[n] (q[v] - sum over k with index[k] = v of p[k])
    """
    f64 = torch.float64
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    N = case["N"]
    if case["op"] == "norm":
        D = case["D"]
        w = s["weight"].to(f64) if case["affine"] else torch.ones(D, dtype=f64, device="cuda")
        b = s["bias"].to(f64) if case["affine"] else torch.zeros(D, dtype=f64, device="cuda")
        ys, means, rstds, dxs, dw, db = [], [], [], [], torch.zeros_like(w), torch.zeros_like(w)
        for r in range(0, N, 8192):
            x = s["x"][r:r + 8192].to(f64)
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            rstd = 1.0 / torch.sqrt(var + _EPS)
            u = (x - mean) * rstd
            ys.append(torch.addcmul(b, u, w))
            means.append(mean[:, 0])
            rstds.append(rstd[:, 0])
            if case["train"]:
                dy = s["dy"][r:r + 8192].to(f64)
                gw = dy * w
                along = gw.mul(u).mean(1, keepdim=True)
                dxs.append((gw - gw.sum(1, keepdim=True) / D - u * along) * rstd)
                dw += dy.mul(u).sum(0)
                db += dy.sum(0)
        out = {"y": torch.cat(ys)}
        if case["stats"]:
            out["mean"], out["rstd"] = torch.cat(means), torch.cat(rstds)
        if case["train"]:
            out["dx"] = torch.cat(dxs)
            if case["affine"]:
                out["dweight"], out["dbias"] = dw, db
        return out
    if case["op"] == "lookup":
        V, D, tokens = case["V"], case["D"], s["tokens"]
        places = torch.nonzero(tokens >= 0)[:, 0]
        kept = tokens[places]
        factor = torch.full((N,), float(s["scale"]) if case["scale"] == "all" else 1.0, dtype=f64, device="cuda")
        if case["scale"] == "each":
            factor = s["scale"].to(f64)
        out = {"out": torch.zeros(N, D, dtype=f64, device="cuda")}
        if case["train"]:
            out["dweight"] = torch.zeros(V, D, dtype=f64, device="cuda")
            dscale = torch.zeros(N, dtype=f64, device="cuda")
        for a in range(0, D, 512):
            cols = slice(a, min(D, a + 512))
            rows = s["weight"][:, cols].index_select(0, kept).to(f64)
            out["out"][places, cols] = factor[places, None] * rows
            if case["train"]:
                dout = s["dout"][:, cols].index_select(0, places).to(f64)
                dscale[places] += dout.mul(rows).sum(1)
                piece = torch.zeros(V, cols.stop - cols.start, dtype=f64, device="cuda")
                out["dweight"][:, cols] = piece.index_add_(0, kept, dout * factor[places, None])
        if case["train"] and case["scale"] == "each":
            out["dscale"] = dscale
        return out
    T, V = case["T"], case["V"]
    a = s["weights"].to(f64) if case["weights"] else torch.ones(N, dtype=f64, device="cuda")
    a = a if case["rows"] else a / a.sum()
    losses = torch.zeros(N, dtype=f64, device="cuda")
    out = {}
    if case["train"]:
        out["dlogits"] = torch.empty(N, V, dtype=f64, device="cuda")
    for r in range(0, N, 512):
        at = slice(r, min(N, r + 512))
        index = s["index"][at]
        there = index >= 0
        some = there.sum(1, keepdim=True) > 0
        log_q = torch.log_softmax(s["logits"][at].to(f64) / T, 1)
        log_p = torch.log_softmax((s["top"][at].to(f64) / T).masked_fill(~there, -1e300), 1)
        p = log_p.exp() * there
        rows = (p * (log_p - log_q.gather(1, index.clamp_min(0)))).masked_fill(~there, 0.0).sum(1)
        losses[at] = T * T * a[at] * rows
        if case["train"]:
            d = log_q.exp_().scatter_add_(1, index.clamp_min(0), -p).mul_(some)
            out["dlogits"][at] = d.mul_((T * case["scale"]) * a[at][:, None])
    out["loss"] = losses if case["rows"] else losses.sum()
    return out
