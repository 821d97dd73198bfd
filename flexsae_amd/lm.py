"""What stands around a dictionary that is trained inside a language model: the layer norm of activations, the rows of a per-token
table that are added to a reconstruction, and the distillation loss that compares the model's logits with the dictionary in it to
the top logits that the model gave without.

    y, mean, rstd = layer_norm_stats(activations)                     # into the encoder; scales the reconstruction back
    x = reconstruction + embedding_lookup(tokens, table, gates)
    loss = distillation_loss(layer_norm(x, w, b) @ unembedding, top_logits, top_indices, row_weights=mask)

Tensors are float32, bfloat16 or float16, on one GPU, of any leading shape; arithmetic and sums are in fp32 and each result is
rounded once.  Everything runs on the current stream of the tensors' device, and nothing synchronises.  The reference has no
counterpart: its losses end at the reconstruction.

The ops under ``flexsae_amd::`` (``layer_norm_fwd``, ``layer_norm_bwd``, ``lookup_fwd``, ``lookup_bwd``, ``distill_fwd``,
``distill_bwd``) are what traced and observed calls see; an ordinary eager call goes through the extension module to the same
kernels.  Gradients have no gradients of their own.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib, ops
from .ops import _DTYPES, _flag_for, _native, _on_device, _ptr, _stream


def _on_one_gpu(*tensors: Tuple[str, Optional[Tensor]]) -> torch.device:
    dev = tensors[0][1].device
    for name, t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError(f"flexsae_amd's operators run on an AMD GPU only (tensors must live on a 'cuda' device), {name} is "
                               f"on {t.device}")
        if t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, {tensors[0][0]} on {dev}")
    return dev


def _float(name: str, t: Tensor) -> None:
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def _indices(name: str, t: Tensor) -> Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")
    return t.to(torch.int64)


def _no_tangents(*tensors: Optional[Tensor]) -> None:
    """The ops have no forward-mode derivatives, and torch would leave them out without a word."""
    if torch.compiler.is_compiling() or forward_ad._current_level < 0:
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("flexsae_amd's operators have no forward-mode derivatives")


def _there(t: Tensor) -> Tensor:
    """A zero tensor, which has no memory, gets some."""
    return torch.zeros(t.shape, dtype=t.dtype, device=t.device) if t.numel() and t.data_ptr() == 0 else t


def _rows(t: Tensor) -> Tuple[Tensor, int]:
    """The tensor, contiguous if need be, and the distance between its rows in elements."""
    t = _there(t)
    cols = t.shape[-1]
    if t.numel() and (cols == 1 or t.stride(-1) == 1):
        rows, stride = 1, cols
        for n, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if rows == 1:
                stride = step
            elif step != stride * rows:
                break
            rows *= n
        else:
            return t, stride
    return t.contiguous(), cols


# ---- layer norm ----------------------------------------------------------------------------


def _check_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> None:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: expected rows of at least one column, got {tuple(x.shape)}")
    _float("x", x)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _float(name, t)
        if tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"layer_norm: {name} is {tuple(t.shape)}, rows have {x.shape[-1]} columns")
    if x.shape[-1] >= 2 ** 27 or x.numel() // x.shape[-1] >= 2 ** 32:
        raise ValueError("sizes beyond the kernels' index range: need fewer than 2^32 rows of fewer than 2^27 columns")
    if not 0 <= eps < math.inf:
        raise ValueError(f"layer_norm: eps must be finite and not negative, got {eps}")
    _on_one_gpu(("x", x), ("weight", weight), ("bias", bias))


def _norm(x: Tensor, x_stride: int, dy_stride: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> _lib.Norm:
    kind = lambda t: _lib.F32 if t is None else _DTYPES[t.dtype]
    return _lib.Norm(x.numel() // x.shape[-1], x.shape[-1], x_stride, dy_stride, eps, _DTYPES[x.dtype], kind(weight), kind(bias))


def _or_null(t: Optional[Tensor]):
    return None if t is None else _ptr(t)


@torch.library.custom_op("flexsae_amd::layer_norm_fwd", mutates_args=())
def _norm_fwd_op(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    _check_norm(x, weight, bias, eps)
    lib = _lib.load()
    with _on_device(x.device):
        x, stride = _rows(x)
        weight, bias = (t if t is None else _there(t).contiguous() for t in (weight, bias))
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mean, rstd = (torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) for _ in range(2))
        n = _norm(x, stride, 0, weight, bias, eps)
        _lib.check(lib.flexsae_layer_norm_fwd(ctypes.byref(n), _ptr(x), _or_null(weight), _or_null(bias), _ptr(y), _ptr(mean),
                                              _ptr(rstd), _stream()), "flexsae_layer_norm_fwd")
    return y, mean, rstd


@_norm_fwd_op.register_fake
def _(x, weight, bias, eps):
    return (x.new_empty(x.shape), *(x.new_empty(x.shape[:-1], dtype=torch.float32) for _ in range(2)))


@torch.library.custom_op("flexsae_amd::layer_norm_bwd", mutates_args=())
def _norm_bwd_op(dy: Tensor, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], mean: Tensor, rstd: Tensor, need_x: bool,
                 need_weight: bool, need_bias: bool) -> Tuple[Tensor, Tensor, Tensor]:
    _check_norm(x, weight, bias, 0.0)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"layer_norm: the gradient is {dy.dtype} {tuple(dy.shape)}, x {x.dtype} {tuple(x.shape)}")
    for t in (mean, rstd):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1]:
            raise ValueError(f"layer_norm: a saved tensor is {t.dtype} {tuple(t.shape)}, x has rows {tuple(x.shape[:-1])}")
    dev = _on_one_gpu(("x", x), ("the gradient", dy), ("mean", mean), ("rstd", rstd))
    lib = _lib.load()
    with _on_device(dev):
        x, x_stride = _rows(x)
        dy, dy_stride = _rows(dy)
        mean, rstd = _there(mean).contiguous(), _there(rstd).contiguous()
        weight = weight if weight is None else _there(weight).contiguous()
        make = lambda shape, t, need: torch.empty(shape if need else (0,), dtype=(x if t is None else t).dtype, device=dev)
        dx = make(x.shape, x, need_x)
        dw, db = make(x.shape[-1:], weight, need_weight), make(x.shape[-1:], bias, need_bias)
        n = _norm(x, x_stride, dy_stride, weight, bias, 0.0)
        nbytes = lib.flexsae_layer_norm_bwd_workspace_bytes(ctypes.byref(n)) if need_weight or need_bias else 0
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        at = lambda t, need: _ptr(t) if need and t.numel() else None
        _lib.check(lib.flexsae_layer_norm_bwd(ctypes.byref(n), _ptr(x), _ptr(dy), _or_null(weight), _ptr(mean), _ptr(rstd),
                                              at(dx, need_x), at(dw, need_weight), at(db, need_bias), _ptr(workspace), nbytes,
                                              _stream()), "flexsae_layer_norm_bwd")
    return dx, dw, db


@_norm_bwd_op.register_fake
def _(dy, x, weight, bias, mean, rstd, need_x, need_weight, need_bias):
    make = lambda shape, t, need: (x if t is None else t).new_empty(shape if need else (0,))
    return make(x.shape, x, need_x), make(x.shape[-1:], weight, need_weight), make(x.shape[-1:], bias, need_bias)


def _norm_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    _, mean, rstd = output
    ctx.save_for_backward(x, weight, bias, mean, rstd)
    ctx.mark_non_differentiable(mean, rstd)
    ctx.set_materialize_grads(False)


def _norm_backward(ctx, dy, *_):
    if dy is None:
        return None, None, None, None
    needs = ctx.needs_input_grad[:3]
    grads = _norm_bwd_op(dy, *ctx.saved_tensors, *needs)
    return (*(g if need else None for g, need in zip(grads, needs)), None)


_norm_fwd_op.register_autograd(_norm_backward, setup_context=_norm_setup)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) * rstd * weight + bias`` of the rows along the last dimension, in x's type, differentiable with respect to x,
    weight and bias; ``rstd = 1 / sqrt(mean((x - mean)**2) + eps)``.

    x: any leading shape, also none or empty; rows at any distance from each other are read where they are, others copied.
    weight, bias: ``[columns]``, each None or of a type of its own, which its gradient has too.  Sums are in fp32, those of the
    weight's gradient over the rows too, in an order that the sizes fix (the same bits on every run)."""
    native = _native(x)
    if native is not None:
        y = native.layer_norm(x, weight, bias, eps, 0)
        if y is not None:
            return y
    _no_tangents(x, weight, bias)
    _check_norm(x, weight, bias, float(eps))
    return _norm_fwd_op(x, weight, bias, float(eps))[0]


def layer_norm_stats(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                     eps: float = 1e-5) -> Tuple[Tensor, Tensor, Tensor]:
    """``(layer_norm(x, weight, bias, eps), mean, rstd)``: with what takes a reconstruction of y back to x's scale
    (``y / rstd[..., None] + mean[..., None]``), fp32 and of x's leading shape.  mean and rstd are constants to autograd."""
    native = _native(x)
    if native is not None:
        out = native.layer_norm(x, weight, bias, eps, 1)
        if out is not None:
            return out
    _no_tangents(x, weight, bias)
    _check_norm(x, weight, bias, float(eps))
    y, mean, rstd = _norm_fwd_op(x, weight, bias, float(eps))
    return y, mean.detach(), rstd.detach()


# ---- lookup --------------------------------------------------------------------------------


def _check_lookup(tokens: Tensor, weight: Tensor, scale: Optional[Tensor], factor: float) -> None:
    if tokens.dtype != torch.int64:
        raise TypeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    _float("weight", weight)
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"embedding_lookup: expected weight[V, D] with at least one element, got {tuple(weight.shape)}")
    if weight.shape[0] >= 2 ** 31 or weight.shape[1] >= 2 ** 29 or tokens.numel() >= 2 ** 32:
        raise ValueError("sizes beyond the kernels' index range: need V < 2^31, D < 2^29 and fewer than 2^32 tokens")
    if scale is not None:
        _float("scale", scale)
        if scale.shape != tokens.shape:
            raise ValueError(f"embedding_lookup: scale is {tuple(scale.shape)}, tokens {tuple(tokens.shape)}")
    if not -math.inf < factor < math.inf:
        raise ValueError(f"embedding_lookup: scale must be finite, got {factor}")
    _on_one_gpu(("weight", weight), ("tokens", tokens), ("scale", scale))


def _lookup(tokens: Tensor, weight: Tensor, scale: Optional[Tensor], factor: float, weight_stride: int,
            dout_stride: int) -> _lib.Lookup:
    return _lib.Lookup(tokens.numel(), weight.shape[0], weight.shape[1], weight_stride, dout_stride, factor, _DTYPES[weight.dtype],
                       _lib.F32 if scale is None else _DTYPES[scale.dtype])


@torch.library.custom_op("flexsae_amd::lookup_fwd", mutates_args=())
def _lookup_fwd_op(tokens: Tensor, weight: Tensor, scale: Optional[Tensor], factor: float) -> Tensor:
    _check_lookup(tokens, weight, scale, factor)
    lib = _lib.load()
    dev = weight.device
    with _on_device(dev):
        tokens = _there(tokens).contiguous()
        weight, stride = _rows(weight)
        scale = scale if scale is None else _there(scale).contiguous()
        out = torch.empty((*tokens.shape, weight.shape[1]), dtype=weight.dtype, device=dev)
        l = _lookup(tokens, weight, scale, factor, stride, 0)
        _lib.check(lib.flexsae_lookup_fwd(ctypes.byref(l), _ptr(tokens), _ptr(weight), _or_null(scale), _ptr(out),
                                          _ptr(_flag_for(dev)), _stream()), "flexsae_lookup_fwd")
        if ops._check_indices:
            ops.check_index_flag(dev)
    return out


@_lookup_fwd_op.register_fake
def _(tokens, weight, scale, factor):
    return weight.new_empty((*tokens.shape, weight.shape[1]))


@torch.library.custom_op("flexsae_amd::lookup_bwd", mutates_args=())
def _lookup_bwd_op(dout: Tensor, tokens: Tensor, weight: Tensor, scale: Optional[Tensor], factor: float, need_weight: bool,
                   need_scale: bool) -> Tuple[Tensor, Tensor]:
    _check_lookup(tokens, weight, scale, factor)
    if dout.dtype != weight.dtype or dout.shape != (*tokens.shape, weight.shape[1]):
        raise ValueError(f"embedding_lookup: the gradient is {dout.dtype} {tuple(dout.shape)}, tokens {tuple(tokens.shape)}, weight "
                         f"{weight.dtype} {tuple(weight.shape)}")
    dev = _on_one_gpu(("weight", weight), ("the gradient", dout))
    need_scale = need_scale and scale is not None
    lib = _lib.load()
    with _on_device(dev):
        tokens = _there(tokens).contiguous()
        weight, weight_stride = _rows(weight)
        dout, dout_stride = _rows(dout)
        scale = scale if scale is None else _there(scale).contiguous()
        dweight = torch.empty(weight.shape if need_weight else (0,), dtype=weight.dtype, device=dev)
        dscale = torch.empty(tokens.shape if need_scale else (0,), dtype=(weight if scale is None else scale).dtype, device=dev)
        l = _lookup(tokens, weight, scale, factor, weight_stride, dout_stride)
        nbytes = lib.flexsae_lookup_bwd_workspace_bytes(ctypes.byref(l))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.check(lib.flexsae_lookup_bwd(ctypes.byref(l), _ptr(tokens), _ptr(weight), _or_null(scale), _ptr(dout),
                                          _ptr(dweight) if need_weight else None,
                                          _ptr(dscale) if need_scale and tokens.numel() else None, _ptr(workspace), nbytes,
                                          _stream()), "flexsae_lookup_bwd")
    return dweight, dscale


@_lookup_bwd_op.register_fake
def _(dout, tokens, weight, scale, factor, need_weight, need_scale):
    return (weight.new_empty(weight.shape if need_weight else (0,)),
            (weight if scale is None else scale).new_empty(tokens.shape if need_scale and scale is not None else (0,)))


def _lookup_setup(ctx, inputs, output):
    tokens, weight, scale, ctx.factor = inputs
    ctx.save_for_backward(tokens, weight, scale)


def _lookup_backward(ctx, dout):
    needs = ctx.needs_input_grad[1:3]
    dweight, dscale = _lookup_bwd_op(dout, *ctx.saved_tensors, ctx.factor, *needs)
    return None, dweight if needs[0] else None, dscale if needs[1] else None, None


_lookup_fwd_op.register_autograd(_lookup_backward, setup_context=_lookup_setup)


def embedding_lookup(tokens: Tensor, weight: Tensor, scale: Union[None, float, Tensor] = None) -> Tensor:
    """``scale * weight[tokens]``: rows of ``weight[V, D]`` by token, ``[*tokens.shape, D]`` in the weight's type, differentiable
    with respect to weight and scale.

    tokens: int64 or int32, any shape.  A token of -1 stands for none (padding): a row of zeros without gradients, whose upstream
    gradient is not looked at.  So does any other outside ``[0, V)``, and is reported by ``check_index_flag``.
    scale: a number, or a tensor that broadcasts to the tokens' shape (a gate of every token), of a type of its own; shares of a
    broadcast scale's gradient are added up in fp32.
    The weight's gradient is dense and written once, summed in fp32 by sorted tokens in a fixed order (the same bits on every
    run)."""
    factor = 1.0
    if isinstance(scale, (int, float)):
        factor, scale = float(scale), None
    elif scale is not None and scale.shape != tokens.shape:
        _float("scale", scale)
        scale = scale.to(torch.float32).expand(tokens.shape)  # (shares of its gradient are added up before they are rounded)
    tokens = _indices("tokens", tokens)
    native = _native(weight)
    if native is not None:
        out = native.embedding_lookup(tokens, weight, scale, factor)
        if out is not None:
            return out
    _no_tangents(weight, scale)
    _check_lookup(tokens, weight, scale, factor)
    return _lookup_fwd_op(tokens, weight, scale, factor)


# ---- distillation --------------------------------------------------------------------------


def _check_distill(logits: Tensor, top: Tensor, index: Tensor, row_weights: Optional[Tensor], temperature: float) -> None:
    _float("logits", logits)
    _float("top_logits", top)
    if index.dtype != torch.int64:
        raise TypeError(f"top_indices must be int64 or int32, got {index.dtype}")
    if logits.dim() < 1 or logits.numel() == 0:
        raise ValueError(f"distillation_loss: expected logits[..., V] with at least one element, got {tuple(logits.shape)}")
    if top.shape != index.shape or top.shape[:-1] != logits.shape[:-1] or top.dim() != logits.dim() or top.shape[-1] == 0:
        raise ValueError(f"distillation_loss: logits {tuple(logits.shape)}, top_logits {tuple(top.shape)}, top_indices "
                         f"{tuple(index.shape)}: expected [..., V] and twice [..., K]")
    if row_weights is not None and (row_weights.shape != logits.shape[:-1] or row_weights.dtype != torch.float32):
        raise ValueError(f"distillation_loss: row_weights is {row_weights.dtype} {tuple(row_weights.shape)}, rows "
                         f"{tuple(logits.shape[:-1])}")
    if not 0 < temperature < math.inf:
        raise ValueError(f"distillation_loss: temperature must be positive and finite, got {temperature}")
    if not 1e-18 < temperature < 1e18:
        raise ValueError(f"distillation_loss: temperature must be within 1e-18 and 1e18, got {temperature}")
    if logits.shape[-1] >= 2 ** 31 or logits.numel() // logits.shape[-1] >= 2 ** 31:
        raise ValueError("sizes beyond the kernels' index range: need fewer than 2^31 rows and V < 2^31")
    _on_one_gpu(("logits", logits), ("top_logits", top), ("top_indices", index), ("row_weights", row_weights))


def _distill(logits: Tensor, stride: int, top: Tensor, temperature: float, by_row: bool) -> _lib.Distill:
    return _lib.Distill(logits.numel() // logits.shape[-1], logits.shape[-1], top.shape[-1], stride, temperature,
                        _DTYPES[logits.dtype], _DTYPES[top.dtype], _lib.DISTILL_BY_ROW if by_row else 0)


@torch.library.custom_op("flexsae_amd::distill_fwd", mutates_args=())
def _distill_fwd_op(logits: Tensor, top: Tensor, index: Tensor, row_weights: Optional[Tensor], temperature: float,
                    by_row: bool) -> Tuple[Tensor, Tensor]:
    _check_distill(logits, top, index, row_weights, temperature)
    lib = _lib.load()
    dev = logits.device
    with _on_device(dev):
        logits, stride = _rows(logits)
        top, index = _there(top).contiguous(), _there(index).contiguous()
        row_weights = row_weights if row_weights is None else _there(row_weights).contiguous()
        d = _distill(logits, stride, top, temperature, by_row)
        loss = torch.empty(logits.shape[:-1] if by_row else (), dtype=torch.float32, device=dev)
        stats = torch.empty(d.rows + 1, 4, dtype=torch.float32, device=dev)
        nbytes = lib.flexsae_distill_workspace_bytes(ctypes.byref(d))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.check(lib.flexsae_distill_fwd(ctypes.byref(d), _ptr(logits), _ptr(top), _ptr(index), _or_null(row_weights), _ptr(loss),
                                           _ptr(stats), None, _ptr(workspace), nbytes, _ptr(_flag_for(dev)), _stream()),
                   "flexsae_distill_fwd")
        if ops._check_indices:
            ops.check_index_flag(dev)
    return loss, stats


@_distill_fwd_op.register_fake
def _(logits, top, index, row_weights, temperature, by_row):
    rows = logits.numel() // logits.shape[-1]
    return (logits.new_empty(logits.shape[:-1] if by_row else (), dtype=torch.float32),
            logits.new_empty((rows + 1, 4), dtype=torch.float32))


@torch.library.custom_op("flexsae_amd::distill_bwd", mutates_args=())
def _distill_bwd_op(grad: Tensor, logits: Tensor, top: Tensor, index: Tensor, row_weights: Optional[Tensor], stats: Tensor,
                    temperature: float, by_row: bool) -> Tensor:
    _check_distill(logits, top, index, row_weights, temperature)
    rows = logits.numel() // logits.shape[-1]
    if grad.shape != (logits.shape[:-1] if by_row else ()):
        raise ValueError(f"distillation_loss: the gradient is {tuple(grad.shape)}, logits {tuple(logits.shape)}")
    if stats.dtype != torch.float32 or stats.shape != (rows + 1, 4):
        raise ValueError(f"distillation_loss: a saved tensor is {stats.dtype} {tuple(stats.shape)}, expected float32 {(rows + 1, 4)}")
    dev = _on_one_gpu(("logits", logits), ("the gradient", grad), ("stats", stats))
    lib = _lib.load()
    with _on_device(dev):
        logits, stride = _rows(logits)
        top, index, stats = (ops._prep(t) for t in (top, index, stats))
        row_weights = row_weights if row_weights is None else _there(row_weights).contiguous()
        grad = _there(grad.to(torch.float32)).contiguous()
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        d = _distill(logits, stride, top, temperature, by_row)
        _lib.check(lib.flexsae_distill_bwd(ctypes.byref(d), _ptr(logits), _ptr(top), _ptr(index), _or_null(row_weights), _ptr(stats),
                                           _ptr(grad), 0, _ptr(dlogits), _stream()), "flexsae_distill_bwd")
    return dlogits


@_distill_bwd_op.register_fake
def _(grad, logits, top, index, row_weights, stats, temperature, by_row):
    return logits.new_empty(logits.shape)


def _distill_setup(ctx, inputs, output):
    logits, top, index, row_weights, ctx.temperature, ctx.by_row = inputs
    ctx.save_for_backward(logits, top, index, row_weights, output[1])
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _distill_backward(ctx, grad, _):
    if grad is None or not ctx.needs_input_grad[0]:
        return (None,) * 6
    return (_distill_bwd_op(grad, *ctx.saved_tensors, ctx.temperature, ctx.by_row), *(None,) * 5)


_distill_fwd_op.register_autograd(_distill_backward, setup_context=_distill_setup)


def distillation_loss(logits: Tensor, top_logits: Tensor, top_indices: Tensor, *, temperature: float = 1.0,
                      row_weights: Optional[Tensor] = None, reduction: str = "mean") -> Tensor:
    """The divergence of a student's ``logits[..., V]`` from a teacher of which only the top logits were stored (fp32),
    differentiable with respect to logits::

        T**2 * sum over k of p[k] * (log p[k] - log q[top_indices[k]])     p = softmax(top_logits / T) over the stored places
                                                                           q = softmax(logits / T)

    top_logits, top_indices: ``[..., K]``, indices int64 or int32.  A place with index -1 holds no logit; neither does one with any
    other index outside ``[0, V)``, which ``check_index_flag`` reports.  An entry may be stored more than once.
    row_weights: of the rows (``logits.shape[:-1]``; a mask, or numbers that are not negative).  A row of weight zero, or without a
    stored logit above minus infinity, counts as zero and has a gradient of zeros, whatever its logits are.
    reduction: "mean", over the rows by their weights (rows without stored logits among them; zero where all weights are), or
    "none", each row's loss times its weight.
    logits: rows at any distance from each other are read where they are.  Their gradient is rounded once.  With the mean it is
    made along with the loss for an upstream gradient of one, except for float16 logits, and made again by a backward pass with
    another, which reads and writes the logits' size once more.  One read serves the loss and that gradient for rows of up to 131072
    logits of 16 bits, or 65536 of fp32, with up to 1024 stored; longer ones are read twice."""
    if reduction not in ("mean", "none"):
        raise ValueError(f"distillation_loss: reduction must be 'mean' or 'none', got {reduction!r}")
    top_indices = _indices("top_indices", top_indices)
    if row_weights is not None:
        if row_weights.dtype != torch.bool and row_weights.dtype not in _DTYPES:
            raise TypeError(f"row_weights must be float32, bfloat16, float16 or bool, got {row_weights.dtype}")
        row_weights = row_weights.detach().to(torch.float32)
    by_row = reduction == "none"
    native = _native(logits)
    if native is not None:
        loss = native.distillation_loss(logits, top_logits, top_indices, row_weights, temperature, int(by_row))
        if loss is not None:
            return loss
    _no_tangents(logits)
    _check_distill(logits, top_logits, top_indices, row_weights, float(temperature))
    return _distill_fwd_op(logits, top_logits.detach(), top_indices, row_weights, float(temperature), by_row)[0]
