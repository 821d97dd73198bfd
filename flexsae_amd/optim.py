"""The optimiser that dictionaries are trained with: AdamW steps over many tensors in one launch, with states in 32 bits or in 8,
the global norm of the gradients, and rows held at length one; as functions over tensors and as ``AdamW``, an optimizer of
torch's kind.

Nothing here synchronises: the number of steps taken, the gradients' norm and whether a step is left out because the norm is not
finite all stay on the device, so a captured graph replays them too.  The reference has no counterpart (its training loop takes
an optimizer of torch, reference example.py:76-77).

The ops under ``flexsae_amd::`` (``grad_norm``, ``adamw_step_``, ``adamw8_step_``, ``adamw8_moments``) are what traced and
observed calls see; an ordinary eager call goes through the extension module to the same kernels.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from .ops import _DTYPES, _native, _on_device, _ptr, _stream

QUANT_BLOCK = 256  # elements that share the maxima of 8-bit states


def _on_gpu(tensors, what) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t.device.type != "cuda":
            raise RuntimeError(f"flexsae_amd's optimiser runs on an AMD GPU only ({what} must live on a 'cuda' device), got {t.device}")
        if t.device != dev:
            raise RuntimeError(f"{what}: tensors on {dev} and on {t.device}")
    return dev


def _layout(shape, unit_rows: bool) -> Tuple[int, int]:
    """(rows, columns) as the blocks of 8-bit states, and rows of length one, follow them."""
    n = math.prod(shape)
    if not unit_rows:
        return 1, n
    cols = shape[-1]
    return (n // cols if cols else 0), cols


def _addressable(t: Tensor, to: int = 0) -> bool:
    return t.is_contiguous() and (not to or t.data_ptr() % to == 0)


# ---- the gradients' norm -------------------------------------------------------------------


@torch.library.custom_op("flexsae_amd::grad_norm", mutates_args=())
def _grad_norm_op(grads: List[Tensor]) -> Tensor:
    dev = _on_gpu(grads, "grads")
    lib = _lib.load()
    with _on_device(dev):
        grads = [g.contiguous() for g in grads]
        table = (_lib.Grad * len(grads))(*((_ptr(g), g.numel(), _DTYPES[g.dtype]) for g in grads))
        nbytes = lib.flexsae_grad_norm_workspace_bytes(len(grads))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        _lib.check(lib.flexsae_grad_norm(table, len(grads), _ptr(norm), _ptr(workspace), nbytes, _stream()), "flexsae_grad_norm")
    return norm


@_grad_norm_op.register_fake
def _(grads):
    return grads[0].new_empty((), dtype=torch.float32)


def grad_norm(grads: Sequence[Tensor]) -> Tensor:
    """The 2-norm of all elements of all tensors together: 0-dim fp32, on their device.  Squares are summed in 64 bits in a fixed
    order (the same bits on every run); infinities and NaN reach the result.  It takes no part in autograd: a penalty on it has no
    gradient."""
    if isinstance(grads, Tensor) or len(grads) == 0:
        raise ValueError("grad_norm: expected a list of at least one tensor")
    native = _native(grads[0])
    if native is not None:
        norm = native.grad_norm(grads)
        if norm is not None:
            return norm
    for g in grads:
        if g.dtype not in _DTYPES:
            raise TypeError(f"grads must be float32, bfloat16 or float16, got {g.dtype}")
    return _grad_norm_op([g.detach() for g in grads])


# ---- the step ------------------------------------------------------------------------------


def adamw_counter(device=None, steps: int = 0) -> Tensor:
    """The ``counter`` of a step's calls: int64[2] on the device, the number of steps taken, and a word that the calls work with."""
    return torch.tensor([steps, 0], dtype=torch.int64, device="cuda" if device is None else device)


def adamw8_state(param: Tensor, unit_rows: bool = False) -> Tuple[Tensor, Tensor]:
    """``(codes, absmax)`` of a parameter that has not been stepped: uint8 ``[*shape, 2]`` and fp32 ``[rows, blocks, 2]``."""
    rows, cols = _layout(param.shape, unit_rows)
    absmax = torch.zeros(rows, -(-cols // QUANT_BLOCK), 2, dtype=torch.float32, device=param.device)
    return torch.zeros(*param.shape, 2, dtype=torch.uint8, device=param.device), absmax


def _check_step(bits, params, grads, state0, state1, masters, counter, lrs, weight_decays, lr, grad_norm, beta1, beta2, eps,
                grad_scale, max_norm, unit_rows):
    """What the kernels take for granted; says what is wrong."""
    n = len(params)
    if n == 0:
        raise ValueError("expected at least one parameter")
    names = ("exp_avgs", "exp_avg_sqs") if bits == 32 else ("codes", "absmax")
    lists = [("grads", grads), (names[0], state0), (names[1], state1)]
    for name, x in lists + [("lr", lrs), ("weight_decay", weight_decays)]:
        if len(x) != n:
            raise ValueError(f"{n} params and {len(x)} {name}")
    narrow = sum(p.dtype != torch.float32 for p in params)
    if masters and len(masters) != narrow:
        raise ValueError(f"{narrow} params of 16 bits and {len(masters)} masters")
    master_of = iter(masters)
    for i, p in enumerate(params):
        if p.dtype not in _DTYPES:
            raise TypeError(f"params must be float32, bfloat16 or float16, got {p.dtype}")
        if unit_rows and p.dim() < 2:
            raise ValueError(f"unit_rows: expected matrices, got params[{i}] of shape {tuple(p.shape)}")
        if grads[i].dtype != p.dtype or grads[i].shape != p.shape:
            raise ValueError(f"grads[{i}] is {grads[i].dtype} {tuple(grads[i].shape)}, params[{i}] {p.dtype} {tuple(p.shape)}")
        rows, cols = _layout(p.shape, unit_rows)
        want = ((torch.float32, tuple(p.shape)), (torch.float32, tuple(p.shape))) if bits == 32 else \
            ((torch.uint8, (*p.shape, 2)), (torch.float32, (rows, -(-cols // QUANT_BLOCK), 2)))
        for name, t, (dtype, shape) in zip(names, (state0[i], state1[i]), want):
            if t.dtype != dtype or tuple(t.shape) != shape:
                raise ValueError(f"{name}[{i}] is {t.dtype} {tuple(t.shape)}, expected {dtype} {shape}")
        master = next(master_of) if masters and p.dtype != torch.float32 else None
        if master is not None and (master.dtype != torch.float32 or master.shape != p.shape):
            raise ValueError(f"the master of params[{i}] is {master.dtype} {tuple(master.shape)}, expected float32 {tuple(p.shape)}")
    for t in (*params, *state0, *state1, *masters):
        if any(n > 1 and step == 0 for n, step in zip(t.shape, t.stride())):
            raise ValueError(f"a tensor of shape {tuple(t.shape)} and strides {t.stride()} has one memory for several elements")
    if counter.dtype != torch.int64 or counter.numel() != 2 or not counter.is_contiguous():
        raise ValueError("counter: expected int64[2] (adamw_counter)")
    for name, t in (("lr", lr), ("grad_norm", grad_norm)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != 1):
            raise ValueError(f"{name}: expected one float32 number, got {t.dtype} {tuple(t.shape)}")
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and eps >= 0):
        raise ValueError(f"expected 0 <= beta < 1 and eps >= 0, got beta1 {beta1}, beta2 {beta2}, eps {eps}")
    if not all(x >= 0 for x in (*lrs, *weight_decays)):
        raise ValueError("lr and weight_decay must not be negative")
    if not (grad_scale > 0 and math.isfinite(grad_scale)):
        raise ValueError(f"grad_scale must be positive and finite, got {grad_scale}")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if max_norm > 0 and grad_norm is None:
        raise ValueError("max_norm needs grad_norm, the norm of the gradients")
    return _on_gpu([*params, *(t for _, x in lists for t in x), *masters, counter,
                    *(t for t in (lr, grad_norm) if t is not None)], "tensors")


def _step(bits, params, grads, state0, state1, masters, counter, lrs, weight_decays, lr, grad_norm, beta1, beta2, eps,
          grad_scale, max_norm, unit_rows) -> None:
    """One call of flexsae_adamw_step.  ``masters``: those of the 16-bit params, in their order, or none (an op may change every
    tensor of this list, so that none of them may be one of the params).  Tensors that are not contiguous are stepped as copies."""
    dev = _check_step(bits, params, grads, state0, state1, masters, counter, lrs, weight_decays, lr, grad_norm, beta1, beta2,
                      eps, grad_scale, max_norm, unit_rows)
    lib = _lib.load()
    back = []

    def at(t: Tensor, to: int = 0) -> int:
        if not _addressable(t, to):
            c = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
            back.append((t, c))
            t = c
        return _ptr(t)

    with _on_device(dev):
        grads = [g.contiguous() for g in grads]
        table = (_lib.AdamwTensor * len(params))()
        master_of = iter(masters)
        for i, p in enumerate(params):
            rows, cols = _layout(p.shape, unit_rows)
            master = at(next(master_of)) if masters and p.dtype != torch.float32 else None
            table[i] = (at(p), _ptr(grads[i]), master, at(state0[i], 0 if bits == 32 else 2), at(state1[i], 0 if bits == 32 else 8),
                        rows, cols, lrs[i], weight_decays[i], _DTYPES[p.dtype])
        config = _lib.AdamwConfig(beta1, beta2, eps, grad_scale, max_norm, None if grad_norm is None else _ptr(grad_norm),
                                  None if lr is None else _ptr(lr), _ptr(counter), bits,
                                  _lib.ADAMW_UNIT_ROWS if unit_rows else 0)
        _lib.check(lib.flexsae_adamw_step(table, len(params), ctypes.byref(config), _stream()), "flexsae_adamw_step")
        for t, c in back:
            t.copy_(c)


@torch.library.custom_op("flexsae_amd::adamw_step_", mutates_args=("params", "exp_avgs", "exp_avg_sqs", "masters", "counter"))
def _adamw_op(params: List[Tensor], grads: List[Tensor], exp_avgs: List[Tensor], exp_avg_sqs: List[Tensor], masters: List[Tensor],
              counter: Tensor, lrs: List[float], weight_decays: List[float], lr: Optional[Tensor], grad_norm: Optional[Tensor],
              beta1: float, beta2: float, eps: float, grad_scale: float, max_norm: float, unit_rows: bool) -> None:
    _step(32, params, grads, exp_avgs, exp_avg_sqs, masters, counter, lrs, weight_decays, lr, grad_norm, beta1, beta2, eps,
          grad_scale, max_norm, unit_rows)


@torch.library.custom_op("flexsae_amd::adamw8_step_", mutates_args=("params", "codes", "absmax", "masters", "counter"))
def _adamw8_op(params: List[Tensor], grads: List[Tensor], codes: List[Tensor], absmax: List[Tensor], masters: List[Tensor],
               counter: Tensor, lrs: List[float], weight_decays: List[float], lr: Optional[Tensor], grad_norm: Optional[Tensor],
               beta1: float, beta2: float, eps: float, grad_scale: float, max_norm: float, unit_rows: bool) -> None:
    _step(8, params, grads, codes, absmax, masters, counter, lrs, weight_decays, lr, grad_norm, beta1, beta2, eps, grad_scale,
          max_norm, unit_rows)


@_adamw_op.register_fake
def _(*args):
    return None


@_adamw8_op.register_fake
def _(*args):
    return None


_Reals = Union[float, Sequence[float]]


def _call(bits, params, grads, state0, state1, masters, counter, lr, weight_decay, beta1, beta2, eps, grad_scale, grad_norm,
          max_norm, unit_rows) -> None:
    if isinstance(params, Tensor) or len(params) == 0:
        raise ValueError("expected a list of at least one parameter")
    if masters is not None and len(masters) == 0:
        masters = None
    max_norm = 0.0 if max_norm is None else max_norm
    native = _native(params[0])
    if native is not None and native.adamw(bits, params, grads, state0, state1, masters, counter, lr, weight_decay, beta1, beta2,
                                           eps, grad_scale, grad_norm, max_norm, unit_rows):
        return
    with torch.no_grad():
        args = _checked(bits, params, grads, state0, state1, masters, counter, lr, weight_decay, beta1, beta2, eps, grad_scale,
                        grad_norm, max_norm, unit_rows)
        op = _adamw_op if bits == 32 else _adamw8_op
        op(*([t.detach() for t in a] if i < 5 else a for i, a in enumerate(args)))


def _checked(bits, params, grads, state0, state1, masters, counter, lr, weight_decay, beta1, beta2, eps, grad_scale, grad_norm,
             max_norm, unit_rows) -> tuple:
    """The op's arguments, which are those of a step."""
    n = len(params)
    on_device = isinstance(lr, Tensor)
    lrs = [1.0] * n if on_device else [float(lr)] * n if isinstance(lr, (int, float)) else [float(x) for x in lr]
    wds = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else [float(x) for x in weight_decay]
    if masters is None:
        masters = []
    elif len(masters) != n:
        raise ValueError(f"{n} params and {len(masters)} masters")
    else:
        masters = [m for m, p in zip(masters, params) if p.dtype != torch.float32]
    args = (params, grads, state0, state1, masters, counter, lrs, wds, lr if on_device else None, grad_norm,
            float(beta1), float(beta2), float(eps), float(grad_scale), float(max_norm), bool(unit_rows))
    _check_step(bits, *args)
    return args


def _call_all(calls) -> None:
    """Steps, each given as the arguments of ``_call``: all of them, or none where one is refused."""
    native = _native(calls[0][1][0])
    if native is not None and native.adamw_all(calls):
        return
    for call in calls:
        _checked(*call)
    for call in calls:
        _call(*call)


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
               counter: Tensor, *, lr: Union[_Reals, Tensor] = 1e-3, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
               weight_decay: _Reals = 0.0, masters: Optional[Sequence[Tensor]] = None, unit_rows: bool = False,
               grad_norm: Optional[Tensor] = None, max_norm: Optional[float] = None, grad_scale: float = 1.0) -> None:
    """One AdamW step of all ``params``, in place; ``t = counter[0] + 1``::

        g = c * grad              c = min(1, max_norm / (grad_norm / grad_scale + 1e-6)) / grad_scale
        m = beta1 * m + (1 - beta1) * g
        v = beta2 * v + (1 - beta2) * g * g
        w = (1 - lr * weight_decay) * w - lr * (m / (1 - beta1**t)) / (sqrt(v / (1 - beta2**t)) + eps)

    params, grads: fp32, bf16 or fp16, of one device, each gradient of its parameter's type and shape; exp_avgs, exp_avg_sqs:
    m and v in fp32; counter: ``adamw_counter()``, shared by no other step.
    lr, weight_decay: a number, or one for each parameter; lr also a 0-dim fp32 tensor, read when the kernel runs.
    masters: fp32 weights that 16-bit params are the rounded copies of (an fp32 parameter's entry is ignored).
    unit_rows: matrices whose rows (along the last dimension) are held at length one: the part of g along the row is left out
    before, and the row divided by its length after.  A row of zeros stays one.  (Lengths between 1e-16 and 1e18: their squares are
    summed in fp32.)
    grad_norm: ``grad_norm(grads)``; one that is not finite makes the call change nothing, ``counter`` neither.  max_norm: clips
    by it (None or 0: does not).  grad_scale: the loss scale that the gradients carry.
    Arithmetic is in fp32; a weight without a master is rounded once.  The gradients are left as they are.  sqrt(v) is taken as
    2^-63 where it is less, which shows where eps is as small: with ``eps=0`` an element without any gradient so far stays where it
    is.  A launch takes up to 66 tensors; with unit_rows, of those that follow each other and go through the same kernel (by type,
    master and number of columns).  No two of the tensors that a call changes may share memory."""
    _call(32, params, grads, exp_avgs, exp_avg_sqs, masters, counter, lr, weight_decay, beta1, beta2, eps, grad_scale, grad_norm,
          max_norm, unit_rows)


def adamw8_step(params: Sequence[Tensor], grads: Sequence[Tensor], codes: Sequence[Tensor], absmax: Sequence[Tensor],
                counter: Tensor, *, lr: Union[_Reals, Tensor] = 1e-3, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                weight_decay: _Reals = 0.0, masters: Optional[Sequence[Tensor]] = None, unit_rows: bool = False,
                grad_norm: Optional[Tensor] = None, max_norm: Optional[float] = None, grad_scale: float = 1.0) -> None:
    """``adamw_step`` with m and v in 8 bits each, ``adamw8_state(param, unit_rows)``: two bytes an element in ``codes``, and two
    fp32 maxima of every block of 256 elements (of a row with unit_rows, else of the flattened parameter) in ``absmax``.  With
    ``a`` the block's maxima of \\|m\\| and of v, the bytes c stand for ``sign(c - 128) ((c - 128) / 127)^2 a`` and
    ``(c / 255)^4 a``, rounded to the nearest on the root's scale; a v above zero never becomes zero.  The step itself uses m and v
    before they are rounded.  A block with an infinity or NaN in m, or in v (the square of a gradient above 1.8e19 is
    one), has NaN there from then on, and in its weights from the next step on."""
    _call(8, params, grads, codes, absmax, masters, counter, lr, weight_decay, beta1, beta2, eps, grad_scale, grad_norm, max_norm,
          unit_rows)


# ---- the values of 8-bit states ------------------------------------------------------------


@torch.library.custom_op("flexsae_amd::adamw8_moments", mutates_args=())
def _moments_op(codes: List[Tensor], absmax: List[Tensor], dtype: torch.dtype) -> List[Tensor]:
    if dtype not in _DTYPES:
        raise TypeError(f"expected float32, bfloat16 or float16, got {dtype}")
    if len(codes) != len(absmax):
        raise ValueError(f"{len(codes)} codes and {len(absmax)} absmax")
    dev = _on_gpu([*codes, *absmax], "codes and absmax")
    codes = [c if _addressable(c, 2) else torch.empty_like(c, memory_format=torch.contiguous_format).copy_(c) for c in codes]
    absmax = [a if _addressable(a, 8) else torch.empty_like(a, memory_format=torch.contiguous_format).copy_(a) for a in absmax]
    out = [torch.empty(c.shape[:-1], dtype=dtype, device=dev) for c in codes for _ in range(2)]
    table = (_lib.Adamw8State * len(codes))()
    for i, (c, a) in enumerate(zip(codes, absmax)):
        rows = a.shape[0] if a.dim() == 3 else 0
        cols = c.numel() // 2 // rows if rows else 0
        if (c.dtype != torch.uint8 or a.dtype != torch.float32 or c.dim() < 1 or c.shape[-1] != 2 or a.dim() != 3
                or rows * cols * 2 != c.numel() or a.shape[2] != 2 or (rows and a.shape[1] != -(-cols // QUANT_BLOCK))):
            raise ValueError(f"codes[{i}] {c.dtype} {tuple(c.shape)} and absmax[{i}] {a.dtype} {tuple(a.shape)} are no state")
        table[i] = (_ptr(c), _ptr(a), _ptr(out[2 * i]), _ptr(out[2 * i + 1]), rows, cols)
    with _on_device(dev):
        _lib.check(_lib.load().flexsae_adamw8_moments(table, len(codes), _DTYPES[dtype], _stream()), "flexsae_adamw8_moments")
    return out


@_moments_op.register_fake
def _(codes, absmax, dtype):
    return [c.new_empty(c.shape[:-1], dtype=dtype) for c in codes for _ in range(2)]


def adamw8_moments(codes: Sequence[Tensor], absmax: Sequence[Tensor], dtype: torch.dtype = torch.float32
                   ) -> Tuple[List[Tensor], List[Tensor]]:
    """The values that 8-bit states stand for: ``(exp_avgs, exp_avg_sqs)`` in ``dtype``, for a log, a checkpoint, or a step with
    states in 32 bits."""
    if isinstance(codes, Tensor) or len(codes) == 0:
        raise ValueError("adamw8_moments: expected lists of at least one tensor")
    if dtype in _DTYPES:
        native = _native(codes[0])
        out = native.adamw8_moments(codes, absmax, _DTYPES[dtype]) if native is not None else None
        if out is not None:
            return out
    out = _moments_op(list(codes), list(absmax), dtype)
    return out[::2], out[1::2]


# ---- the optimizer -------------------------------------------------------------------------


_OPTIONS = ("lr", "betas", "eps", "weight_decay", "state_bits", "unit_rows", "master_weights")  # of a group


def _not_captured(device: torch.device, what: str) -> None:
    """Refuses what every replay of a captured step would do again."""
    if device.type == "cuda":
        with _on_device(device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"AdamW: a step in which {what} cannot be captured: take one with the same gradients first")


class AdamW(torch.optim.Optimizer):
    """AdamW of ``adamw_step`` / ``adamw8_step`` as an optimizer of torch's kind: parameter groups, schedulers, state_dict.

    Options of a group: ``lr`` (a float, or a 0-dim fp32 tensor on the device, which a captured step reads at every replay),
    ``betas``, ``eps``, ``weight_decay``, ``state_bits`` (32 or 8), ``unit_rows``, ``master_weights`` (16-bit parameters are
    stepped in fp32 and rounded; on unless switched off).
    max_norm: the gradients of all groups are clipped to this norm together.  skip_nonfinite: a step whose gradients hold an
    infinity or NaN changes nothing, as always with max_norm.  After a step with either ``grad_norm`` is the norm of the gradients
    as they were, on the device.
    Parameters without a gradient are left out of a step, their number of steps too.  A step is captured after one with gradients of
    the same parameters, which makes their states.  Whoever changes 16-bit parameters with master weights from outside calls
    ``reset_masters()``."""

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, unit_rows: bool = False, master_weights: bool = True,
                 max_norm: Optional[float] = None, skip_nonfinite: bool = False):
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      unit_rows=unit_rows, master_weights=master_weights))
        self.max_norm, self.skip_nonfinite = max_norm, skip_nonfinite
        self.grad_norm: Optional[Tensor] = None

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            if group["state_bits"] not in (32, 8):
                raise ValueError(f"state_bits must be 32 or 8, got {group['state_bits']}")
            if not (all(0 <= b < 1 for b in group["betas"]) and group["eps"] >= 0 and group["weight_decay"] >= 0):
                raise ValueError("expected 0 <= betas < 1, eps >= 0 and weight_decay >= 0")
            if not isinstance(group["lr"], Tensor) and not group["lr"] >= 0:
                raise ValueError(f"lr must not be negative, got {group['lr']}")
            if len(set(group["params"])) != len(group["params"]):
                raise ValueError("a parameter stands twice in a group: one step would change it in two places at once")
            if group["unit_rows"] and any(p.dim() < 2 for p in group["params"]):
                raise ValueError("unit_rows: expected matrices")
        except ValueError:
            self.param_groups.pop()
            raise

    def _new_state(self, p: Tensor, group, counter: Tensor) -> dict:
        s = {"counter": counter}
        if group["state_bits"] == 8:
            s["codes"], s["absmax"] = adamw8_state(p, group["unit_rows"])
        else:
            s["exp_avg"], s["exp_avg_sq"] = (torch.zeros(p.shape, dtype=torch.float32, device=p.device) for _ in range(2))
        if group["master_weights"] and p.dtype != torch.float32:
            s["master"] = p.detach().to(torch.float32).contiguous()
        return s

    def _cohorts(self, group):
        """What a step takes of the group: (params, grads, moments, masters, counter) of the parameters with gradients that have
        taken the same steps.  A parameter that now has none stays behind: the count of those it was stepped with goes on
        without it."""
        cohorts, behind, new, state = {}, {}, {}, self.state
        first, second = ("exp_avg", "exp_avg_sq") if group["state_bits"] == 32 else ("codes", "absmax")
        for p in group["params"]:
            g, s = p.grad, state.get(p)
            if g is None:
                if s:
                    behind.setdefault(id(s["counter"]), []).append(s)
                continue
            if not s:
                if g.is_sparse:
                    raise RuntimeError("AdamW takes dense gradients")
                _not_captured(p.device, "a parameter's states begin")
                if p.device not in new:
                    new[p.device] = adamw_counter(p.device)
                s = state[p] = self._new_state(p, group, new[p.device])
            counter = s["counter"]
            cohort = cohorts.get(id(counter))
            if cohort is None:
                cohort = cohorts[id(counter)] = ([], [], [], [], [], counter)
            cohort[0].append(p)
            cohort[1].append(g)
            cohort[2].append(s[first])
            cohort[3].append(s[second])
            cohort[4].append(s.get("master", p))
        for key, states in behind.items():
            if key in cohorts:
                _not_captured(states[0]["counter"].device, "a parameter without a gradient gets a count of its own")
                own = states[0]["counter"].clone()
                for s in states:
                    s["counter"] = own
        return list(cohorts.values())

    def step(self, closure=None, *, grad_scale: float = 1.0):
        """One step; ``grad_scale``: the loss scale that the gradients carry (they are left as they are).  Within a compiled function
        it runs as outside of one: which parameters are stepped together is up to the host."""
        if torch.compiler.is_compiling():
            return _uncompiled_step(self, closure, grad_scale)
        return self._step(closure, grad_scale)

    def _step(self, closure, grad_scale: float):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        cohorts = [(group, cohort) for group in self.param_groups for cohort in self._cohorts(group)]
        if not cohorts:
            return loss
        norm = None
        if self.max_norm is not None or self.skip_nonfinite:
            norm = self.grad_norm = grad_norm([g for _, cohort in cohorts for g in cohort[1]])
        calls = []
        for group, (params, grads, first, second, masters, counter) in cohorts:
            beta1, beta2 = group["betas"]
            calls.append((group["state_bits"], params, grads, first, second, masters if group["master_weights"] else None, counter,
                          group["lr"], group["weight_decay"], beta1, beta2, group["eps"], grad_scale, norm, self.max_norm or 0.0,
                          group["unit_rows"]))
        if len(calls) == 1:
            _call(*calls[0])
        else:
            _call_all(calls)
        return loss

    def moments(self, p: Tensor, dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
        """The first and second moment of a parameter that has been stepped, in ``dtype``."""
        s = self.state.get(p)
        if not s:
            raise KeyError("moments: the parameter has not been stepped")
        if "codes" in s:
            m, v = adamw8_moments([s["codes"]], [s["absmax"]], dtype)
            return m[0], v[0]
        return s["exp_avg"].to(dtype), s["exp_avg_sq"].to(dtype)

    def reset_masters(self) -> None:
        """Master weights from the parameters as they are: for whoever has changed those from outside (a step would otherwise bring
        back what the masters hold)."""
        for p, s in self.state.items():
            if "master" in s:
                s["master"].copy_(p.detach())

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite, "grad_norm": None}

    def load_state_dict(self, state_dict) -> None:
        """As torch's, with states kept in their own types (torch's own would turn them into the parameter's).  Parameters of a
        group that have taken the same number of steps share a count again."""
        loaded = {}

        def take(_, state_dict):  # what the hooks before it have left: the groups are torch's business
            if (any("counter" not in s for s in state_dict["state"].values())
                    or any(k not in group for group in state_dict["param_groups"] for k in _OPTIONS)):
                raise ValueError("load_state_dict: the states are not those of this optimizer")
            loaded.update(state_dict)
            return {**state_dict, "state": {}}

        def fill(_):
            saved = loaded["state"]
            for group, old in zip(self.param_groups, loaded["param_groups"]):
                counters = {}
                for p, key in zip(group["params"], old["params"]):
                    if key not in saved:
                        continue
                    s = {k: v.detach().to(p.device).clone() if isinstance(v, Tensor) else v for k, v in saved[key].items()}
                    counter = s["counter"]
                    s["counter"] = counters.setdefault((p.device, int(counter[0])), counter)
                    self.state[p] = s

        before = self.register_load_state_dict_pre_hook(take)  # (the last of them)
        after = self.register_load_state_dict_post_hook(fill, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            before.remove()
            after.remove()


@torch._disable_dynamo  # (torch.compiler.disable, but for the compiler's import here)
def _uncompiled_step(opt: AdamW, closure, grad_scale: float):
    return opt._step(closure, grad_scale)
