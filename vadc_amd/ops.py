"""Operators on device tensors: what a streaming layer of one's own is made of, to run beside the models of vadc_amd.engine on the same GPU.

    linear       act(x W^T + b) + r                       matrix product with bias, activation and residual
    gated_delta  the gated delta rule                      a recurrence with one state per stream and head: many steps per call, or one
    group_norm   group norm with an activation or a gate   channels last; positions of a sequence together, or each token alone

Tensors are torch tensors on one gfx950 device, of one type (float32, float16 or bfloat16); the work is enqueued on torch's current stream of that device and may be captured into a
graph.  Sums, statistics and states are float32, an output is rounded once.  Strided tensors are taken as they are, as long as the innermost dimension is contiguous.  The operators
have no gradients: tensors that ask for them are refused while autograd records.  All arithmetic happens in libvadc_amd.so (include/vadc_amd.h: vadc_amd_linear, ...); a wrong
argument raises ValueError or TypeError before the device is touched, a failure of the library VadcAmdError.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _lib
from .engine import VadcAmdError

__all__ = ["linear", "group_norm", "gated_delta", "ACTIVATIONS"]

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# the C structs of include/vadc_amd.h, field by field
_LINEAR = struct.Struct("=5Q7q4i")
_NORM = struct.Struct("=7Qq4q6q3if")
_DELTA = struct.Struct("=9Qq6q12q4qqf3i")

Tensor = torch.Tensor


def _call(fn, packed: bytes, device: int):
    rc = fn(packed, torch._C._cuda_getCurrentRawStream(device))
    if rc != 0:
        raise VadcAmdError(rc, _lib.load().vadc_amd_last_error().decode())


def _bytes(fn, packed: bytes) -> int:
    n = fn(packed)
    if n < 0:
        raise VadcAmdError(n, _lib.load().vadc_amd_last_error().decode())
    return n


def _no_grad(what: str, *ts: Optional[Tensor]):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no gradient: call it under torch.no_grad() or with tensors that ask for none")


def _device(what: str, first: Tensor, *ts: Optional[Tensor]) -> int:
    d = first.device
    for t in ts:
        if t is not None and t.device != d:
            raise ValueError(f"{what}: tensors on {d} and on {t.device}")
    if d.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a gfx950 device, not on {d} (vadc_amd has no CPU fallback)")
    return d.index


def _activation(what: str, name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{what}: activation {name!r} is none of {', '.join(ACTIVATIONS)}") from None


def _dtype(what: str, first: Tensor, *ts: Optional[Tensor]) -> int:
    dt = first.dtype
    code = _DTYPES.get(dt)
    if code is None:
        raise TypeError(f"{what}: {dt} is none of float32, float16, bfloat16")
    for t in ts:
        if t is not None and t.dtype != dt:
            raise TypeError(f"{what}: tensors of {dt} and of {t.dtype}")
    return code


def _floats(what: str, name: str, t: Tensor):
    if t.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be float32, not {t.dtype}")


def _inner(what: str, **ts: Optional[Tensor]):
    for name, t in ts.items():
        if t is not None and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{what}: the last dimension of {name} must be contiguous")


def _span(t: Tensor):
    lo = t.data_ptr()
    return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else lo


def _apart(what: str, name: str, out: Tensor, **ts: Optional[Tensor]):
    lo, hi = _span(out)
    for other, t in ts.items():
        if t is not None:
            a, b = _span(t)
            if a < hi and lo < b:
                raise ValueError(f"{what}: {name} overlaps {other}")


def _same_or_apart(what: str, out: Tensor, **ts: Optional[Tensor]):
    for name, t in ts.items():
        if t is not None and not (t.data_ptr() == out.data_ptr() and t.stride() == out.stride()):
            _apart(what, "out", out, **{name: t})


def _lengths(what: str, lengths: Optional[Tensor], n: int):
    if lengths is None:
        return
    if lengths.dtype != torch.int32:
        raise TypeError(f"{what}: lengths must be int32, not {lengths.dtype}")
    if lengths.dim() != 1 or lengths.shape[0] != n or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths must be a contiguous tensor of {n}")


def _ptr(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: Tensor):
    """a tensor [..., n] as rows [m, n] without a copy, or None"""
    if t.dim() == 2:
        return t
    if t.dim() == 1:
        return t[None]
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        return None


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "none", residual: Optional[Tensor] = None,
           residual_first: bool = False, out: Optional[Tensor] = None) -> Tensor:
    """act(x W^T + bias) + residual, or with residual_first act(x W^T + bias + residual).

    x [..., in], weight [out, in], bias [out], residual [..., out]; returns [..., out] (in `out`, if given, which may be the residual).  Leading dimensions must make up rows at one
    distance.  activation: none, relu, silu, gelu (with erf), sigmoid."""
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    n, k = weight.shape
    shape = x.shape[:-1] + (n,)
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"linear: bias {tuple(bias.shape)} is not [{n}]")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"linear: residual {tuple(residual.shape)} is not {tuple(shape)}")
    if out is not None and out.shape != shape:
        raise ValueError(f"linear: out {tuple(out.shape)} is not {tuple(shape)}")
    act = _activation("linear", activation)
    dtype = _dtype("linear", x, weight, bias, residual, out)
    _inner("linear", x=x, weight=weight, bias=bias, residual=residual, out=out)
    _no_grad("linear", x, weight, bias, residual, out)
    device = _device("linear", x, weight, bias, residual, out)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    else:
        _apart("linear", "out", out, x=x, weight=weight, bias=bias)
        _same_or_apart("linear", out, residual=residual)
    if out.numel() == 0:
        return out
    xr, rr, yr = _rows(x) if k else x.new_empty((out.numel() // n, 0)), residual if residual is None else _rows(residual), _rows(out)
    if xr is None or yr is None or (rr is None and residual is not None):
        raise ValueError("linear: the leading dimensions of a tensor are not rows at one distance")
    m = yr.shape[0]
    _call(_lib.load().vadc_amd_linear, _LINEAR.pack(
        xr.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(rr), yr.data_ptr(), m, k, n, xr.stride(0), weight.stride(0), 0 if rr is None else rr.stride(0), yr.stride(0),
        dtype, act, bool(residual_first), device), device)
    return out


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5, activation: str = "none",
               gate: Optional[Tensor] = None, lengths: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """Group norm with channels last: per sequence and group, y = (x - mean) / sqrt(var + eps) weight + bias; returns act(y), or y act(gate) if a gate is given.

    x [sequences, positions, channels], or [tokens, channels] (each token a sequence of one position); gate like x; weight, bias [channels].  lengths [sequences] (int32): sequence n
    has its first lengths[n] positions only; what lies behind them is not read, and stays as it is in `out` (zero, where no `out` is given).  `out` may be x or gate."""
    if x.dim() not in (2, 3):
        raise ValueError(f"group_norm: x {tuple(x.shape)} is neither [sequences, positions, channels] nor [tokens, channels]")
    n, l, c = x.shape if x.dim() == 3 else (x.shape[0], 1, x.shape[1])
    if groups < 1 or c % groups:
        raise ValueError(f"group_norm: {c} channels do not divide into {groups} groups")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"group_norm: eps {eps} must be finite and not negative")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (c,):
            raise ValueError(f"group_norm: {name} {tuple(t.shape)} is not [{c}]")
    for name, t in (("gate", gate), ("out", out)):
        if t is not None and t.shape != x.shape:
            raise ValueError(f"group_norm: {name} {tuple(t.shape)} is not {tuple(x.shape)}")
    _lengths("group_norm", lengths, n)
    act = _activation("group_norm", activation)
    dtype = _dtype("group_norm", x, weight, bias, gate, out)
    _inner("group_norm", x=x, weight=weight, bias=bias, gate=gate, out=out)
    _no_grad("group_norm", x, weight, bias, gate, out)
    device = _device("group_norm", x, weight, bias, gate, lengths, out)
    if out is None:
        out = (torch.empty if lengths is None else torch.zeros)(x.shape, dtype=x.dtype, device=x.device)
    else:
        _apart("group_norm", "out", out, weight=weight, bias=bias, lengths=lengths)
        _same_or_apart("group_norm", out, x=x, gate=gate)
    if out.numel() == 0:
        return out

    def strides(t):
        return (0, 0) if t is None else (t.stride(0), t.stride(1)) if t.dim() == 3 else (t.stride(0), 0)

    L = _lib.load()
    sizes = (n, l, c, groups, *strides(x), *strides(gate), *strides(out), dtype, act, device, eps)
    pointers = (x.data_ptr(), _ptr(weight), _ptr(bias), _ptr(gate), out.data_ptr(), _ptr(lengths))
    space, need = None, 0
    if l > 1:                                        # a single position never needs any
        need = _bytes(L.vadc_amd_group_norm_workspace, _NORM.pack(*pointers, 0, 0, *sizes))
        space = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call(L.vadc_amd_group_norm, _NORM.pack(*pointers, _ptr(space), need, *sizes), device)
    return out


def gated_delta(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, state: Tensor, scale: Optional[float] = None, normalize: bool = False,
                lengths: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """The gated delta rule.  Per stream and head, for each step: S = e^log_decay S; u = beta (v - S^T k); S = S + k u^T; out = scale S^T q.

    q, k [streams, steps, key_heads, key_dim], v [streams, steps, heads, value_dim], log_decay, beta [streams, steps, heads] (float32), state [streams, heads, key_dim, value_dim]
    (float32), which is UPDATED in place; returns [streams, steps, heads, value_dim].  heads is a multiple of key_heads (consecutive heads share a key head); key_dim is 256 at most.
    scale: 1 / sqrt(key_dim) by default.  normalize: q and k are brought to unit length (x / sqrt(sum x^2 + 1e-6)).  lengths [streams] (int32): stream b has its first lengths[b] steps
    only; what lies behind them is not read, and stays as it is in `out` (zero, where no `out` is given); a stream of no steps keeps its state."""
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"gated_delta: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    b, t, hk, dk = q.shape
    h, dv = v.shape[2:]
    if hk < 1 or h % hk:
        raise ValueError(f"gated_delta: {h} heads are no multiple of {hk} key heads")
    if not 1 <= dk <= 256:
        raise ValueError(f"gated_delta: key_dim {dk} is not in 1 ... 256")
    if log_decay.shape != (b, t, h) or beta.shape != (b, t, h):
        raise ValueError(f"gated_delta: log_decay {tuple(log_decay.shape)} and beta {tuple(beta.shape)} must be [{b}, {t}, {h}]")
    if state.shape != (b, h, dk, dv):
        raise ValueError(f"gated_delta: state {tuple(state.shape)} is not [{b}, {h}, {dk}, {dv}]")
    if out is not None and out.shape != v.shape:
        raise ValueError(f"gated_delta: out {tuple(out.shape)} is not {tuple(v.shape)}")
    _lengths("gated_delta", lengths, b)
    dtype = _dtype("gated_delta", q, k, v, out)
    _floats("gated_delta", "log_decay", log_decay)
    _floats("gated_delta", "beta", beta)
    _floats("gated_delta", "state", state)
    _inner("gated_delta", q=q, k=k, v=v, log_decay=log_decay, beta=beta, out=out)
    if not state.is_contiguous() and not state[0].is_contiguous():
        raise ValueError("gated_delta: each stream's part of state must be contiguous")
    if scale is None:
        scale = dk ** -0.5
    _no_grad("gated_delta", q, k, v, log_decay, beta, state, out)
    device = _device("gated_delta", q, k, v, log_decay, beta, state, lengths, out)
    if out is None:
        out = (torch.empty if lengths is None else torch.zeros)(v.shape, dtype=v.dtype, device=v.device)
    else:
        _apart("gated_delta", "out", out, q=q, k=k, v=v, log_decay=log_decay, beta=beta, state=state, lengths=lengths)
    if out.numel() == 0:
        return out
    L = _lib.load()
    sizes = (b, t, hk, h, dk, dv, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *log_decay.stride()[:2], *beta.stride()[:2], state.stride(0),
             scale, bool(normalize), dtype, device)
    pointers = (q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(), out.data_ptr(), _ptr(lengths))
    space, need = None, 0
    if t > 1:                                        # a single step never needs any
        need = _bytes(L.vadc_amd_gated_delta_workspace, _DELTA.pack(*pointers, 0, 0, *sizes))
        space = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call(L.vadc_amd_gated_delta, _DELTA.pack(*pointers, _ptr(space), need, *sizes), device)
    return out
