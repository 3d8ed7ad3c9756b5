"""Operators on device tensors: what a streaming layer of one's own is made of, to run beside the models of vadc_amd.engine on the same GPU.

    linear       act(x W^T + b) + r                       matrix product with bias, activation and residual
    gated_delta  the gated delta rule                      a recurrence with one state per stream and head: many steps per call, or one
    group_norm   group norm with an activation or a gate   channels last; positions of a sequence together, or each token alone

Tensors are torch tensors on one gfx950 device, of one type (float32, float16 or bfloat16); the work is enqueued on torch's current stream of that device and may be captured into a
graph.  Sums, statistics and states are float32, an output is rounded once.  Strided tensors are taken as they are, as long as the innermost dimension is contiguous.  The operators
have no gradients: tensors that ask for them are refused while autograd records, as are tensors with a forward-mode tangent.  What a call writes in place (`out`, `state`) counts as changed for autograd, as by torch's own in-place
operations: a graph that saved it raises in its backward.  All arithmetic happens in libvadc_amd.so (include/vadc_amd.h: vadc_amd_linear, ...); a wrong
argument raises ValueError or TypeError before the device is touched, a failure of the library VadcAmdError.
"""
from __future__ import annotations

import functools
import numbers
import struct
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

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


# A call's checks go by its tensors' layouts (shape, strides, type, device) alone, so each set of layouts is checked once and what the checks found is kept: the fields behind the
# pointers, the workspace's size, the bytes that each tensor spans.  A step of one stream is a matter of microseconds, and checking it is half of them.
class _Plan(NamedTuple):
    fields: tuple            # of the struct, behind its pointers (and its workspace)
    shape: tuple             # of the output
    device: int
    spans: tuple             # bytes from each tensor's first to its last element, in the order of the layouts; the output's is last
    workspace: int
    empty: bool              # nothing to do


_KEPT = 1024                 # plans, the least recently used go first; by the arguments' types as well: 2.0 equals 2, but is refused as a number of groups, whatever ran before


class _Layout(NamedTuple):
    shape: torch.Size
    stride: tuple
    dtype: torch.dtype
    device: torch.device


def _layout(t: Optional[Tensor]):
    try:
        return None if t is None else (t.shape, t.stride(), t.dtype, t.device)
    except (AttributeError, RuntimeError):           # an array, a list; a tensor without strides
        raise TypeError(f"the operators take strided torch tensors, not {type(t).__name__}") from None


def _layouts(*ls):
    return [None if v is None else _Layout(*v) for v in ls]


_EINVAL = -1                 # of include/vadc_amd.h


def _check(rc: int) -> int:
    if rc < 0:
        said = _lib.load().vadc_amd_last_error().decode()
        raise ValueError(said) if rc == _EINVAL else VadcAmdError(rc, said)
    return rc


def _no_grad(what: str, *ts: Optional[Tensor]):
    for t in ts:
        if t is not None and t.requires_grad:
            raise ValueError(f"{what} has no gradient: call it under torch.no_grad() or with tensors that ask for none")


def _no_tangent(what: str, *ts: Optional[Tensor]):
    """inside a dual level of forward mode, which torch.no_grad() leaves on"""
    for t in ts:
        if t is not None and torch._C._is_fwd_grad_enabled() and (torch._C._functorch.is_functorch_wrapped_tensor(t) or forward_ad.unpack_dual(t).tangent is not None):
            raise ValueError(f"{what} has no forward-mode derivative: call it with tensors that carry no tangent")


def _same_device(what: str, *ls: Optional[_Layout]) -> int:
    d = ls[0].device
    for v in ls:
        if v is not None and v.device != d:
            raise ValueError(f"{what}: tensors on {d} and on {v.device}")
    if d.type != "cuda":
        raise ValueError(f"{what}: tensors must be on a gfx950 device, not on {d} (vadc_amd has no CPU fallback)")
    return d.index


_LARGEST = 3.4e38            # of float32, short of its last digits


def _given(what: str, **ls: Optional[_Layout]):
    for name, v in ls.items():
        if v is None:
            raise TypeError(f"{what}: {name} must be a tensor, not None")


def _flag(what: str, **flags):
    for name, v in flags.items():
        if not isinstance(v, (bool, int)):           # a tensor's truth would be read once and kept
            raise TypeError(f"{what}: {name} must be True or False, not {v!r}")


def _activation(what: str, name: str) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"{what}: activation {name!r} is none of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def _same_dtype(what: str, *ls: Optional[_Layout]) -> int:
    dt = ls[0].dtype
    if dt not in _DTYPES:
        raise TypeError(f"{what}: {dt} is none of float32, float16, bfloat16")
    for v in ls:
        if v is not None and v.dtype != dt:
            raise TypeError(f"{what}: tensors of {dt} and of {v.dtype}")
    return _DTYPES[dt]


def _float32(what: str, **ls: _Layout):
    for name, v in ls.items():
        if v.dtype != torch.float32:
            raise TypeError(f"{what}: {name} must be float32, not {v.dtype}")


def _shaped(what: str, shape: tuple, **ls: Optional[_Layout]):
    for name, v in ls.items():
        if v is not None and tuple(v.shape) != tuple(shape):
            raise ValueError(f"{what}: {name} {tuple(v.shape)} is not {list(shape)}")


def _inner(what: str, **ls: Optional[_Layout]):
    for name, v in ls.items():
        if v is not None and v.shape[-1] > 1 and v.stride[-1] != 1:
            raise ValueError(f"{what}: the last dimension of {name} must be contiguous")


def _distinct(what: str, v: Optional[_Layout]):
    """no two entries of an output at one place: taken by falling stride, each dimension steps over all that the smaller ones span"""
    if v is not None and 0 not in v.shape:
        reach = 1
        for stride, n in sorted(zip(v.stride, v.shape)):
            if n > 1:
                if stride < reach:
                    raise ValueError(f"{what}: entries of out lie on top of each other (strides {v.stride})")
                reach = stride * (n - 1) + reach


def _lengths(what: str, v: Optional[_Layout], n: int):
    if v is not None:
        if v.dtype != torch.int32:
            raise TypeError(f"{what}: lengths must be int32, not {v.dtype}")
        if tuple(v.shape) != (n,) or (n > 1 and v.stride[0] != 1):
            raise ValueError(f"{what}: lengths must be a contiguous tensor of {n}")


def _span(v: Optional[_Layout]) -> int:
    if v is None or 0 in v.shape:
        return 0
    return (sum((n - 1) * s for n, s in zip(v.shape, v.stride)) + 1) * v.dtype.itemsize


def _pieces(shape: tuple, stride: tuple, size: int):
    """the bytes of a tensor: runs of equal length, and the (distance, count) of their repetitions, the furthest apart first"""
    run, repeats = size, []
    for distance, n in sorted((s * size, n) for s, n in zip(stride, shape) if n > 1 and s):
        if not repeats and distance <= run:
            run += distance * (n - 1)
        else:
            repeats.append((distance, n))
    return run, repeats[::-1]


_FEW = 8                     # repetitions looked at one by one


def _meet(by: int, run_a: int, a: list, run_b: int, b: list) -> bool:
    """whether two tensors' _pieces share a byte, the second's first one `by` behind the first's.  Repetitions at one distance are taken together; where too many would have to be looked
    at one by one, the answer is yes."""
    reach_a, reach_b = (run + sum(s * (n - 1) for s, n in t) for run, t in ((run_a, a), (run_b, b)))
    if by >= reach_a or by + reach_b <= 0:
        return False
    if not a and not b:
        return True
    s = max(t[0][0] for t in (a, b) if t)
    n_a, n_b = (t[0][1] if t and t[0][0] == s else 1 for t in (a, b))
    a, b = (t[1:] if t and t[0][0] == s else t for t in (a, b))
    reach_a, reach_b = reach_a - s * (n_a - 1), reach_b - s * (n_b - 1)
    near = range(max(1 - n_a, (-reach_b - by) // s + 1), min(n_b - 1, (reach_a - 1 - by) // s) + 1)      # differences between the repetitions whose spans meet
    return len(near) > _FEW or any(_meet(by + j * s, run_a, a, run_b, b) for j in near)


def _shares(x: Tensor, y: Tensor) -> bool:
    return _meet(y.data_ptr() - x.data_ptr(), *_pieces(x.shape, x.stride(), x.element_size()), *_pieces(y.shape, y.stride(), y.element_size()))


def _apart(what: str, spans: tuple, out: Tensor, ts: tuple, same: tuple = (), written: str = "out"):
    """out (or what is `written` else) overlaps none of `ts` (named, in the order of the plan's spans; out's is last); those in `same` may be out itself, entry for entry.  Spans that meet are
    looked at closely: rows may hold both."""
    lo = out.data_ptr()
    hi = lo + spans[-1]
    for (name, t), span in zip(ts, spans):
        if t is not None:
            at = t.data_ptr()
            if at < hi and lo < at + span and not (name in same and at == lo and t.stride() == out.stride()) and _shares(out, t):
                raise ValueError(f"{what}: {written} overlaps {name}")


def _rows(what: str, name: str, v: Optional[_Layout]):
    """a tensor [..., n] as rows at one distance: that distance"""
    if v is None:
        return 0
    distance = count = None
    for n, stride in zip(reversed(v.shape[:-1]), reversed(v.stride[:-1])):
        if n == 1:
            continue
        if distance is None:
            distance, count = stride, n
        elif stride == distance * count:
            count *= n
        else:
            raise ValueError(f"{what}: the leading dimensions of {name} are not rows at one distance (strides {v.stride})")
    return v.shape[-1] if distance is None else distance


@functools.lru_cache(_KEPT, typed=True)
def _plan_linear(x, weight, bias, residual, out, activation, residual_first) -> _Plan:
    x, weight, bias, residual, out = _layouts(x, weight, bias, residual, out)
    _given("linear", x=x, weight=weight)
    if len(weight.shape) != 2 or len(x.shape) < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    n, k = weight.shape
    shape = tuple(x.shape[:-1]) + (n,)
    _shaped("linear", (n,), bias=bias)
    _shaped("linear", shape, residual=residual, out=out)
    act = _activation("linear", activation)
    _flag("linear", residual_first=residual_first)
    dtype = _same_dtype("linear", x, weight, bias, residual, out)
    _inner("linear", x=x, weight=weight, bias=bias, residual=residual, out=out)
    _distinct("linear", out)
    m = 1
    for d in shape[:-1]:
        m *= d
    empty = m == 0 or n == 0
    strides = (0, 0, 0, 0) if empty else (_rows("linear", "x", x) if k else 0, weight.stride[0], _rows("linear", "residual", residual), _rows("linear", "out", out) if out else n)
    device = _same_device("linear", x, weight, bias, residual, out)
    return _Plan((m, k, n, *strides, dtype, act, bool(residual_first), device), shape, device, tuple(map(_span, (x, weight, bias, residual, out))), 0, empty)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "none", residual: Optional[Tensor] = None,
           residual_first: bool = False, out: Optional[Tensor] = None) -> Tensor:
    """act(x W^T + bias) + residual, or with residual_first act(x W^T + bias + residual).

    x [..., in], weight [out, in], bias [out], residual [..., out]; returns [..., out] (in `out`, if given, which may be the residual).  Leading dimensions must make up rows at one
    distance.  activation: none, relu, silu, gelu (with erf), sigmoid."""
    plan = _plan_linear(_layout(x), _layout(weight), _layout(bias), _layout(residual), _layout(out), activation, residual_first)
    if torch.is_grad_enabled():
        _no_grad("linear", x, weight, bias, residual, out)
    if forward_ad._current_level >= 0:
        _no_tangent("linear", x, weight, bias, residual, out)
    fresh = out is None
    if fresh:
        out = x.new_empty(plan.shape)
    else:
        _apart("linear", plan.spans, out, (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)), ("residual",))
    if not plan.empty:
        _check(_lib.load().vadc_amd_linear(_LINEAR.pack(
            x.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if residual is None else residual.data_ptr(), out.data_ptr(), *plan.fields),
            torch._C._cuda_getCurrentRawStream(plan.device)))
        if not fresh:
            increment_version(out)
    return out


@functools.lru_cache(_KEPT, typed=True)
def _plan_norm(x, groups, weight, bias, eps, activation, gate, lengths, out) -> _Plan:
    x, weight, bias, gate, lengths, out = _layouts(x, weight, bias, gate, lengths, out)
    _given("group_norm", x=x)
    if len(x.shape) not in (2, 3):
        raise ValueError(f"group_norm: x {tuple(x.shape)} is neither [sequences, positions, channels] nor [tokens, channels]")
    n, l, c = x.shape if len(x.shape) == 3 else (x.shape[0], 1, x.shape[1])
    if not isinstance(groups, numbers.Integral) or not isinstance(eps, numbers.Real):
        raise TypeError(f"group_norm: groups must be a whole number, eps a number, not {groups!r}, {eps!r}")
    if groups < 1 or c % groups:
        raise ValueError(f"group_norm: {c} channels do not divide into {groups} groups")
    if not 0 <= eps <= _LARGEST:
        raise ValueError(f"group_norm: eps {eps} must be finite and not negative")
    _shaped("group_norm", (c,), weight=weight, bias=bias)
    _shaped("group_norm", x.shape, gate=gate, out=out)
    _lengths("group_norm", lengths, n)
    act = _activation("group_norm", activation)
    dtype = _same_dtype("group_norm", x, weight, bias, gate, out)
    _inner("group_norm", x=x, weight=weight, bias=bias, gate=gate, out=out)
    _distinct("group_norm", out)
    device = _same_device("group_norm", x, weight, bias, gate, lengths, out)
    empty = 0 in x.shape

    def strides(v):
        return (0, 0) if v is None else (v.stride[0], v.stride[1]) if len(v.shape) == 3 else (v.stride[0], c)

    fields = (n, l, c, groups, *strides(x), *strides(gate), *(strides(out) if out else (l * c, c)), dtype, act, device, eps)
    space = 0 if empty else _check(_lib.load().vadc_amd_group_norm_workspace(_NORM.pack(*(0,) * 8, *fields)))
    return _Plan(fields, tuple(x.shape), device, tuple(map(_span, (x, weight, bias, gate, lengths, out))), space, empty)


def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5, activation: str = "none",
               gate: Optional[Tensor] = None, lengths: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """Group norm with channels last: per sequence and group, y = (x - mean) / sqrt(var + eps) weight + bias; returns act(y), or y act(gate) if a gate is given.

    x [sequences, positions, channels], or [tokens, channels] (each token a sequence of one position); gate like x; weight, bias [channels].  lengths [sequences] (int32): sequence n
    has its first lengths[n] positions only; what lies behind them is not read, and stays as it is in `out` (zero, where no `out` is given).  `out` may be x or gate."""
    plan = _plan_norm(_layout(x), groups, _layout(weight), _layout(bias), eps, activation, _layout(gate), _layout(lengths), _layout(out))
    if torch.is_grad_enabled():
        _no_grad("group_norm", x, weight, bias, gate, out)
    if forward_ad._current_level >= 0:
        _no_tangent("group_norm", x, weight, bias, gate, out)
    fresh = out is None
    if fresh:
        out = x.new_empty(plan.shape) if lengths is None else x.new_zeros(plan.shape)
    else:
        _apart("group_norm", plan.spans, out, (("x", x), ("weight", weight), ("bias", bias), ("gate", gate), ("lengths", lengths)), ("x", "gate"))
    if not plan.empty:
        space = torch.empty(plan.workspace, dtype=torch.uint8, device=x.device) if plan.workspace else None
        _check(_lib.load().vadc_amd_group_norm(_NORM.pack(
            x.data_ptr(), 0 if weight is None else weight.data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if gate is None else gate.data_ptr(), out.data_ptr(),
            0 if lengths is None else lengths.data_ptr(), 0 if space is None else space.data_ptr(), plan.workspace, *plan.fields),
            torch._C._cuda_getCurrentRawStream(plan.device)))
        if not fresh:
            increment_version(out)
    return out


@functools.lru_cache(_KEPT, typed=True)
def _plan_delta(q, k, v, log_decay, beta, state, scale, normalize, lengths, out) -> _Plan:
    q, k, v, log_decay, beta, state, lengths, out = _layouts(q, k, v, log_decay, beta, state, lengths, out)
    _given("gated_delta", q=q, k=k, v=v, log_decay=log_decay, beta=beta, state=state)
    if len(q.shape) != 4 or k.shape != q.shape or len(v.shape) != 4 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"gated_delta: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    b, t, hk, dk = q.shape
    h, dv = v.shape[2:]
    if hk < 1 or h % hk:
        raise ValueError(f"gated_delta: {h} heads are no multiple of {hk} key heads")
    if not 1 <= dk <= 256:
        raise ValueError(f"gated_delta: key_dim {dk} is not in 1 ... 256")
    _shaped("gated_delta", (b, t, h), log_decay=log_decay, beta=beta)
    _shaped("gated_delta", (b, h, dk, dv), state=state)
    _shaped("gated_delta", v.shape, out=out)
    _lengths("gated_delta", lengths, b)
    dtype = _same_dtype("gated_delta", q, k, v, out)
    _float32("gated_delta", log_decay=log_decay, beta=beta, state=state)
    _inner("gated_delta", q=q, k=k, v=v, log_decay=log_decay, beta=beta, out=out)
    _distinct("gated_delta", out)
    part = dk * dv
    if 0 not in state.shape and any(n > 1 and have != want for n, have, want in zip(state.shape[1:], state.stride[1:], (part, dv, 1))):
        raise ValueError("gated_delta: each stream's part of state must be contiguous")
    _flag("gated_delta", normalize=normalize)
    if scale is not None and not isinstance(scale, numbers.Real):
        raise TypeError(f"gated_delta: scale must be a number, not {scale!r}")
    scale = dk ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _LARGEST:
        raise ValueError(f"gated_delta: scale {scale} must be finite")
    device = _same_device("gated_delta", q, k, v, log_decay, beta, state, lengths, out)
    empty = 0 in v.shape
    fields = (b, t, hk, h, dk, dv, *q.stride[:3], *k.stride[:3], *v.stride[:3], *(out.stride[:3] if out else (t * h * dv, h * dv, dv)), *log_decay.stride[:2], *beta.stride[:2],
              state.stride[0] if b > 1 else h * part, scale, bool(normalize), dtype, device)
    space = 0 if empty else _check(_lib.load().vadc_amd_gated_delta_workspace(_DELTA.pack(*(0,) * 10, *fields)))
    return _Plan(fields, tuple(v.shape), device, tuple(map(_span, (q, k, v, log_decay, beta, state, lengths, out))), space, empty)


def _state_apart(spans: tuple, q, k, v, log_decay, beta, state, lengths):
    """state, which is written, overlaps no input"""
    _apart("gated_delta", (*spans[:5], spans[6], spans[5]), state, (("q", q), ("k", k), ("v", v), ("log_decay", log_decay), ("beta", beta), ("lengths", lengths)), written="state")


def gated_delta(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, state: Tensor, scale: Optional[float] = None, normalize: bool = False,
                lengths: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """The gated delta rule.  Per stream and head, for each step: S = e^log_decay S; u = beta (v - S^T k); S = S + k u^T; out = scale S^T q.

    q, k [streams, steps, key_heads, key_dim], v [streams, steps, heads, value_dim], log_decay, beta [streams, steps, heads] (float32), state [streams, heads, key_dim, value_dim]
    (float32), which is UPDATED in place and overlaps no input; returns [streams, steps, heads, value_dim].  heads is a multiple of key_heads (consecutive heads share a key head); key_dim is 256 at most.
    scale: 1 / sqrt(key_dim) by default.  normalize: q and k are brought to unit length (x / sqrt(sum x^2 + 1e-6)).  lengths [streams] (int32): stream b has its first lengths[b] steps
    only; what lies behind them is not read, and stays as it is in `out` (zero, where no `out` is given); a stream of no steps keeps its state.  Many steps go in blocks where key_dim is 8 to
    128, one by one with longer keys.  A value that is not finite, an infinity as well, makes NaN of what it reaches: its column of the state and of the outputs from its step on (a key or gate: every column of its head; a query: its own outputs)."""
    plan = _plan_delta(_layout(q), _layout(k), _layout(v), _layout(log_decay), _layout(beta), _layout(state), scale, normalize, _layout(lengths), _layout(out))
    if torch.is_grad_enabled():
        _no_grad("gated_delta", q, k, v, log_decay, beta, state, out)
    if forward_ad._current_level >= 0:
        _no_tangent("gated_delta", q, k, v, log_decay, beta, state, out)
    fresh = out is None
    if fresh:
        out = v.new_empty(plan.shape) if lengths is None else v.new_zeros(plan.shape)
    else:
        _apart("gated_delta", plan.spans, out, (("q", q), ("k", k), ("v", v), ("log_decay", log_decay), ("beta", beta), ("state", state), ("lengths", lengths)))
    if not plan.empty:
        at_q, at_k, at_v, at_g, at_b, lo, at_n = q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(), 0 if lengths is None else lengths.data_ptr()
        n_q, n_k, n_v, n_g, n_b, n_s, n_n, _ = plan.spans
        hi = lo + n_s
        if (at_q < hi and lo < at_q + n_q or at_k < hi and lo < at_k + n_k or at_v < hi and lo < at_v + n_v or at_g < hi and lo < at_g + n_g or at_b < hi and lo < at_b + n_b
                or at_n < hi and lo < at_n + n_n):   # in line: 0.3 us of a step's 8
            _state_apart(plan.spans, q, k, v, log_decay, beta, state, lengths)
        space = torch.empty(plan.workspace, dtype=torch.uint8, device=v.device) if plan.workspace else None
        _check(_lib.load().vadc_amd_gated_delta(_DELTA.pack(at_q, at_k, at_v, at_g, at_b, lo, out.data_ptr(), at_n, 0 if space is None else space.data_ptr(), plan.workspace, *plan.fields),
                                                torch._C._cuda_getCurrentRawStream(plan.device)))
        increment_version((state,) if fresh else (state, out))
    return out
