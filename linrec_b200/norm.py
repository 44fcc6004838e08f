"""Group norm of channels-last tensors with an activation or an activated gate: what stands behind the gated
recurrence in a layer with heads (`linrec_gated_norm`), where every position is a sample of its own and the
heads are the groups, and the usual group norm of (samples, positions, channels) tensors.

    y = group_norm_act(x, groups, weight, bias)                # act(norm(x) * weight + bias)
    y = group_norm_act(x, groups, weight, bias, gate=g)        # (norm(x) * weight + bias) * act(g)

Storage types float32, bfloat16 and float16; statistics, parameters and their gradients are float32.

Derivatives are backward ones.  Forward-mode derivatives, torch.func transforms, recording by torch.jit.trace or make_fx
and fake tensors are refused; torch.compile runs the calls between its graphs.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _capi
from .ops import _DTYPES, _row_layout

__all__ = ["group_norm_act"]

_STORAGE = (torch.float32, torch.bfloat16, torch.float16)
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_TINIEST, _HUGEST = 2.0 ** -150, 2.0 ** 128 - 2.0 ** 103      # what lies between them is neither zero nor infinite in float32
_ACTIVATIONS = {None: 0, "silu": 1, "sigmoid": 2}
# (looked up once: they are asked for at every call, and a small call is host work)
_Tensor = torch.Tensor
_functorch_stack = torch._C._functorch.peek_interpreter_stack
_functorch_wrapped = torch._C._functorch.is_functorch_wrapped_tensor
_jit_tracing = torch._C._is_tracing
_dispatch_modes = torch._C._len_torch_dispatch_stack
_dispatch_mode = torch._C._get_dispatch_mode
_no_dispatch = torch._C._disabled_torch_dispatch_impl
_RECORDERS = (torch._C._TorchDispatchModeKey.PROXY, torch._C._TorchDispatchModeKey.FAKE)


def _fail(what: str):
    raise RuntimeError(f"linrec: {what}")


def _refuse_transforms(ts) -> None:
    for t in ts:
        if t is None:
            continue
        if _functorch_wrapped(t):
            _fail("torch.func transforms are not supported")
        if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
            _fail("forward-mode derivatives are not supported")
    if _jit_tracing() or any(_dispatch_mode(k) is not None for k in _RECORDERS):
        _fail("calls cannot be recorded by a tracer (torch.compile runs them between its graphs)")


def _check_memory(t) -> None:
    if type(t).__torch_dispatch__ is not _no_dispatch:
        _fail(f"{type(t).__name__} is not a tensor with memory of its own")


def _check_tensors(first, *others) -> None:
    """Tensors that the C library can take: real ones, all on one GPU.  It computes out of sight of PyTorch's
    transforms and tracers, and what those would make of the calls around it is a wrong answer."""
    if _forward_ad._current_level >= 0 or _dispatch_modes() or _jit_tracing() or _functorch_stack() is not None:
        _refuse_transforms((first, *others))
    if type(first) is not _Tensor:
        _check_memory(first)
    if not first.is_cuda:
        _fail("tensors must be CUDA tensors (there is no CPU implementation)")
    device = first.device
    for t in others:
        if t is not None:
            if type(t) is not _Tensor:
                _check_memory(t)
            if t.device != device:
                _fail("tensors must be CUDA tensors (there is no CPU implementation)" if not t.is_cuda else
                      "tensors must be on the same device")


def _as_rows(t: torch.Tensor):
    """(`t` or a dense copy, elements between consecutive rows): the kernels take rows at one stride."""
    if t.is_contiguous():
        return t, t.size(-1)
    layout = _row_layout(t) if t.numel() and (t.size(-1) == 1 or t.stride(-1) == 1) else None
    if layout is None:
        t = t.contiguous()
        return t, t.size(-1)
    return t, layout[2]


def _as_float(t):
    """A parameter or state as dense float32 (the cast is autograd's to undo)."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.float().contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*ts) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _empty_dense(t: torch.Tensor) -> torch.Tensor:
    """A dense tensor of the sizes and type of `t`."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _backward_once(raw):
    """`once_differentiable(raw)` without its bookkeeping where no gradient of the gradient was asked for."""
    refusing = once_differentiable(raw)

    def backward(ctx, *grads):
        return (refusing if torch.is_grad_enabled() else raw)(ctx, *grads)

    return staticmethod(backward)


def _on(device: torch.device, launch) -> None:
    """`launch(stream)` with `device` current."""
    if _current_device() == device.index:
        launch(_raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            launch(_raw_stream(device.index))


@functools.lru_cache(maxsize=4096)
def _scratch_size(dtype, nsamples, positions, C, groups, bwd, params) -> int:
    a = _capi.GroupNormArgs(dtype=dtype, nsamples=nsamples, positions=positions, nchan=C, groups=groups, eps=1.0)
    a.dweight = 16 if params else None
    return _capi.lib.linrec_b200_group_norm_scratch_size(ctypes.byref(a), bwd)


def _call(bwd, x, gate, weight, bias, groups, act, eps, stats, y=None, dy=None, dx=None, dgate=None, dw=None, db=None) -> None:
    N, C = x.size(0), x.size(-1)
    L = x.numel() // (N * C)
    dtype = _DTYPES[x.dtype]
    x, sx = _as_rows(x)
    gate, sg = (None, 0) if gate is None else _as_rows(gate)
    dy, sdy = (None, 0) if dy is None else _as_rows(dy)
    need = _scratch_size(dtype, N, L, C, groups, bwd, dw is not None or db is not None)
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    # (the field order of linrec_group_norm_args)
    a = _capi.GroupNormArgs(x.data_ptr(), _ptr(gate), sx, sg, _ptr(weight), _ptr(bias), eps, act, dtype, N, L, C, groups, _ptr(stats), _ptr(y),
                            _ptr(dy), sdy, _ptr(dx), _ptr(dgate), _ptr(dw), _ptr(db), _ptr(scratch), need)
    entry, name = ((_capi.lib.linrec_b200_group_norm_bwd, "linrec_b200_group_norm_bwd") if bwd else
                   (_capi.lib.linrec_b200_group_norm_fwd, "linrec_b200_group_norm_fwd"))
    _on(x.device, lambda stream: _capi.raise_for(entry(ctypes.byref(a), stream), name))


def _forward(x, gate, weight, bias, groups, act, eps, want_stats):
    y = _empty_dense(x)
    stats = torch.empty(x.size(0) * groups * 2, dtype=torch.float32, device=x.device) if want_stats else None
    if y.numel():
        _call(False, x, gate, weight, bias, groups, act, eps, stats, y=y)
    return y, stats


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, weight, bias, groups, act, eps):
        y, stats = _forward(x, gate, weight, bias, groups, act, eps, True)
        ctx.save_for_backward(x, gate, weight, bias, stats)
        ctx.args = (groups, act, eps)
        return y

    @_backward_once
    def backward(ctx, dy):
        x, gate, weight, bias, stats = ctx.saved_tensors
        dx = _empty_dense(x)
        dgate = None if gate is None else _empty_dense(x)
        make = torch.empty_like if x.numel() else torch.zeros_like
        dw = make(weight) if weight is not None and ctx.needs_input_grad[2] else None
        db = make(bias) if bias is not None and ctx.needs_input_grad[3] else None
        if x.numel():
            _call(True, x, gate, weight, bias, *ctx.args, stats, dy=dy, dx=dx, dgate=dgate, dw=dw, db=db)
        return dx, dgate, dw, db, None, None, None


def _check(x, groups, weight, bias, gate, activation, eps) -> None:
    shape = x.shape
    if len(shape) < 2:
        _fail("x needs a sample and a channel dimension")
    if x.dtype not in _STORAGE:
        _fail(f"dtype {x.dtype} is not supported (float32, bfloat16, float16)")
    if isinstance(groups, bool) or not isinstance(groups, int) or groups < 1 or shape[-1] % groups:
        _fail("groups must divide the channels")
    if activation not in _ACTIVATIONS:
        _fail(f"activation {activation!r} is not one of {list(_ACTIVATIONS)}")
    if not _TINIEST < float(eps) < _HUGEST:
        _fail("eps must be positive and finite in float32")
    channels = shape[-1:]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != channels or not t.is_floating_point()):
            _fail(f"{name} must have one floating-point value per channel")
    if gate is not None and (gate.shape != shape or gate.dtype != x.dtype):
        _fail("gate must have the sizes and the dtype of x")
    _check_tensors(x, gate, weight, bias)


def _apply(x, groups, weight, bias, gate, activation, eps) -> torch.Tensor:
    weight, bias = _as_float(weight), _as_float(bias)
    args = (x, gate, weight, bias, groups, _ACTIVATIONS[activation], float(eps))
    if _wants_grad(x, gate, weight, bias):
        return _GroupNormFn.apply(*args)
    return _forward(*args, False)[0]


def group_norm_act(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                   gate: torch.Tensor | None = None, activation: str | None = "silu", eps: float = 1e-5) -> torch.Tensor:
    """Group norm of `x`, (samples, ..., channels): mean and (biased) variance over the dimensions between and
    the channels of a group, `groups` groups of adjacent channels; then weight and bias per channel; then
    the activation of the result, or the product with the activated gate where one is given.

    For statistics of every position by itself give x as (positions, channels).
    activation   "silu", "sigmoid" or None
    weight, bias (channels,), ones and zeros by default; gate has the sizes and dtype of x

    Differentiable once with respect to x, gate, weight and bias."""
    _check(x, groups, weight, bias, gate, activation, eps)
    return _apply(x, groups, weight, bias, gate, activation, eps)
