"""Gated linear recurrence on channels-last tensors: the recurrence of `linrec` with its multiplier and
input factor computed from gate logits inside the kernels, over batches or packed sequences, with states
carried in and out in float32, a backward pass, and a form for single tokens on a state cache.

    y = linrec_gated(inputs, forget)                                     # a = s(f), h = a h + (1 - a) x
    y = linrec_gated(inputs, forget, input_gate=i, decay=L)              # log a = -k softplus(L) s(f),
                                                                         # h = a h + sqrt(1 - a^2) s(i) x
    y, state = linrec_gated(..., initial_state=h0, return_state=True)
    y = linrec_gated(inputs, forget, cu_seqlens=offsets)                 # (rows, D), sequences end to end
    y = linrec_gated_step(inputs, forget, state, slots=slots)            # one token each, state in place

    y = linrec_gated_norm(inputs, forget, gate, groups, weight, bias)    # recurrence, norm per head, gate

(s is the logistic function.)  `linrec_general(x, c, dim=1)` scans the same layout with finished
coefficients in the storage type; rounded to 16 bits a multiplier near one is off by more than its distance
from one, and it takes no states and no packed sequences, which is what these operators are for.  The
reference's operators take finished coefficients too (linrec/impl/cuda/ops.py:17-101).

Storage types float32, bfloat16 and float16; gates, products and states are float32.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _capi
from .norm import _as_rows, _check_cuda, _fail, _ptr, _STORAGE, group_norm_act
from .ops import _DTYPES, _on_device, _workspace

__all__ = ["linrec_gated", "linrec_gated_step", "linrec_gated_norm", "linrec_gated_norm_step"]


# ---- arguments ---------------------------------------------------------------------------------------
def _check_operands(inputs, forget, input_gate, decay, decay_scale) -> None:
    """What the scan and the step have in common."""
    if inputs.dtype not in _STORAGE:
        _fail(f"dtype {inputs.dtype} is not supported (float32, bfloat16, float16)")
    for name, t in (("forget", forget), ("input_gate", input_gate)):
        if t is None:
            continue
        if t.shape != inputs.shape:
            _fail(f"{name} must have the sizes of the inputs")
        if t.dtype != inputs.dtype:
            _fail(f"{name} must have the dtype of the inputs")
    if (input_gate is None) != (decay is None):
        _fail("input_gate and decay come together (decay form) or not at all (forget form)")
    if decay is not None:
        if decay.shape != inputs.shape[-1:]:
            _fail("decay must have one value per channel")
        if not decay.is_floating_point():
            _fail("decay must be a floating-point tensor")
        if not float(decay_scale) > 0.0 or float(decay_scale) == float("inf"):
            _fail("decay_scale must be positive and finite")


def _check_index(name: str, t) -> None:
    if t.dtype not in (torch.int32, torch.int64):
        _fail(f"{name} must be int32 or int64")
    if t.dim() != 1:
        _fail(f"{name} must have one dimension")


def _scratch(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """The stream's workspace.  Inside a graph capture a fresh one that belongs to the graph: graphs that
    were captured on one stream may be replayed side by side on others."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return _workspace(device, stream, nbytes)


# ---- the scan ----------------------------------------------------------------------------------------
def _describe(inputs, forget, input_gate, decay, scale, cu, nseq, reverse):
    """The C struct for one problem, and the row-uniform tensors it points to."""
    D = inputs.size(-1)
    nrows = inputs.numel() // D if D else 0
    a = _capi.GatedArgs()
    x, a.x_stride = _as_rows(inputs)
    f, a.forget_stride = _as_rows(forget)
    a.x, a.forget = x.data_ptr(), f.data_ptr()
    i = None
    if input_gate is not None:
        i, a.input_gate_stride = _as_rows(input_gate)
        a.input_gate, a.decay, a.decay_scale = i.data_ptr(), decay.data_ptr(), scale
    a.dtype, a.reverse = _DTYPES[inputs.dtype], int(reverse)
    a.nseq, a.nrows, a.nchan = nseq, nrows, D
    if cu is None:
        a.seqlen = inputs.size(-2)
    else:
        a.cu_seqlens, a.cu_is_64 = cu.data_ptr(), int(cu.dtype == torch.int64)
    return a, (x, f, i)


def _run(entry, name, device, a) -> None:
    with _on_device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        ws = _scratch(device, stream, _capi.lib.linrec_b200_gated_workspace_size(ctypes.byref(a)))
        _capi.raise_for(entry(ctypes.byref(a), None, ws.data_ptr(), ws.numel(), stream), name)


def _states_like(other, shape, device, always: bool):
    """Final states (or their gradients' counterpart): what sequences without rows keep is filled in here."""
    if other is not None and always:
        return other.clone(memory_format=torch.contiguous_format)
    make = torch.zeros if always else torch.empty
    return make(shape, dtype=torch.float32, device=device)


def _forward(inputs, forget, input_gate, decay, initial, cu, scale, reverse, want_state, want_checkpoints):
    D = inputs.size(-1)
    lead = inputs.shape[:-2] if cu is None else (cu.numel() - 1,)
    nseq = 1
    for n in lead:
        nseq *= n
    a, keep = _describe(inputs, forget, input_gate, decay, scale, cu, nseq, reverse)
    y = torch.empty(inputs.shape, dtype=inputs.dtype, device=inputs.device)
    a.y, a.initial_state = y.data_ptr(), _ptr(initial)
    final = None
    if want_state:
        final = _states_like(initial, (*lead, D), inputs.device, always=cu is not None or inputs.size(-2) == 0)
        a.final_state = final.data_ptr()
    checkpoints = None
    if want_checkpoints:
        checkpoints = torch.empty(_capi.lib.linrec_b200_gated_checkpoint_rows(ctypes.byref(a)) * D, dtype=torch.float32,
                                  device=inputs.device)
        a.checkpoints = checkpoints.data_ptr()
    if y.numel():
        _run(_capi.lib.linrec_b200_gated_fwd, "linrec_b200_gated_fwd", inputs.device, a)
    return y, final, checkpoints


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, forget, input_gate, decay, initial, cu, scale, reverse, want_state):
        y, final, checkpoints = _forward(inputs, forget, input_gate, decay, initial, cu, scale, reverse, want_state, True)
        ctx.save_for_backward(inputs, forget, input_gate, decay, initial, cu, checkpoints)
        ctx.scale, ctx.reverse = scale, reverse
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        inputs, forget, input_gate, decay, initial, cu, checkpoints = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 9
        D, dev = inputs.size(-1), inputs.device
        nseq = cu.numel() - 1 if cu is not None else (inputs.numel() // (inputs.size(-2) * D) if inputs.numel() else 0)
        a, keep = _describe(inputs, forget, input_gate, decay, ctx.scale, cu, nseq, ctx.reverse)
        dy = torch.zeros_like(inputs) if dy is None else dy
        dy, a.dy_stride = _as_rows(dy)
        a.dy, a.checkpoints, a.initial_state = dy.data_ptr(), checkpoints.data_ptr(), _ptr(initial)
        if dfinal is not None:
            dfinal = dfinal.contiguous()
            a.d_final_state = dfinal.data_ptr()
        dx, df = (torch.empty(inputs.shape, dtype=inputs.dtype, device=dev) for _ in range(2))
        a.dx, a.dforget = dx.data_ptr(), df.data_ptr()
        di = ddecay = dinitial = scratch = None
        if decay is not None:
            di = torch.empty(inputs.shape, dtype=inputs.dtype, device=dev)
            ddecay = torch.empty_like(decay) if inputs.numel() else torch.zeros_like(decay)
            scratch = torch.empty(_capi.lib.linrec_b200_gated_scratch_size(ctypes.byref(a)), dtype=torch.uint8, device=dev)
            a.dinput_gate, a.ddecay = di.data_ptr(), ddecay.data_ptr()
            a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch.numel()
        if initial is not None and ctx.needs_input_grad[4]:
            dinitial = _states_like(dfinal, initial.shape, dev, always=cu is not None or inputs.size(-2) == 0)
            a.d_initial_state = dinitial.data_ptr()
        if inputs.numel():
            _run(_capi.lib.linrec_b200_gated_bwd, "linrec_b200_gated_bwd", dev, a)
        return dx, df, di, ddecay, dinitial, None, None, None, None


def linrec_gated(inputs: torch.Tensor, forget: torch.Tensor, *, input_gate: torch.Tensor | None = None,
                 decay: torch.Tensor | None = None, decay_scale: float = 8.0,
                 initial_state: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                 reverse: bool = False, return_state: bool = False):
    """Gated recurrence along the sequence of `inputs`, (..., T, D), or (rows, D) with `cu_seqlens`.

    inputs, forget, input_gate   one shape and dtype; any row stride (slices of one projection are fine)
    decay                        (D,); with input_gate: the decay form, without both: the forget form
    initial_state                (..., D), with cu_seqlens (sequences, D); zeros by default
    cu_seqlens                   int32 or int64 offsets on the device, non-decreasing, sequences + 1 of them;
                                 rows in front of the first and behind the last give zeros
    reverse                      scan every sequence from its last row to its first
    return_state                 also return the state behind each sequence's last scanned row, float32

    Differentiable once with respect to inputs, forget, input_gate, decay and initial_state."""
    if inputs.dim() < 2:
        _fail("inputs need a sequence and a channel dimension")
    _check_operands(inputs, forget, input_gate, decay, decay_scale)
    lead = inputs.shape[:-2]
    if cu_seqlens is not None:
        _check_index("cu_seqlens", cu_seqlens)
        if inputs.dim() != 2:
            _fail("packed inputs have two dimensions (rows, channels)")
        if cu_seqlens.numel() < 1:
            _fail("cu_seqlens holds one offset more than there are sequences")
        lead = (cu_seqlens.numel() - 1,)
    if initial_state is not None:
        if tuple(initial_state.shape) != (*lead, inputs.size(-1)):
            _fail("initial_state must have one row of channels per sequence")
        if not initial_state.is_floating_point():
            _fail("initial_state must be a floating-point tensor")
    _check_cuda(inputs, forget, input_gate, decay, initial_state, cu_seqlens)
    # casts outside the operator: autograd casts the gradients back
    decay = None if decay is None else decay.float().contiguous()
    initial_state = None if initial_state is None else initial_state.float().contiguous()
    cu_seqlens = None if cu_seqlens is None else cu_seqlens.contiguous()
    args = (inputs, forget, input_gate, decay, initial_state, cu_seqlens, float(decay_scale), bool(reverse), bool(return_state))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:5]):
        y, final = _GatedFn.apply(*args)
    else:
        y, final, _ = _forward(*args, False)
    return (y, final) if return_state else y


# ---- one token ---------------------------------------------------------------------------------------
def linrec_gated_step(inputs: torch.Tensor, forget: torch.Tensor, state: torch.Tensor, *,
                      input_gate: torch.Tensor | None = None, decay: torch.Tensor | None = None,
                      decay_scale: float = 8.0, slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of the recurrence for every row of `inputs` (rows, D); `state` (slots, D), float32, is
    updated in place and y (rows, D) returned.

    slots   (rows,) int32 or int64: the state row each row advances.  A slot outside the cache (such as -1)
            marks a padding row: zeros in y, no state touched.  Rows of the same slot are consecutive tokens
            of one sequence.  Without it row r advances state row r, and the two have as many rows.

    For decoding: refuses operands that need a gradient (`linrec_gated` over one position has one)."""
    if inputs.dim() != 2:
        _fail("inputs must have two dimensions (rows, channels)")
    _check_operands(inputs, forget, input_gate, decay, decay_scale)
    rows, D = inputs.shape
    if state.dim() != 2 or state.size(1) != D:
        _fail("state must have two dimensions, one row of channels per slot")
    if state.dtype != torch.float32:
        _fail("state must be float32")
    if state.numel() and ((D > 1 and state.stride(1) != 1) or (state.size(0) > 1 and state.stride(0) < D)):
        _fail("state rows must be dense and must not overlap: they are updated in place")
    if slots is None:
        if state.size(0) != rows:
            _fail("without slots the state has one row per row of the inputs")
    else:
        _check_index("slots", slots)
        if slots.numel() != rows:
            _fail("slots must name one state row per row of the inputs")
    _check_cuda(inputs, forget, input_gate, decay, state, slots)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (inputs, forget, input_gate, decay, state)):
        _fail("linrec_gated_step updates its state in place and has no backward pass; use linrec_gated")
    y = torch.empty((rows, D), dtype=inputs.dtype, device=inputs.device)
    if y.numel() == 0:
        return y
    x, sx = _as_rows(inputs)
    f, sf = _as_rows(forget)
    i, si = (None, 0) if input_gate is None else _as_rows(input_gate)
    decay = None if decay is None else decay.float().contiguous()
    slots = None if slots is None else slots.contiguous()
    with _on_device(inputs.device):
        stream = torch.cuda.current_stream(inputs.device).cuda_stream
        rc = _capi.lib.linrec_b200_gated_step(x.data_ptr(), f.data_ptr(), _ptr(i), sx, sf, si, _ptr(decay), float(decay_scale),
                                              y.data_ptr(), state.data_ptr(), max(state.stride(0), D), state.size(0),
                                              _ptr(slots), int(slots is not None and slots.dtype == torch.int64),
                                              rows, D, _DTYPES[inputs.dtype], stream)
    _capi.raise_for(rc, "linrec_b200_gated_step")
    torch.autograd.graph.increment_version(state)
    return y


# ---- with the norm behind it ---------------------------------------------------------------------------
def linrec_gated_norm(inputs: torch.Tensor, forget: torch.Tensor, gate: torch.Tensor | None, groups: int,
                      weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, activation: str | None = "silu",
                      eps: float = 1e-5, return_state: bool = False, **recurrence):
    """The mixing of a gated recurrence layer with heads: `linrec_gated(inputs, forget, **recurrence)`, then
    every position normalised head by head (`groups` heads of adjacent channels) and multiplied with the
    activated gate, `group_norm_act(h, groups, weight, bias, gate=gate)`.  Differentiable once."""
    r = linrec_gated(inputs, forget, return_state=return_state, **recurrence)
    h, state = r if return_state else (r, None)
    D = h.size(-1)
    if gate is not None and gate.shape != inputs.shape:
        _fail("gate must have the sizes of the inputs")
    y = group_norm_act(h.reshape(-1, D) if D else h, groups, weight, bias, gate=None if gate is None else gate.reshape(-1, D) if D else gate,
                       activation=activation, eps=eps).reshape(inputs.shape)
    return (y, state) if return_state else y


def linrec_gated_norm_step(inputs: torch.Tensor, forget: torch.Tensor, gate: torch.Tensor | None, state: torch.Tensor, groups: int,
                           weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
                           activation: str | None = "silu", eps: float = 1e-5, **recurrence) -> torch.Tensor:
    """`linrec_gated_norm` for one token per row: `linrec_gated_step`, then the norm and the gate.  A padding
    row's norm is that of zeros, act of the bias times the gate."""
    h = linrec_gated_step(inputs, forget, state, **recurrence)
    return group_norm_act(h, groups, weight, bias, gate=gate, activation=activation, eps=eps)
