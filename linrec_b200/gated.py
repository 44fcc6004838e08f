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

Derivatives are backward ones.  Forward-mode derivatives, torch.func transforms, recording by torch.jit.trace or make_fx
and fake tensors are refused; torch.compile runs the calls between its graphs.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _capi
from .norm import (_HUGEST, _STORAGE, _TINIEST, _as_float, _as_rows, _backward_once, _check_tensors, _empty_dense, _fail, _on, _ptr,
                   _wants_grad, group_norm_act)
from .norm import _apply as _apply_norm, _check as _check_norm
from .ops import _DTYPES, _workspace

_capturing = torch._C._cuda_isCurrentStreamCapturing

__all__ = ["linrec_gated", "linrec_gated_step", "linrec_gated_norm", "linrec_gated_norm_step"]


# ---- arguments ---------------------------------------------------------------------------------------
def _check_operands(inputs, forget, input_gate, decay, decay_scale) -> None:
    """What the scan and the step have in common."""
    shape, dtype = inputs.shape, inputs.dtype
    if dtype not in _STORAGE:
        _fail(f"dtype {dtype} is not supported (float32, bfloat16, float16)")
    for name, t in (("forget", forget), ("input_gate", input_gate)):
        if t is None:
            continue
        if t.shape != shape:
            _fail(f"{name} must have the sizes of the inputs")
        if t.dtype != dtype:
            _fail(f"{name} must have the dtype of the inputs")
    if (input_gate is None) != (decay is None):
        _fail("input_gate and decay come together (decay form) or not at all (forget form)")
    if decay is not None:
        if decay.shape != shape[-1:]:
            _fail("decay must have one value per channel")
        if not decay.is_floating_point():
            _fail("decay must be a floating-point tensor")
        if not _TINIEST < float(decay_scale) < _HUGEST:
            _fail("decay_scale must be positive and finite in float32")


def _check_index(name: str, t) -> None:
    if t.dtype not in (torch.int32, torch.int64):
        _fail(f"{name} must be int32 or int64")
    if t.dim() != 1:
        _fail(f"{name} must have one dimension")


def _scratch(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """The stream's workspace.  Inside a graph capture a fresh one that belongs to the graph: graphs that
    were captured on one stream may be replayed side by side on others."""
    if _capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return _workspace(device, stream, nbytes)


# ---- the scan ----------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _sizes(nseq, seqlen, nrows, D, packed):
    """Workspace bytes and checkpoint rows of a problem (the same in both passes and for every type)."""
    a = _capi.GatedArgs(nseq=nseq, seqlen=seqlen, nrows=nrows, nchan=D, cu_seqlens=16 if packed else None)
    ref = ctypes.byref(a)
    return _capi.lib.linrec_b200_gated_workspace_size(ref), _capi.lib.linrec_b200_gated_checkpoint_rows(ref)


class _Problem:
    """One scan: sizes, and the C struct for its passes."""

    def __init__(self, inputs, forget, input_gate, decay, initial, cu, scale, reverse):
        shape = inputs.shape
        self.D = D = shape[-1]
        self.nrows = math.prod(shape[:-1]) if D else 0
        self.seqlen = shape[-2]
        if cu is not None:
            self.nseq = cu.numel() - 1
            self.lead = (self.nseq,)
        else:
            self.lead = shape[:-2]
            self.nseq = math.prod(self.lead)
        self.sizes = _sizes(self.nseq, self.seqlen, self.nrows, D, cu is not None) if self.nrows else (0, 0)
        self.dtype, self.device = inputs.dtype, inputs.device
        x, sx = _as_rows(inputs)
        f, sf = _as_rows(forget)
        i, si = (None, 0) if input_gate is None else _as_rows(input_gate)
        self.keep = (x, f, i)
        # (the field order of linrec_gated_args)
        self.args = _capi.GatedArgs(x.data_ptr(), f.data_ptr(), _ptr(i), sx, sf, si, _ptr(decay), scale, _DTYPES[self.dtype], reverse,
                                    cu is not None and cu.dtype == torch.int64, _ptr(cu), self.nseq, self.seqlen, self.nrows, D,
                                    _ptr(initial))

    def run(self, bwd: bool) -> None:
        entry, name = ((_capi.lib.linrec_b200_gated_bwd, "linrec_b200_gated_bwd") if bwd else
                       (_capi.lib.linrec_b200_gated_fwd, "linrec_b200_gated_fwd"))

        def launch(stream):
            ws = _scratch(self.device, stream, self.sizes[0])
            _capi.raise_for(entry(ctypes.byref(self.args), None, ws.data_ptr(), ws.numel(), stream), name)

        _on(self.device, launch)


def _states_like(other, shape, device, always: bool):
    """Final states (or their gradients' counterpart): what sequences without rows keep is filled in here."""
    if other is not None and always:
        return other.clone(memory_format=torch.contiguous_format)
    make = torch.zeros if always else torch.empty
    return make(shape, dtype=torch.float32, device=device)


def _forward(inputs, forget, input_gate, decay, initial, cu, scale, reverse, want_state, want_checkpoints):
    p = _Problem(inputs, forget, input_gate, decay, initial, cu, scale, reverse)
    y = _empty_dense(inputs)
    p.args.y = y.data_ptr()
    final = checkpoints = None
    if want_state:
        final = _states_like(initial, (*p.lead, p.D), p.device, always=cu is not None or p.seqlen == 0)
        p.args.final_state = final.data_ptr()
    if want_checkpoints:
        checkpoints = torch.empty(p.sizes[1] * p.D, dtype=torch.float32, device=p.device)
        p.args.checkpoints = checkpoints.data_ptr()
    if p.nrows:
        p.run(False)
    return y, final, checkpoints


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, forget, input_gate, decay, initial, cu, scale, reverse, want_state):
        y, final, checkpoints = _forward(inputs, forget, input_gate, decay, initial, cu, scale, reverse, want_state, True)
        ctx.save_for_backward(inputs, forget, input_gate, decay, initial, cu, checkpoints)
        ctx.scale, ctx.reverse = scale, reverse
        ctx.set_materialize_grads(False)
        return y, final

    @_backward_once
    def backward(ctx, dy, dfinal):
        inputs, forget, input_gate, decay, initial, cu, checkpoints = ctx.saved_tensors
        if dy is None and dfinal is None:
            return (None,) * 9
        p = _Problem(inputs, forget, input_gate, decay, initial, cu, ctx.scale, ctx.reverse)
        a, dev = p.args, p.device
        dy = torch.zeros_like(inputs) if dy is None else dy
        dy, a.dy_stride = _as_rows(dy)
        a.dy, a.checkpoints = dy.data_ptr(), checkpoints.data_ptr()
        if dfinal is not None:
            dfinal = dfinal.contiguous()
            a.d_final_state = dfinal.data_ptr()
        dx, df = _empty_dense(inputs), _empty_dense(inputs)
        a.dx, a.dforget = dx.data_ptr(), df.data_ptr()
        di = ddecay = dinitial = scratch = None
        if decay is not None:
            di = _empty_dense(inputs)
            ddecay = torch.empty_like(decay) if p.nrows else torch.zeros_like(decay)
            scratch = torch.empty(p.sizes[1] * p.D, dtype=torch.float32, device=dev)
            a.dinput_gate, a.ddecay = di.data_ptr(), ddecay.data_ptr()
            a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch.numel() * 4
        if initial is not None and ctx.needs_input_grad[4]:
            dinitial = _states_like(dfinal, initial.shape, dev, always=cu is not None or p.seqlen == 0)
            a.d_initial_state = dinitial.data_ptr()
        if p.nrows:
            p.run(True)
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
    shape = inputs.shape
    if len(shape) < 2:
        _fail("inputs need a sequence and a channel dimension")
    _check_operands(inputs, forget, input_gate, decay, decay_scale)
    lead = shape[:-2]
    if cu_seqlens is not None:
        _check_index("cu_seqlens", cu_seqlens)
        if len(shape) != 2:
            _fail("packed inputs have two dimensions (rows, channels)")
        if cu_seqlens.numel() < 1:
            _fail("cu_seqlens holds one offset more than there are sequences")
        lead = (cu_seqlens.numel() - 1,)
    if initial_state is not None:
        if initial_state.shape != (*lead, shape[-1]):
            _fail("initial_state must have one row of channels per sequence")
        if not initial_state.is_floating_point():
            _fail("initial_state must be a floating-point tensor")
    _check_tensors(inputs, forget, input_gate, decay, initial_state, cu_seqlens)
    # casts outside the operator: autograd casts the gradients back
    decay, initial_state = _as_float(decay), _as_float(initial_state)
    cu_seqlens = None if cu_seqlens is None else cu_seqlens.contiguous()
    args = (inputs, forget, input_gate, decay, initial_state, cu_seqlens, float(decay_scale), bool(reverse), bool(return_state))
    if _wants_grad(inputs, forget, input_gate, decay, initial_state):
        y, final = _GatedFn.apply(*args)
    else:
        y, final, _ = _forward(*args, False)
    return (y, final) if return_state else y


# ---- one token ---------------------------------------------------------------------------------------
def _span(t):
    """First byte of `t` and the one behind its last."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _check_apart(state, *operands) -> None:
    """Names the refusal of operands in the memory between the state's first and last element."""
    for t in operands:
        if t is not None and t.numel() and state.numel():
            (first, behind), (lo, hi) = _span(t), _span(state)
            if first < hi and lo < behind:
                _fail("operands must not share memory with the state, which is updated in place")


def linrec_gated_step(inputs: torch.Tensor, forget: torch.Tensor, state: torch.Tensor, *,
                      input_gate: torch.Tensor | None = None, decay: torch.Tensor | None = None,
                      decay_scale: float = 8.0, slots: torch.Tensor | None = None) -> torch.Tensor:
    """One token of the recurrence for every row of `inputs` (rows, D); `state` (slots, D), float32, is
    updated in place and y (rows, D) returned.  No operand may lie in the memory from the state's first element to
    its last, but for other columns of the same rows.

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
    if not state.is_contiguous() and state.numel() and ((D > 1 and state.stride(1) != 1) or (state.size(0) > 1 and state.stride(0) < D)):
        _fail("state rows must be dense and must not overlap: they are updated in place")
    if slots is None:
        if state.size(0) != rows:
            _fail("without slots the state has one row per row of the inputs")
    else:
        _check_index("slots", slots)
        if slots.numel() != rows:
            _fail("slots must name one state row per row of the inputs")
    _check_tensors(inputs, forget, input_gate, decay, state, slots)
    if _wants_grad(inputs, forget, input_gate, decay, state):
        _fail("linrec_gated_step updates its state in place and has no backward pass; use linrec_gated")
    y = _empty_dense(inputs)
    if y.numel() == 0:
        return y
    x, sx = _as_rows(inputs)
    f, sf = _as_rows(forget)
    i, si = (None, 0) if input_gate is None else _as_rows(input_gate)
    decay = _as_float(decay)
    slots = None if slots is None else slots.contiguous()
    args = (x.data_ptr(), f.data_ptr(), _ptr(i), sx, sf, si, _ptr(decay), float(decay_scale), y.data_ptr(), state.data_ptr(), max(state.stride(0), D),
            state.size(0), _ptr(slots), slots is not None and slots.dtype == torch.int64, rows, D, _DTYPES[inputs.dtype])

    def launch(stream):
        rc = _capi.lib.linrec_b200_gated_step(*args, stream)
        if rc == _capi.ERR_OVERLAP:
            _check_apart(state, inputs, forget, input_gate, decay, slots)
        _capi.raise_for(rc, "linrec_b200_gated_step")

    _on(inputs.device, launch)
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
    _check_norm(inputs, groups, weight, bias, gate, activation, eps)      # before the state moves
    h = linrec_gated_step(inputs, forget, state, **recurrence)
    return _apply_norm(h, groups, weight, bias, gate, activation, eps)
