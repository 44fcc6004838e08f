"""Refusals of the gated recurrence and its step that need no GPU: every check runs before a device is
touched, and tensors outside a GPU are refused like everywhere in the package."""
import ctypes

import pytest
import torch

import linrec_b200 as lb
from linrec_b200 import _capi

X = torch.zeros(2, 5, 8)
P = torch.zeros(10, 8)


@pytest.mark.parametrize("why,call", [
    ("sequence and a channel", lambda: lb.linrec_gated(torch.zeros(8), torch.zeros(8))),
    ("not supported", lambda: lb.linrec_gated(X.double(), X.double())),
    ("not supported", lambda: lb.linrec_gated(X.long(), X.long())),
    ("forget must have the sizes", lambda: lb.linrec_gated(X, X[:, :4])),
    ("forget must have the dtype", lambda: lb.linrec_gated(X, X.bfloat16())),
    ("input_gate must have the sizes", lambda: lb.linrec_gated(X, X, input_gate=X[:1], decay=torch.zeros(8))),
    ("come together", lambda: lb.linrec_gated(X, X, input_gate=X)),
    ("come together", lambda: lb.linrec_gated(X, X, decay=torch.zeros(8))),
    ("one value per channel", lambda: lb.linrec_gated(X, X, input_gate=X, decay=torch.zeros(1))),
    ("floating-point", lambda: lb.linrec_gated(X, X, input_gate=X, decay=torch.zeros(8, dtype=torch.int32))),
    ("decay_scale", lambda: lb.linrec_gated(X, X, input_gate=X, decay=torch.zeros(8), decay_scale=0.0)),
    ("decay_scale", lambda: lb.linrec_gated(X, X, input_gate=X, decay=torch.zeros(8), decay_scale=float("nan"))),
    ("decay_scale", lambda: lb.linrec_gated(X, X, input_gate=X, decay=torch.zeros(8), decay_scale=float("inf"))),
    ("one row of channels per sequence", lambda: lb.linrec_gated(X, X, initial_state=torch.zeros(8))),
    ("one row of channels per sequence", lambda: lb.linrec_gated(P, P, initial_state=torch.zeros(3, 8), cu_seqlens=torch.zeros(3, dtype=torch.int32))),
    ("floating-point", lambda: lb.linrec_gated(X, X, initial_state=torch.zeros(2, 8, dtype=torch.int64))),
    ("int32 or int64", lambda: lb.linrec_gated(P, P, cu_seqlens=torch.zeros(3))),
    ("one dimension", lambda: lb.linrec_gated(P, P, cu_seqlens=torch.zeros(3, 1, dtype=torch.int32))),
    ("one offset more", lambda: lb.linrec_gated(P, P, cu_seqlens=torch.zeros(0, dtype=torch.int32))),
    ("two dimensions", lambda: lb.linrec_gated(X, X, cu_seqlens=torch.zeros(3, dtype=torch.int32))),
    ("CUDA tensors", lambda: lb.linrec_gated(X, X)),
    ("CUDA tensors", lambda: lb.linrec_gated(P, P, cu_seqlens=torch.zeros(3, dtype=torch.int32))),
    ("two dimensions", lambda: lb.linrec_gated_step(X, X, P)),
    ("one row of channels per slot", lambda: lb.linrec_gated_step(P, P, torch.zeros(10, 7))),
    ("state must be float32", lambda: lb.linrec_gated_step(P, P, P.bfloat16())),
    ("must not overlap", lambda: lb.linrec_gated_step(P, P, torch.zeros(1, 8).expand(10, 8))),
    ("must not overlap", lambda: lb.linrec_gated_step(P, P, torch.zeros(8, 10).t())),
    ("one row per row", lambda: lb.linrec_gated_step(P, P, torch.zeros(9, 8))),
    ("int32 or int64", lambda: lb.linrec_gated_step(P, P, P, slots=torch.zeros(10))),
    ("one state row per row", lambda: lb.linrec_gated_step(P, P, P, slots=torch.zeros(9, dtype=torch.int32))),
    ("come together", lambda: lb.linrec_gated_step(P, P, P, decay=torch.zeros(8))),
    ("CUDA tensors", lambda: lb.linrec_gated_step(P, P, P)),
])
def test_refusals(why, call):
    with pytest.raises(RuntimeError, match=why):
        call()


def _args(**kw):
    a = _capi.GatedArgs()
    base = {"nseq": 2, "seqlen": 5, "nrows": 10, "nchan": 8, "x": 16, "forget": 16, "x_stride": 8, "forget_stride": 8, "y": 16}
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("code,kw", [
    (_capi.ERR_INVALID_ARG, {"nrows": -1}),
    (_capi.ERR_INVALID_ARG, {"nrows": 11}),
    (_capi.ERR_INVALID_ARG, {"nseq": 3}),
    (_capi.ERR_INVALID_ARG, {"x_stride": 7}),
    (_capi.ERR_INVALID_ARG, {"x": None}),
    (_capi.ERR_INVALID_ARG, {"y": None}),
    (_capi.ERR_INVALID_ARG, {"decay": 16}),
    (_capi.ERR_INVALID_ARG, {"nrows": 1 << 40, "seqlen": 1 << 39}),
    (_capi.ERR_NOT_IMPLEMENTED, {"dtype": _capi.DTYPE_F64}),
    (_capi.ERR_NOT_IMPLEMENTED, {"dtype": 17}),
    (_capi.ERR_WORKSPACE, {}),
])
def test_c_entry_refuses(code, kw):
    a = _args(**kw)
    assert _capi.lib.linrec_b200_gated_fwd(ctypes.byref(a), None, None, 0, None) == code


def test_c_entry_options_and_sizes():
    a = _args()
    opts, keep = _capi.make_opts({"kStages": 2})
    assert _capi.lib.linrec_b200_gated_fwd(ctypes.byref(a), opts, None, 0, None) == _capi.ERR_NOT_IMPLEMENTED
    assert _capi.lib.linrec_b200_gated_fwd(None, None, None, 0, None) == _capi.ERR_INVALID_ARG
    assert _capi.lib.linrec_b200_gated_bwd(ctypes.byref(a), None, None, 0, None) == _capi.ERR_INVALID_ARG
    # no rows or channels: nothing to do, whatever the pointers are
    assert _capi.lib.linrec_b200_gated_fwd(ctypes.byref(_args(nrows=0, seqlen=0, x=None)), None, None, 0, None) == _capi.OK
    assert _capi.lib.linrec_b200_gated_checkpoint_rows(ctypes.byref(a)) == 1
    assert _capi.lib.linrec_b200_gated_checkpoint_rows(ctypes.byref(_args(nseq=3, seqlen=600, nrows=1800))) == 30
    assert _capi.lib.linrec_b200_gated_scratch_size(ctypes.byref(a)) == 0
    assert _capi.lib.linrec_b200_gated_step(None, None, None, 8, 8, 8, None, 8.0, None, None, 8, 4, None, 0, 4, 8, 0, None) == _capi.ERR_INVALID_ARG


@pytest.mark.parametrize("why,kw", [
    ("groups must divide", {"groups": 3}),
    ("activation", {"activation": "relu"}),
    ("eps", {"eps": 0.0}),
    ("weight must have", {"weight": torch.zeros(7)}),
    ("bias must have", {"bias": torch.zeros(7)}),
    ("gate must have the sizes", {"gate": P[:5]}),
    ("gate must have the sizes", {"gate": P.bfloat16()}),
])
def test_a_refused_norm_step_leaves_the_state(why, kw, monkeypatch):
    from linrec_b200 import gated
    steps = []
    monkeypatch.setattr(gated, "linrec_gated_step", lambda x, *a, **k: steps.append(1) or x)
    args = {"gate": None, "groups": 2, **kw}
    with pytest.raises(RuntimeError, match=why):
        lb.linrec_gated_norm_step(P, P, args.pop("gate"), P.clone(), args.pop("groups"), **args)
    assert not steps


def test_step_refuses_operands_in_the_memory_of_its_state():
    # rows are advanced by different blocks: one would read what another has already advanced
    from linrec_b200.gated import _check_apart
    cache = torch.zeros(20, 8)
    for state, operand in ((cache[5:15], cache[:10]), (cache[:10], cache[:10]), (cache[:10], cache[9]), (cache[:, :4], cache[:, 4:])):
        with pytest.raises(RuntimeError, match="share memory with the state"):
            _check_apart(state, P, None, operand)
    _check_apart(cache[10:], cache[:10], P, None, P[0])
    _check_apart(cache[:0], cache, cache[:10])


def _entry_points():
    d = torch.zeros(8)
    return {
        "scan": lambda x: lb.linrec_gated(x, P),
        "scan, decay": lambda x: lb.linrec_gated(P, x, input_gate=P, decay=d),
        "scan, state": lambda x: lb.linrec_gated(X, X, initial_state=x[:2]),
        "step": lambda x: lb.linrec_gated_step(P, x, P),
        "step, state": lambda x: lb.linrec_gated_step(P, P, x),
        "norm": lambda x: lb.group_norm_act(x, 2),
        "norm, gate": lambda x: lb.group_norm_act(P, 2, gate=x),
        "norm, weight": lambda x: lb.group_norm_act(P, 2, x[0]),
        "layer": lambda x: lb.linrec_gated_norm(x, x, x, 2),
        "layer step": lambda x: lb.linrec_gated_norm_step(P, P, x, P, 2),
    }


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", _entry_points())
def test_what_pytorch_cannot_see_through_is_refused(name):
    """The calls allocate a result and fill it out of PyTorch's sight: a tangent would be dropped and a recording
    would hold an empty tensor."""
    call = _entry_points()[name]
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode derivatives"):
            call(forward_ad.make_dual(P, torch.ones_like(P)))
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call(P)                       # no tangent, nothing to refuse
    for transform in (lambda: torch.func.vmap(call)(P[None]), lambda: torch.func.jvp(call, (P,), (P,)),
                      lambda: torch.func.grad(lambda x: call(x).sum())(P)):
        with pytest.raises(RuntimeError, match="torch.func transforms"):
            transform()
    with pytest.raises(RuntimeError, match="recorded by a tracer"):
        torch.jit.trace(call, (P,), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(RuntimeError, match="recorded by a tracer"):
            make_fx(call, tracing_mode=mode)(P)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = torch.empty(10, 8, device="cuda")
        with pytest.raises(RuntimeError, match="recorded by a tracer"):
            call(fake)
    with pytest.raises(RuntimeError, match="FakeTensor is not a tensor with memory|CUDA tensors"):
        call(mode.from_tensor(P))


def test_columns_beside_the_state_are_told_from_shared_memory():
    """The C entry's answer for every operand in turn, against sets of bytes.  A result that lies between elements,
    which is looked at later, keeps the accepted calls from going further."""
    def bytes_of(t):
        at = torch.zeros(1, dtype=torch.int64)
        for n, s in zip(t.shape, t.stride()):
            at = (at[:, None] + torch.arange(n) * s).flatten()
        first = t.data_ptr() + at * t.element_size()
        return set((first[:, None] + torch.arange(t.element_size())).flatten().tolist())

    code = {torch.float32: _capi.DTYPE_F32, torch.bfloat16: _capi.DTYPE_BF16}
    lone = torch.zeros(64)
    apart = lone.data_ptr()

    def step(state, dtype, rows, D, x=(apart, 8), forget=(apart, 8), gate=(apart, 8), y=apart + 129, decay=apart, slots=None):
        return _capi.lib.linrec_b200_gated_step(x[0], forget[0], gate[0], x[1], forget[1], gate[1], decay, 8.0, y, state.data_ptr(), state.stride(0),
                                                state.size(0), slots, 0, rows, D, dtype, None)

    buf = torch.zeros(12, 24)
    half, index = buf.view(torch.bfloat16), buf.view(torch.int32)
    states = [buf[2:8, 4:12], buf[:, :8], buf[3:4, :8], buf.view(6, 48)[:, 4:12]]
    operands = [buf[:, 12:20], buf[2:8, 12:20], buf[:4, 8:16], buf[2:8, 11:19], buf[:2, 4:12], buf[8:, 4:12], buf.view(6, 48)[:, 12:20],
                buf.view(6, 48)[:, 40:], half[:, 24:32], half[2:8, :8], half[:, 23:31], half[8:, 8:16], half[3:4, 8:16], buf.view(36, 8)[:9]]
    answers = set()
    for state in states:
        slots = torch.zeros(64, dtype=torch.int32).data_ptr()
        for t in operands:
            shared = bool(bytes_of(state) & bytes_of(t))
            for name in ("x", "forget", "gate"):
                rc = step(state, code[t.dtype], t.size(0), 8, slots=slots, **{name: (t.data_ptr(), t.stride(0))})
                assert rc in ((_capi.ERR_OVERLAP,) if shared else (_capi.ERR_OVERLAP, _capi.ERR_INVALID_ARG))
                # columns of their own in rows at the state's distance, and memory on either side of it, are no overlap
                if t.stride(0) * t.element_size() == state.stride(0) * 4 and not shared:
                    assert rc == _capi.ERR_INVALID_ARG
                answers.add((shared, rc))
        if state.size(0) > 1:
            inside = state.data_ptr() + state.stride(0) * 4
            assert step(state, 0, 2, 8, slots=inside) == step(state, 0, 2, 8, decay=inside, slots=slots) == _capi.ERR_OVERLAP
            assert step(state, 0, 2, 8, y=inside, slots=slots) == _capi.ERR_OVERLAP
    assert (True, _capi.ERR_OVERLAP) in answers and (False, _capi.ERR_INVALID_ARG) in answers


@pytest.mark.parametrize("dtype,kw", [
    (_capi.DTYPE_F32, {"x": 18}), (_capi.DTYPE_F32, {"forget": 18}), (_capi.DTYPE_F32, {"y": 18}), (_capi.DTYPE_BF16, {"x": 17}),
    (_capi.DTYPE_F16, {"y": 17}), (_capi.DTYPE_BF16, {"initial_state": 18}), (_capi.DTYPE_BF16, {"final_state": 18}), (_capi.DTYPE_BF16, {"checkpoints": 18}),
    (_capi.DTYPE_BF16, {"cu_seqlens": 18}), (_capi.DTYPE_BF16, {"cu_seqlens": 20, "cu_is_64": 1}),
    (_capi.DTYPE_BF16, {"decay": 18, "input_gate": 16, "input_gate_stride": 8}), (_capi.DTYPE_F32, {"decay": 16, "input_gate": 18, "input_gate_stride": 8}),
])
def test_c_entry_refuses_pointers_between_elements(dtype, kw):
    # a workspace that is never reached: refused before it is looked at
    a = _args(dtype=dtype, **kw)
    assert _capi.lib.linrec_b200_gated_fwd(ctypes.byref(a), None, 256, 1 << 40, None) == _capi.ERR_INVALID_ARG
    back = {"dy": 16, "dy_stride": 8, "dx": 16, "dforget": 16, "checkpoints": 16}
    for n in back:
        if n != "dy_stride":
            b = _args(dtype=dtype, **{**back, n: 17})
            assert _capi.lib.linrec_b200_gated_bwd(ctypes.byref(b), None, 256, 1 << 40, None) == _capi.ERR_INVALID_ARG


@pytest.mark.parametrize("at", range(6))
def test_c_step_refuses_pointers_between_elements(at):
    p = [(i + 1) << 20 for i in range(6)]      # x, forget, input_gate, decay, y, state
    p[at] += 2
    call = lambda slots, wide: _capi.lib.linrec_b200_gated_step(p[0], p[1], p[2], 8, 8, 8, p[3], 8.0, p[4], p[5], 8, 4, slots, wide, 4, 8, _capi.DTYPE_F32, None)
    assert call(None, 0) == _capi.ERR_INVALID_ARG
    p[at] -= 2
    assert call(18, 0) == call(20, 1) == _capi.ERR_INVALID_ARG


@pytest.mark.parametrize("value", [1e39, 2.0 ** 128 - 2.0 ** 103, 1e-46, 2.0 ** -150])
def test_scalars_that_float32_cannot_hold(value):
    """They would reach the kernels as infinity or zero; the largest and smallest that it holds are taken."""
    d = torch.zeros(8)
    assert ctypes.c_float(value).value in (0.0, float("inf"))
    for call, why in ((lambda v: lb.linrec_gated(X, X, input_gate=X, decay=d, decay_scale=v), "decay_scale"),
                      (lambda v: lb.linrec_gated_step(P, P, P, input_gate=P, decay=d, decay_scale=v), "decay_scale"),
                      (lambda v: lb.group_norm_act(P, 2, eps=v), "eps")):
        with pytest.raises(RuntimeError, match=why):
            call(value)
        for good in (2.0 ** 128 - 2.0 ** 104, 2.0 ** -149, torch.tensor(8.0)):
            with pytest.raises(RuntimeError, match="CUDA tensors"):
                call(good)
