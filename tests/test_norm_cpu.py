"""Refusals of the group norm that need no GPU."""
import ctypes

import pytest
import torch

import linrec_b200 as lb
from linrec_b200 import _capi

X = torch.zeros(4, 5, 12)
W = torch.ones(12)


@pytest.mark.parametrize("why,call", [
    ("sample and a channel", lambda: lb.group_norm_act(W, 3)),
    ("not supported", lambda: lb.group_norm_act(X.double(), 3)),
    ("groups must divide", lambda: lb.group_norm_act(X, 5)),
    ("groups must divide", lambda: lb.group_norm_act(X, 0)),
    ("groups must divide", lambda: lb.group_norm_act(X, True)),
    ("groups must divide", lambda: lb.group_norm_act(X, 3.0)),
    ("activation", lambda: lb.group_norm_act(X, 3, activation="gelu")),
    ("eps", lambda: lb.group_norm_act(X, 3, eps=0.0)),
    ("eps", lambda: lb.group_norm_act(X, 3, eps=float("nan"))),
    ("weight must have", lambda: lb.group_norm_act(X, 3, torch.ones(3))),
    ("bias must have", lambda: lb.group_norm_act(X, 3, W, torch.ones(12, dtype=torch.int32))),
    ("gate must have", lambda: lb.group_norm_act(X, 3, gate=X[:1])),
    ("gate must have", lambda: lb.group_norm_act(X, 3, gate=X.bfloat16())),
    ("CUDA tensors", lambda: lb.group_norm_act(X, 3, W, W, gate=X)),
    ("CUDA tensors", lambda: lb.linrec_gated_norm(X, X, X, 3, W)),
    ("CUDA tensors", lambda: lb.linrec_gated_norm_step(X[0], X[0], X[0], X[0], 3, W)),
])
def test_refusals(why, call):
    with pytest.raises(RuntimeError, match=why):
        call()


def _args(**kw):
    a = _capi.GroupNormArgs()
    base = {"x": 16, "x_stride": 12, "y": 16, "eps": 1e-5, "nsamples": 4, "positions": 5, "nchan": 12, "groups": 3}
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("code,kw", [
    (_capi.ERR_INVALID_ARG, {"groups": 5}),
    (_capi.ERR_INVALID_ARG, {"groups": 0}),
    (_capi.ERR_INVALID_ARG, {"eps": 0.0}),
    (_capi.ERR_INVALID_ARG, {"nsamples": -1}),
    (_capi.ERR_INVALID_ARG, {"x": None}),
    (_capi.ERR_INVALID_ARG, {"y": None}),
    (_capi.ERR_INVALID_ARG, {"x_stride": 11}),
    (_capi.ERR_INVALID_ARG, {"gate": 16, "gate_stride": 0}),
    (_capi.ERR_INVALID_ARG, {"nsamples": 1 << 40, "positions": 1 << 40}),
    (_capi.ERR_NOT_IMPLEMENTED, {"activation": 3}),
    (_capi.ERR_NOT_IMPLEMENTED, {"dtype": _capi.DTYPE_F64}),
    (_capi.ERR_WORKSPACE, {}),
    (_capi.OK, {"nsamples": 0, "x": None}),
])
def test_c_entry_refuses(code, kw):
    assert _capi.lib.linrec_b200_group_norm_fwd(ctypes.byref(_args(**kw)), None) == code


def test_c_backward_refuses():
    full = {"dy": 16, "dy_stride": 12, "dx": 16, "stats": 16}
    for missing in full:
        assert _capi.lib.linrec_b200_group_norm_bwd(ctypes.byref(_args(**{**full, missing: None if missing != "dy_stride" else 0})), None) == _capi.ERR_INVALID_ARG
    # parameter gradients need scratch
    assert _capi.lib.linrec_b200_group_norm_bwd(ctypes.byref(_args(**full, dweight=16)), None) == _capi.ERR_WORKSPACE
    assert _capi.lib.linrec_b200_group_norm_bwd(None, None) == _capi.ERR_INVALID_ARG


@pytest.mark.parametrize("name", ["x", "y", "gate", "weight", "bias", "stats", "dy", "dx", "dgate", "dweight", "dbias"])
def test_c_entries_refuse_pointers_between_elements(name):
    good = {"gate": 16, "gate_stride": 12, "dy": 16, "dy_stride": 12, "dx": 16, "dgate": 16, "stats": 16, "scratch": 16, "scratch_bytes": 1 << 40}
    at = 20 if name == "stats" else 18      # (pairs of floats)
    forward = _capi.lib.linrec_b200_group_norm_fwd(ctypes.byref(_args(**{**good, name: at})), None)
    back = _capi.lib.linrec_b200_group_norm_bwd(ctypes.byref(_args(**{**good, "dweight": 16, "dbias": 16, name: at})), None)
    assert forward == back == _capi.ERR_INVALID_ARG
    if name in ("x", "y", "gate", "dy", "dx", "dgate"):
        a = _args(**{**good, name: 17}, dtype=_capi.DTYPE_BF16)
        assert _capi.lib.linrec_b200_group_norm_fwd(ctypes.byref(a), None) == _capi.ERR_INVALID_ARG
