"""Group norm with an activation or a gate on the GPU, against a 64-bit evaluation that carries the error
bound of a float32 one (tests/norm_oracle.py), and the gated recurrence with the norm behind it.  Results
in 16 bits may be off by half a step of their type on top of that."""
import numpy as np
import pytest
import torch

import gated_oracle as go
import norm_oracle as no
from test_gated_gpu import _case as _scan_case, _check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = {"x": "dx", "weight": "dweight", "bias": "dbias", "gate": "dgate"}


def _lb():
    import linrec_b200
    return linrec_b200


def _case(shape, dtype, gate=True, affine=True, seed=0, shift=0.5, scale=1.0):
    g = torch.Generator().manual_seed(seed + 11)
    C = shape[-1]
    c = {"x": (scale * torch.randn(shape, generator=g) + shift * torch.randn(C, generator=g)).to(dtype),
         "dy": torch.randn(shape, generator=g).to(dtype)}
    if gate:
        c["gate"] = (2.0 * torch.randn(shape, generator=g)).to(dtype)
    if affine:
        c["weight"], c["bias"] = 1.0 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    return c


def _oracle(c, groups, act, eps=1e-5):
    n = {k: v.double().numpy() for k, v in c.items()}
    return no.evaluate(n["x"], groups, n.get("weight"), n.get("bias"), n.get("gate"), act, eps, n["dy"])


def _run(c, groups, act, place=None, eps=1e-5):
    dev = {k: (place or (lambda _, t: t.to(DEV)))(k, v) for k, v in c.items()}
    leaves = {k: dev[k].requires_grad_(True) for k in NAMES if k in dev}
    y = _lb().group_norm_act(leaves["x"], groups, leaves.get("weight"), leaves.get("bias"), gate=leaves.get("gate"), activation=act, eps=eps)
    got = torch.autograd.grad(y, list(leaves.values()), dev["dy"])
    with torch.no_grad():
        plain = _lb().group_norm_act(leaves["x"], groups, leaves.get("weight"), leaves.get("bias"), gate=leaves.get("gate"), activation=act, eps=eps)
    assert torch.equal(plain.isnan(), y.isnan()) and torch.equal(plain.nan_to_num(), y.nan_to_num())
    return {"y": y, **{NAMES[k]: t for k, t in zip(leaves, got)}}


def _compare(got, want):
    for n, t in got.items():
        _check(t, want[n], n)


# (shape, groups): one position per sample, several, whole rows as one group, odd sizes, groups wider than a warp
SHAPES = [((1, 16), 1), ((3, 64), 2), ((7, 96), 6), ((33, 1000), 8), ((5, 1002), 6), ((4, 4096), 32), ((300, 256), 16), ((2, 8192), 1),
          ((3, 5000), 1), ((9, 17 * 24), 17), ((2, 40, 64), 8), ((3, 7, 5, 48), 3), ((2, 333, 1002), 6), ((1, 2000, 32), 32), ((4, 100, 6), 1),
          ((65, 2, 130), 2), ((2, 600, 512), 4), ((1, 33, 16384), 2), ((1, 40000), 5),
          ((1500, 3, 24), 3), ((5000, 48), 3), ((900, 1), 1)]


@pytest.mark.parametrize("shape,groups", SHAPES, ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else f"g{s}")
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_values_and_gradients(shape, groups, dtype):
    for gate in (False, True):
        for act in ("silu", "sigmoid", None):
            c = _case(shape, dtype, gate, affine=act != "sigmoid" or gate, seed=shape[-1])
            _compare(_run(c, groups, act), _oracle(c, groups, act))


def test_far_from_zero():
    """A mean far above the spread, and constant groups (variance zero: eps alone)."""
    for shape, groups in (((6, 512), 4), ((2, 300, 64), 4)):
        c = _case(shape, torch.float32, shift=0.0)
        c["x"] = c["x"] + 1000.0
        _compare(_run(c, groups, "silu"), _oracle(c, groups, "silu"))
        c["x"] = torch.full(shape, 3.0)
        got = _run(c, groups, "silu")
        want = _oracle(c, groups, "silu")
        _compare(got, want)
        assert all(torch.isfinite(t).all() for t in got.values())


def test_a_sample_keeps_its_infinities():
    for shape, groups in (((40, 256), 8), ((5, 70, 96), 3)):
        c = _case(shape, torch.bfloat16)
        clean = _run(c, groups, "silu")
        c["x"] = c["x"].clone()
        c["x"][3, ..., 5] = float("inf")
        dirty = _run(c, groups, "silu")
        width = shape[-1] // groups
        for n in ("y", "dx", "dgate"):
            keep = torch.ones(shape, dtype=torch.bool, device=DEV)
            keep[3, ..., :width] = False
            assert torch.equal(clean[n][keep], dirty[n][keep]), n
            assert not torch.isfinite(dirty[n][3, ..., :width]).all(), n


def test_layouts():
    """Operands that are slices of wider tensors, starting anywhere, and a gradient in another layout."""
    for shape, groups, wide, starts in (((50, 64), 4, 256, (0, 64)), ((50, 40), 5, 137, (1, 45)), ((4, 30, 72), 3, 300, (4, 80)), ((3, 20, 65), 5, 131, (0, 66))):
        for dtype in (torch.float32, torch.bfloat16):
            c = _case(shape, dtype)
            base = torch.full((*shape[:-1], wide), float("nan"), dtype=dtype, device=DEV)

            def place(k, t):
                if k in ("x", "gate"):
                    at = starts[k == "gate"]
                    v = base[..., at:at + shape[-1]]
                    v.copy_(t)
                    return v.detach()
                if k == "dy":
                    return t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
                return t.to(DEV)

            _compare(_run(c, groups, "silu", place), _oracle(c, groups, "silu"))


def test_differences():
    for shape, groups in (((2, 12), 2), ((2, 3, 8), 2)):
        for gate in (False, True):
            for act in ("silu", "sigmoid"):
                c = _case(shape, torch.float32, gate)
                got = _run(c, groups, act)
                c = {k: v.double() for k, v in c.items()}
                loss = lambda: (_oracle(c, groups, act)["y"][0] * c["dy"].numpy()).sum()
                step = 1e-4
                for k, n in NAMES.items():
                    if k not in c:
                        continue
                    for at in np.ndindex(*c[k].shape):
                        keep = c[k][at].item()
                        c[k][at] = keep + step
                        up = loss()
                        c[k][at] = keep - step
                        down = loss()
                        c[k][at] = keep
                        # third derivatives below 1e3 at this spread: step^2/6 * 1e3 < 2e-6
                        assert abs((up - down) / (2 * step) - got[n][at].item()) < 2e-5 + 1e-4 * abs(got[n][at].item()), (n, at)


def test_same_bits_every_time():
    for shape, groups in (((500, 1024), 8), ((3, 700, 256), 8)):
        c = _case(shape, torch.bfloat16)
        one = _run(c, groups, "silu")
        for _ in range(3):
            two = _run(c, groups, "silu")
            assert all(torch.equal(one[n], two[n]) for n in one)


def test_nothing_to_do():
    lb = _lb()
    for shape in ((0, 16), (2, 0, 16), (0, 3, 16)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w = torch.ones(16, device=DEV, requires_grad=True)
        y = lb.group_norm_act(x, 4, w)
        gx, gw = torch.autograd.grad(y, [x, w], torch.empty(shape, device=DEV))
        assert y.shape == gx.shape == x.shape and (gw == 0).all()


def test_parameters_in_16_bits():
    lb = _lb()
    c = _case((30, 64), torch.bfloat16)
    w, b = (c[k].bfloat16().to(DEV).requires_grad_(True) for k in ("weight", "bias"))
    y = lb.group_norm_act(c["x"].to(DEV), 4, w, b)
    gw, gb = torch.autograd.grad(y, [w, b], c["dy"].to(DEV))
    assert gw.dtype == gb.dtype == torch.bfloat16
    c["weight"], c["bias"] = w.detach().cpu().float(), b.detach().cpu().float()
    del c["gate"]
    want = _oracle(c, 4, "silu")
    _check(y, want["y"], "y")
    _check(gw, want["dweight"], "dweight")


def test_captured_and_replayed():
    lb = _lb()
    for shape, groups in (((200, 512), 8), ((3, 300, 64), 4)):
        c = {k: v.to(DEV) for k, v in _case(shape, torch.bfloat16).items()}
        leaves = [c[k].requires_grad_(True) for k in NAMES]

        def step():
            y = lb.group_norm_act(leaves[0], groups, leaves[1], leaves[2], gate=leaves[3])
            return [y, *torch.autograd.grad(y, leaves, c["dy"])]

        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = step()
        fresh = _case(shape, torch.bfloat16, seed=9)
        for k, v in fresh.items():
            c[k].detach().copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = _oracle(fresh, groups, "silu")
        for n, t in zip(("y", *NAMES.values()), outs):
            _check(t, want[n], n)


# ---- the recurrence with the norm behind it ----------------------------------------------------------------
def test_training_step_of_a_layer():
    """Recurrence, norm and gate over packed sequences: the same bits as the two operators, each of which is
    held to its own oracle, and gradients of every operand."""
    lb = _lb()
    offsets = [0, 70, 70, 300, 512]
    for dtype in (torch.float32, torch.bfloat16):
        c = _scan_case((520, 128), True, dtype, nseq=4)
        g = torch.Generator().manual_seed(5)
        c |= {"gate": torch.randn(520, 128, generator=g).to(dtype), "weight": 1 + 0.2 * torch.randn(128, generator=g), "bias": 0.2 * torch.randn(128, generator=g)}
        dev = {k: v.to(DEV) for k, v in c.items()}
        leaves = [dev[k].requires_grad_(True) for k in ("inputs", "forget", "input_gate", "decay", "initial_state", "gate", "weight", "bias")]
        x, f, i, d, h0, gate, w, b = leaves
        kw = {"input_gate": i, "decay": d, "initial_state": h0, "cu_seqlens": torch.tensor(offsets, dtype=torch.int32, device=DEV)}
        y, end = lb.linrec_gated_norm(x, f, gate, 8, w, b, return_state=True, **kw)
        grads = torch.autograd.grad([y, end], leaves, [dev["dy"], dev["dfinal"]])
        h, end2 = lb.linrec_gated(x, f, return_state=True, **kw)
        cut = h.detach().requires_grad_(True)
        y2 = lb.group_norm_act(cut, 8, w, b, gate=gate)
        dh, *second = torch.autograd.grad(y2, [cut, gate, w, b], dev["dy"])
        first = torch.autograd.grad([h, end2], leaves[:5], [dh, dev["dfinal"]])
        assert torch.equal(y, y2) and torch.equal(end, end2)
        assert all(torch.equal(p, q) for p, q in zip(grads, [*first, *second]))
        # each half against its oracle, at the values that reach it
        n = lambda t: t.detach().double().cpu().numpy()
        ref = no.evaluate(n(cut), 8, n(w), n(b), n(gate), "silu", 1e-5, n(dev["dy"]))
        for name, t in zip(("y", "dx", "dgate", "dweight", "dbias"), (y, dh, *second)):
            _check(t, ref[name], name)
        ref = go.evaluate(n(x), n(f), n(i), n(d), h0=n(h0), offsets=offsets, dy=n(dh), dfinal=n(dev["dfinal"]),
                          fast=dtype != torch.float32)
        for name, t in zip(("final", "dx", "dforget", "dinput", "ddecay", "dinitial"), (end, *first)):
            _check(t, ref[name], name)


def test_prefill_then_decode():
    """A prompt through the scan, then tokens one by one on the cache, against the whole in 64 bits."""
    lb = _lb()
    B, T, P, D, G = 3, 90, 70, 128, 4
    c = _scan_case((B, T, D), True, torch.float32)
    g = torch.Generator().manual_seed(6)
    gate, w, b = torch.randn(B, T, D, generator=g), 1 + 0.2 * torch.randn(D, generator=g), 0.2 * torch.randn(D, generator=g)
    n = lambda t: t.double().numpy()
    h = go.evaluate(n(c["inputs"]), n(c["forget"]), n(c["input_gate"]), n(c["decay"]))["y"]
    want = no.evaluate(h[0].reshape(B * T, D), G, n(w), n(b), n(gate).reshape(B * T, D), "silu", ex=h[1].reshape(B * T, D))["y"]
    want = tuple(t.reshape(B, T, D) for t in want)
    dev = {k: v.to(DEV) for k, v in c.items()}
    gate, w, b = gate.to(DEV), w.to(DEV), b.to(DEV)
    y, end = lb.linrec_gated_norm(dev["inputs"][:, :P], dev["forget"][:, :P], gate[:, :P], G, w, b, return_state=True,
                                  input_gate=dev["input_gate"][:, :P], decay=dev["decay"])
    _check(y, tuple(t[:, :P] for t in want), "prompt")
    cache = torch.full((8, D), float("nan"), device=DEV)
    slots = torch.tensor([6, 0, 3, -1], device=DEV)
    cache[slots[:3]] = end
    pad = lambda t: torch.cat([t, torch.full_like(t[:1], float("nan"))])
    for t in range(P, T):
        at = {k: pad(dev[k][:, t]) for k in ("inputs", "forget", "input_gate")}
        y = lb.linrec_gated_norm_step(at["inputs"], at["forget"], pad(gate[:, t]), cache, G, w, b, input_gate=at["input_gate"],
                                      decay=dev["decay"], slots=slots)
        _check(y[:3], tuple(v[:, t] for v in want), f"token {t}")
    assert torch.isnan(cache[[1, 2, 4, 5, 7]]).all()


@pytest.mark.parametrize("width", [264, 300, 384, 500, 512, 683, 1000, 1024])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_wide_groups(width, dtype):
    """Groups of 257 to 1024 channels, one position per sample, whose lanes have many pieces each: operands on
    16-byte boundaries, one element off them, and parameters off them; more rows than the CTAs take in one turn."""
    for rows, groups, off in ((1000, 3, None), (1000, 3, "x"), (41, 1, "weight"), (1, 2, "x")):
        for gate, act in ((True, "silu"), (False, "sigmoid")):
            C = groups * width
            c = _case((rows, C), dtype, gate, affine=gate or off == "weight", seed=width)
            # memory that the results will get: an element that nothing writes shows
            del [torch.full((rows, C), float("nan"), dtype=dtype, device=DEV) for _ in range(8)][:]

            def place(k, t):
                if k == off or (off == "x" and k in ("gate", "dy")):
                    wide = torch.full((*t.shape[:-1], C + 1), float("nan"), dtype=t.dtype, device=DEV)
                    wide[..., 1:] = t.to(DEV)
                    return wide[..., 1:].detach()
                return t.to(DEV)

            _compare(_run(c, groups, act, place), _oracle(c, groups, act))


def test_an_outlier_in_front():
    """Whole sequences whose first position is far from all others: the statistics hold although every thread
    that meets the outlier counts its distances from it first."""
    lb = _lb()
    g = torch.Generator(device=DEV).manual_seed(3)
    # 223 samples fill the device with one slice each: 8 channels of 600 positions per thread (16-byte accesses), or
    # one channel of 600 (rows off 16-byte boundaries)
    for C, groups, skip in ((2048, 32, 0), (256, 4, 1)):
        for far in (30.0, 1000.0, 1e4):
            base = torch.randn(223, 600, C + skip, generator=g, device=DEV)
            x = base[..., skip:]
            x[:, 0, ::C // groups] = far
            y = lb.group_norm_act(x, groups, activation=None, eps=1e-5)
            # a few samples in 64 bits
            for n in (0, 100, 222):
                v = x[n].double().reshape(600, groups, -1)
                d = v - v.mean((0, 2), keepdim=True)
                want = (d / torch.sqrt((d * d).mean((0, 2), keepdim=True) + 1e-5)).reshape(600, C)
                # A thread adds 8 * 600 / 2 squares one after the other at most, and fewer than 32 partial sums follow.
                # Counted about elements of the data the squares come to twice those about the mean (once, where an
                # outlier made the thread count about its mean), so the variance is off by 2 (2400 + 32) 2^-24 of
                # itself and its root by half of that; the mean by as many steps of the distance from those elements,
                # which is on average below the sum of both ends' distances from zero.
                steps = (2400 + 32) * 2.0 ** -24
                tol = steps * (want.abs() + 2 * v.abs().mean() / v.std()) + 1e-6
                assert (y[n].double() - want).abs().le(tol).all(), (C, far, n, ((y[n].double() - want).abs() / tol).max())
            del base, x, y
