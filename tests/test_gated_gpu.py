"""Gated recurrence, its gradients and its one-token step on the GPU, against a sequential evaluation in 64
bits (tests/gated_oracle.py, which also carries the error bound of a float32 evaluation).  Results in 16 bits
may be off by half a step of their type on top of that."""
import numpy as np
import pytest
import torch

import gated_oracle as go

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = {"inputs": "dx", "forget": "dforget", "input_gate": "dinput", "decay": "ddecay", "initial_state": "dinitial"}


def _lb():
    import linrec_b200
    return linrec_b200


def _check(got, want, what):
    value, bound = want
    dt = got.dtype
    g = got.detach().double().cpu().numpy().reshape(value.shape)
    tol = bound + 1e-37
    if dt != torch.float32:
        # half a step of the type at the largest value the bound allows; subnormal steps of fp16
        tol = tol + (np.abs(value) + bound) * torch.finfo(dt).eps / 2 + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    bad = ~(np.abs(g - value) <= tol)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.abs(g - value) / tol, 0)), bad.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside, worst at {at}: {g[at]} for {value[at]} +- {tol[at]}")


def _case(shape, decay, dtype, seed=0, states=True, nseq=None, spread=4.0):
    g = torch.Generator().manual_seed(seed + 1)
    D = shape[-1]
    lead = shape[:-2] if nseq is None else (nseq,)
    c = {"inputs": torch.randn(shape, generator=g), "forget": torch.rand(D, generator=g) * spread + torch.randn(shape, generator=g),
         "dy": torch.randn(shape, generator=g)}
    if decay:
        c["input_gate"] = torch.randn(shape, generator=g)
        c["decay"] = torch.rand(D, generator=g) * 5.0 - 5.0
    if states:
        c["initial_state"] = torch.randn(*lead, D, generator=g)
        c["dfinal"] = torch.randn(*lead, D, generator=g)
    for n in ("inputs", "forget", "input_gate", "dy"):
        if n in c:
            c[n] = c[n].to(dtype)
    return c


def _oracle(c, **kw):
    n = {k: (v.double().numpy() if v is not None else None) for k, v in c.items()}
    return go.evaluate(n["inputs"], n["forget"], n.get("input_gate"), n.get("decay"), h0=n.get("initial_state"), dy=n["dy"],
                       dfinal=n.get("dfinal"), fast=c["inputs"].dtype != torch.float32, **kw)


def _run(c, place=None, **kw):
    """Forward and backward through the public entry point: dict of results."""
    dev = {k: (place or (lambda _, t: t.to(DEV)))(k, v) for k, v in c.items()}
    leaves = {k: dev[k].requires_grad_(True) for k in NAMES if k in dev}
    y, final = _lb().linrec_gated(leaves["inputs"], leaves["forget"], return_state=True, **kw,
                                  **{k: v for k, v in leaves.items() if k not in ("inputs", "forget")})
    outs, grads = ([y, final], [dev["dy"], dev["dfinal"]]) if "dfinal" in dev else ([y], [dev["dy"]])
    got = torch.autograd.grad(outs, list(leaves.values()), grads)
    return {"y": y, "final": final, **{NAMES[k]: t for k, t in zip(leaves, got)}}


def _compare(got, want):
    for n, t in got.items():
        _check(t, want[n], n)
    _lb().check_status()


SHAPES = [(1, 1, 1), (2, 1, 64), (1, 63, 65), (2, 64, 8), (3, 130, 72), (2, 512, 136), (1, 1000, 33), (5, 129, 64), (1, 4100, 16),
          (33, 3, 66), (2, 3, 70, 40), (4, 384, 128), (70, 128)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_scan_and_gradients(shape, decay, dtype):
    for reverse in (False, True):
        for states in (False, True):
            c = _case(shape, decay, dtype, seed=len(shape) + shape[-1], states=states)
            _compare(_run(c, reverse=reverse), _oracle(c, reverse=reverse))


LENGTHS = {"mixed": (0, [0, 1, 0, 5, 200, 0, 64, 1, 1, 0], 0), "gaps": (3, [130, 1, 128, 77], 19), "one": (0, [300], 0),
           "singles": (0, [1] * 150, 2), "none": (0, [], 40), "empty": (5, [0, 0], 70), "long": (0, [3, 2500, 0, 700], 64)}


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_packed_sequences(name, decay, dtype):
    front, lens, tail = LENGTHS[name]
    offsets = [front]
    for n in lens:
        offsets.append(offsets[-1] + n)
    for D, reverse, kind in ((72, False, torch.int32), (40, True, torch.int64), (67, False, torch.int64)):
        c = _case((offsets[-1] + tail, D), decay, dtype, nseq=len(lens), seed=D)
        # what lies outside the sequences must not matter
        outside = torch.ones(offsets[-1] + tail, dtype=torch.bool)
        outside[offsets[0]:offsets[-1]] = False
        want = _oracle(c, offsets=offsets, reverse=reverse)
        for i, n in enumerate(k for k in ("inputs", "forget", "input_gate", "dy") if k in c):
            c[n] = c[n].clone()
            c[n][outside] = [float("nan"), float("inf"), -float("inf"), float("nan")][i]
        got = _run(c, cu_seqlens=torch.tensor(offsets, dtype=kind, device=DEV), reverse=reverse)
        _compare(got, want)
        for n in ("y", "dx", "dforget", "dinput"):
            if n in got:
                assert (got[n][outside.to(DEV)] == 0).all(), n


def test_a_sequence_keeps_its_infinities():
    """NaN and infinity in one sequence, its states included, leave the others' bits alone."""
    offsets = [0, 100, 164, 230, 500]
    for decay in (False, True):
        for reverse in (False, True):
            cu = torch.tensor(offsets, dtype=torch.int32, device=DEV)
            c = _case((500, 66), decay, torch.float32, nseq=4)
            clean = _run(c, cu_seqlens=cu, reverse=reverse)
            for n in c:
                if n in ("initial_state", "dfinal"):
                    c[n] = c[n].clone()
                    c[n][2] = float("nan")
                elif n != "decay":
                    c[n] = c[n].clone()
                    c[n][180:200] = float("inf") if n == "forget" else float("nan")
            dirty = _run(c, cu_seqlens=cu, reverse=reverse)
            for n in clean:
                if n == "ddecay":
                    continue
                keep = torch.ones(clean[n].shape[0], dtype=torch.bool, device=DEV)
                if clean[n].shape[0] == 500:
                    keep[164:230] = False
                else:
                    keep[2] = False
                assert torch.equal(clean[n][keep], dirty[n][keep]), n
                assert not torch.isfinite(dirty[n][~keep]).all(), n


@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
def test_extreme_logits(decay):
    """Open and shut gates: multipliers of exactly one and zero, input factors next to nothing."""
    T, D = 150, 64
    c = _case((1, T, D), decay, torch.float32)
    c["forget"] = torch.tensor([-200.0, -100.0, -20.0, -1e-30, 0.0, 3.0, 17.0, 100.0, 200.0, float("inf"), -float("inf")])[
        torch.randint(0, 11, (1, T, D), generator=torch.Generator().manual_seed(3))]
    if decay:
        c["decay"] = torch.linspace(-60.0, 12.0, D)
        c["input_gate"] = 30.0 * c["input_gate"]
    got = _run(c)
    c["forget"] = c["forget"].clamp(-1e4, 1e4)
    want = _oracle(c)
    for n, t in got.items():
        assert torch.isfinite(t).all(), n
        # below 1.2e-38 values lose their bits; log a reaches the results through its root, 1.1e-19, times
        # operands whose products stay below 1e4 here
        _check(t, (want[n][0], want[n][1] + 2e-15), n)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("value", ["inf", "lowest"])
def test_masked_rows_hold_the_state(dtype, value):
    """Logits of minus infinity, or of the type's lowest value: the decay form keeps its state to the bit and takes
    nothing in, the forget form replaces it; of plus infinity the forget form keeps it."""
    lb = _lb()
    low = -float("inf") if value == "inf" else torch.finfo(dtype).min
    g = torch.Generator().manual_seed(1)
    x, i, h0 = torch.randn(2, 200, 72, generator=g).to(DEV, dtype), torch.randn(2, 200, 72, generator=g).to(DEV, dtype), torch.randn(2, 72, generator=g).to(DEV)
    i[:, 5:9] = low
    d = torch.linspace(-6.0, 3.0, 72, device=DEV)
    for state in (h0, torch.zeros_like(h0)):
        shut = torch.full_like(x, low)
        y, end = lb.linrec_gated(x, shut, input_gate=i, decay=d, initial_state=state, return_state=True)
        assert torch.equal(end, state) and torch.equal(y, state[:, None].to(dtype).expand_as(y))
        y, end = lb.linrec_gated(x, -shut, initial_state=state, return_state=True)
        assert torch.equal(end, state) and torch.equal(y, state[:, None].to(dtype).expand_as(y))
        y, end = lb.linrec_gated(x, shut, initial_state=state, return_state=True)
        assert torch.equal(y, x) and torch.equal(end, x[:, -1].float())
        one = state.clone()
        assert torch.equal(lb.linrec_gated_step(x[:, 0], shut[:, 0], one, input_gate=i[:, 0], decay=d), state.to(dtype))
        assert torch.equal(one, state)
    # a masked stretch in the middle of a sequence: the rows around it do not notice
    f = torch.randn(2, 200, 72, generator=g).to(DEV, dtype)
    f[:, 60:140] = low
    keep = torch.ones(200, dtype=torch.bool, device=DEV)
    keep[60:140] = False
    whole, end = lb.linrec_gated(x, f, input_gate=i, decay=d, initial_state=h0, return_state=True)
    short, end2 = lb.linrec_gated(x[:, keep], f[:, keep], input_gate=i[:, keep], decay=d, initial_state=h0, return_state=True)
    # (tiles begin elsewhere, so products of multipliers round elsewhere)
    assert torch.allclose(whole[:, keep].float(), short.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
    assert torch.allclose(end, end2, rtol=1e-4, atol=1e-5)
    # held: a run of positions is entered through the joined runs before it, fewer than 20 products and sums of terms
    # below 10, each rounded: 20 * 10 * 2^-24 = 1.2e-5
    assert torch.allclose(whole[:, 60:140].float(), whole[:, 59:60].float().expand(-1, 80, -1), rtol=torch.finfo(dtype).eps, atol=1.2e-5)


def test_inference_mode():
    lb = _lb()
    with torch.inference_mode():
        c = {k: v.to(DEV) for k, v in _case((3, 40, 64), True, torch.bfloat16).items()}
        y, end = lb.linrec_gated(c["inputs"], c["forget"], input_gate=c["input_gate"], decay=c["decay"], return_state=True)
        z = lb.linrec_gated_step(c["inputs"][:, 0], c["forget"][:, 0], end, input_gate=c["input_gate"][:, 0], decay=c["decay"])
        assert torch.isfinite(lb.group_norm_act(z, 4)).all()


def test_expanded_gradient():
    """The gradient of a sum is one number seen everywhere."""
    c = _case((2, 130, 72), True, torch.float32, states=False)
    c["dy"] = torch.ones(2, 130, 72)
    _compare(_run(c, lambda k, t: torch.ones((), device=DEV).expand(t.shape) if k == "dy" else t.to(DEV)), _oracle(c))


def test_differences():
    """Gradients against central differences of the 64-bit evaluation."""
    for decay in (False, True):
        for reverse in (False, True):
            offsets = [0, 4, 4, 9]
            c = _case((9, 3), decay, torch.float32, nseq=3, spread=1.0)
            got = _run(c, cu_seqlens=torch.tensor(offsets, dtype=torch.int32, device=DEV), reverse=reverse)

            def loss(c):
                r = _oracle(c, offsets=offsets, reverse=reverse)
                return (r["y"][0] * c["dy"].numpy()).sum() + (r["final"][0] * c["dfinal"].numpy()).sum()

            step = 1e-4
            c = {k: v.double() for k, v in c.items()}
            for k, n in NAMES.items():
                if k not in c:
                    continue
                for at in np.ndindex(*c[k].shape):
                    keep = c[k][at].item()
                    c[k][at] = keep + step
                    up = loss(c)
                    c[k][at] = keep - step
                    down = loss(c)
                    c[k][at] = keep
                    # third derivatives of this loss stay below 1e4: step^2/6 * 1e4 < 2e-5; float32 results of size < 100
                    assert abs((up - down) / (2 * step) - got[n][at].item()) < 2e-5 + 1e-4 * abs(got[n][at].item()), (n, at)


def test_slices_of_one_projection():
    """Operands that are slices of a wider tensor, starting anywhere, and a gradient in another layout."""
    for D, wide, starts in ((64, 256, (0, 64, 128)), (40, 137, (1, 45, 91)), (72, 300, (4, 80, 200)), (65, 260, (0, 65, 130))):
        for dtype in (torch.float32, torch.bfloat16):
            c = _case((3, 140, D), True, dtype, seed=D)
            base = torch.full((3, 140, wide), float("nan"), dtype=dtype, device=DEV)
            at = dict(zip(("inputs", "forget", "input_gate"), starts))

            def place(k, t):
                if k in at:
                    v = base[..., at[k]:at[k] + D]
                    v.copy_(t)
                    return v.detach()
                if k == "dy":
                    return t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
                return t.to(DEV)

            _compare(_run(c, place), _oracle(c))


def test_rows_far_apart():
    """Row offsets beyond 2^31 elements, in the operands and in the state cache."""
    stride, D, T = (1 << 30) + 8, 64, 4
    wide = torch.empty(stride * (T - 1) + D, dtype=torch.bfloat16, device=DEV)
    c = _case((1, T, D), False, torch.bfloat16, states=False)

    def place(k, t):
        if k != "inputs":
            return t.to(DEV)
        v = wide.as_strided((1, T, D), (stride * T, stride, 1))
        v.copy_(t)
        return v

    got = _run(c, place)
    _compare(got, _oracle(c))
    del got, wide
    state = torch.empty(stride * 2 + D, dtype=torch.float32, device=DEV).as_strided((3, D), (stride, 1))
    state.copy_(torch.ones(3, D))
    x = torch.zeros(3, D, device=DEV)
    y = _lb().linrec_gated_step(x, x, state)
    assert (y == 0.5).all() and (state == 0.5).all()


def test_states_chain_calls():
    """A sequence scanned in pieces, state handed on, is the sequence scanned whole."""
    lb = _lb()
    for decay in (False, True):
        c = {k: v.to(DEV) for k, v in _case((2, 700, 96), decay, torch.float32).items()}
        kw = {"decay": c["decay"]} if decay else {}
        whole, end = lb.linrec_gated(c["inputs"], c["forget"], input_gate=c.get("input_gate"), initial_state=c["initial_state"],
                                     return_state=True, **kw)
        h, parts = c["initial_state"], []
        for lo, hi in ((0, 1), (1, 129), (129, 129), (129, 640), (640, 700)):
            y, h = lb.linrec_gated(c["inputs"][:, lo:hi], c["forget"][:, lo:hi],
                                   input_gate=c["input_gate"][:, lo:hi] if decay else None, initial_state=h, return_state=True, **kw)
            parts.append(y)
        # two float32 evaluations of one recurrence with multipliers below 0.9994: each within 1e-5 of the truth
        # (bound of the oracle, checked above) at values up to 10
        assert torch.allclose(torch.cat(parts, 1), whole, rtol=1e-4, atol=1e-4)
        assert torch.allclose(h, end, rtol=1e-4, atol=1e-4)


def test_same_bits_every_time():
    c = _case((2, 1500, 200), True, torch.bfloat16)
    one = _run(c)
    for _ in range(3):
        two = _run(c)
        assert all(torch.equal(one[n], two[n]) for n in one)
    # a few columns only: how far the look-back walks differs from run to run, the bits do not
    c = _case((1, 20000, 64), True, torch.float32)
    one = _run(c)
    for _ in range(5):
        two = _run(c)
        assert all(torch.equal(one[n], two[n]) for n in one)
    _lb().check_status()


def test_many_tiles_in_flight():
    """Few channels and many positions: every resident CTA waits in the look-back of one column."""
    for T, D, dtype in ((20000, 64, torch.float32), (15001, 72, torch.bfloat16)):
        for decay in (False, True):
            c = _case((1, T, D), decay, dtype, spread=8.0)
            _compare(_run(c), _oracle(c))


def test_captured_and_replayed():
    """Forward and backward in CUDA graphs captured on one stream, replayed side by side on others, on new data."""
    lb = _lb()
    cases = [_case((2, 900, 128), True, torch.bfloat16, seed=s) for s in (1, 2)]
    graphs = []
    stream = torch.cuda.Stream()
    for c in cases:
        dev = {k: v.to(DEV) for k, v in c.items()}
        leaves = [dev[k].requires_grad_(True) for k in NAMES]
        torch.cuda.synchronize()

        def step():
            y, final = lb.linrec_gated(leaves[0], leaves[1], input_gate=leaves[2], decay=leaves[3], initial_state=leaves[4], return_state=True)
            return [y, final, *torch.autograd.grad([y, final], leaves, [dev["dy"], dev["dfinal"]])]

        with torch.cuda.stream(stream):
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = step()
        graphs.append((graph, outs, dev, leaves))
    fresh = [_case((2, 900, 128), True, torch.bfloat16, seed=s) for s in (3, 4)]
    for (_, _, dev, _), c in zip(graphs, fresh):
        for k, v in c.items():
            dev[k].detach().copy_(v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for (graph, _, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, outs, _, _), c in zip(graphs, fresh):
        want = _oracle(c)
        for n, t in zip(("y", "final", *NAMES.values()), outs):
            _check(t, want[n], n)


def test_side_streams():
    lb = _lb()
    c = _case((2, 600, 128), False, torch.float32)
    want = _oracle(c)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(_run(c))
    torch.cuda.synchronize()
    for g in got:
        _compare(g, want)


def test_gradients_asked_for_in_part():
    lb = _lb()
    c = {k: v.to(DEV) for k, v in _case((2, 70, 64), True, torch.float32).items()}
    full = _run({k: v.cpu() for k, v in c.items()})
    for k, n in NAMES.items():
        t = c[k].clone().requires_grad_(True)
        kw = {m: c[m] for m in NAMES if m != k}
        kw[k] = t
        y, final = lb.linrec_gated(kw.pop("inputs"), kw.pop("forget"), return_state=True, **kw)
        got, = torch.autograd.grad([y, final], [t], [c["dy"], c["dfinal"]])
        assert torch.equal(got, full[n]), n
    # gradient through the state alone
    x = c["inputs"].clone().requires_grad_(True)
    _, final = lb.linrec_gated(x, c["forget"], return_state=True)
    got, = torch.autograd.grad(final, x, c["dfinal"])
    want = go.evaluate(c["inputs"].double().cpu().numpy(), c["forget"].double().cpu().numpy(), dfinal=c["dfinal"].double().cpu().numpy())
    _check(got, want["dx"], "dx")
    # 16-bit parameters and states are cast, their gradients cast back
    d, h = c["decay"].bfloat16().requires_grad_(True), c["initial_state"].bfloat16().requires_grad_(True)
    y = lb.linrec_gated(c["inputs"], c["forget"], input_gate=c["input_gate"], decay=d, initial_state=h)
    gd, gh = torch.autograd.grad(y, [d, h], c["dy"])
    assert gd.dtype == gh.dtype == torch.bfloat16


def test_no_rows():
    lb = _lb()
    h0 = torch.randn(2, 8, device=DEV, requires_grad=True)
    x = torch.empty(2, 0, 8, device=DEV, requires_grad=True)
    d = torch.randn(8, device=DEV, requires_grad=True)
    y, h = lb.linrec_gated(x, x, input_gate=x, decay=d, initial_state=h0, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(h, h0)
    gx, gd, gh = torch.autograd.grad(h, [x, d, h0], torch.ones_like(h))
    assert gx.shape == x.shape and (gd == 0).all() and (gh == 1).all()
    assert lb.linrec_gated(torch.empty(0, 5, 8, device=DEV), torch.empty(0, 5, 8, device=DEV)).shape == (0, 5, 8)
    assert lb.linrec_gated_step(torch.empty(0, 8, device=DEV), torch.empty(0, 8, device=DEV), torch.empty(0, 8, device=DEV)).shape == (0, 8)


# ---- one token ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 64), (7, 257), (33, 1000), (2, 2048), (130, 40), (600, 4100), (600, 1003)])
@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_step(rows, D, decay, dtype):
    lb = _lb()
    c = _case((rows, 1, D), decay, dtype)
    want = _oracle(c)
    args = [c[k].to(DEV)[:, 0] for k in ("inputs", "forget")]
    kw = {"input_gate": c["input_gate"].to(DEV)[:, 0], "decay": c["decay"].to(DEV)} if decay else {}
    state = c["initial_state"].to(DEV)
    y = lb.linrec_gated_step(*args, state, **kw)
    _check(y, want["y"], "y")
    _check(state, want["final"], "state")
    # through slots of a larger, padded cache, 64-bit and 32-bit indexes, with padding rows
    slots = torch.randperm(rows + 5, generator=torch.Generator().manual_seed(rows))[:rows]
    for kind in (torch.int64, torch.int32):
        cache = torch.full((rows + 5, D + 3), 7.0, device=DEV)
        view = cache[:, 1:D + 1]
        view[slots.to(DEV)] = c["initial_state"].to(DEV)
        use = slots.to(kind).to(DEV).clone()
        if rows > 2:
            use[1], use[2] = -1, rows + 5
        y = lb.linrec_gated_step(*args, view, slots=use, **kw)
        live = torch.ones(rows, dtype=torch.bool)
        if rows > 2:
            live[1:3] = False
            assert (y[1:3] == 0).all()
            assert torch.equal(view[slots[1:3].to(DEV)], c["initial_state"].to(DEV)[1:3])
        _check(y[live.to(DEV)], tuple(t[live.numpy()] for t in want["y"]), "y")
        _check(view[slots.to(DEV)[live.to(DEV)]], tuple(t[live.numpy()] for t in want["final"]), "state")
        untouched = torch.ones(rows + 5, dtype=torch.bool, device=DEV)
        untouched[slots.to(DEV)] = False
        assert (cache[untouched] == 7.0).all() and (cache[:, 0] == 7.0).all() and (cache[:, D + 1:] == 7.0).all()


@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
def test_steps_are_a_scan(decay):
    lb = _lb()
    B, T, D = 3, 9, 200
    c = _case((B, T, D), decay, torch.float32)
    want = _oracle(c)
    dev = {k: v.to(DEV) for k, v in c.items()}
    kw = (lambda t: {"input_gate": dev["input_gate"][:, t], "decay": dev["decay"]}) if decay else (lambda t: {})
    state = dev["initial_state"].clone()
    ys = [lb.linrec_gated_step(dev["inputs"][:, t], dev["forget"][:, t], state, **kw(t)) for t in range(T)]
    _check(torch.stack(ys, 1), want["y"], "y")
    _check(state, want["final"], "state")
    # the same tokens as rows of one call: rows that share a slot are one sequence, in row order
    order = torch.randperm(B * T, generator=torch.Generator().manual_seed(5))
    seq = (torch.arange(B * T) % B)[order]                     # which sequence each row belongs to
    pos = torch.empty(B * T, dtype=torch.long)
    for q in range(B):
        pos[seq == q] = torch.arange(T)
    rows = {k: dev[k][seq, pos] for k in ("inputs", "forget", "input_gate") if k in dev}
    state = dev["initial_state"].clone()
    kw = {"input_gate": rows["input_gate"], "decay": dev["decay"]} if decay else {}
    y = lb.linrec_gated_step(rows["inputs"], rows["forget"], state, slots=seq.to(torch.int32).to(DEV), **kw)
    _check(y, tuple(t[seq.numpy(), pos.numpy()] for t in want["y"]), "y")
    _check(state, want["final"], "state")


def test_step_replayed():
    """A captured decode step advances its cache at every replay."""
    lb = _lb()
    c = _case((4, 6, 128), True, torch.bfloat16)
    want = _oracle(c)
    dev = {k: v.to(DEV) for k, v in c.items()}
    x, f, i = (dev[k][:, 0].clone() for k in ("inputs", "forget", "input_gate"))
    state = dev["initial_state"].clone()
    keep = state.clone()
    lb.linrec_gated_step(x, f, state, input_gate=i, decay=dev["decay"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lb.linrec_gated_step(x, f, state, input_gate=i, decay=dev["decay"])
    state.copy_(keep)
    for t in range(6):
        for buf, k in ((x, "inputs"), (f, "forget"), (i, "input_gate")):
            buf.copy_(dev[k][:, t])
        graph.replay()
        _check(y, tuple(v[:, t] for v in want["y"]), "y")
    _check(state, want["final"], "state")


@pytest.mark.parametrize("which", ["inputs", "forget"])
def test_step_refuses_operands_in_the_memory_of_its_state(which):
    cache, x = torch.randn(20, 8, device=DEV), torch.randn(10, 8, device=DEV)
    before = cache.clone()
    args = {"inputs": x, "forget": x, which: cache[:10]}
    with pytest.raises(RuntimeError, match="share memory with the state"):
        _lb().linrec_gated_step(args["inputs"], args["forget"], cache[5:15])
    assert torch.equal(cache, before)
    _lb().linrec_gated_step(args["inputs"], args["forget"], cache[10:])      # side by side in one buffer


def test_a_refused_norm_step_leaves_the_state():
    x, state = torch.randn(10, 8, device=DEV), torch.randn(10, 8, device=DEV)
    before = state.clone()
    for kw in ({"groups": 3}, {"groups": 2, "weight": torch.ones(8)}, {"groups": 2, "eps": 0.0}):
        with pytest.raises(RuntimeError):
            _lb().linrec_gated_norm_step(x, x, None, state, **kw)
    assert torch.equal(state, before)


EXTREME = [-200.0, -110.0, -89.0, -88.0, -87.5, -87.0, -86.0, -85.0, -84.0, -83.0, -82.0, -80.0, -75.0, -60.0, -45.0, -20.0, 0.0, 3.0, 17.0, 90.0, 200.0]


@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_extreme_logits_in_every_type(dtype, decay):
    """Gates that are next to nothing without being nothing, beside gates of ordinary size, in scan, gradients and step."""
    lb = _lb()
    T, D = 150, 64
    # rates of the decay form: from below 2^-149 to 96, and below 1/4 in all channels (a series of its own)
    for lo, hi, wide in ((-110.0, 12.0, 1.0), (-110.0, -4.0, 1.0), (-20.0, -5.0, 30.0)):
        c = _case((1, T, D), decay, dtype)
        c["forget"] = torch.tensor(EXTREME)[torch.randint(0, len(EXTREME), (1, T, D), generator=torch.Generator().manual_seed(3))].to(dtype)
        c["inputs"][:, ::7] = 0.0
        if decay:
            c["decay"] = torch.linspace(lo, hi, D)
            c["input_gate"] = wide * c["input_gate"]
        got, want = _run(c), _oracle(c)
        for n, t in got.items():
            assert torch.isfinite(t).all(), n
            # below 1.2e-38 values lose their bits; log a reaches the results through its root, 1.1e-19, times
            # operands whose products stay below 1e4 here; an input gate below e^-44 counts as shut
            _check(t, (want[n][0], want[n][1] + 2e-15), n)
        state = c["initial_state"].to(DEV)
        kw = {"input_gate": c["input_gate"][:, 0].to(DEV), "decay": c["decay"].to(DEV)} if decay else {}
        y = lb.linrec_gated_step(c["inputs"][:, 0].to(DEV), c["forget"][:, 0].to(DEV), state, **kw)
        _check(y, tuple(t[:, 0] + e for t, e in zip(want["y"], (0.0, 2e-15))), "step")
        lb.check_status()
        if not decay:
            break


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_nan_logits_show(dtype):
    """A NaN gate is not a shut gate: the state is NaN from there on, at the sequence's first row as well."""
    for decay in (False, True):
        for at in (0, 1, 40):
            for name in ("forget", "input_gate") if decay else ("forget",):
                c = _case((1, 70, 64), decay, dtype, states=False)
                c[name][:, at, 3] = float("nan")
                y = _lb().linrec_gated(*(c[k].to(DEV) for k in ("inputs", "forget")),
                                       **({k: c[k].to(DEV) for k in ("input_gate", "decay")} if decay else {}))
                bad = torch.zeros(70, 64, dtype=torch.bool, device=DEV)
                bad[at:, 3] = True
                assert torch.equal(y[0].isnan(), bad), (decay, at, name)


@pytest.mark.parametrize("D", [66, 72, 1280], ids=lambda d: f"D{d}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_sequence_keeps_its_nan_logits(dtype, D):
    """NaN in the logits of a sequence's first or last scanned positions leaves all other sequences' values and gradients
    alone, bit for bit, packed and in a batch of short sequences on one axis."""
    offsets = [0, 100, 164, 230, 500]
    for decay in (False, True):
        for reverse in (False, True):
            for packed in (True, False):
                kw = {"cu_seqlens": torch.tensor(offsets, dtype=torch.int32, device=DEV)} if packed else {}
                lo, hi = (164, 230) if packed else (2 * 77, 3 * 77)
                c = _case((500, D) if packed else (5, 77, D), decay, dtype, nseq=4 if packed else None)
                clean = _run(c, reverse=reverse, **kw)
                for at in ([0], [1], [5, 6], [-1], [-2], [20]):
                    d = {k: v.clone() for k, v in c.items()}
                    for n in ("forget", "input_gate") if decay else ("forget",):
                        d[n].view(-1, D)[torch.tensor(at) + (lo if at[0] >= 0 else hi)] = float("nan")
                    dirty = _run(d, reverse=reverse, **kw)
                    for n in clean:
                        if n == "ddecay":
                            continue
                        whole, part = clean[n].flatten(0, -2), dirty[n].flatten(0, -2)
                        keep = torch.ones(len(whole), dtype=torch.bool, device=DEV)
                        if len(whole) < 10:
                            keep[2] = False
                        else:
                            keep[lo:hi] = False
                        assert torch.equal(whole[keep], part[keep]), (n, at, reverse, packed)
                        if n in ("dx", "dforget"):
                            assert part[~keep].isnan().any(), (n, at)


@pytest.mark.filterwarnings("ignore")
def test_under_modes_that_only_look_on_and_compiled():
    """Counting and profiling modes, and torch.compile, which runs the calls between its graphs."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Onlooker(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    lb = _lb()
    c = _case((2, 70, 64), True, torch.float32, states=False)
    x, f, i, d = (c[k].to(DEV) for k in ("inputs", "forget", "input_gate", "decay"))

    def layer(x):
        y = lb.linrec_gated_norm(2.0 * x, f, i, 4, input_gate=i, decay=d)
        state = torch.zeros(2, 64, device=DEV)
        with torch.no_grad():
            z = lb.linrec_gated_norm_step(x[:, 0], f[:, 0], i[:, 0], state, 4, input_gate=i[:, 0], decay=d)
        return y + 1.0, z, state

    def run(fn):
        leaf = x.clone().requires_grad_(True)
        out = fn(leaf)
        return (*out, *torch.autograd.grad(out[0], leaf, c["dy"].to(DEV)))

    want = run(layer)
    with Onlooker():
        got = run(layer)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = run(torch.compile(layer, backend="eager"))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_step_on_columns_of_one_buffer():
    """State and float32 operands as column blocks of the same rows; 16-bit and index views of the state's memory are
    refused."""
    lb = _lb()
    D = 24
    g = torch.Generator().manual_seed(2)
    buf = torch.randn(10, 3 * D, generator=g).to(DEV)
    state, x, f = buf[:, :D], buf[:, D:2 * D], buf[:, 2 * D:]
    alone = state.clone()
    want = lb.linrec_gated_step(x.clone(), f.clone(), alone)
    keep = buf[:, D:].clone()
    assert torch.equal(lb.linrec_gated_step(x, f, state), want)
    assert torch.equal(state, alone) and torch.equal(buf[:, D:], keep)
    state = torch.zeros(10, D, device=DEV)
    h = torch.zeros(10, D, dtype=torch.bfloat16, device=DEV)
    for args, kw in (((state.view(torch.bfloat16)[:, :D], h), {}), ((h, state.view(torch.float16)[:, D:].view(torch.bfloat16)), {}),
                     ((h, h), {"slots": state.view(torch.int32)[0, :10]})):
        with pytest.raises(RuntimeError, match="share memory with the state"):
            lb.linrec_gated_step(*args, state, **kw)
    assert (state == 0).all()


# Sizes that reach every way a tile is linked to the one before it, on a device of 148 SMs, rows on 16-byte boundaries
# (columns: blocks of 64 channels times batch entries; `test_scan_and_gradients` has look-back).
#   12, 20, 19 and 50 columns   clusters of eight, seven, seven and two CTAs, with turns in which some have no tile
#   80                          clusters of one: a CTA keeps a column to itself
#   160                         eight warps, jobs of four tiles
#   300                         that forward in 16 bits, backward four warps
#   450                         four warps in both directions (16 bits), jobs of four tiles and a shorter one
COLUMNS = {12: (1, 1100, 768), 20: (2, 1100, 640), 19: (1, 2300, 1216), 50: (5, 600, 640), 80: (8, 600, 640),
           160: (1, 700, 10240), 300: (2, 520, 9600), 450: (1, 330, 28800)}


def _added_up(want, positions):
    """The decay gradient is a sum over positions, `positions` of them one after the other in 32 bits; its bound
    holds 50 roundings of every term already."""
    if "ddecay" in want:
        value, bound = want["ddecay"]
        want["ddecay"] = (value, bound * (1 + (positions + 8) / 50))
    return want


@pytest.mark.parametrize("columns,dtype", [(n, t) for n in COLUMNS for t in DTYPES if t != torch.float16 or n in (12, 450)],
                         ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
def test_every_way_of_linking_tiles(columns, dtype, decay):
    shape = COLUMNS[columns]
    for reverse in (False, True):
        c = _case(shape, decay, dtype, seed=columns, states=reverse == decay)
        got = _run(c, reverse=reverse)
        # a thread has every fourth run of the column's positions at least
        _compare(got, _added_up(_oracle(c, reverse=reverse), shape[-2] / 4))
        again = _run(c, reverse=reverse)
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("columns,rows", [(12, 1100), (50, 700), (80, 450), (160, 700), (450, 330)], ids=lambda n: str(n))
@pytest.mark.parametrize("decay", [False, True], ids=["forget", "decay"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_packed_in_every_way_of_linking_tiles(columns, rows, decay, dtype):
    for reverse, kind in ((False, torch.int32), (True, torch.int64)):
        # empty and one-row sequences, one that starts where a tile does, one over several tiles, rows of none
        offsets = [5, 5, 64, 65, 65, 128, 200, rows - 30, rows - 17]
        c = _case((rows, columns * 64), decay, dtype, nseq=len(offsets) - 1, seed=columns)
        want = _added_up(_oracle(c, offsets=offsets, reverse=reverse), rows / 4)
        outside = torch.ones(rows, dtype=torch.bool)
        outside[offsets[0]:offsets[-1]] = False
        for i, n in enumerate(k for k in ("inputs", "forget", "input_gate", "dy") if k in c):
            c[n] = c[n].clone()
            c[n][outside] = [float("nan"), float("inf"), -float("inf"), float("nan")][i]
        cu = torch.tensor(offsets, dtype=kind, device=DEV)
        got = _run(c, cu_seqlens=cu, reverse=reverse)
        _compare(got, want)
        for n in ("y", "dx", "dforget", "dinput"):
            if n in got:
                assert (got[n][outside.to(DEV)] == 0).all(), n
        again = _run(c, cu_seqlens=cu, reverse=reverse)
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("columns", [12, 80, 160, 450])
def test_linked_tiles_on_side_streams_and_replayed(columns):
    """Two graphs captured on one stream and replayed side by side on others while the call runs eagerly on a third."""
    lb = _lb()
    _, T, D = COLUMNS[columns]
    cases = [_case((1, T, D), True, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [_run(c) for c in cases]
    stream, graphs = torch.cuda.Stream(), []
    for c in cases:
        dev = {k: v.to(DEV) for k, v in c.items()}
        leaves = [dev[k].requires_grad_(True) for k in NAMES]
        torch.cuda.synchronize()

        def step():
            y, final = lb.linrec_gated(leaves[0], leaves[1], input_gate=leaves[2], decay=leaves[3], initial_state=leaves[4], return_state=True)
            return [y, final, *torch.autograd.grad([y, final], leaves, [dev["dy"], dev["dfinal"]])]

        with torch.cuda.stream(stream):
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = step()
        graphs.append((graph, outs, dev, leaves))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = _run(cases[0])
    torch.cuda.synchronize()
    for w, (_, outs, *_) in zip(want, graphs):
        assert all(torch.equal(w[n], t) for n, t in zip(("y", "final", *NAMES.values()), outs))
    assert all(torch.equal(want[0][n], eager[n]) for n in eager)
    lb.check_status()


def test_scale_as_a_tensor():
    """A scale that is no Python number means the same to the step as to the scan."""
    lb = _lb()
    c = {k: v.to(DEV) for k, v in _case((3, 1, 64), True, torch.float32).items()}
    x, f, i = (c[k] for k in ("inputs", "forget", "input_gate"))
    want, end = lb.linrec_gated(x, f, input_gate=i, decay=c["decay"], decay_scale=4.0, initial_state=c["initial_state"], return_state=True)
    for scale in (4.0, 4, torch.tensor(4.0), np.float32(4.0)):
        state = c["initial_state"].clone()
        y = lb.linrec_gated_step(x[:, 0], f[:, 0], state, input_gate=i[:, 0], decay=c["decay"], decay_scale=scale)
        # one position: the same products, each rounded once, whichever kernel forms them (bound of the oracle below 1e-6)
        assert torch.allclose(y, want[:, 0], rtol=1e-5, atol=1e-6) and torch.allclose(state, end, rtol=1e-5, atol=1e-6)
