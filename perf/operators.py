"""Cases, inputs and plain forms of the gated recurrence operators and of the group norm that follows them.

    linrec_gated        h[t] = a[t] * h[t-1] + b[t] * u[t] along the sequence of channels-last tensors, with
                        gates computed from logits, packed sequences, carried states, and its backward pass
    linrec_gated_step   the same recurrence for one token of each sequence on a state cache updated in place
    group_norm_act      group norm over channels-last tensors, with an activation or an activated gate

`run` computes an operator in elementary torch operations (32 bits inside, one rounding at the end) unless the
module's `own` is set, where it calls the operators of this package.  `exact` is the definition in 64 bits.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SCALE = 8.0
_EPS = 1e-5


def listed():
    return [
        # decode of a handful of sequences, every row its own state: latency counts
        {"name": "step 4x2048", "op": "step", "form": "forget", "dtype": "bf16", "rows": 4, "D": 2048, "slots": 0, "pads": 0},
        # a full serving batch against a larger state cache, padded to the captured batch size
        {"name": "step 512x8192 slots", "op": "step", "form": "decay", "dtype": "bf16", "rows": 512, "D": 8192, "slots": 768, "pads": 7},
        # two short prompts: latency of the scan itself
        {"name": "scan 2x16x512", "op": "scan", "form": "forget", "dtype": "fp16", "B": 2, "T": 16, "D": 512, "train": False, "state": True, "reverse": False},
        # prefill of one long document: few columns, the sequence has to supply the parallelism
        {"name": "scan 1x32768x2048", "op": "scan", "form": "decay", "dtype": "bf16", "B": 1, "T": 32768, "D": 2048, "train": False, "state": True, "reverse": False},
        # an ordinary training step
        {"name": "train 4x2048x2048", "op": "scan", "form": "forget", "dtype": "bf16", "B": 4, "T": 2048, "D": 2048, "train": True, "state": False, "reverse": False},
        # training on packed documents of very different lengths, with unused rows at the end of the buffer
        {"name": "train packed 16384x4096", "op": "packed", "form": "decay", "dtype": "bf16", "N": 16384, "S": 61, "tail": 37, "D": 4096, "train": True, "state": True, "reverse": False},
        # odd sizes in 32 bits, scanned backwards (the second half of a bidirectional layer)
        {"name": "train 3x1001x1001 reverse", "op": "scan", "form": "forget", "dtype": "fp32", "B": 3, "T": 1001, "D": 1001, "train": True, "state": True, "reverse": True},
        # a large training step
        {"name": "train 8x4096x4096", "op": "scan", "form": "decay", "dtype": "bf16", "B": 8, "T": 4096, "D": 4096, "train": True, "state": False, "reverse": False},
        # the norm behind a decode step: one position of each sequence, heads as groups
        {"name": "norm 16x2048 gate", "op": "norm", "dtype": "bf16", "N": 16, "L": 1, "C": 2048, "G": 16, "gate": True, "act": "silu", "train": False},
        # the norm behind the recurrence of a training step: every position has its own statistics
        {"name": "norm train 16384x4096 gate", "op": "norm", "dtype": "bf16", "N": 16384, "L": 1, "C": 4096, "G": 32, "gate": True, "act": "silu", "train": True},
        # statistics over a whole sequence (encoders), no gate
        {"name": "norm train 4x4096x1024", "op": "norm", "dtype": "bf16", "N": 4, "L": 4096, "C": 1024, "G": 32, "gate": False, "act": "silu", "train": True},
        # odd sizes in 32 bits
        {"name": "norm 5x333x1002", "op": "norm", "dtype": "fp32", "N": 5, "L": 333, "C": 1002, "G": 6, "gate": True, "act": "sigmoid", "train": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["step", "scan", "packed", "norm", "scan", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    most = 8 * 4096 * 4096 // (2 if dtype == "fp32" else 1)
    if op == "step":
        rows = _log_int(rng, 1, 512)
        slots = 0 if rng.random() < 0.4 else rows + _log_int(rng, 1, 512)
        return {"op": op, "form": rng.choice(["forget", "decay"]), "dtype": dtype, "rows": rows, "D": _log_int(rng, 64, 8192),
                "slots": slots, "pads": 0 if not slots else rng.randint(0, rows // 4)}
    if op == "norm":
        per_position = rng.random() < 0.5
        G = _log_int(rng, 1, 64)
        # groups of a few elements normalise to almost nothing but rounding: none smaller than 16 elements
        c = _log_int(rng, 16 if per_position else 1, 256)
        C = G * c if rng.random() < 0.7 else G * (8 * max(1, c // 8))
        train = rng.random() < 0.6
        if per_position:
            N, L = _log_int(rng, 1, min(32768, most // (2 * C))), 1
        else:
            L = _log_int(rng, 16, min(8192, most // (4 * C)))
            N = _log_int(rng, 1, min(64, max(1, most // (4 * C * L))))
        return {"op": op, "dtype": dtype, "N": N, "L": L, "C": C, "G": G, "gate": rng.random() < 0.5,
                "act": rng.choice(["silu", "silu", "sigmoid", "none"]), "train": train}
    D = _log_int(rng, 64, 4096)
    if rng.random() < 0.6:
        D = max(64, D // 16 * 16)
    common = {"form": rng.choice(["forget", "decay"]), "dtype": dtype, "D": D, "train": rng.random() < 0.6,
              "state": rng.random() < 0.5, "reverse": rng.random() < 0.3}
    if op == "scan":
        T = _log_int(rng, 1, min(32768, most // (2 * D)))
        B = _log_int(rng, 1, max(1, min(32, most // (2 * D * T))))
        return {"op": op, "B": B, "T": T, **common}
    N = _log_int(rng, 64, min(32768, most // (2 * D)))
    return {"op": op, "N": N, "S": _log_int(rng, 1, max(1, N // 8)), "tail": rng.choice([0, 0, rng.randint(1, 1 + N // 8)]), **common}


# ---- inputs ------------------------------------------------------------------------------------------
def _offsets(case, seed):
    """Sequence offsets: uneven lengths, an empty sequence now and then, `tail` rows that belong to none."""
    if case["op"] == "scan":
        return [b * case["T"] for b in range(case["B"] + 1)]
    r = random.Random(seed * 7919 + 13)
    used = case["N"] - case["tail"]
    w = [math.exp(r.gauss(0.0, 1.0)) if r.random() > 0.03 else 0.0 for _ in range(case["S"])]
    total, acc, offs = sum(w) or 1.0, 0.0, [0]
    for v in w:
        acc += v
        offs.append(min(used, int(round(used * acc / total))))
    offs[-1] = used
    return offs


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    dt = _DT[case["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=dev).to(dtype)

    s = SimpleNamespace(case=dict(case))
    if case["op"] == "norm":
        N, L, C = case["N"], case["L"], case["C"]
        shape = (N, C) if L == 1 else (N, L, C)
        s.x = (randn(*shape) + 0.5 * randn(C)).to(dt)
        s.weight, s.bias = 1.0 + 0.2 * randn(C), 0.2 * randn(C)
        s.gate = randn(*shape, dtype=dt) if case["gate"] else None
        s.dy = randn(*shape, dtype=dt) if case["train"] else None
        if case["train"]:
            for t in (s.x, s.weight, s.bias, s.gate):
                if t is not None:
                    t.requires_grad_(True)
        return s

    D, decay = case["D"], case["form"] == "decay"
    s.decay = None
    if decay:
        # a per-channel decay between 0.9 and 0.999 where the recurrence gate is open
        a = 0.9 + 0.099 * torch.rand(D, generator=g, device=dev)
        s.decay = torch.log(torch.expm1(-torch.log(a) / _SCALE))
        centre = torch.zeros(D, device=dev)
    else:
        # forget gates between about 0.5 and 0.998
        centre = 6.0 * torch.rand(D, generator=g, device=dev)
    if case["op"] == "step":
        rows, slots = case["rows"], case["slots"]
        s.x = randn(rows, D, dtype=dt)
        s.forget = (centre + randn(rows, D)).to(dt)
        s.input_gate = randn(rows, D, dtype=dt) if decay else None
        s.state = randn(slots or rows, D)
        s.slots = None
        if slots:
            index = torch.randperm(slots, generator=g, device=dev)[:rows]
            if case["pads"]:
                index[-case["pads"]:] = -1
            s.slots = index.to(torch.int32)
        return s

    packed = case["op"] == "packed"
    offs = _offsets(case, seed)
    S = len(offs) - 1
    shape = (case["N"], D) if packed else (case["B"], case["T"], D)
    s.x = randn(*shape, dtype=dt)
    s.forget = (centre + randn(*shape)).to(dt)
    s.input_gate = randn(*shape, dtype=dt) if decay else None
    s.initial = randn(S, D) if case["state"] else None
    s.cu = torch.tensor(offs, dtype=torch.int32, device=dev) if packed else None
    s.dy = randn(*shape, dtype=dt) if case["train"] else None
    s.dfinal = randn(S, D) if case["train"] and case["state"] else None
    if case["train"]:
        for t in (s.x, s.forget, s.input_gate, s.decay, s.initial):
            if t is not None:
                t.requires_grad_(True)
    # rows of the flattened (rows, D) view in scan order, for the plain form
    n = s.x.numel() // D
    full = [q for q in range(S) if offs[q + 1] > offs[q]]
    first = [offs[q] if not case["reverse"] else n - offs[q + 1] for q in full]
    last = [offs[q + 1] - 1 if not case["reverse"] else n - 1 - offs[q] for q in full]
    s.offsets, s.longest = offs, max([offs[q + 1] - offs[q] for q in full], default=0)
    s.full, s.first, s.last = (torch.tensor(v, dtype=torch.long, device=dev) for v in (full, first, last))
    inside = torch.zeros(n, 1, device=dev)
    inside[offs[0]:offs[-1]] = 1.0
    s.inside = inside.flip(0) if case["reverse"] else inside
    return s


# ---- plain forms -------------------------------------------------------------------------------------
def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _gates(x, f, i, lam):
    """Multiplier a, input factor b, gated input u, all in 32 bits; for the decay form also log a and the gates."""
    if lam is None:
        return torch.sigmoid(f), torch.sigmoid(-f), x, None, None, None
    r, g = torch.sigmoid(f), torch.sigmoid(i)
    la = -_SCALE * _softplus(lam) * r
    return torch.exp(la), torch.sqrt(-torch.expm1(2.0 * la)), g * x, la, r, g


def _scan(a, v, longest):
    """All h[t] = a[t] h[t-1] + v[t] down the rows by doubling; a is zero where a sequence starts."""
    d = 1
    while d < longest:
        shifted = v[:-d] * a[d:]
        product = a[:-d] * a[d:]
        v, a = v.clone(), a.clone()
        v[d:] += shifted
        a[d:] = product
        d *= 2
    return v


def _plain_scan(s):
    case = s.case
    D, dt, rev = case["D"], s.x.dtype, case["reverse"]

    def rows(t):
        if t is None:
            return None
        t = t.detach().reshape(-1, D).float()
        return t.flip(0) if rev else t

    def back(t):
        t = t.flip(0) if rev else t
        return t.to(dt).reshape(s.x.shape)

    x, f, i = rows(s.x), rows(s.forget), rows(s.input_gate)
    lam = None if s.decay is None else s.decay.detach().float()
    h0 = None if s.initial is None else s.initial.detach()
    a, b, u, la, r, g = _gates(x, f, i, lam)
    a, b = a * s.inside, b * s.inside
    carry, v = a.clone(), b * u
    carry[s.first] = 0.0
    if h0 is not None:
        v[s.first] += a[s.first] * h0[s.full]
    h = _scan(carry, v, s.longest)
    final = None
    if h0 is not None:
        final = h0.clone()
        final[s.full] = h[s.last]
    if not case["train"]:
        return {"y": back(h), "final": final}

    # adjoint: w[t] = dy[t] + a[t+1] w[t+1], back to front
    dy = rows(s.dy)
    if s.dfinal is not None:
        dy[s.last] += s.dfinal[s.full]
    shifted = torch.zeros_like(carry)
    shifted[:-1] = carry[1:]
    w = _scan(shifted.flip(0), dy.flip(0), s.longest).flip(0) * s.inside
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[s.first] = 0.0 if h0 is None else h0[s.full]
    out = {"y": back(h), "final": final, "dx": None, "dforget": None, "dinput": None, "ddecay": None, "dinitial": None}
    if lam is None:
        out["dx"] = back(w * b)
        out["dforget"] = back(w * a * b * (before - x))
    else:
        dla = w * (a * before - u * a * a / torch.where(b > 0, b, torch.ones_like(b)))
        out["dx"] = back(w * b * g)
        out["dinput"] = back(w * b * x * g * torch.sigmoid(-i))
        out["dforget"] = back(dla * la * torch.sigmoid(-f))
        out["ddecay"] = ((dla * -_SCALE * r).double().sum(0) * torch.sigmoid(lam).double()).float()
    if h0 is not None:
        d0 = s.dfinal.clone()
        d0[s.full] = (a * w)[s.first]
        out["dinitial"] = d0
    return out


def _plain_step(s):
    x, f = s.x.float(), s.forget.float()
    i = None if s.input_gate is None else s.input_gate.float()
    a, b, u, _, _, _ = _gates(x, f, i, s.decay)
    if s.slots is None:
        s.state.copy_(a * s.state + b * u)
        return {"y": s.state.to(s.x.dtype), "state": s.state}
    keep = s.slots >= 0
    at = s.slots.long().clamp(min=0)
    h = (a * s.state[at] + b * u) * keep[:, None]
    # rows that stand for padding write to a row behind the cache
    grown = torch.cat([s.state, s.state[:1]])
    grown[torch.where(keep, at, torch.full_like(at, s.state.shape[0]))] = h
    s.state.copy_(grown[:-1])
    return {"y": h.to(s.x.dtype), "state": s.state}


def _act(kind, v):
    """The activation and its derivative."""
    if kind == "none":
        return v, torch.ones_like(v)
    p = torch.sigmoid(v)
    if kind == "sigmoid":
        return p, p * (1.0 - p)
    return v * p, p * (1.0 + v * (1.0 - p))


def _plain_norm(s):
    case = s.case
    N, L, C, G = case["N"], case["L"], case["C"], case["G"]
    dt, shape = s.x.dtype, (N, L, G, C // G)
    x = s.x.detach().float().reshape(shape)
    w, bias = s.weight.detach().reshape(1, 1, G, -1), s.bias.detach().reshape(1, 1, G, -1)
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    inv = torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + _EPS)
    xhat = centred * inv
    z = xhat * w + bias
    if s.gate is None:
        y, dz = _act(case["act"], z)
    else:
        gate = s.gate.detach().float().reshape(shape)
        dz, slope = _act(case["act"], gate)
        y = z * dz
    out = {"y": y.to(dt).reshape(s.x.shape)}
    if not case["train"]:
        return out
    dy = s.dy.float().reshape(shape)
    if s.gate is not None:
        out["dgate"] = (dy * z * slope).to(dt).reshape(s.x.shape)
    dz = dy * dz
    dxhat = dz * w
    m1 = dxhat.mean((1, 3), keepdim=True)
    m2 = (dxhat * xhat).mean((1, 3), keepdim=True)
    out["dx"] = (inv * (dxhat - m1 - xhat * m2)).to(dt).reshape(s.x.shape)
    out["dweight"] = (dz * xhat).sum((0, 1), dtype=torch.float64).float().reshape(-1)
    out["dbias"] = dz.sum((0, 1), dtype=torch.float64).float().reshape(-1)
    return out


# ---- the framework's operators -----------------------------------------------------------------------
def _own_scan(s):
    import linrec_b200 as lb
    case = s.case
    kw = {"input_gate": s.input_gate, "decay": s.decay, "decay_scale": _SCALE, "initial_state": s.initial,
          "cu_seqlens": s.cu, "reverse": case["reverse"], "return_state": case["state"]}
    if not case["train"]:
        r = lb.linrec_gated(s.x, s.forget, **kw)
        y, final = r if case["state"] else (r, None)
        return {"y": y, "final": final}
    r = lb.linrec_gated(s.x, s.forget, **kw)
    y, final = r if case["state"] else (r, None)
    names = ["dx", "dforget", "dinput", "ddecay", "dinitial"]
    leaves = [s.x, s.forget, s.input_gate, s.decay, s.initial]
    asked = [(n, t) for n, t in zip(names, leaves) if t is not None]
    outs, douts = ((y, final), (s.dy, s.dfinal)) if case["state"] else ((y,), (s.dy,))
    grads = torch.autograd.grad(outs, [t for _, t in asked], douts)
    out = {"y": y.detach(), "final": None if final is None else final.detach(), **dict.fromkeys(names)}
    out.update({n: d for (n, _), d in zip(asked, grads)})
    return out


def _own_step(s):
    import linrec_b200 as lb
    y = lb.linrec_gated_step(s.x, s.forget, s.state, input_gate=s.input_gate, decay=s.decay, decay_scale=_SCALE, slots=s.slots)
    return {"y": y, "state": s.state}


def _own_norm(s):
    import linrec_b200 as lb
    case = s.case
    act = None if case["act"] == "none" else case["act"]
    y = lb.group_norm_act(s.x, case["G"], s.weight, s.bias, gate=s.gate, activation=act, eps=_EPS)
    if not case["train"]:
        return {"y": y}
    asked = [("dx", s.x), ("dweight", s.weight), ("dbias", s.bias)] + ([("dgate", s.gate)] if case["gate"] else [])
    grads = torch.autograd.grad(y, [t for _, t in asked], s.dy)
    return {"y": y.detach(), **{n: d for (n, _), d in zip(asked, grads)}}


def run(state):
    op = state.case["op"]
    if own:
        return _own_step(state) if op == "step" else _own_norm(state) if op == "norm" else _own_scan(state)
    return _plain_step(state) if op == "step" else _plain_norm(state) if op == "norm" else _plain_scan(state)


# ---- cost --------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["N"] * case["L"] * case["C"]
        arrays = 2 + case["gate"] + (2 + case["gate"] if case["train"] else 0)
        return {"bytes": n * size * arrays + case["C"] * 4 * (4 if case["train"] else 2), "flops": n * (45 if case["train"] else 15)}
    D, decay = case["D"], case["form"] == "decay"
    if case["op"] == "step":
        n = case["rows"] * D
        live = (case["rows"] - case["pads"]) * D
        return {"bytes": n * size * (4 if decay else 3) + live * 8, "flops": n * (25 if decay else 12)}
    n = case["N"] * D if case["op"] == "packed" else case["B"] * case["T"] * D
    S = case["S"] if case["op"] == "packed" else case["B"]
    inputs = 3 if decay else 2
    arrays = inputs + 1 + (1 + inputs if case["train"] else 0)
    states = (2 + (2 if case["train"] else 0)) * S * D * 4 if case["state"] else 0
    return {"bytes": n * size * arrays + states, "flops": n * ((25 if decay else 12) + (60 if decay else 30) * case["train"])}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _exact_scan(case, s):
    """One position after the other; the sequences of a batch of equal lengths side by side, packed ones in turn."""
    D, B = case["D"], case.get("B", 1)
    f64 = lambda t: None if t is None else t.detach().double().reshape(B, -1, D)  # noqa: E731
    x, f, i, dy = f64(s.x), f64(s.forget), f64(s.input_gate), f64(s.dy)
    T = x.shape[1]
    if s.decay is None:
        a = 1.0 / (1.0 + torch.exp(-f))
        b, u = 1.0 / (1.0 + torch.exp(f)), x
    else:
        lam = s.decay.detach().double()
        speed = torch.log1p(torch.exp(-lam.abs())) + lam.clamp(min=0.0)
        rate = 1.0 / (1.0 + torch.exp(-f))
        gate = 1.0 / (1.0 + torch.exp(-i))
        la = -_SCALE * speed * rate
        a, b, u = torch.exp(la), torch.sqrt(-torch.expm1(2.0 * la)), gate * x
    runs = [(0, T)] if case["op"] == "scan" else list(zip(s.offsets[:-1], s.offsets[1:]))
    S = len(s.offsets) - 1
    h0 = None if s.initial is None else s.initial.detach().double()
    final = None if h0 is None else h0.clone()
    at = (lambda q: slice(0, B)) if case["op"] == "scan" else (lambda q: slice(q, q + 1))
    y, prev = torch.zeros_like(x), torch.zeros_like(x)
    v = b * u
    for q, (lo, hi) in enumerate(runs):
        if hi == lo:
            continue
        h = torch.zeros(B, D, dtype=torch.float64, device=x.device) if h0 is None else h0[at(q)].clone()
        for t in (range(hi - 1, lo - 1, -1) if case["reverse"] else range(lo, hi)):
            prev[:, t] = h
            h = torch.addcmul(v[:, t], a[:, t], h)
            y[:, t] = h
        if final is not None:
            final[at(q)] = h
    if not case["train"]:
        return {"y": y.reshape(s.x.shape), "final": final}
    dfinal = None if s.dfinal is None else s.dfinal.double()
    d0 = None if dfinal is None else dfinal.clone()
    w = torch.zeros_like(x)
    for q, (lo, hi) in enumerate(runs):
        if hi == lo:
            continue
        c = torch.zeros(B, D, dtype=torch.float64, device=x.device) if dfinal is None else dfinal[at(q)].clone()
        for t in (range(lo, hi) if case["reverse"] else range(hi - 1, lo - 1, -1)):
            c = c + dy[:, t]
            w[:, t] = c
            c = c * a[:, t]
        if d0 is not None:
            d0[at(q)] = c
    shape = s.x.shape
    out = {"y": y.reshape(shape), "final": final, "dx": None, "dforget": None, "dinput": None, "ddecay": None, "dinitial": d0}
    if s.decay is None:
        out["dx"] = (w * b).reshape(shape)
        out["dforget"] = (w * (prev - x) * a * (1.0 - a)).reshape(shape)
        return out
    slope_b = torch.where(b > 0, a * a / b, torch.zeros_like(b))
    dla = w * prev * a - w * u * slope_b
    out["dx"] = (w * b * gate).reshape(shape)
    out["dinput"] = (w * b * x * gate * (1.0 - gate)).reshape(shape)
    out["dforget"] = (dla * la * (1.0 - rate)).reshape(shape)
    out["ddecay"] = (dla * rate).sum((0, 1)) * -_SCALE / (1.0 + torch.exp(-lam))
    return out


def _exact_norm(case, s):
    N, L, C, G = case["N"], case["L"], case["C"], case["G"]
    x = s.x.detach().double().reshape(N, L, G, C // G).permute(0, 2, 1, 3).reshape(N, G, -1)
    var, mean = torch.var_mean(x, dim=2, correction=0, keepdim=True)
    inv = 1.0 / torch.sqrt(var + _EPS)
    xhat = (x - mean) * inv
    lay = lambda t: t.reshape(N, L, G, C // G).permute(0, 2, 1, 3).reshape(N, G, -1)  # noqa: E731
    unlay = lambda t: t.reshape(N, G, L, C // G).permute(0, 2, 1, 3).reshape(s.x.shape)  # noqa: E731
    w = lay(s.weight.detach().double().expand(N, L, C))
    z = xhat * w + lay(s.bias.detach().double().expand(N, L, C))
    src = z if s.gate is None else lay(s.gate.detach().double())
    sig = 1.0 / (1.0 + torch.exp(-src))
    value = {"none": src, "sigmoid": sig, "silu": src * sig}[case["act"]]
    slope = {"none": torch.ones_like(src), "sigmoid": sig * (1.0 - sig), "silu": sig + src * sig * (1.0 - sig)}[case["act"]]
    out = {"y": unlay(value if s.gate is None else z * value)}
    if not case["train"]:
        return out
    dy = lay(s.dy.double())
    if s.gate is None:
        dz = dy * slope
    else:
        dz, out["dgate"] = dy * value, unlay(dy * z * slope)
    k = dz * w
    out["dx"] = unlay((k - k.mean(2, keepdim=True) - xhat * (k * xhat).mean(2, keepdim=True)) * inv)
    out["dweight"] = unlay(dz * xhat).reshape(-1, C).sum(0)
    out["dbias"] = unlay(dz).reshape(-1, C).sum(0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["op"] != "step":
        return _exact_scan(case, s)
    f = s.forget.double()
    if s.decay is None:
        a, v = 1.0 / (1.0 + torch.exp(-f)), s.x.double() / (1.0 + torch.exp(f))
    else:
        lam = s.decay.double()
        la = -_SCALE * (torch.log1p(torch.exp(-lam.abs())) + lam.clamp(min=0.0)) / (1.0 + torch.exp(-f))
        a, v = torch.exp(la), torch.sqrt(-torch.expm1(2.0 * la)) * s.x.double() / (1.0 + torch.exp(-s.input_gate.double()))
    state, y = s.state.double(), torch.zeros_like(a)
    for row, slot in enumerate(range(a.shape[0]) if s.slots is None else s.slots.tolist()):
        if slot >= 0:
            state[slot] = a[row] * state[slot] + v[row]
            y[row] = state[slot]
    return {"y": y, "state": state}
