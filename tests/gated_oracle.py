"""Oracle of the gated recurrence: one position after the other in 64 bits, and beside every result a bound
on the error of a float32 evaluation, carried along by the same recurrence.

With u = 2^-24 and all quantities relative: logistic values, exp, reciprocal and square root are taken as
within 6u; log a (product of three factors, one of them a softplus) as within 12u, which reaches a = exp(log a)
multiplied by |log a|; b = sqrt(1 - a^2) as within 40u (where the difference is taken, a^2/(1 - a^2) <= 3.6
and a is off by less than 8u there: 2 * 8 * 3.6 / 2 + the rounding of the difference < 40).
Operands of 16 bits are evaluated with exp(v) = 2^(v log2 e): rounding the product and the constant puts
1.3 |v| u on top of 4u of the power, so that logistic values are within (8 + 1.3 |v|) u there (a value next
to one: its distance from one is).  Whatever order
the products and sums of a scan are taken in, a contribution that travels n positions meets at most 2n
roundings, i.e. 2u per position on top of the error of a.
"""
import numpy as np

U = 2.0 ** -24


def logistic(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def softplus(v):
    return np.log1p(np.exp(-np.abs(v))) + np.maximum(v, 0.0)


def gates(x, f, i, decay, scale, fast=False):
    """a, b, u, log a, s(f), s(i) and the relative errors of a and of b * u."""
    k = 1.3 if fast else 0.0
    with np.errstate(over="ignore"):
        ef = (8 + k * np.abs(f)) * U if fast else 6 * U + 0 * f
        if decay is None:
            return logistic(f), logistic(-f), x, None, logistic(f), None, 2 * U + ef * np.minimum(1.0, np.exp(-f)), ef + 8 * U
        la = -scale * softplus(decay) * logistic(f)
        a = np.exp(la)
        # (the series gives 1 - a, which counts as much as 1 - a is of a, at most 1.3 |log a| below 1/4)
        ea = (5 + 1.3 * (12 + k * np.abs(f)) * np.abs(la)) * U
        eb = 40 * U + (k * np.abs(f) + k * np.abs(la)) * U
        return a, np.sqrt(-np.expm1(2 * la)), logistic(i) * x, la, logistic(f), logistic(i), ea, eb + (12 + k * np.abs(i)) * U


def runs_of(shape, offsets, reverse):
    """[(sequence, rows in scan order)] over the flattened rows."""
    if offsets is None:
        T = shape[-2]
        n = int(np.prod(shape[:-2]))
        spans = [(q * T, (q + 1) * T) for q in range(n)]
    else:
        spans = list(zip(offsets[:-1], offsets[1:]))
    return [(q, list(range(lo, hi))[::-1] if reverse else list(range(lo, hi))) for q, (lo, hi) in enumerate(spans)]


def evaluate(x, f, i=None, decay=None, scale=8.0, h0=None, offsets=None, reverse=False, dy=None, dfinal=None, fast=False):
    """dict name -> (value, bound); x, f, i, dy as (..., T, D) or (rows, D) float64 arrays; fast: the
    operands were of 16 bits."""
    shape, D = x.shape, x.shape[-1]
    flat = lambda t: None if t is None else np.asarray(t, np.float64).reshape(-1, D)
    x, f, i, dy, h0, dfinal = (flat(t) for t in (x, f, i, dy, h0, dfinal))
    a, b, u, la, rate, gate, ea, ev = gates(x, f, i, decay, scale, fast)
    k13 = 1.3 * U if fast else 0.0
    elog = lambda t: 10 * U + k13 * np.abs(t)      # of s(t) and s(-t)
    v = b * u
    runs = runs_of(shape, offsets, reverse)
    S = len(runs)
    zero = lambda: np.zeros_like(x)
    h, eh, big, prev, eprev, bprev = zero(), zero(), zero(), zero(), zero(), zero()
    final = np.zeros((S, D)) if h0 is None else h0.copy()
    efinal = np.zeros((S, D))
    for q, rows in runs:
        hv, e = final[q].copy(), np.zeros(D)
        m = np.abs(hv)
        for t in rows:
            prev[t], eprev[t], bprev[t] = hv, e, m
            hv = a[t] * hv + v[t]
            e = a[t] * (e + (ea[t] + 2 * U) * m) + ev[t] * np.abs(v[t])
            m = a[t] * m + np.abs(v[t])
            e = e + 2 * U * m
            h[t], eh[t], big[t] = hv, e, m
        final[q], efinal[q] = hv, e
    out = {"y": (h.reshape(shape), eh.reshape(shape)), "final": (final, efinal)}
    if dy is None and dfinal is None:
        return out
    dy = zero() if dy is None else dy
    w, ew, bw = zero(), zero(), zero()
    d0 = np.zeros((S, D)) if dfinal is None else dfinal.copy()
    ed0 = np.zeros((S, D))
    for q, rows in runs:
        c, e = d0[q].copy(), np.zeros(D)
        m = np.abs(c)
        for t in reversed(rows):
            c = c + dy[t]
            m = m + np.abs(dy[t])
            e = e + 2 * U * m
            w[t], ew[t], bw[t] = c, e, m
            c = a[t] * c
            e = a[t] * (e + (ea[t] + 2 * U) * m)
            m = a[t] * m
        d0[q], ed0[q] = c, e
    out["dinitial"] = (d0, ed0)
    if decay is None:
        k, ak = a * b, np.abs(bprev) + np.abs(x)
        out["dx"] = (w * b, b * (ew + (6 * U + elog(f)) * bw))
        out["dforget"] = (w * k * (prev - x), k * (ew * ak + bw * (eprev + (4 * U + 2 * elog(f)) * ak)))
    else:
        # a^2/b has the error of b and twice that of a
        sl = np.divide(a * a, b, out=np.zeros_like(b), where=b > 0)
        eb = ev + 2 * ea + 20 * U
        out["dx"] = (w * b * gate, b * gate * (ew + eb * bw))
        k = b * np.abs(x) * gate * (1 - gate)
        # 1 - s(i) is a difference: off by 6u s(i), i.e. by 6u relative to one
        out["dinput"] = (w * b * x * gate * (1 - gate), k * (ew + eb * bw) + elog(i) * bw * b * np.abs(x) * gate)
        mag = a * bprev + np.abs(u) * sl
        dla = w * (a * prev - u * sl)
        edla = ew * mag + bw * (a * eprev + eb * mag)
        low = logistic(-f)
        out["dforget"] = (dla * la * low, np.abs(la) * low * (edla + (20 * U + 2 * elog(f)) * bw * mag))
        L = logistic(decay)
        inside = np.zeros(len(x), bool)
        for _, rows in runs:
            inside[rows] = True
        terms, eterms = dla * rate, rate * (edla + (50 * U + elog(f)) * bw * mag)
        out["ddecay"] = (-scale * L * terms[inside].sum(0), scale * L * eterms[inside].sum(0))
    for n in ("dx", "dforget", "dinput"):
        if n in out:
            out[n] = tuple(t.reshape(shape) for t in out[n])
    return out
