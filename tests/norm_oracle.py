"""Oracle of the group norm in 64 bits, with a bound on the error of a float32 evaluation beside every result.

u = 2^-24.  A sum of n terms taken by threads and a tree is off by at most (32 + n/64) u times the sum of the
absolute terms: no thread adds more than n/64 of them one after the other, and the trees and shared-memory
passes above it add fewer than 32.  A variance may be formed from sums of squares about any element of the
same channel, so its error counts the squares of the largest distance from the channel's mean.  Logistic
values are within 6u, for 16-bit operands within (8 + 1.3 |v|) u, which 16u and 20u below cover for |v| < 6 and
half a step of the result's type by far beyond; slopes of activations are below 1.1, second slopes below 0.5.
"""
import numpy as np

from gated_oracle import U, logistic


def _act(kind, v):
    p = logistic(v)
    if kind is None:
        return v, np.ones_like(v)
    if kind == "sigmoid":
        return p, p * (1 - p)
    return v * p, p * (1 + v * (1 - p))


def evaluate(x, groups, w=None, b=None, gate=None, act="silu", eps=1e-5, dy=None, ex=None):
    """dict name -> (value, bound) for x (samples, ..., channels), all float64; ex: error that x carries already."""
    shape, C = x.shape, x.shape[-1]
    N, G = shape[0], groups
    lay = lambda t: np.asarray(t, np.float64).reshape(N, -1, G, C // G)
    x = lay(x)
    w = np.ones(C) if w is None else w
    b = np.zeros(C) if b is None else b
    W, Bi = w.reshape(1, 1, G, -1), b.reshape(1, 1, G, -1)
    n = x.shape[1] * x.shape[3]
    red = lambda t: t.mean((1, 3), keepdims=True)
    steps = (32 + n / 64) * U
    mean = red(x)
    far = np.abs(x - x.mean(1, keepdims=True)).max((1, 3), keepdims=True) + np.abs(x.mean(1, keepdims=True) - mean).max(3, keepdims=True)
    em = steps * red(np.abs(x))
    if ex is not None:
        em = em + red(lay(ex))
    d = x - mean
    var = red(d * d)
    inv = 1 / np.sqrt(var + eps)
    ed = em + U * (np.abs(x) + np.abs(mean)) + (0 if ex is None else lay(ex))
    big = ed.max((1, 3), keepdims=True)
    evar = steps * (var + far * far) + 2 * big * red(np.abs(d)) + big * big
    einv = evar / (2 * (var + eps)) * 1.5 + 8 * U
    xhat = d * inv
    exh = inv * ed + np.abs(xhat) * (einv + 4 * U)
    z = xhat * W + Bi
    ez = np.abs(W) * exh + 4 * U * (np.abs(W * xhat) + np.abs(Bi))
    out = {}
    back = lambda v, e: (v.reshape(shape), e.reshape(shape))
    if gate is None:
        v, s = _act(act, z)
        ev, es = 1.1 * ez + 16 * U * np.abs(v), 0.5 * ez + 16 * U * (1 + np.abs(z))
        out["y"] = back(v, ev)
    else:
        g = lay(gate)
        v, s = _act(act, g)
        ev, es = 16 * U * np.abs(v), 16 * U * (1 + np.abs(g)) * logistic(np.abs(g))
        out["y"] = back(z * v, np.abs(v) * ez + 20 * U * np.abs(z * v))
    if dy is None:
        return out
    dy = lay(dy)
    if gate is None:
        dz, edz = dy * s, np.abs(dy) * es + 2 * U * np.abs(dy * s)
    else:
        dz, edz = dy * v, np.abs(dy) * ev + 2 * U * np.abs(dy * v)
        out["dgate"] = back(dy * z * s, np.abs(dy) * (ez * np.abs(s) + np.abs(z) * es) + 4 * U * np.abs(dy * z * s))
    k, ek = dz * W, np.abs(W) * edz + 2 * U * np.abs(dz * W)
    m1, e1 = red(k), red(ek) + steps * red(np.abs(k))
    kx = k * xhat
    ekx = ek * np.abs(xhat) + np.abs(k) * exh + 2 * U * np.abs(kx)
    m2, e2 = red(kx), red(ekx) + steps * red(np.abs(kx))
    inner = k - m1 - xhat * m2
    mag = np.abs(k) + np.abs(m1) + np.abs(xhat * m2)
    ein = ek + e1 + np.abs(xhat) * e2 + exh * np.abs(m2) + 4 * U * mag
    out["dx"] = back(inv * inner, inv * (ein + (einv + 4 * U) * np.abs(inner)))
    rows = N * x.shape[1]
    far = (64 + rows / 16) * U
    t, et = dz * xhat, np.abs(xhat) * edz + np.abs(dz) * exh
    out["dweight"] = (t.sum((0, 1)).reshape(-1), (et + far * np.abs(t)).sum((0, 1)).reshape(-1))
    out["dbias"] = (dz.sum((0, 1)).reshape(-1), (edz + far * np.abs(dz)).sum((0, 1)).reshape(-1))
    return out
