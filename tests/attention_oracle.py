"""The attention operators in 64 bits (numpy), with bounds on what their kernels
may differ by.

u is half a step of the kernels' type, eps / 2.  Bounds count roundings along the
longest chain of each result, so that they hold whatever order a sum takes.
"""
from __future__ import annotations

import numpy as np


def half_step(dtype) -> float:
    return float(np.finfo(dtype).eps) / 2


# ------------------------------------------------------------------ rotation

def frequencies(rotary, base=10000.0):
    return base ** (-2.0 * np.arange(rotary // 2) / rotary)


def pairs(rotary, layout):
    """Indices of the pairs' first and second elements."""
    if layout == "half":
        return np.arange(rotary // 2), np.arange(rotary // 2, rotary)
    return np.arange(0, rotary, 2), np.arange(1, rotary, 2)


def turn(x, positions, freq, layout, magnitude=1.0, inverse=False):
    """(turned heads, |a| + |b| of each element's pair times the magnitude): x is
    [batch, heads, tokens, extent], positions [tokens] or [batch, tokens]."""
    x = np.asarray(x, np.float64)
    positions = np.broadcast_to(np.asarray(positions), (x.shape[0], x.shape[2]))
    angle = (positions[:, None, :, None].astype(np.float64) * freq) * (-1 if inverse else 1)
    a, b = pairs(2 * len(freq), layout)
    y, size = x.copy(), np.abs(x)
    y[..., a] = magnitude * (x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle))
    y[..., b] = magnitude * (x[..., b] * np.cos(angle) + x[..., a] * np.sin(angle))
    size[..., a] = size[..., b] = abs(magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


# cos and sin: the reduced angle's rounding (1/2 u of a turn below 1), the
# function (2 steps: 4 u), the magnitude (u); then a product and the sum (2 u).
TURN = 8


def norm(x, weight, epsilon):
    x = np.asarray(x, np.float64)
    d = np.sqrt(np.mean(x * x, -1, keepdims=True) + epsilon)
    return x / d * weight, d


# Squares (u), their sum in a tree (3 additions in a lane, 6 between lanes), the
# quotient and epsilon: 12 u of d * d, 6 u of d; the root, 1 / d, and two products.
NORM = 10


def norm_backward(x, weight, gradient, epsilon):
    """(dx, dw, bound scale of dx, of dw) for the gradient before the rotation."""
    x, g = np.asarray(x, np.float64), np.asarray(gradient, np.float64)
    d = np.sqrt(np.mean(x * x, -1, keepdims=True) + epsilon)
    h = x / d
    gw = g * weight
    dx = (gw - h * np.mean(gw * h, -1, keepdims=True)) / d
    scale = (np.abs(gw) + np.abs(h) * np.mean(np.abs(gw * h), -1, keepdims=True)) / d
    axes = (0, 1, 2)
    return dx, (g * h).sum(axes), scale, np.abs(g * h).sum(axes)


# ----------------------------------------------------------------- attention

def visible(queries, keys, lengths, window, sinks):
    """[batch, queries, keys] of truth values."""
    lengths = np.clip(np.asarray(lengths, np.int64), 0, keys)
    p = (lengths[:, None] - queries + np.arange(queries))[:, :, None]
    j = np.arange(keys)
    seen = j <= p
    if window:
        seen = seen & ((p - j < window) | (j < sinks))
    return seen


class Attention:
    """Forward and backward with bounds for kernels of `dtype`.  query [batch,
    heads, queries, extent], key and value [batch, key heads, keys, extent]."""

    def __init__(self, query, key, value, window=0, sinks=0, scale=None, lengths=None,
                 dtype=np.float32):
        b, h, t, d = query.shape
        hk, s = key.shape[1], key.shape[2]
        self.group = h // hk
        self.u = half_step(dtype)
        self.scale = 1 / np.sqrt(d) if scale is None else scale
        lengths = [s] * b if lengths is None else lengths
        self.seen = visible(t, s, lengths, window, sinks)[:, None]
        # what no query sees has no part, whatever it holds
        used = np.broadcast_to(self.seen.any((1, 2))[:, None, :, None], key.shape)
        self.q = np.where(self.seen.any(-1)[..., None], np.asarray(query, np.float64), 0.0)
        self.k = np.repeat(np.where(used, np.asarray(key, np.float64), 0.0), self.group, 1)
        self.v = np.repeat(np.where(used, np.asarray(value, np.float64), 0.0), self.group, 1)
        scores = np.where(self.seen, self.scale * (self.q @ self.k.swapaxes(2, 3)), -np.inf)
        top = scores.max(-1, keepdims=True, initial=-np.inf)
        top = np.where(np.isneginf(top), 0.0, top)
        e = np.exp(scores - top)
        total = e.sum(-1, keepdims=True)
        self.p = e / np.where(total == 0, 1.0, total)
        with np.errstate(divide="ignore"):
            self.logsumexp = (top + np.log(total))[..., 0]
        self.output = self.p @ self.v
        # A score: its products and their sum (d u), the scale in q and log2(e) (3 u).
        # A weight: its score and the row's maximum or logsumexp, each as far off as a
        # score, and as far as u of itself; the exponential (4 u).
        score = abs(self.scale) * (np.abs(self.q) @ np.abs(self.k).swapaxes(2, 3))
        score = np.where(self.seen, score, 0.0).max(-1, keepdims=True, initial=0.0)
        self.weight = self.u * (2 * (d + 4) * score + 4 * score + s + 8)
        # sums over keys: a rounding each, and those of the waves' and parts' joining
        self.output_bound = (np.abs(self.p) @ np.abs(self.v)) * (
            2 * self.weight + self.u * (s + 32))
        self.logsumexp_bound = self.weight[..., 0] + 4 * self.u * np.abs(
            np.where(np.isfinite(self.logsumexp), self.logsumexp, 0.0))

    def backward(self, gradient):
        """dq, dk, dv and the bounds of each."""
        d = self.q.shape[-1]
        u = self.u
        g = np.where(self.seen.any(-1)[..., None], np.asarray(gradient, np.float64), 0.0)
        dp = g @ self.v.swapaxes(2, 3)
        delta = (g * self.output).sum(-1, keepdims=True)
        ds = self.p * (dp - delta)
        size = np.abs(g) @ np.abs(self.v).swapaxes(2, 3) + (
            np.abs(g) * np.abs(self.output)).sum(-1, keepdims=True)
        ds_bound = self.p * (2 * self.weight * np.abs(dp - delta) + u * (d + 8) * size
                             + (np.abs(g) * self.output_bound).sum(-1, keepdims=True))
        rows = self.q.shape[2] * self.group + 80  # a rounding each, and the parts' joining

        def grouped(x):  # sums over the heads of a group
            b, h, s, w = x.shape
            return x.reshape(b, h // self.group, self.group, s, w).sum(2)

        t = (0, 1, 3, 2)
        dq = self.scale * (ds @ self.k)
        dq_bound = abs(self.scale) * (ds_bound @ np.abs(self.k) + u * (self.k.shape[2] + 32) * (
            np.abs(ds) @ np.abs(self.k)))
        dk = self.scale * grouped(ds.transpose(t) @ self.q)
        dk_bound = abs(self.scale) * grouped(
            ds_bound.transpose(t) @ np.abs(self.q)
            + u * rows * (np.abs(ds).transpose(t) @ np.abs(self.q)))
        dv = grouped(self.p.transpose(t) @ g)
        dv_bound = grouped((self.p * 2 * self.weight).transpose(t) @ np.abs(g)
                           + u * rows * (self.p.transpose(t) @ np.abs(g)))
        return (dq, dk, dv), (dq_bound, dk_bound, dv_bound)


def assert_within(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, f"{what}: shape {got.shape} != {want.shape}"
    tiny = np.finfo(np.float32).tiny
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        ok = same | (np.abs(got - want) <= bound + tiny)
    if not ok.all():
        i = np.unravel_index(np.flatnonzero(~ok.ravel())[0], got.shape)
        raise AssertionError(f"{what}: {int((~ok).sum())} of {got.size} off; first at {i}: got "
                             f"{got[i]!r} want {want[i]!r} bound {np.broadcast_to(bound, got.shape)[i]!r}")
