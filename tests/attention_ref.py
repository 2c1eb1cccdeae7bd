"""Attention in float64 with its gradients, and per-element bounds on what a
float32 computation of it may be off by."""
import math

import numpy as np

U = 2.0 ** -24  # half a step of float32, relative
# A product of two float32 operands that are each cut into two float16 parts
# (the first two of their bits' three groups of products are kept): each part
# is cut off at 11 bits, so an operand is off by at most 2^-21 of itself and
# the product of the two second parts, 2^-20 of the whole, is left out.
ETA = 2.0 ** -19
# The second part has no bits below 2^-40 of the largest operand of its block,
# 2^-19 of which times ETA covers it.
FLOOR = 2.0 ** -20


def heads_of(x, batch, heads):
    n, c = x.shape
    return x.reshape(batch, n // batch, heads, c // heads).transpose(0, 2, 1, 3).astype(np.float64)


def rows_of(x):
    b, h, n, d = x.shape
    return x.transpose(0, 2, 1, 3).reshape(b * n, h * d)


def visible(batch, sq, sk, causal, lengths):
    i, j = np.arange(sq)[:, None], np.arange(sk)[None, :]
    seen = np.broadcast_to(j < (np.full(batch, sk) if lengths is None else np.clip(lengths, 0, sk))[:, None, None, None],
                           (batch, 1, sq, sk))
    return seen & (j <= i + sk - sq) if causal else seen


def attention(q, k, v, batch, heads, kv_heads, causal=False, lengths=None, scale=None, g=None):
    """{"y", and with g "dq", "dk", "dv"}: (value, bound) pairs of matrices."""
    sq, sk, group = q.shape[0] // batch, k.shape[0] // batch, heads // kv_heads
    q = heads_of(q, batch, heads)
    d = q.shape[3]
    scale = d ** -0.5 if scale is None else float(np.float32(scale))
    seen = visible(batch, sq, sk, causal, lengths)
    # What a hidden key holds never matters.
    live = np.broadcast_to(seen.any(axis=2)[:, :, :, None] if not causal else
                           visible(batch, sq, sk, False, lengths).any(axis=2)[:, :, :, None], (batch, 1, sk, 1))
    k, v = (np.where(np.repeat(live, heads, 1), np.repeat(heads_of(x, batch, kv_heads), group, 1), 0.0) for x in (k, v))

    def mag(x):  # an operand's magnitude with the part of its block's largest that its error is at most ETA of
        return np.abs(x) + FLOOR * np.abs(x).max()

    t = lambda x: x.transpose(0, 1, 3, 2)  # noqa: E731
    eta = ETA + (d + 4) * U
    s = np.where(seen, q @ t(k) * scale, -np.inf)
    top = np.where(seen.any(3, keepdims=True), s.max(3, keepdims=True), 0.0)
    e = np.exp(s - top)
    total = e.sum(3, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    # exp's argument is off by its product's error (and the maximum's, the same
    # for the whole row, is made up for by the sum) and by the roundings of
    # arguments up to |s|; exp2 itself by 2^-22.
    ds_abs = eta * scale * (mag(q) @ t(mag(k))) + 4 * U * np.where(seen, np.abs(q @ t(k)) * scale + np.abs(top), 0.0) + 2.0 ** -21
    rho = 2 * np.where(seen, ds_abs, 0.0).max(3, keepdims=True) + (sk + 8) * U + ETA
    pm = np.where(seen, p + 2.0 ** -13 / np.where(total == 0, 1.0, total), 0.0)
    y = p @ v
    yb = (pm * rho) @ mag(v) + (eta + sk * U) * (pm @ mag(v)) + 1e-38
    out = {"y": (rows_of(y), rows_of(yb))}
    if g is None:
        return out
    g = heads_of(g, batch, heads)
    dp = g @ t(v)
    delta = (g * y).sum(3, keepdims=True)
    ds = p * (dp - delta)
    # The scores' gradient keeps 2^-38 of the largest it could have been.
    worst = d * np.abs(g).max() * np.abs(v).max()
    dsb = (pm * rho) * (np.abs(dp) + np.abs(delta)) + pm * (
        eta * (mag(g) @ t(mag(v))) + eta * (np.abs(g) * np.abs(y)).sum(3, keepdims=True) +
        (np.abs(g) * yb).sum(3, keepdims=True)) + np.where(seen, 2.0 ** -38 * worst, 0.0)
    dsm = np.abs(ds) + dsb
    dv = t(p) @ g
    dvb = t(pm * rho) @ mag(g) + (eta + group * sq * U) * (t(pm) @ mag(g))
    dq, dk = ds @ k * scale, t(ds) @ q * scale
    dqb = (dsb @ mag(k) + (eta + sk * U) * (dsm @ mag(k))) * scale
    dkb = (t(dsb) @ mag(q) + (eta + group * sq * U) * (t(dsm) @ mag(q))) * scale

    def fold(x):  # the heads that share a key head
        return rows_of(x.reshape(batch, kv_heads, group, sk, d).sum(2))

    out["dq"] = rows_of(dq), rows_of(dqb) + 1e-38
    out["dk"] = fold(dk), fold(dkb) + 1e-38
    out["dv"] = fold(dv), fold(dvb) + 1e-38
    return out
