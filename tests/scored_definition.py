"""Scored attention's definition in 64 bits, all rows of a sequence at once, with
the error that f32 arithmetic may make (the derivation of test_gpu_scored, whose
constants these are). What a row does not see enters neither its result nor its
bound."""

from __future__ import annotations

import math

import numpy as np

from test_gpu_scored import BLOCK, H, SIGMA

# Half a step of the rows' type; f16 and bf16 rows take weights rounded to f16,
# and V of 8-bit pools too.
STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def visible(length, m, window=0, sinks=0, prefix=None, first=None):
    """[m][length]: which positions each row sees (none before position 0)."""
    p = np.arange(length - m, length)[:, None]
    t = np.arange(length)[None, :]
    f = np.zeros((m, 1), np.int64) if first is None else np.maximum(np.asarray(first, np.int64), 0)[:, None]
    see = ((t <= p) | (t < (0 if prefix is None else prefix))) & (t >= f) & (p >= 0)
    if window:
        see &= (t > p - window) | (t - f < sinks)
    return see


def definition(q, held, tables, lens, starts, heads, hd, rows="f32", eight=False, scale=None, softcap=0.0, slopes=None,
               window=0, sinks=0, prefix=None, first=None):
    """(result, bound, finite): finite is False for the rows that see an infinity
    or NaN, whose result is not finite either. A cap's error: tanh to 16 half
    steps of itself; 16-bit rows of caps up to 256 to 16 half steps of the cap."""
    k_all, v_all = held
    g = heads // (k_all.shape[1] // hd)
    scale = float(np.float32(1 / math.sqrt(hd) if scale is None else scale))
    q = q.astype(np.float64)
    out, bound, finite = np.zeros_like(q), np.zeros_like(q), np.ones(q.shape[0], bool)
    for i, length in enumerate(lens):
        lo, m = starts[i], starts[i + 1] - starts[i]
        if length == 0 or m == 0:
            continue
        t = np.arange(length)
        cells = np.maximum(tables[i], 0)[t // BLOCK].astype(np.int64) * BLOCK + t % BLOCK
        see = visible(length, m, window, sinks, None if prefix is None else prefix[i],
                      None if first is None else first[lo:lo + m])
        k, v = k_all[cells], v_all[cells]
        bad = ~(np.isfinite(k).all(axis=1) & np.isfinite(v).all(axis=1))
        finite[lo:lo + m] = ~(see & bad).any(axis=1)
        k, v = np.where(bad[:, None], 0, k), np.where(bad[:, None], 0, v)
        dist = np.abs(np.arange(length - m, length)[:, None] - t[None, :])
        some, count = see.any(axis=1), see.sum(axis=1)
        for h in range(heads):
            a, qs = h // g * hd, q[lo:lo + m, h * hd:(h + 1) * hd]
            kh, vh = k[:, a:a + hd], v[:, a:a + hd]
            s = qs @ kh.T * scale
            off = np.minimum(np.abs(qs) @ np.abs(kh).T, 6 * np.sqrt(qs ** 2 @ (kh ** 2).T)) * abs(scale)
            off = SIGMA * math.sqrt(hd + 16) * H * off
            if softcap:
                s = softcap * np.tanh(s / softcap)
                off = off + 16 * H * (softcap if rows != "f32" and softcap <= 256 else np.abs(s))
            if slopes is not None:
                s = s - float(slopes[h]) * dist
                off = off + 2 * H * float(slopes[h]) * dist
            off = np.where(see, off + 4 * H * np.abs(s), 0).max(axis=1)
            s = np.where(see, s, -np.inf)
            top = np.where(some, s.max(axis=1), 0)
            w = np.exp(s - top[:, None])
            w /= np.where(some, w.sum(axis=1), 1)[:, None]
            o, mass = w @ vh, w @ np.abs(vh)
            largest = np.where(see, np.abs(vh).max(axis=1)[None, :], 0).max(axis=1)
            small = 2.0 ** -30 * w.max(axis=1) * count * largest
            b = (2 * off + SIGMA * np.sqrt(count + 32) * H)[:, None] * mass + small[:, None]
            if rows != "f32":
                b += (2 + eight) * 2.0 ** -11 * mass + STEP[rows] * np.abs(o) + 2.0 ** -25
            out[lo:lo + m, h * hd:(h + 1) * hd] = o
            bound[lo:lo + m, h * hd:(h + 1) * hd] = b
    return out, bound, finite


def compare(got, want):
    out, bound, finite = want
    assert np.isfinite(got[finite]).all(), f"rows {np.flatnonzero(~np.isfinite(got).all(axis=1) & finite)[:8]}"
    err = np.abs(got.astype(np.float64) - out)[finite]
    bound = bound[finite] + 1e-30
    assert (err <= bound).all(), f"error {err.max():.3e}, {(err / bound).max():.2f} times what rounding allows"
