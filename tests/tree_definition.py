"""Attention of drafted trees by its definition in 64 bits, with the error that
f32 arithmetic may make (the derivation of test_gpu_scored, whose constants these
are; f16 and bf16 rows take weights rounded to f16, and V of 8-bit and f32 pools
too, the cap's tanh is off by up to 16 half steps). What a row does not see enters
neither its result nor its bound."""

from __future__ import annotations

import math

import numpy as np

from test_gpu_scored import BLOCK, H, SIGMA

STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def random_tree(rng, m, branch=0.4, roots=0.0):
    """Parents of m tokens: each continues the last, branches off an earlier one
    or is a root of its own."""
    out = []
    for j in range(m):
        r = rng.random()
        if j == 0 or r < roots:
            out.append(-1)
        else:
            out.append(int(rng.integers(0, j)) if r < roots + branch else j - 1)
    return out


def ancestors(parents):
    """[m][m]: the tokens on each token's way up, itself among them."""
    m = len(parents)
    see = np.zeros((m, m), bool)
    for j, p in enumerate(parents):
        if 0 <= p < j:
            see[j] = see[p]
        see[j, j] = True
    return see


def depths(parents):
    return ancestors(parents).sum(axis=1) - 1 if len(parents) else np.zeros(0, np.int64)


def words_of(see, words):
    """Mask words of [m][m'] visibility; rows from 32 * words on have no bit."""
    bits = np.zeros((see.shape[0], words * 32), bool)
    n = min(see.shape[1], words * 32)
    bits[:, :n] = see[:, :n]
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(see.shape[0], words)


def visible(length, drafted, window=0, positions=None):
    """[m][length]: what each of m rows sees, drafted [m][m] of its own cells."""
    m = drafted.shape[0]
    ctx = length - m
    t = np.arange(length)
    see = np.zeros((m, length), bool)
    for r in range(m):
        context = t < ctx
        if window:
            context &= t > max(int(positions[r]), ctx, 0) - window
        see[r] = context
        own = t[t >= max(ctx, 0)] - ctx
        see[r, t >= max(ctx, 0)] = drafted[r, own]
    return see


def definition(q, held, tables, lens, starts, heads, hd, sees, rows="f32", eight=False, scale=None, softcap=0.0):
    """(result, bound, finite) of all rows; sees[i] [m][lens[i]]. finite is False
    for the rows that see an infinity or NaN."""
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
        see = sees[i]
        k, v = k_all[cells], v_all[cells]
        bad = ~(np.isfinite(k).all(axis=1) & np.isfinite(v).all(axis=1))
        finite[lo:lo + m] = ~(see & bad).any(axis=1)
        k, v = np.where(bad[:, None], 0, k), np.where(bad[:, None], 0, v)
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
