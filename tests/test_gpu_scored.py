"""Scored attention (capped scores, distance biases, windows, prefixes,
documents) against the definition in 64 bits over the rows the pool holds.

Tolerances: a score is an f32 sum of head_dim products of Q and K, with some 16
roundings more (Q as two f16 parts, the scale, the cap and the bias). Each
rounds a partial sum by at most half a step, 2^-24 of it; partial sums are at
most the products' magnitudes together, and six times the root of their squares
(six sigma of their signs). Roundings are independent: n of them add up to
6 / sqrt(3) sqrt(n) of one's bound (six sigma of a uniform error) rather than to
n. A weight is then off by as much relatively, twice (numerator and sum), the
f32 sums over L positions by L + 32 roundings (32: exp2, the weights as two f16
parts, the folds), and f16 / bf16 rows by one f16 rounding per weight (2^-11, in
numerator and sum) and the rounding of the result to its type.
Small weights are off absolutely: the lo part of a weight is an f16 number, a
multiple of 2^-24, and a largest weight enters the products as at least 2^6 (8-bit
pools: as at least 2^6 over the largest scale, times quants of up to 127), so a
weight is off by at most 2^-25 / 2^6 = 2^-31 of the largest, times at most the
largest |V| the position could hold: 2^-30 w_max L max |V| in all, where a
position with a tiny weight holds the only value of its column."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BLOCK = 16
H = 2.0 ** -24  # half a step of f32
SIGMA = 6 / math.sqrt(3)


def held_rows(kv, layer=0):
    """K and V of a layer as the pool holds them, f64 [cells][kv_dim]."""
    k, v = kv.read_pool(layer)
    out = []
    if kv.dtype in ("q8_0", "q4_0"):
        for q, s in zip((k, v), kv.read_scales(layer)):
            d = s.view(np.float16).astype(np.float64)  # [block][group][slot]
            d = np.repeat(d.transpose(0, 2, 1), 32, axis=2)
            out.append((q.astype(np.float64) * d).reshape(-1, kv.kv_dim))
    else:
        for x in (k, v):
            x = x.view(np.float16) if kv.dtype == "f16" else x
            out.append(x.astype(np.float64).reshape(-1, kv.kv_dim))
    return out


def build(kvd, lens, dtype, seed, device=0, slack=2, stream=None, layers=1, edit=None):
    """A cache with len(lens) sequences of random rows in a permuted pool, and
    its tables. edit(i, k, v) may change sequence i's rows before the write."""
    import torch

    from langtrain_studio_amd import KvCache

    rng = np.random.default_rng(seed)
    blocks = sum(-(-n // BLOCK) for n in lens) + slack
    kv = KvCache(layers, kvd, blocks * BLOCK, dtype=dtype, device=device, stream=stream)
    kv.init_free_order(rng.permutation(blocks))
    dev = torch.device("cuda", device)
    for i, n in enumerate(lens):
        if n == 0:
            continue
        sm = kv.append_batch(np.full(n, i, np.uint32), np.arange(n, dtype=np.uint64))
        size = np.exp(0.3 * rng.standard_normal(kvd)).astype(np.float32)
        for layer in range(layers):
            k = (rng.standard_normal((n, kvd), dtype=np.float32) * size).astype(np.float32)
            v = rng.standard_normal((n, kvd), dtype=np.float32)
            if edit:
                edit(i, k, v)
            kv.write_batch(layer, torch.from_numpy(sm).to(dev), torch.from_numpy(k).to(dev),
                           torch.from_numpy(v).to(dev))
    return kv, kv.block_tables(np.arange(len(lens), dtype=np.uint32))


def expect(q, held, tables, lens, starts, heads, hd, scale=None, softcap=0.0, slopes=None, window=0, sinks=0,
           prefix=None, first=None):
    """(result, bound of the f32 error, weights times |V|) per row, 64 bits."""
    k_all, v_all = held
    kv_heads = k_all.shape[1] // hd
    g = heads // kv_heads
    scale = float(np.float32(1 / math.sqrt(hd) if scale is None else scale))
    out = np.zeros(q.shape, np.float64)
    bound, mass = np.zeros_like(out), np.zeros_like(out)
    q = q.astype(np.float64)
    for i, length in enumerate(lens):
        rows = range(starts[i], starts[i + 1])
        if length == 0 or not len(rows):
            continue
        cells = tables[i][np.arange(length) // BLOCK].astype(np.int64) * BLOCK + np.arange(length) % BLOCK
        for j, r in enumerate(rows):
            p = length - len(rows) + j
            if p < 0:
                continue
            t = np.arange(length)
            f = 0 if first is None else int(first[r])
            see = (t <= p) | (t < (0 if prefix is None else prefix[i]))
            see &= t >= f
            if window:
                see &= (t > p - window) | (t - f < sinks)
            t = t[see]
            if t.size == 0:
                continue
            k, v = k_all[cells[t]], v_all[cells[t]]
            for h in range(heads):
                a, qs = h // g * hd, q[r, h * hd:(h + 1) * hd]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k[:, a:a + hd] @ qs * scale
                    mag = np.abs(k[:, a:a + hd]) @ np.abs(qs) * abs(scale)
                    mag = np.minimum(mag, 6 * np.sqrt(k[:, a:a + hd] ** 2 @ qs ** 2) * abs(scale))
                    off = SIGMA * math.sqrt(hd + 16) * H * mag
                    if softcap:
                        s = softcap * np.tanh(s / softcap)
                        off = off + 16 * H * softcap
                    if slopes is not None:
                        s = s - float(slopes[h]) * np.abs(p - t)
                        off = off + 2 * H * float(slopes[h]) * np.abs(p - t)
                    off = off + 4 * H * np.abs(s)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    o, m = w @ v[:, a:a + hd], w @ np.abs(v[:, a:a + hd])
                    out[r, h * hd:(h + 1) * hd] = o
                    mass[r, h * hd:(h + 1) * hd] = m
                    small = 2.0 ** -30 * w.max() * t.size * np.abs(v[:, a:a + hd]).max()
                    bound[r, h * hd:(h + 1) * hd] = (2 * off.max() + SIGMA * math.sqrt(t.size + 32) * H) * m + small
    return out, bound, mass


def check(got, want, rows):
    out, bound, mass = want
    if rows != "f32":  # one f16 rounding per weight, then the result's
        step = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}[rows]
        bound = bound + 2 * 2.0 ** -11 * mass + step * np.abs(out) + 2.0 ** -25
    err = np.abs(got.astype(np.float64) - out)
    assert np.isfinite(got).all()
    worst = (err / (bound + 1e-30)).max() if err.size else 0.0
    assert (err <= bound + 1e-30).all(), f"error {err.max():.3e}, {worst:.2f} times what rounding allows"
    return worst


def run(kv, q, tables, lens, heads, hd, rows="f32", starts=None, out=None, **how):
    import torch

    dev = torch.device("cuda", kv.device)
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[rows]

    def up(a, dtype):
        return None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(dev)

    for name, dtype in (("slopes", np.float32), ("prefix", np.int32), ("first", np.int32)):
        if name in how:
            how[name] = up(how[name], dtype)
    qd = torch.from_numpy(np.ascontiguousarray(q, np.float32)).to(dev).to(dt)
    got = kv.scored_attention(0, qd, up(tables, np.int32), up(lens, np.int32), heads, hd,
                              row_starts=up(starts, np.int32), out=out, **how)
    kv.synchronize()
    return got.float().cpu().numpy(), qd.float().cpu().numpy()


def slopes_of(heads):
    return np.array([2.0 ** (-8.0 * (i + 1) / heads) for i in range(heads)], np.float32)


# (heads, kv heads, head_dim): tuned widths and groups, and ones outside them
SHAPES = [(8, 2, 128), (7, 1, 128), (4, 4, 64), (9, 3, 64), (16, 1, 64), (6, 2, 96), (20, 1, 80), (2, 2, 256),
          (3, 1, 40)]


def shape_dtype():
    for shape in SHAPES:
        for dtype in ("f16", "f32", "q8_0", "q4_0"):
            if dtype in ("q8_0", "q4_0") and shape[1] * shape[2] % 32:
                continue
            yield shape, dtype


MODS = {
    "plain": {},
    "cap": {"softcap": 5.0},
    "alibi": {"slopes": True},
    "window": {"window": 23, "sinks": 3},
    "all": {"softcap": 8.0, "slopes": True, "window": 40, "sinks": 1},
}


@pytest.mark.parametrize("mods", MODS)
@pytest.mark.parametrize("shape,dtype", list(shape_dtype()))
def test_single_tokens(gpu, shape, dtype, mods):
    """One row per sequence: lengths of zero, one, block and tile borders."""
    heads, kv_heads, hd = shape
    lens = [1, 0, 15, 16, 17, 33, 64, 65, 200, 517]
    kv, tables = build(kv_heads * hd, lens, dtype, 1)
    q = np.random.default_rng(2).standard_normal((len(lens), heads * hd)).astype(np.float32) * 2
    how = dict(MODS[mods])
    if how.get("slopes"):
        how["slopes"] = slopes_of(heads)
    got, qr = run(kv, q, tables, lens, heads, hd, **how)
    want = expect(qr, held_rows(kv), tables, lens, list(range(len(lens) + 1)), heads, hd, **how)
    check(got, want, "f32")


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mods", MODS)
@pytest.mark.parametrize("shape,dtype", list(shape_dtype()))
def test_chunks(gpu, shape, dtype, mods, rows):
    """Ragged chunks beside single tokens, empty sequences among them."""
    heads, kv_heads, hd = shape
    if rows != "f32" and mods in ("cap", "alibi"):
        pytest.skip("covered with f32 rows")
    lens = [70, 5, 0, 150, 33, 260]
    new = [70, 1, 0, 37, 2, 130]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 3)
    q = np.random.default_rng(4).standard_normal((starts[-1], heads * hd)).astype(np.float32) * 2
    how = dict(MODS[mods])
    if how.get("slopes"):
        how["slopes"] = slopes_of(heads)
    got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=max(new), **how)
    want = expect(qr, held_rows(kv), tables, lens, starts, heads, hd, **how)
    check(got, want, rows)


@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 96])
def test_prefix_and_documents(gpu, dtype, hd):
    """A bidirectional prefix (also one longer than the context, and none), and
    documents that start inside a tile, at a row's own position and behind it
    (nothing visible)."""
    heads, kv_heads = 6, 2
    lens, new = [90, 140, 50, 30], [90, 60, 50, 1]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 5)
    rng = np.random.default_rng(6)
    q = rng.standard_normal((starts[-1], heads * hd)).astype(np.float32)
    prefix = [40, 0, 900, 30]
    first = np.zeros(starts[-1], np.int32)
    for i, (n, m) in enumerate(zip(lens, new)):
        for j in range(m):
            p = n - m + j
            first[starts[i] + j] = p // 37 * 37 if i != 2 else p - j % 3 + 1  # sequence 2: at or behind its row
    first[0] = -5
    for how in ({"prefix": prefix}, {"first": first}, {"prefix": prefix, "first": first, "window": 20, "sinks": 4},
                {"prefix": prefix, "slopes": slopes_of(heads), "softcap": 4.0}):
        got, qr = run(kv, q, tables, lens, heads, hd, starts=starts, max_rows=90, **how)
        want = expect(qr, held_rows(kv), tables, lens, starts, heads, hd,
                      **{**how, **({"first": np.maximum(first, 0)} if "first" in how else {})})
        check(got, want, "f32")


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("shape", [(8, 2, 128), (9, 3, 64)])
def test_long_contexts(gpu, shape, dtype, rows):
    """Contexts long enough to be split, single tokens and a short chunk."""
    heads, kv_heads, hd = shape
    lens, new = [5000, 2049, 3500], [1, 1, 20]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 7)
    q = np.random.default_rng(8).standard_normal((starts[-1], heads * hd)).astype(np.float32) * 2
    for how in ({}, {"window": 1500, "sinks": 70}, {"softcap": 10.0, "slopes": slopes_of(heads) / 16}):
        got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=20, **how)
        check(got, expect(qr, held_rows(kv), tables, lens, starts, heads, hd, **how), rows)


@pytest.mark.parametrize("shape", [(8, 2, 128), (4, 4, 64), (6, 2, 96)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_unseen_positions_may_hold_anything(gpu, shape, dtype):
    """Infinities and NaN in K and V at positions a row does not see: outside
    the window, before the document, behind the row, behind the context. Rows
    that see such a position have a NaN result; the others' results are those
    of finite rows."""
    import torch

    heads, kv_heads, hd = shape
    lens, new = [100, 300, 64], [100, 1, 3]
    starts = np.concatenate([[0], np.cumsum(new)])
    bad = {0: [40, 41], 1: [0, 5, 130, 207], 2: [63]}  # sequence 2: the last row's own position

    def poison(i, k, v):
        for n, p in enumerate(bad[i]):
            k[p, :] = [np.nan, np.inf][n % 2]
            v[p, :] = [np.nan, -np.inf][n % 2]

    kv, tables = build(kv_heads * hd, lens, dtype, 9, edit=poison)
    clean, ctables = build(kv_heads * hd, lens, dtype, 9)
    q = np.random.default_rng(10).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    window = 25
    for lens_now in (lens, [100, 240, 64]):  # 240: stale cells behind the context
        got, _ = run(kv, q, tables, lens_now, heads, hd, starts=starts, max_rows=100, window=window)
        base, _ = run(clean, q, ctables, lens_now, heads, hd, starts=starts, max_rows=100, window=window)
        for i, m in enumerate(new):
            for j in range(m):
                r, p = starts[i] + j, lens_now[i] - m + j
                sees = any(p - window < b <= p for b in bad[i])
                if sees:
                    assert np.isnan(got[r]).all(), (i, j)
                else:
                    np.testing.assert_allclose(got[r], base[r], rtol=1e-5, atol=1e-5)
    assert torch.cuda.is_available()


def test_rows_of_no_sequence_stay(gpu):
    """Rows before the first start and behind the last are left as they were,
    and a sequence may have more rows than max_rows says."""
    import torch

    heads, kv_heads, hd = 4, 2, 64
    lens = [50, 200]
    starts = np.array([3, 20, 150], np.int32)
    kv, tables = build(kv_heads * hd, lens, "f16", 11)
    q = np.random.default_rng(12).standard_normal((160, heads * hd)).astype(np.float32)
    for max_rows in (1, 20, 160):
        out = torch.full((160, heads * hd), 7.5, device="cuda")
        got, qr = run(kv, q, tables, lens, heads, hd, starts=starts, max_rows=max_rows, out=out)
        assert (got[:3] == 7.5).all() and (got[150:] == 7.5).all()
        want = expect(qr, held_rows(kv), tables, lens, starts, heads, hd)
        check(got[3:150], [w[3:150] for w in want], "f32")


def test_more_rows_than_context_and_lengths_past_the_table(gpu):
    """Rows that stand before position 0 give zeros; lengths are cut to the
    table."""
    heads, kv_heads, hd = 4, 2, 128
    kv, tables = build(kv_heads * hd, [10, 64], "f16", 13)
    starts = np.array([0, 14, 20], np.int32)
    q = np.random.default_rng(14).standard_normal((20, heads * hd)).astype(np.float32)
    got, qr = run(kv, q, tables[:, :4], [10, 99999], heads, hd, starts=starts, max_rows=14)
    assert (got[:4] == 0).all()
    check(got, expect(qr, held_rows(kv), tables, [10, 64], starts, heads, hd), "f32")


@pytest.mark.parametrize("dtype", ["f16", "q4_0"])
def test_large_queries(gpu, dtype):
    """Q of large and of tiny magnitude beside each other, per head."""
    heads, kv_heads, hd = 8, 2, 128
    lens = [40, 300]
    kv, tables = build(kv_heads * hd, lens, dtype, 15)
    q = np.random.default_rng(16).standard_normal((2, heads, hd)).astype(np.float32)
    q *= (10.0 ** np.array([-30, -6, 0, 3, 6, 8, 20, 30]))[None, :, None].astype(np.float32)
    for h, f in enumerate(10.0 ** np.array([-30, -6, 0, 3, 6, 8, 20, 30])):
        one = np.zeros_like(q)
        one[:, h] = q[:, h]
        scale = float(0.1 / max(f, 1.0))  # scores of ordinary size
        got, qr = run(kv, one.reshape(2, -1), tables, lens, heads, hd, scale=scale)
        check(got, expect(qr, held_rows(kv), tables, lens, [0, 1, 2], heads, hd, scale=scale), "f32")


def test_bad_table_entries_are_reported(gpu):
    from langtrain_studio_amd import KvError

    heads, kv_heads, hd = 4, 2, 64
    kv, tables = build(kv_heads * hd, [100, 100], "f16", 17)
    q = np.zeros((2, heads * hd), np.float32)
    bad = tables.copy()
    bad[1, 3] = 1 << 20
    with pytest.raises(KvError, match="outside the pool"):
        run(kv, q, bad, [100, 100], heads, hd)
    run(kv, q, bad, [100, 100], heads, hd, window=20)  # not read: position 48..63 is outside the window
    run(kv, q, bad, [100, 40], heads, hd)              # nor behind the length


def test_refusals(gpu):
    import torch

    from langtrain_studio_amd import KvError

    heads, kv_heads, hd = 4, 2, 64
    kv, tables = build(kv_heads * hd, [20, 20], "f16", 19)
    dev = torch.device("cuda", 0)
    t = torch.from_numpy(tables).to(dev)
    lens = torch.tensor([20, 20], dtype=torch.int32, device=dev)
    q = torch.zeros((2, heads * hd), device=dev)
    ok = dict(layer=0, q=q, tables=t, lens=lens, n_heads=heads, head_dim=hd)

    def no(err, match=None, **kw):
        with pytest.raises(err, match=match):
            kv.scored_attention(**{**ok, **kw})

    no(KvError, "out of range", layer=1)
    no(KvError, "softcap", softcap=-1.0)
    no(KvError, "softcap", softcap=math.nan)
    no(KvError, "softcap", softcap=math.inf)
    no(KvError, "scale", scale=math.inf)
    no(KvError, "sinks need a window", sinks=2)
    no(ValueError, "negative", window=-1)
    no(TypeError, "float32, float16 or bfloat16", q=q.double())
    no(ValueError, "one row per sequence", q=torch.zeros((3, heads * hd), device=dev))
    no(ValueError, "row_starts", row_starts=torch.zeros(2, dtype=torch.int32, device=dev))
    no(ValueError, "slopes", slopes=torch.zeros(3, device=dev))
    no(ValueError, "prefix", prefix=torch.zeros(3, dtype=torch.int32, device=dev))
    no(ValueError, "first", first=torch.zeros(3, dtype=torch.int32, device=dev))
    no(TypeError, "int32", first=torch.zeros(2, dtype=torch.int64, device=dev))
    no(ValueError, "out must match", out=torch.zeros((1, heads * hd), device=dev))
    no(TypeError, "out must be", out=torch.zeros((2, heads * hd), device=dev, dtype=torch.float16))
    no(ValueError, "contiguous", q=torch.zeros((heads * hd, 2), device=dev).t())
    no(KvError, "multiple of n_kv_heads", n_heads=3, q=torch.zeros((2, 3 * hd), device=dev))
    kv.scored_attention(**ok)
    none = kv.scored_attention(**{**ok, "q": q[:0], "tables": t[:0], "lens": lens[:0]})
    assert none.shape == (0, heads * hd)
    kv.synchronize()
