"""The 4-bit cache and scored attention as measurable cases.

One pass of a case is one pass through an operator as a user's program calls
it. Where ``own`` is false the pass runs the operator's plain form (elementary
torch operations), where it is true the framework's entry points:

* "ingest": rows appended to a 4-bit cache (``write_batch``) and read back as
  f32 values (``gather_values``), as when a prompt is stored and its rows go to
  code that takes contiguous values.
* "step": a decode step on a 4-bit cache: new rows appended, then attention
  (``append_decode_attention``).
* "decode": decode attention over a 4-bit cache (``decode_attention``).
* "scored": attention whose scores are capped by a tanh, get a bias that grows
  with distance, and are masked by a window, a prefix or document starts
  (``scored_attention``), single tokens and prompt chunks alike.

The 4-bit format: each 32 elements of a row share a scale d; e is the element
of largest magnitude (the positive one where both signs reach it; magnitudes
over 65280 count as 65280 and NaN as 0), d is -e / 8 rounded to bf16 and then
to f16 (nearest even), an element is held as the nearest q in -8 .. 7 to x / d
(nearest even; 0 where d is 0) and read back as q * d.

Lengths, prefixes and document starts are a function of the case alone (its
"spread" seed), values of the seed given to ``prepare``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16
LIMIT = 65280.0

# (query heads, kv heads, head_dim)
LLAMA3_8B = (32, 8, 128)
QWEN25_7B = (28, 4, 128)
TINYLLAMA = (32, 4, 64)
SMOLLM2 = (9, 3, 64)


def _case(name, kind, shape, **kw):
    heads, kv_heads, head_dim = shape
    return {"name": name, "kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, **kw}


def _scored(name, shape, **kw):
    base = {"dtype": "f16", "rows": "f32", "gain": 1.0, "softcap": 0.0, "alibi": False, "window": 0, "sinks": 0,
            "prefix": False, "docs": False, "chunks": 0, "chunk_lo": 1, "chunk": 1, "decodes": 0}
    base.update(kw)
    return _case(name, "scored", shape, **base)


def listed():
    return [
        # A small local model, four short chats on a 4-bit cache: launch latency.
        _case("step-tiny-q4", "step", TINYLLAMA, batch=4, lo=128, hi=512, spread=1),
        # A server's prompts of one scheduling round, stored and read back.
        _case("ingest-prompts-q4", "ingest", LLAMA3_8B, seqs=16, lo=200, hi=1000, spread=2),
        # One prompt at another row width (10 groups of 32), an odd length.
        _case("ingest-odd-q4", "ingest", (20, 4, 80), seqs=1, lo=777, hi=777, spread=3),
        # One user's chat in mid-conversation: the interactive stream.
        _case("decode-chat-q4", "decode", LLAMA3_8B, batch=1, lo=5003, hi=5003, spread=4),
        # The server's full decode batch.
        _case("decode-batch-q4", "decode", LLAMA3_8B, batch=64, lo=2048, hi=4096, spread=5),
        # Long documents, which the 4-bit cache is for.
        _case("decode-long-q4", "decode", QWEN25_7B, batch=8, lo=32700, hi=32768, spread=6),
        # A decode batch with capped scores and a sliding window behind sink tokens.
        _scored("scored-step-window", LLAMA3_8B, gain=3.0, softcap=30.0, window=1024, sinks=4, decodes=32, lo=300,
                hi=4000, spread=7),
        # A small model with distance biases on an 8-bit cache.
        _scored("scored-step-alibi-q8", SMOLLM2, dtype="q8_0", alibi=True, decodes=12, lo=50, hi=3000, spread=8),
        # One long prompt with capped scores, half-precision activations.
        _scored("scored-prompt-cap", LLAMA3_8B, rows="bf16", gain=3.0, softcap=30.0, chunks=1, chunk_lo=4096,
                chunk=4096, lo=0, hi=0, spread=9),
        # Prompt chunks behind their contexts, sliding window, 4-bit cache.
        _scored("scored-chunks-q4", QWEN25_7B, dtype="q4_0", window=2048, sinks=4, chunks=6, chunk_lo=400, chunk=512,
                lo=0, hi=6000, spread=10),
        # Packed documents with a shared bidirectional prefix, ragged chunks.
        _scored("scored-docs-prefix", TINYLLAMA, alibi=True, prefix=True, docs=True, chunks=5, chunk_lo=30, chunk=700,
                lo=0, hi=900, spread=11),
        # Decodes beside a prompt chunk, f16 activations, an f32 cache of another head width.
        _scored("scored-mixed-f32", (20, 4, 80), dtype="f32", rows="f16", gain=2.0, softcap=20.0, chunks=1,
                chunk_lo=90, chunk=90, decodes=12, lo=17, hi=900, spread=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# Shapes of the repository's configurations and tests; the last four are
# outside the common head_dim 64 / 128 and groups of up to 8.
COMMON = [LLAMA3_8B, QWEN25_7B, TINYLLAMA, SMOLLM2]
OTHER = [(32, 8, 96), (16, 1, 128), (8, 1, 256), (20, 4, 80)]


def draw(rng):
    kind = rng.choice(["ingest", "step", "decode", "decode", "scored", "scored", "scored", "scored", "scored"])
    spread = rng.randrange(1 << 20)
    if kind == "ingest":
        seqs = _log(rng, 1, 16)
        hi = _log(rng, 20, 9000 // seqs)
        return _case("", "ingest", rng.choice(COMMON + OTHER), seqs=seqs, lo=max(1, hi // rng.choice([1, 8])), hi=hi,
                     spread=spread)
    if kind in ("step", "decode"):
        other = rng.random() < 0.2
        batch = _log(rng, 1, 96)
        hi = min(_log(rng, 32, 32768), (6000 if other else 200000) // batch + 32)
        return _case("", kind, rng.choice(OTHER if other else COMMON), batch=batch,
                     lo=max(1, hi // rng.choice([1, 2, 8]) - rng.randrange(7)), hi=hi, spread=spread)
    other = rng.random() < 0.2
    chunks = rng.choice([0, 1, _log(rng, 1, 6)])
    chunk = _log(rng, 2, 200 if other else 1500)
    hi = min(_log(rng, 16, 900 if other else 5000), 5000000 // (max(1, chunks) * chunk))
    window = rng.choice([0, 0, _log(rng, 8, 3000)])
    prefix = rng.random() < 0.2
    return _scored("", rng.choice(OTHER if other else COMMON), dtype=rng.choice(["f16", "f16", "q8_0", "q4_0", "f32"]),
                   rows=rng.choice(["f32", "f16", "bf16"]), gain=rng.choice([1.0, 3.0]),
                   softcap=rng.choice([0.0, 15.0, 50.0]), alibi=rng.random() < 0.4, window=window,
                   sinks=rng.choice([0, 4]) if window else 0, prefix=prefix, docs=rng.random() < 0.2, chunks=chunks,
                   chunk_lo=max(1, chunk // rng.choice([1, 4])), chunk=chunk,
                   decodes=_log(rng, 1, 48) if chunks == 0 else rng.choice([0, _log(rng, 1, 20)]),
                   lo=hi // rng.choice([1, 2, 8]), hi=hi, spread=spread)


# ---- sizes of a case ----------------------------------------------------------


def _dims(case):
    return case["heads"], case["kv_heads"], case["head_dim"], case["kv_heads"] * case["head_dim"]


CELL = {"f16": 2.0, "f32": 4.0, "q8_0": 1.0 + 2.0 / 32, "q4_0": 0.5 + 2.0 / 32}
ROWS = {"f32": 4, "f16": 2, "bf16": 2}


def _lens(case, n):
    r = np.random.default_rng(case["spread"])
    return [int(x) for x in r.integers(case["lo"], case["hi"] + 1, n)]


def _layout(case):
    """A scored case's sequences: context lengths (all rows included), rows of
    each, prefix lengths, and the first visible position of every row."""
    r = np.random.default_rng(case["spread"] + 1)
    n = case["chunks"] + case["decodes"]
    new = [int(x) for x in r.integers(case["chunk_lo"], case["chunk"] + 1, case["chunks"])] + [1] * case["decodes"]
    lens = [c + m for c, m in zip(_lens(case, n), new)]
    prefix = [int(x * length) for x, length in zip(r.random(n), lens)] if case["prefix"] else None
    first = None
    if case["docs"]:
        first = []
        for length, m in zip(lens, new):
            # documents of a random length follow each other; a row sees from its own's start
            start, pos = 0, length - m
            ends = np.cumsum(r.integers(1, max(2, length // 2), 64))
            for p in range(pos, length):
                while p >= ends[start] and start < 63:
                    start += 1
                first.append(int(ends[start - 1]) if start else 0)
    return lens, new, prefix, first


def _visible(case, length, m, prefix, first):
    """[m][length] on the host: which positions each row sees."""
    pos = np.arange(length - m, length)[:, None]
    t = np.arange(length)[None, :]
    see = t <= pos
    if prefix is not None:
        see = see | (t < prefix)
    f = np.zeros((m, 1), np.int64) if first is None else np.asarray(first)[:, None]
    see = see & (t >= f)
    if case["window"]:
        see = see & ((t > pos - case["window"]) | (t - f < case["sinks"]))
    return see


def work(case):
    heads, _, hd, kvd = _dims(case)
    kind = case["kind"]
    cell = CELL[case.get("dtype", "q4_0")]
    if kind == "ingest":
        rows = sum(_lens(case, case["seqs"]))
        return {"bytes": rows * 2 * kvd * (4 + 2 * cell + 4), "flops": 0.0}
    if kind in ("step", "decode"):
        lens = _lens(case, case["batch"])
        total, n = sum(lens), len(lens)
        new = n * 2 * kvd * 4 if kind == "step" else 0
        return {"bytes": 2 * total * kvd * cell + 2 * n * heads * hd * 4 + new, "flops": 4.0 * heads * hd * total}
    lens, new, prefix, first = _layout(case)
    pairs = cells = row = 0
    for i, (length, m) in enumerate(zip(lens, new)):
        see = _visible(case, length, m, prefix[i] if prefix else None, first[row:row + m] if first else None)
        pairs += int(see.sum())
        cells += int(see.any(axis=0).sum())
        row += m
    return {"bytes": 2 * cells * kvd * cell + 2 * row * heads * hd * ROWS[case["rows"]], "flops": 4.0 * heads * hd * pairs}


# ---- inputs -------------------------------------------------------------------


def _normal(seed, stream, rows, dim):
    """N(0, 1) f32 rows on the GPU, a function of (seed, stream) alone."""
    g = torch.Generator(device="cuda").manual_seed((seed * 1000003 + stream * 7919) % (1 << 62))
    return torch.randn((rows, dim), generator=g, device="cuda")


def _kv_rows(case, seed, seq, rows):
    """K and V rows of a sequence. Channels differ in size, as a model's do."""
    kvd = _dims(case)[3]
    size = torch.exp(0.4 * _normal(seed, 1, 2, kvd))
    return _normal(seed, 8 + 4 * seq, rows, kvd) * size[0], _normal(seed, 9 + 4 * seq, rows, kvd) * size[1]


def _queries(case, seed, rows):
    heads, _, hd, _ = _dims(case)
    q = _normal(seed, 2, rows, heads * hd) * case.get("gain", 1.0)
    return q.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[case.get("rows", "f32")])


def _slopes(case):
    h = case["heads"]
    return np.array([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], np.float32)


def _cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def _context(case):
    """Every sequence's length with this pass's rows, and the rows of each."""
    if case["kind"] == "ingest":
        lens = _lens(case, case["seqs"])
        return lens, lens
    if case["kind"] in ("step", "decode"):
        lens = _lens(case, case["batch"])
        return lens, [1] * len(lens)
    lens, new, _, _ = _layout(case)
    return lens, new


def prepare(case, seed):
    heads, _, hd, kvd = _dims(case)
    kind = case["kind"]
    lens, new = _context(case)
    n = len(lens)
    need = [-(-x // BLOCK) for x in lens]
    n_blocks = sum(need) + sum(need) // 10 + 1
    order = np.random.default_rng(seed).permutation(n_blocks)  # a fragmented pool
    cells = []
    tables = np.zeros((n, max(need)), np.int32)
    at = 0
    for i, (length, b) in enumerate(zip(lens, need)):
        blocks = order[at:at + b]
        at += b
        tables[i, :b] = blocks
        cells.append((blocks[np.arange(length) // BLOCK] * BLOCK + np.arange(length) % BLOCK).astype(np.int32))
    dtype = case.get("dtype", "q4_0")
    st = {"case": case, "lens": _cuda(np.array(lens, np.int32)), "lens_host": lens, "new": new, "dtype": dtype}
    if own:
        from langtrain_studio_amd import KvCache

        kv = st["kv"] = KvCache(1, kvd, n_blocks * BLOCK, dtype=dtype, stream=torch.cuda.current_stream())
        kv.init_free_order(order)
        for i, length in enumerate(lens):
            kv.append_batch(np.full(length, i, np.uint32), np.arange(length, dtype=np.uint64))
        st["tables"] = _cuda(kv.block_tables(np.arange(n, dtype=np.uint32)))

        def store(where, k, v):
            kv.write_batch(0, where, k, v)
    else:
        st["tables"] = _cuda(tables)
        st["pool"] = [_empty_pool(dtype, n_blocks, kvd) for _ in range(2)]

        def store(where, k, v):
            _store(dtype, st["pool"][0], where, k)
            _store(dtype, st["pool"][1], where, v)

    if kind != "ingest":  # the context is in the cache already
        for i in range(n):
            k, v = _kv_rows(case, seed, i, lens[i])
            store(_cuda(cells[i]), k, v)
            if kind == "step":
                st.setdefault("new_rows", []).append((k[-1:], v[-1:]))
    if kind == "ingest":
        rows = [_kv_rows(case, seed, i, lens[i]) for i in range(n)]
        st["k"], st["v"] = torch.cat([r[0] for r in rows]), torch.cat([r[1] for r in rows])
        st["cells"] = _cuda(np.concatenate(cells))
        st["offsets"] = _cuda(np.concatenate([[0], np.cumsum(lens)[:-1]]).astype(np.int64))
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        torch.cuda.synchronize()
        return st
    st["q"] = _queries(case, seed, sum(new))
    if own:
        st["out"] = torch.empty_like(st["q"])
    if kind == "step":
        st["k"] = torch.cat([r[0] for r in st["new_rows"]]).contiguous()
        st["v"] = torch.cat([r[1] for r in st.pop("new_rows")]).contiguous()
        st["cells"] = _cuda(np.array([c[-1] for c in cells], np.int32))
    if kind == "scored":
        _, _, prefix, first = _layout(case)
        st["starts_host"] = [0] + [int(x) for x in np.cumsum(new)]
        st["starts"] = _cuda(np.array(st["starts_host"], np.int32))
        st["slopes"] = _cuda(_slopes(case)) if case["alibi"] else None
        st["prefix"] = _cuda(np.array(prefix, np.int32)) if prefix else None
        st["first"] = _cuda(np.array(first, np.int32)) if first else None
    torch.cuda.synchronize()
    return st


# ---- the plain forms ------------------------------------------------------------


def _quantise(x):
    """(q, d) of f32 rows [n][kvd]: whole numbers and scales per 32 elements."""
    g = torch.nan_to_num(x, nan=0.0, posinf=LIMIT, neginf=-LIMIT).clamp(-LIMIT, LIMIT).reshape(x.shape[0], -1, 32)
    top, low = g.amax(dim=2, keepdim=True), g.amin(dim=2, keepdim=True)
    e = torch.where(top >= -low, top, low)
    d = (e * -0.125).to(torch.bfloat16).to(torch.float16)
    wide = d.double()
    q = torch.round(g.double() / torch.where(wide == 0, torch.ones_like(wide), wide)).clamp(-8, 7)
    return torch.where(wide == 0, torch.zeros_like(q), q).to(torch.int8).reshape(x.shape), d.reshape(x.shape[0], -1)


def _empty_pool(dtype, n_blocks, kvd):
    n = n_blocks * BLOCK
    if dtype in ("f16", "f32"):
        return torch.zeros((n, kvd), dtype=torch.float16 if dtype == "f16" else torch.float32, device="cuda")
    return (torch.zeros((n, kvd), dtype=torch.int8, device="cuda"),
            torch.zeros((n, kvd // 32), dtype=torch.float16, device="cuda"))


def _store(dtype, pool, cells, x):
    """Rows x into cells of a plain pool, rounded or quantised as it holds them."""
    cells = cells.long()
    if dtype in ("f16", "f32"):
        pool[cells] = x.to(pool.dtype)
    elif dtype == "q4_0":
        pool[0][cells], pool[1][cells] = _quantise(x)
    else:  # 8 bits: d = amax / 127, nearest, halves away from zero
        g = x.reshape(x.shape[0], -1, 32)
        d = g.abs().amax(dim=2, keepdim=True) / torch.full((1, 1, 1), 127.0, device="cuda")
        t = g * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
        q = torch.trunc(t)
        q = (q + torch.sign(t) * ((t - q).abs() >= 0.5)).clamp(-128, 127)
        pool[0][cells], pool[1][cells] = q.to(torch.int8).reshape(x.shape), d.half().reshape(x.shape[0], -1)


def _load(dtype, pool, table, length):
    """The f32 values of positions 0 .. length - 1 behind a block table."""
    at = torch.arange(length, device="cuda")
    cells = table.long()[at // BLOCK] * BLOCK + at % BLOCK
    if dtype in ("f16", "f32"):
        return pool[cells].float()
    q, d = pool[0][cells].float(), pool[1][cells].float()
    return (q.reshape(length, -1, 32) * d[:, :, None]).reshape(length, -1)


def _plain_attention(case, q, k, v, see, bias_at, slopes):
    """q [m][heads * hd], k and v [length][kvd] (f32); see [m][length] or None
    (all); bias_at [m][length]: distances, with slopes."""
    heads, kv_heads, hd, _ = _dims(case)
    g, m, length = heads // kv_heads, q.shape[0], k.shape[0]
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    qh = q.reshape(m, kv_heads, g, hd).permute(1, 2, 0, 3).reshape(kv_heads, g * m, hd).contiguous()
    kh = k.reshape(length, kv_heads, hd).permute(1, 2, 0).contiguous()
    vh = v.reshape(length, kv_heads, hd).permute(1, 0, 2).contiguous()
    s = (torch.matmul(qh, kh) * scale).reshape(kv_heads, g, m, length)
    cap = case.get("softcap", 0.0)
    if cap > 0:
        s = torch.tanh(s / cap) * cap
    if slopes is not None:
        s = s - slopes.reshape(kv_heads, g, 1, 1) * bias_at
    if see is not None:
        s = torch.where(see, s, torch.full_like(s, -math.inf))
    top = s.amax(dim=3, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.reshape(kv_heads, g * m, length), vh)
    return o.reshape(kv_heads, g, m, hd).permute(2, 0, 1, 3).reshape(m, heads * hd)


def _run_plain(st):
    case, dtype = st["case"], st["dtype"]
    kind = case["kind"]
    if kind == "ingest":
        kp, vp = st["pool"]
        _store(dtype, kp, st["cells"], st["k"])
        _store(dtype, vp, st["cells"], st["v"])
        ks = [_load(dtype, kp, st["tables"][i], n) for i, n in enumerate(st["lens_host"])]
        vs = [_load(dtype, vp, st["tables"][i], n) for i, n in enumerate(st["lens_host"])]
        return torch.cat(ks), torch.cat(vs)
    if kind == "step":
        _store(dtype, st["pool"][0], st["cells"], st["k"])
        _store(dtype, st["pool"][1], st["cells"], st["v"])
    out = torch.empty_like(st["q"])
    row = 0
    for i, (length, m) in enumerate(zip(st["lens_host"], st["new"])):
        k = _load(dtype, st["pool"][0], st["tables"][i], length)
        v = _load(dtype, st["pool"][1], st["tables"][i], length)
        for r in range(0, m, 1024):  # rows in pieces: the scores of a long prompt are many
            c = min(1024, m - r)
            q = st["q"][row + r:row + r + c].float()
            see = dist = None
            if kind == "scored":
                pos = torch.arange(length - m + r, length - m + r + c, device="cuda")[:, None]
                t = torch.arange(length, device="cuda")[None, :]
                see = t <= pos
                if st["prefix"] is not None:
                    see = see | (t < st["prefix"][i])
                f = 0 if st["first"] is None else st["first"][row + r:row + r + c].long()[:, None]
                see = see & (t >= f)
                if case["window"]:
                    see = see & ((t > pos - case["window"]) | (t - f < case["sinks"]))
                dist = (pos - t).abs().float()
            out[row + r:row + r + c] = _plain_attention(case, q, k, v, see, dist, st.get("slopes")).to(out.dtype)
        row += m
    return out


def run(st):
    if not own:
        return _run_plain(st)
    case, kv = st["case"], st["kv"]
    heads, _, hd, _ = _dims(case)
    if case["kind"] == "ingest":
        kv.write_batch(0, st["cells"], st["k"], st["v"])
        kv.gather_values(0, st["tables"], st["lens"], st["offsets"], st["k_out"], st["v_out"])
        return st["k_out"], st["v_out"]
    if case["kind"] == "step":
        return kv.append_decode_attention(0, st["cells"], st["k"], st["v"], st["q"], st["tables"], st["lens"], heads,
                                          hd, out=st["out"])
    if case["kind"] == "decode":
        return kv.decode_attention(0, st["q"], st["tables"], st["lens"], heads, hd, out=st["out"])
    return kv.scored_attention(0, st["q"], st["tables"], st["lens"], heads, hd, row_starts=st["starts"],
                               max_rows=max(st["new"]), softcap=case["softcap"], slopes=st["slopes"],
                               window=case["window"], sinks=case["sinks"], prefix=st["prefix"], first=st["first"],
                               out=st["out"])


# ---- the definition in 64 bits ----------------------------------------------------


def _held(dtype, x):
    """f32 rows as a cache of this type holds them, in 64 bits."""
    if dtype == "f16":
        return x.half().double()
    if dtype == "f32":
        return x.double()
    rows = x.double().view(x.shape[0], x.shape[1] // 32, 32)
    if dtype == "q8_0":
        # the format's scale and reciprocal are single-precision numbers
        d = (rows.abs().max(dim=2, keepdim=True).values.float().div(torch.tensor(127.0, device="cuda")))
        inv = torch.where(d > 0, torch.ones_like(d).div(d), torch.zeros_like(d))
        y = (x.view(rows.shape) * inv).double()
        q = torch.floor(y.abs() + 0.5).copysign(y).clamp(-128, 127)
        return (q * d.half().double()).view(x.shape)
    big, small = rows.max(dim=2, keepdim=True).values, rows.min(dim=2, keepdim=True).values
    e = torch.where(big + small >= 0, big, small).clamp(-LIMIT, LIMIT)
    d = (e / -8.0).float().bfloat16().half().double()
    y = torch.where(d != 0, rows / d, torch.zeros_like(rows))
    floor = torch.floor(y)
    up = (y - floor > 0.5) | ((y - floor == 0.5) & (floor.remainder(2.0) == 1))
    return ((floor + up).clamp(-8, 7) * d).view(x.shape)


def exact(case, seed):
    heads, kv_heads, hd, _ = _dims(case)
    lens, new = _context(case)
    dtype = case.get("dtype", "q4_0")
    if case["kind"] == "ingest":
        rows = [_kv_rows(case, seed, i, n) for i, n in enumerate(lens)]
        return tuple(torch.cat([_held(dtype, r[j]) for r in rows]) for j in range(2))
    q = _queries(case, seed, sum(new)).double()
    out = torch.zeros_like(q)
    scored = case["kind"] == "scored"
    prefix = first = None
    if scored:
        _, _, prefix, first = _layout(case)
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    row = 0
    for i, (length, m) in enumerate(zip(lens, new)):
        ks, vs = (_held(dtype, x) for x in _kv_rows(case, seed, i, length))
        hide = dist = None
        if scored:
            see = _visible(case, length, m, prefix[i] if prefix else None, first[row:row + m] if first else None)
            hide = _cuda(~see)
            dist = _cuda(np.abs(np.arange(length - m, length)[:, None] - np.arange(length)[None, :]).astype(np.float64))
        for h in range(heads):
            a = h // (heads // kv_heads) * hd
            s = torch.mm(q[row:row + m, h * hd:(h + 1) * hd].contiguous(), ks[:, a:a + hd].t().contiguous()) * scale
            if scored:
                if case["softcap"] > 0:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                if case["alibi"]:
                    s = s - float(_slopes(case)[h]) * dist
                s = s.masked_fill(hide, -math.inf)
            lse = torch.logsumexp(s, dim=1, keepdim=True)
            w = torch.exp(s - lse).masked_fill(lse == -math.inf, 0.0)
            out[row:row + m, h * hd:(h + 1) * hd] = torch.mm(w, vs[:, a:a + hd].contiguous())
        row += m
    return out
