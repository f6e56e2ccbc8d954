"""Decoding with trees of drafted tokens as measurable cases.

A step of such decoding lays out its drafted tokens on the GPU, appends their
rotated rows, attends over the cache with a tree's mask, and keeps the drafts
that the model agrees with. One pass of a case is one pass through an operator
as a user's program calls it. Where ``own`` is false the pass runs the
operator's plain form (elementary torch operations), where it is true the
framework's entry points:

* "layout": row starts, lengths, block tables, slots, positions and ancestor
  masks of a step from its requests' lengths (``step_layout``).
* "append": K rotated into its cells, V appended, Q rotated, with rotary
  frequencies scaled for long contexts and rows of 32 or 16 bits
  (``write_rope_rows``); the cells are read back as f32 values
  (``gather_values``), as code that takes contiguous rows does.
* "tree": attention of drafted rows over the cache (``tree_attention``).
* "accept": the end of a step: drafted rows appended in every layer, the
  accepted path found and its rows moved together (``accept_tree``), and the
  last blocks of every sequence read back.

Rotary positions: pair i of a head has the angle position * f_i in 64 bits; its
cosine and sine, times a magnitude, are held in single precision, and so is each
product and sum of the rotation. A drafted row sees its context and the drafted
rows whose bits its mask holds.

Lengths and trees are a function of the case alone (its "spread" seed), values
of the seed given to ``prepare``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16
LIMIT = 65280.0  # largest magnitude of a 4-bit cache

# (query heads, kv heads, head_dim)
LLAMA3_8B = (32, 8, 128)
QWEN25_7B = (28, 4, 128)
TINYLLAMA = (32, 4, 64)
SMOLLM2 = (9, 3, 64)


def _case(name, kind, shape, **kw):
    heads, kv_heads, head_dim = shape
    return {"name": name, "kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, **kw}


def _rope(name, kind, shape, **kw):
    base = {"dtype": "f16", "rows": "f32", "base": 10000.0, "rope_dim": shape[2], "half": True, "scaling": "none",
            "factor": 1.0, "original": 0}
    base.update(kw)
    return _case(name, kind, shape, **base)


def _tree(name, shape, **kw):
    base = {"dtype": "f16", "rows": "f32", "gain": 1.0, "softcap": 0.0, "window": 0, "branch": 0.4}
    base.update(kw)
    return _case(name, "tree", shape, **base)


def listed():
    return [
        # The server's decode batch, each request with a tree of drafts: launch latency.
        _case("layout-trees", "layout", LLAMA3_8B, batch=64, lo=1000, hi=4096, new_lo=16, new=64, tree=True, branch=0.4,
              spread=1),
        # A scheduling round that admits long prompts beside running decodes.
        _case("layout-prompts", "layout", LLAMA3_8B, batch=48, lo=0, hi=9000, new_lo=1, new=4096, tree=False,
              branch=0.0, spread=2),
        # A decode step's rows, half-precision activations, long-context frequencies.
        _rope("append-step", "append", LLAMA3_8B, rows="bf16", base=500000.0, scaling="llama3", factor=8.0,
              original=8192, batch=64, lo=1, hi=1, at=100000, spread=3),
        # Prompts of one scheduling round of a model stretched past its trained length.
        _rope("append-prompts", "append", QWEN25_7B, rows="bf16", base=1000000.0, scaling="yarn", factor=4.0,
              original=32768, batch=8, lo=500, hi=2000, at=30000, spread=4),
        # The interleaved layout on part of the head, f32 activations, an 8-bit cache.
        _rope("append-part-q8", "append", (32, 8, 96), dtype="q8_0", rope_dim=48, half=False, scaling="linear",
              factor=2.0, batch=3, lo=300, hi=900, at=0, spread=5),
        # A small local model, a short chat with a few drafts: launch latency.
        _tree("tree-chat", TINYLLAMA, batch=1, lo=400, hi=400, new_lo=8, new=8, spread=6),
        # The server's full decode batch with a small tree each, half-precision rows.
        _tree("tree-batch", LLAMA3_8B, rows="bf16", batch=64, lo=2048, hi=4096, new_lo=10, new=16, spread=7),
        # Long documents on an 8-bit cache, wide trees.
        _tree("tree-long-q8", QWEN25_7B, dtype="q8_0", batch=8, lo=32000, hi=32700, new_lo=40, new=48, spread=8),
        # A 4-bit cache, capped scores and a sliding window, trees of 64.
        _tree("tree-cap-q4", LLAMA3_8B, dtype="q4_0", rows="f16", gain=3.0, softcap=30.0, window=2048, batch=16,
              lo=500, hi=6000, new_lo=64, new=64, spread=9),
        # Another head width on an f32 cache, ragged trees.
        _tree("tree-odd-f32", (20, 4, 80), dtype="f32", batch=5, lo=17, hi=1500, new_lo=1, new=29, spread=10),
        # One user's step on a small model with an 8-bit cache.
        _rope("accept-chat-q8", "accept", TINYLLAMA, dtype="q8_0", rows="f16", batch=1, lo=777, hi=777, new_lo=13,
              new=13, branch=0.4, layers=2, spread=11),
        # The server's batch.
        _rope("accept-batch", "accept", LLAMA3_8B, rows="bf16", base=500000.0, batch=48, lo=100, hi=700, new_lo=20,
              new=64, branch=0.4, layers=4, spread=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# Shapes of the repository's configurations and tests; the last four are
# outside the common head_dim 64 / 128 and groups of up to 8.
COMMON = [LLAMA3_8B, QWEN25_7B, TINYLLAMA, SMOLLM2]
OTHER = [(32, 8, 96), (16, 1, 128), (8, 1, 256), (20, 4, 80)]


def _draw_rope(rng, shape):
    part = rng.random() < 0.3
    kind = rng.choice(["none", "linear", "ntk", "yarn", "llama3"])
    return {"dtype": rng.choice(["f16", "f16", "f32", "q8_0", "q4_0"]), "rows": rng.choice(["f32", "f16", "bf16"]),
            "base": rng.choice([10000.0, 500000.0, 1000000.0]),
            "rope_dim": shape[2] // 2 if part else shape[2], "half": rng.random() < 0.6, "scaling": kind,
            "factor": 1.0 if kind == "none" else rng.choice([2.0, 4.0, 8.0]),
            "original": rng.choice([4096, 8192]) if kind in ("yarn", "llama3") else 0}


def draw(rng):
    kind = rng.choice(["layout", "append", "append", "tree", "tree", "tree", "tree", "accept"])
    spread = rng.randrange(1 << 20)
    if kind == "layout":
        tree = rng.random() < 0.5
        batch = _log(rng, 1, 200)
        new = _log(rng, 1, 150) if tree else _log(rng, 1, max(2, 90000 // batch))
        hi = _log(rng, 1, 9000)
        return _case("", "layout", rng.choice(COMMON), batch=batch, lo=rng.choice([0, hi // 2]), hi=hi,
                     new_lo=rng.choice([0, 1, new]), new=new, tree=tree, branch=rng.choice([0.1, 0.5, 0.9]),
                     spread=spread)
    if kind == "append":
        shape = rng.choice(COMMON + OTHER)
        r = _draw_rope(rng, shape)
        if shape[2] % 32:  # (8-bit and 4-bit caches rotate whole groups of 32 elements)
            r["dtype"] = rng.choice(["f16", "f32"])
        batch = _log(rng, 1, 96)
        hi = _log(rng, 1, max(2, 9000 // batch))
        return _rope("", "append", shape, **r, batch=batch, lo=rng.choice([1, hi]), hi=hi,
                     at=rng.choice([0, rng.randrange(120000 - hi)]), spread=spread)
    if kind == "accept":
        shape = rng.choice(COMMON)
        new = _log(rng, 1, 80)
        batch = _log(rng, 1, min(64, max(2, 2500 // new)))
        hi = _log(rng, 1, 800)
        return _rope("", "accept", shape, **_draw_rope(rng, shape), batch=batch, lo=rng.choice([0, hi]), hi=hi,
                     new_lo=rng.choice([1, new]), new=new, branch=rng.choice([0.1, 0.4, 0.8]),
                     layers=rng.choice([1, 2, 4]), spread=spread)
    other = rng.random() < 0.2
    new = _log(rng, 1, 64)
    batch = _log(rng, 1, 72)
    hi = min(_log(rng, 16, 32768), (30000 if other else 200000) // batch + 16, (1000000 if other else 10000000) // (batch * new))
    return _tree("", rng.choice(OTHER if other else COMMON), dtype=rng.choice(["f16", "f16", "q8_0", "q4_0", "f32"]),
                 rows=rng.choice(["f32", "f16", "bf16"]), gain=rng.choice([1.0, 3.0]),
                 softcap=rng.choice([0.0, 0.0, 20.0]), window=rng.choice([0, 0, 0, _log(rng, 8, 3000)]), batch=batch,
                 lo=max(0, hi // rng.choice([1, 2, 8]) - rng.randrange(5)), hi=hi, new_lo=rng.choice([1, new]), new=new,
                 branch=rng.choice([0.1, 0.4, 0.8]), spread=spread)


# ---- sizes of a case ----------------------------------------------------------


def _dims(case):
    return case["heads"], case["kv_heads"], case["head_dim"], case["kv_heads"] * case["head_dim"]


CELL = {"f16": 2.0, "f32": 4.0, "q8_0": 1.0 + 2.0 / 32, "q4_0": 0.5 + 2.0 / 32}
ROWS = {"f32": 4, "f16": 2, "bf16": 2}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _requests(case):
    """Context lengths and new tokens of every request."""
    r = np.random.default_rng(case["spread"])
    n = case["batch"]
    if case["kind"] == "append":  # the context is not in this pass's cache
        return [case["at"]] * n, [int(x) for x in r.integers(case["lo"], case["hi"] + 1, n)]
    return ([int(x) for x in r.integers(case["lo"], case["hi"] + 1, n)],
            [int(x) for x in r.integers(case["new_lo"], case["new"] + 1, n)])


def _parents(case):
    """The parent of every drafted token, in its request: -1 for a root. A token
    continues the last one or branches off an earlier one."""
    r = np.random.default_rng(case["spread"] + 1)
    trees = []
    for m in _requests(case)[1]:
        trees.append([-1] + [int(r.integers(0, j)) if r.random() < case["branch"] else j - 1 for j in range(1, m)])
    return [t[:m] for t, m in zip(trees, _requests(case)[1])]


def _words(case):
    return (max(1, max(_requests(case)[1])) + 31) // 32


def _path(parents, tokens, targets):
    """The drafts of one request that its model agrees with."""
    path = [0] if parents else []
    while path:
        nxt = [j for j in range(path[-1] + 1, len(parents))
               if parents[j] == path[-1] and tokens[j] == targets[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path


def work(case):
    heads, kv_heads, hd, kvd = _dims(case)
    ctx, new = _requests(case)
    rows, n = sum(new), len(new)
    kind = case["kind"]
    if kind == "layout":
        blocks = sum((c + m + BLOCK - 1) // BLOCK for c, m in zip(ctx, new))
        masks = rows * (4 + 4 * _words(case)) if case["tree"] else 0
        return {"bytes": float(8 * blocks + 8 * rows + 20 * n + masks), "flops": 0.0}
    size = ROWS[case["rows"]]
    cell = CELL[case["dtype"]]
    append = rows * (2 * kvd * (size + cell) + 2 * heads * hd * size)
    rotate = 3.0 * rows * (heads + kv_heads) * case.get("rope_dim", 0)
    if kind == "append":
        return {"bytes": append + rows * 2 * kvd * (cell + 4), "flops": rotate}
    if kind == "accept":
        layers = case["layers"]
        tail = sum(c % BLOCK + m for c, m in zip(ctx, new))
        return {"bytes": layers * (append + tail * 2 * kvd * (cell + 4)) + rows * 12.0, "flops": layers * rotate}
    total = cells = 0
    for c, m, see in zip(ctx, new, _visible(case)):
        total += int(see.sum())
        cells += int(see.any(axis=0).sum())
    return {"bytes": 2 * cells * kvd * cell + 2 * rows * heads * hd * size, "flops": 4.0 * heads * hd * total}


def _visible(case):
    """Of every request, [m][context + m] on the host: the positions that its rows see."""
    out = []
    for c, m, parents in zip(*_requests(case), _parents(case)):
        see = np.zeros((m, c + m), bool)
        depth = np.zeros(m, np.int64)
        for j, p in enumerate(parents):
            if p >= 0:
                see[j, c:] = see[p, c:]
                depth[j] = depth[p] + 1
            see[j, c + j] = True
        see[:, :c] = True
        if case.get("window"):
            see[:, :c] = np.arange(c)[None, :] > c + depth[:, None] - case["window"]
        out.append(see)
    return out


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


def _cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def _projections(case, seed, layer, rows):
    """One layer's Q, K and V rows as the projections leave them."""
    heads, _, hd, kvd = _dims(case)
    dtype = TYPES[case["rows"]]
    q, k, v = (_normal(seed, 16 + 3 * layer + j, rows, w) for j, w in ((0, heads * hd), (1, kvd), (2, kvd)))
    return q.to(dtype), (k * torch.exp(0.4 * _normal(seed, 1, 1, kvd))).to(dtype), v.to(dtype)


def _words_of(see, ctx, words):
    """Mask words of [m][context + m] visibility: bit j % 32 of word j / 32 is drafted row j."""
    m = see.shape[0]
    bits = np.zeros((m, words * 32), bool)
    bits[:, :m] = see[:, ctx:]
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)


def _tokens(case, seed):
    """Drafted tokens, and the model's token behind each of them: a likely draft's
    or another one."""
    r = np.random.default_rng(seed * 7 + case["spread"])
    tokens, targets = [], []
    for parents in _parents(case):
        m = len(parents)
        tok = [int(x) for x in r.integers(0, 32000, m)]
        want = []
        for j in range(m):
            below = [k for k in range(j + 1, m) if parents[k] == j]
            want.append(tok[below[int(r.integers(0, len(below)))]] if below and r.random() < 0.8 else
                        int(r.integers(0, 32000)))
        tokens += tok
        targets += want
    return tokens, targets


def _cells(table, positions):
    return (np.asarray(table)[positions // BLOCK] * BLOCK + positions % BLOCK).astype(np.int32)


def prepare(case, seed):
    heads, _, hd, kvd = _dims(case)
    kind = case["kind"]
    ctx, new = _requests(case)
    n, rows = len(new), sum(new)
    dtype = case.get("dtype", "f16")
    held = [0] * n if kind == "append" else ctx  # tokens of the context in this cache
    need = [-(-(c + m) // BLOCK) for c, m in zip(held, new)]
    width = max(1, max(need))
    n_blocks = sum(need) + sum(need) // 10 + 1
    order = np.random.default_rng(seed).permutation(n_blocks)  # a fragmented pool
    layers = case.get("layers", 1)
    tables = np.full((n, width), -1, np.int32)
    at = 0
    for i, b in enumerate(need):
        tables[i, :b] = order[at:at + b]
        at += b
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    st = {"case": case, "ctx": ctx, "new": new, "dtype": dtype, "layers": layers}
    small = kind == "layout"  # no rows of K and V
    if own:
        from langtrain_studio_amd import KvCache

        kv = st["kv"] = KvCache(layers, 32 if small else kvd, n_blocks * BLOCK, dtype=dtype,
                                stream=torch.cuda.current_stream())
        kv.init_free_order(order)
        for i, (c, m) in enumerate(zip(held, new)):
            kv.append_batch(np.full(c + m, i, np.uint32), np.arange(c + m, dtype=np.uint64))

        def store(layer, where, k, v):
            kv.write_batch(layer, where, k, v)
    elif not small:
        st["pool"] = [[_empty_pool(dtype, n_blocks, kvd) for _ in range(2)] for _ in range(layers)]

        def store(layer, where, k, v):
            _store(dtype, st["pool"][layer][0], where, k)
            _store(dtype, st["pool"][layer][1], where, v)

    if kind == "layout":
        st["lens"], st["counts"] = _cuda(np.array(ctx, np.int32)), _cuda(np.array(new, np.int32))
        st["parents"] = None
        st["words"] = _words(case) if case["tree"] else 0
        if case["tree"]:
            st["parents"] = _cuda(np.array(sum(_parents(case), []), np.int32))
        st["capacity"] = rows + rows // 8 + 1  # a captured step's arrays have room for more
        if st["parents"] is not None:
            st["parents"] = torch.nn.functional.pad(st["parents"], (0, st["capacity"] - rows), value=-1)
        st["width"] = width
        if own:
            st["rows"] = _cuda(kv.seq_rows(np.arange(n, dtype=np.uint32)))
            st["out"] = kv.step_layout(st["rows"], st["lens"], st["counts"], st["capacity"], width,
                                       parents=st["parents"], mask_words=st["words"])
        else:
            st["resident"] = _cuda(tables)
        torch.cuda.synchronize()
        return st
    st["lens"] = _cuda(np.array([c + m for c, m in zip(held, new)], np.int32))
    st["tables"] = _cuda(np.maximum(tables, 0))
    st["starts"] = _cuda(starts)
    if kind in ("append", "accept"):
        st["slots"] = _cuda(np.concatenate([_cells(tables[i], held[i] + np.arange(m)) for i, m in enumerate(new)]))
        if kind == "append":
            depth = [np.arange(m) for m in new]
        else:
            depth = [_depths(p) for p in _parents(case)]
        st["positions"] = _cuda(np.concatenate([c + d for c, d in zip(ctx, depth)]).astype(np.int32))
        top = max(c + m for c, m in zip(ctx, new))
        if own:
            kv.rope_init_scaled(case["base"], case["rope_dim"], hd, case["half"], top, kind=case["scaling"],
                                factor=case["factor"], original=case["original"])
        else:
            st["rope"] = _rope_table(case, top)
        st["qkv"] = [_projections(case, seed, layer, rows) for layer in range(layers)]
        st["q_out"] = [torch.empty_like(q) for q, _, _ in st["qkv"]]
        # the blocks that this pass's rows lie in, read back whole
        first = [c // BLOCK for c in held]
        tails = [need[i] - first[i] for i in range(n)]
        tail = np.zeros((n, max(1, max(tails))), np.int32)
        for i in range(n):
            tail[i, :tails[i]] = tables[i, first[i]:need[i]]
        st["tail"] = _cuda(tail)
        st["tail_lens_host"] = [c % BLOCK + m for c, m in zip(held, new)]
        st["tail_lens"] = _cuda(np.array(st["tail_lens_host"], np.int32))
        total = sum(st["tail_lens_host"])
        st["offsets"] = _cuda(np.concatenate([[0], np.cumsum(st["tail_lens_host"])[:-1]]).astype(np.int64))
        st["k_out"] = [torch.empty((total, kvd), device="cuda") for _ in range(layers)]
        st["v_out"] = [torch.empty((total, kvd), device="cuda") for _ in range(layers)]
    if kind == "accept":
        for i in range(n):  # the rows in front of the drafts in their first block
            p = np.arange(ctx[i] // BLOCK * BLOCK, ctx[i])
            if p.size:
                k, v = _kv_rows(case, seed, i, p.size)
                for layer in range(layers):
                    store(layer, _cuda(_cells(tables[i], p)), k, v)
        tokens, targets = _tokens(case, seed)
        st["tokens"], st["targets"] = _cuda(np.array(tokens, np.int32)), _cuda(np.array(targets, np.int32))
        st["parents"] = _cuda(np.array(sum(_parents(case), []), np.int32))
    if kind == "tree":
        for i, (c, m) in enumerate(zip(ctx, new)):  # contexts and drafted rows are in the cache already
            k, v = _kv_rows(case, seed, i, c + m)
            store(0, _cuda(_cells(tables[i], np.arange(c + m))), k, v)
        st["q"] = (_normal(seed, 2, rows, heads * hd) * case["gain"]).to(TYPES[case["rows"]])
        see = _visible(case)
        st["positions"] = _cuda(np.concatenate([c + _depths(p) for c, p in zip(ctx, _parents(case))]).astype(np.int32))
        st["masks"] = _cuda(np.concatenate([_words_of(s, c, _words(case)) for s, c in zip(see, ctx)]))
        st["out"] = torch.empty_like(st["q"])
    torch.cuda.synchronize()
    return st


def _depths(parents):
    depth = np.zeros(len(parents), np.int64)
    for j, p in enumerate(parents):
        depth[j] = depth[p] + 1 if p >= 0 else 0
    return depth


# ---- the plain forms ------------------------------------------------------------


def _frequencies(case):
    """Angle a position adds to each pair, and the rotation's magnitude."""
    base, d, kind, factor, original = (case[x] for x in ("base", "rope_dim", "scaling", "factor", "original"))
    if kind == "ntk":
        base = base * factor ** (d / (d - 2.0))
    f = [base ** (-2.0 * i / d) for i in range(d // 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    if kind == "llama3":
        low, high = 1.0, 4.0
        for i, x in enumerate(f):
            turns = original * x / (2.0 * math.pi)
            blend = min(max((turns - low) / (high - low), 0.0), 1.0)
            f[i] = x / factor * (1.0 - blend) + x * blend
    if kind == "yarn":
        slow, fast = 1.0, 32.0

        def pair(turns):
            return d * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), d - 1)
        for i, x in enumerate(f):
            blend = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f[i] = x / factor * blend + x * (1.0 - blend)
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rope_table(case, top):
    """(cosines, sines) f32 [top][rope_dim / 2], their magnitude included."""
    f, size = _frequencies(case)
    size = float(np.float32(size))
    angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * torch.tensor(f, device="cuda",
                                                                                        dtype=torch.float64)
    return (torch.cos(angle) * size).float(), (torch.sin(angle) * size).float()


def _rotate(case, x, cos, sin):
    """f32 rows [n][heads * hd] rotated by [n][rope_dim / 2] cosines and sines."""
    hd, d = case["head_dim"], case["rope_dim"]
    x = x.reshape(x.shape[0], -1, hd)
    cos, sin = cos[:, None, :], sin[:, None, :]
    a, b = (x[..., :d // 2], x[..., d // 2:d]) if case["half"] else (x[..., 0:d:2], x[..., 1:d:2])
    u = a * cos
    u = u - b * sin
    w = a * sin
    w = w + b * cos
    y = x.clone()
    if case["half"]:
        y[..., :d // 2], y[..., d // 2:d] = u, w
    else:
        y[..., 0:d:2], y[..., 1:d:2] = u, w
    return y.reshape(x.shape[0], -1)


def _quantise4(x):
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
        pool[0][cells], pool[1][cells] = _quantise4(x)
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


def _plain_layout(st):
    """Row starts, lengths, tables, slots, positions and masks of a step."""
    lens, counts, capacity, width = st["lens"].long(), st["counts"].long(), st["capacity"], st["width"]
    ends = torch.cumsum(counts, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    after = lens + counts
    block = torch.arange(width, device="cuda")[None, :]
    tables = torch.where(block < (after[:, None] + BLOCK - 1) // BLOCK, st["resident"],
                         torch.full_like(st["resident"], -1))
    token = torch.arange(capacity, device="cuda")
    req = torch.searchsorted(ends, token, right=True)
    live = req < counts.numel()
    req = req.clamp(max=counts.numel() - 1)
    place = token - starts[req]
    cell = lens[req] + place
    entry = tables[req, (cell // BLOCK).clamp(max=width - 1)].long()
    slots = torch.where(live, entry * BLOCK + cell % BLOCK, torch.full_like(cell, -1))
    positions = cell
    out = {"row_starts": starts.int(), "lens": after.int(), "tables": tables, "slot_mapping": slots.int()}
    if st["parents"] is not None:
        words = st["words"]
        masks = torch.zeros((capacity, words), dtype=torch.int64, device="cuda")
        depth = torch.full_like(token, -1)
        node, here = place, live
        parents = st["parents"].long()
        for _ in range(int(st["case"]["new"])):  # every row at once, a step up its tree a time
            depth = depth + here
            word = torch.where(here, node // 32, torch.zeros_like(node))
            bit = torch.where(here, 1 << (node % 32), torch.zeros_like(node))
            masks[token, word] |= bit
            node = torch.where(here, parents[(starts[req] + node).clamp(0, capacity - 1)], node)
            here = here & (node >= 0)
        out["masks"] = torch.where(masks >= 1 << 31, masks - (1 << 32), masks).int()
        positions = lens[req] + depth
    out["positions"] = torch.where(live, positions, torch.full_like(positions, -1)).int()
    return out


def _plain_append(st, layer):
    case, dtype = st["case"], st["dtype"]
    q, k, v = st["qkv"][layer]
    at = st["positions"].long()
    cos, sin = st["rope"][0][at], st["rope"][1][at]
    _store(dtype, st["pool"][layer][0], st["slots"], _rotate(case, k.float(), cos, sin))
    _store(dtype, st["pool"][layer][1], st["slots"], v.float())
    return _rotate(case, q.float(), cos, sin).to(q.dtype)


def _plain_tail(st, layer):
    return tuple(torch.cat([_load(st["dtype"], st["pool"][layer][j], st["tail"][i], m)
                            for i, m in enumerate(st["tail_lens_host"])]) for j in range(2))


def _plain_accept(st):
    """The accepted path of every request, and its rows moved together."""
    case, starts = st["case"], st["starts"].long()
    n, rows = starts.numel() - 1, st["tokens"].numel()
    first, count = starts[:-1], starts[1:] - starts[:-1]
    top = int(case["new"])
    j = torch.arange(top, device="cuda")[None, :]
    inside = j < count[:, None]
    at = (first[:, None] + j).clamp(max=rows - 1)
    parents = torch.where(inside, st["parents"].long()[at], torch.full_like(at, -2))
    tokens, targets = st["tokens"].long()[at], st["targets"].long()[at]
    path = torch.full((n, top), -1, dtype=torch.int64, device="cuda")
    accepted = torch.zeros(n, dtype=torch.int64, device="cuda")
    cur, going = torch.zeros(n, dtype=torch.int64, device="cuda"), count > 0
    after = torch.full_like(cur, -1)
    for _ in range(top):
        path.scatter_(1, accepted[:, None].clamp(max=top - 1),
                      torch.where(going, cur, path.gather(1, accepted[:, None].clamp(max=top - 1))[:, 0])[:, None])
        accepted = accepted + going
        want = targets.gather(1, cur[:, None])
        after = torch.where(going, want[:, 0], after)
        match = inside & (parents == cur[:, None]) & (tokens == want) & (j > cur[:, None])
        going = going & match.any(dim=1)
        cur = torch.where(going, match.int().argmax(dim=1), cur)
    base = st["lens"].long() - count
    moves = path >= 0
    tables = st["tables"].long()

    def cell(position):
        p = torch.where(moves, position, torch.zeros_like(position))
        return tables.gather(1, p // BLOCK) * BLOCK + p % BLOCK

    src, dst = cell(base[:, None] + path)[moves], cell(base[:, None] + j.expand(n, -1))[moves]
    for layer in st["pool"]:
        for pool in layer:
            for part in pool if isinstance(pool, tuple) else (pool,):
                part[dst] = part[src]
    flat = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    flat[at[inside]] = path[inside]
    return {"accepted": accepted.int(), "path": flat.int(), "next": after.int(), "lens": (base + accepted).int()}


def _plain_attention(case, q, k, v, see):
    """q [m][heads * hd], k and v [length][kvd] (f32); see [m][length]."""
    heads, kv_heads, hd, _ = _dims(case)
    g, m, length = heads // kv_heads, q.shape[0], k.shape[0]
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    qh = q.reshape(m, kv_heads, g, hd).permute(1, 2, 0, 3).reshape(kv_heads, g * m, hd).contiguous()
    kh = k.reshape(length, kv_heads, hd).permute(1, 2, 0).contiguous()
    vh = v.reshape(length, kv_heads, hd).permute(1, 0, 2).contiguous()
    s = (torch.matmul(qh, kh) * scale).reshape(kv_heads, g, m, length)
    if case["softcap"] > 0:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    top = s.amax(dim=3, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=3, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p.reshape(kv_heads, g * m, length), vh)
    return o.reshape(kv_heads, g, m, hd).permute(2, 0, 1, 3).reshape(m, heads * hd)


def _plain_tree(st):
    case, dtype = st["case"], st["dtype"]
    out = torch.empty_like(st["q"])
    row = 0
    for i, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        if m == 0:
            continue
        k = _load(dtype, st["pool"][0][0], st["tables"][i], c + m)
        v = _load(dtype, st["pool"][0][1], st["tables"][i], c + m)
        node = torch.arange(m, device="cuda")
        words = st["masks"][row:row + m].long()
        drafted = (words[:, node // 32] >> (node % 32)[None, :]) & 1
        t = torch.arange(c, device="cuda")[None, :]
        before = t >= 0
        if case["window"]:
            before = t > st["positions"][row:row + m].long()[:, None] - case["window"]
        see = torch.cat([before.expand(m, c), drafted > 0], dim=1)
        out[row:row + m] = _plain_attention(case, st["q"][row:row + m].float(), k, v, see).to(out.dtype)
        row += m
    return out


def _run_plain(st):
    kind = st["case"]["kind"]
    if kind == "layout":
        return _plain_layout(st)
    if kind == "tree":
        return _plain_tree(st)
    if kind == "append":
        q = _plain_append(st, 0)
        return (q,) + _plain_tail(st, 0)
    q = [_plain_append(st, layer) for layer in range(st["layers"])]
    out = _plain_accept(st)
    tails = [_plain_tail(st, layer) for layer in range(st["layers"])]
    return {**out, "q": q, "k": [t[0] for t in tails], "v": [t[1] for t in tails]}


def run(st):
    if not own:
        return _run_plain(st)
    case, kv = st["case"], st["kv"]
    heads, _, hd, _ = _dims(case)
    if case["kind"] == "layout":
        step = kv.step_layout(st["rows"], st["lens"], st["counts"], st["capacity"], st["width"],
                              parents=st["parents"], mask_words=st["words"], out=st["out"])
        out = {"row_starts": step.row_starts, "lens": step.lens, "tables": step.tables,
               "slot_mapping": step.slot_mapping, "positions": step.positions}
        if st["parents"] is not None:
            out["masks"] = step.masks
        return out
    if case["kind"] == "tree":
        return kv.tree_attention(0, st["q"], st["tables"], st["lens"], heads, hd, st["starts"],
                                 positions=st["positions"], masks=st["masks"], max_rows=max(st["new"]),
                                 softcap=case["softcap"], window=case["window"], out=st["out"])

    def append(layer):
        q, k, v = st["qkv"][layer]
        kv.write_rope_rows(layer, st["slots"], st["positions"], k, v, q=q, n_heads=heads, out=st["q_out"][layer])

    def tail(layer):
        kv.gather_values(layer, st["tail"], st["tail_lens"], st["offsets"], st["k_out"][layer], st["v_out"][layer])

    if case["kind"] == "append":
        append(0)
        tail(0)
        return st["q_out"][0], st["k_out"][0], st["v_out"][0]
    for layer in range(st["layers"]):
        append(layer)
    done = kv.accept_tree(st["tables"], st["lens"], st["starts"], st["parents"], st["tokens"], st["targets"])
    for layer in range(st["layers"]):
        tail(layer)
    return {"accepted": done.accepted, "path": done.path, "next": done.next, "lens": done.lens, "q": st["q_out"],
            "k": st["k_out"], "v": st["v_out"]}


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


def _turned(case, x, positions):
    """Rows turned by their positions' angles: in 64 bits, with the roundings to
    single precision that the definition has."""
    hd, d = case["head_dim"], case["rope_dim"]
    f, size = _frequencies(case)
    size = float(np.float32(size))
    z = x.double().view(x.shape[0], -1, hd).clone()
    for i in range(d // 2):
        angle = positions.double() * f[i]
        c, s = ((t * size).float().double()[:, None] for t in (angle.cos(), angle.sin()))
        a, b = (i, i + d // 2) if case["half"] else (2 * i, 2 * i + 1)
        p, r = z[:, :, a].clone(), z[:, :, b].clone()
        z[:, :, a] = ((p * c).float().double() - (r * s).float().double()).float().double()
        z[:, :, b] = ((p * s).float().double() + (r * c).float().double()).float().double()
    return z.view(x.shape)


def _exact_tree(case, seed):
    heads, kv_heads, hd, _ = _dims(case)
    ctx, new = _requests(case)
    q = (_normal(seed, 2, sum(new), heads * hd) * case["gain"]).to(TYPES[case["rows"]]).double()
    out = torch.zeros_like(q)
    scale = float(np.float32(1.0 / math.sqrt(hd)))
    row = 0
    for i, (c, m, see) in enumerate(zip(ctx, new, _visible(case))):
        ks, vs = (_held(case["dtype"], x) for x in _kv_rows(case, seed, i, c + m))
        hide = _cuda(~see)
        for h in range(heads):
            a = h // (heads // kv_heads) * hd
            s = torch.mm(q[row:row + m, h * hd:(h + 1) * hd].contiguous(), ks[:, a:a + hd].t().contiguous()) * scale
            if case["softcap"] > 0:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s = s.masked_fill(hide, -math.inf)
            lse = torch.logsumexp(s, dim=1, keepdim=True)
            w = torch.exp(s - lse).masked_fill(lse == -math.inf, 0.0)
            out[row:row + m, h * hd:(h + 1) * hd] = torch.mm(w, vs[:, a:a + hd].contiguous())
        row += m
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "tree":
        return _exact_tree(case, seed)
    ctx, new = _requests(case)
    if kind == "layout":  # whole numbers: the plain form's are exact
        return None
    if kind == "append":
        positions = _cuda(np.concatenate([c + np.arange(m) for c, m in zip(ctx, new)]))
        q, k, v = (x.float() for x in _projections(case, seed, 0, sum(new)))
        return (_turned(case, q, positions), _held(case["dtype"], _turned(case, k, positions).float()),
                _held(case["dtype"], v))
    parents = _parents(case)
    tokens, targets = _tokens(case, seed)
    at = np.concatenate([[0], np.cumsum(new)])
    paths = [_path(p, tokens[a:b], targets[a:b]) for p, a, b in zip(parents, at, at[1:])]
    positions = _cuda(np.concatenate([c + _depths(p) for c, p in zip(ctx, parents)]))
    res = {"q": [], "k": [], "v": []}
    for layer in range(case["layers"]):
        q, k, v = (x.float() for x in _projections(case, seed, layer, sum(new)))
        res["q"].append(_turned(case, q, positions))
        kept = {"k": _held(case["dtype"], _turned(case, k, positions).float()), "v": _held(case["dtype"], v)}
        for name in ("k", "v"):
            tails = []
            for i, (c, path) in enumerate(zip(ctx, paths)):
                part = kept[name][at[i]:at[i + 1]].clone()
                part[:len(path)] = kept[name][at[i]:at[i + 1]][path]
                if c % BLOCK:
                    before = _kv_rows(case, seed, i, c % BLOCK)[0 if name == "k" else 1]
                    part = torch.cat([_held(case["dtype"], before), part])
                tails.append(part)
            res[name].append(torch.cat(tails))
    return {"accepted": None, "path": None, "next": None, "lens": None, **res}
