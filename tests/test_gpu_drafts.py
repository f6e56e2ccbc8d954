"""Steps with drafted tokens from end to end: begin_drafts, draft_layer and accept of
the backend against the same tokens decoded one at a time, captured layers, other
streams, and calls that overlap."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_scored import BLOCK, held_rows
from test_gpu_tree import Trees, up
from tree_definition import compare, definition, depths, random_tree, visible, ancestors

pytestmark = pytest.mark.gpu

HEADS, KVH, HD, LAYERS = 8, 2, 64, 2


def backend(dtype="f16", tokens=2000, stream=None):
    from langtrain_studio_amd import PagedKvBackend

    b = PagedKvBackend(LAYERS, HEADS, KVH, HD, tokens, n_seq_max=8, n_batch=256, dtype=dtype, stream=stream)
    b.kv.rope_init_scaled(10000.0, HD, HD, True, 512, kind="yarn", factor=2.0, original=128)
    return b


def projections(token, layer, dtype):
    """One layer's Q, K and V rows of a token: a function of the token alone."""
    import torch

    r = np.random.default_rng(1000 * layer + token)
    return [torch.from_numpy(r.standard_normal((1, w), dtype=np.float32)).to("cuda", dtype)
            for w in (HEADS * HD, KVH * HD, KVH * HD)]


def rows_of(tokens, layer, dtype):
    import torch

    return [torch.cat(x).contiguous() for x in zip(*(projections(t, layer, dtype) for t in tokens))]


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
def test_drafted_steps_match_single_tokens(gpu, dtype, rows):
    """Three steps of three sequences (two forked from one prompt): every kept
    row's attention is the definition's over its own sequence, the sequences' rows
    are those of the tokens kept, bit by bit, and shared blocks stay the other
    sequence's."""
    import torch

    from langtrain_studio_amd import Drafts

    td = {"f32": torch.float32, "bf16": torch.bfloat16}[rows]
    b, plain = backend(dtype), backend(dtype)
    rng = np.random.default_rng(7)
    history = {0: list(rng.integers(0, 50, 37)), 1: [], 2: list(rng.integers(0, 50, 5))}
    for x in (b, plain):
        for s in (0, 2):
            n = len(history[s])
            cells = x.kv.append_batch(np.full(n, s, np.uint32), np.arange(n, dtype=np.uint64))
            for layer in range(LAYERS):
                _, k, v = rows_of(history[s], layer, td)
                x.kv.write_rope_rows(layer, up(cells, np.int32), up(np.arange(n), np.int32), k, v)
        x.kv_copy(0, 1, 30)  # a block shared in part
    history[1] = history[0][:30]
    for step in range(3):
        trees, tokens, targets = [], [], []
        for s in range(3):
            m = int(rng.integers(1, 40))
            parents = random_tree(rng, m, 0.3)
            tok = rng.integers(0, 50, m)
            want = rng.integers(0, 50, m)
            for j in range(1, m):
                if rng.random() < 0.7:
                    want[parents[j]] = tok[j]
            trees.append(parents)
            tokens.append(tok)
            targets.append(want)
        lens = [len(history[s]) for s in range(3)]
        at = b.begin_drafts([Drafts(s, p) for s, p in enumerate(trees)])
        flat = [int(t) for x in tokens for t in x]
        outs, held = [], []
        for layer in range(LAYERS):
            q, k, v = rows_of(flat, layer, td)
            outs.append(b.draft_layer(at, layer, q, k, v).float().cpu().numpy())
            held.append(held_rows(b.kv, layer))
        # the definition over this cache's rows (before they move), Q turned as the cache turns it
        tables, starts = at.layout.tables.cpu().numpy(), at.layout.row_starts.cpu().numpy()
        sees = [visible(c + len(p), ancestors(p)) for c, p in zip(lens, trees)]
        for layer in range(LAYERS):
            q, k, v = rows_of(flat, layer, td)
            turned = plain.kv.write_rope_rows(layer, torch.full_like(at.layout.slot_mapping, -1), at.layout.positions,
                                              k, v, q=q, n_heads=HEADS)
            compare(outs[layer], definition(turned.float().cpu().numpy(), held[layer], tables,
                                            [c + len(p) for c, p in zip(lens, trees)], starts, HEADS, HD, sees, rows=rows,
                                            eight=dtype in ("q8_0", "f32")))
        kept, done = b.accept(at, up(np.concatenate(tokens), np.int32), up(np.concatenate(targets), np.int32))
        for s in range(3):
            path = [j for j in done.path[starts[s]:starts[s + 1]].tolist() if j >= 0]
            assert len(path) == kept[s] and path[0] == 0
            for a, c in zip(path, path[1:]):
                assert trees[s][c] == a and tokens[s][c] == targets[s][a]
            new = [int(tokens[s][j]) for j in path]
            pos = np.arange(lens[s], lens[s] + len(new), dtype=np.uint64)
            for i, t in enumerate(new):  # one token at a time
                cell = plain.kv.append_batch(np.array([s], np.uint32), pos[i:i + 1])
                for layer in range(LAYERS):
                    _, k, v = projections(t, layer, td)
                    plain.kv.write_rope_rows(layer, up(cell, np.int32), up(pos[i:i + 1], np.int32), k, v)
            history[s] = history[s] + new
    plain.kv.synchronize()
    for s in range(3):
        n = len(history[s])
        assert b.kv.len(s) == plain.kv.len(s) == n
        p = np.arange(n)
        a, c = (x.kv.block_table(s)[p // BLOCK] * BLOCK + p % BLOCK for x in (b, plain))
        for layer in range(LAYERS):
            for x, y in zip(held_rows(b.kv, layer), held_rows(plain.kv, layer)):
                np.testing.assert_array_equal(x[a], y[c])


def test_begin_drafts_is_all_or_nothing(gpu):
    from langtrain_studio_amd import Drafts, KvCacheFull

    b = backend(tokens=64)
    b.kv.append_batch(np.zeros(20, np.uint32), np.arange(20, dtype=np.uint64))
    free = b.kv.free_blocks()
    with pytest.raises(KvCacheFull):
        b.begin_drafts([Drafts(0, [-1] + list(range(9))), Drafts(1, [-1] + list(range(60)))])
    assert b.kv.len(0) == 20 and b.kv.len(1) == 0 and b.kv.free_blocks() == free
    for match, bad in [("distinct", [Drafts(0, [-1]), Drafts(0, [-1])]), ("at least one", [Drafts(0, [])]),
                       ("parents of sequence 0", [Drafts(0, [-1, 1])]), ("parents", [Drafts(0, [0])]),
                       ("n_batch", [Drafts(0, [-1] + list(range(256)))])]:
        with pytest.raises(ValueError, match=match):
            b.begin_drafts(bad)
    step = b.begin_drafts([Drafts(0, [-1, 0])])
    b.kv_remove(0, 21)
    with pytest.raises(RuntimeError, match="changed since"):
        b.accept(step, step.parents, step.parents)
    empty = b.begin_drafts([])
    assert empty.n == 0


def test_captured_layers(gpu):
    """A step's layers captured once and replayed with other rows, eager work and
    synchronizations between: each replay gives the eager result."""
    import torch

    from langtrain_studio_amd import Drafts

    side = torch.cuda.Stream()
    b = backend(stream=side)
    rng = np.random.default_rng(3)
    with torch.cuda.stream(side):
        n = 300
        cells = b.kv.append_batch(np.zeros(n, np.uint32), np.arange(n, dtype=np.uint64))
        for layer in range(LAYERS):
            _, k, v = rows_of(rng.integers(0, 50, n), layer, torch.float32)
            b.kv.write_rope_rows(layer, up(cells, np.int32), up(np.arange(n), np.int32), k, v)
        step = b.begin_drafts([Drafts(0, random_tree(rng, 20, 0.3)), Drafts(1, random_tree(rng, 7, 0.3))])
        fixed = [rows_of(rng.integers(0, 50, step.n), layer, torch.bfloat16) for layer in range(LAYERS)]
        out = [torch.zeros_like(x[0]) for x in fixed]
        for layer in range(LAYERS):  # (sizes what is sized on demand)
            b.draft_layer(step, layer, *fixed[layer], out=out[layer])
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for layer in range(LAYERS):
            b.draft_layer(step, layer, *fixed[layer], out=out[layer])
    for turn in range(4):
        with torch.cuda.stream(side):
            for layer in range(LAYERS):
                for x, y in zip(fixed[layer], rows_of(rng.integers(0, 50, step.n), layer, torch.bfloat16)):
                    x.copy_(y)
        side.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [x.clone() for x in out]
        with torch.cuda.stream(side):
            for layer in range(LAYERS):
                out[layer].zero_()
                b.draft_layer(step, layer, *fixed[layer], out=out[layer])
                assert torch.equal(out[layer], replayed[layer]), (turn, layer)
            if turn == 1:  # an acceptance's launch between
                b.kv.accept_tree(step.layout.tables, step.layout.lens, step.layout.row_starts, step.parents,
                                 torch.zeros_like(step.parents), torch.ones_like(step.parents))
        b.kv.synchronize()


def test_captured_acceptance(gpu):
    """Layers and the acceptance in one graph, replayed with other choices of the
    model: paths, lengths and the moved rows are those of eager calls."""
    import torch

    from langtrain_studio_amd import AcceptedTree, Drafts

    side = torch.cuda.Stream()
    rng = np.random.default_rng(5)
    trees = [random_tree(rng, 24, 0.3), random_tree(rng, 9, 0.2)]
    tokens = rng.integers(0, 3, 33)
    made = []
    for _ in range(2):  # a cache that replays and one that is eager
        b = backend("q8_0", stream=side)
        with torch.cuda.stream(side):
            cells = b.kv.append_batch(np.zeros(37, np.uint32), np.arange(37, dtype=np.uint64))
            for layer in range(LAYERS):
                _, k, v = rows_of(np.arange(37), layer, torch.float32)
                b.kv.write_rope_rows(layer, up(cells, np.int32), up(np.arange(37), np.int32), k, v)
            step = b.begin_drafts([Drafts(0, trees[0]), Drafts(1, trees[1])])
        rows = [rows_of(tokens, layer, torch.bfloat16) for layer in range(LAYERS)]
        made.append((b, step, rows, up(tokens, np.int32), up(np.zeros(33), np.int32),
                     AcceptedTree(*[torch.empty(m, dtype=torch.int32, device="cuda") for m in (2, 33, 2, 2)]),
                     [torch.empty_like(x[0]) for x in rows]))
    torch.cuda.synchronize()

    def run(b, step, rows, drafted, targets, done, outs):
        at = step.layout
        for layer in range(LAYERS):
            b.draft_layer(step, layer, *rows[layer], out=outs[layer])
        b.kv.accept_tree(at.tables, at.lens, at.row_starts, step.parents, drafted, targets, out=done)

    with torch.cuda.stream(side):
        for x in made:
            run(*x)  # (sizes what is sized on demand)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(*made[0])
    kept = set()
    for turn in range(4):
        targets = up(rng.integers(0, 3, 33), np.int32)
        for x in made:
            x[4].copy_(targets)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            run(*made[1])
        for x in made:
            x[0].kv.synchronize()
        for g, w in zip(made[0][5], made[1][5]):
            assert torch.equal(g, w), turn
        kept.add(tuple(made[0][5].accepted.tolist()))
        for layer in range(LAYERS):
            assert torch.equal(made[0][6][layer], made[1][6][layer])
            for x, y in zip(made[0][0].kv.read_pool(layer), made[1][0].kv.read_pool(layer)):
                np.testing.assert_array_equal(x, y)
    assert len(kept) > 1


@pytest.mark.parametrize("shape", [(8, 8, 128), (51, 51, 20)])
@pytest.mark.parametrize("dtype,size", [("f16", 2), ("f32", 4), ("q8_0", 1), ("q4_0", 0.5)])
def test_cells_past_32_bits(gpu, dtype, size, shape):
    """Rows that lie more than 2^32 bytes behind a pool's start: the same bits as in a
    small cache."""
    import torch

    from langtrain_studio_amd import KvCache

    heads, kvh, hd = shape
    kvd = heads * hd
    if kvd % 32 and dtype in ("q8_0", "q4_0"):
        kvd, kvh = 1280, 64  # (whole groups)
        heads = kvh
    blocks = int((1 << 32) / (kvd * size * BLOCK)) + 40
    rng = np.random.default_rng(6)
    ctx, new = 53, 13
    parents = random_tree(rng, new, 0.4)
    n = ctx + new
    x = [up(rng.standard_normal((n, kvd)), np.float32).to(torch.bfloat16) for _ in range(3)]
    tokens, targets = (up(rng.integers(0, 2, new), np.int32) for _ in range(2))
    results = []
    for total in (40, blocks):
        kv = KvCache(1, kvd, total * BLOCK, dtype=dtype)
        order = np.arange(total)[::-1].copy()
        kv.init_free_order(order)
        cells = kv.append_batch(np.zeros(n, np.uint32), np.arange(n, dtype=np.uint64))
        if min(kv.block_table(0)) < total - 40:  # (the other end is handed out first)
            kv = KvCache(1, kvd, total * BLOCK, dtype=dtype)
            kv.init_free_order(order[::-1].copy())
            cells = kv.append_batch(np.zeros(n, np.uint32), np.arange(n, dtype=np.uint64))
        assert min(kv.block_table(0)) >= total - 40
        if hd % 8 == 0:
            kv.rope_init_scaled(10000.0, hd, hd, True, 128)
            kv.write_rope_rows(0, up(cells, np.int32), up(np.arange(n), np.int32), x[1], x[2])
        else:
            kv.write_batch(0, up(cells, np.int32), x[1].float(), x[2].float())
        at = kv.step_layout(up(kv.seq_rows(np.arange(1)), np.int32), up([ctx], np.int32), up([new], np.int32), new, 6,
                            parents=up(parents, np.int32), mask_words=1)
        out = kv.tree_attention(0, x[0][:new], at.tables, at.lens, heads, hd, at.row_starts, masks=at.masks)
        done = kv.accept_tree(at.tables, at.lens, at.row_starts, up(parents, np.int32), tokens, targets)
        got = [torch.zeros((n, kvd), device="cuda") for _ in range(2)]
        kv.gather_values(0, at.tables, at.lens, torch.zeros(1, dtype=torch.int64, device="cuda"), *got)
        kv.synchronize()
        results.append([out, *done, *got])
        del kv
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert bool(results[0][0].float().isfinite().all()) and bool((results[0][0] != 0).any())


def test_captured_before_its_partials_exist(gpu):
    """A capture that would have to grow the partials is refused, and works after
    one eager call."""
    import torch

    from langtrain_studio_amd import KvError

    side = torch.cuda.Stream()
    t = Trees((32, 8, 128), "f16", [200], [60], 3, stream=side, rows="bf16")
    args, masks = t.args(), up(t.masks, np.int32)
    out = torch.zeros_like(t.q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        torch.zeros(1, device="cuda")
        with pytest.raises(KvError, match="before capturing"):
            t.kv.tree_attention(0, *args, masks=masks, max_rows=60, out=out)
    with torch.cuda.stream(side):
        want = t.kv.tree_attention(0, *args, masks=masks, max_rows=60)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        t.kv.tree_attention(0, *args, masks=masks, max_rows=60, out=out)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_two_caches_on_two_streams(gpu):
    """Calls of two caches that run at once, each on its own stream."""
    import torch

    streams = [torch.cuda.Stream() for _ in range(2)]
    trees = [Trees((8, 2, 128), "f16", [3000, 50, 700], [9, 30, 1], 20 + i, stream=s) for i, s in enumerate(streams)]
    torch.cuda.synchronize()
    outs = [torch.zeros_like(t.q) for t in trees]
    args = [(t.args(), up(t.masks, np.int32)) for t in trees]
    torch.cuda.synchronize()
    for _ in range(5):
        for t, o, (a, m) in zip(trees, outs, args):
            t.kv.tree_attention(0, *a, masks=m, out=o)
    for t in trees:
        t.kv.synchronize()
    for t, o in zip(trees, outs):
        compare(o.cpu().numpy(), t.want())


def test_the_same_inputs_give_the_same_bits(gpu):
    import torch

    t = Trees((32, 8, 128), "q8_0", [4000, 100, 2500], [33, 64, 2], 30)
    a, m = t.args(), up(t.masks, np.int32)
    first = t.kv.tree_attention(0, *a, masks=m)
    for _ in range(3):
        assert torch.equal(t.kv.tree_attention(0, *a, masks=m), first)


@pytest.mark.parametrize("hint", [1, 3, 17, 200])
def test_rows_beyond_the_hint(gpu, hint):
    """max_rows sizes the tiles; any value gives the definition."""
    t = Trees((8, 2, 128), "f16", [100, 7, 40], [17, 3, 1], 31)
    t.check(max_rows=hint)


def test_wide_tables_and_a_cache_without_blocks(gpu):
    """Tables far wider than the contexts, and a cache that holds no block: zeros."""
    import torch

    from langtrain_studio_amd import KvCache

    t = Trees((8, 2, 128), "f16", [100, 7], [5, 3], 32)
    t.tables = np.pad(t.tables, ((0, 0), (0, 8000)), constant_values=-1)
    t.check()
    kv = KvCache(1, 128, 0)
    q = torch.randn((2, 256), device="cuda")
    got = kv.tree_attention(0, q, torch.full((1, 1), -1, dtype=torch.int32, device="cuda"), up([2], np.int32), 4, 64,
                            up([0, 2], np.int32))
    kv.synchronize()
    assert (got == 0).all()


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30, 30.0])
@pytest.mark.parametrize("dtype", ["f16", "q8_0"])
def test_scales(gpu, dtype, scale):
    t = Trees((8, 2, 64), dtype, [200, 3], [9, 4], 33)
    got = t.run(scale=scale)
    compare(got, t.want(scale=scale))


@pytest.mark.parametrize("cap", [1e-3, 300.0, 1e30])
@pytest.mark.parametrize("rows", ["f32", "f16"])
def test_caps(gpu, rows, cap):
    t = Trees((8, 2, 64), "f16", [200, 3], [9, 4], 34, rows=rows, gain=3.0)
    t.check(softcap=cap)
