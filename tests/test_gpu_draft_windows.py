"""Layers with a window over drafted steps: a draft sees what the same token decoded
alone sees, however deep its tree is; and the masks that make it so."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_drafts import HD, HEADS, KVH, backend, rows_of
from test_gpu_scored import held_rows
from test_gpu_steps import cache, down
from test_gpu_tree import up
from tree_definition import ancestors, compare, definition, depths, random_tree, words_of

pytestmark = pytest.mark.gpu


def inside(see, positions, window):
    """[m][m] visibility without the rows that the window hides."""
    p = np.asarray(positions, np.int64)
    return see & (p[None, :] > p[:, None] - window)


@pytest.mark.parametrize("window", [1, 3, 8, 40])
@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
def test_drafts_deeper_than_the_window(gpu, dtype, window):
    """Every row by the definition, the window bounding ancestors as it bounds the
    context."""
    import torch

    from langtrain_studio_amd import Drafts

    b = backend(dtype)
    rng = np.random.default_rng(window)
    ctx = [37, 0, 5]
    for s, c in enumerate(ctx):
        cells = b.kv.append_batch(np.full(c, s, np.uint32), np.arange(c, dtype=np.uint64))
        if c:
            _, k, v = rows_of(rng.integers(0, 50, c), 0, torch.float32)
            b.kv.write_rope_rows(0, up(cells, np.int32), up(np.arange(c), np.int32), k, v)
    trees = [random_tree(rng, 45, 0.05), [-1] + list(range(59)), random_tree(rng, 9, 0.5)]
    step = b.begin_drafts([Drafts(s, p) for s, p in enumerate(trees)])
    q, k, v = rows_of(rng.integers(0, 50, step.n), 0, torch.float32)
    out = b.draft_layer(step, 0, q, k, v, window=window)
    b.kv.synchronize()
    at = step.layout
    turned = b.kv.write_rope_rows(0, torch.full_like(at.slot_mapping, -1), at.positions, k, v, q=q, n_heads=HEADS)
    b.kv.synchronize()
    sees = []
    for c, p in zip(ctx, trees):
        pos = c + depths(p)
        see = np.zeros((len(p), c + len(p)), bool)
        see[:, :c] = np.arange(c)[None, :] > pos[:, None] - window
        see[:, c:] = inside(ancestors(p), pos, window)
        sees.append(see)
    want = definition(down(turned), held_rows(b.kv), down(at.tables), [c + len(p) for c, p in zip(ctx, trees)],
                      down(at.row_starts), HEADS, HD, sees, eight=dtype in ("q8_0", "f32"))
    compare(down(out), want)
    if window < 40:  # (the test would see drafts that the window does not bound)
        free = b.kv.tree_attention(0, turned, at.tables, at.lens, HEADS, HD, at.row_starts, positions=at.positions,
                                   masks=at.masks, window=window)
        with pytest.raises(AssertionError):
            compare(down(free), want)


def test_a_chain_is_its_tokens_decoded_alone(gpu):
    """Row by row: scored attention of a single token with the same window."""
    import torch

    from langtrain_studio_amd import Drafts

    b = backend()
    m, window = 50, 7
    step = b.begin_drafts([Drafts(0, [-1] + list(range(m - 1)))])
    q, k, v = rows_of(range(m), 0, torch.float32)
    out = b.draft_layer(step, 0, q, k, v, window=window)
    at = step.layout
    turned = b.kv.write_rope_rows(0, torch.full_like(at.slot_mapping, -1), at.positions, k, v, q=q, n_heads=HEADS)
    sees = [np.tril(np.ones((m, m), bool)) & ~np.tril(np.ones((m, m), bool), -window)]
    want = definition(down(turned), held_rows(b.kv), down(at.tables), [m], [0, m], HEADS, HD, sees)
    compare(down(out), want)
    alone = torch.cat([b.kv.scored_attention(0, turned[j:j + 1], at.tables, up([j + 1], np.int32), HEADS, HD,
                                             window=window) for j in range(m)])
    b.kv.synchronize()
    compare(down(alone), want)


def test_captured_with_a_window(gpu):
    """A captured layer bounds its masks in each replay."""
    import torch

    from langtrain_studio_amd import Drafts

    side = torch.cuda.Stream()
    b = backend(stream=side)
    with torch.cuda.stream(side):
        step = b.begin_drafts([Drafts(0, [-1] + list(range(29)))])
        fixed = rows_of(range(30), 0, torch.bfloat16)
        out = torch.zeros_like(fixed[0])
        b.draft_layer(step, 0, *fixed, window=4, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.draft_layer(step, 0, *fixed, window=4, out=out)
    for turn in range(4):
        with torch.cuda.stream(side):
            for x, y in zip(fixed, rows_of(np.arange(30) + 7 * turn, 0, torch.bfloat16)):
                x.copy_(y)
        side.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        with torch.cuda.stream(side):
            b.draft_layer(step, 0, *fixed, window=4, out=out)
        b.kv.synchronize()
        assert torch.equal(out, replayed), turn


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("window", [1, 2, 30, 10 ** 9])
def test_window_masks(gpu, window, in_place):
    """Masks of several words, rows of no sequence, sequences without rows and bits
    of rows that a sequence does not have; positions of any size."""
    kv = cache([1])
    rng = np.random.default_rng(window)
    news = [1, 0, 70, 33, 5]
    starts = 3 + np.concatenate([[0], np.cumsum(news)])
    rows, words = int(starts[-1]) + 4, 3
    masks = rng.integers(-2 ** 31, 2 ** 31, (rows, words)).astype(np.int32)
    positions = rng.integers(0, 60, rows).astype(np.int32)
    positions[starts[3]:starts[4]] += 2 ** 31 - 100
    positions[starts[2]] = -1
    want = np.zeros_like(masks)
    for a, m in zip(starts, news):
        bits = np.unpackbits(masks[a:a + m].view(np.uint8), axis=1, bitorder="little").astype(bool)[:, :m]
        want[a:a + m] = words_of(inside(bits, positions[a:a + m], window), words)
    given = up(masks, np.int32)
    got = kv.window_masks(up(starts, np.int32), up(positions, np.int32), given, window, out=given if in_place else None)
    kv.synchronize()
    np.testing.assert_array_equal(down(got), want)
    assert (got is given) == in_place and (in_place or (down(given) == masks).all())


def test_window_masks_refusals(gpu):
    from langtrain_studio_amd import KvError

    kv = cache([1])
    starts, positions, masks = up([0, 4], np.int32), up(np.arange(4), np.int32), up(np.ones((4, 1)), np.int32)
    call = kv.window_masks
    with pytest.raises(ValueError, match="one word"):
        call(starts, positions, masks[:, :0], 2)
    with pytest.raises(ValueError, match="positions"):
        call(starts, positions[:3], masks, 2)
    with pytest.raises(ValueError, match="window"):
        call(starts, positions, masks, 0)
    with pytest.raises(ValueError, match="out must match"):
        call(starts, positions, masks, 2, out=masks[:3])
    with pytest.raises(TypeError, match="masks must be"):
        call(starts, positions, masks.long(), 2)
    with pytest.raises(KvError, match="overlap"):
        call(starts, positions, masks, 2, out=positions.view(4, 1))
    falling = call(up([9, -3], np.int32), positions, masks, 2)  # no row of any sequence
    none = call(starts[:1], positions, masks, 2)
    kv.synchronize()
    assert (down(falling) == 0).all() and (down(none) == 0).all()
