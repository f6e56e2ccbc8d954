"""Forms of a drafted step's layer: rows of every type, turned by the cache or by the
caller, with caps and windows, into given outputs, captured on another stream than
the step's; and acceptance where lengths end in front of the rows."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_drafts import HD, HEADS, backend, rows_of
from test_gpu_scored import held_rows
from test_gpu_steps import cache, down, raw_rows, up
from test_gpu_tree import types
from tree_definition import ancestors, compare, definition, depths, random_tree, visible

pytestmark = pytest.mark.gpu


def begun(b, rng, ctx, trees):
    """A step behind random contexts (layer 0 is written)."""
    import torch

    from langtrain_studio_amd import Drafts

    for s, c in enumerate(ctx):
        cells = b.kv.append_batch(np.full(c, s, np.uint32), np.arange(c, dtype=np.uint64))
        if c:
            _, k, v = rows_of(rng.integers(0, 50, c), 0, torch.float32)
            b.kv.write_rope_rows(0, up(cells, np.int32), up(np.arange(c), np.int32), k, v)
    return b.begin_drafts([Drafts(s, p) for s, p in enumerate(trees)])


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("how", [{}, {"softcap": 5.0}, {"window": 30}, {"softcap": 8.0, "window": 21}])
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
def test_layers(gpu, dtype, rows, rotate, how, given):
    import torch

    b = backend(dtype)
    rng = np.random.default_rng(8)
    ctx, trees = [37, 0, 100], [random_tree(rng, 19, 0.3), random_tree(rng, 40, 0.6), random_tree(rng, 3, 0.0)]
    step = begun(b, np.random.default_rng(9), ctx, trees)
    assert step.depth < 21  # (in all windows: every draft sees its ancestors)
    td = types()[rows]
    q, k, v = rows_of(rng.integers(0, 50, step.n), 0, td)
    at = step.layout
    if rotate:
        turned = b.kv.write_rope_rows(0, torch.full_like(at.slot_mapping, -1), at.positions, k, v, q=q, n_heads=HEADS)
    else:
        turned, k, v = q, k.float(), v.float()
    out = torch.full_like(q, float("nan")) if given else None
    got = b.draft_layer(step, 0, q, k, v, out=out, rotate=rotate, **how)
    b.kv.synchronize()
    assert got.dtype is td and (got is out or not given)
    if not rotate:  # (k and v as they were given)
        plain = backend(dtype)
        begun(plain, np.random.default_rng(9), ctx, trees)
        plain.kv.write_batch(0, at.slot_mapping, k, v)
        plain.kv.synchronize()
        for x, y in zip(raw_rows(b.kv, 0), raw_rows(plain.kv, 0)):
            np.testing.assert_array_equal(x, y)
    sees = [visible(c + len(p), ancestors(p), how.get("window", 0), c + depths(p)) for c, p in zip(ctx, trees)]
    compare(got.float().cpu().numpy(),
            definition(turned.float().cpu().numpy(), held_rows(b.kv), down(at.tables),
                       [c + len(p) for c, p in zip(ctx, trees)], down(at.row_starts), HEADS, HD, sees, rows=rows,
                       eight=dtype in ("q8_0", "f32"), softcap=how.get("softcap", 0.0)))


def test_layers_captured_on_another_stream(gpu):
    """A step begun on one stream, its layers recorded on another."""
    import torch

    own, side = torch.cuda.Stream(), torch.cuda.Stream()
    b = backend(stream=own)
    rng = np.random.default_rng(6)
    with torch.cuda.stream(own):
        step = begun(b, rng, [37], [random_tree(rng, 19, 0.3)])
        fixed = rows_of(rng.integers(0, 50, step.n), 0, torch.bfloat16)
        out = torch.zeros_like(fixed[0])
        b.draft_layer(step, 0, *fixed, out=out)  # (sizes what is sized on demand)
    torch.cuda.synchronize()
    for s, c in zip(step.seqs, step.lens):
        b.kv.truncate(s, c)
    from langtrain_studio_amd import Drafts

    with torch.cuda.stream(own):
        step = b.begin_drafts([Drafts(0, random_tree(rng, 19, 0.3))])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.kv.set_stream(side)
        b.draft_layer(step, 0, *fixed, out=out)
    for turn in range(4):
        with torch.cuda.stream(side):
            for x, y in zip(fixed, rows_of(rng.integers(0, 50, step.n), 0, torch.bfloat16)):
                x.copy_(y)
            graph.replay()
            replayed = out.clone()
            b.draft_layer(step, 0, *fixed, out=out)
        torch.cuda.synchronize()
        assert torch.equal(out, replayed), turn


@pytest.mark.parametrize("dtype", ["f16", "q8_0"])
def test_acceptance_in_front_of_the_first_position(gpu, dtype):
    """Lengths below the rows: kept rows whose cell does not exist are not moved, the
    others are, nothing is reported."""
    kv = cache([20, 20], kvd=64, layers=2, dtype=dtype)
    rng = np.random.default_rng(3)
    tables = kv.block_tables([0, 1], 2)
    cells = np.concatenate([t[np.arange(20) // 16] * 16 + np.arange(20) % 16 for t in tables]).astype(np.int32)
    for layer in (0, 1):
        kv.write_batch(layer, up(cells, np.int32), *(up(rng.standard_normal((40, 64)), np.float32) for _ in "kv"))
    kv.synchronize()
    before = [raw_rows(kv, layer) for layer in (0, 1)]
    # four rows over two positions, and two over none
    parents, tokens, targets = [-1, 0, 0, 2, -1, 0], [1, 2, 3, 4, 9, 9], [3, 0, 4, 7, 9, 5]
    got = kv.accept_tree(up(tables, np.int32), up([2, 0], np.int32), up([0, 4, 6], np.int32),
                         *(up(x, np.int32) for x in (parents, tokens, targets)))
    kv.synchronize()
    assert down(got.path).tolist() == [0, 2, 3, -1, 0, 1]
    assert down(got.accepted).tolist() == [3, 2] and down(got.next).tolist() == [7, 5]
    assert down(got.lens).tolist() == [1, 0]
    for layer in (0, 1):
        for a, b in zip(raw_rows(kv, layer), before[layer]):
            b[cells[0]] = b[cells[1]]  # the path's third token: position -2 + 3 to -2 + 2
            np.testing.assert_array_equal(a, b)
