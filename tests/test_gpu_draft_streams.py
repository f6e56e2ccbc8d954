"""Steps with drafted tokens whose cache changes streams between begin_drafts,
draft_layer and accept, with work in front of the layout on the old stream: every
call reads the arrays that the layout made."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_drafts import HD, HEADS, KVH, LAYERS, backend, rows_of
from test_gpu_scored import BLOCK, held_rows
from test_gpu_tree import up
from tree_definition import random_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("current", ["same", "other"])
@pytest.mark.parametrize("moved", ["never", "layer", "accept"])
def test_steps_on_moved_streams(gpu, moved, current):
    """The step's outputs, the kept path and the pool are those of a step that waits
    for everything. The layout is held back by some milliseconds of work in front
    of it; the arrays that it writes hold what another step left there."""
    import torch

    from langtrain_studio_amd import Drafts

    rng = np.random.default_rng(4)
    prompt = rng.integers(0, 50, 37)
    trees = [random_tree(rng, 24, 0.3), random_tree(rng, 9, 0.2)]
    tokens, targets = rng.integers(0, 3, 33), rng.integers(0, 3, 33)
    rows = [rows_of(tokens, layer, torch.bfloat16) for layer in range(LAYERS)]
    big = torch.ones(1 << 28, device="cuda")
    results = []
    for wait in (True, False):
        own, side = torch.cuda.Stream(), torch.cuda.Stream()
        b = backend(stream=own)
        drafted, wanted = up(tokens, np.int32), up(targets, np.int32)
        torch.cuda.synchronize()
        cells = b.kv.append_batch(np.zeros(37, np.uint32), np.arange(37, dtype=np.uint64))
        for layer in range(LAYERS):
            _, k, v = rows_of(prompt, layer, torch.float32)
            at = up(cells, np.int32), up(np.arange(37), np.int32)
            torch.cuda.synchronize()
            b.kv.write_rope_rows(layer, *at, k, v)
        torch.cuda.synchronize()
        if not wait:
            with torch.cuda.stream(own):
                for _ in range(40):  # some 15 ms of work in front of the layout
                    big.mul_(1.0)
        with torch.cuda.stream(own if current == "same" else side):
            step = b.begin_drafts([Drafts(0, trees[0]), Drafts(1, trees[1])])
        if wait:
            torch.cuda.synchronize()
        elif moved == "layer":
            b.kv.set_stream(side)
        if not wait and moved == "accept":  # no layer in between: the paths alone
            b.kv.set_stream(side)
            outs = []
        else:
            outs = [b.draft_layer(step, layer, *rows[layer]) for layer in range(LAYERS)]
        if wait:
            torch.cuda.synchronize()
        kept, done = b.accept(step, drafted, wanted)
        torch.cuda.synchronize()
        n = [b.kv.len(s) for s in (0, 1)]
        pools = []
        for layer in range(LAYERS):
            k, v = held_rows(b.kv, layer)
            for s in (0, 1):
                p = np.arange(n[s])
                cell = b.kv.block_table(s)[p // BLOCK] * BLOCK + p % BLOCK
                pools += [k[cell], v[cell]]
        results.append((kept, [x.cpu() for x in (*done, *outs)], pools))
    (kept, arrays, pools), (kept2, arrays2, pools2) = results
    assert kept == kept2 and max(kept) > 1
    for a, b in zip(arrays, arrays2):
        assert torch.equal(a, b)
    if moved == "accept":  # (its rows were never written)
        return
    assert len(arrays) == len(arrays2) == 4 + LAYERS
    for a, b in zip(pools, pools2):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("n", [1, 8])
def test_uploads_outlive_their_step(gpu, n):
    """A step begun on another stream than the cache's and dropped at once: its layout,
    held back, still reads what was uploaded, whatever the current stream allocates."""
    import torch

    from langtrain_studio_amd import Drafts

    own, side = torch.cuda.Stream(), torch.cuda.Stream()
    big = torch.ones(1 << 28, device="cuda")
    rng = np.random.default_rng(n)
    trees = [random_tree(rng, 20, 0.3) for _ in range(n)]
    want = None
    for late in (False, True):
        b = backend(stream=own)
        for s in range(n):
            b.kv.append_batch(np.full(s, s, np.uint32), np.arange(s, dtype=np.uint64))
        torch.cuda.synchronize()
        if late:
            with torch.cuda.stream(own):
                for _ in range(40):  # some 15 ms of work in front of the layout
                    big.mul_(1.0)
        with torch.cuda.stream(side):
            step = b.begin_drafts([Drafts(s, p) for s, p in enumerate(trees)])
            layout, size = step.layout, step.parents.untyped_storage().nbytes() // 4
            del step
            filled = [torch.full((size,), 99, dtype=torch.int32, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        b.kv.synchronize()
        got = [x.cpu() for x in layout]
        want = want or got
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        del filled


@pytest.mark.parametrize("descriptor", ["tables", "resident"])
def test_uploads_of_plain_steps_outlive_their_plan(gpu, descriptor):
    import torch

    from langtrain_studio_amd import BatchToken, PagedKvBackend

    own, side = torch.cuda.Stream(), torch.cuda.Stream()
    big = torch.ones(1 << 28, device="cuda")
    n, want = 40, None
    q, k, v = rows_of(range(n), 0, torch.float32)
    for late in (False, True):
        b = PagedKvBackend(LAYERS, HEADS, KVH, HD, 2000, n_seq_max=n, descriptor=descriptor, stream=own)
        with torch.cuda.stream(side):
            plan = b.begin_step([BatchToken(0, 0, s) for s in range(n)])
        b.layer(plan, 0, q, k, v)  # (sizes what is sized on demand)
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        if late:
            with torch.cuda.stream(own):
                for _ in range(40):
                    big.mul_(1.0)
        with torch.cuda.stream(side):
            plan = b.begin_step([BatchToken(0, 1, s) for s in range(n)])
            size = plan.lens.untyped_storage().nbytes() // 4
            b.layer(plan, 0, q, k, v, out=out)
            del plan
            filled = [torch.full((size,), 99, dtype=torch.int32, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        b.kv.synchronize()
        want = out if want is None else want
        assert torch.equal(out, want)
        del filled
