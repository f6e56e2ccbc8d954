"""Tokens outside the RoPE table: what rotary appends leave of them, and drafted
steps that would reach past the table."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_drafts import HD, LAYERS, backend, rows_of
from test_gpu_steps import down, rope_case, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
def test_skipped_rows_of_a_new_output_are_zeros(gpu, rows, own):
    """Whatever the memory of the new rows held before, on the cache's stream and
    on another one."""
    import torch

    kv, slots, positions, q, k, v = rope_case("f16", rows, (4, 2, 64), 64, True, "none", 6, 7, top=100)
    if own:
        torch.cuda.synchronize()
        kv.set_stream(torch.cuda.Stream())
    positions[[1, 4]] = [-1, 100]
    sd, pd = up(slots, np.int32), up(positions, np.int32)
    with kv._ordered():
        stale = [torch.full_like(q, float("nan")) for _ in range(64)]
    torch.cuda.synchronize()
    del stale
    out = kv.write_rope_rows(0, sd, pd, k, v, q=q, n_heads=4)
    kv.synchronize()
    o = down(out.float())
    assert (o[[1, 4]] == 0).all() and np.isfinite(o).all() and (o[[0, 2, 3, 5]] != 0).any(axis=1).all()


def test_steps_past_the_table_are_refused(gpu):
    """A step whose deepest token has no row in the table is refused by its layers,
    with nothing written; one that ends with the table, and one whose rows are
    turned already, are not."""
    import torch

    from langtrain_studio_amd import Drafts

    b = backend()
    top = 300
    b.kv.rope_init_scaled(10000.0, HD, HD, True, top)
    n = top - 3
    b.kv.append_batch(np.zeros(n, np.uint32), np.arange(n, dtype=np.uint64))
    long = b.begin_drafts([Drafts(1, [-1, 0]), Drafts(0, [-1, 0, 1, 2, 2])])  # positions 297 ... 300
    before = [b.kv.read_pool(layer) for layer in range(LAYERS)]
    q, k, v = rows_of(range(7), 0, torch.bfloat16)
    with pytest.raises(ValueError, match="reaches position 300"):
        b.draft_layer(long, 0, q, k, v)
    b.kv.synchronize()
    for layer in range(LAYERS):
        for x, y in zip(before[layer], b.kv.read_pool(layer)):
            np.testing.assert_array_equal(x, y)
    assert b.draft_layer(long, 0, q.float(), k.float(), v.float(), rotate=False).isfinite().all()
    for s, c in zip(long.seqs, long.lens):
        b.kv.truncate(s, c)
    short = b.begin_drafts([Drafts(0, [-1, 0, 1, 1, 0, 0])])  # six tokens, positions 297 ... 299
    q, k, v = rows_of(range(6), 0, torch.bfloat16)
    out = b.draft_layer(short, 0, q, k, v)
    b.kv.synchronize()
    assert bool(out.float().isfinite().all()) and bool((out != 0).any(dim=1).all())
    b.kv.rope_init(10000.0, HD, HD, True, top - 1)  # (a shorter table afterwards)
    with pytest.raises(ValueError, match="the RoPE table 299 positions"):
        b.draft_layer(short, 0, q, k, v)
