"""Positions that a row does not see: huge, infinite or stale cells there change
nothing for it, and table entries that no row needs are not reported."""

from __future__ import annotations

import numpy as np
import pytest

from scored_definition import compare, definition
from test_gpu_scored import BLOCK, build, held_rows, run

pytestmark = pytest.mark.gpu


KERNELS = [(dtype, hd) for dtype in ("f16", "f32", "q8_0", "q4_0") for hd in (64, 128, 96, 256)]


# lengths as built, lengths of the call, rows, positions with a huge cell, masks
def scenario(name):
    if name == "window":
        return [100, 300, 64], [100, 300, 64], [100, 1, 3], {0: [40], 1: [5, 130], 2: [20]}, {"window": 25}
    if name == "sinks":
        return [200, 150], [200, 150], [120, 40], {0: [60, 130], 1: [70]}, {"window": 20, "sinks": 3}
    if name == "documents":
        first = np.concatenate([np.arange(150) // 37 * 37, np.arange(30, 90) // 37 * 37]).astype(np.int32)
        return [150, 90], [150, 90], [150, 60], {0: [10, 80], 1: [50]}, {"first": first}
    if name == "behind":
        return [100, 80, 90], [70, 33, 81], [70, 20, 2], {0: [75, 99], 1: [33, 40], 2: [82]}, {}
    return [200], [200], [200], {0: [130]}, {}  # causal: behind most rows


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["window", "sinks", "documents", "behind", "causal"])
@pytest.mark.parametrize("dtype,hd", KERNELS)
def test_huge_cells(gpu, dtype, hd, name, rows):
    """V of ordinary and of small size beside cells of 1e3, of the largest that a
    quantised type holds, and of what becomes an infinity there."""
    heads, kv_heads = 8, 2
    built, lens, new, where, how = scenario(name)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = np.random.default_rng(62).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    for size in (1.0, 1e-3):
        for huge in (1e3, 8e6, 1e12, 1e30):
            def edit(i, k, v):
                v *= np.float32(size)
                for n, p in enumerate(where[i]):
                    k[p] *= np.float32(huge)
                    v[p] = np.float32(huge if n % 2 else -huge)

            kv, tables = build(kv_heads * hd, built, dtype, 61, edit=edit)
            got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=max(new), **dict(how))
            compare(got, definition(qr, held_rows(kv), tables, lens, starts, heads, hd, rows=rows,
                                    eight=dtype == "q8_0", **how))


@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("hd", [64, 96, 20])
def test_entries_that_no_row_needs(gpu, dtype, hd):
    """Two documents, a window and sinks in one tile of rows: blocks between a
    document's sinks and its window may have been given back."""
    heads, kv_heads = 32, 8
    lens, new = [160, 40], [70, 3]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 63)
    first = np.where(np.arange(90, 160) < 100, 0, 100)
    first = np.concatenate([first, [0, 0, 0]]).astype(np.int32)
    q = np.random.default_rng(64).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    how = {"window": 16, "sinks": 4, "first": first}
    given = tables.copy()
    given[0, 1:4] = [-1, 1 << 20, -1]  # rows 90 .. 99 see 0 .. 3 and from 75 on
    got, qr = run(kv, q, given, lens, heads, hd, starts=starts, max_rows=70, **dict(how))
    compare(got, definition(qr, held_rows(kv), tables, lens, starts, heads, hd, **how))
    # one that a single row needs is reported
    from langtrain_studio_amd import KvError

    given[0, 4] = -1
    assert 75 // BLOCK == 4
    with pytest.raises(KvError, match="outside the pool"):
        run(kv, q, given, lens, heads, hd, starts=starts, max_rows=70, **dict(how))


@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("hd", [64, 96, 20])
@pytest.mark.parametrize("new", [[1, 1], [3, 1], [30, 1]])
def test_entries_before_a_window_and_of_rows_that_see_nothing(gpu, dtype, hd, new):
    """A document that began before the window, without sinks, and one that
    begins behind its row: the blocks of their first positions are not needed."""
    heads, kv_heads = 32, 8
    lens = [160, 40]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 65)
    first = np.array([37] * new[0] + [45], np.int32)
    q = np.random.default_rng(66).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    how = {"window": 16, "first": first}
    given = tables.copy()
    given[0, :7] = -1  # the first row stands at 130 or later and sees from 115 on
    given[1, :] = -1
    got, qr = run(kv, q, given, lens, heads, hd, starts=starts, max_rows=max(new), **dict(how))
    assert (got[-1] == 0).all()
    compare(got, definition(qr, held_rows(kv), tables, lens, starts, heads, hd, **how))
