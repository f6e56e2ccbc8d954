"""Positions that a row does not see: huge, infinite or stale cells there change
nothing for it."""

from __future__ import annotations

import numpy as np
import pytest

from scored_definition import compare, definition
from test_gpu_scored import build, held_rows, run

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
