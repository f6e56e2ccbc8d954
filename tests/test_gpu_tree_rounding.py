"""Rows of 16 bits are computed to f32 accuracy and rounded once, whatever the pool
holds: the f32 rows' bound, and the type's half step."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_scored import held_rows
from test_gpu_tree import Trees
from tree_definition import definition, visible

pytestmark = pytest.mark.gpu

# half a step of each type, relative, and of f16's subnormal numbers
HALF = {"f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}


@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("rows", ["f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("shape", [(8, 2, 128), (32, 2, 128), (9, 3, 64), (6, 2, 96), (2, 2, 256), (65, 1, 32)])
def test_16_bit_rows_are_rounded_once(gpu, shape, dtype, rows, window):
    """Few positions a row in most trees, where a weight's own rounding would show."""
    t = Trees(shape, dtype, [0, 2, 60, 300], [40, 20, 9, 3], 21, rows=rows, gain=1.0)
    got = t.run(window=window).astype(np.float64)
    sees, row = [], 0
    for length, d in zip(t.lens, t.drafted):
        sees.append(visible(length, d, window, t.positions[row:row + d.shape[0]]))
        row += d.shape[0]
    want, bound, _ = definition(t.q.float().cpu().numpy(), held_rows(t.kv), t.tables, t.lens, t.starts, t.heads, t.hd,
                                sees)
    half, least = HALF[rows]
    bound = bound + np.maximum(half * (np.abs(want) + bound), least)
    off = np.abs(got - want)
    assert (off <= bound).all(), f"{(off / (bound + 1e-30)).max():.3f} times what one rounding allows"
