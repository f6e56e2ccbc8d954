"""Tree attention with drafts deeper than the window, at every kernel's shapes: the
window bounds the context, masks (or the rows in front) the drafts."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_tree import Trees

pytestmark = pytest.mark.gpu

# head widths and groups of the generic kernel, and two of the tile kernel beside them
SHAPES = [(3, 1, 20), (2, 1, 320), (65, 1, 32), (8, 2, 128), (6, 2, 96)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [1, 5, 23])
@pytest.mark.parametrize("shape", SHAPES)
def test_chains_deeper_than_the_window(gpu, shape, window, causal):
    """Chains over several blocks and more than a generic round of 256 positions,
    behind contexts of none to a few blocks."""
    Trees(shape, "f16", [40, 0, 3, 300], [40, 70, 1, 290], 1, branch=0.0, roots=0.0, causal=causal).check(window=window)


@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("shape", [(65, 1, 32), (2, 1, 320)])
def test_far_positions(gpu, shape, dtype):
    """Rows whose positions lie far behind the context's end, or wrap the window's
    start: they see no context, and their drafts all the same; rows that see
    nothing give zeros."""
    t = Trees(shape, dtype, [0, 20, 0], [3, 4, 1], 9)
    t.masks[:] = 0
    t.masks[1] = 1  # the second row of the first tree sees its first one
    for d in t.drafted:
        d[:] = False
    t.drafted[0][1, 0] = True
    t.masks[4] = 1  # a far row that sees the first draft of its tree
    t.drafted[1][1, 0] = True
    t.positions[3:7] = [20, 10 ** 6, 2 ** 31 - 1, 0]
    t.check(window=7)
    got = t.run(window=7)
    assert (got[[0, 2, 5, 7]] == 0).all() and (got[[1, 3, 4, 6]] != 0).any(axis=1).all()


@pytest.mark.parametrize("value", [np.inf, np.nan, 3e38])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_what_a_generic_row_does_not_see(gpu, dtype, value):
    """Infinities and NaN in siblings, behind windows and in front of them stay out
    of the rows that do not see them, in the generic kernel too."""
    from tree_definition import words_of

    ctx, new = [70, 5], [30, 4]

    def edit(i, k, v):
        if i == 0:
            for x in (k, v):
                x[[3, 40, ctx[0] + 2], ::3] = value  # (3 and 40: outside the windows)
        else:
            v[ctx[1] + 1, 1::2] = value

    with np.errstate(over="ignore", invalid="ignore"):
        t = Trees((3, 1, 20), dtype, ctx, new, 10, edit=edit)
        for d, bad in zip(t.drafted, (2, 1)):
            d[:, bad] = False
        t.masks = np.concatenate([words_of(d, t.words) for d in t.drafted])
        t.check(window=20)
