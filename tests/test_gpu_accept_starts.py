"""Acceptance with row starts that fall or leave the call's rows: nothing outside
d_path is written, and a request's path stays its own."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_steps import cache, down, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts,paths,counts", [
    # the last request ends in front of its first row: the rows behind that belong to none
    ([0, 6, -5], [0, 1, 2, 3, 4, 5, -1, -1], [6, 0]),
    ([0, 6, 2], [0, 1, 2, 3, 4, 5, -1, -1], [6, 0]),
    ([3, 8, 0], [-1, -1, -1, 0, 1, 2, 3, 4], [5, 0]),
    # every start is negative, or behind the last row
    ([-9, -8, -7], [-1] * 8, [0, 0]),
    ([8, 20, 10 ** 9], [-1] * 8, [0, 0]),
    ([-4, 3, 2 ** 31 - 1], [0, 1, 2, 0, 1, 2, 3, 4], [3, 5]),
])
def test_falling_starts(gpu, starts, paths, counts):
    from langtrain_studio_amd import AcceptedTree

    kv = cache([20, 20], kvd=64)
    tables, lens = up(kv.block_tables([0, 1], 2), np.int32), up([20, 20], np.int32)
    parents = np.full(8, 9)  # (each request's own chain, wherever it begins)
    begins = [min(max(starts[i], 0), 8) for i in range(2)]
    for i, b in enumerate(begins):
        for j in range(counts[i]):
            parents[b + j] = j - 1
    # every child is its parent's target: all rows of a request are kept
    parents, tokens, targets = up(parents, np.int32), up(np.zeros(8), np.int32), up(np.zeros(8), np.int32)
    for _ in range(8):
        guarded = up(np.full(64 + 8 + 64, 77), np.int32)
        out = AcceptedTree(up([7, 7], np.int32), guarded[64:72], up([7, 7], np.int32), up([7, 7], np.int32))
        got = kv.accept_tree(tables, lens, up(starts, np.int32), parents, tokens, targets, out=out)
        kv.synchronize()
        assert (down(guarded)[:64] == 77).all() and (down(guarded)[72:] == 77).all(), "written outside the path"
        assert down(got.path).tolist() == paths
        assert down(got.accepted).tolist() == counts and down(got.lens).tolist() == [20, 20]
        assert down(got.next).tolist() == [0 if c else -1 for c in counts]
