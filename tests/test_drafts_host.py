"""Refusals of the calls for drafted tokens that need no GPU: a metadata-only cache,
and arguments that the Python face checks by itself."""

from __future__ import annotations

import numpy as np
import pytest

from tree_definition import ancestors, depths, random_tree, words_of


def test_metadata_only_cache():
    import torch

    from langtrain_studio_amd import KvCache, KvError

    kv = KvCache(1, 64, 256, device=None)
    with pytest.raises(KvError, match="metadata-only"):
        kv.rope_init_scaled(10000.0, 64, 64, True, 128)
    x = torch.zeros((2, 64))
    with pytest.raises(TypeError, match="rope_rows|device tensor|device"):
        kv.tree_attention(0, x, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1, 64,
                          torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="device"):
        kv.write_rope_rows(0, torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), x, x)
    with pytest.raises(TypeError, match="device tensor"):
        i = torch.zeros(1, dtype=torch.int32)
        kv.step_layout(i, i, i, 2, 2)
    with pytest.raises(TypeError, match="device tensor"):
        i = torch.zeros(1, dtype=torch.int32)
        kv.accept_tree(i.view(1, 1), i, torch.zeros(2, dtype=torch.int32), i, i, i)


def test_arguments():
    import torch

    from langtrain_studio_amd import KvCache

    kv = KvCache(1, 64, 256, device=None)
    i = torch.zeros(3, dtype=torch.int32)
    for match, call in [
            ("kind", lambda: kv.rope_init_scaled(1e4, 64, 64, True, 128, kind="linear ")),
            ("must not be negative", lambda: kv.rope_init_scaled(1e4, -8, 64, True, 128)),
            ("magnitude", lambda: kv.rope_init_scaled(1e4, 64, 64, True, 128, magnitude=0.0)),
            ("rope_dim / 2", lambda: kv.rope_init_scaled(1e4, 64, 64, True, 128, divisors=[1.0])),
            ("match slot_mapping", lambda: kv.write_rope_rows(0, i, i, torch.zeros((3, 63)), torch.zeros((3, 63)))),
            ("positions", lambda: kv.write_rope_rows(0, i, i[:2], torch.zeros((3, 64)), torch.zeros((3, 64)))),
            ("equal length", lambda: kv.step_layout(i, i[:2], None, 3, 2)),
            ("parents", lambda: kv.step_layout(i, i, None, 4, 2, parents=i, mask_words=1)),
            ("must not be negative", lambda: kv.step_layout(i, i, None, -1, 2)),
            ("row_starts", lambda: kv.accept_tree(i.view(3, 1), i, i, i, i, i)),
            ("equal length", lambda: kv.accept_tree(i.view(3, 1), i, torch.zeros(4), i[:2], i, i)),
            ("n_rows", lambda: kv.tree_attention(0, torch.zeros((3, 63)), i.view(3, 1), i, 1, 64, i)),
            ("row_starts", lambda: kv.tree_attention(0, torch.zeros((3, 64)), i.view(3, 1), i, 1, 64, i)),
            ("one word", lambda: kv.tree_attention(0, torch.zeros((3, 64)), i.view(3, 1), i, 1, 64, torch.zeros(4),
                                                   masks=torch.zeros((3, 0))))]:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(TypeError, match="k must be"):
        kv.write_rope_rows(0, i, i, torch.zeros((3, 64)).double(), torch.zeros((3, 64)).double())


def test_the_oracle_of_trees():
    """The tests' own restatement: ancestors by walking up, bits by definition."""
    rng = np.random.default_rng(1)
    for m in (1, 2, 33, 70):
        parents = random_tree(rng, m, 0.4, 0.1)
        see = ancestors(parents)
        for j in range(m):
            way, node = set(), j
            while node >= 0:
                way.add(node)
                node = parents[node]
            assert set(np.flatnonzero(see[j])) == way and depths(parents)[j] == len(way) - 1
        words = words_of(see, 3).view(np.uint32)
        assert all(bool(words[j, i // 32] >> (i % 32) & 1) == see[j, i] for j in range(m) for i in range(m))
