"""begin_drafts claims everything or nothing: blocks shared by sequences, caches
that are full, and failures behind the claim, on metadata-only caches."""

from __future__ import annotations

import numpy as np
import pytest


@pytest.fixture
def on_host(monkeypatch):
    """(no GPU: nothing is captured, and no layout is made)"""
    import torch

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def backend(blocks):
    from langtrain_studio_amd import PagedKvBackend

    return PagedKvBackend(1, 4, 2, 64, blocks * 16, n_seq_max=8, n_batch=256, device=None)


def fill(b, seq, n):
    b.kv.append_batch(np.full(n, seq, np.uint32), np.arange(n, dtype=np.uint64))


def state(b, seqs):
    return (b.kv.free_blocks(), b.kv.cow_copies(), [b.kv.len(s) for s in seqs],
            [b.kv.block_table(s).tolist() for s in seqs])


def chain(m):
    return [-1] + list(range(m - 1))


def test_a_refused_claim_copies_nothing(on_host):
    """Two sequences share a partial block; the first one's claim would copy it, the
    second one's does not fit."""
    from langtrain_studio_amd import Drafts, KvCacheFull

    b = backend(3)
    fill(b, 0, 20)
    b.kv_copy(0, 1, 20)
    before = state(b, (0, 1))
    with pytest.raises(KvCacheFull):
        b.begin_drafts([Drafts(0, chain(1)), Drafts(1, chain(30))])
    assert state(b, (0, 1)) == before


class Laid(Exception):
    pass


def claims(b, drafts):
    """Whether begin_drafts claims the drafts (its layout is refused, without a GPU)."""
    from langtrain_studio_amd import KvCacheFull

    def upload(arrays):
        raise Laid

    b._upload = upload
    try:
        b.begin_drafts(drafts)
    except KvCacheFull:
        return False
    except Laid:
        return True
    raise AssertionError("neither")


@pytest.mark.parametrize("free", range(0, 7))
def test_the_room_is_what_the_claims_need(on_host, free):
    """Three owners of a partial block, of whom two or all draft, beside whole blocks
    and a sequence of its own: refused exactly where the cache itself would run full."""
    from langtrain_studio_amd import Drafts, KvCacheFull

    for counts in ([1, 1, 0, 0], [1, 1, 1, 0], [13, 1, 12, 3], [12, 12, 12, 17], [1, 0, 0, 16], [30, 2, 1, 1]):
        made = []
        for _ in range(2):
            b = backend(3 + 5 + free)
            fill(b, 0, 20)  # two blocks, the second in part
            b.kv_copy(0, 1, 20)
            b.kv_copy(0, 2, 20)
            fill(b, 3, 16)  # a whole block
            fill(b, 9, 80)  # the others
            assert b.kv.free_blocks() == free
            made.append(b)
        seqs = [s for s in range(4) if counts[s]]
        got = claims(made[0], [Drafts(s, chain(counts[s])) for s in seqs])
        try:
            for s in seqs:
                c = made[1].kv.len(s)
                made[1].kv.append_batch(np.full(counts[s], s, np.uint32), np.arange(c, c + counts[s], dtype=np.uint64))
            fits = True
        except KvCacheFull:
            fits = False
        assert got == fits, counts


@pytest.mark.parametrize("where", ["seq_rows", "_upload", "step_layout"])
def test_failures_behind_the_claim(on_host, monkeypatch, where):
    """Whatever fails behind the claim, the sequences have their lengths back, and
    the next step claims what this one did."""
    from langtrain_studio_amd import Drafts

    b = backend(8)
    fill(b, 0, 20)
    fill(b, 1, 3)
    if where != "_upload":
        b._upload = lambda arrays: (arrays, None)

    def refuse(*args, **how):
        raise MemoryError(where)

    monkeypatch.setattr(b if where == "_upload" else b.kv, where, refuse, raising=True)
    before = state(b, (0, 1, 2))
    with pytest.raises(MemoryError, match=where):
        b.begin_drafts([Drafts(0, chain(9)), Drafts(2, chain(40)), Drafts(1, chain(2))])
    assert state(b, (0, 1, 2)) == before
