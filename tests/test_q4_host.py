"""The 4-bit cache's host side, without a GPU: creation, sizes, block
bookkeeping, and that device ops on a metadata-only cache are refused."""

from __future__ import annotations

import numpy as np
import pytest


def test_creation_and_bookkeeping():
    from langtrain_studio_amd import KvCache, KvError

    with pytest.raises(KvError, match="multiple of 32"):
        KvCache(1, 48, 256, dtype="q4_0", device=None)
    with pytest.raises(ValueError, match="q4_0"):
        KvCache(1, 64, 256, dtype="q5_0", device=None)
    kv = KvCache(3, 64, 100, dtype="q4_0", device=None)
    assert kv.capacity() == 112 and kv.kv_dim == 64
    assert kv.bytes() == 2 * 3 * 112 * (32 + 2 * 2)
    f16 = KvCache(3, 64, 100, device=None)
    for c in (kv, f16):
        c.append_batch(np.zeros(40, np.uint32), np.arange(40))
        c.share(0, 1, 20)
        c.append(1, 20)
    assert kv.cow_copies() == f16.cow_copies() == 1
    np.testing.assert_array_equal(kv.block_tables([0, 1]), f16.block_tables([0, 1]))


def test_device_ops_need_a_device():
    from langtrain_studio_amd import KvCache, KvError, _lib

    kv = KvCache(1, 64, 64, dtype="q4_0", device=None)
    for call in (lambda: kv.read_pool(0), lambda: kv.read_scales(0), lambda: kv.set_attention_engine("valu")):
        with pytest.raises(KvError):
            call()
    rc = kv._lib.ltkv_gather_values(kv._h, 0, 1, None, 1, None, None, None, None)
    assert rc == _lib.ERR_ARG and "metadata-only" in _lib.last_error()
    rc = kv._lib.ltkv_scored_attention(kv._h, 0, 1, 1, 1, 2, 32, 1.0, 0.0, None, 0, 0, None, None, 0, None, None, 1,
                                       None, None, None)
    assert rc == _lib.ERR_ARG and "metadata-only" in _lib.last_error()
    assert kv._lib.ltkv_scored_attention(None, 0, 1, 1, 1, 2, 32, 1.0, 0.0, None, 0, 0, None, None, 0, None, None, 1,
                                         None, None, None) == _lib.ERR_ARG


def test_plans_on_the_host():
    """A plan of a 4-bit cache has no groups: every query reads its own context."""
    from langtrain_studio_amd import KvCache

    kv = KvCache(1, 256, 64 * 16, dtype="q4_0", device=None)
    kv.append_batch(np.zeros(200, np.uint32), np.arange(200))
    kv.share(0, 1, 200)
    st = kv.plan_attention([0, 1], [200, 200], 8, 128)
    assert st["queries"] == 2 and st["groups"] == 0
