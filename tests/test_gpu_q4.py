"""The 4-bit cache: append bit-exact against the format's definition, block
copies, read-back as values, and every decode attention entry point against the
definition in 64 bits over the held values (tolerances as test_gpu_scored)."""

from __future__ import annotations

import numpy as np
import pytest

from helpers import special_f32
from test_gpu_scored import BLOCK, build, check, expect, held_rows

pytestmark = pytest.mark.gpu

LIMIT = 65280.0


def f16_of_bf16(x):
    """f32 -> bf16 -> f16, nearest even both times (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    u = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
    return u.view(np.float32).astype(np.float16)


def quantise(x):
    """(q int8, d f16) of f32 rows [n][kv_dim], by the format's definition."""
    g = np.where(np.isnan(x), np.float32(0), np.clip(x, -LIMIT, LIMIT)).astype(np.float64)
    g = g.reshape(x.shape[0], -1, 32)
    top, low = g.max(axis=2), g.min(axis=2)
    d = f16_of_bf16((np.where(top >= -low, top, low) * -0.125).astype(np.float32))
    w = d.astype(np.float64)[:, :, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(w == 0, 0, np.clip(np.rint(g / w), -8, 7))
    return q.astype(np.int8).reshape(x.shape), np.where(d == 0, np.float16(0), d)


def pool_rows(kv, sm, layer=0):
    """(q [n][kv_dim], d [n][groups]) of the cells sm, for K and V."""
    out = []
    for q, s in zip(kv.read_pool(layer), kv.read_scales(layer)):
        d = s.view(np.float16).transpose(0, 2, 1).reshape(-1, kv.kv_dim // 32)
        out.append((q.reshape(-1, kv.kv_dim)[sm], d[sm]))
    return out


def up(a, dev):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def rows_of(rng, n, kvd, kind):
    if kind == "special":
        x = special_f32(rng, max(n * kvd, 256))[:n * kvd].reshape(n, kvd)
    elif kind == "ties":
        # the extreme is 8 (d = -1), the rest halves: every border of a level
        x = (rng.integers(-16, 17, (n, kvd)) * 0.5).astype(np.float32)
        x[:, ::32] = np.where(rng.random((n, kvd // 32)) < 0.5, 8.0, -8.0)
    elif kind == "tiny":
        x = (rng.standard_normal((n, kvd)) * 10.0 ** rng.integers(-9, -3, (n, 1))).astype(np.float32)
    else:
        x = (rng.standard_normal((n, kvd)) * np.exp(rng.standard_normal(kvd))).astype(np.float32)
    return x


@pytest.mark.parametrize("kind", ["normal", "special", "ties", "tiny"])
@pytest.mark.parametrize("kvd", [32, 96, 320, 1024])
def test_append_is_the_formats(gpu, kvd, kind):
    from langtrain_studio_amd import KvCache

    rng = np.random.default_rng(kvd)
    n = 75
    kv = KvCache(2, kvd, 10 * BLOCK, dtype="q4_0")
    kv.init_free_order(rng.permutation(10))
    assert kv.bytes() == 2 * 2 * 10 * BLOCK * (kvd // 2 + kvd // 32 * 2)
    sm = kv.append_batch(np.repeat([0, 1, 2], 25), np.tile(np.arange(25), 3))
    k, v = rows_of(rng, n, kvd, kind), rows_of(rng, n, kvd, kind)
    skip = sm.copy()
    skip[::9] = -1  # left out: the cells stay zero
    skip[4] = 10 * BLOCK  # outside the pool: skipped
    kv.write_batch(1, up(skip, gpu), up(k, gpu), up(v, gpu))
    kv.synchronize()
    for (q, d), x in zip(pool_rows(kv, sm, 1), (k, v)):
        wq, wd = quantise(x)
        gone = (skip < 0) | (skip >= 10 * BLOCK)
        wq[gone], wd[gone] = 0, 0
        np.testing.assert_array_equal(d.view(np.uint16), wd.view(np.uint16))
        np.testing.assert_array_equal(q, wq)
        # a held value is an f16 number
        val = q.astype(np.float32).reshape(n, -1, 32) * d.astype(np.float32)[:, :, None]
        assert (val.astype(np.float16).astype(np.float32) == val).all() and np.isfinite(val).all()
    for q, d in pool_rows(kv, sm, 0):  # the other layer is untouched
        assert (q == 0).all() and (d == 0).all()


def test_append_orders_and_host_rows(gpu):
    from langtrain_studio_amd import KvCache

    rng = np.random.default_rng(3)
    kvd, n = 64, 40
    k, v = rows_of(rng, n, kvd, "normal"), rows_of(rng, n, kvd, "normal")
    pools = []
    for form in range(3):
        kv = KvCache(1, kvd, 3 * BLOCK, dtype="q4_0")
        sm = kv.append_batch(np.zeros(n, np.uint32), np.arange(n))
        if form == 0:
            kv.write_batch(0, up(sm, gpu), up(k, gpu), up(v, gpu))
        elif form == 1:
            order = kv.cell_order(sm)[::-1].copy()
            kv.write_batch_ordered(0, up(sm, gpu), up(k, gpu), up(v, gpu), up(order, gpu))
        else:
            for i in range(n):
                kv.write(0, int(sm[i]) // BLOCK, int(sm[i]) % BLOCK, k[i], v[i])
        pools.append(kv.read_pool(0) + kv.read_scales(0))
    for p in pools[1:]:
        for a, b in zip(p, pools[0]):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("neox", [False, True])
def test_rope_append_is_rotate_then_append(gpu, neox):
    """The q8_0 append's rotation (bit-exact against the oracle), read from an
    f32 cache, then this format's quants."""
    from langtrain_studio_amd import KvCache

    rng = np.random.default_rng(4)
    hd, kvh, heads, n = 64, 2, 4, 33
    k = rng.standard_normal((n, kvh * hd), dtype=np.float32)
    v = rng.standard_normal((n, kvh * hd), dtype=np.float32)
    q = rng.standard_normal((n, heads * hd), dtype=np.float32)
    res = {}
    for dtype in ("f32", "q4_0"):
        kv = KvCache(1, kvh * hd, 3 * BLOCK, dtype=dtype)
        kv.rope_init(10000.0, hd, hd, neox, 100)
        sm = kv.append_batch(np.zeros(n, np.uint32), np.arange(n))
        qd = up(q, gpu)
        kv.write_rope(0, up(sm, gpu), up(np.arange(n, dtype=np.int32), gpu), up(k, gpu), up(v, gpu), qd, heads)
        kv.synchronize()
        res[dtype] = (kv, sm, qd.cpu().numpy())
    np.testing.assert_array_equal(res["f32"][2], res["q4_0"][2])
    kr, vr = res["f32"][0].rows(0, 0, n)
    for (got_q, got_d), x in zip(pool_rows(res["q4_0"][0], res["q4_0"][1]), (kr, vr)):
        wq, wd = quantise(x)
        np.testing.assert_array_equal(got_q, wq)
        np.testing.assert_array_equal(got_d.view(np.uint16), wd.view(np.uint16))


def test_copy_on_write_and_block_copies(gpu):
    rng = np.random.default_rng(5)
    kvd = 96
    kv, _ = build(kvd, [20], "q4_0", 6, slack=8, layers=2)
    kv.share(0, 1, 20)
    sm = kv.append_batch(np.array([1], np.uint32), np.array([20], np.uint64))  # shared last block: copied
    assert kv.cow_copies() == 1
    k, v = rows_of(rng, 1, kvd, "normal"), rows_of(rng, 1, kvd, "normal")
    kv.write_batch(1, up(sm, gpu), up(k, gpu), up(v, gpu))
    kv.synchronize()
    t0, t1 = kv.block_table(0), kv.block_table(1)
    assert t0[0] == t1[0] and t0[1] != t1[1]
    for layer in range(2):
        for a in kv.read_pool(layer):
            np.testing.assert_array_equal(a[t1[1]][:4], a[t0[1]][:4])
        for a in kv.read_scales(layer):
            np.testing.assert_array_equal(a[t1[1]][:, :4], a[t0[1]][:, :4])
    for (q, d), x in zip(pool_rows(kv, sm, 1), (k, v)):
        wq, wd = quantise(x)
        np.testing.assert_array_equal(q, wq)
    free = [b for b in range(kv.n_blocks) if kv.refcount(b) == 0][0]
    kv.copy_blocks(up(np.array([[t0[0], free]], np.int32), gpu))
    kv.synchronize()
    for layer in range(2):
        for a in kv.read_pool(layer) + kv.read_scales(layer):
            np.testing.assert_array_equal(a[free], a[t0[0]])


@pytest.mark.parametrize("kvd,dtype", [(32, "q4_0"), (320, "q4_0"), (320, "q8_0"), (64, "f16"), (10, "f16"), (7, "f32"),
                                       (1024, "q4_0"), (36, "f32")])
def test_gather_values(gpu, kvd, dtype):
    import torch

    lens = [1, 0, 16, 45]
    kv, tables = build(kvd, lens, dtype, 8)
    offs = np.array([50, 0, 3, 100], np.int64)
    k = torch.full((160, kvd), -3.0, device=gpu)
    v = torch.full((160, kvd), -3.0, device=gpu)
    kv.gather_values(0, up(tables, gpu), up(np.array(lens, np.int32), gpu), up(offs, gpu), k, v)
    kv.synchronize()
    held = held_rows(kv)
    for got, h in zip((k.cpu().numpy(), v.cpu().numpy()), held):
        want = np.full((160, kvd), -3.0)
        for i, n in enumerate(lens):
            t = np.arange(n)
            want[offs[i]:offs[i] + n] = h[tables[i][t // BLOCK] * BLOCK + t % BLOCK]
        np.testing.assert_array_equal(got, want.astype(np.float32))


def test_gather_values_faults_and_refusals(gpu):
    import torch

    from langtrain_studio_amd import KvError

    kv, tables = build(32, [40], "q4_0", 9)
    bad = tables.copy()
    bad[0, 1] = -1
    k, v = torch.zeros((40, 32), device=gpu), torch.zeros((40, 32), device=gpu)
    args = (up(np.array([40], np.int32), gpu), up(np.array([0], np.int64), gpu))
    kv.gather_values(0, up(bad, gpu), *args, k, v)
    with pytest.raises(KvError, match="outside the pool"):
        kv.synchronize()
    kv.gather_values(0, up(tables, gpu), *args, k, v)
    kv.synchronize()
    with pytest.raises(TypeError, match="float32"):
        kv.gather_values(0, up(tables, gpu), *args, k.half(), v.half())
    with pytest.raises(KvError, match="16-byte"):
        flat = torch.zeros(40 * 32 + 1, device=gpu)[1:].view(40, 32)
        kv.gather_values(0, up(tables, gpu), *args, flat, v)
    with pytest.raises(KvError, match="gather_values"):
        kv.gather(0, up(tables, gpu), *args, k.to(torch.int8), v.to(torch.int8))
    with pytest.raises(KvError, match="gather_values"):
        kv.rows(0, 0, 10)
    with pytest.raises(KvError, match="Q4_0"):
        kv.set_attention_engine("valu")


SHAPES = [(8, 2, 128), (32, 8, 64), (7, 1, 128), (9, 3, 64), (16, 1, 128), (6, 2, 96), (20, 4, 80), (8, 1, 256),
          (34, 1, 64), (3, 3, 32)]
LENS = [1, 0, 15, 16, 17, 31, 33, 64, 127, 129, 300, 1025, 1700]


@pytest.mark.parametrize("shape", SHAPES)
def test_decode_attention(gpu, shape):
    heads, kvh, hd = shape
    if kvh * hd % 32:
        pytest.skip("not a q4_0 row")
    kv, tables = build(kvh * hd, LENS, "q4_0", 10)
    q = np.random.default_rng(11).standard_normal((len(LENS), heads * hd)).astype(np.float32) * 2
    qd, td, ld = up(q, gpu), up(tables, gpu), up(np.array(LENS, np.int32), gpu)
    want = expect(q, held_rows(kv), tables, LENS, list(range(len(LENS) + 1)), heads, hd)
    got = kv.decode_attention(0, qd, td, ld, heads, hd)
    kv.synchronize()
    check(got.cpu().numpy(), want, "f32")
    # the other entry points: the same bits
    same = {"noalloc": kv.decode_attention(0, qd, td, ld, heads, hd, noalloc=True)}
    rows = up(kv.seq_rows(np.arange(len(LENS), dtype=np.uint32)), gpu)
    same["rows"] = kv.decode_attention_rows(0, qd, rows, ld, heads, hd)
    for shared in (False, True):
        kv.plan_attention(np.arange(len(LENS)), LENS, heads, hd, shared_prefix=shared)
        same[f"planned {shared}"] = kv.planned_attention(0, qd)
    kv.synchronize()
    for name, x in same.items():
        assert (x == got).all(), name
    # and a query's result does not depend on its batch
    for i in (0, 6, 10, 12):
        one = kv.decode_attention(0, qd[i:i + 1], td[i:i + 1], ld[i:i + 1], heads, hd)
        assert (one[0] == got[i]).all(), i
    big = kv.decode_attention(0, qd.repeat(40, 1), td.repeat(40, 1), ld.repeat(40), heads, hd)
    assert (big.view(40, len(LENS), -1) == got).all()


@pytest.mark.parametrize("part", [64, 192])
def test_fixed_partitions(gpu, part):
    heads, kvh, hd = 8, 2, 128
    kv, tables = build(kvh * hd, LENS, "q4_0", 12)
    q = np.random.default_rng(13).standard_normal((len(LENS), heads * hd)).astype(np.float32)
    kv.set_attention_partition(part)
    got = kv.decode_attention(0, up(q, gpu), up(tables, gpu), up(np.array(LENS, np.int32), gpu), heads, hd)
    kv.synchronize()
    check(got.cpu().numpy(), expect(q, held_rows(kv), tables, LENS, list(range(len(LENS) + 1)), heads, hd), "f32")


@pytest.mark.parametrize("shape", [(8, 2, 128), (9, 3, 64)])
def test_long_contexts(gpu, shape):
    heads, kvh, hd = shape
    lens = [9000, 4097, 20011]
    kv, tables = build(kvh * hd, lens, "q4_0", 14)
    q = np.random.default_rng(15).standard_normal((3, heads * hd)).astype(np.float32) * 2
    qd, td, ld = up(q, gpu), up(tables, gpu), up(np.array(lens, np.int32), gpu)
    got = kv.decode_attention(0, qd, td, ld, heads, hd)
    kv.synchronize()
    check(got.cpu().numpy(), expect(q, held_rows(kv), tables, lens, [0, 1, 2, 3], heads, hd), "f32")
    one = kv.decode_attention(0, qd[2:], td[2:], ld[2:], heads, hd)
    assert (one[0] == got[2]).all()


def test_append_decode_attention(gpu):
    heads, kvh, hd = 8, 2, 64
    rng = np.random.default_rng(16)
    lens = [5, 16, 40, 300]
    kv, _ = build(kvh * hd, lens, "q4_0", 17, slack=6)
    ref, _ = build(kvh * hd, lens, "q4_0", 17, slack=6)
    seqs = np.arange(4, dtype=np.uint32)
    n = 4
    k, v = rows_of(rng, n, kvh * hd, "normal"), rows_of(rng, n, kvh * hd, "normal")
    q = up(rng.standard_normal((n, heads * hd), dtype=np.float32), gpu)
    outs = []
    for c in (kv, ref):
        sm = up(c.append_batch(seqs, np.array(lens, np.uint64)), gpu)
        t, ld = up(c.block_tables(seqs), gpu), up(np.array(lens, np.int32) + 1, gpu)
        if c is kv:
            outs.append(c.append_decode_attention(0, sm, up(k, gpu), up(v, gpu), q, t, ld, heads, hd))
        else:
            c.write_batch(0, sm, up(k, gpu), up(v, gpu))
            outs.append(c.decode_attention(0, q, t, ld, heads, hd))
        c.synchronize()
    assert (outs[0] == outs[1]).all()
    for a, b in zip(kv.read_pool(0) + kv.read_scales(0), ref.read_pool(0) + ref.read_scales(0)):
        np.testing.assert_array_equal(a, b)


def test_large_queries(gpu):
    heads, kvh, hd = 4, 2, 128
    lens = [30, 500]
    kv, tables = build(kvh * hd, lens, "q4_0", 18)
    for f in (1e-30, 1e-3, 1e6, 1e30):
        q = (np.random.default_rng(19).standard_normal((2, heads * hd)) * f).astype(np.float32)
        scale = float(np.float32(0.1 / f))
        got = kv.decode_attention(0, up(q, gpu), up(tables, gpu), up(np.array(lens, np.int32), gpu), heads, hd, scale)
        kv.synchronize()
        check(got.cpu().numpy(), expect(q, held_rows(kv), tables, lens, [0, 1, 2], heads, hd, scale=scale), "f32")


def test_bad_tables_are_reported(gpu):
    from langtrain_studio_amd import KvError

    heads, kvh, hd = 4, 2, 64
    kv, tables = build(kvh * hd, [100, 700], "q4_0", 20)
    bad = tables.copy()
    bad[1, 30] = -7
    q = up(np.zeros((2, heads * hd), np.float32), gpu)
    kv.decode_attention(0, q, up(bad, gpu), up(np.array([100, 700], np.int32), gpu), heads, hd)
    with pytest.raises(KvError, match="outside the pool.*1"):
        kv.synchronize()
    kv.decode_attention(0, q, up(bad, gpu), up(np.array([100, 480], np.int32), gpu), heads, hd)
    kv.synchronize()


@pytest.mark.parametrize("descriptor", ["tables", "resident", "planned"])
def test_backend_steps(gpu, descriptor):
    """Prompt chunk, decodes, a fork and its copy-on-write through the engine's
    backend on a 4-bit cache, against 64 bits over the held rows."""
    from langtrain_studio_amd.backend import BatchToken, PagedKvBackend

    heads, kvh, hd, layers = 8, 2, 64, 2
    rng = np.random.default_rng(21)
    be = PagedKvBackend(layers, heads, kvh, hd, 64 * BLOCK, n_seq_max=4, dtype="q4_0", descriptor=descriptor)
    steps = [[(0, p) for p in range(37)], [(0, 37)], "fork", [(0, 38), (1, 38)], [(1, 39), (0, 39)]]
    for step in steps:
        if step == "fork":
            be.kv_copy(0, 1, 38)
            continue
        plan = be.begin_step([BatchToken(0, p, s) for s, p in step])
        n = len(step)
        for layer in range(layers):
            k, v = rows_of(rng, n, kvh * hd, "normal"), rows_of(rng, n, kvh * hd, "normal")
            q = rng.standard_normal((n, heads * hd), dtype=np.float32)
            got = be.layer(plan, layer, up(q, gpu), up(k, gpu), up(v, gpu))
            be.kv.synchronize()
            tables = be.kv.block_tables([s for s, _ in step])
            lens = [p + 1 for _, p in step]
            want = expect(q, held_rows(be.kv, layer), tables, lens, list(range(n + 1)), heads, hd)
            check(got.cpu().numpy(), want, "f32")
