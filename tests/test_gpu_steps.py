"""Steps with drafted tokens around their attention: layouts from lengths, rotary
appends of rows of any type, and acceptance, against plain restatements."""

from __future__ import annotations

import copy
import math

import numpy as np
import pytest

from test_gpu_scored import BLOCK, held_rows
from tree_definition import ancestors, depths, random_tree, words_of

pytestmark = pytest.mark.gpu


def up(a, dtype):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def down(t):
    return t.cpu().numpy()


# ---- layout -------------------------------------------------------------------


def cache(lens, layers=1, kvd=32, dtype="f16", slack=3, seed=0, stream=None):
    from langtrain_studio_amd import KvCache

    blocks = sum(-(-n // BLOCK) for n in lens) + slack
    kv = KvCache(layers, kvd, blocks * BLOCK, dtype=dtype, stream=stream)
    kv.init_free_order(np.random.default_rng(seed).permutation(blocks))
    for i, n in enumerate(lens):
        if n:
            kv.append_batch(np.full(n, i, np.uint32), np.arange(n, dtype=np.uint64))
    return kv


def layout_of(kv, lens, new, n_tokens, stride, parents=None, words=0):
    """The step's arrays, from the host's own tables."""
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tables = np.full((len(lens), stride), -1, np.int32)
    slots, pos = np.full(n_tokens, -1, np.int32), np.full(n_tokens, -1, np.int32)
    masks = np.zeros((n_tokens, words), np.int32)
    for i, (c, m) in enumerate(zip(lens, new)):
        need = -(-(c + m) // BLOCK)
        full = kv.block_table(i) if c + m else np.zeros(0, np.int32)
        tables[i, :need] = full[:need]
        p = c + np.arange(m)
        slots[starts[i]:starts[i + 1]] = full[p // BLOCK] * BLOCK + p % BLOCK
        tree = None if parents is None else parents[i]
        pos[starts[i]:starts[i + 1]] = c + (np.arange(m) if tree is None else depths(tree))
        if tree is not None and m:
            masks[starts[i]:starts[i + 1]] = words_of(ancestors(tree), words)
    return starts, np.add(lens, new).astype(np.int32), tables, slots, pos, masks


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("n,top,new", [(1, 0, 1), (3, 40, 5), (64, 300, 17), (300, 20, 3), (2, 5000, 2000), (5, 100, 130)])
def test_layout(gpu, n, top, new, tree):
    rng = np.random.default_rng(n + new)
    lens, news = rng.integers(0, top + 1, n).tolist(), rng.integers(0, new + 1, n).tolist()
    news[0] = new
    kv = cache([c + m for c, m in zip(lens, news)])
    n_tokens, stride = sum(news) + 7, max(-(-(c + m) // BLOCK) for c, m in zip(lens, news)) + 2
    parents = [random_tree(rng, m, 0.3, 0.1) for m in news] if tree else None
    words = (new + 31) // 32 if tree else 0
    flat = None
    if tree:
        flat = up(np.concatenate([np.array(p, np.int64) for p in parents] + [np.full(7, 3)]), np.int32)
    rows = up(kv.seq_rows(np.arange(n)), np.int32)
    got = kv.step_layout(rows, up(lens, np.int32), up(news, np.int32), n_tokens, stride, parents=flat, mask_words=words)
    kv.synchronize()
    want = layout_of(kv, lens, news, n_tokens, stride, parents, words)
    for name, g, w in zip(got._fields, got, want):
        if g is not None:
            np.testing.assert_array_equal(down(g), w, err_msg=name)


def test_layout_of_single_tokens_and_absent_requests(gpu):
    """No counts: one token each; a row of -1 (or past the tables) is no request;
    negative counts and lengths are none."""
    kv = cache([17, 5, 33])
    rows = kv.seq_rows(np.arange(3))
    r = up([rows[0], -1, rows[2], 10 ** 6, rows[1], rows[1]], np.int32)
    lens = up([16, 9, 32, 4, -3, 2], np.int32)
    got = kv.step_layout(r, lens, None, 6, 3)
    kv.synchronize()
    assert down(got.row_starts).tolist() == [0, 1, 1, 2, 2, 3, 4]
    assert down(got.lens).tolist() == [17, 0, 33, 0, 1, 3]
    t0, t2, t1 = (kv.block_table(i) for i in (0, 2, 1))
    assert down(got.slot_mapping).tolist() == [t0[1] * 16, t2[2] * 16, t1[0] * 16, t1[0] * 16 + 2, -1, -1]
    assert down(got.positions).tolist() == [16, 32, 0, 2, -1, -1]
    assert down(got.tables).tolist() == [[*t0, -1], [-1] * 3, [*t2], [-1] * 3, [t1[0], -1, -1], [t1[0], -1, -1]]
    counts = up([1, 5, -2, 0, 0, 1], np.int32)
    got = kv.step_layout(r, lens, counts, 6, 3)
    kv.synchronize()
    assert down(got.row_starts).tolist() == [0, 1, 1, 1, 1, 1, 2]


def test_layout_faults(gpu):
    """Tokens beyond the arrays, the blocks or the tables' width are reported,
    and what is written stays inside."""
    from langtrain_studio_amd import KvError

    kv = cache([20, 40])
    rows = up(kv.seq_rows(np.arange(2)), np.int32)
    lens = up([10, 30], np.int32)
    got = kv.step_layout(rows, lens, up([4, 4], np.int32), 6, 3)
    with pytest.raises(KvError, match="step layout: request 1"):
        kv.synchronize()
    assert down(got.row_starts).tolist() == [0, 4, 6] and down(got.lens).tolist() == [14, 32]
    got = kv.step_layout(rows, lens, up([30, 4], np.int32), 40, 3)
    with pytest.raises(KvError, match="step layout: request 0"):
        kv.synchronize()
    assert (down(got.slot_mapping)[:22] >= 0).all() and (down(got.slot_mapping)[22:30] == -1).all()
    kv.step_layout(rows, lens, up([1, 1], np.int32), 2, 1)
    with pytest.raises(KvError, match="step layout: request 1"):
        kv.synchronize()
    kv.synchronize()


def test_layout_odd_parents(gpu):
    """A parent that is no earlier token makes a root; tokens past the mask's
    words have no bit, in long chains too."""
    kv = cache([2000])
    rows, lens = up(kv.seq_rows([0]), np.int32), up([3], np.int32)
    got = kv.step_layout(rows, lens, up([6], np.int32), 6, 125, parents=up([5, 0, 2, -7, 3, 10 ** 9], np.int32),
                         mask_words=1)
    assert down(got.positions).tolist() == [3, 4, 3, 3, 4, 3]
    assert down(got.masks)[:, 0].tolist() == [1, 3, 4, 8, 24, 32]
    m = 1500  # more than a work-group holds
    chain = np.arange(-1, m - 1)
    got = kv.step_layout(rows, lens, up([m], np.int32), m, 125, parents=up(chain, np.int32), mask_words=2)
    kv.synchronize()
    assert down(got.positions).tolist() == [3 + j for j in range(m)]
    np.testing.assert_array_equal(down(got.masks), words_of(np.tril(np.ones((m, m), bool)), 2))


def test_layout_follows_the_tables(gpu):
    """Appends, truncations and forks between steps reach the next layout; the
    arrays of an earlier call are filled again; another stream than torch's."""
    import torch

    side = torch.cuda.Stream()
    kv = cache([30, 10], stream=side)
    rows = up(kv.seq_rows(np.arange(2)), np.int32)
    lens, counts = up([20, 9], np.int32), up([2, 1], np.int32)
    torch.cuda.synchronize()
    out = kv.step_layout(rows, lens, counts, 4, 4)
    kv.truncate(0, 17)
    kv.share(0, 2, 17)
    kv.append_batch(np.full(5, 0, np.uint32), np.arange(17, 22, dtype=np.uint64))
    again = kv.step_layout(rows, lens, counts, 4, 4, out=out)
    kv.synchronize()
    assert again is out
    copied = copy.deepcopy(out)  # a copy's arrays are its own
    for t in (out.lens, copied.lens):
        t.zero_()
    torch.cuda.synchronize()
    kv.step_layout(rows, lens, counts, 4, 4, out=copied)
    kv.synchronize()
    assert down(copied.lens).tolist() == [22, 10] and down(out.lens).tolist() == [0, 0]
    out = copied
    for name, g, w in zip(out._fields, out, layout_of(kv, [20, 9], [2, 1], 4, 4)):
        if g is not None:
            np.testing.assert_array_equal(down(g), w, err_msg=name)


def test_layout_without_tokens(gpu):
    """Requests that get no tokens (with and without parents), and no requests."""
    import torch

    kv = cache([17, 5])
    rows = kv.seq_rows(np.arange(2))
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    for parents, words in ((None, 0), (empty, 2)):
        got = kv.step_layout(up(rows, np.int32), up([17, 5], np.int32), up([0, 0], np.int32), 0, 2, parents=parents,
                             mask_words=words)
        kv.synchronize()
        assert down(got.row_starts).tolist() == [0, 0, 0] and down(got.lens).tolist() == [17, 5]
        assert down(got.tables).tolist() == [list(kv.block_table(0)), [kv.block_table(1)[0], -1]]
    got = kv.step_layout(empty, empty, empty, 3, 2, parents=up([-1, 0, 0], np.int32), mask_words=1)
    kv.synchronize()
    assert down(got.row_starts).tolist() == [0] and down(got.slot_mapping).tolist() == [-1] * 3
    assert down(got.masks).tolist() == [[0]] * 3
    done = kv.accept_tree(empty.view(0, 1), empty, up([0], np.int32), *[up([0, 0], np.int32)] * 3)
    kv.synchronize()
    assert down(done.path).tolist() == [-1, -1] and done.accepted.numel() == 0


def test_outputs_do_not_take_memory_in_use_on_the_current_stream(gpu):
    """New outputs of a cache on another stream than the current one lie in none of
    the memory that work of the current stream still reads."""
    import torch

    n = 1 << 16
    kv = cache([n + 64], kvd=32, stream=torch.cuda.Stream())
    rows, lens = up(kv.seq_rows(np.arange(1)), np.int32), up([0], np.int32)
    counts = up([n], np.int32)
    stride = n // BLOCK + 4
    big = torch.ones(1 << 28, device="cuda")
    want = kv.step_layout(rows, lens, counts, n, stride)  # (its kernel and memory are there)
    kv.synchronize()
    size = want.row_starts.untyped_storage().nbytes() // 4
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        held = torch.full((size,), 7, dtype=torch.int32, device="cuda")
        for _ in range(40):  # some 15 ms of work in front of the copy
            big.mul_(1.0)
        copied = held + 0
        del held
        got = kv.step_layout(rows, lens, counts, n, stride)
    torch.cuda.synchronize()
    assert bool((copied == 7).all())
    for a, b in zip(got[:5], want[:5]):
        assert torch.equal(a, b)


def test_layout_refusals(gpu):
    import torch

    from langtrain_studio_amd import KvError

    kv = cache([20])
    rows, lens, counts = up(kv.seq_rows([0]), np.int32), up([10], np.int32), up([2], np.int32)
    with pytest.raises(ValueError, match="equal length"):
        kv.step_layout(rows, up([1, 2], np.int32), counts, 2, 2)
    with pytest.raises(ValueError, match="parents"):
        kv.step_layout(rows, lens, counts, 2, 2, parents=counts, mask_words=1)
    with pytest.raises(KvError, match="one word"):
        kv.step_layout(rows, lens, counts, 2, 2, parents=up([-1, 0], np.int32))
    with pytest.raises(KvError, match="table_stride"):
        kv.step_layout(rows, lens, counts, 2, 0)
    with pytest.raises(TypeError, match="lens must be"):
        kv.step_layout(rows, lens.long(), counts, 2, 2)
    out = kv.step_layout(rows, lens, counts, 2, 2)
    with pytest.raises(ValueError, match="out.tables"):
        kv.step_layout(rows, lens, counts, 2, 3, out=out)
    with pytest.raises(KvError, match="overlap"):
        kv.step_layout(rows, lens, counts, 2, 2, out=out._replace(lens=lens))
    with pytest.raises(KvError, match="overlap"):
        kv.step_layout(rows, lens, counts, 2, 2, out=out._replace(positions=out.slot_mapping))
    side = torch.cuda.Stream()
    kv.synchronize()
    kv.set_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        torch.zeros(1, device="cuda")
        with pytest.raises(KvError, match="capture"):
            kv.step_layout(rows, lens, counts, 2, 2, out=out)
    none = kv.step_layout(rows[:0], lens[:0], None, 3, 2)
    assert down(none.row_starts).tolist() == [0] and down(none.slot_mapping).tolist() == [-1] * 3


# ---- rotary appends -----------------------------------------------------------


def frequencies(base, d, kind, factor=1.0, original=0, low=None, high=None):
    if kind == "ntk":
        base = base * factor ** (d / (d - 2.0))
    f = np.array([base ** (-2.0 * i / d) for i in range(d // 2)])
    if kind == "linear":
        return f / factor, 1.0
    if kind == "llama3":
        low, high = low or 1.0, high or 4.0
        wave = 2 * np.pi / f
        smooth = (original / wave - low) / (high - low)
        mid = (1 - smooth) * f / factor + smooth * f
        return np.where(wave < original / high, f, np.where(wave > original / low, f / factor, mid)), 1.0
    if kind == "yarn":
        low, high = low or 1.0, high or 32.0
        dim = [d * math.log(original / (x * 2 * math.pi)) / (2 * math.log(base)) for x in (high, low)]
        lo, hi = max(math.floor(dim[0]), 0), min(math.ceil(dim[1]), d - 1)
        ramp = np.clip((np.arange(d // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0


def rotate(x, positions, hd, d, half, f, magnitude):
    """f32 rows turned by 64-bit angles: the 64-bit result."""
    x = x.astype(np.float64).reshape(x.shape[0], -1, hd).copy()
    angle = positions[:, None, None].astype(np.float64) * f[None, None, :]
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    i = np.arange(d // 2)
    a, b = (i, i + d // 2) if half else (2 * i, 2 * i + 1)
    u, w = x[:, :, a].copy(), x[:, :, b].copy()
    x[:, :, a], x[:, :, b] = u * c - w * s, u * s + w * c
    size = np.zeros_like(x)
    size[:, :, a] = np.abs(u * c) + np.abs(w * s)
    size[:, :, b] = np.abs(u * s) + np.abs(w * c)
    return x.reshape(x.shape[0], -1), size.reshape(x.shape[0], -1)


KINDS = {"none": {}, "linear": dict(factor=4.0), "ntk": dict(factor=3.0),
         "yarn": dict(factor=4.0, original=4096), "llama3": dict(factor=8.0, original=8192)}
# half steps of a value of each type, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def rope_case(dtype, rows, shape, d, half, kind, n, seed, base=10000.0, top=100001, **extra):
    """A cache with n rows appended; everything the check needs."""
    import torch

    heads, kvh, hd = shape
    kv = cache([n], kvd=kvh * hd, dtype=dtype, seed=seed)
    rng = np.random.default_rng(seed)
    table = kv.block_table(0)
    p = np.arange(n)
    slots = (table[p // BLOCK] * BLOCK + p % BLOCK).astype(np.int32)
    positions = np.sort(rng.integers(0, top, n)).astype(np.int32)
    positions[:1] = 0
    positions[-1:] = top - 1
    kv.rope_init_scaled(base, d, hd, half, top, kind=kind, **KINDS[kind], **extra)
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[rows]
    q, k, v = (up(rng.standard_normal((n, w)) * 2, np.float32).to(t) for w in (heads * hd, kvh * hd, kvh * hd))
    return kv, slots, positions, q, k, v


def check_rotation(got, x, positions, hd, d, half, f, mag, rows):
    """A rotated value has the table's two roundings, two products' and a sum's of
    f32 (each 2^-24 of the products' magnitude), and its own type's."""
    want, size = rotate(x, positions, hd, d, half, f, np.float64(np.float32(mag)))
    turned = np.broadcast_to(np.arange(hd) < d, (x.shape[0], x.shape[1] // hd, hd)).reshape(x.shape)
    bound = np.where(turned, 3 * HALF["f32"] * size, 0)
    if rows != "f32":
        bound = bound + HALF[rows] * (np.abs(want) + bound) + (2.0 ** -25 if rows == "f16" else 0)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= bound).all(), f"{(err / (bound + 1e-30)).max():.2f} times what rounding allows"


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,d", [((8, 2, 128), 128), ((4, 2, 64), 32), ((6, 2, 96), 48), ((5, 1, 80), 40),
                                     ((2, 1, 256), 64), ((3, 1, 512), 512), ((3, 3, 8), 8)])
def test_rotation(gpu, shape, d, half, kind):
    """Every scaling, layout and part of a head, near and far positions: Q, and K
    and V as f32 pools hold them."""
    heads, kvh, hd = shape
    if kind in ("yarn", "ntk") and d == 8:
        pytest.skip("(rope_dim 8 has too few pairs to blend)")
    kv, slots, positions, q, k, v = rope_case("f32", "f32", shape, d, half, kind, 45, 3)
    f, mag = frequencies(10000.0, d, kind, **KINDS[kind])
    out = kv.write_rope_rows(0, up(slots, np.int32), up(positions, np.int32), k, v, q=q, n_heads=heads)
    kv.synchronize()
    check_rotation(down(out), down(q), positions, hd, d, half, f, mag, "f32")
    ks, vs = held_rows(kv)
    check_rotation(ks[slots], down(k), positions, hd, d, half, f, mag, "f32")
    np.testing.assert_array_equal(vs[slots], down(v))


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("shape,d", [((8, 2, 128), 128), ((9, 3, 64), 64), ((4, 2, 96), 48), ((3, 1, 96), 40),
                                     ((2, 2, 256), 256)])
def test_types(gpu, shape, d, half, dtype, rows):
    """Rows and cells of every type: the pool's bits are ltkv_write's of the
    rotated rows that an f32 pool holds, Q's rows their rounding."""
    import torch

    heads, kvh, hd = shape
    n = 37
    kv, slots, positions, q, k, v = rope_case(dtype, rows, shape, d, half, "yarn", n, 4)
    f32 = rope_case("f32", rows, shape, d, half, "yarn", n, 4)[0]
    plain = cache([n], kvd=kvh * hd, dtype=dtype, seed=4)
    sd, pd = up(slots, np.int32), up(positions, np.int32)
    out = kv.write_rope_rows(0, sd, pd, k, v, q=q, n_heads=heads)
    wide = f32.write_rope_rows(0, sd, pd, k.float(), v.float(), q=q.float(), n_heads=heads)
    for c in (kv, f32):
        c.synchronize()
    k32, v32 = (x[slots].astype(np.float32) for x in held_rows(f32))
    plain.write_batch(0, sd, up(k32, np.float32), up(v32, np.float32))
    plain.synchronize()
    for a, b in zip(kv.read_pool(0), plain.read_pool(0)):
        np.testing.assert_array_equal(a, b)
    if dtype in ("q8_0", "q4_0"):
        for a, b in zip(kv.read_scales(0), plain.read_scales(0)):
            np.testing.assert_array_equal(a, b)
    assert torch.equal(out, wide.to(out.dtype))


@pytest.mark.parametrize("dtype", ["f16", "q8_0"])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("shape,d", [((8, 2, 128), 128), ((9, 3, 64), 40), ((1, 1, 32), 32)])
@pytest.mark.parametrize("n", [1025, 2560, 2563])
def test_many_rows(gpu, n, shape, d, half, dtype):
    """A call of many rows gives the bits of calls of a few."""
    import torch

    heads, kvh, hd = shape
    few, slots, positions, q, k, v = rope_case(dtype, "bf16", shape, d, half, "yarn", n, 7)
    many = rope_case(dtype, "bf16", shape, d, half, "yarn", n, 7)[0]
    sd, pd = up(slots, np.int32), up(positions, np.int32)
    out = many.write_rope_rows(0, sd, pd, k, v, q=q, n_heads=heads)
    parts = [few.write_rope_rows(0, sd[i:i + 400], pd[i:i + 400], k[i:i + 400], v[i:i + 400], q=q[i:i + 400],
                                 n_heads=heads) for i in range(0, n, 400)]
    for c in (few, many):
        c.synchronize()
    assert torch.equal(out, torch.cat(parts))
    for a, b in zip(many.read_pool(0), few.read_pool(0)):
        np.testing.assert_array_equal(a, b)
    if dtype == "q8_0":
        for a, b in zip(many.read_scales(0), few.read_scales(0)):
            np.testing.assert_array_equal(a, b)


def test_rope_rows_with_the_plain_table_match_write_rope(gpu):
    """On rope_init's table and f32 rows: write_rope's bits, in place too."""
    shape, n = (8, 2, 128), 20
    for dtype in ("f16", "f32", "q8_0"):
        kv, slots, positions, q, k, v = rope_case(dtype, "f32", shape, 128, True, "none", n, 5, top=500)
        ref = cache([n], kvd=256, dtype=dtype, seed=5)
        for c in (kv, ref):
            c.rope_init(10000.0, 128, 128, True, 500)
        q2 = q.clone()
        sd, pd = up(slots, np.int32), up(positions, np.int32)
        ref.write_rope(0, sd, pd, k, v, q=q2, n_heads=8)
        same = kv.write_rope_rows(0, sd, pd, k, v, q=q, n_heads=8, out=q)
        kv.synchronize(), ref.synchronize()
        assert same is q
        np.testing.assert_array_equal(down(q), down(q2))
        for a, b in zip(kv.read_pool(0), ref.read_pool(0)):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("shape,d,half", [((8, 2, 128), 128, True), ((3, 1, 512), 512, True), ((5, 1, 80), 40, True),
                                          ((6, 2, 96), 96, False)])
def test_columns_of_one_buffer_in_place(gpu, shape, d, half):
    """[q | k | v] rows of a fused projection, Q rotated where it lies; many rows
    (a wave a token) and few."""
    import torch

    heads, kvh, hd = shape
    for n in (3, 2500):
        kv, slots, positions, q, k, v = rope_case("f16", "bf16", shape, d, half, "linear", n, 6, top=4096)
        ref = rope_case("f16", "bf16", shape, d, half, "linear", n, 6, top=4096)[0]
        sd, pd = up(slots, np.int32), up(positions, np.int32)
        want = ref.write_rope_rows(0, sd, pd, k, v, q=q, n_heads=heads)
        buf = torch.cat([q, k, v], dim=1)
        a, b = heads * hd, heads * hd + kvh * hd
        kv.write_rope_rows(0, sd, pd, buf[:, a:b], buf[:, b:], q=buf[:, :a], n_heads=heads, out=buf[:, :a])
        kv.synchronize(), ref.synchronize()
        assert torch.equal(buf[:, :a], want) and torch.equal(buf[:, a:], torch.cat([k, v], dim=1))
        for x, y in zip(kv.read_pool(0), ref.read_pool(0)):
            np.testing.assert_array_equal(x, y)


def test_skipped_tokens(gpu):
    """A position outside the table: nothing written, Q's row too; a cell outside
    the pool: Q alone."""
    kv, slots, positions, q, k, v = rope_case("f16", "f32", (4, 2, 64), 64, True, "none", 6, 7, top=100)
    before = kv.read_pool(0)[1].copy()
    positions[[1, 4]] = [-1, 100]
    slots[[2, 3]] = [-1, 10 ** 8]
    out = q.new_full(q.shape, 5.0)
    kv.write_rope_rows(0, up(slots, np.int32), up(positions, np.int32), k, v, q=q, n_heads=4, out=out)
    kv.synchronize()
    o = down(out)
    assert (o[[1, 4]] == 5).all() and (o[[0, 2, 3, 5]] != 5).any(axis=1).all()
    after = kv.read_pool(0)[1].reshape(-1, 128)
    changed = np.flatnonzero((after != before.reshape(-1, 128)).any(axis=1))
    assert sorted(changed.tolist()) == sorted(slots[[0, 5]].tolist())


def test_scaled_table_serves_write_rope(gpu):
    """rope_init_scaled's table in the f32 append, with divisors and a magnitude."""
    div = np.linspace(1, 3, 32).astype(np.float32)
    kv, slots, positions, q, k, v = rope_case("f32", "f32", (4, 2, 64), 64, False, "none", 9, 8, top=3000)
    kv.rope_init_scaled(500000.0, 64, 64, False, 3000, divisors=div, magnitude=1.25)
    f = frequencies(500000.0, 64, "none")[0] / div.astype(np.float64)
    q2 = q.clone()
    kv.write_rope(0, up(slots, np.int32), up(positions, np.int32), k, v, q=q2, n_heads=4)
    kv.synchronize()
    check_rotation(down(q2), down(q), positions, 64, 64, False, f, 1.25, "f32")


def test_rope_refusals(gpu):
    import torch

    from langtrain_studio_amd import KvCache, KvError

    kv, slots, positions, q, k, v = rope_case("f16", "f32", (4, 2, 64), 64, True, "none", 4, 9, top=100)
    sd, pd = up(slots, np.int32), up(positions, np.int32)
    init = kv.rope_init_scaled
    for match, args, how in [("rope_dim", (1e4, 20, 64, True, 10), {}), ("head_dim", (1e4, 8, 60, True, 10), {}),
                             ("max_positions", (1e4, 64, 64, True, 0), {}), ("base", (0.0, 64, 64, True, 10), {}),
                             ("factor", (1e4, 64, 64, True, 10), dict(kind="linear", factor=0.0)),
                             ("original", (1e4, 64, 64, True, 10), dict(kind="yarn", factor=2.0)),
                             ("low < high", (1e4, 64, 64, True, 10),
                              dict(kind="llama3", factor=2.0, original=64, low=4.0, high=4.0)),
                             ("divisors must be", (1e4, 64, 64, True, 10), dict(divisors=np.zeros(32)))]:
        with pytest.raises(KvError, match=match):
            init(*args, **how)
    for match, how in [("kind", dict(kind="other")), ("rope_dim / 2", dict(divisors=np.ones(3))),
                       ("magnitude", dict(magnitude=-1.0)), ("negative", dict(original=-1))]:
        with pytest.raises(ValueError, match=match):
            init(1e4, 64, 64, True, 10, **how)
    call = kv.write_rope_rows
    with pytest.raises(ValueError, match="match slot_mapping"):
        call(0, sd[:-1], pd, k, v)
    with pytest.raises(TypeError, match="v must be"):
        call(0, sd, pd, k, v.half())
    with pytest.raises(TypeError, match="k must be"):
        call(0, sd, pd, k.double(), v.double())
    with pytest.raises(ValueError, match="n_heads"):
        call(0, sd, pd, k, v, q=q, n_heads=3)
    with pytest.raises(ValueError, match="same row stride"):
        call(0, sd, pd, torch.cat([k, k], dim=1)[:, :128], v)
    with pytest.raises(ValueError, match="unit stride"):
        call(0, sd, pd, k.t().contiguous().t(), v.t().contiguous().t())
    with pytest.raises(KvError, match="16-byte"):
        wide = torch.zeros((4, 136), device="cuda")
        call(0, sd, pd, wide[:, 1:129], wide[:, 1:129])
    with pytest.raises(KvError, match="whole 16-byte"):
        wide = torch.zeros((4, 130), device="cuda")
        call(0, sd, pd, wide[:, :128], wide[:, :128])
    with pytest.raises(KvError, match="overlap"):
        wide = torch.zeros((5, 256), device="cuda")
        call(0, sd, pd, k, v, q=wide[:4], n_heads=4, out=wide[1:])
    with pytest.raises(KvError, match="overlaps the rows"):
        wide = torch.zeros((4, 384), device="cuda")
        call(0, sd, pd, wide[:, 128:256], wide[:, 256:], q=wide[:, :256], n_heads=4, out=wide[:, :256])
    with pytest.raises(KvError, match="no RoPE table"):
        KvCache(1, 128, 64).write_rope_rows(0, sd, pd, k, v)
    with pytest.raises(KvError, match="multiple of 32"):
        c = KvCache(1, 160, 64, dtype="q8_0")
        c.rope_init_scaled(1e4, 40, 80, True, 100)
        c.write_rope_rows(0, sd, pd, torch.zeros((4, 160), device="cuda"), torch.zeros((4, 160), device="cuda"))
    with pytest.raises(KvError, match="at most 512"):
        c = KvCache(1, 1024, 64)
        c.rope_init_scaled(1e4, 1024, 1024, True, 100)
        c.write_rope_rows(0, sd, pd, torch.zeros((4, 1024), device="cuda"), torch.zeros((4, 1024), device="cuda"))


# ---- acceptance ---------------------------------------------------------------


def accepted(parents, tokens, targets):
    path = [0] if len(parents) else []
    while path:
        below = [j for j in range(path[-1] + 1, len(parents)) if parents[j] == path[-1] and tokens[j] == targets[path[-1]]]
        if not below:
            break
        path.append(below[0])
    return path


def raw_rows(kv, layer):
    """The pool's cells, with their scales, as comparable rows."""
    parts = [x.reshape(-1, kv.kv_dim) for x in kv.read_pool(layer)]
    if kv.dtype in ("q8_0", "q4_0"):
        parts += [s.transpose(0, 2, 1).reshape(-1, kv.kv_dim // 32) for s in kv.read_scales(layer)]
    return parts


@pytest.mark.parametrize("dtype,kvd", [("f16", 64), ("f16", 3), ("f32", 64), ("f32", 5), ("q8_0", 96), ("q4_0", 96),
                                       ("f16", 4104)])
@pytest.mark.parametrize("news", [[1, 0, 5, 13], [64, 65, 1], [200, 3]])
def test_acceptance(gpu, dtype, kvd, news):
    """Paths, counts, next tokens and moved rows of every layer, cells behind
    the kept ones as they were; repeated tokens among siblings."""
    rng = np.random.default_rng(sum(news))
    ctx = [0, 5, 30, 16][:len(news)]
    lens = [c + m for c, m in zip(ctx, news)]
    layers = 3
    kv = cache(lens, layers=layers, kvd=kvd, dtype=dtype, seed=2)
    cells = []
    for i, n in enumerate(lens):
        p = np.arange(n)
        t = kv.block_table(i) if n else np.zeros(1, np.int64)
        cells.append(t[p // BLOCK] * BLOCK + p % BLOCK)
    flat = np.concatenate(cells).astype(np.int32)
    for layer in range(layers):
        kv.write_batch(layer, up(flat, np.int32), *(up(rng.standard_normal((flat.size, kvd)), np.float32) for _ in "kv"))
    parents = [random_tree(rng, m, 0.2, 0.02) for m in news]
    tokens = [rng.integers(0, 3, m) for m in news]
    # the model often chooses a child's token
    targets = []
    for p, t in zip(parents, tokens):
        want = rng.integers(0, 3, len(p))
        for j in range(len(p)):
            below = [k for k in range(len(p)) if p[k] == j]
            if below and rng.random() < 0.95:
                want[j] = t[below[-1]]
        targets.append(want)
    starts = np.concatenate([[0], np.cumsum(news)])
    before = [raw_rows(kv, layer) for layer in range(layers)]
    stride = max(1, max(-(-n // BLOCK) for n in lens))
    got = kv.accept_tree(up(kv.block_tables(np.arange(len(lens)), stride), np.int32), up(lens, np.int32),
                         up(starts, np.int32), *(up(np.concatenate(x), np.int32) for x in (parents, tokens, targets)))
    kv.synchronize()
    for i, m in enumerate(news):
        path = accepted(parents[i], tokens[i], targets[i])
        assert down(got.accepted)[i] == len(path) and down(got.lens)[i] == ctx[i] + len(path)
        assert down(got.next)[i] == (targets[i][path[-1]] if path else -1)
        row = np.full(m, -1)
        row[:len(path)] = path
        np.testing.assert_array_equal(down(got.path)[starts[i]:starts[i + 1]], row)
        for parts in before:
            for x in parts:
                x[cells[i][ctx[i]:ctx[i] + len(path)]] = x[cells[i][ctx[i]:][path]]
    for layer in range(layers):
        for a, b in zip(raw_rows(kv, layer), before[layer]):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0"])
def test_acceptance_of_long_paths(gpu, dtype):
    """Paths of many moves, their tokens between decoys, over more drafts than a
    wave has lanes: rows move onto rows that are sources themselves."""
    rng = np.random.default_rng(5)
    ctx, kept = 21, 150
    parents, tokens, targets, path = [-1], [0], [100], [0]
    for k in range(1, kept):
        for _ in range(int(rng.integers(0, 4))):  # children of the path that the model did not choose
            parents.append(path[-1])
            tokens.append(7)
            targets.append(int(rng.integers(100, 110)))
        parents.append(path[-1])
        tokens.append(targets[path[-1]])
        targets.append(100 + k % 10)
        path.append(len(parents) - 1)
    m = len(parents)
    kv = cache([ctx + m], layers=2, kvd=64, dtype=dtype)
    p = np.arange(ctx + m)
    cells = (kv.block_table(0)[p // BLOCK] * BLOCK + p % BLOCK).astype(np.int32)
    for layer in (0, 1):
        kv.write_batch(layer, up(cells, np.int32), *(up(rng.standard_normal((ctx + m, 64)), np.float32) for _ in "kv"))
    before = [raw_rows(kv, layer) for layer in (0, 1)]
    got = kv.accept_tree(up(kv.block_tables([0]), np.int32), up([ctx + m], np.int32), up([0, m], np.int32),
                         *(up(x, np.int32) for x in (parents, tokens, targets)))
    kv.synchronize()
    assert m > 200 and down(got.accepted).tolist() == [kept] and down(got.path)[:kept].tolist() == path
    for layer in (0, 1):
        for a, b in zip(raw_rows(kv, layer), before[layer]):
            b[cells[ctx:ctx + kept]] = b[cells[ctx:][path]]
            np.testing.assert_array_equal(a, b)


def test_acceptance_of_padded_batches_and_bad_entries(gpu):
    """Rows of no request get -1; falling starts, lengths below the rows and
    entries outside the pool move nothing out of place."""
    from langtrain_studio_amd import KvError

    kv = cache([20, 20], kvd=64, layers=2)
    rng = np.random.default_rng(3)
    tables = kv.block_tables([0, 1], 2)
    cells = np.concatenate([t[np.arange(20) // BLOCK] * BLOCK + np.arange(20) % BLOCK for t in tables])
    for layer in (0, 1):
        kv.write_batch(layer, up(cells, np.int32), *(up(rng.standard_normal((40, 64)), np.float32) for _ in "kv"))
    before = [raw_rows(kv, layer) for layer in (0, 1)]
    # [0, 2): no request; 2..6 of the first; none of the second; 6.. none
    parents, tokens = [-1, -1, -1, 0, 0, 2, -1, -1], [9, 9, 1, 2, 3, 4, 9, 9]
    targets = [9, 9, 3, 0, 4, 7, 9, 9]  # 0 -> 2 (token 3) -> none below 2 but 3 (token 4)
    args = [up(x, np.int32) for x in (parents, tokens, targets)]
    got = kv.accept_tree(up(tables, np.int32), up([20, 20], np.int32), up([2, 6, 4], np.int32), *args)
    kv.synchronize()
    assert down(got.path).tolist() == [-1, -1, 0, 2, 3, -1, -1, -1]
    assert down(got.accepted).tolist() == [3, 0] and down(got.next).tolist() == [7, -1]
    assert down(got.lens).tolist() == [19, 20]
    for layer in (0, 1):
        for a, b in zip(raw_rows(kv, layer), before[layer]):
            b[cells[[17, 18]]] = b[cells[[18, 19]]]
            np.testing.assert_array_equal(a, b)
    bad = tables.copy()
    bad[0, 1] = 10 ** 7
    before = [raw_rows(kv, layer) for layer in (0, 1)]
    got = kv.accept_tree(up(bad, np.int32), up([20, 20], np.int32), up([2, 6, 6], np.int32), *args)
    with pytest.raises(KvError, match="block-table entry"):
        kv.synchronize()
    got = kv.accept_tree(up(tables, np.int32), up([2, 0], np.int32), up([2, 6, 8], np.int32), *args)
    try:
        kv.synchronize()
    except KvError:
        pass
    assert down(got.lens)[0] == 1
    for layer in (0, 1):
        for a, b in zip(raw_rows(kv, layer), before[layer]):
            keep = np.ones(a.shape[0], bool)
            keep[cells[0]] = False  # (the last call's kept row may move there)
            np.testing.assert_array_equal(a[keep], b[keep])


def test_acceptance_refusals(gpu):
    from langtrain_studio_amd import KvError

    kv = cache([20], kvd=64)
    tables, lens, starts = up(kv.block_tables([0]), np.int32), up([20], np.int32), up([0, 2], np.int32)
    p = up([-1, 0], np.int32)
    tok, want = up([1, 2], np.int32), up([2, 3], np.int32)
    with pytest.raises(ValueError, match="row_starts"):
        kv.accept_tree(tables, lens, starts[:1], p, tok, want)
    with pytest.raises(ValueError, match="equal length"):
        kv.accept_tree(tables, lens, starts, p, tok, want[:1])
    with pytest.raises(TypeError, match="tokens must be"):
        kv.accept_tree(tables, lens, starts, p, tok.long(), want)
    out = kv.accept_tree(tables, lens, starts, p, tok, want)
    with pytest.raises(KvError, match="overlap"):
        kv.accept_tree(tables, lens, starts, p, tok, want, out=out._replace(lens=lens))
    with pytest.raises(KvError, match="overlap"):
        kv.accept_tree(tables, lens, starts, p, tok, want, out=out._replace(next=out.accepted))
    with pytest.raises(ValueError, match="out.path"):
        kv.accept_tree(tables, lens, starts, p, tok, want, out=out._replace(path=out.next))
    none = kv.accept_tree(tables[:0], lens[:0], starts[:1], p, tok, want)
    assert down(none.path).tolist() == [-1, -1]
