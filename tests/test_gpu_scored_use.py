"""Scored attention and the 4-bit cache as they are used together: captured and
replayed steps, other streams, batches larger than the chip's waves, padded
batches, extreme scales, and a sequence's life from prompt to forked decodes.
Numbers against the definition in 64 bits (test_gpu_scored's tolerances);
captured against eager calls bit by bit."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_scored import BLOCK, build, check, expect, held_rows, run, slopes_of

pytestmark = pytest.mark.gpu


def up(a, dtype):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


# (dtype, heads, kv heads, head_dim, lens, new rows): single tokens in parts, a
# chunk split over positions beside single tokens, packs of rows, the generic kernel
CAPTURES = {
    "rows": ("q4_0", 8, 2, 128, [3000, 40, 700], [1, 1, 1]),
    "chunks": ("f16", 8, 2, 64, [1500, 9, 600], [200, 1, 1]),
    "packs": ("f32", 10, 2, 80, [900, 20, 300], [30, 1, 4]),
    "any": ("f16", 3, 1, 20, [90, 20, 33], [10, 1, 4]),
}


@pytest.mark.parametrize("name", CAPTURES)
def test_captured_and_replayed(gpu, name):
    """Each replay, with eager calls and other sizes between, gives the eager
    result for the inputs of that moment."""
    import torch

    dtype, heads, kvh, hd, lens, new = CAPTURES[name]
    starts = np.concatenate([[0], np.cumsum(new)])
    side = torch.cuda.Stream()
    kv, tables = build(kvh * hd, lens, dtype, 31, stream=side)
    kv.synchronize()
    gen = torch.Generator(device="cuda").manual_seed(5)
    with torch.cuda.stream(side):
        q = torch.randn((starts[-1], heads * hd), generator=gen, device="cuda")
        out = torch.zeros_like(q)
        t, ld, sd = up(tables, np.int32), up(lens, np.int32), up(starts, np.int32)
        slopes = up(slopes_of(heads), np.float32)
    side.synchronize()

    def call(out=None):
        return kv.scored_attention(0, q, t, ld, heads, hd, row_starts=sd, max_rows=max(new), softcap=9.0,
                                   slopes=slopes, out=out)

    with torch.cuda.stream(side):
        call()  # (sizes what is sized on demand)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(out)
    for i in range(4):
        with torch.cuda.stream(side):
            q.normal_(generator=gen)
            ld.copy_(up([max(n - 17 * i, 0) for n in lens], np.int32))
            graph.replay()
            got = out.clone()
            want = call()
            # partials of another size, in memory of their own once they outgrow the captured call's
            big = kv.scored_attention(0, q[:3].repeat(30 * (i + 1), 1), t.repeat(30 * (i + 1), 1),
                                      ld.repeat(30 * (i + 1)), heads, hd)
        side.synchronize()
        assert torch.equal(got, want), i
        assert torch.isfinite(big).all()
        lens_now = ld.cpu().tolist()
        check(got.cpu().numpy(), expect(q.cpu().numpy(), held_rows(kv), tables, lens_now, starts, heads, hd,
                                        softcap=9.0, slopes=slopes_of(heads)), "f32")


def test_captured_decode_of_the_4bit_cache(gpu):
    import torch

    heads, kvh, hd, lens = 8, 2, 128, [2500, 77, 1, 600]
    side = torch.cuda.Stream()
    kv, tables = build(kvh * hd, lens, "q4_0", 32, slack=8, stream=side)
    kv.synchronize()
    gen = torch.Generator(device="cuda").manual_seed(6)
    n = len(lens)
    sm = up(kv.append_batch(np.arange(n, dtype=np.uint32), np.array(lens, np.uint64)), np.int32)
    t, ld = up(kv.block_tables(np.arange(n, dtype=np.uint32)), np.int32), up(np.array(lens) + 1, np.int32)
    q, k, v = (torch.randn((n, w), generator=gen, device="cuda") for w in (heads * hd, kvh * hd, kvh * hd))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        kv.append_decode_attention(0, sm, k, v, q, t, ld, heads, hd)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kv.append_decode_attention(0, sm, k, v, q, t, ld, heads, hd, out=out)
    for _ in range(3):
        with torch.cuda.stream(side):
            for x in (q, k, v):
                x.normal_(generator=gen)
            graph.replay()
            got = out.clone()
            want = kv.decode_attention(0, q, t, ld, heads, hd)
        side.synchronize()
        assert torch.equal(got, want)
        check(got.cpu().numpy(), expect(q.cpu().numpy(), held_rows(kv), t.cpu().numpy(), [x + 1 for x in lens],
                                        list(range(n + 1)), heads, hd), "f32")


def test_a_capture_without_partials_is_refused(gpu):
    """Nothing is allocated in a capture: the call is refused there, the capture
    goes on, and the call is captured once it ran eagerly."""
    import torch

    from langtrain_studio_amd import KvError

    heads, kvh, hd, lens = 32, 8, 128, [6000] * 12
    side = torch.cuda.Stream()
    kv, tables = build(kvh * hd, lens, "q4_0", 33, stream=side)
    kv.synchronize()
    # 94 parts x 12 x 32 rows of 130 floats: 18.8 MB, more than the at most 16 MiB that a cache holds
    # from its creation (at the default partition it would be 4.8 MB)
    kv.set_attention_partition(64)
    q = torch.randn((12, heads * hd), device="cuda")
    t, ld = up(tables, np.int32), up(lens, np.int32)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out.fill_(3.0)
        with pytest.raises(KvError, match="before capturing"):
            kv.decode_attention(0, q, t, ld, heads, hd, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 3.0).all()
    with torch.cuda.stream(side):
        want = kv.decode_attention(0, q, t, ld, heads, hd)
    side.synchronize()
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again, stream=side):
        kv.decode_attention(0, q, t, ld, heads, hd, out=out)
    again.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["q4_0", "q8_0", "f16"])
@pytest.mark.parametrize("how", ["plain", "all"])
def test_batches_beyond_the_resident_waves(gpu, dtype, how):
    """200 single rows, some of the same sequence, some of no context: parts of
    many sequences share a wave, and a row's bits are those of its own call."""
    heads, kvh, hd = 16, 8, 64
    some = [1, 0, 33, 700, 2100, 64, 129, 1025]
    kv, tables = build(kvh * hd, some, dtype, 34)
    rng = np.random.default_rng(35)
    pick = rng.integers(0, len(some), 200)
    lens = [some[i] for i in pick]
    q = rng.standard_normal((200, heads * hd)).astype(np.float32) * 2
    mods = {} if how == "plain" else {"softcap": 8.0, "slopes": slopes_of(heads), "window": 300, "sinks": 5}
    got, qr = run(kv, q, tables[pick], lens, heads, hd, **mods)
    check(got, expect(qr, held_rows(kv), tables[pick], lens, list(range(201)), heads, hd,
                      **({} if how == "plain" else {"softcap": 8.0, "slopes": slopes_of(heads), "window": 300,
                                                    "sinks": 5})), "f32")
    for i in (0, 3, 77, 199):
        mods = {} if how == "plain" else {"softcap": 8.0, "slopes": slopes_of(heads), "window": 300, "sinks": 5}
        one, _ = run(kv, q[i:i + 1], tables[pick[i]:pick[i] + 1], lens[i:i + 1], heads, hd, **mods)
        np.testing.assert_array_equal(one[0], got[i])


@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("new", [[1, 1], [40, 33]])
def test_scales_of_any_sign(gpu, dtype, new):
    heads, kvh, hd, lens = 8, 2, 64, [300, 50]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kvh * hd, lens, dtype, 36)
    q = np.random.default_rng(37).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    for scale in (-0.3, 0.0, 1.5):
        for softcap in (0.0, 2.0):
            got, qr = run(kv, q, tables, lens, heads, hd, starts=starts, max_rows=max(new), scale=scale,
                          softcap=softcap)
            check(got, expect(qr, held_rows(kv), tables, lens, starts, heads, hd, scale=scale, softcap=softcap), "f32")


@pytest.mark.parametrize("dtype,sizes", [("q8_0", (1e-7, 1e6)), ("f32", (1e-30, 1e-6, 1e6, 1e30)), ("f16", (1e-4, 1e4)),
                                         ("q4_0", (1e-4, 1e4))])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [[1, 1], [37, 20]])
def test_rows_of_any_magnitude(gpu, dtype, sizes, hd, new):
    """K and V of one magnitude, from the smallest the type holds well to near
    its largest, with scores of ordinary size."""
    heads, kvh, lens = 4, 2, [200, 70]
    starts = np.concatenate([[0], np.cumsum(new)])
    q = np.random.default_rng(38).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    for size in sizes:
        def times(i, k, v):
            k *= np.float32(size)
            v *= np.float32(size)

        kv, tables = build(kvh * hd, lens, dtype, 39, edit=times)
        scale = float(np.float32(0.1 / size))
        got, qr = run(kv, q, tables, lens, heads, hd, starts=starts, max_rows=max(new), scale=scale)
        check(got, expect(qr, held_rows(kv), tables, lens, starts, heads, hd, scale=scale), "f32")


@pytest.mark.parametrize("part", [64, 192])
@pytest.mark.parametrize("dtype", ["q4_0", "f32"])
def test_fixed_partitions(gpu, part, dtype):
    heads, kvh, hd, lens, new = 8, 2, 96, [700, 30, 400], [1, 20, 1]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kvh * hd, lens, dtype, 40)
    q = np.random.default_rng(41).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    kv.set_attention_partition(part)
    got, qr = run(kv, q, tables, lens, heads, hd, starts=starts, max_rows=20)
    check(got, expect(qr, held_rows(kv), tables, lens, starts, heads, hd), "f32")


@pytest.mark.parametrize("rows", ["f32", "bf16"])
def test_splits_of_several_sequences(gpu, rows):
    """Few tiles of long contexts: every tile's positions are split, tiles of
    several sequences with odd numbers of rows and empty sequences between."""
    heads, kvh, hd = 8, 2, 128
    lens, new = [2000, 0, 1300, 900, 40], [70, 0, 33, 3, 40]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kvh * hd, lens, "f16", 42)
    q = np.random.default_rng(43).standard_normal((starts[-1], heads * hd)).astype(np.float32) * 2
    for how in ({}, {"window": 700, "sinks": 3}):
        got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=70, **how)
        check(got, expect(qr, held_rows(kv), tables, lens, starts, heads, hd, **how), rows)


def test_padded_batches_and_empty_calls(gpu):
    """Padding rows (length 0, any table) give zeros; no rows and no sequences
    are no work."""
    import torch

    heads, kvh, hd = 8, 2, 64
    kv, tables = build(kvh * hd, [100, 40], "q4_0", 44)
    t = np.full((6, tables.shape[1]), -1, np.int32)
    t[:2] = tables
    lens = [100, 40, 0, 0, 0, 0]
    q = np.random.default_rng(45).standard_normal((6, heads * hd)).astype(np.float32)
    got, qr = run(kv, q, t, lens, heads, hd)
    assert (got[2:] == 0).all()
    check(got[:2], expect(qr[:2], held_rows(kv), tables, lens[:2], [0, 1, 2], heads, hd), "f32")
    td, ld = up(t, np.int32), up(lens, np.int32)
    dec = kv.decode_attention(0, up(q, np.float32), td, ld, heads, hd)
    kv.synchronize()
    np.testing.assert_array_equal(dec.cpu().numpy(), got)
    none = kv.scored_attention(0, torch.zeros((0, heads * hd), device="cuda"), td, ld, heads, hd,
                               row_starts=torch.zeros(7, dtype=torch.int32, device="cuda"), max_rows=9)
    kv.synchronize()
    assert none.shape == (0, heads * hd)


@pytest.mark.parametrize("dtype", ["q4_0", "q8_0", "f16"])
def test_a_sequences_life(gpu, dtype):
    """A prompt in two chunks, its rows read back, a fork, and decodes of both
    sequences through the append and the scored entry points."""
    import torch

    from langtrain_studio_amd import KvCache

    heads, kvh, hd = 8, 2, 64
    rng = np.random.default_rng(46)
    kv = KvCache(1, kvh * hd, 40 * BLOCK, dtype=dtype)

    def rows(n):
        return (up(rng.standard_normal((n, kvh * hd)), np.float32) for _ in range(2))

    done = 0
    for m in (75, 130):
        sm = up(kv.append_batch(np.zeros(m, np.uint32), np.arange(done, done + m, dtype=np.uint64)), np.int32)
        kv.write_batch(0, sm, *rows(m))
        done += m
        q = rng.standard_normal((m, heads * hd)).astype(np.float32)
        tables = kv.block_tables([0])
        for how in ({}, {"softcap": 6.0, "window": 64, "sinks": 2}):
            got, qr = run(kv, q, tables, [done], heads, hd, starts=[0, m], max_rows=m, **how)
            check(got, expect(qr, held_rows(kv), tables, [done], [0, m], heads, hd, **how), "f32")
    k_out, v_out = (torch.full((done + 1, kvh * hd), 9.0, device="cuda") for _ in range(2))
    kv.gather_values(0, up(tables, np.int32), up([done], np.int32), up([0], np.int64), k_out, v_out)
    kv.synchronize()
    cells = np.concatenate([b * BLOCK + np.arange(BLOCK) for b in tables[0]])[:done]
    for got, held in zip((k_out, v_out), held_rows(kv)):
        np.testing.assert_array_equal(got[:done].cpu().numpy(), held[cells].astype(np.float32))
        assert (got[done] == 9.0).all()
    kv.share(0, 1, done)
    for step in range(3):
        sm = up(kv.append_batch([0, 1], np.full(2, done + step, np.uint64)), np.int32)
        k, v = rows(2)
        q = rng.standard_normal((2, heads * hd)).astype(np.float32)
        tables, lens = kv.block_tables([0, 1]), [done + step + 1] * 2
        dec = kv.append_decode_attention(0, sm, k, v, up(q, np.float32), up(tables, np.int32), up(lens, np.int32),
                                         heads, hd)
        kv.synchronize()
        got, qr = run(kv, q, tables, lens, heads, hd, slopes=slopes_of(heads))
        held = held_rows(kv)
        check(got, expect(qr, held, tables, lens, [0, 1, 2], heads, hd, slopes=slopes_of(heads)), "f32")
        if dtype == "q4_0":
            check(dec.cpu().numpy(), expect(q, held, tables, lens, [0, 1, 2], heads, hd), "f32")
            plain, _ = run(kv, q, tables, lens, heads, hd)
            np.testing.assert_array_equal(plain, dec.cpu().numpy())
    assert kv.cow_copies() > 0


@pytest.mark.parametrize("dtype", ["f16", "f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("rows", ["f32", "f16"])
@pytest.mark.parametrize("new", [[1, 1], [40, 33]])
def test_the_smallest_caps(gpu, dtype, rows, new):
    """Caps so small that a score over the cap is no number: the weights are
    equal, also where q.k is exactly zero."""
    heads, kvh, hd, lens = 8, 2, 64, [300, 50]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kvh * hd, lens, dtype, 47)
    q = np.random.default_rng(48).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    q[0] = 0
    for softcap in (1e-45, 1e-38, 1e-20):
        got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=max(new), softcap=softcap)
        check(got, expect(np.zeros_like(qr), held_rows(kv), tables, lens, starts, heads, hd), rows)


def test_q_and_out_lie_apart(gpu):
    import torch

    from langtrain_studio_amd import KvError

    heads, kvh, hd = 4, 2, 64
    kv, tables = build(kvh * hd, [20, 20], "f16", 49)
    both = torch.zeros((3, heads * hd), device="cuda")
    t, ld = up(tables, np.int32), up([20, 20], np.int32)
    for out in (both[:2], both[1:]):
        with pytest.raises(KvError, match="overlap"):
            kv.scored_attention(0, both[:2], t, ld, heads, hd, out=out)
    kv.synchronize()
