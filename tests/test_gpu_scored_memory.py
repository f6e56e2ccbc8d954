"""Memory and streams of scored attention and 4-bit decodes: partials of wide
tables, growth beside a full device, refused calls, outputs made by the call."""

from __future__ import annotations

import numpy as np
import pytest

from scored_definition import compare, definition
from test_gpu_scored import BLOCK, build, held_rows, run

pytestmark = pytest.mark.gpu

MIB = 1 << 20


def up(a, dtype):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def wide(tables, stride):
    t = np.full((tables.shape[0], stride), -1, np.int32)
    t[:, :tables.shape[1]] = tables
    return t


def free_bytes():
    import torch

    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("own_stream", [True, False])
def test_new_outputs_on_the_caches_stream(gpu, own_stream):
    """The rows of no sequence in a new output are cleared before the call writes
    the others, whatever the current stream is busy with (a cache without a stream
    of its own: on the null stream)."""
    import torch

    heads, kvh, hd, lens, new = 8, 2, 64, [300, 50], [40, 33]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kvh * hd, lens, "f16", 71, stream=torch.cuda.Stream() if own_stream else None)
    kv.synchronize()
    q = torch.randn((80, heads * hd), device="cuda")
    t, ld, sd = up(tables, np.int32), up(lens, np.int32), up(starts, np.int32)
    a = torch.randn((8192, 8192), device="cuda").half()
    torch.cuda.synchronize()
    current = torch.cuda.current_stream() if own_stream else torch.cuda.Stream()
    with torch.cuda.stream(current):
        for _ in range(40):  # some 40 ms before the current stream gets to anything else
            a = a @ a
        got = kv.scored_attention(0, q, t, ld, heads, hd, row_starts=sd, max_rows=40)
    torch.cuda.synchronize()
    got = got.cpu().numpy()
    assert (got[73:] == 0).all()
    compare(got[:73], definition(q[:73].cpu().numpy(), held_rows(kv), tables, lens, starts, heads, hd))


def test_a_refused_append_writes_nothing(gpu):
    """A 4-bit append with attention that a capture cannot hold is refused whole:
    the append is not recorded either."""
    import torch

    from langtrain_studio_amd import KvError

    heads, kvh, hd, lens = 32, 8, 128, [6000] * 12
    side = torch.cuda.Stream()
    kv, tables = build(kvh * hd, lens, "q4_0", 72, slack=16, stream=side)
    kv.synchronize()
    kv.set_attention_partition(64)  # 94 parts x 12 x 32 rows of 130 floats: over the 16 MiB held
    n = len(lens)
    sm = up(kv.append_batch(np.arange(n, dtype=np.uint32), np.array(lens, np.uint64)), np.int32)
    t, ld = up(kv.block_tables(np.arange(n, dtype=np.uint32)), np.int32), up(np.array(lens) + 1, np.int32)
    q, k, v = (torch.randn((n, w), device="cuda") for w in (heads * hd, kvh * hd, kvh * hd))
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    before = kv.read_pool(0) + kv.read_scales(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out.fill_(3.0)
        with pytest.raises(KvError, match="before capturing"):
            kv.append_decode_attention(0, sm, k, v, q, t, ld, heads, hd, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 3.0).all()
    for x, y in zip(before, kv.read_pool(0) + kv.read_scales(0)):
        np.testing.assert_array_equal(x, y)
    with torch.cuda.stream(side):
        kv.append_decode_attention(0, sm, k, v, q, t, ld, heads, hd, out=out)
    kv.synchronize()
    compare(out.cpu().numpy(), definition(q.cpu().numpy(), held_rows(kv), t.cpu().numpy(), [x + 1 for x in lens],
                                          list(range(n + 1)), heads, hd))


def test_partials_grow_beside_a_full_device(gpu):
    """Twice the old size does not fit, what the call needs does; a call whose
    partials do not fit is refused, and the next one runs."""
    import torch

    from langtrain_studio_amd import KvError

    heads, kvh, hd, stride = 32, 8, 128, 8192
    kv, tables = build(kvh * hd, [1], "q4_0", 73)
    # 257 parts of up to 131 072 positions a sequence: 32 x 257 x 130 floats
    need = {n: n * (32 * 257 * 130 * 4 + 4) for n in (192, 256)}
    q = torch.randn((256, heads * hd), device="cuda")
    t = torch.full((256, stride), -1, dtype=torch.int32, device="cuda")
    t[:, 0] = int(tables[0, 0])
    ld = torch.ones(256, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    q2, t2, ld2 = (x.repeat(2, *[1] * (x.dim() - 1)) for x in (q, t, ld))  # twice the sequences: too many
    want = kv.decode_attention(0, q[:1], t[:1, :1].contiguous(), ld[:1], heads, hd)
    # room for the first call's partials, then for the second's and 300 MiB, not for twice the first's
    room = need[192] + need[256] + 300 * MIB
    assert need[256] + 300 * MIB < 2 * need[192]
    ballast = []
    try:
        for size in (free_bytes() // MIB * 3 // 4, 4096, 64):  # MiB a piece, until the device is full
            try:
                while len(ballast) < 256:
                    ballast.append(torch.empty(size * MIB, dtype=torch.uint8, device="cuda"))
            except torch.OutOfMemoryError:
                torch.cuda.empty_cache()
            if size == 4096:
                ballast.pop()  # (in small pieces, some of which are given back)
                torch.cuda.empty_cache()
        pieces = -(-room // (64 * MIB))
        assert len(ballast) < 256 and ballast[-pieces].numel() == 64 * MIB
        del ballast[-pieces:]
        torch.cuda.empty_cache()
        kv.decode_attention(0, q[:192], t[:192], ld[:192], heads, hd, out=out[:192])
        kv.synchronize()
        with pytest.raises(KvError, match="out of memory"):
            kv.decode_attention(0, q2, t2, ld2, heads, hd, out=q2)
        kv.decode_attention(0, q, t, ld, heads, hd, out=out)
        kv.synchronize()
    finally:
        ballast.clear()
        torch.cuda.empty_cache()
    assert torch.equal(out[0], want[0])
    v = held_rows(kv)[1][int(tables[0, 0]) * BLOCK].reshape(kvh, 1, hd).repeat(heads // kvh, axis=1).reshape(-1)
    np.testing.assert_allclose(out.cpu().numpy(), np.tile(v, (256, 1)), rtol=1e-6)
    kv.close()


@pytest.mark.parametrize("dtype", ["f16", "q4_0"])
def test_partials_of_wide_tables_beside_chunks(gpu, dtype):
    """A chunk beside 255 single tokens on tables of 131 072 positions: partials
    follow what the launch can use, not the tables' width."""
    import torch

    heads, kvh, hd = 32, 8, 128
    lens, new = [300] + [1 + i * 7 % 400 for i in range(255)], [64] + [1] * 255
    lens[9], lens[200] = 5000, 2100
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kvh * hd, lens, dtype, 74)
    q = np.random.default_rng(75).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    run(kv, q[:1], tables[:1], [1], heads, hd)
    qd, t, ld, sd = up(q, np.float32), up(wide(tables, 8192), np.int32), up(lens, np.int32), up(starts, np.int32)
    out = torch.empty_like(qd)
    before = free_bytes()
    kv.scored_attention(0, qd, t, ld, heads, hd, row_starts=sd, max_rows=64, out=out)
    kv.synchronize()
    assert before - free_bytes() < 256 * MIB
    compare(out.cpu().numpy(), definition(q, held_rows(kv), tables, lens, starts, heads, hd))
    kv.close()
