"""Memory and streams of scored attention and 4-bit decodes: outputs made by the
call, refused calls."""

from __future__ import annotations

import numpy as np
import pytest

from scored_definition import compare, definition
from test_gpu_scored import build, held_rows, run

pytestmark = pytest.mark.gpu


def up(a, dtype):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


def test_new_outputs_on_the_caches_stream(gpu):
    """The rows of no sequence in a new output are cleared before the call writes
    the others, whatever the current stream is busy with."""
    import torch

    heads, kvh, hd, lens, new = 8, 2, 64, [300, 50], [40, 33]
    starts = np.concatenate([[0], np.cumsum(new)])
    side = torch.cuda.Stream()
    kv, tables = build(kvh * hd, lens, "f16", 71, stream=side)
    kv.synchronize()
    q = torch.randn((80, heads * hd), device="cuda")
    t, ld, sd = up(tables, np.int32), up(lens, np.int32), up(starts, np.int32)
    a = torch.randn((8192, 8192), device="cuda").half()
    torch.cuda.synchronize()
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
