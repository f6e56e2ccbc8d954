"""Memory and streams of scored attention and 4-bit decodes: outputs made by the
call."""

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
