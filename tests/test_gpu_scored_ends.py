"""Scored attention and 4-bit decodes at the ends of their ranges: shapes of the
generic kernel on quantised pools, single tokens of 16-bit rows, values near the
largest f32."""

from __future__ import annotations

import numpy as np
import pytest

from scored_definition import compare, definition
from test_gpu_scored import build, held_rows, run, slopes_of

pytestmark = pytest.mark.gpu

# (heads, kv heads, head_dim) that no matrix-core kernel takes on these pools
GENERIC = [("q4_0", (16, 8, 20)), ("q4_0", (4, 4, 264)), ("q8_0", (16, 8, 20)), ("q8_0", (6, 2, 80)),
           ("q8_0", (4, 4, 264)), ("f32", (4, 2, 160)), ("f16", (2, 1, 1024)), ("q4_0", (2, 1, 1024))]


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype,shape", GENERIC)
def test_generic_shapes(gpu, dtype, shape, rows):
    heads, kv_heads, hd = shape
    lens, new = [70, 1, 0, 300, 33], [40, 1, 0, 5, 2]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 81)
    q = np.random.default_rng(82).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    first = np.concatenate([np.arange(n - m, n) // 37 * 37 for n, m in zip(lens, new)]).astype(np.int32)
    for how in ({}, {"softcap": 3.0, "slopes": slopes_of(heads)}, {"window": 20, "sinks": 3, "first": first},
                {"prefix": [50, 1, 9, 299, 40]}):
        got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=40, **dict(how))
        compare(got, definition(qr, held_rows(kv), tables, lens, starts, heads, hd, rows=rows, **how))


@pytest.mark.parametrize("shape", [(16, 8, 20), (4, 4, 264), (2, 1, 1024)])
def test_generic_decodes_of_the_4bit_cache(gpu, shape):
    """Tables and the fused append of shapes that only the generic kernel takes."""
    import torch

    heads, kv_heads, hd = shape
    lens = [40, 1, 300]
    kv, tables = build(kv_heads * hd, lens, "q4_0", 83, slack=4)
    n = len(lens)
    rng = np.random.default_rng(84)

    def up(a, dtype):
        return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()

    q = rng.standard_normal((n, heads * hd)).astype(np.float32)
    out = kv.decode_attention(0, up(q, np.float32), up(tables, np.int32), up(lens, np.int32), heads, hd)
    kv.synchronize()
    starts = list(range(n + 1))
    compare(out.cpu().numpy(), definition(q, held_rows(kv), tables, lens, starts, heads, hd))
    sm = kv.append_batch(np.arange(n, dtype=np.uint32), np.array(lens, np.uint64))
    tables = kv.block_tables(np.arange(n, dtype=np.uint32))
    k, v = (rng.standard_normal((n, kv_heads * hd)).astype(np.float32) for _ in range(2))
    lens = [x + 1 for x in lens]
    out = kv.append_decode_attention(0, up(sm, np.int32), up(k, np.float32), up(v, np.float32), up(q, np.float32),
                                     up(tables, np.int32), up(lens, np.int32), heads, hd)
    kv.synchronize()
    compare(out.cpu().numpy(), definition(q, held_rows(kv), tables, lens, starts, heads, hd))


@pytest.mark.parametrize("rows", ["f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("shape", [(8, 2, 128), (9, 3, 64), (6, 2, 96)])
def test_single_tokens_of_16_bit_rows(gpu, shape, dtype, rows):
    heads, kv_heads, hd = shape
    lens = [1, 0, 15, 16, 17, 33, 64, 65, 200, 517, 1500]
    kv, tables = build(kv_heads * hd, lens, dtype, 85)
    q = np.random.default_rng(86).standard_normal((len(lens), heads * hd)).astype(np.float32) * 2
    for how in ({}, {"softcap": 5.0}, {"softcap": 8.0, "slopes": slopes_of(heads), "window": 40, "sinks": 1}):
        got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, **dict(how))
        compare(got, definition(qr, held_rows(kv), tables, lens, list(range(len(lens) + 1)), heads, hd, rows=rows, **how))


@pytest.mark.parametrize("shape", [(8, 2, 128), (6, 2, 96), (4, 2, 160)])
@pytest.mark.parametrize("lens,new", [([300, 50], [1, 1]), ([3000, 40], [1, 1]), ([300, 50], [40, 33]),
                                      ([3000, 700], [5, 20])])
def test_values_near_the_largest_f32(gpu, shape, lens, new):
    """An average of values is no larger than the largest: sums that pass f32's
    range on the way are not formed."""
    heads, kv_heads, hd = shape
    starts = np.concatenate([[0], np.cumsum(new)])
    q = np.random.default_rng(88).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    for size in (1e30, 1e35, 3e37):
        def large(i, k, v):
            np.clip(v, -4, 4, out=v)
            v *= np.float32(size)

        kv, tables = build(kv_heads * hd, lens, "f32", 87, edit=large)
        got, qr = run(kv, q, tables, lens, heads, hd, starts=starts, max_rows=max(new))
        compare(got, definition(qr, held_rows(kv), tables, lens, starts, heads, hd))
