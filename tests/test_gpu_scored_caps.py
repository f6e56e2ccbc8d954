"""Capped scores: 16-bit rows, whose caps the chunk kernel takes in a form of its
own, caps from the smallest to the largest, and scores whose factor is near the
ends of f32."""

from __future__ import annotations

import numpy as np
import pytest

from scored_definition import compare, definition
from test_gpu_scored import build, held_rows, run, slopes_of

pytestmark = pytest.mark.gpu


def both(kv, q, tables, lens, starts, heads, hd, rows, max_rows, **how):
    got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=max_rows, **dict(how))
    compare(got, definition(qr, held_rows(kv), tables, lens, starts, heads, hd, rows=rows, eight=kv.dtype == "q8_0",
                            **how))


@pytest.mark.parametrize("rows", ["f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("shape", [(8, 2, 128), (7, 1, 128), (4, 4, 64), (9, 3, 64), (6, 2, 96)])
def test_chunks_of_16_bit_rows(gpu, shape, dtype, rows):
    """Ragged chunks beside single tokens: caps alone, with windows, prefixes and
    documents, and scales of either sign."""
    heads, kv_heads, hd = shape
    lens, new = [70, 5, 0, 150, 33, 260], [70, 1, 0, 37, 2, 130]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 51)
    q = np.random.default_rng(52).standard_normal((starts[-1], heads * hd)).astype(np.float32) * 3
    first = np.concatenate([np.arange(n - m, n) // 37 * 37 for n, m in zip(lens, new)]).astype(np.int32)
    for how in ({"softcap": 5.0}, {"softcap": 30.0}, {"softcap": 256.0}, {"softcap": 5.0, "window": 23, "sinks": 3},
                {"softcap": 5.0, "prefix": [40, 0, 3, 90, 33, 900]}, {"softcap": 20.0, "first": first},
                {"softcap": 4.0, "scale": -0.2}, {"scale": -0.2}, {"softcap": 4.0, "scale": 0.0},
                {"softcap": 5.0, "slopes": slopes_of(heads)}, {"slopes": slopes_of(heads)}, {}):
        both(kv, q, tables, lens, starts, heads, hd, rows, max(new), **how)


@pytest.mark.parametrize("rows", ["f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0"])
def test_split_chunks_of_16_bit_rows(gpu, dtype, rows):
    """Contexts long enough to be split over their positions."""
    heads, kv_heads, hd = 8, 2, 128
    lens, new = [5000, 2049, 3500], [1, 40, 20]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 53)
    q = np.random.default_rng(54).standard_normal((starts[-1], heads * hd)).astype(np.float32) * 3
    for how in ({"softcap": 8.0}, {"softcap": 30.0, "window": 1500, "sinks": 70}, {"softcap": 8.0, "scale": -0.1}):
        both(kv, q, tables, lens, starts, heads, hd, rows, 40, **how)


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype,shape", [("f16", (8, 2, 128)), ("q8_0", (4, 4, 64)), ("q4_0", (9, 3, 64)),
                                         ("f16", (6, 2, 96)), ("f32", (6, 2, 96)), ("f16", (6, 2, 20))])
@pytest.mark.parametrize("new", [[1, 1], [60, 33]])
def test_large_caps(gpu, dtype, shape, new, rows):
    """A cap far above the scores changes little, and costs no bits."""
    heads, kv_heads, hd = shape
    lens = [300, 50]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 55)
    q = np.random.default_rng(56).standard_normal((starts[-1], heads * hd)).astype(np.float32) * 3
    for softcap in (257.0, 1e3, 1e4, 1e5, 1e6, 1e7, 1e12, 1e25, 3e38):
        for slopes in ({}, {"slopes": slopes_of(heads)}):
            both(kv, q, tables, lens, starts, heads, hd, rows, max(new), softcap=softcap, **slopes)


@pytest.mark.parametrize("rows", ["f32", "f16"])
@pytest.mark.parametrize("dtype,size", [("f32", 1e8), ("q8_0", 1e6), ("f16", 1e4), ("q4_0", 1e4)])
@pytest.mark.parametrize("shape", [(8, 2, 64), (6, 2, 96)])
@pytest.mark.parametrize("new", [[1, 1], [40, 33]])
def test_the_smallest_caps_of_large_rows(gpu, dtype, size, shape, new, rows):
    """Scores over caps so small are no numbers, and some are exactly zero."""
    heads, kv_heads, hd = shape
    lens = [300, 50]
    starts = np.concatenate([[0], np.cumsum(new)])

    def large(i, k, v):
        k *= np.float32(size)
        k[::7] = 0

    kv, tables = build(kv_heads * hd, lens, dtype, 57, edit=large)
    q = np.random.default_rng(58).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    q[0] = 0
    for softcap in (1e-45, 1e-38, 1e-30):
        # (the weights are equal: a capped score is at most the cap)
        got, qr = run(kv, q, tables, lens, heads, hd, rows=rows, starts=starts, max_rows=max(new), softcap=softcap)
        compare(got, definition(np.zeros_like(qr), held_rows(kv), tables, lens, starts, heads, hd, rows=rows,
                                eight=dtype == "q8_0"))


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f16", "q8_0", "q4_0", "f32"])
@pytest.mark.parametrize("shape", [(8, 2, 64), (6, 2, 96)])
@pytest.mark.parametrize("new", [[1, 1], [40, 33]])
def test_factors_near_the_ends_of_f32(gpu, dtype, shape, new, rows):
    """Scales and queries whose product is below or near the top of f32's range."""
    heads, kv_heads, hd = shape
    lens = [300, 50]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, tables = build(kv_heads * hd, lens, dtype, 59)
    q = np.random.default_rng(60).standard_normal((starts[-1], heads * hd)).astype(np.float32)
    for size, scale in ((1e-30, 1e-25), (1.0, 1e-38), (1e-30, -1e-25), (1e-25, 1e24), (1e30, 1e-31)):
        for softcap in (0.0, 7.0):
            both(kv, (q * np.float32(size)).astype(np.float32), tables, lens, starts, heads, hd, rows, max(new),
                 scale=scale, softcap=softcap)
