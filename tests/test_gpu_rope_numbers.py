"""Numbers of scaled rotary positions that are no f32 numbers: the frequencies are
those of the 64-bit numbers, at positions where their rounding to f32 would show."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_gpu_scored import held_rows
from test_gpu_steps import check_rotation, down, frequencies, rope_case, up

pytestmark = pytest.mark.gpu

KINDS = {"none": {}, "linear": dict(factor=1.3), "ntk": dict(factor=1.7),
         "yarn": dict(factor=3.3, original=4096, low=1.1, high=30.3),
         "llama3": dict(factor=6.7, original=8192, low=1.1, high=4.3)}


@pytest.mark.parametrize("divisors", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_numbers_of_64_bits(gpu, kind, divisors):
    top, base, d = 131072, 10000.1, 128
    div = np.linspace(1.1, 3.3, d // 2) if divisors else None
    kv, slots, positions, q, k, v = rope_case("f32", "f32", (8, 2, 128), d, True, "none", 45, 3, top=top)
    kv.rope_init_scaled(base, d, 128, True, top, kind=kind, divisors=div, **KINDS[kind])
    f, mag = frequencies(base, d, kind, **KINDS[kind])
    if divisors:
        f = f / div
    out = kv.write_rope_rows(0, up(slots, np.int32), up(positions, np.int32), k, v, q=q, n_heads=8)
    kv.synchronize()
    check_rotation(down(out), down(q), positions, 128, d, True, f, mag, "f32")
    check_rotation(held_rows(kv)[0][slots], down(k), positions, 128, d, True, f, mag, "f32")


def test_numbers_of_32_bits(gpu):
    """The entry for f32 numbers: the table of those numbers as they are."""
    from langtrain_studio_amd import _lib

    made = []
    div = np.linspace(1.1, 3.3, 32).astype(np.float32)
    for wide in (False, True):
        kv, slots, positions, q, k, v = rope_case("f32", "f32", (4, 2, 64), 64, False, "none", 20, 5, top=5000)
        base, factor, low, high = (float(np.float32(x)) for x in (10000.1, 3.3, 1.1, 4.3))
        if wide:
            kv.rope_init_scaled(base, 64, 64, False, 5000, kind="llama3", factor=factor, original=2048, low=low, high=high,
                                divisors=div.astype(np.float64), magnitude=1.25)
        else:
            assert _lib.load().ltkv_rope_init_scaled(kv._h, base, 64, 64, 0, 5000, _lib.ROPE_LLAMA3, factor, 2048, low,
                                                     high, div.ctypes.data_as(C.c_void_p), 1.25) == 0
        made.append(kv.write_rope_rows(0, up(slots, np.int32), up(positions, np.int32), k, v, q=q, n_heads=4))
        kv.synchronize()
    assert (made[0] == made[1]).all()


def test_refusals(gpu):
    from langtrain_studio_amd import KvError, _lib

    kv = rope_case("f16", "f32", (4, 2, 64), 64, True, "none", 4, 9, top=100)[0]
    for match, how in [("out of range", dict(kind="linear", factor=1e-308)), ("out of range", dict(divisors=[1e-308] * 32)),
                       ("divisors must be", dict(divisors=[float("nan")] * 32)),
                       ("factor", dict(kind="ntk", factor=float("inf")))]:
        with pytest.raises(KvError, match=match):
            kv.rope_init_scaled(1e4, 64, 64, True, 1000, **how)
    assert _lib.load().ltkv_rope_init_scaled64(kv._h, 64, 64, 0, 100, 0, 0, None, None, 0.0) == _lib.ERR_ARG


@pytest.mark.parametrize("factor,magnitude", [(0.25, 1.0), (1.0, 1.0), (1e-6, 1.0), (2.0, 0.1 * np.log(2.0) + 1.0)])
def test_yarn_magnitudes(gpu, factor, magnitude):
    """Contexts that are not stretched keep the rows' size; a magnitude given is taken."""
    for own in (True, False):
        kv, slots, positions, q, k, v = rope_case("f32", "f32", (4, 2, 64), 64, True, "none", 20, 5, top=500)
        kv.rope_init_scaled(10000.0, 64, 64, True, 500, kind="yarn", factor=factor, original=128,
                            magnitude=None if own else 0.75)
        f, _ = frequencies(10000.0, 64, "yarn", factor, 128)
        out = kv.write_rope_rows(0, up(slots, np.int32), up(positions, np.int32), k, v, q=q, n_heads=4)
        kv.synchronize()
        check_rotation(down(out), down(q), positions, 64, 64, True, f, magnitude if own else 0.75, "f32")
