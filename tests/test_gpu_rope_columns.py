"""Rotary appends whose rows and outputs are columns of one buffer, and steps without
sequences."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_steps import rope_case, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 5, 1500])
@pytest.mark.parametrize("order", ["qkvo", "oqkv", "kovq"])
def test_outputs_as_columns(gpu, order, n, rows):
    """q, k, v and the output in any order of columns of one buffer."""
    import torch

    ref, slots, positions, q, k, v = rope_case("f16", rows, (4, 2, 64), 64, True, "linear", n, 6, top=4096)
    kv = rope_case("f16", rows, (4, 2, 64), 64, True, "linear", n, 6, top=4096)[0]
    sd, pd = up(slots, np.int32), up(positions, np.int32)
    want = ref.write_rope_rows(0, sd, pd, k, v, q=q, n_heads=4)
    parts = {"q": q, "k": k, "v": v, "o": torch.zeros_like(q)}
    buf = torch.cat([parts[x] for x in order], dim=1)
    col, at = {}, 0
    for x in order:
        col[x] = buf[:, at:at + parts[x].shape[1]]
        at += parts[x].shape[1]
    kv.write_rope_rows(0, sd, pd, col["k"], col["v"], q=col["q"], n_heads=4, out=col["o"])
    kv.synchronize(), ref.synchronize()
    assert torch.equal(col["o"], want)
    for x in "qkv":
        assert torch.equal(col[x], parts[x])
    for a, b in zip(kv.read_pool(0), ref.read_pool(0)):
        np.testing.assert_array_equal(a, b)


def test_overlapping_columns_are_refused(gpu):
    import torch

    from langtrain_studio_amd import KvError

    kv, slots, positions, q, k, v = rope_case("f16", "f32", (4, 2, 64), 64, True, "none", 4, 9, top=100)
    sd, pd = up(slots, np.int32), up(positions, np.int32)
    wide = torch.zeros((5, 1024), device="cuda")
    for a, b, at in [(wide[:4, :256], wide[:4, 128:384], 128), (wide[:4, 512:768], wide[:4, 384:640], 0),
                     (wide[:4, :256], wide[1:, 4:260], 128), (wide[1:, :256], wide[:4, 252:508], 128)]:
        with pytest.raises(KvError, match="q and its output overlap"):
            kv.write_rope_rows(0, sd, pd, k, v, q=a, n_heads=4, out=b)
        other = torch.zeros((5, 1024), device="cuda")[:4, :128]
        for x, y in ((a[:, at:at + 128], other), (other, a[:, at:at + 128])):
            with pytest.raises(KvError, match="overlaps the rows of K or V"):
                kv.write_rope_rows(0, sd, pd, x, y, q=q, n_heads=4, out=b)
    # (a row's end that reaches the next row's begin)
    narrow = torch.zeros((5, 512), device="cuda")
    with pytest.raises(KvError, match="q and its output overlap"):
        kv.write_rope_rows(0, sd, pd, k, v, q=narrow[:4, :256], n_heads=4,
                           out=narrow.view(-1)[260:260 + 4 * 512].view(4, 512)[:, :256])


def test_steps_without_sequences(gpu):
    import torch

    from test_gpu_drafts import HD, HEADS, KVH, backend

    b = backend()
    step = b.begin_drafts([])
    rows = [torch.zeros((0, w), device="cuda", dtype=torch.bfloat16) for w in (HEADS * HD, KVH * HD, KVH * HD)]
    assert b.draft_layer(step, 0, *rows, window=3).shape == (0, HEADS * HD)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    kept, done = b.accept(step, none, none)
    assert kept == [] and done.path.numel() == 0
