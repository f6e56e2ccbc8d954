"""Paged KV cache on one MI355X: the Python face of libltkv.so.

``KvCache`` mirrors ``langtrain_native::kv::KvCache``
(engine/crates/native/src/kv.rs:15-188): same constructor arguments, same
method names, same errors ("KV cache full", "seq S: position P is not
contiguous (length L)"), same block-allocation order. K and V live in HBM;
``write``/``rows`` take and return host rows like the reference, and the
batched device ops take torch device tensors (torch supplies device memory
and streams only; all compute is the HIP kernels of libltkv.so).
"""

from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Sequence

import numpy as np

from . import _lib

BLOCK = _lib.BLOCK  # kv.rs:13


class KvError(RuntimeError):
    """An error returned by the C ABI (code = LTKV_ERR_*)."""

    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


class KvCacheFull(KvError):
    """kv.rs:71 "KV cache full"."""


class NonContiguous(KvError):
    """kv.rs:88-91 "seq S: position P is not contiguous (length L)"."""


_ERROR_TYPES = {_lib.ERR_FULL: KvCacheFull, _lib.ERR_NONCONTIG: NonContiguous}


def _check(rc: int) -> None:
    if rc != _lib.OK:
        raise _ERROR_TYPES.get(rc, KvError)(rc, _lib.last_error())


def _np_ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


_torch = None


def _dev_ptr(t, dtype, name: str, device: int) -> int:
    """Device address of a contiguous torch tensor of the given dtype. A
    decode call checks seven tensors, ~0.7 us each with the module lookup,
    ``t.device`` object and ctypes pointer of each, so the good case takes the
    cheapest form of the same tests."""
    global _torch
    if _torch is None:
        import torch as _torch
    if not isinstance(t, _torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a HIP device tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, cache is on device {device}")
    return t.data_ptr()


_types = None


def _row_types() -> dict:
    """LTKV_ROWS_* code of each torch type that rows may have."""
    global _types
    if _types is None:
        import torch

        _types = {torch.float32: _lib.ROWS_F32, torch.float16: _lib.ROWS_F16, torch.bfloat16: _lib.ROWS_BF16}
    return _types


def _int32_parts(sizes, empty):
    """int32 tensors of these sizes in one allocation of empty(shape, dtype), and
    their addresses (each 16-byte aligned)."""
    import torch

    starts, total = [], 0
    for size in sizes:
        starts.append(total)
        total += -(-size // 4) * 4
    buf = empty((total,), torch.int32)
    base = buf.data_ptr()
    return [buf[at:at + size] for at, size in zip(starts, sizes)], [base + 4 * at for at in starts]


class StepLayout(NamedTuple):
    """The device arrays of a step (KvCache.step_layout), int32."""

    row_starts: "object"    # [n + 1]: request i has tokens row_starts[i]..row_starts[i+1]
    lens: "object"          # [n]: lengths, the step's tokens included
    tables: "object"        # [n][stride]: block tables, -1 behind their ends
    slot_mapping: "object"  # [n_tokens]: each token's cell, -1 behind the last token
    positions: "object"     # [n_tokens]: each token's position, -1 behind the last token
    masks: "object" = None  # [n_tokens][words]: a drafted token's ancestors and itself


class _OwnLayout(StepLayout):
    """A layout as step_layout made it: its sizes and the addresses of its arrays."""

    sizes = None
    pointers = None


class AcceptedTree(NamedTuple):
    """What KvCache.accept_tree kept, int32 on the device."""

    accepted: "object"  # [n]: tokens kept
    path: "object"      # [n_rows]: the kept tokens of each request in order, -1 behind them
    next: "object"      # [n]: the token behind the last kept one
    lens: "object"      # [n]: lengths after it


class KvCache:
    """kv.rs KvCache with its pools in HBM.

    ``KvCache(n_layers, kv_dim, n_tokens)`` is ``KvCache::new`` (kv.rs:35-48);
    ``dtype`` selects the storage ("f16" as the reference, "f32", "q8_0":
    int8 quants with one f16 scale per 32 elements, quant.rs:785-791, or
    "q4_0": 4-bit quants with one) and ``device`` the HIP device (``None`` = a metadata-only cache with no
    pools, whose device ops raise).
    """

    def __init__(self, n_layers: int, kv_dim: int, n_tokens: int, dtype: str = "f16",
                 device: Optional[int] = 0, stream=None):
        codes = {"f16": _lib.F16, "f32": _lib.F32, "q8_0": _lib.Q8_0, "q4_0": _lib.Q4_0}
        if dtype not in codes:
            raise ValueError("dtype must be 'f16', 'f32', 'q8_0' or 'q4_0'")
        self._lib = _lib.load()
        h = C.c_void_p()
        dev = _lib.NO_DEVICE if device is None else int(device)
        _check(self._lib.ltkv_create(n_layers, kv_dim, n_tokens, codes[dtype], dev, C.byref(h)))
        self._h = h
        self.n_layers = n_layers
        self.dtype = dtype
        self.elem = {"f16": 2, "f32": 4, "q8_0": 1, "q4_0": 0.5}[dtype]  # bytes per element, scales apart
        self.device = device
        self.n_blocks = self._lib.ltkv_n_blocks(h)
        self._kv_dim = self._lib.ltkv_kv_dim(h)
        self._plan_shape = None
        self._rope_dims = self._rope_positions = 0  # head_dim and positions of the RoPE table
        self._stream = 0
        if stream is not None:
            self.set_stream(stream)

    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            self._lib.ltkv_destroy(h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def set_stream(self, stream) -> None:
        """Enqueue device work on ``stream`` (a torch.cuda.Stream or a raw hipStream_t)."""
        raw = int(getattr(stream, "cuda_stream", stream) or 0)
        _check(self._lib.ltkv_set_stream(self._h, C.c_void_p(raw)))
        self._stream = raw

    # ---- kv.rs:17-18,50-60,185-187 --------------------------------------------------
    @property
    def kv_dim(self) -> int:
        return self._kv_dim

    def capacity(self) -> int:
        return self._lib.ltkv_capacity(self._h)

    def bytes(self) -> int:
        return self._lib.ltkv_bytes(self._h)

    def len(self, seq: int) -> int:
        return self._lib.ltkv_len(self._h, seq)

    def free_blocks(self) -> int:
        return self._lib.ltkv_free_blocks(self._h)

    def refcount(self, block: int) -> int:
        return self._lib.ltkv_refcount(self._h, block)

    def cow_copies(self) -> int:
        return self._lib.ltkv_cow_copies(self._h)

    # ---- kv.rs:85-121 ---------------------------------------------------------------
    def append(self, seq: int, pos: int) -> tuple[int, int]:
        """Reserve the cell of ``pos`` (== len(seq)); returns (block, slot)."""
        b, s = C.c_uint32(), C.c_uint32()
        _check(self._lib.ltkv_append(self._h, seq, pos, C.byref(b), C.byref(s)))
        return b.value, s.value

    def append_batch(self, seqs, positions) -> np.ndarray:
        """The cell claim of model.rs:380-383: slot mapping block*16+slot per token."""
        seqs = np.ascontiguousarray(seqs, dtype=np.uint32)
        pos = np.ascontiguousarray(positions, dtype=np.uint64)
        if seqs.shape != pos.shape:
            raise ValueError("seqs and positions differ in length")
        out = np.full(seqs.size, -1, dtype=np.int32)
        done = C.c_size_t()
        rc = self._lib.ltkv_append_batch(self._h, seqs.size, _np_ptr(seqs), _np_ptr(pos), _np_ptr(out),
                                         C.byref(done))
        if rc != _lib.OK:
            err = _ERROR_TYPES.get(rc, KvError)(rc, _lib.last_error())
            err.n_done = done.value
            err.slot_mapping = out
            raise err
        return out

    # ---- kv.rs:123-131 --------------------------------------------------------------
    def write(self, layer: int, block: int, slot: int, k, v) -> None:
        """Write one token's K and V rows (f32, kv_dim each) into (block, slot)."""
        k = np.ascontiguousarray(k, dtype=np.float32).reshape(-1)
        v = np.ascontiguousarray(v, dtype=np.float32).reshape(-1)
        if k.size != self.kv_dim or v.size != self.kv_dim:
            raise ValueError(f"rows must have kv_dim={self.kv_dim} elements")
        _check(self._lib.ltkv_write_row(self._h, layer, block, slot, _np_ptr(k), _np_ptr(v)))

    # ---- kv.rs:133-150 --------------------------------------------------------------
    def rows(self, layer: int, seq: int, n: int) -> tuple[np.ndarray, np.ndarray]:
        """K and V rows of positions 0..n of seq as host [n][kv_dim] arrays
        (uint16 f16 bits, or float32)."""
        dt = np.uint16 if self.elem == 2 else np.float32
        k = np.empty((n, self.kv_dim), dtype=dt)
        v = np.empty((n, self.kv_dim), dtype=dt)
        _check(self._lib.ltkv_rows(self._h, layer, seq, n, _np_ptr(k), _np_ptr(v)))
        return k, v

    # ---- kv.rs:153-183 --------------------------------------------------------------
    def truncate(self, seq: int, from_: int) -> None:
        self._lib.ltkv_truncate(self._h, seq, from_)

    def share(self, src: int, dst: int, length: int) -> None:
        self._lib.ltkv_share(self._h, src, dst, length)

    # ---- tables ---------------------------------------------------------------------
    def block_table(self, seq: int) -> np.ndarray:
        n = C.c_size_t()
        self._lib.ltkv_block_table(self._h, seq, None, 0, C.byref(n))
        out = np.empty(n.value, dtype=np.int32)
        _check(self._lib.ltkv_block_table(self._h, seq, _np_ptr(out), out.size, C.byref(n)))
        return out

    def block_tables(self, seqs, stride: Optional[int] = None) -> np.ndarray:
        seqs = np.ascontiguousarray(seqs, dtype=np.uint32)
        if stride is None:
            stride = max([1] + [math.ceil(self.len(int(s)) / BLOCK) for s in seqs])
        out = np.empty((seqs.size, stride), dtype=np.int32)
        _check(self._lib.ltkv_block_tables(self._h, seqs.size, _np_ptr(seqs), _np_ptr(out), stride))
        return out

    def init_free_order(self, order) -> None:
        o = np.ascontiguousarray(order, dtype=np.uint32)
        _check(self._lib.ltkv_init_free_order(self._h, _np_ptr(o), o.size))

    # ---- device ops (torch device tensors) ------------------------------------------
    def write_batch(self, layer: int, slot_mapping, k, v) -> None:
        """Kernel 1: rows of k, v ([n][>=kv_dim] f32) into cells slot_mapping[n] (int32)."""
        import torch

        n = slot_mapping.numel()
        if k.dim() != 2 or k.shape != v.shape or k.shape[0] != n or k.shape[1] < self.kv_dim:
            raise ValueError("k and v must be [n][>=kv_dim] and match slot_mapping")
        _check(self._lib.ltkv_write(
            self._h, layer, n, _dev_ptr(slot_mapping, torch.int32, "slot_mapping", self.device),
            _dev_ptr(k, torch.float32, "k", self.device), _dev_ptr(v, torch.float32, "v", self.device),
            k.shape[1]))

    def cell_order(self, slot_mapping) -> np.ndarray:
        """Host: the rows of a claimed batch grouped by block in ascending
        block order (ltkv_cell_order), skipped cells left out (int32)."""
        sm = np.ascontiguousarray(slot_mapping, dtype=np.int32)
        order = np.empty(sm.size, dtype=np.int32)
        m = C.c_size_t(0)
        _check(self._lib.ltkv_cell_order(self._h, sm.size, _np_ptr(sm), _np_ptr(order), C.byref(m)))
        return order[:m.value]

    def write_batch_ordered(self, layer: int, slot_mapping, k, v, order) -> None:
        """Kernel 1 over the rows order[m] (int32, device) of a batch:
        row order[j] of k, v into cell slot_mapping[order[j]]."""
        import torch

        n = slot_mapping.numel()
        if k.dim() != 2 or k.shape != v.shape or k.shape[0] != n or k.shape[1] < self.kv_dim:
            raise ValueError("k and v must be [n][>=kv_dim] and match slot_mapping")
        _check(self._lib.ltkv_write_ordered(
            self._h, layer, n, _dev_ptr(slot_mapping, torch.int32, "slot_mapping", self.device),
            _dev_ptr(k, torch.float32, "k", self.device), _dev_ptr(v, torch.float32, "v", self.device),
            k.shape[1], order.numel(), _dev_ptr(order, torch.int32, "order", self.device)))

    def rope_init(self, base: float, rope_dim: int, head_dim: int, neox: bool, max_positions: int) -> None:
        """RoPE table of Model::rope (model.rs:263-265, 291-308) for write_rope."""
        _check(self._lib.ltkv_rope_init(self._h, float(base), rope_dim, head_dim, 1 if neox else 0,
                                        max_positions))
        self._rope_dims, self._rope_positions = head_dim, max_positions

    def write_rope(self, layer: int, slot_mapping, positions, k, v, q=None, n_heads: int = 0) -> None:
        """Kernel 1 with RoPE (model.rs:414-429): k rotated into its cell, v appended,
        q ([n][n_heads*head_dim] f32, optional) rotated in place."""
        import torch

        n = slot_mapping.numel()
        if k.dim() != 2 or k.shape != v.shape or k.shape[0] != n or k.shape[1] < self.kv_dim:
            raise ValueError("k and v must be [n][>=kv_dim] and match slot_mapping")
        if positions.numel() != n:
            raise ValueError("positions must match slot_mapping")
        qp, qs = None, 0
        if q is not None:
            if q.dim() != 2 or q.shape[0] != n:
                raise ValueError("q must be [n][n_heads*head_dim]")
            qp, qs = _dev_ptr(q, torch.float32, "q", self.device), q.shape[1]
        _check(self._lib.ltkv_write_rope(
            self._h, layer, n, _dev_ptr(slot_mapping, torch.int32, "slot_mapping", self.device),
            _dev_ptr(positions, torch.int32, "positions", self.device),
            _dev_ptr(k, torch.float32, "k", self.device), _dev_ptr(v, torch.float32, "v", self.device),
            k.shape[1], qp, qs, n_heads))

    def rope_init_scaled(self, base: float, rope_dim: int, head_dim: int, neox: bool, max_positions: int,
                         kind: str = "none", factor: float = 1.0, original: int = 0, low: Optional[float] = None,
                         high: Optional[float] = None, divisors=None, magnitude: Optional[float] = None) -> None:
        """rope_init with frequencies scaled for long contexts
        (ltkv_rope_init_scaled64): kind "none", "linear", "ntk", "yarn" or "llama3" by
        `factor`; yarn and llama3 keep the frequencies of pairs that turn `high`
        (32; 4) times within `original` positions and scale those that turn up to
        `low` (1) times. divisors: one per pair. magnitude: of the cosines and
        sines (default: the kind's own)."""
        kinds = {"none": (_lib.ROPE_PLAIN, 1.0, 1.0), "linear": (_lib.ROPE_LINEAR, 1.0, 1.0),
                 "ntk": (_lib.ROPE_NTK, 1.0, 1.0), "yarn": (_lib.ROPE_YARN, 1.0, 32.0),
                 "llama3": (_lib.ROPE_LLAMA3, 1.0, 4.0)}
        if kind not in kinds:
            raise ValueError(f"kind must be one of {sorted(kinds)}")
        if rope_dim < 0 or head_dim < 0 or max_positions < 0 or original < 0:
            raise ValueError("rope_dim, head_dim, max_positions and original must not be negative")
        if magnitude is not None and not magnitude > 0:
            raise ValueError("magnitude must be positive")
        code, lo, hi = kinds[kind]
        if divisors is not None:
            divisors = np.ascontiguousarray(divisors, dtype=np.float64).reshape(-1)
            if divisors.size != rope_dim // 2:
                raise ValueError("divisors must have rope_dim / 2 entries")
        numbers = np.array([base, factor, lo if low is None else low, hi if high is None else high], np.float64)
        _check(self._lib.ltkv_rope_init_scaled64(
            self._h, rope_dim, head_dim, 1 if neox else 0, max_positions, code, original, _np_ptr(numbers),
            None if divisors is None else _np_ptr(divisors), 0.0 if magnitude is None else float(magnitude)))
        self._rope_dims, self._rope_positions = head_dim, max_positions

    def write_rope_rows(self, layer: int, slot_mapping, positions, k, v, q=None, n_heads: int = 0, out=None):
        """write_rope for f32, f16 or bf16 rows: k rotated into its cell, v
        appended, and q ([n][n_heads*head_dim], optional) rotated into out, which
        is returned (default: a new tensor; out=q rotates in place). A token whose
        position is outside the RoPE table is skipped: no cell of it is written, and
        its row of q is left as it was (zeros in a new out). Rows may be columns of a
        wider tensor (unit stride within a row)."""
        import torch

        n = slot_mapping.numel()
        dtype, dev = k.dtype, self.device
        code = _row_types().get(dtype)
        if code is None:
            raise TypeError(f"k must be float32, float16 or bfloat16, got {dtype}")
        shape = k.shape
        if len(shape) != 2 or shape != v.shape or shape[0] != n or shape[1] != self._kv_dim:
            raise ValueError("k and v must be [n][kv_dim] and match slot_mapping")
        if positions.numel() != n:
            raise ValueError("positions must match slot_mapping")

        def rows(t, name):
            if t.dtype is not dtype:
                raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
            if not t.is_cuda or t.get_device() != dev:
                raise ValueError(f"{name} must be on the cache's device")
            across, along = t.stride()
            if along != 1 or across < 0:
                raise ValueError(f"{name} must have rows of unit stride")
            # (the stride of a single row may be anything)
            return t.data_ptr(), across if n > 1 else -(-t.shape[1] // 8) * 8

        kp, ks = rows(k, "k")
        vp, vs = rows(v, "v")
        if ks != vs:
            raise ValueError("k and v must have the same row stride")
        qp = op = None
        qs = os = 0
        if q is not None:
            shape = q.shape
            if len(shape) != 2 or shape[0] != n or (self._rope_dims and n_heads * self._rope_dims != shape[1]):
                raise ValueError("q must be [n][n_heads*head_dim]")
            if out is None:
                out = self._zeros_like(q)  # (rows of skipped tokens)
            elif out.shape != shape:
                raise ValueError("out must match q")
            qp, qs = rows(q, "q")
            op, os = (qp, qs) if out is q else rows(out, "out")
        elif out is not None:
            raise ValueError("out without q")
        _check(self._lib.ltkv_write_rope_rows(
            self._h, layer, n, _dev_ptr(slot_mapping, torch.int32, "slot_mapping", dev),
            _dev_ptr(positions, torch.int32, "positions", dev), code, kp, vp, ks, qp, qs, n_heads, op, os))
        return out

    def copy_blocks(self, pairs) -> None:
        """Kernel 2: copy block pairs[i,0] -> pairs[i,1] (all layers, K and V)."""
        import torch

        if pairs.dim() != 2 or pairs.shape[1] != 2:
            raise ValueError("pairs must be [n][2]")
        _check(self._lib.ltkv_copy_blocks(self._h, pairs.shape[0],
                                          _dev_ptr(pairs, torch.int32, "pairs", self.device)))

    def gather(self, layer: int, tables, lens, out_offsets, k_out, v_out) -> None:
        """Kernel 3: rows 0..lens[i] of each table to k_out/v_out rows out_offsets[i]..."""
        import torch

        dt = {0.5: torch.int8, 1: torch.int8, 2: torch.float16, 4: torch.float32}[self.elem]
        n = self._gather_args(tables, lens, out_offsets, k_out, v_out)
        _check(self._lib.ltkv_gather(
            self._h, layer, n, _dev_ptr(tables, torch.int32, "tables", self.device), tables.shape[1],
            _dev_ptr(lens, torch.int32, "lens", self.device),
            _dev_ptr(out_offsets, torch.int64, "out_offsets", self.device),
            _dev_ptr(k_out, dt, "k_out", self.device), _dev_ptr(v_out, dt, "v_out", self.device)))

    def _gather_args(self, tables, lens, out_offsets, k_out, v_out) -> int:
        n = lens.numel()
        if tables.dim() != 2 or tables.shape[0] != n or out_offsets.numel() != n:
            raise ValueError("tables must be [n][stride]; lens and out_offsets [n]")
        if k_out.dim() != 2 or k_out.shape[1] != self.kv_dim or v_out.shape != k_out.shape:
            raise ValueError("k_out and v_out must be [rows][kv_dim]")
        return n

    def gather_values(self, layer: int, tables, lens, out_offsets, k_out, v_out) -> None:
        """gather with the rows as f32 values, for caches of every dtype: rows
        0..lens[i] of each table to the f32 k_out/v_out rows out_offsets[i]..."""
        import torch

        n = self._gather_args(tables, lens, out_offsets, k_out, v_out)
        _check(self._lib.ltkv_gather_values(
            self._h, layer, n, _dev_ptr(tables, torch.int32, "tables", self.device), tables.shape[1],
            _dev_ptr(lens, torch.int32, "lens", self.device),
            _dev_ptr(out_offsets, torch.int64, "out_offsets", self.device),
            _dev_ptr(k_out, torch.float32, "k_out", self.device),
            _dev_ptr(v_out, torch.float32, "v_out", self.device)))

    def scored_attention(self, layer: int, q, tables, lens, n_heads: int, head_dim: int, row_starts=None,
                         max_rows: Optional[int] = None, scale: Optional[float] = None, softcap: float = 0.0,
                         slopes=None, window: int = 0, sinks: int = 0, prefix=None, first=None, out=None):
        """Attention with capped scores, distance biases and masks
        (ltkv_scored_attention) for single tokens and prompt chunks: sequence i
        has rows row_starts[i]..row_starts[i+1] of q ([n_rows][n_heads*head_dim],
        f32, f16 or bf16; row_starts int32 [n+1], None: one row each), the last
        of its lens[i] positions. softcap > 0: scores become softcap *
        tanh(score / softcap). slopes (f32 [n_heads]): score minus slope *
        distance. window > 0: a row sees that many positions up to its own, and
        the first `sinks`. prefix (int32 [n]): positions every row of the
        sequence sees. first (int32 [n_rows]): the first position of the row's
        document. max_rows: the most rows of one sequence (a hint; default: as
        many as there are). Rows of no sequence are left as they were (zeros in a
        new out)."""
        import torch

        n = lens.numel()
        types = _row_types()
        if q.dim() != 2 or q.shape[1] != n_heads * head_dim:
            raise ValueError("q must be [n_rows][n_heads*head_dim]")
        if q.dtype not in types:
            raise TypeError(f"q must be float32, float16 or bfloat16, got {q.dtype}")
        if tables.dim() != 2 or tables.shape[0] != n:
            raise ValueError("tables must be [n][stride]")
        n_rows = q.shape[0]
        if row_starts is None:
            if n_rows != n:
                raise ValueError("without row_starts q must have one row per sequence")
        elif row_starts.numel() != n + 1:
            raise ValueError("row_starts must have one entry per sequence and one more")
        if out is None:
            out = self._zeros_like(q) if row_starts is not None else torch.empty_like(q)
        elif out.shape != q.shape:
            raise ValueError("out must match q")
        if scale is None:
            scale = 1.0 / math.sqrt(head_dim)  # model.rs:402
        if window < 0 or sinks < 0 or (max_rows is not None and max_rows < 0):
            raise ValueError("window, sinks and max_rows must not be negative")

        def given(t, dtype, name, size):
            if t is None:
                return None
            if t.numel() != size:
                raise ValueError(f"{name} must have {size} entries")
            return _dev_ptr(t, dtype, name, self.device)

        _check(self._lib.ltkv_scored_attention(
            self._h, layer, n, n_rows, n_rows if max_rows is None else max_rows, n_heads, head_dim, float(scale),
            float(softcap), given(slopes, torch.float32, "slopes", n_heads), window, sinks,
            given(prefix, torch.int32, "prefix", n), given(first, torch.int32, "first", n_rows), types[q.dtype],
            _dev_ptr(q, q.dtype, "q", self.device), _dev_ptr(tables, torch.int32, "tables", self.device),
            tables.shape[1], _dev_ptr(lens, torch.int32, "lens", self.device),
            given(row_starts, torch.int32, "row_starts", n + 1), _dev_ptr(out, q.dtype, "out", self.device)))
        return out

    def tree_attention(self, layer: int, q, tables, lens, n_heads: int, head_dim: int, row_starts, positions=None,
                       masks=None, max_rows: Optional[int] = None, scale: Optional[float] = None,
                       softcap: float = 0.0, window: int = 0, out=None):
        """Attention of drafted rows over the cache (ltkv_tree_attention):
        sequence i has rows row_starts[i]..row_starts[i+1] of q
        ([n_rows][n_heads*head_dim], f32, f16 or bf16), the last cells of its
        lens[i] positions. A row sees the context in front of them (with window >
        0: less than that many positions back from positions[row], int32
        [n_rows]) and the rows whose bits its masks (int32 [n_rows][words]) hold,
        window or not (window_masks bounds them by it); without masks the rows up
        to its own. softcap > 0: scores become softcap
        * tanh(score / softcap). max_rows: the most rows of one sequence (a hint;
        default: as many as there are). Rows of no sequence are left as they were
        (zeros in a new out)."""
        import torch

        n = lens.numel()
        types = _row_types()
        if q.dim() != 2 or q.shape[1] != n_heads * head_dim:
            raise ValueError("q must be [n_rows][n_heads*head_dim]")
        if q.dtype not in types:
            raise TypeError(f"q must be float32, float16 or bfloat16, got {q.dtype}")
        if tables.dim() != 2 or tables.shape[0] != n:
            raise ValueError("tables must be [n][stride]")
        n_rows = q.shape[0]
        if row_starts.numel() != n + 1:
            raise ValueError("row_starts must have one entry per sequence and one more")
        words = 0
        if masks is not None:
            if masks.dim() != 2 or masks.shape[0] != n_rows or masks.shape[1] == 0:
                raise ValueError("masks must be [n_rows][words], of at least one word")
            words = masks.shape[1]
        if positions is not None and positions.numel() != n_rows:
            raise ValueError("positions must have one entry per row")
        if window < 0 or (max_rows is not None and max_rows < 0):
            raise ValueError("window and max_rows must not be negative")
        if out is None:
            out = self._zeros_like(q)
        elif out.shape != q.shape:
            raise ValueError("out must match q")
        if scale is None:
            scale = 1.0 / math.sqrt(head_dim)  # model.rs:402
        _check(self._lib.ltkv_tree_attention(
            self._h, layer, n, n_rows, n_rows if max_rows is None else max_rows, n_heads, head_dim, float(scale),
            float(softcap), window,
            None if positions is None else _dev_ptr(positions, torch.int32, "positions", self.device),
            None if masks is None else _dev_ptr(masks, torch.int32, "masks", self.device), words, types[q.dtype],
            _dev_ptr(q, q.dtype, "q", self.device), _dev_ptr(tables, torch.int32, "tables", self.device),
            tables.shape[1], _dev_ptr(lens, torch.int32, "lens", self.device),
            _dev_ptr(row_starts, torch.int32, "row_starts", self.device), _dev_ptr(out, q.dtype, "out", self.device)))
        return out

    def step_layout(self, rows, lens, counts, n_tokens: int, table_stride: int, parents=None, mask_words: int = 0,
                    out: Optional[StepLayout] = None) -> StepLayout:
        """The arrays of a step from its requests' lengths, on the device
        (ltkv_step_layout): request i holds lens[i] tokens of the sequence in
        resident table row rows[i] (seq_rows; -1: no request) and gets counts[i]
        new ones (None: one each), whose cells are claimed. parents ([n_tokens]):
        each token's parent among its request's (-1: a root), for positions by
        depth and the masks of tree_attention. All int32 device tensors; out: the
        arrays of an earlier call to fill again."""
        import torch

        n = rows.numel()
        if n_tokens < 0 or table_stride < 0 or mask_words < 0:
            raise ValueError("n_tokens, table_stride and mask_words must not be negative")
        if lens.numel() != n or (counts is not None and counts.numel() != n):
            raise ValueError("rows, lens and counts must have equal length")
        if parents is not None and parents.numel() != n_tokens:
            raise ValueError("parents must have n_tokens entries")
        int32, dev = torch.int32, self.device
        sizes = (n, n_tokens, table_stride, mask_words if parents is not None else None, dev)
        if out is None:
            parts, pointers = _int32_parts(
                [n + 1, n, n * table_stride, n_tokens, n_tokens] +
                ([n_tokens * mask_words] if parents is not None else []), self._empty)
            parts[2] = parts[2].view(n, table_stride)
            if parents is not None:
                parts[5] = parts[5].view(n_tokens, mask_words)
            else:
                parts.append(None)
                pointers.append(None)
            out = _OwnLayout(*parts)
            out.sizes, out.pointers = sizes, pointers
        pointers = None
        if isinstance(out, _OwnLayout) and out.sizes == sizes and out.row_starts.data_ptr() == out.pointers[0]:
            pointers = out.pointers
        else:  # arrays of the caller's own (or a copy of a layout)
            shapes = [(n + 1,), (n,), (n, table_stride), (n_tokens,), (n_tokens,),
                      (n_tokens, mask_words) if parents is not None else None]
            for name, t, shape in zip(StepLayout._fields, out, shapes):
                if (t is None) != (shape is None) or (t is not None and tuple(t.shape) != shape):
                    raise ValueError(f"out.{name} must have shape {shape}")
            pointers = [None if t is None else _dev_ptr(t, int32, f"out.{name}", dev)
                        for name, t in zip(StepLayout._fields, out)]
        if n == 0:  # nothing to lay out: every token is behind the last one
            with self._ordered():
                out.row_starts.zero_()
                for t in (out.slot_mapping, out.positions):
                    t.fill_(-1)
                if out.masks is not None:
                    out.masks.zero_()
            return out
        if n_tokens == 0:  # (empty tensors have no address)
            parents, pointers = None, [*pointers[:5], None]
        _check(self._lib.ltkv_step_layout(
            self._h, n, _dev_ptr(rows, int32, "rows", dev), _dev_ptr(lens, int32, "lens", dev),
            None if counts is None else _dev_ptr(counts, int32, "counts", dev), n_tokens, table_stride,
            None if parents is None else _dev_ptr(parents, int32, "parents", dev),
            mask_words if parents is not None else 0, *pointers))
        return out

    def window_masks(self, row_starts, positions, masks, window: int, out=None):
        """masks (int32 [n_rows][words]) without the rows that lie `window`
        positions or more in front of the one that sees them (ltkv_window_masks),
        for the layers of a model that have a window. All int32 device tensors,
        as step_layout gives them; out: a new tensor, or one to fill (masks
        itself, too)."""
        import torch

        if masks.dim() != 2 or masks.shape[1] == 0:
            raise ValueError("masks must be [n_rows][words], of at least one word")
        n, n_rows = row_starts.numel() - 1, masks.shape[0]
        if n < 0:
            raise ValueError("row_starts must have one entry per sequence and one more")
        if positions.numel() != n_rows:
            raise ValueError("positions must have one entry per row")
        if window <= 0:
            raise ValueError("window must be positive")
        int32, dev = torch.int32, self.device
        if out is None:
            out = self._empty(masks.shape, int32)
        elif out.shape != masks.shape:
            raise ValueError("out must match masks")
        if n == 0 or n_rows == 0:
            with self._ordered():
                out.zero_()
            return out
        _check(self._lib.ltkv_window_masks(
            self._h, n, n_rows, _dev_ptr(row_starts, int32, "row_starts", dev),
            _dev_ptr(positions, int32, "positions", dev), _dev_ptr(masks, int32, "masks", dev), masks.shape[1], window,
            _dev_ptr(out, int32, "out", dev)))
        return out

    def accept_tree(self, tables, lens, row_starts, parents, tokens, targets,
                    out: Optional[AcceptedTree] = None) -> AcceptedTree:
        """Keeps what the model agrees with of every request's drafted tree
        (ltkv_accept_tree), in all layers: rows as in tree_attention; token j of a
        request has parent parents[j] and the model chose targets[j] behind it.
        Token 0 is kept, then from each kept token the lowest child that is its
        target; their K and V rows move together behind the context. All int32
        device tensors; truncate the sequences to the lens returned."""
        import torch

        n, n_rows = lens.numel(), tokens.numel()
        if tables.dim() != 2 or tables.shape[0] != n:
            raise ValueError("tables must be [n][stride]")
        if row_starts.numel() != n + 1:
            raise ValueError("row_starts must have one entry per sequence and one more")
        if parents.numel() != n_rows or targets.numel() != n_rows:
            raise ValueError("parents, tokens and targets must have equal length")
        int32, dev = torch.int32, self.device
        sizes = (n, n_rows, n, n)
        if out is None:
            parts, pointers = _int32_parts(sizes, self._empty)
            out = AcceptedTree(*parts)
        else:
            pointers = []
            for name, t, size in zip(AcceptedTree._fields, out, sizes):
                if t.numel() != size:
                    raise ValueError(f"out.{name} must have {size} entries")
                pointers.append(_dev_ptr(t, int32, f"out.{name}", dev))
        if n == 0:
            with self._ordered():
                out.path.fill_(-1)
            return out
        _check(self._lib.ltkv_accept_tree(
            self._h, n, n_rows, _dev_ptr(tables, int32, "tables", dev), tables.shape[1],
            _dev_ptr(lens, int32, "lens", dev), _dev_ptr(row_starts, int32, "row_starts", dev),
            _dev_ptr(parents, int32, "parents", dev), _dev_ptr(tokens, int32, "tokens", dev),
            _dev_ptr(targets, int32, "targets", dev), *pointers))
        return out

    def _ordered(self):
        """Context in which torch works on the cache's stream, in order with its
        launches."""
        import torch

        if not self._stream:  # (the null stream; ExternalStream(0) is a new one)
            return torch.cuda.stream(torch.cuda.default_stream(self.device))
        return torch.cuda.stream(torch.cuda.ExternalStream(self._stream, device=self.device))

    def _empty(self, shape, dtype):
        """Memory whose earlier use is in order with the cache's launches, whatever
        the current stream is."""
        import torch

        if self.device is None:  # (the call refuses)
            return torch.empty(shape, dtype=dtype)
        current = torch.cuda.current_stream(self.device)
        if current.cuda_stream == self._stream:
            return torch.empty(shape, dtype=dtype, device=current.device)
        with self._ordered():
            out = torch.empty(shape, dtype=dtype, device=current.device)
        out.record_stream(current)  # the caller's: the memory is not reused under its work
        return out

    def _zeros_like(self, t):
        """Zeros cleared on the cache's stream, in order with its launches, whatever
        the current stream is."""
        import torch

        if not t.is_cuda or t.get_device() != self.device:
            return torch.zeros_like(t)  # (the call refuses t)
        current = torch.cuda.current_stream(self.device)
        if current.cuda_stream == self._stream:
            return torch.zeros_like(t)
        with self._ordered():
            out = torch.zeros_like(t)
        out.record_stream(current)  # the caller's: the memory is not reused under its work
        return out

    def decode_attention(self, layer: int, q, tables, lens, n_heads: int, head_dim: int,
                         scale: Optional[float] = None, out=None, noalloc: bool = False):
        """Kernel 4: GQA paged decode attention; q, out are [n][n_heads*head_dim] f32.
        noalloc: ltkv_decode_attention_noalloc (partials in the device's static
        scratch; nothing allocated, same result bits)."""
        import torch

        n = lens.numel()
        if q.dim() != 2 or q.shape != (n, n_heads * head_dim):
            raise ValueError("q must be [n][n_heads*head_dim]")
        if tables.dim() != 2 or tables.shape[0] != n:
            raise ValueError("tables must be [n][stride]")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape:
            raise ValueError("out must match q")
        if scale is None:
            scale = 1.0 / math.sqrt(head_dim)  # model.rs:402
        fn = self._lib.ltkv_decode_attention_noalloc if noalloc else self._lib.ltkv_decode_attention
        _check(fn(
            self._h, layer, n, n_heads, head_dim, float(scale),
            _dev_ptr(q, torch.float32, "q", self.device),
            _dev_ptr(tables, torch.int32, "tables", self.device), tables.shape[1],
            _dev_ptr(lens, torch.int32, "lens", self.device),
            _dev_ptr(out, torch.float32, "out", self.device)))
        return out

    # ---- resident block tables (device step descriptor)
    def seq_rows(self, seqs: Sequence[int]) -> np.ndarray:
        """Row of each sequence in the resident tables (-1: no blocks)."""
        seqs_a = np.ascontiguousarray(seqs, dtype=np.uint32)
        out = np.empty(seqs_a.shape, dtype=np.int32)
        _check(self._lib.ltkv_seq_rows(self._h, seqs_a.size, _np_ptr(seqs_a), _np_ptr(out)))
        return out

    def sync_tables(self) -> None:
        """Enqueue the upload of the block-table changes since the last one."""
        _check(self._lib.ltkv_sync_tables(self._h))

    def resident_tables(self):
        """(tables [rows][stride], lengths [rows]) of the resident tables,
        copied to host after pending uploads (synchronous)."""
        t, l = C.c_void_p(), C.c_void_p()
        stride, rows = C.c_size_t(), C.c_size_t()
        _check(self._lib.ltkv_resident_tables(self._h, C.byref(t), C.byref(l), C.byref(stride),
                                              C.byref(rows)))
        tables = np.empty((rows.value, stride.value), dtype=np.int32)
        lengths = np.empty((rows.value,), dtype=np.int32)
        _check(self._lib.ltkv_read_resident_tables(self._h, _np_ptr(tables), _np_ptr(lengths)))
        return tables, lengths

    def slot_mapping(self, rows, pos, out=None):
        """Slot mapping of tokens (row, position) from the resident tables,
        computed on the device; rows int32, pos int64 device tensors."""
        import torch

        n = rows.numel()
        if pos.numel() != n:
            raise ValueError("rows and pos must have equal length")
        if out is None:
            out = torch.empty((n,), dtype=torch.int32, device=rows.device)
        _check(self._lib.ltkv_slot_mapping(self._h, n, _dev_ptr(rows, torch.int32, "rows", self.device),
                                           _dev_ptr(pos, torch.int64, "pos", self.device),
                                           _dev_ptr(out, torch.int32, "out", self.device)))
        return out

    def decode_attention_rows(self, layer: int, q, rows, lens, n_heads: int, head_dim: int,
                              scale: Optional[float] = None, out=None):
        """decode_attention over the resident tables: query i reads the
        sequence in row rows[i] (device int32)."""
        import torch

        n = lens.numel()
        if q.dim() != 2 or q.shape != (n, n_heads * head_dim):
            raise ValueError("q must be [n][n_heads*head_dim]")
        if rows.numel() != n:
            raise ValueError("rows must have one entry per query")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape:
            raise ValueError("out must match q")
        if scale is None:
            scale = 1.0 / math.sqrt(head_dim)  # model.rs:402
        _check(self._lib.ltkv_decode_attention_rows(
            self._h, layer, n, n_heads, head_dim, float(scale),
            _dev_ptr(q, torch.float32, "q", self.device),
            _dev_ptr(rows, torch.int32, "rows", self.device),
            _dev_ptr(lens, torch.int32, "lens", self.device),
            _dev_ptr(out, torch.float32, "out", self.device)))
        return out

    def table_uploads(self) -> int:
        """Resident-table entries uploaded so far."""
        v = C.c_uint64()
        _check(self._lib.ltkv_table_uploads(self._h, C.byref(v)))
        return int(v.value)

    def append_decode_attention(self, layer: int, slot_mapping, k, v, q, tables, lens, n_heads: int,
                                head_dim: int, scale: Optional[float] = None, out=None):
        """write_batch(layer, slot_mapping, k, v) then decode_attention in one
        launch (tuned shapes): slot_mapping[i] must be position lens[i] - 1 of
        query i's table, one new token per sequence."""
        import torch

        n = lens.numel()
        if q.dim() != 2 or q.shape != (n, n_heads * head_dim):
            raise ValueError("q must be [n][n_heads*head_dim]")
        if tables.dim() != 2 or tables.shape[0] != n:
            raise ValueError("tables must be [n][stride]")
        if k.shape != (n, self.kv_dim) or v.shape != k.shape or slot_mapping.numel() != n:
            raise ValueError("k, v must be [n][kv_dim] and slot_mapping [n]")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape:
            raise ValueError("out must match q")
        if scale is None:
            scale = 1.0 / math.sqrt(head_dim)  # model.rs:402
        _check(self._lib.ltkv_append_decode_attention(
            self._h, layer, n, n_heads, head_dim, float(scale),
            _dev_ptr(q, torch.float32, "q", self.device),
            _dev_ptr(tables, torch.int32, "tables", self.device), tables.shape[1],
            _dev_ptr(lens, torch.int32, "lens", self.device),
            _dev_ptr(slot_mapping, torch.int32, "slot_mapping", self.device),
            _dev_ptr(k, torch.float32, "k", self.device), _dev_ptr(v, torch.float32, "v", self.device),
            k.stride(0), _dev_ptr(out, torch.float32, "out", self.device)))
        return out

    def plan_attention(self, seqs: Sequence[int], lens: Sequence[int], n_heads: int, head_dim: int,
                       shared_prefix: bool = True, f16_products: bool = False) -> dict:
        """Step descriptor for planned_attention: query i reads positions
        [0, lens[i]) of sequence seqs[i]; with shared_prefix, queries forked
        from a common prefix attend to its shared blocks once, together (with
        f16_products, on products of f16-rounded Q and weights: faster, ~3e-4
        relative error instead of f32 accuracy). Returns the plan's figures."""
        seqs_a = np.ascontiguousarray(seqs, dtype=np.uint32)
        lens_a = np.ascontiguousarray(lens, dtype=np.uint32)
        if seqs_a.shape != lens_a.shape or seqs_a.ndim != 1:
            raise ValueError("seqs and lens must be 1-D of equal length")
        _check(self._lib.ltkv_plan_attention(self._h, len(seqs_a), _np_ptr(seqs_a), _np_ptr(lens_a),
                                             n_heads, head_dim,
                                             (1 if shared_prefix else 0) | (2 if f16_products else 0)))
        self._plan_shape = (len(seqs_a), n_heads * head_dim, head_dim)
        return self.plan_stats()

    def plan_stats(self) -> dict:
        out = np.zeros(6, dtype=np.uint64)
        _check(self._lib.ltkv_plan_stats(self._h, _np_ptr(out)))
        keys = ("queries", "groups", "grouped", "shared_blocks", "prefix_workgroups", "table_width")
        return {k: int(v) for k, v in zip(keys, out)}

    def planned_attention(self, layer: int, q, scale: Optional[float] = None, out=None):
        """Attention of the planned batch on one layer; q, out [n][n_heads*head_dim] f32."""
        import torch

        if self._plan_shape is None:
            raise KvError(_lib.ERR_ARG, "no attention plan (plan_attention)")
        n, width, head_dim = self._plan_shape
        if q.dim() != 2 or q.shape != (n, width):
            raise ValueError("q must be [n][n_heads*head_dim] of the plan")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape:
            raise ValueError("out must match q")
        if scale is None:
            scale = 1.0 / math.sqrt(head_dim)  # model.rs:402
        _check(self._lib.ltkv_planned_attention(
            self._h, layer, float(scale), _dev_ptr(q, torch.float32, "q", self.device),
            _dev_ptr(out, torch.float32, "out", self.device)))
        return out

    def set_attention_partition(self, tokens: int) -> None:
        _check(self._lib.ltkv_set_attention_partition(self._h, tokens))

    def set_attention_engine(self, engine: str) -> None:
        """'auto' (matrix cores for f16 and q8_0 pools) or 'valu' (f16 pools on
        the vector-ALU kernels, as f32 pools always are)."""
        codes = {"auto": _lib.ENGINE_AUTO, "valu": _lib.ENGINE_VALU}
        if engine not in codes:
            raise ValueError(f"engine must be one of {sorted(codes)}")
        _check(self._lib.ltkv_set_attention_engine(self._h, codes[engine]))

    def read_pool(self, layer: int = 0) -> tuple[np.ndarray, np.ndarray]:
        """Raw K and V pools of one layer, [n_blocks][16][kv_dim] on the host
        (f16 bits as uint16, float32, or q8_0 and q4_0 quants as int8)."""
        dt = {0.5: np.int8, 1: np.int8, 2: np.uint16, 4: np.float32}[self.elem]
        shape = (self.n_blocks, BLOCK, self.kv_dim)
        k = np.empty(shape, dtype=dt)
        v = np.empty(shape, dtype=dt)
        _check(self._lib.ltkv_read_pool(self._h, layer, _np_ptr(k), _np_ptr(v)))
        return k, v

    def read_scales(self, layer: int = 0) -> tuple[np.ndarray, np.ndarray]:
        """K and V scale pools of one layer of a q8_0 or q4_0 cache,
        [n_blocks][kv_dim/32][16] f16 bits (uint16) on the host: the scale of
        slot s, 32-element group g of block b is [b][g][s]."""
        shape = (self.n_blocks, self.kv_dim // 32, BLOCK)
        k = np.empty(shape, dtype=np.uint16)
        v = np.empty(shape, dtype=np.uint16)
        _check(self._lib.ltkv_read_scales(self._h, layer, _np_ptr(k), _np_ptr(v)))
        return k, v

    def synchronize(self) -> None:
        _check(self._lib.ltkv_synchronize(self._h))
