"""A paged cache of keys and values in 8 bits with the attention that reads it.

`QuantKVCache` holds what `KVCache` (model.py) holds for models -- keys and values of sequences with their lengths -- for callers
that drive their own layers: one byte a value with an fp32 scale per head and position, in pages of 64 positions.  A step
brings rows: `append` normalises, rotates and quantises them, `attention` answers their queries over everything committed
and the rows themselves (a chain, or a `tree` of drafted tokens), `commit` keeps the accepted ones and `read` gives values back.
Lengths live on the device; all of these are asynchronous on the context's stream and can be captured: with device arrays, `out` arrays, and
steps and trees that live as long as the graph (a call without `out`, or with host arrays, takes memory that a replay would not have).

bf16 rows are `np.uint16` arrays, the upper halves of float32 (a torch tensor's memory as it is); `to_bf16` / `from_bf16` convert on the host.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import numpy as np

from .device import Context, DeviceArray, as_device

SCHEMES = ("int8", "fp8")
PAGE = 64
MAX_DRAFT = 64            # rows of a tree, and rows that commit may pick from
_END = 1 << 31            # whole numbers go to the library in 32 bits
_DTYPES = {"f32": (0, np.dtype(np.float32)), "bf16": (1, np.dtype(np.uint16))}


def to_bf16(x) -> np.ndarray:
    """float32 -> bf16 bits, to nearest even (NaN stays NaN)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(x) -> np.ndarray:
    return (np.asarray(x, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def _ptr(a):
    return None if a is None else a.ptr


def _below_2_31(**numbers):
    for name, n in numbers.items():
        if not 0 <= n < _END:
            raise ValueError(f"{name} {n} outside 0 .. 2^31 - 1")


def _in_32_bits(ctx: Context, a, name: str) -> DeviceArray:
    """Whole numbers on the device; those of the host have to fit."""
    if not isinstance(a, DeviceArray):
        a = np.asarray(a.data if hasattr(a, "requires_grad") else a)
        if a.size and a.dtype != np.int32 and (a.min() < -_END or a.max() >= _END):
            raise ValueError(f"{name} holds a number that 32 bits do not")
    return as_device(ctx, a, np.int32)


class Step:
    """Rows of a ragged step on the device: entry e brings `counts[e]` rows for sequence `slots[e]`, one after another."""

    __slots__ = ("entries", "T", "rows", "counts", "_buf", "ents", "row_ent")

    def __init__(self, cache: "QuantKVCache", slots, counts):
        slots, counts = np.asarray(list(slots), np.int64).reshape(-1), np.asarray(list(counts), np.int64).reshape(-1)
        if slots.shape != counts.shape:
            raise ValueError(f"{slots.size} sequences with {counts.size} counts")
        if slots.size and (slots.min() < 0 or slots.max() >= cache.max_batch):
            raise IndexError(f"sequence outside the cache's {cache.max_batch}")
        if np.unique(slots).size != slots.size:
            raise ValueError("a sequence may come once in a step")
        if counts.size and (counts.min() < 0 or counts.max() > cache.max_seq):
            raise ValueError(f"counts outside 0 .. {cache.max_seq}")
        n, m = slots.size, int(counts.sum())
        if m >= 1 << 31:
            raise ValueError("a step has fewer than 2^31 rows")
        ents = np.zeros((n, 4), np.int32)
        ents[:, 0], ents[:, 2] = slots, counts
        if n:
            ents[1:, 1] = np.cumsum(counts)[:-1]
        self.entries, self.T, self.rows, self.counts = n, int(counts.max()) if n else 0, m, counts
        self._buf = cache.ctx.from_numpy(np.concatenate([ents.reshape(-1), np.repeat(np.arange(n, dtype=np.int32), counts), np.zeros(4, np.int32)]))
        self.ents, self.row_ent = self._buf.ptr, self._buf.ptr + 16 * n


class Tree:
    """What the rows of a tree see of one another, on the device."""

    __slots__ = ("T", "counts", "per_row", "_buf", "seen", "depth")

    def __init__(self, ctx: Context, seen: np.ndarray, depth: np.ndarray, T: int, counts: Optional[np.ndarray]):
        """counts: rows of every entry of the step that the tables go by; None: one tree for all entries."""
        self.T, self.counts, self.per_row = T, counts, int(counts is not None)
        self._buf = ctx.from_numpy(np.concatenate([seen.astype(np.uint64).view(np.uint8), depth.astype(np.int32).view(np.uint8), np.zeros(16, np.uint8)]))
        self.seen, self.depth = self._buf.ptr, self._buf.ptr + 8 * seen.size


def _tree_of(parents):
    """(seen, depth) of one list of parents: -1, or the place of an earlier row."""
    p = np.asarray(parents, np.int64).reshape(-1)
    if p.size > MAX_DRAFT:
        raise ValueError(f"a tree has at most {MAX_DRAFT} rows, not {p.size}")
    seen, depth = np.zeros(p.size, np.uint64), np.zeros(p.size, np.int32)
    for i, q in enumerate(p.tolist()):
        if q < -1 or q >= i:
            raise ValueError(f"row {i}: its parent {q} is not an earlier row or -1")
        seen[i] = (seen[q] if q >= 0 else np.uint64(0)) | np.uint64(1 << i)
        depth[i] = depth[q] + 1 if q >= 0 else 0
    return seen, depth


class QuantKVCache:
    """Keys and values of `max_batch` sequences of up to `max_seq` positions (rounded up to pages), `n_kv_head` heads of `head_dim`
    (a multiple of 8, at most 256) under `n_head` query heads.

    scheme "int8" or "fp8" (e4m3); dtype "bf16" or "f32": type of the rows and results.  pages = 0: every sequence owns its pages; else
    a pool of that many, handed out with `set_pages`."""

    def __init__(self, ctx: Context, max_batch: int, max_seq: int, n_head: int, n_kv_head: int, head_dim: int, scheme: str = "int8", dtype: str = "bf16", pages: int = 0):
        if scheme not in SCHEMES:
            raise ValueError(f"unknown scheme {scheme!r}, expected one of {SCHEMES}")
        if dtype not in _DTYPES:
            raise ValueError(f"unknown dtype {dtype!r}, expected one of {tuple(_DTYPES)}")
        self.handle = None
        _below_2_31(max_batch=max_batch, max_seq=max_seq, n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, pages=pages)
        self.ctx, self.scheme, self.dtype = ctx, scheme, dtype
        self.max_batch, self.n_head, self.n_kv_head, self.head_dim = int(max_batch), int(n_head), int(n_kv_head), int(head_dim)
        self._code, self._np = _DTYPES[dtype]
        self._lib, self._scale = ctx.lib, self.head_dim ** -0.5
        h = C.c_void_p()
        ctx._check(ctx.lib.vn_qkv_create(ctx.handle, self.max_batch, int(max_seq), self.n_head, self.n_kv_head, self.head_dim, scheme.encode(), self._code, int(pages),
                                         C.byref(h)))
        self.handle = h
        self.max_pages = -(-int(max_seq) // PAGE)
        self.max_seq = self.max_pages * PAGE
        self.pages = int(pages) or self.max_batch * self.max_pages

    def _here(self, a: DeviceArray) -> DeviceArray:
        if a.ctx is not self.ctx and a.ctx.device != self.ctx.device:
            raise ValueError(f"an array on device {a.ctx.device} for a cache on device {self.ctx.device}")
        return a

    # -- lengths and pages ---------------------------------------------------
    @property
    def per_seq_lens(self) -> np.ndarray:
        out = np.zeros(self.max_batch, np.int32)
        self.ctx._check(self.ctx.lib.vn_qkv_lengths(self.handle, out.ctypes.data_as(C.c_void_p)))
        return out

    def set_lengths(self, lens):
        """Committed positions of every sequence: a host array (checked), or a device array (copied in stream order)."""
        if isinstance(lens, DeviceArray):
            if lens.shape != (self.max_batch,) or lens.dtype != np.int32:
                raise ValueError(f"lens must be int32 of shape ({self.max_batch},)")
            self.ctx._check(self.ctx.lib.vn_qkv_set_lengths(self.handle, self._here(lens).ptr, 1))
            return
        lens = np.asarray(lens)
        if lens.shape != (self.max_batch,):
            raise ValueError(f"lens must have shape ({self.max_batch},)")
        if lens.size and (lens.min() < 0 or lens.max() > self.max_seq):
            raise RuntimeError(f"a length outside 0 .. {self.max_seq}")
        lens = np.ascontiguousarray(lens, np.int32)
        self.ctx._check(self.ctx.lib.vn_qkv_set_lengths(self.handle, lens.ctypes.data_as(C.c_void_p), 0))

    def reset(self):
        self.set_lengths(np.zeros(self.max_batch, np.int32))

    def set_pages(self, table):
        """table (max_batch, max_pages): the page of every 64 positions of a sequence, -1 for none."""
        t = np.asarray(table)
        if t.shape != (self.max_batch, self.max_pages):
            raise ValueError(f"the table must have shape ({self.max_batch}, {self.max_pages})")
        if t.size and (t.min() < -1 or t.max() >= self.pages):
            raise IndexError(f"a page outside the pool of {self.pages}")
        t = np.ascontiguousarray(t, np.int32)
        self.ctx._check(self.ctx.lib.vn_qkv_set_pages(self.handle, t.ctypes.data_as(C.c_void_p)))

    # -- steps -----------------------------------------------------------------
    def step(self, slots, counts) -> Step:
        return Step(self, slots, counts)

    def tree(self, parents, step: Optional[Step] = None) -> Tree:
        """What rows with these parents see: their ancestors and themselves.  `parents`: one list for every entry (row 0 is the last
        committed token's, -1: a child of nothing), or, with `step`, a list for each entry."""
        if step is not None and len(parents) and not np.isscalar(parents[0]):
            if len(parents) != step.entries or any(len(p) != n for p, n in zip(parents, step.counts)):
                raise ValueError("a list of parents for every entry, one parent a row, is needed")
            made = [_tree_of(p) for p in parents]
            return Tree(self.ctx, np.concatenate([m[0] for m in made]), np.concatenate([m[1] for m in made]), step.T, step.counts)
        seen, depth = _tree_of(parents)
        return Tree(self.ctx, seen, depth, seen.size, None)

    def _rows(self, shape, tail, step):
        """(entries, ents, row_ent, T, M) of rows of this shape, whose last axes are `tail`."""
        k = len(shape) - len(tail)
        lead = shape[:k]
        if shape[k:] != tail or k < 0:
            raise ValueError(f"rows of shape {tuple(shape)} do not end in {tuple(tail)}")
        if step is not None:
            if step._buf.ctx is not self.ctx:
                self._here(step._buf)
            m = math.prod(lead)
            if m < step.rows:
                raise ValueError(f"{m} rows for a step of {step.rows}")
            return step.entries, step.ents, step.row_ent, step.T, step.rows
        if k != 2 or lead[0] > self.max_batch or lead[0] * lead[1] >= _END:
            raise ValueError(f"rows of shape (sequences, rows, ..) with at most {self.max_batch} sequences and fewer than 2^31 rows, or a step, are needed")
        return lead[0], None, None, lead[1], lead[0] * lead[1]

    def _tree(self, tree, step, T, M):
        if tree is None:
            return None, None, 0
        if tree.per_row:
            if step is None or (tree.counts is not step.counts and not np.array_equal(tree.counts[tree.counts > 0], step.counts[step.counts > 0])):
                raise ValueError("this tree was made for another step")
        elif tree.T < T:
            raise ValueError(f"a tree of {tree.T} rows for entries of {T}")
        if T > MAX_DRAFT:
            raise ValueError(f"a tree has at most {MAX_DRAFT} rows, not {T}")
        if tree._buf.ctx is not self.ctx:
            self._here(tree._buf)
        return tree.seen, tree.depth, tree.per_row

    def _in(self, x):
        if isinstance(x, DeviceArray):
            if x.dtype != self._np:
                raise TypeError(f"device array has dtype {x.dtype}, need {self._np}")
            return x if x.ctx is self.ctx else self._here(x)
        x = np.asarray(x)
        if self.dtype == "bf16" and x.dtype != np.uint16:
            x = to_bf16(x)
        elif self.dtype == "f32" and x.dtype == np.uint16:
            raise TypeError("bf16 rows for a cache of float32 ones")
        return as_device(self.ctx, x, self._np)

    def _out(self, out, shape, dtype):
        if out is None:
            return self.ctx.empty(shape, dtype)
        if not isinstance(out, DeviceArray) or out.dtype != dtype or out.size < math.prod(shape):
            raise ValueError(f"out must be a device array of {np.dtype(dtype)} with room for {tuple(shape)}")
        return out if out.ctx is self.ctx else self._here(out)

    def _weight(self, a, name):
        a = self._here(as_device(self.ctx, a, np.float32))
        if a.shape != (self.head_dim,):
            raise ValueError(f"{name} must have shape ({self.head_dim},)")
        return a

    def append(self, rows, step: Optional[Step] = None, tree: Optional[Tree] = None, offset: int = 0, queries: bool = True, q_norm=None, k_norm=None, eps: float = 1e-6,
               rope=None, interleaved: bool = False, out: Optional[DeviceArray] = None) -> Optional[DeviceArray]:
        """Write a step's keys and values behind the committed positions (`offset` further on) and return its queries (rows, n_head, head_dim).

        rows: (sequences, rows of each, width), or (rows, width) with `step`; width = the query heads (unless `queries` is False), the key
        heads, the value heads, as one projection gives them.  q_norm / k_norm: weights (head_dim,) of an RMS norm of every
        query / key head; rope: (cos, sin) tables (positions, pairs) for rotating the first 2 * pairs dimensions of queries and keys
        (half-split, or neighbours when `interleaved`).  Lengths stay: `commit` moves them."""
        if not 0 <= offset < _END:
            _below_2_31(offset=offset)
        x = self._in(rows)
        H, d = self.n_head if queries else 0, self.head_dim
        width = (H + 2 * self.n_kv_head) * d
        E, ents, row_ent, T, M = self._rows(x.shape, (width,), step)
        _, depth, per_row = self._tree(tree, step, T, M)
        qn = self._weight(q_norm, "q_norm") if q_norm is not None else None
        kn = self._weight(k_norm, "k_norm") if k_norm is not None else None
        cs = sn = None
        pairs = rope_rows = 0
        if rope is not None:
            cs, sn = rope
            cs, sn = self._here(as_device(self.ctx, cs, np.float32)), self._here(as_device(self.ctx, sn, np.float32))
            if cs.ndim != 2 or cs.shape != sn.shape or 2 * cs.shape[1] > d:
                raise ValueError(f"rope: two tables (positions, pairs) with at most {d // 2} pairs are needed")
            rope_rows, pairs = cs.shape
            if pairs and rope_rows < self.max_seq:
                raise ValueError(f"rope: tables of {rope_rows} positions for a cache of {self.max_seq}")
        q = self._out(out, x.shape[:-1] + (H, d), self._np) if queries else None
        st = self._lib.vn_qkv_append(self.handle, x.ptr, width, queries, E, ents, row_ent, T, M, offset, depth, per_row, _ptr(qn), _ptr(kn), eps, _ptr(cs), _ptr(sn),
                                     rope_rows, pairs, interleaved, _ptr(q))
        if st:
            self.ctx._check(st)
        return q

    def attention(self, q, step: Optional[Step] = None, tree: Optional[Tree] = None, window: int = 0, scale: Optional[float] = None, out: Optional[DeviceArray] = None) -> DeviceArray:
        """softmax(scale q k^T) v of a step's queries (.., n_head, head_dim) over the committed positions and the step's own rows, which
        `append` has written: row i of an entry sees the rows up to itself, or its ancestors in `tree`.  window > 0: only the last
        `window` positions, of its path where there is a tree.  scale: 1 / sqrt(head_dim) unless given.  A row that sees nothing gets zeros."""
        if not 0 <= window < _END:
            _below_2_31(window=window)
        q = self._in(q)
        E, ents, row_ent, T, M = self._rows(q.shape, (self.n_head, self.head_dim), step)
        seen, depth, per_row = self._tree(tree, step, T, M)
        out = self._out(out, q.shape, self._np)
        st = self._lib.vn_qkv_attention(self.handle, q.ptr, E, ents, row_ent, T, M, seen, depth, per_row, window, self._scale if scale is None else scale, out.ptr)
        if st:
            self.ctx._check(st)
        return out

    def commit(self, n_new: int, n_keep, keep_idx=None, keep_add: int = 0):
        """Keep `n_keep[b] + keep_add` of the `n_new` positions appended to sequence b: the first ones (chain), or those listed in
        `keep_idx[b]` (tree path), as KVCache.commit."""
        if not (0 <= n_new < _END and -_END <= keep_add < _END):
            raise ValueError(f"n_new {n_new} outside 0 .. 2^31 - 1, or keep_add {keep_add} outside 32 bits")
        nk = self._here(_in_32_bits(self.ctx, n_keep, "n_keep"))
        if nk.size < self.max_batch:
            raise ValueError(f"n_keep must have {self.max_batch} values")
        ki, stride = None, 0
        if keep_idx is not None:
            ki = self._here(_in_32_bits(self.ctx, keep_idx, "keep_idx"))
            if ki.ndim != 2 or ki.shape[0] < self.max_batch or ki.shape[1] < n_new:
                raise ValueError(f"keep_idx must have shape ({self.max_batch}, {n_new})")
            stride = ki.shape[-1]
        st = self._lib.vn_qkv_commit(self.handle, n_new, _ptr(ki), stride, nk.ptr, keep_add)
        if st:
            self.ctx._check(st)

    def read(self, step, start: Optional[int] = None, offset: int = 0, back: bool = False, dtype: Optional[str] = None, out=None):
        """(k, v) values (rows, n_kv_head, head_dim) of a step's positions, as `dtype` (the cache's unless given): positions start .. of every
        entry; those behind its committed ones (`offset` further on) when `start` is None; its last committed ones with `back`.
        step: a Step, or (sequences, rows of each)."""
        if isinstance(step, Step):
            self._here(step._buf)
            E, ents, row_ent, T, M = step.entries, step.ents, step.row_ent, step.T, step.rows
            lead = (M,)
        else:
            E, T = (int(n) for n in step)
            if E < 0 or E > self.max_batch or T < 0 or max(T, E * T) >= _END:
                raise ValueError(f"at most {self.max_batch} sequences and fewer than 2^31 rows")
            ents, row_ent, M, lead = None, None, E * T, (E, T)
        if start is not None and (back or not 0 <= start < _END):
            raise ValueError("start is a position, and excludes `back`")
        if not 0 <= offset < _END:
            _below_2_31(offset=offset)
        if dtype is not None and dtype not in _DTYPES:
            raise ValueError(f"unknown dtype {dtype!r}, expected one of {tuple(_DTYPES)}")
        code, kind = _DTYPES[dtype or self.dtype]
        shape = lead + (self.n_kv_head, self.head_dim)
        k, v = out if out is not None else (None, None)
        k, v = self._out(k, shape, kind), self._out(v, shape, kind)
        st = self._lib.vn_qkv_read(self.handle, E, ents, row_ent, T, M, -2 if back else -1 if start is None else start, offset, code, k.ptr, v.ptr)
        if st:
            self.ctx._check(st)
        return k, v

    def get(self, seq_idx: int = 0, n_positions: Optional[int] = None):
        """(k, v) float32 ndarrays (n_positions, n_kv_head, head_dim) of one sequence, as KVCache.get."""
        if not 0 <= seq_idx < self.max_batch:
            raise IndexError(f"sequence {seq_idx} outside the cache's {self.max_batch}")
        n = int(self.per_seq_lens[seq_idx]) if n_positions is None else int(n_positions)
        k, v = self.read(self.step([seq_idx], [n]), start=0, dtype="f32")
        return k.numpy(), v.numpy()

    def check(self):
        """Raise what kernels have met since the last call: RuntimeError for a position without room, IndexError for an index out of range."""
        self.ctx._check(self.ctx.lib.vn_qkv_status(self.handle, None, None))

    def __del__(self):
        try:
            if self.handle:
                self.ctx.lib.vn_qkv_destroy(self.handle)
                self.handle = None
        except Exception:
            pass
