"""QuantKVCache without a GPU: trees, steps, bf16 on the host, and every refusal that the Python layer and the C entry points make."""

import ctypes as C

import numpy as np
import pytest

from versenext_b200 import _lib
from versenext_b200 import quant_cache as Q
from versenext_b200.device import DeviceArray


class FakeLib:
    """Records calls; every entry point succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


class FakeCtx:
    def __init__(self):
        self.lib, self.handle, self.device, self.held = FakeLib(), None, 0, []

    def _check(self, status):
        assert status == 0

    def from_numpy(self, a):
        a = np.ascontiguousarray(a)
        self.held.append(a)
        return DeviceArray(self, a.ctypes.data, a.shape, a.dtype)

    def empty(self, shape, dtype):
        return self.from_numpy(np.zeros(shape, dtype))


def cache(**kw):
    a = dict(max_batch=3, max_seq=100, n_head=4, n_kv_head=2, head_dim=16)
    a.update(kw)
    return Q.QuantKVCache(FakeCtx(), **a)


def host(ptr, shape, dtype):
    n = int(np.prod(shape))
    return np.frombuffer((C.c_byte * (n * np.dtype(dtype).itemsize)).from_address(ptr), dtype).reshape(shape).copy()


def test_bf16_on_the_host_rounds_to_nearest_even():
    import torch
    x = np.concatenate([np.random.default_rng(0).normal(0, 1, 5000).astype(np.float32) * np.float32(10) ** np.random.default_rng(1).integers(-30, 30, 5000),
                        np.array([0.0, -0.0, np.inf, -np.inf, 1.00390625, 1.01171875, 3.4e38, 1e-40], np.float32)]).astype(np.float32)
    want = torch.from_numpy(x).bfloat16().float().numpy()
    np.testing.assert_array_equal(Q.from_bf16(Q.to_bf16(x)), want)
    assert np.isnan(Q.from_bf16(Q.to_bf16(np.array([np.nan, np.uint32(0x7F800001).view(np.float32)], np.float32)))).all()


def test_tree_tables():
    seen, depth = Q._tree_of([-1, 0, 0, 1, 3, -1])
    assert depth.tolist() == [0, 1, 1, 2, 3, 0]
    assert [bin(int(s)) for s in seen] == ["0b1", "0b11", "0b101", "0b1011", "0b11011", "0b100000"]
    seen, depth = Q._tree_of(list(range(-1, 63)))
    assert int(seen[63]) == (1 << 64) - 1 and depth[63] == 63
    for bad in ([0], [-2], [-1, 1], [-1, 5], list(range(-1, 64))):
        with pytest.raises(ValueError):
            Q._tree_of(bad)
    c = cache()
    t = c.tree([-1, 0, 1])
    assert host(t.seen, 3, np.uint64).tolist() == [1, 3, 7] and host(t.depth, 3, np.int32).tolist() == [0, 1, 2] and not t.per_row
    s = c.step([2, 0], [2, 3])
    t = c.tree([[-1, -1], [-1, 0, 0]], s)
    assert host(t.seen, 5, np.uint64).tolist() == [1, 2, 1, 3, 5] and host(t.depth, 5, np.int32).tolist() == [0, 0, 0, 1, 1] and t.per_row
    with pytest.raises(ValueError):
        c.tree([[-1, -1]], s)
    with pytest.raises(ValueError):
        c.tree([[-1], [-1, 0, 0]], s)


def test_step_tables_and_refusals():
    c = cache()
    s = c.step([2, 0, 1], [3, 0, 2])
    assert (s.entries, s.T, s.rows) == (3, 3, 5)
    assert host(s.ents, (3, 4), np.int32).tolist() == [[2, 0, 3, 0], [0, 3, 0, 0], [1, 3, 2, 0]]
    assert host(s.row_ent, 5, np.int32).tolist() == [0, 0, 0, 2, 2]
    assert s.ents % 16 == 0
    e = c.step([], [])
    assert (e.entries, e.T, e.rows) == (0, 0, 0)
    for slots, counts, kind in (([0], [1, 2], ValueError), ([3], [1], IndexError), ([-1], [1], IndexError), ([0, 0], [1, 1], ValueError), ([0], [-1], ValueError),
                                ([0], [129], ValueError)):
        with pytest.raises(kind):
            c.step(slots, counts)


def test_construction_refusals():
    for kw in (dict(scheme="int3"), dict(dtype="f16")):
        with pytest.raises(ValueError):
            cache(**kw)
    c = cache()
    assert c.max_seq == 128 and c.pages == 6
    assert cache(pages=5).pages == 5


def test_lengths_and_pages_refusals():
    c = cache()
    with pytest.raises(ValueError):
        c.set_lengths([1, 2])
    for bad in ([-1, 0, 0], [0, 129, 0], [0, 1 << 40, 0]):
        with pytest.raises(RuntimeError):
            c.set_lengths(bad)
    with pytest.raises(ValueError):
        c.set_lengths(c.ctx.from_numpy(np.zeros(3, np.int64)))
    with pytest.raises(ValueError):
        c.set_pages(np.zeros((3, 3), int))
    for bad in (-2, 6, 1 << 33):
        with pytest.raises(IndexError):
            c.set_pages(np.full((3, 2), bad))
    c.set_pages(np.full((3, 2), -1))
    assert c.ctx.lib.calls[-1][0] == "vn_qkv_set_pages"


def test_row_refusals():
    c = cache(dtype="f32")
    x = np.zeros((2, 3, 128), np.float32)
    n = len(c.ctx.lib.calls)
    for bad in (np.zeros((2, 3, 127), np.float32), np.zeros((4, 3, 128), np.float32), np.zeros((6, 128), np.float32)):
        with pytest.raises(ValueError):
            c.append(bad)
    with pytest.raises(ValueError):
        c.append(x, queries=False)
    with pytest.raises(ValueError):
        c.append(x[0], step=c.step([0], [4]))
    with pytest.raises(TypeError):
        c.append(c.ctx.from_numpy(np.zeros((2, 3, 128), np.uint16)))
    with pytest.raises(ValueError):
        c.append(x, q_norm=np.ones(15, np.float32))
    table = np.zeros((128, 8), np.float32)
    for rope in ((table[:127], table[:127]), (table, table[:, :7]), (np.zeros((128, 9), np.float32),) * 2, (table[0], table[0])):
        with pytest.raises(ValueError):
            c.append(x, rope=rope)
    with pytest.raises(ValueError):
        c.append(x, tree=c.tree([-1, 0]))
    with pytest.raises(ValueError):
        c.append(x, out=c.ctx.from_numpy(np.zeros((2, 3, 4, 15), np.float32)))
    q = np.zeros((2, 3, 4, 16), np.float32)
    with pytest.raises(ValueError):
        c.attention(q[..., :15])
    with pytest.raises(ValueError):
        c.attention(q, tree=c.tree([[-1, 0, 1]], c.step([0], [3])))
    with pytest.raises(ValueError):
        c.attention(np.zeros((1, 65, 4, 16), np.float32), tree=c.tree(range(-1, 63)))
    with pytest.raises(ValueError):
        c.attention(q, out=np.zeros_like(q))
    for kw in (dict(step=(4, 1)), dict(step=(1, -1)), dict(step=(1, 1), start=-1), dict(step=(1, 1), start=0, back=True), dict(step=(1, 1), dtype="f64")):
        with pytest.raises(ValueError):
            c.read(**kw)
    with pytest.raises(ValueError):
        c.commit(3, [1, 2])
    with pytest.raises(ValueError):
        c.commit(3, [1, 2, 3], np.zeros((3, 2), np.int32))
    with pytest.raises(IndexError):
        c.get(3)
    assert all(name not in ("vn_qkv_append", "vn_qkv_attention", "vn_qkv_read", "vn_qkv_commit") for name, _ in c.ctx.lib.calls[n:])
    c.append(x, rope=(table, table))
    assert c.ctx.lib.calls[-1][0] == "vn_qkv_append"


def test_c_entry_points_refuse_null():
    lib = _lib.load()
    out = C.c_void_p()
    assert lib.vn_qkv_create(None, 1, 1, 1, 1, 16, b"int8", 0, 0, C.byref(out)) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_destroy(None) == _lib.VN_OK
    assert lib.vn_qkv_set_pages(None, None) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_lengths(None, None) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_set_lengths(None, None, 0) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_status(None, None, None) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_append(None, None, 0, 0, 0, None, None, 0, 0, 0, None, 0, None, None, 0.0, None, None, 0, 0, 0, None) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_attention(None, None, 0, None, None, 0, 0, None, None, 0, 0, 1.0, None) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_read(None, 0, None, None, 0, 0, 0, 0, 0, None, None) == _lib.VN_ERR_INVALID
    assert lib.vn_qkv_commit(None, 0, None, 0, None, 0) == _lib.VN_ERR_INVALID
