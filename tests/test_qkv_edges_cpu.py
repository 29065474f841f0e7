"""QuantKVCache without a GPU: numbers that the library's 32 bits do not hold, and arrays that it cannot read, are refused before a call."""

import numpy as np
import pytest

from test_qkv_cpu import cache


@pytest.mark.parametrize("name,call", [
    ("vn_qkv_append", lambda c, n: c.append(np.zeros((2, 3, 128), np.float32), offset=n)),
    ("vn_qkv_attention", lambda c, n: c.attention(np.zeros((2, 3, 4, 16), np.float32), window=n)),
    ("vn_qkv_read", lambda c, n: c.read((1, 2), start=n)),
    ("vn_qkv_read", lambda c, n: c.read((1, 2), offset=n)),
    ("vn_qkv_read", lambda c, n: c.read(c.step([1], [2]), offset=n)),
    ("vn_qkv_commit", lambda c, n: c.commit(n, [1, 2, 3])),
    ("vn_qkv_commit", lambda c, n: c.commit(3, [1, 2, 3], keep_add=n)),
    ("vn_qkv_commit", lambda c, n: c.commit(3, [1, n, 3])),
    ("vn_qkv_commit", lambda c, n: c.commit(3, np.array([n, 2, 3]))),
    ("vn_qkv_commit", lambda c, n: c.commit(3, [1, 2, 3], [[0, 1, 2], [0, 1, n], [0, 1, 2]])),
])
def test_numbers_of_more_than_32_bits(name, call):
    c = cache(dtype="f32")
    call(c, 2)
    assert c.ctx.lib.calls[-1][0] == name
    n = len(c.ctx.lib.calls)
    for bad in (1 << 31, 1 << 32, (1 << 32) + 5, (1 << 62) + 1, -(1 << 31) - 1, -(1 << 32)):
        with pytest.raises(ValueError):
            call(c, bad)
    assert len(c.ctx.lib.calls) == n


@pytest.mark.parametrize("which", ["max_batch", "max_seq", "n_head", "n_kv_head", "head_dim", "pages"])
@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 8, 8 - (1 << 32), -1])
def test_sizes_of_more_than_32_bits(which, n):
    with pytest.raises(ValueError):
        cache(**{which: n})


def test_rows_of_more_than_32_bits():
    c = cache(dtype="f32")
    n = len(c.ctx.lib.calls)
    for step in ((1, 1 << 31), (0, 1 << 32), (3, 1 << 30)):
        with pytest.raises(ValueError):
            c.read(step, out=(None, None))
    assert len(c.ctx.lib.calls) == n


def test_bf16_rows_are_not_taken_for_whole_numbers():
    c = cache(dtype="f32")
    n = len(c.ctx.lib.calls)
    with pytest.raises(TypeError):
        c.append(np.zeros((2, 3, 128), np.uint16))
    with pytest.raises(TypeError):
        c.attention(np.zeros((2, 3, 4, 16), np.uint16))
    assert len(c.ctx.lib.calls) == n
    c.append(np.zeros((2, 3, 128), np.int32))
    c.attention(np.zeros((2, 3, 4, 16), np.float64))


def test_a_tree_of_another_step():
    """The tables go by the rows of the step: one with as many rows, but others for an entry, is another step."""
    c = cache(dtype="f32")
    a, b = c.step([0, 1], [1, 2]), c.step([0, 1], [2, 1])
    t = c.tree([[-1], [-1, -1]], a)
    x, q = np.zeros((3, 128), np.float32), np.zeros((3, 4, 16), np.float32)
    n = len(c.ctx.lib.calls)
    for step in (b, c.step([0], [3]), c.step([0, 1, 2], [1, 1, 1]), None):
        with pytest.raises(ValueError):
            c.append(x if step else x[None], step=step, tree=t)
        with pytest.raises(ValueError):
            c.attention(q if step else q[None], step=step, tree=t)
    assert len(c.ctx.lib.calls) == n
    for step in (a, c.step([2, 0], [1, 2]), c.step([2, 1, 0], [1, 0, 2])):     # other sequences, the same rows
        c.append(x, step=step, tree=t)
        c.attention(q, step=step, tree=t)


def test_arrays_of_another_device():
    """A kernel of this device cannot read them."""
    c, other = cache(dtype="f32"), cache(dtype="f32")
    other.ctx.device = 1
    there = other.ctx.from_numpy
    x, q, w = np.zeros((2, 3, 128), np.float32), np.zeros((2, 3, 4, 16), np.float32), np.ones(16, np.float32)
    table = np.zeros((128, 8), np.float32)
    i3 = np.zeros(3, np.int32)
    step, far = c.step([0], [3]), other.step([0], [3])
    calls = [
        lambda f: c.append(f(x)), lambda f: c.append(x, out=f(q)), lambda f: c.append(x, q_norm=f(w)), lambda f: c.append(x, k_norm=f(w)),
        lambda f: c.append(x, rope=(f(table), table)), lambda f: c.append(x, rope=(table, f(table))),
        lambda f: c.append(x[0], step=far if f == there else step), lambda f: c.append(x, tree=(other if f == there else c).tree([-1, 0, 0])),
        lambda f: c.attention(f(q)), lambda f: c.attention(q, out=f(q)), lambda f: c.attention(q[0], step=far if f == there else step),
        lambda f: c.read((2, 3), out=(f(np.zeros((2, 3, 2, 16), np.float32)), None)), lambda f: c.read((2, 3), out=(None, f(np.zeros((2, 3, 2, 16), np.float32)))),
        lambda f: c.read(far if f == there else step), lambda f: c.commit(3, f(i3)), lambda f: c.commit(3, i3, f(np.zeros((3, 3), np.int32))), lambda f: c.set_lengths(f(i3)),
    ]
    for call in calls:
        n = len(c.ctx.lib.calls)
        with pytest.raises(ValueError):
            call(there)
        assert len(c.ctx.lib.calls) == n
        call(c.ctx.from_numpy)
        assert len(c.ctx.lib.calls) == n + 1


def test_the_probe_refuses_null():
    import ctypes as C
    from versenext_b200 import _lib
    assert _lib.load().vn_qkv_probe_wait(None, 1, C.byref(C.c_int64())) == _lib.VN_ERR_INVALID
