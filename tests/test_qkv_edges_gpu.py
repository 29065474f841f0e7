"""QuantKVCache on the device where it is easiest to get wrong: scores that differ much between the parts of a sequence, values that differ
much in size, rows that are not finite, tables out of range, very long sequences, trees of their own for every entry, offsets, narrow windows,
graphs in turn, and a loop whose rounds are the plain cache's."""

import numpy as np
import pytest

import qkv_cases as R
from test_qkv_gpu import back, check_attention, fill, new, stored, tables

pytestmark = pytest.mark.gpu


def write(c, k, v):
    """Positions 0 .. of sequence 0; k, v (n, KH, d)."""
    n = len(k)
    c.append(np.concatenate([k.reshape(n, -1), v.reshape(n, -1)], 1), step=c.step([0], [n]), queries=False)


def check_one(c, q, k, v, n_com, dtype, parents=None, window=0):
    """Attention of sequence 0 over `n_com` committed positions and the rows q brings, against 64 bits."""
    n, d = len(q), c.head_dim
    write(c, k, v)
    c.set_lengths([n_com] + [0] * (c.max_batch - 1))
    tree = c.tree(parents) if parents is not None else None
    got = back(c.attention(q[None], tree=tree, window=window))[0]
    c.check()
    depth, seen = R.depth_and_seen(parents, n)
    out, weight, reach = R.attention(q, R.in_8_bits(k, c.scheme), R.in_8_bits(v, c.scheme), n_com, depth, seen, window, d ** -0.5)
    tol = R.tolerance(out, weight, reach, d, n_com + n, dtype, c.scheme == "int8")
    assert np.isfinite(got).all()
    assert (np.abs(got - out) <= tol).all(), float(np.max(np.abs(got - out) / tol))


# ---- parts of a sequence whose scores lie far apart ---------------------------------------------------------------------
@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,H,KH,d,T", [("f32", 1, 1, 256, 1), ("bf16", 2, 1, 256, 1), ("bf16", 4, 2, 192, 2), ("f32", 3, 1, 248, 1), ("bf16", 5, 1, 136, 4), ("f32", 2, 1, 192, 24),
                                            ("bf16", 8, 2, 128, 1), ("f32", 2, 1, 64, 1), ("bf16", 2, 1, 64, 20), ("bf16", 6, 1, 128, 5), ("bf16", 4, 1, 96, 9)])
@pytest.mark.parametrize("n,hot", [(620, [(619, 110)]), (700, [(650, 380)]), (1000, [(990, 150)]), (1000, [(560, 120), (999, 260)]), (1000, [(3, 200)]), (1400, [(1390, 300)]),
                                   (2600, [(1300, 130), (2590, 270)]), (1000, [(700, 60)])])
def test_a_score_far_above_those_of_the_other_parts(scheme, dtype, H, KH, d, T, n, hot):
    """A sequence of n positions is cut into parts of at least four blocks of 32 (two pages of 64 for many rows): 5 to 21 of them here.
    One or two positions have a score of `hot` above the others', which are small."""
    rng = np.random.default_rng(n + d)
    c = new(1, n + T, H, KH, d, scheme=scheme, dtype=dtype)
    along = rng.normal(0, 1, (KH, d))
    along /= np.linalg.norm(along, axis=-1, keepdims=True)
    q = stored(np.repeat(along, H // KH, 0)[None] * 4 + rng.normal(0, 0.1, (T, H, d)), dtype)
    k = rng.normal(0, 0.3, (n + T, KH, d))
    for at, gap in hot:
        k[at] = along * gap * d ** 0.5 / 4
    check_one(c, q, stored(k, dtype), stored(rng.normal(0, 1, (n + T, KH, d)), dtype), n, dtype)


# ---- rows that are not finite -----------------------------------------------------------------------------------------
def shown(c, seen, depth):
    """A tree of rows that see what `seen` says, on the device."""
    from versenext_b200.quant_cache import Tree
    return Tree(c.ctx, np.asarray(seen, np.uint64), np.asarray(depth, np.int32), len(seen), None)


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,H,d,T", [("f32", 1, 64, 4), ("bf16", 1, 64, 4), ("bf16", 2, 64, 12), ("bf16", 4, 128, 40), ("bf16", 1, 256, 4), ("bf16", 4, 96, 30), ("f32", 2, 192, 20)])
@pytest.mark.parametrize("bad", [-np.inf, np.inf, np.nan])
def test_a_query_that_is_not_finite(scheme, dtype, H, d, T, bad):
    """Every score of the row is then infinite or no number, of one sign too where all keys have the same sign in that channel: no soft-max
    exists, and the row is NaN.  A row that sees nothing is zero whatever its query."""
    rng = np.random.default_rng(d + T)
    n = 200
    c = new(1, n + T, H, 1, d, scheme=scheme, dtype=dtype)
    k = rng.normal(0, 1, (n + T, 1, d))
    k[..., 3] = rng.uniform(1, 2, (n + T, 1))
    write(c, stored(k, dtype), stored(rng.normal(0, 1, (n + T, 1, d)), dtype))
    c.set_lengths([n])
    q = stored(rng.normal(0, 1, (1, T, H, d)), dtype)
    good = back(c.attention(q))
    q[0, 1, 0, 3] = bad
    got = back(c.attention(q))
    assert np.isnan(got[0, 1, 0]).all()
    good[0, 1, 0] = got[0, 1, 0]
    np.testing.assert_array_equal(got, good)
    c.set_lengths([0])
    out = back(c.attention(q, tree=shown(c, [0] * T, [0] * T)))
    assert (out == 0).all()
    c.check()


# ---- device tables out of range -----------------------------------------------------------------------------------------
def test_device_lengths_out_of_range_are_reported():
    c = new(3, 100, 2, 1, 16, dtype="f32")
    for bad, want in (([-1, 5, 128], [0, 5, 128]), ([3, 1 << 30, 129], [3, 128, 128]), ([-(1 << 31), 0, (1 << 31) - 1], [0, 0, 128])):
        c.set_lengths(c.ctx.from_numpy(np.array(bad, np.int32)))
        with pytest.raises(IndexError):
            c.check()
        assert c.per_seq_lens.tolist() == want
    c.set_lengths(c.ctx.from_numpy(np.array([0, 128, 7], np.int32)))
    c.check()
    assert c.per_seq_lens.tolist() == [0, 128, 7]
    assert c.get(1)[0].shape == (128, 1, 16)


def test_positions_that_pass_32_bits_have_no_room():
    far = (1 << 31) - 1
    c = new(2, 128, 2, 1, 16, dtype="f32")
    ones = np.ones((2, 3, 64), np.float32)
    c.append(ones)
    c.set_lengths([3, 100])
    for start in (dict(start=far), dict(start=far - 1), dict(offset=far), dict(offset=far - 2), dict(offset=far, back=True)):
        for step in ((2, 3), c.step([1, 0], [2, 3])):
            k, v = c.read(step, dtype="f32", **start)
            with pytest.raises(RuntimeError):
                c.check()
            assert (k.numpy() == 0).all() and (v.numpy() == 0).all()
    before = [c.get(b, 128) for b in range(2)]
    for offset in (far, far - 1, far - 102):
        q = c.append(2 * ones, offset=offset, rope=tables(128, 8))
        assert np.isfinite(q.numpy()).all()
        with pytest.raises(RuntimeError):
            c.check()
    for b in range(2):
        for x, y in zip(before[b], c.get(b, 128)):
            np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("dtype,H,d", [("f32", 2, 64), ("bf16", 2, 64), ("bf16", 16, 64), ("bf16", 16, 128), ("bf16", 16, 96)])
@pytest.mark.parametrize("wrong,counts_as", [([100, -10, 3], [63, 0, 3]), ([0, 1 << 30, -(1 << 31)], [0, 63, 0]), ([64, 2, (1 << 31) - 1], [63, 2, 63])])
def test_depths_out_of_range_are_reported(dtype, H, d, wrong, counts_as):
    """A row of a tree is 0 to 63 tokens behind the committed ones; what is outside counts as the nearest of them."""
    rng = np.random.default_rng(d)
    c = new(2, 500, H, 1, d, dtype=dtype)
    fill(c, rng, [400, 90], dtype)
    c.append(stored(rng.normal(0, 1, (2, 3, 2 * d)), dtype), queries=False)
    q = stored(rng.normal(0, 1, (2, 3, H, d)), dtype)
    seen = [1, 3, 5]
    for window in (1, 40, 200):
        want = back(c.attention(q, tree=shown(c, seen, counts_as), window=window))
        c.check()
        got = back(c.attention(q, tree=shown(c, seen, wrong), window=window))
        with pytest.raises(IndexError):
            c.check()
        np.testing.assert_array_equal(got, want)


def test_positions_outside_the_rotation_tables_are_reported():
    rng = np.random.default_rng(1)
    c = new(1, 64, 1, 1, 16, dtype="f32")
    rope = tables(64, 8)
    x = rng.normal(0, 1, (1, 2, 48)).astype(np.float32)
    c.set_lengths([10])
    c.append(x, tree=shown(c, [1, 3], [-10, 53]), rope=rope)     # positions 0 and 63
    c.check()
    for depth in ([0, 54], [-11, 0], [0, (1 << 31) - 1], [-(1 << 31), 0]):
        c.append(x, tree=shown(c, [1, 3], depth), rope=rope)
        with pytest.raises(IndexError):
            c.check()
        c.append(x, tree=shown(c, [1, 3], depth))
        c.check()                                                 # without rotation there is no such position


def test_a_step_whose_rows_belong_to_nobody():
    """No entries, and rows that name none: everything is left as it was."""
    from versenext_b200._lib import VN_OK
    for dtype, d in (("f32", 16), ("bf16", 64)):
        c = new(2, 64, 2, 1, d, dtype=dtype)
        ctx, lib = c.ctx, c.ctx.lib
        nobody = ctx.from_numpy(np.full(4, -1, np.int32))
        x = ctx.from_numpy(np.full((4, 4 * d), 1, c._np))
        out = ctx.from_numpy(np.full((4, 2, d), 9, c._np))
        for T in (1, 40):
            assert lib.vn_qkv_append(c.handle, x.ptr, 4 * d, 1, 0, nobody.ptr, nobody.ptr, T, 4, 0, None, 0, None, None, 1e-6, None, None, 0, 0, 0, out.ptr) == VN_OK
            assert lib.vn_qkv_attention(c.handle, x.ptr, 0, nobody.ptr, nobody.ptr, T, 4, None, None, 0, 0, 1.0, out.ptr) == VN_OK
            assert lib.vn_qkv_read(c.handle, 0, nobody.ptr, nobody.ptr, T, 4, 0, 0, c._code, out.ptr, out.ptr) == VN_OK
        c.check()
        assert (out.numpy() == 9).all()


# ---- errors -------------------------------------------------------------------------------------------------------------
def test_a_failed_allocation_is_told_once():
    """The call that fails says so; the next one is good."""
    c = new(1, 64, 2, 1, 16, dtype="f32")
    x = c.ctx.from_numpy(np.ones((1, 3, 64), np.float32))
    want = c.attention(c.append(x)).numpy()                       # (127 times 1 / 127 in 32 bits is not quite 1)
    for _ in range(2):
        with pytest.raises(MemoryError):
            c.ctx.alloc(1 << 50)
        np.testing.assert_array_equal(c.attention(c.append(x)).numpy(), want)
    c.check()


# ---- sequences that may be very long ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,H,KH,d,T", [("bf16", 8, 8, 16, 1), ("f32", 4, 2, 16, 30), ("bf16", 8, 2, 64, 40)])
def test_room_for_2_30_positions(dtype, H, KH, d, T):
    """A pool of a few pages under a table for 2^30 positions."""
    rng = np.random.default_rng(T)
    c = new(1, 1 << 30, H, KH, d, dtype=dtype, pages=6)
    table = np.full((1, c.max_pages), -1, np.int32)
    table[0, :6] = [5, 0, 3, 1, 4, 2]
    c.set_pages(table)
    check_attention(c, rng, [300], [T], dtype)


def test_more_blocks_than_32_bits_count():
    """65 heads of 2^30 - 64 positions whose pages are one page: 2.18 10^9 blocks.  Every key is zero, so the result is the
    mean of the values, which are the head's own: sums of equal terms that 24 bits hold."""
    KH, d = 65, 16
    c = new(1, 1 << 30, KH, KH, d, pages=2)
    table = np.zeros((1, c.max_pages), np.int32)
    table[0, -1] = 1
    c.set_pages(table)
    sign = np.where(np.arange(KH) % 3 == 0, -1.0, 1.0) * 2.0 ** (np.arange(KH) % 7)
    v = np.full((64, KH, d), 64.0) * sign[None, :, None]
    v[..., 0] = 127.0 * sign                                      # the scale: the others have the code 64
    write(c, np.zeros((64, KH, d), np.float32), v)
    c.set_lengths([(1 << 30) - 64])
    c.append(np.concatenate([np.zeros((1, KH, d)), v[:1]], 1).reshape(1, 1, -1), queries=False)
    out = back(c.attention(np.ones((1, 1, KH, d), np.float32)))[0, 0]
    c.check()
    # sums of weights and values are exact in a part (a few 10^6 equal terms, in 32 at a time); parts join with 2^-24 for each of
    # some 30, and the result is rounded to bf16
    np.testing.assert_allclose(out[:, 1:], v[0, :, 1:], rtol=2.0 ** -8)


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,H,d,T", [("bf16", 2, 64, 1), ("f32", 2, 64, 1), ("bf16", 4, 128, 16), ("bf16", 2, 256, 3), ("f32", 2, 80, 20)])
@pytest.mark.parametrize("order", [1, -1, 0])
def test_values_that_differ_much_in_size(scheme, dtype, H, d, T, order):
    """Heads of values from 10^-15 to 10^15, smallest first, largest first, or mixed."""
    rng = np.random.default_rng(d + order)
    n = 900
    size = np.linspace(-15, 15, n + T)[::order or 1]
    size = 10.0 ** (rng.permutation(size) if order == 0 else size)
    c = new(1, n + T, H, 1, d, scheme=scheme, dtype=dtype)
    q, k = stored(rng.normal(0, 1, (T, H, d)), dtype), stored(rng.normal(0, 1, (n + T, 1, d)), dtype)
    check_one(c, q, k, stored(rng.normal(0, 1, (n + T, 1, d)) * size[:, None, None], dtype), n, dtype)


# ---- trees, windows, offsets ------------------------------------------------------------------------------------------
def grown(rng, n):
    return [int(rng.integers(-1, i)) if i else -1 for i in range(n)]


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,H,KH,d,most", [("bf16", 4, 4, 64, 15), ("bf16", 8, 2, 128, 40), ("f32", 2, 1, 64, 30), ("bf16", 4, 2, 96, 64)])
@pytest.mark.parametrize("window", [0, 2, 50])
def test_a_tree_for_every_entry(scheme, dtype, H, KH, d, most, window):
    rng = np.random.default_rng(d + window)
    B, lens, counts = 5, [200, 0, 31, 500, 64], [most, 1, 0, most // 2, 7]
    slots = [3, 0, 4, 1, 2]
    c = new(B, 600, H, KH, d, scheme=scheme, dtype=dtype)
    lens = np.asarray(lens)
    old = fill(c, rng, lens.tolist(), dtype)
    trees = [grown(rng, n) for n in counts]
    trees[0] = [i - 1 for i in range(most)]                # a path
    M = sum(counts)
    cs, sn = tables(c.max_seq, d // 2)
    x = stored(rng.normal(0, 1, (M + 3, (H + 2 * KH) * d)), dtype)
    step = c.step(slots, counts)
    tree = c.tree(trees, step)
    out = c.ctx.from_numpy(np.full((M + 3, H, d), 7, c._np))
    q = c.append(x, step=step, tree=tree, rope=(cs, sn))
    got = back(c.attention(q, step=step, tree=tree, window=window, out=out))
    assert (out.numpy()[M:] == 7).all()
    q = back(q)
    k, v = (a.numpy() for a in c.read(step, dtype="f32"))
    c.check()
    at = 0
    for b, n, parents in zip(slots, counts, trees):
        if n:
            depth, seen = R.depth_and_seen(parents, n)
            h = x[at:at + n].reshape(n, H + 2 * KH, d)
            both = R.heads_in(h[:, :H + KH], None, 0, lens[b] + depth, cs, sn, False)
            # two products and a sum in 32 bits, relative to the larger of a pair's channels; half a step of the type, half a code
            size = np.abs(both).max(-1, keepdims=True)
            off = 2.0 ** -24 * 4 * 2 * size
            assert (np.abs(q[at:at + n] - both[:, :H]) <= off[:, :H] + (2.0 ** -8 if dtype == "bf16" else 0) * np.abs(both[:, :H]) * 1.001).all()
            code = size[:, H:] / 127 / 2 if scheme == "int8" else np.maximum(np.abs(both[:, H:]) * 2.0 ** -4, size[:, H:] / 448 * 2.0 ** -10)
            assert (np.abs(k[at:at + n] - both[:, H:]) <= code * 1.001 + 2 * off[:, H:]).all()
            np.testing.assert_array_equal(v[at:at + n], R.in_8_bits(h[:, H + KH:], scheme))
            kk, vv = np.concatenate([old[b][0], k[at:at + n]]), np.concatenate([old[b][1], v[at:at + n]])
            want, weight, reach = R.attention(q[at:at + n], kk, vv, lens[b], depth, seen, window, d ** -0.5)
            tol = R.tolerance(want, weight, reach, d, lens[b] + n, dtype, scheme == "int8")
            assert (np.abs(got[at:at + n] - want) <= tol).all(), (b, float(np.max(np.abs(got[at:at + n] - want) / tol)))
        at += n


@pytest.mark.parametrize("dtype,H,d", [("bf16", 1, 64), ("bf16", 1, 256), ("f32", 2, 64), ("f32", 1, 16)])
@pytest.mark.parametrize("window", [1, 2, 3, 5, 17])
def test_windows_narrower_than_a_path_with_few_rows(dtype, H, d, window):
    rng = np.random.default_rng(window + d)
    c = new(3, 300, H, 1, d, dtype=dtype)
    check_attention(c, rng, [250, 0, 64], [8] * 3, dtype, parents=[-1, 0, 1, 2, 3, 1, 5, 6], window=window)
    check_attention(c, rng, [250, 0, 64], [8] * 3, dtype, window=window)


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_offsets(scheme, dtype):
    """A step brought in three portions, each `offset` further on, is the step brought at once; `read` finds each portion."""
    rng = np.random.default_rng(18)
    B, H, KH, d, n = 3, 4, 2, 64, 70
    lens = [0, 61, 130]
    cs, sn = tables(256, 32)
    w = rng.normal(1, 0.3, d).astype(np.float32)
    x = stored(rng.normal(0, 1, (B, n, (H + 2 * KH) * d)), dtype)
    kw = dict(q_norm=w, k_norm=w, rope=(cs, sn))
    a, b = (new(B, 250, H, KH, d, scheme=scheme, dtype=dtype) for _ in "ab")
    for c in (a, b):
        fill(c, np.random.default_rng(19), lens, dtype)
    whole = back(a.append(x, **kw))
    ka, va = (t.numpy() for t in a.read((B, n), dtype="f32"))
    for lo, hi in ((3, 40), (0, 3), (40, n)):
        np.testing.assert_array_equal(back(b.append(np.ascontiguousarray(x[:, lo:hi]), offset=lo, **kw)), whole[:, lo:hi])
        k, v = (t.numpy() for t in b.read((B, hi - lo), offset=lo, dtype="f32"))
        np.testing.assert_array_equal(k, ka[:, lo:hi])
        np.testing.assert_array_equal(v, va[:, lo:hi])
    for i in range(B):
        want = R.heads_in(x[i].reshape(n, H + 2 * KH, d)[:, :H], w, 1e-6, lens[i] + np.arange(n), cs, sn, False)
        size = np.abs(want).max(-1, keepdims=True)
        assert (np.abs(whole[i] - want) <= 2.0 ** -24 * 32 * size + (2.0 ** -8 if dtype == "bf16" else 0) * np.abs(want) * 1.001).all()     # as in the test of append
    s = b.step([2, 0], [2, 5])
    k, v = (t.numpy() for t in b.read(s, offset=7, dtype="f32"))
    np.testing.assert_array_equal(k, np.concatenate([ka[2, 7:9], ka[0, 7:12]]))
    np.testing.assert_array_equal(v, np.concatenate([va[2, 7:9], va[0, 7:12]]))
    b.check()
    np.testing.assert_array_equal(back(a.attention(whole)), back(b.attention(whole)))


# ---- a loop: every round against the plain cache ------------------------------------------------------------------------
@pytest.mark.parametrize("scheme,dtype,H,KH,d", [("int8", "f32", 8, 2, 64), ("fp8", "bf16", 4, 2, 128), ("int8", "bf16", 2, 2, 80)])
def test_a_loop_whose_rounds_are_the_plain_caches(scheme, dtype, H, KH, d):
    """Prompt, then rounds of a tree: norms, rotation, attention, commit.  Keys are within half a code of the formulas', values are the
    definition's, and the attention is that of what the cache then holds."""
    rng = np.random.default_rng(20)
    B, n = 3, 16
    c = new(B, 400, H, KH, d, scheme=scheme, dtype=dtype)
    cs, sn = tables(c.max_seq, d // 2)
    w = rng.normal(1, 0.2, (2, d)).astype(np.float32)
    held = [np.zeros((2, 0, KH, d), np.float32) for _ in range(B)]
    for r, T in enumerate([90, n, n, n, n]):
        parents = R.TREE16 if r else None
        x = stored(rng.normal(0, 1, (B, T, (H + 2 * KH) * d)), dtype)
        tree = c.tree(parents) if r else None
        q = c.append(x, tree=tree, q_norm=w[0], k_norm=w[1], rope=(cs, sn))
        got = back(c.attention(q, tree=tree))
        q = back(q)
        k, v = (a.numpy() for a in c.read((B, T), dtype="f32"))
        keep = np.zeros((B, T), np.int32)
        if r:
            paths = ([0, 1, 5, 13], [0], [0, 3, 10])
            kept = [len(p) for p in paths]
            for b, p in enumerate(paths):
                keep[b, :len(p)] = p
        else:
            kept, paths = [90, 71, 0], [list(range(90)), list(range(71)), []]
        c.commit(T, np.asarray(kept, np.int32), keep if r else None)
        depth, seen = R.depth_and_seen(parents, T)
        for b in range(B):
            m = held[b].shape[1]
            h = x[b].reshape(T, H + 2 * KH, d)
            for key in (False, True):
                want = R.heads_in(h[:, H:H + KH] if key else h[:, :H], w[int(key)], 1e-6, m + depth, cs, sn, False)
                size = np.abs(want).max(-1, keepdims=True)
                if key:
                    step = size / 254 if scheme == "int8" else np.maximum(np.abs(want) * 2.0 ** -4, size / 448 * 2.0 ** -10)
                else:
                    step = (2.0 ** -8 if dtype == "bf16" else 0) * np.abs(want)
                assert (np.abs((k if key else q)[b] - want) <= 2.0 ** -24 * 64 * size + step * 1.001).all()       # 32-bit steps as in the test of append
            np.testing.assert_array_equal(v[b], R.in_8_bits(h[:, H + KH:], scheme))
            kk, vv = np.concatenate([held[b][0], k[b]]), np.concatenate([held[b][1], v[b]])
            out, weight, reach = R.attention(q[b], kk, vv, m, depth, seen, 0, d ** -0.5)
            tol = R.tolerance(out, weight, reach, d, m + T, dtype, scheme == "int8")
            assert (np.abs(got[b] - out) <= tol).all(), (r, b, float(np.max(np.abs(got[b] - out) / tol)))
            held[b] = np.concatenate([held[b], np.stack([k[b], v[b]])[:, paths[b]]], 1)
        assert c.per_seq_lens.tolist() == [x.shape[1] for x in held]
        for b in range(B):
            kb, vb = c.get(b)
            np.testing.assert_array_equal(kb, held[b][0])
            np.testing.assert_array_equal(vb, held[b][1])
    c.check()


def test_two_captured_graphs_in_turn():
    """Both use the context's workspace; replayed in any order, with eager calls between, each gives what it gave eagerly."""
    import ctypes as C
    rng = np.random.default_rng(21)
    few, many = new(16, 2200, 16, 8, 64), new(4, 1500, 8, 1, 128, scheme="fp8")
    fill(few, rng, [2000] * 16, "bf16", loud=False)
    fill(many, rng, [1400, 3, 0, 700], "bf16", loud=False)
    few.set_lengths([2000 - 1] * 16)
    many.set_lengths([1400 - 30, 3, 0, 600])
    ctx, lib = few.ctx, few.ctx.lib
    made = []
    for c, T in ((few, 1), (many, 30)):
        q = ctx.from_numpy(rng.integers(0x3c00, 0x4000, (c.max_batch, T, c.n_head, c.head_dim)).astype(np.uint16))
        want = c.attention(q).numpy()
        o = ctx.zeros(want.shape, np.uint16)
        ctx._check(lib.vn_graph_begin(ctx.handle))
        c.attention(q, out=o)
        graph = C.c_void_p()
        ctx._check(lib.vn_graph_end(ctx.handle, C.byref(graph)))
        made.append((c, q, o, want, graph))
    for which in rng.integers(0, 4, 40):
        c, q, o, want, graph = made[which % 2]
        if which < 2:
            ctx._check(lib.vn_memset(ctx.handle, C.c_void_p(o.ptr), 0, o.nbytes))
            ctx._check(lib.vn_graph_launch(ctx.handle, graph))
        np.testing.assert_array_equal((o if which < 2 else c.attention(q)).numpy(), want)
    for _ in range(20):                                           # nothing read between
        for c, q, o, want, graph in made:
            ctx._check(lib.vn_graph_launch(ctx.handle, graph))
    for c, q, o, want, graph in made:
        np.testing.assert_array_equal(o.numpy(), want)
        ctx._check(lib.vn_graph_destroy(ctx.handle, graph))
        c.check()


def test_a_copy_that_does_not_come_is_reported():
    """A wait that runs out sets the condition; it is told once, and the next call is good."""
    import ctypes as C
    from versenext_b200._lib import VN_ERR_INVALID
    rng = np.random.default_rng(22)
    c = new(1, 300, 2, 1, 64, dtype="f32")
    check_attention(c, rng, [200], [3], "f32")
    q = rng.normal(0, 1, (1, 3, 2, 64)).astype(np.float32)
    want = c.attention(q).numpy()
    waited = C.c_int64()
    c.ctx._check(c.ctx.lib.vn_qkv_probe_wait(c.handle, 2_000_000, C.byref(waited)))       # about a millisecond
    assert 2_000_000 <= waited.value < 200_000_000
    with pytest.raises(RuntimeError):
        c.check()
    c.check()
    np.testing.assert_array_equal(c.attention(q).numpy(), want)
    for cycles in (0, 1 << 40):
        assert c.ctx.lib.vn_qkv_probe_wait(c.handle, cycles, None) == VN_ERR_INVALID


# ---- large values that a row does not see -------------------------------------------------------------------------------
@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,H,d,T", [("f32", 2, 64, 4), ("bf16", 1, 64, 6), ("bf16", 2, 128, 8), ("bf16", 2, 64, 20), ("bf16", 4, 128, 30), ("bf16", 4, 96, 20), ("bf16", 2, 256, 20), ("f32", 2, 128, 40)])
@pytest.mark.parametrize("size", [1e4, 1e10, 1e18, 1e30, 3e38])
@pytest.mark.parametrize("where", ["chain", "tree", "window"])
def test_values_that_a_row_does_not_see_do_not_touch_it(scheme, dtype, H, d, T, size, where):
    """A later row of a chain, a row of a tree that no other sees, a position behind the window of the later rows, with values `size` times as
    large as the others'.  A row's weights are held relative to the largest scale that it sees itself, or to 2^-117 of the largest that one of
    its neighbours sees: on tcgen05 2^-150 of that is lost at most for every key, as 2^-33 of the row's own largest, else 2^-156 and 2^-39."""
    rng = np.random.default_rng(T + d)
    n = 300
    c = new(1, n + T, H, 1, d, scheme=scheme, dtype=dtype)
    q, k, v = (stored(rng.normal(0, 1, s), dtype) for s in ((T, H, d), (n + T, 1, d), (n + T, 1, d)))
    window, parents, at = 0, None, n + T - 1
    if where == "tree":
        parents, at = [-1] + [0] * (T - 1), n + T // 2
    if where == "window":
        window, at = 200, n - 200 + T // 2                        # seen by the first half of the rows
    v[at] = stored(v[at] / np.abs(v[at]).max() * size, dtype)
    write(c, k, v)
    c.set_lengths([n])
    got = back(c.attention(q[None], tree=c.tree(parents) if parents else None, window=window))[0]
    c.check()
    depth, seen = R.depth_and_seen(parents, T)
    out, weight, reach = R.attention(q, R.in_8_bits(k, scheme), R.in_8_bits(v, scheme), n, depth, seen, window, d ** -0.5)
    tol = R.tolerance(out, weight, reach, d, n + T, dtype, scheme == "int8")
    if dtype == "bf16":
        tol = tol + 2.0 ** -150 * size * (n + T)
    assert np.isfinite(got).all() and (np.abs(got - out) <= tol).all(), float(np.max(np.abs(got - out) / tol))
