"""QuantKVCache on the device against a plain cache in 64 bits: append, attention, read, commit, alone and as a decoding loop uses them."""

import numpy as np
import pytest

import qkv_cases as R

pytestmark = pytest.mark.gpu


def new(*a, **kw):
    import versenext_b200 as vn
    return vn.QuantKVCache(vn.Context.get(0), *a, **kw)


def stored(x, dtype):
    """float32 values that rows of this type hold."""
    from versenext_b200.quant_cache import from_bf16, to_bf16
    return from_bf16(to_bf16(x)) if dtype == "bf16" else np.asarray(x, np.float32)


def back(a):
    from versenext_b200.quant_cache import from_bf16
    x = a.numpy()
    return from_bf16(x) if x.dtype == np.uint16 else x


def tables(positions, pairs):
    ang = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(pairs) / max(pairs, 1))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def fill(c, rng, lens, dtype, loud=True):
    """Committed positions of every sequence; returns the values (k, v) that the cache then stands for."""
    kv = [rng.normal(0, 1, (2, n, c.n_kv_head, c.head_dim)) * (10.0 ** rng.uniform(-2, 2, (2, n, 1, 1)) if loud else 1.0) for n in lens]
    for x in kv:
        x[0] /= np.maximum(np.abs(x[0]).max(-1, keepdims=True), 1e-30) / 3
    kv = [stored(x, dtype) for x in kv]
    c.reset()
    if sum(lens):
        rows = np.concatenate([x.transpose(1, 0, 2, 3).reshape(n, 2 * c.n_kv_head * c.head_dim) for x, n in zip(kv, lens)])
        c.append(rows, step=c.step(range(len(lens)), lens), queries=False)
    c.set_lengths(np.asarray(list(lens) + [0] * (c.max_batch - len(lens))))
    return [R.in_8_bits(x, c.scheme) for x in kv]


# ---- append and read ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,d", [(1, 8), (2, 16), (3, 64), (8, 128), (2, 72), (1, 80), (2, 96), (1, 192), (2, 256), (5, 248)])
def test_codes_are_the_definitions(scheme, dtype, kv, d):
    rng = np.random.default_rng(d)
    c = new(3, 200, kv, kv, d, scheme=scheme, dtype=dtype)
    c.set_pages(rng.permutation(c.pages).reshape(3, -1))
    lens = [130, 0, 65]
    vals = fill(c, rng, lens, dtype)
    for b, n in enumerate(lens):
        k, v = c.get(b)
        np.testing.assert_array_equal(k, vals[b][0])
        np.testing.assert_array_equal(v, vals[b][1])
    k, v = c.read((3, 20), start=45, dtype="bf16")
    np.testing.assert_array_equal(back(k)[0], stored(vals[0][0][45:65], "bf16"))
    np.testing.assert_array_equal(back(v)[2], stored(vals[2][1][45:65], "bf16"))
    k, v = c.read(c.step([2, 0], [5, 9]), back=True, dtype="f32")
    np.testing.assert_array_equal(k.numpy()[:5], vals[2][0][-5:])
    np.testing.assert_array_equal(v.numpy()[5:], vals[0][1][-9:])
    c.check()


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
def test_zeros_ties_and_values_that_are_not_finite(scheme):
    c = new(1, 64, 1, 1, 64, scheme=scheme, dtype="f32")
    top = 127.0 if scheme == "int8" else 448.0
    k = np.zeros((8, 64), np.float32)
    k[1, :5] = [top, 0.5, 1.5, 2.5, -3.5]                 # scale 1: halves between two codes, to even
    k[2, 0], k[2, 1:4] = -top, [17.0, 19.0, 0.0009765625]  # e4m3: 17 and 19 lie between 16, 18, 20; half the smallest number
    k[3, 7] = np.nan
    k[4, 63] = -np.inf
    k[5] = 1e-42                                          # below the smallest scale
    k[6, 0] = 3.4e38
    k[7] = -7.0
    v = k[::-1].copy()
    c.append(np.concatenate([k, v], 1)[None], queries=False)
    gk, gv = (x.numpy()[0, :, 0] for x in c.read((1, 8), dtype="f32"))
    np.testing.assert_array_equal(gk, R.in_8_bits(k, scheme))
    np.testing.assert_array_equal(gv, R.in_8_bits(v, scheme))
    assert np.isnan(gk[3]).all() and np.isnan(gk[4]).all() and np.isfinite(gk[[0, 1, 2, 5, 6, 7]]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,KH,d,pairs,inter,norm,T,tree", [
    (4, 2, 64, 32, False, True, 3, False), (4, 2, 64, 32, True, False, 3, False), (6, 3, 128, 64, False, True, 1, False), (2, 1, 256, 128, False, True, 16, True),
    (8, 8, 16, 4, False, False, 16, True), (5, 1, 72, 36, False, True, 2, False), (3, 1, 80, 10, False, True, 7, False), (2, 2, 8, 3, True, True, 5, False),
    (4, 4, 192, 0, False, True, 5, False), (16, 8, 96, 41, False, False, 5, False), (4, 1, 248, 124, True, True, 4, False)])
def test_append_norms_and_rotates(dtype, H, KH, d, pairs, inter, norm, T, tree):
    rng = np.random.default_rng(H * 1000 + d)
    B, lens = 3, [0, 61, 17]
    c = new(B, 90, H, KH, d, scheme="int8", dtype=dtype)
    fill(c, rng, lens, dtype)
    x = stored(rng.normal(0, 2, (B, T, (H + 2 * KH) * d)), dtype)
    qw, kw = (rng.normal(1, 0.3, d).astype(np.float32) if norm else None for _ in "qk")
    cs, sn = tables(c.max_seq, pairs)
    parents = R.TREE16 if tree else None
    t = c.tree(parents) if tree else None
    q = back(c.append(x, tree=t, q_norm=qw, k_norm=kw, eps=1e-5, rope=(cs, sn) if pairs else None, interleaved=inter))
    k, v = (a.numpy() for a in c.read((B, T), dtype="f32"))
    depth, _ = R.depth_and_seen(parents, T)
    for b in range(B):
        h = x[b].reshape(T, H + 2 * KH, d)
        both = R.heads_in(h[:, :H], qw, 1e-5, lens[b] + depth, cs if pairs else None, sn, inter)
        # 32-bit steps: d squares (2^-24 each, pairwise at least over lanes), root, division, weight, rotation: 16 of them are plenty
        # of room for 12, relative to the larger of a pair's two channels; then half a step of the type
        size = np.abs(both).max(-1, keepdims=True)
        tol = 2.0 ** -24 * 16 * 2 * size + (2.0 ** -8 if dtype == "bf16" else 0) * np.abs(both) * 1.001
        assert (np.abs(q[b] - both) <= tol).all()
        want = R.heads_in(h[:, H:H + KH], kw, 1e-5, lens[b] + depth, cs if pairs else None, sn, inter)
        # keys may fall on the other side of a step's middle: half a code and what the value is off
        step = np.abs(want).max(-1, keepdims=True) / 127
        assert (np.abs(k[b] - want) <= step * 0.5 + 2.0 ** -24 * 40 * np.abs(want).max(-1, keepdims=True)).all()
        np.testing.assert_array_equal(v[b], R.in_8_bits(h[:, H + KH:], "int8"))
    c.check()


def test_rows_of_a_packed_projection_and_rows_of_nobody():
    """Rows behind a step's last stay as they were; unaligned and strided rows through the C entry point."""
    import ctypes as C
    rng = np.random.default_rng(3)
    c = new(4, 64, 2, 1, 24, scheme="int8", dtype="f32")
    s = c.step([3, 1], [2, 3])
    x = rng.normal(0, 1, (9, 96)).astype(np.float32)
    out = c.ctx.from_numpy(np.full((9, 2, 24), 7.0, np.float32))
    c.append(x, step=s, out=out)
    got = out.numpy()
    np.testing.assert_array_equal(got[:5], x[:5, :48].reshape(5, 2, 24))
    assert (got[5:] == 7.0).all()
    out2 = c.ctx.from_numpy(np.full((9, 2, 24), 7.0, np.float32))
    c.attention(out, step=s, out=out2)
    assert (out2.numpy()[5:] == 7.0).all()
    wide = c.ctx.from_numpy(rng.normal(0, 1, (5, 101)).astype(np.float32))
    ptr = C.c_void_p(wide.ptr + 4)                         # one value in: aligned to 4 bytes only
    c.ctx._check(c.ctx.lib.vn_qkv_append(c.handle, ptr, 101, 1, s.entries, s.ents, s.row_ent, s.T, s.rows, 0, None, 0, None, None, 1e-6, None, None, 0, 0, 0, out.ptr))
    np.testing.assert_array_equal(out.numpy()[:5], wide.numpy()[:, 1:49].reshape(5, 2, 24))
    k, _ = c.read(s, dtype="f32")
    np.testing.assert_array_equal(k.numpy()[:, 0], R.in_8_bits(wide.numpy()[:, 49:73], "int8"))


# ---- attention ------------------------------------------------------------------------------------------------------
def check_attention(c, rng, lens, counts, dtype, parents=None, window=0, scale=None, ragged=False, q_size=1.0):
    H, KH, d = c.n_head, c.n_kv_head, c.head_dim
    old = fill(c, rng, lens, dtype)
    B, T = len(lens), max(counts)
    M = sum(counts)
    q = stored(rng.normal(0, q_size, (M, H, d)), dtype)
    kv = stored(rng.normal(0, 1, (M, 2, KH, d)), dtype)
    step = c.step(range(B), counts) if ragged else None
    rows = np.concatenate([q.reshape(M, -1), kv.reshape(M, -1)], 1)
    tree = c.tree(parents) if parents is not None else None
    got_q = c.append(rows if ragged else rows.reshape(B, T, -1), step=step, tree=tree)
    np.testing.assert_array_equal(back(got_q).reshape(M, H, d), q)
    got = back(c.attention(got_q, step=step, tree=tree, window=window, scale=scale)).reshape(M, H, d)
    c.check()
    at = 0
    for b, n in enumerate(counts):
        depth, seen = R.depth_and_seen(parents, n)
        k = np.concatenate([old[b][0], R.in_8_bits(kv[at:at + n, 0], c.scheme)])
        v = np.concatenate([old[b][1], R.in_8_bits(kv[at:at + n, 1], c.scheme)])
        out, weight, reach = R.attention(q[at:at + n], k, v, lens[b], depth, seen, window, d ** -0.5 if scale is None else scale)
        tol = R.tolerance(out, weight, reach, d, lens[b] + n, dtype, c.scheme == "int8")
        worst = np.abs(got[at:at + n] - out) / tol
        assert np.isfinite(got[at:at + n]).all() and (worst <= 1).all(), (b, float(np.nanmax(worst)))
        at += n


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,KH,d", [(4, 4, 16), (8, 2, 64), (8, 1, 128), (6, 2, 96), (5, 1, 72), (3, 1, 80), (4, 2, 192), (16, 2, 256), (2, 2, 8), (24, 1, 128)])
def test_decoding(scheme, dtype, H, KH, d):
    rng = np.random.default_rng(H + d)
    c = new(4, 700, H, KH, d, scheme=scheme, dtype=dtype)
    c.set_pages(rng.permutation(c.pages).reshape(4, -1))
    check_attention(c, rng, [0, 31, 64, 613], [1] * 4, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,T", [([0], 1), ([1], 1), ([0, 0], 2), ([63, 64, 65], 1), ([31, 32, 33, 127, 128], 5), ([500], 64), ([0], 200), ([100, 3], 70)])
def test_lengths(dtype, lens, T):
    rng = np.random.default_rng(T)
    c = new(len(lens), max(lens) + T, 8, 2, 64, scheme="int8", dtype=dtype)
    check_attention(c, rng, lens, [T] * len(lens), dtype)


@pytest.mark.parametrize("scheme,dtype,H,KH,d", [("int8", "bf16", 16, 8, 64), ("fp8", "bf16", 32, 8, 128), ("int8", "f32", 4, 1, 96), ("fp8", "bf16", 8, 1, 256)])
@pytest.mark.parametrize("window", [0, 40])
def test_trees(scheme, dtype, H, KH, d, window):
    rng = np.random.default_rng(d)
    c = new(3, 300, H, KH, d, scheme=scheme, dtype=dtype)
    check_attention(c, rng, [0, 250, 47], [16] * 3, dtype, parents=R.TREE16, window=window)


def test_trees_of_one_to_sixty_four_rows():
    rng = np.random.default_rng(9)
    for n in (1, 2, 33, 64):
        c = new(2, 200, 4, 2, 64)
        parents = [int(rng.integers(-1, i)) if i else -1 for i in range(n)]
        check_attention(c, rng, [100, 5], [n] * 2, "bf16", parents=parents)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 5000])
def test_windows(window):
    rng = np.random.default_rng(window)
    c = new(3, 400, 4, 2, 64, dtype="f32")
    check_attention(c, rng, [300, 0, 90], [70] * 3, "f32", window=window)
    check_attention(c, rng, [300, 0, 90], [1] * 3, "f32", window=window)


def test_ragged_steps():
    rng = np.random.default_rng(5)
    c = new(6, 400, 8, 2, 64)
    check_attention(c, rng, [300, 0, 90, 7, 64, 200], [1, 130, 0, 5, 64, 1], "bf16", ragged=True)
    check_attention(c, rng, [300, 0, 90, 7, 64, 200], [3, 0, 16, 1, 9, 16], "bf16", parents=R.TREE16, ragged=True)
    check_attention(c, rng, [0, 0, 0, 0, 0, 1], [0, 0, 0, 0, 0, 1], "bf16", ragged=True)


def test_scales_of_the_scores_and_large_queries():
    rng = np.random.default_rng(6)
    c = new(2, 300, 4, 2, 64, dtype="f32")
    check_attention(c, rng, [250, 10], [3, 3], "f32", scale=1.0)
    check_attention(c, rng, [250, 10], [3, 3], "f32", scale=1e-3, q_size=1e4)
    check_attention(c, rng, [250, 10], [3, 3], "f32", q_size=1e-30)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_long_context(dtype):
    rng = np.random.default_rng(7)
    c = new(1, 20100, 8, 2, 128, scheme="fp8", dtype=dtype)
    check_attention(c, rng, [20011], [4], dtype)


def test_many_sequences():
    rng = np.random.default_rng(8)
    n = 300
    c = new(n, 128, 2, 1, 32)
    check_attention(c, rng, [int(x) for x in rng.integers(0, 120, n)], [2] * n, "bf16")


def test_sequences_share_pages():
    """Two sequences over the same first pages: what one appends behind them the other does not see."""
    rng = np.random.default_rng(10)
    c = new(2, 192, 4, 2, 64, pages=5, dtype="f32")
    c.set_pages([[3, 0, -1], [-1, -1, -1]])
    old = fill(c, rng, [128], "f32")[0]
    c.set_pages([[3, 0, 1], [3, 0, 4]])
    c.set_lengths([128, 128])
    q, kv = rng.normal(0, 1, (2, 1, 4, 64)).astype(np.float32), rng.normal(0, 1, (2, 1, 2, 2, 64)).astype(np.float32)
    got = c.attention(c.append(np.concatenate([q.reshape(2, 1, -1), kv.reshape(2, 1, -1)], 2))).numpy()
    for b in range(2):
        k, v = (np.concatenate([old[i], R.in_8_bits(kv[b, :, i], "int8")]) for i in (0, 1))
        out, weight, reach = R.attention(q[b], k, v, 128, np.zeros(1, int), np.ones((1, 1), bool), 0, 0.125)
        assert (np.abs(got[b] - out) <= R.tolerance(out, weight, reach, 64, 129, "f32")).all()
    c.check()


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
def test_bad_heads_reach_only_the_rows_that_see_them(scheme):
    """A position that reads as NaN, an infinite query: the rows that see them, and no others."""
    rng = np.random.default_rng(11)
    for which in (0, 1):
        c = new(1, 200, 4, 2, 64, scheme=scheme, dtype="f32")
        kv = rng.normal(0, 1, (100, 2, 2, 64)).astype(np.float32)
        kv[20, which, 1, 5] = np.inf
        kv[97, which, 0, 3] = np.nan
        c.append(kv.reshape(1, 100, -1), queries=False)
        c.set_lengths([90])
        q = rng.normal(0, 1, (1, 10, 4, 64)).astype(np.float32)
        got = c.attention(q, window=60).numpy()[0]                 # the window hides position 20
        bad = np.isnan(got).any(-1)
        assert bad[7:, :2].all() and not bad[:7].any() and not bad[:, 2:].any()
        got = c.attention(q, window=0).numpy()[0]
        bad = np.isnan(got).all(-1)
        assert bad[:, 2:].all() and not np.isnan(got[:7, :2]).any() and bad[7:, :2].all()
    q[0, 3, 2] = np.inf
    q[0, 4, 0, 9] = np.nan
    c.set_lengths([0])
    bad = np.isnan(c.attention(q).numpy()[0]).any(-1)
    assert bad[3, 2] and bad[4, 0] and bad.sum() == 2


def test_nothing_stale_is_seen():
    """Positions behind the step's rows hold NaN and large values from before."""
    rng = np.random.default_rng(12)
    c = new(2, 200, 4, 2, 64, dtype="f32")
    old = np.full((2, 200, 256), 1e30, np.float32)
    old[:, ::3] = np.nan
    c.append(old, queries=False)
    check_attention(c, rng, [70, 0], [3, 3], "f32")


# ---- commit, and everything together -----------------------------------------------------------------------------------
@pytest.mark.parametrize("scheme,KH,d", [("int8", 2, 64), ("fp8", 8, 128), ("int8", 1, 256), ("fp8", 3, 24)])
def test_commit(scheme, KH, d):
    rng = np.random.default_rng(d)
    lens, n = [0, 60, 119, 33], 16
    c = new(4, 140, KH, KH, d, scheme=scheme, dtype="f32")
    c.set_pages(rng.permutation(c.pages).reshape(4, -1))
    old = fill(c, rng, lens, "f32")
    kv = rng.normal(0, 1, (4, n, 2, KH, d)).astype(np.float32)
    c.append(kv.reshape(4, n, -1), queries=False)
    keep = np.zeros((4, n), np.int32)
    keep[0, :5], keep[1, :16], keep[2, :1], keep[3, :4] = [0, 2, 5, 9, 15], range(16), [15], [3, 2, 1, 0]
    kept = [5, 16, 1, 4]
    c.commit(n, np.asarray(kept) - 1, keep, keep_add=1)
    assert c.per_seq_lens.tolist() == [a + b for a, b in zip(lens, kept)]
    for b in range(4):
        k, v = c.get(b)
        np.testing.assert_array_equal(k, np.concatenate([old[b][0], R.in_8_bits(kv[b, keep[b, :kept[b]], 0], scheme)]))
        np.testing.assert_array_equal(v, np.concatenate([old[b][1], R.in_8_bits(kv[b, keep[b, :kept[b]], 1], scheme)]))
    c.commit(3, [0, 3, 1, 2])
    assert c.per_seq_lens.tolist() == [5, 79, 121, 39]
    c.check()


def test_what_does_not_fit_is_left_out_and_reported():
    c = new(2, 64, 2, 1, 16, dtype="f32")
    rows = np.ones((2, 3, 64), np.float32)
    c.set_lengths([62, 10])
    c.append(rows)
    with pytest.raises(RuntimeError):
        c.check()
    c.check()                                                     # told once
    k, _ = c.read((2, 2), start=62, dtype="f32")
    assert (k.numpy()[0] == 1).all()
    c.read((1, 2), start=63)
    with pytest.raises(RuntimeError):
        c.check()
    c.commit(3, [3, 1])                                           # 62 + 3 > 64
    with pytest.raises(IndexError):
        c.check()
    assert c.per_seq_lens.tolist() == [64, 11]
    c.commit(2, [0, 2], np.array([[0, 1], [0, 7]], np.int32))
    with pytest.raises(IndexError):
        c.check()
    c = new(2, 128, 2, 1, 16, dtype="f32", pages=2)               # nobody has a page
    c.append(rows)
    with pytest.raises(RuntimeError):
        c.check()
    c.set_pages([[0, -1], [1, -1]])
    c.append(rows)
    c.check()
    c.set_lengths([70, 0])                                        # says more than it has pages for
    out = c.attention(np.ones((2, 1, 2, 16), np.float32)).numpy()
    assert np.isfinite(out).all()
    with pytest.raises(RuntimeError):
        c.check()


def test_device_tables_out_of_range_are_left_out():
    c = new(2, 64, 2, 1, 16, dtype="f32")
    s = c.step([0, 1], [1, 1])
    ents = np.array([[0, 0, 1, 0], [7, 1, 1, 0]], np.int32)
    s._buf = c.ctx.from_numpy(np.concatenate([ents.reshape(-1), np.array([0, 1], np.int32)]))
    s.ents, s.row_ent = s._buf.ptr, s._buf.ptr + 32
    q = c.append(np.ones((2, 64), np.float32), step=s)
    with pytest.raises(IndexError):
        c.check()
    out = c.attention(q, step=s).numpy()
    np.testing.assert_allclose(out[0], 1, rtol=2.0 ** -20)
    with pytest.raises(IndexError):
        c.check()


def test_argument_refusals_of_the_library():
    import versenext_b200 as vn
    ctx = vn.Context.get(0)
    for a in ((0, 64, 2, 1, 16), (1, 0, 2, 1, 16), (1, 64, 3, 2, 16), (1, 64, 2, 1, 12), (1, 64, 2, 1, 264), (1, 64, 0, 1, 16), (70000, 64, 2, 1, 16)):
        with pytest.raises(ValueError):
            vn.QuantKVCache(ctx, *a)
    with pytest.raises(MemoryError):
        vn.QuantKVCache(ctx, 60000, 1 << 20, 8, 8, 128, pages=1 << 30)
    c = new(2, 64, 2, 1, 16, dtype="f32")
    for kw in (dict(window=-1), dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            c.attention(np.zeros((1, 1, 2, 16), np.float32), **kw)
    with pytest.raises(ValueError):
        c.append(np.zeros((1, 1, 64), np.float32), offset=-1)
    with pytest.raises(ValueError):
        c.commit(65, [1, 1], np.zeros((2, 65), np.int32))
    c.attention(np.zeros((0, 0, 2, 16), np.float32))
    c.append(np.zeros((0, 64), np.float32), step=c.step([], []))


def test_a_decoding_loop_and_its_captured_replay():
    """Prompt, then rounds of a tree: append, attention, commit, all on device lengths, eager and as a replayed graph; the same
    results bit for bit, and those of the plain cache."""
    import ctypes as C
    rng = np.random.default_rng(13)
    B, H, KH, d, n = 3, 8, 2, 64, 16
    rows = rng.normal(0, 1, (4, B, n, (H + 2 * KH) * d)).astype(np.float32)
    prompt = rng.normal(0, 1, (B, 90, (H + 2 * KH) * d)).astype(np.float32)
    keep = np.zeros((B, n), np.int32)
    keep[0, :4], keep[1, :1], keep[2, :3] = [0, 1, 5, 13], [0], [0, 3, 10]
    nk = np.array([4, 1, 3], np.int32)

    def run(captured):
        c = new(B, 200, H, KH, d, dtype="f32")
        ctx, lib = c.ctx, c.ctx.lib
        cs, sn = (ctx.from_numpy(t) for t in tables(c.max_seq, 32))
        qw = ctx.from_numpy(np.full(d, 1.5, np.float32))
        outs = [c.attention(c.append(prompt, q_norm=qw, k_norm=qw, rope=(cs, sn))).numpy()]
        c.commit(90, np.full(B, 90, np.int32))
        tree, dk, dn = c.tree(R.TREE16), ctx.from_numpy(keep), ctx.from_numpy(nk)
        x, q, o = ctx.empty((B, n, (H + 2 * KH) * d)), ctx.empty((B, n, H, d)), ctx.empty((B, n, H, d))

        def once():
            c.append(x, tree=tree, q_norm=qw, k_norm=qw, rope=(cs, sn), out=q)
            c.attention(q, tree=tree, out=o)
            c.commit(n, dn, dk)
        graph = None
        if captured:
            ctx._check(lib.vn_graph_begin(ctx.handle))
            once()
            graph = C.c_void_p()
            ctx._check(lib.vn_graph_end(ctx.handle, C.byref(graph)))
        for r in range(4):
            x.copy_from_host(rows[r])
            if captured:
                ctx._check(lib.vn_graph_launch(ctx.handle, graph))
            else:
                once()
            outs.append(o.numpy())
        if graph:
            ctx._check(lib.vn_graph_destroy(ctx.handle, graph))
        c.check()
        return outs, c.per_seq_lens.tolist(), [c.get(b) for b in range(B)], (cs.numpy(), sn.numpy())

    a, lens, kv, (cs, sn) = run(False)
    b, lens2, kv2, _ = run(True)
    assert lens == lens2 == [90 + 16, 90 + 4, 90 + 12]
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)
    for x, y in zip(kv, kv2):
        np.testing.assert_array_equal(x[0], y[0])
        np.testing.assert_array_equal(x[1], y[1])
    # the last round from the plain cache: committed values as read back, its own rows from the definition
    depth, seen = R.depth_and_seen(R.TREE16, n)
    w = np.full(d, 1.5)
    for s in range(B):
        m = lens[s] - nk[s]
        x = rows[3, s].reshape(n, H + 2 * KH, d)
        q, k = (R.heads_in(x[:, h0:h1], w, 1e-6, m + depth, cs, sn, False) for h0, h1 in ((0, H), (H, H + KH)))
        k, v = (R.in_8_bits(t, "int8") for t in (k, x[:, H + KH:]))
        k, v = np.concatenate([kv[s][0][:m], k]), np.concatenate([kv[s][1][:m], v])
        out, weight, reach = R.attention(q.astype(np.float32), k, v, m, depth, seen, 0, 0.125)
        # keys whose quotient lies at a code's edge may have the neighbouring code here: one step of one channel, 1 / 127 of the
        # head's maximum, moves a score by at most max|q| max|k| / 127 / 8, and the weights by twice that
        edge = 2 * np.abs(q).max() * np.abs(k).max() / 127 * 0.125
        assert (np.abs(a[-1][s] - out) <= R.tolerance(out, weight, reach, d, m + n, "f32") + 2 * edge * weight).all()


def test_two_caches_on_one_context_do_not_meet():
    rng = np.random.default_rng(14)
    a, b = new(1, 5000, 8, 1, 128, dtype="f32"), new(2, 3000, 8, 2, 64, dtype="f32")
    fill(a, rng, [4900], "f32")
    fill(b, rng, [2900, 100], "f32")
    qa, qb = rng.normal(0, 1, (1, 1, 8, 128)).astype(np.float32), rng.normal(0, 1, (2, 1, 8, 64)).astype(np.float32)
    a.set_lengths([4899])
    b.set_lengths([2899, 99])
    wa, wb = a.attention(qa).numpy(), b.attention(qb).numpy()
    outs = [(a.attention(qa), b.attention(qb)) for _ in range(20)]
    for x, y in outs:
        np.testing.assert_array_equal(x.numpy(), wa)
        np.testing.assert_array_equal(y.numpy(), wb)


# ---- many rows of bf16, and shapes one after another ---------------------------------------------------------------------
@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("H,KH,d,lens,T", [
    (8, 2, 64, [4300, 5], 70),                             # units of 68 pages, cut among shares
    (24, 1, 128, [9000], 5), (20, 1, 64, [6100, 0, 63], 1),  # one row block, few units: a unit in many shares
    (4, 4, 128, [700, 64, 0, 1], 33), (2, 1, 40, [500], 20), (6, 2, 120, [129, 300], 9), (17, 1, 8, [400], 1),
    (12, 3, 56, [3, 900], 31), (4, 1, 64, [0], 300)])
def test_many_rows(scheme, H, KH, d, lens, T):
    rng = np.random.default_rng(H * T + d)
    c = new(len(lens), max(lens) + T, H, KH, d, scheme=scheme)
    c.set_pages(rng.permutation(c.pages).reshape(len(lens), -1))
    check_attention(c, rng, lens, [T] * len(lens), "bf16")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [1, 64, 100, 5000])
def test_windows_of_many_rows(d, window):
    rng = np.random.default_rng(window + d)
    c = new(3, 900, 4, 2, d)
    check_attention(c, rng, [800, 0, 90], [70] * 3, "bf16", window=window)
    check_attention(c, rng, [800, 0, 90], [16] * 3, "bf16", window=window, parents=R.TREE16)
    check_attention(c, rng, [800, 0, 90], [1, 70, 33], "bf16", window=window, ragged=True)


def test_steps_of_every_shape_one_after_another():
    """Units of 8 rows leave a list of cuts with high share numbers behind; those of 128 rows come next, with other places for their parts."""
    rng = np.random.default_rng(15)
    few, many = new(16, 2200, 16, 8, 64), new(4, 1500, 8, 1, 128, scheme="fp8")
    exact = new(2, 900, 4, 1, 64, dtype="f32")
    for _ in range(2):
        check_attention(few, rng, [int(x) for x in rng.integers(1500, 2100, 16)], [1] * 16, "bf16")
        check_attention(many, rng, [1300, 0, 70, 900], [16] * 4, "bf16", parents=R.TREE16)
        check_attention(few, rng, [2100] * 4 + [30] * 12, [4] * 16, "bf16", window=1000)
        check_attention(exact, rng, [600, 800], [40] * 2, "f32")
        check_attention(many, rng, [1400, 3, 0, 600], [60] * 4, "bf16")
        check_attention(few, rng, [2000] + [0] * 15, [10] * 16, "bf16")


def test_shapes_in_turn_give_the_same_bits_without_waits_between_them():
    """Launched back to back, nothing read between: each as by itself."""
    rng = np.random.default_rng(16)
    few, many = new(32, 3000, 16, 8, 64), new(8, 1600, 16, 4, 64)
    fill(few, rng, [2900] * 32, "bf16", loud=False)
    fill(many, rng, [1500] * 8, "bf16", loud=False)
    few.set_lengths([2900 - 5] * 32)
    many.set_lengths([1500 - 64] * 8)
    rows = lambda *s: few.ctx.from_numpy(rng.integers(0x3c00, 0x4000, s).astype(np.uint16))
    q1, q5, q16, q64 = rows(32, 1, 16, 64), rows(32, 5, 16, 64), rows(8, 16, 16, 64), rows(8, 64, 16, 64)
    tree = many.tree(R.TREE16)
    calls = [lambda: few.attention(q1), lambda: many.attention(q16, tree=tree), lambda: few.attention(q5, window=700), lambda: many.attention(q64), lambda: many.attention(q16, tree=tree)]
    want = [f().numpy() for f in calls]
    for _ in range(10):
        for w, g in zip(want, [f() for f in calls]):
            np.testing.assert_array_equal(g.numpy(), w)
    few.check()
    many.check()


@pytest.mark.parametrize("scheme", ["int8", "fp8"])
@pytest.mark.parametrize("d", [64, 128])
def test_bad_heads_and_many_rows_of_bf16(scheme, d):
    rng = np.random.default_rng(17)
    for which in (0, 1):
        c = new(1, 400, 4, 2, d, scheme=scheme)
        kv = rng.normal(0, 1, (300, 2, 2, d)).astype(np.float32)
        kv[20, which, 1, 5] = np.inf
        kv[285, which, 0, 3] = np.nan
        c.append(stored(kv, "bf16").reshape(1, 300, -1), queries=False)
        c.set_lengths([270])
        q = stored(rng.normal(0, 1, (1, 30, 4, d)), "bf16")
        bad = np.isnan(back(c.attention(q, window=100))[0])
        assert bad[15:, :2].all() and not bad[:15].any() and not bad[:, 2:].any()
        bad = np.isnan(back(c.attention(q))[0])
        assert bad[:, 2:].all() and bad[15:, :2].all() and not bad[:15, :2].any()
    q[0, 14, 2, 0] = np.inf
    q[0, 4, 0, 7] = np.nan
    c.set_lengths([0])
    bad = np.isnan(back(c.attention(q))[0]).any(-1)
    assert bad[14, 2] and bad[4, 0] and bad[:20].sum() == 2 and bad[20:, 2:].all() and not bad[20:, :2].any()


def test_commit_of_more_rows_than_a_length_can_count():
    c = new(2, 64, 1, 1, 8, dtype="f32")
    c.set_lengths([62, 10])
    c.commit(2 ** 31 - 1, np.array([2 ** 31 - 1, 1], np.int32))
    with pytest.raises(IndexError):
        c.check()
    assert c.per_seq_lens.tolist() == [64, 11]
