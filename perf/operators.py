"""The operators of the 8-bit cache of keys and values -- append, attention, commit, read -- with their plain forms.

A case names its operator and sizes.  `prepare` makes what a program holds before the call (a filled cache, the step's rows, the
tree), `run` is one pass: the plain form in elementary torch, or the calls of the library where `own` is true.  `exact` gives the
same outputs in 64 bits from the definition.

Sequences have different lengths (`_lens`), their pages are scattered over the pool, and a step brings `new` rows a sequence
(`ragged`: between none and `new`).
"""

import math

import numpy as np
import torch

own = False

PAGE = 64
# 16 nodes behind the last committed token (row 0 is that token): the shape of the framework's tree proposals
TREE16 = [-1, 0, 0, 0, 0, 1, 1, 2, 2, 3, 3, 4, 4, 5, 5, 6]


# ---- the cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a decoding step of 64 requests: norms of the query and key heads, rotation, and the cache, in one launch
        {"name": "append_decode_64", "op": "append", "batch": 64, "new": 1, "ctx": 4000, "heads": 32, "kv": 8, "dim": 128, "scheme": "int8", "dtype": "bf16",
         "norm": True, "rotary": 128, "interleaved": False},
        # prompts of four requests, heads of the mate-shaped target
        {"name": "append_prompt_4x2000", "op": "append", "batch": 4, "new": 2000, "ctx": 0, "heads": 16, "kv": 8, "dim": 64, "scheme": "fp8", "dtype": "bf16",
         "norm": False, "rotary": 64, "interleaved": False},
        # one long request's keys and values in bf16 again, as for a kernel that knows no 8 bits
        {"name": "read_one_50000", "op": "read", "batch": 1, "count": 50000, "kv": 8, "dim": 128, "scheme": "int8", "dtype": "bf16"},
        # some hundred positions of many requests
        {"name": "read_32x500", "op": "read", "batch": 32, "count": 500, "kv": 8, "dim": 64, "scheme": "fp8", "dtype": "f32"},
        # the accepted path of a tree is kept in 32 requests
        {"name": "commit_tree_32x16", "op": "commit", "batch": 32, "new": 16, "tree": True, "ctx": 1000, "heads": 16, "kv": 8, "dim": 128, "scheme": "int8",
         "dtype": "bf16", "norm": False, "rotary": 128, "interleaved": False},
        # the accepted prefix of a chain of one request
        {"name": "commit_chain_1x5", "op": "commit", "batch": 1, "new": 5, "tree": False, "ctx": 500, "heads": 16, "kv": 8, "dim": 64, "scheme": "fp8",
         "dtype": "bf16", "norm": False, "rotary": 64, "interleaved": False},
        # decoding of 64 requests of mixed lengths
        {"name": "decode_64", "op": "attention", "batch": 64, "new": 1, "ctx": 4000, "heads": 32, "kv": 8, "dim": 128, "scheme": "int8", "dtype": "bf16", "window": 0},
        # one request with a long context: the keys are split over the whole machine
        {"name": "decode_1_120000", "op": "attention", "batch": 1, "new": 1, "ctx": 120000, "heads": 64, "kv": 8, "dim": 128, "scheme": "fp8", "dtype": "bf16", "window": 0},
        # the verification step of the speculative workload: 32 requests, k = 4, a window of 1024
        {"name": "verify_32x5", "op": "attention", "batch": 32, "new": 5, "ctx": 1500, "heads": 16, "kv": 8, "dim": 64, "scheme": "int8", "dtype": "bf16", "window": 1024},
        # tree verification: 8 requests, 16 rows, a context of 2048
        {"name": "tree_8x16", "op": "attention", "batch": 8, "new": 16, "tree": True, "ctx": 2048, "heads": 32, "kv": 8, "dim": 128, "scheme": "int8", "dtype": "bf16", "window": 0},
        # a step of the CPU-sized model in the default float32: launches and latency
        {"name": "small_f32", "op": "attention", "batch": 1, "new": 5, "ctx": 33, "heads": 4, "kv": 4, "dim": 16, "scheme": "int8", "dtype": "f32", "window": 0},
        # portions of two prompts
        {"name": "prompt_2x1000", "op": "attention", "batch": 2, "new": 1000, "ctx": 1500, "heads": 16, "kv": 8, "dim": 128, "scheme": "int8", "dtype": "bf16", "window": 0,
         "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "commit", "attention", "attention", "attention", "attention"])
    kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([16, 32, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256])
    c = {"op": op, "kv": kv, "dim": dim, "scheme": rng.choice(["int8", "fp8"]), "dtype": rng.choice(["bf16", "bf16", "bf16", "f32"])}
    if op == "read":
        b = _log(rng, 1, 64)
        return dict(c, batch=b, count=_log(rng, 1, 25_000_000 // (b * kv * dim)))
    c.update(heads=kv * group)
    if op in ("append", "commit"):
        rotary = rng.choice([0, dim, dim, dim // 2 & ~7])
        c.update(norm=rng.random() < 0.5, rotary=rotary, interleaved=rng.random() < 0.3, ctx=_log(rng, 1, 4000))
        if op == "commit":
            tree = rng.random() < 0.7
            return dict(c, batch=_log(rng, 1, 64), new=16 if tree else rng.randint(1, 9), tree=tree)
        b = _log(rng, 1, 64)
        return dict(c, batch=b, new=_log(rng, 1, max(1, 2000 // b)), ragged=rng.random() < 0.3)
    kind = rng.choice(["decode", "decode", "verify", "tree", "prompt"])
    b = _log(rng, 1, 64)
    c.update(batch=b, window=rng.choice([0, 0, 0, 100, 1024]))
    if kind == "prompt":
        b = rng.randint(1, 2)
        new = _log(rng, 20, 700)
        return dict(c, batch=b, new=new, ctx=_log(rng, 1, max(1, min(1500, 4_000_000_000 // (b * new * kv * group * dim) - new))), ragged=rng.random() < 0.5)
    most = min(100000, 120_000_000 // (b * kv * dim), 4_000_000_000 // (b * (1 if kind == "decode" else 8 if kind == "verify" else 16) * kv * group * dim))
    ctx = _log(rng, 1, max(1, most))
    if kind == "decode":
        return dict(c, new=1, ctx=ctx)
    if kind == "verify":
        return dict(c, new=rng.randint(2, 8), ctx=ctx, ragged=rng.random() < 0.3)
    return dict(c, new=16, tree=True, ctx=ctx)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _lens(case):
    """Committed tokens of every sequence: the first has `ctx`, the others between a quarter of it and all of it."""
    b, n = case["batch"], case.get("ctx", case.get("count"))
    return [n - (n * 3 * (i * 7 % 11)) // 44 for i in range(b)] if case["op"] != "read" else [n] * b


def _counts(case):
    """New rows of every sequence."""
    n = case.get("new", 0)
    return [n - (n * (i * 5 % 9)) // 8 if case.get("ragged") else n for i in range(case["batch"])]


def _positions(case):
    """Room for the longest sequence, in whole pages."""
    return -(-(max(_lens(case)) + case.get("new", 0) + 1) // PAGE) * PAGE


def _depth(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _seen(case):
    """[new, new] truth values: row i sees new row j."""
    n = case["new"]
    if not case.get("tree"):
        return torch.ones(n, n, dtype=torch.bool).tril()
    m = torch.eye(n, dtype=torch.bool)
    for i, p in enumerate(TREE16):
        if p >= 0:
            m[i] |= m[p]
    return m


def _kept(case):
    """(how many new rows stay, which ones) for every sequence: a path of the tree, or a prefix of the chain."""
    n, idx = [], []
    for b in range(case["batch"]):
        if case["tree"]:
            at, path = [5, 9, 15, 3, 0, 12][b % 6], []
            while at >= 0:
                path.append(at)
                at = TREE16[at]
            path = path[::-1]
        else:
            path = list(range(b * 3 % case["new"] + 1))
        n.append(len(path))
        idx.append(path + [0] * (case["new"] - len(path)))
    return n, idx


def _values(case, g, rows):
    """Keys and values as projections give them: some channels of the keys are many times as large as the others."""
    shape = (rows, case["kv"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda")
    wide = torch.randn((case["kv"], case["dim"]), generator=g, device="cuda")
    k = k * (1 + 4 * (wide > 1.5)) * (0.5 + torch.rand((rows, 1, 1), generator=g, device="cuda"))
    v = torch.randn(shape, generator=g, device="cuda") * (0.3 + torch.rand((rows, 1, 1), generator=g, device="cuda"))
    return k.to(_type(case)), v.to(_type(case))


def _inputs(case, seed):
    """Everything that the seed decides, the same for every form of the operator."""
    g = _gen(seed)
    B, dev = case["batch"], "cuda"
    lens, counts = _lens(case), _counts(case)
    pages = _positions(case) // PAGE
    table = torch.randperm(B * pages, generator=g, device=dev).to(torch.int32).reshape(B, pages)
    s = {"lens": torch.tensor(lens, device=dev), "table": table}
    if case["op"] != "append":
        s["k"], s["v"] = _values(case, g, sum(lens))
        if case["op"] == "commit":                          # the committed part is not looked at
            s["k"], s["v"] = s["k"][:0], s["v"][:0]
    if case["op"] == "attention":
        s["k_new"], s["v_new"] = _values(case, g, sum(counts))
        s["q"] = (torch.randn((sum(counts), case["heads"], case["dim"]), generator=g, device=dev) * 1.5).to(_type(case))
    if case["op"] in ("append", "commit"):
        H, KH, d = case["heads"], case["kv"], case["dim"]
        s["rows"] = (torch.randn((sum(counts), (H + 2 * KH) * d), generator=g, device=dev)
                     * (0.5 + torch.rand((sum(counts), 1), generator=g, device=dev))).to(_type(case))
        if case["norm"]:
            s["q_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
            s["k_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
        if case["rotary"]:
            pairs = case["rotary"] // 2
            freq = 10000.0 ** (-torch.arange(pairs, device=dev, dtype=torch.float64) / pairs)
            ang = torch.arange(_positions(case), device=dev, dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    return s


def _quantise(x, scheme):
    """Codes and scales of heads x [..., d]: as they stand in the cache.  (Divisions by tensors: one by a number is torch's product with
    the number's reciprocal.)"""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    one = torch.ones_like(top)
    if scheme == "int8":
        scale = torch.where(top > 0, top, one) / (127 * one)
        return torch.round(x / scale).clamp(-127, 127).to(torch.int8), scale
    scale = torch.where(top > 0, top, one) / (448 * one)
    return (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.int8), scale


def _values_of(codes, scale, scheme, ftype):
    """What the codes stand for."""
    return (codes if scheme == "int8" else codes.view(torch.float8_e4m3fn)).to(ftype) * scale.to(ftype)


def _entries(counts, device="cuda"):
    """(sequence, place among its new rows) of every row of a step."""
    n = torch.tensor(counts, device=device)
    seq = torch.repeat_interleave(torch.arange(len(counts), device=device), n)
    first = torch.cumsum(n, 0) - n
    return seq, torch.arange(int(sum(counts)), device=device) - first[seq]


# ---- what a program holds before the call -----------------------------------------------------------------------------
def _device(t):
    """A torch tensor as an array of the library: the same memory."""
    from versenext_b200 import Context
    from versenext_b200.device import DeviceArray
    kind = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int32: np.int32}[t.dtype]
    return DeviceArray(Context.get(0), t.data_ptr(), tuple(t.shape), kind, base=t)


def _own_cache(case, x):
    import versenext_b200 as vn
    ctx = vn.Context.get(0)
    torch.cuda.synchronize()
    c = vn.QuantKVCache(ctx, case["batch"], _positions(case), case.get("heads", case["kv"]), case["kv"], case["dim"], scheme=case["scheme"], dtype=case["dtype"])
    c.set_pages(x["table"].cpu().numpy())
    lens = x["lens"].tolist()

    def write(k, v, counts):
        rows = torch.cat([k.flatten(1), v.flatten(1)], 1)
        torch.cuda.synchronize()
        c.append(_device(rows), step=c.step(range(len(counts)), counts), queries=False)
        ctx.sync()

    if "k" in x and len(x["k"]):
        write(x["k"], x["v"], lens)
    if case["op"] != "read":
        c.set_lengths(np.asarray(lens, np.int32))
    if "k_new" in x:
        write(x["k_new"], x["v_new"], _counts(case))
    return c


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case, "x": x}
    counts = _counts(case)
    if own:
        c = s["cache"] = _own_cache(case, x)
        s["step"] = c.step(range(case["batch"]), counts) if case["op"] != "read" else c.step(range(case["batch"]), [case["count"]] * case["batch"])
        s["tree"] = c.tree(TREE16, s["step"]) if case.get("tree") else None
        s["dev"] = {n: _device(t) for n, t in x.items() if n in ("q", "rows", "q_norm", "k_norm", "cos", "sin")}
        if case["op"] == "commit":
            n, idx = _kept(case)
            s["n_keep"], s["keep"] = c.ctx.from_numpy(np.asarray(n, np.int32)), c.ctx.from_numpy(np.asarray(idx, np.int32))
            s["lens"] = c.ctx.from_numpy(np.asarray(_lens(case), np.int32))
            s["kept"] = c.step(range(case["batch"]), n)
        c.ctx.sync()
        return s
    # a pool of pages of codes [pages, 64, kv, dim] with their scales, keys and values
    n = x["table"].numel()
    s["pool"] = [(torch.zeros((n, PAGE, case["kv"], case["dim"]), dtype=torch.int8, device="cuda"), torch.ones((n, PAGE, case["kv"], 1), device="cuda")) for _ in "kv"]
    s["seq"], s["at"] = _entries(counts)
    s["depth"] = torch.tensor(_depth(TREE16) if case.get("tree") else range(case.get("new", 0)), dtype=torch.int64, device="cuda")
    s["seen"] = _seen(case).cuda() if "new" in case else None
    if "k" in x and len(x["k"]):
        seq, at = _entries(_lens(case))
        _write(s, seq, at, x["k"], x["v"])
    if "k_new" in x:
        _write(s, s["seq"], x["lens"][s["seq"]] + s["at"], x["k_new"], x["v_new"])
    if case["op"] == "commit":
        n, idx = _kept(case)
        seq, i = _entries(n)
        s["kept"] = seq, i, torch.tensor(idx, device="cuda")[seq, i]
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _where(s, seq, pos):
    return s["x"]["table"].long()[seq, pos // PAGE], pos % PAGE


def _write(s, seq, pos, k, v):
    page, at = _where(s, seq, pos)
    for (codes, scales), x in zip(s["pool"], (k, v)):
        q, sc = _quantise(x, s["case"]["scheme"])
        codes[page, at], scales[page, at] = q, sc


def _read(s, seq, pos, ftype):
    page, at = _where(s, seq, pos)
    return [_values_of(codes[page, at], scales[page, at], s["case"]["scheme"], torch.float32).to(ftype) for codes, scales in s["pool"]]


def _normed_rotated(x, w, eps, cos, sin, interleaved):
    """Heads x [rows, heads, d] normalised and rotated; cos, sin [rows, 1, pairs] or None."""
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    if cos is None:
        return x
    n = cos.shape[-1]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    y, z = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_append(s):
    case, x = s["case"], s["x"]
    H, KH, d = case["heads"], case["kv"], case["dim"]
    rows = x["rows"].float().reshape(-1, H + 2 * KH, d)
    pos = x["lens"][s["seq"]] + s["at"]                       # where a row stands in the cache
    turn = x["lens"][s["seq"]] + s["depth"][s["at"]]          # and how far it is from the beginning
    cos, sin = (x["cos"][turn][:, None], x["sin"][turn][:, None]) if case["rotary"] else (None, None)
    q = _normed_rotated(rows[:, :H], x.get("q_norm"), 1e-6, cos, sin, case["interleaved"])
    k = _normed_rotated(rows[:, H:H + KH], x.get("k_norm"), 1e-6, cos, sin, case["interleaved"])
    _write(s, s["seq"], pos, k, rows[:, H + KH:])
    return q.to(_type(case)), pos


def _plain_attention(s):
    case, x = s["case"], s["x"]
    B, T, H, KH, d = case["batch"], case["new"], case["heads"], case["kv"], case["dim"]
    k, v = (_values_of(codes[x["table"].long()], scales[x["table"].long()], case["scheme"], torch.float32).reshape(B, -1, KH, d) for codes, scales in s["pool"])
    q = torch.zeros((B, T, H, d), device="cuda")
    q[s["seq"], s["at"]] = x["q"].float()
    L, lens = k.shape[1], x["lens"]
    key = torch.arange(L, device="cuda")
    turn = lens[:, None] + s["depth"][None]                   # [B, T]
    seen = key < lens[:, None, None]                          # [B, 1, L] committed
    if case["window"]:
        seen = seen & (turn[..., None] - key < case["window"])
    new = key - lens[:, None]                                 # [B, L] place among the new rows
    inside = (new >= 0) & (new < T)
    drafted = s["seen"][:, new.clamp(0, T - 1)].permute(1, 0, 2) & inside[:, None]
    if case["window"]:                                        # (a tree is never deeper than the windows here)
        drafted = drafted & (turn[..., None] - (lens[:, None] + s["depth"][new.clamp(0, T - 1)])[:, None] < case["window"])
    seen = (seen | drafted)[:, None, None]                    # [B, 1, 1, T, L]
    a = torch.matmul(q.reshape(B, T, KH, H // KH, d).permute(0, 2, 3, 1, 4).reshape(B, KH, -1, d), k.permute(0, 2, 3, 1)) * d ** -0.5
    a = torch.where(seen, a.reshape(B, KH, H // KH, T, L), float("-inf"))
    m = a.amax(-1, keepdim=True)
    e = torch.exp(a - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(B, KH, -1, L), v.permute(0, 2, 1, 3)).reshape(B, KH, H // KH, T, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, d)[s["seq"], s["at"]].to(_type(case))


def _plain(s):
    case, x = s["case"], s["x"]
    if case["op"] == "attention":
        return _plain_attention(s)
    if case["op"] == "read":
        n = case["count"]
        pos = torch.arange(n, device="cuda").expand(case["batch"], n)
        seq = torch.arange(case["batch"], device="cuda")[:, None].expand(case["batch"], n)
        return [t.flatten(0, 1) for t in _read(s, seq, pos, _type(case))]
    q, pos = _plain_append(s)
    if case["op"] == "append":
        return [q] + _read(s, s["seq"], pos, torch.bfloat16)
    seq, i, src = s["kept"]
    base = x["lens"][seq]
    page, at = _where(s, seq, base + src)
    to_page, to_at = _where(s, seq, base + i)
    for codes, scales in s["pool"]:
        codes[to_page, to_at], scales[to_page, to_at] = codes[page, at], scales[page, at]
    return [q] + _read(s, seq, base + i, torch.bfloat16)


# ---- the library's calls ------------------------------------------------------------------------------------------------
def _own_read(s, step, ftype, **at):
    case, c = s["case"], s["cache"]
    k, v = (torch.empty((step.rows, case["kv"], case["dim"]), dtype=ftype, device="cuda") for _ in "kv")
    c.read(step, out=(_device(k), _device(v)), dtype="f32" if ftype == torch.float32 else "bf16", **at)
    return [k, v]


def _own(s):
    case, c, dev = s["case"], s["cache"], s["dev"]
    if case["op"] == "read":
        return _own_read(s, s["step"], _type(case), start=0)
    q = torch.empty((s["step"].rows, case["heads"], case["dim"]), dtype=_type(case), device="cuda")
    if case["op"] == "attention":
        c.attention(dev["q"], step=s["step"], tree=s["tree"], window=case["window"], out=_device(q))
        return q
    if case["op"] == "commit":
        c.set_lengths(s["lens"])
    c.append(dev["rows"], step=s["step"], tree=s["tree"], q_norm=dev.get("q_norm"), k_norm=dev.get("k_norm"), eps=1e-6,
             rope=(dev["cos"], dev["sin"]) if case["rotary"] else None, interleaved=case["interleaved"], out=_device(q))
    if case["op"] == "append":
        return [q] + _own_read(s, s["step"], torch.bfloat16)
    c.commit(case["new"], s["n_keep"], s["keep"])
    # what was kept ends at the new length: read it from where the old one was
    return [q] + _own_read(s, s["kept"], torch.bfloat16, back=True)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    KH, d, es = case["kv"], case["dim"], 4 if case["dtype"] == "f32" else 2
    cell = KH * (2 * d + 8)                                   # a position's codes and scales
    if case["op"] == "read":
        n = case["batch"] * case["count"]
        return {"bytes": n * (cell + 2.0 * KH * d * es), "flops": 2.0 * n * KH * d}
    H, counts, lens = case["heads"], _counts(case), _lens(case)
    M = sum(counts)
    if case["op"] in ("append", "commit"):
        total = M * ((2 * H + 2 * KH) * d * es + cell)        # rows in, queries out, codes out
        kept = M if case["op"] == "append" else sum(_kept(case)[0])
        moved = 0 if case["op"] == "append" else sum(i != j for idx, n in zip(*_kept(case)[::-1]) for i, j in enumerate(idx[:n]))
        return {"bytes": total + kept * (cell + 4.0 * KH * d) + 2.0 * moved * cell, "flops": 10.0 * M * (H + KH) * d}
    seen = _seen(case)
    pairs = keys = 0
    for n, l in zip(counts, lens):
        w = case["window"] or 1 << 40
        depth = _depth(TREE16) if case.get("tree") else range(n)
        first = [max(0, l + t - w + 1) for t in depth]
        if n:
            keys += l + n - min(min(first), l)
            inside = int(seen[:n, :n].sum()) if n <= w else sum(min(i + 1, w) for i in range(n))
            pairs += sum(max(0, l - f) for f in first) + inside
    return {"bytes": keys * cell + 2.0 * M * H * d * es, "flops": 4.0 * H * d * pairs}


# ---- the same outputs in 64 bits ----------------------------------------------------------------------------------------
def _exact_heads(x, w, eps, pos, case, cos, sin):
    x = x.double()
    if w is not None:
        x = x * w.double() / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + eps).pow(0.5)
    if not case["rotary"]:
        return x
    n = case["rotary"] // 2
    turn = torch.complex(cos.double(), sin.double())[pos][:, None]
    out = x.clone()
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case["interleaved"] else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., lo], x[..., hi]) * turn
    out[..., lo], out[..., hi] = z.real, z.imag
    return out


def _exact_in_8_bits(x, scheme):
    """The nearest values that a head's scale and codes can stand for.  Scales and quotients have 32 bits by definition: 16-bit values
    meet the middle between two codes often, and the side they fall on is decided there."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    if scheme == "int8":
        s = (torch.where(top > 0, top, 1.0) / 127).float().double()
        return torch.round((x / s).float().double()) * s
    s = (torch.where(top > 0, top, 1.0) / 448).float().double()
    y = (x / s).float().double()
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * s


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "read":
        # the inputs are the codes: what the cache holds is decided in 32 bits
        return [_values_of(*_quantise(t, case["scheme"]), case["scheme"], torch.float64) for t in (x["k"], x["v"])]
    H, KH, d = case["heads"], case["kv"], case["dim"]
    lens, counts = _lens(case), _counts(case)
    depth = _depth(TREE16) if case.get("tree") else list(range(case["new"]))
    if case["op"] in ("append", "commit"):
        pos = torch.tensor([l + depth[i] for l, n in zip(lens, counts) for i in range(n)], device="cuda")
        rows = x["rows"].reshape(-1, H + 2 * KH, d)
        q = _exact_heads(rows[:, :H], x.get("q_norm"), 1e-6, pos, case, x.get("cos"), x.get("sin"))
        k = _exact_in_8_bits(_exact_heads(rows[:, H:H + KH], x.get("k_norm"), 1e-6, pos, case, x.get("cos"), x.get("sin")), case["scheme"])
        v = _exact_in_8_bits(rows[:, H + KH:], case["scheme"])
        if case["op"] == "append":
            return [q, k, v]
        n, idx = _kept(case)
        at = torch.tensor([b * case["new"] + i for b in range(case["batch"]) for i in idx[b][:n[b]]], device="cuda")
        return [q, k[at], v[at]]
    seen = _seen(case).cuda()
    k, v, kn, vn = (_values_of(*_quantise(x[n], case["scheme"]), case["scheme"], torch.float64) for n in ("k", "v", "k_new", "v_new"))
    if sum(lens) * H * d * case["new"] > 1 << 42:
        return None
    outs, lo, new_lo = [], 0, 0
    dep = torch.tensor(depth, device="cuda")
    for l, n in zip(lens, counts):
        at = torch.cat([torch.arange(l, device="cuda"), l + dep[:n]])
        for h in range(H):
            g = h // (H // KH)
            keys, vals = torch.cat([k[lo:lo + l, g], kn[new_lo:new_lo + n, g]]), torch.cat([v[lo:lo + l, g], vn[new_lo:new_lo + n, g]])
            a = x["q"][new_lo:new_lo + n, h].double() @ keys.T / math.sqrt(d)
            ok = torch.cat([torch.ones((n, l), dtype=torch.bool, device="cuda"), seen[:n, :n]], 1)
            if case["window"]:
                ok &= (l + dep[:n])[:, None] - at < case["window"]
            outs.append(torch.softmax(a.masked_fill(~ok, float("-inf")), -1) @ vals)
        lo, new_lo = lo + l, new_lo + n
    per, i = [], 0
    for n in counts:
        per.append(torch.stack(outs[i:i + H], 1))
        i += H
    return torch.cat(per)
