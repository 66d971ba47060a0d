"""Cases of the grouped-query decode operators: products with 4-bit weights, the paged 8-bit cache's append and the
attention that reads it. ``run`` computes each in plain torch operations, or (``own``) by the package's kernels."""

import math

import torch

own = False

FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a draft layer's key projection for one token: a megabyte of weights, all latency
        dict(name="w4 one row 1024x1024", op="w4", rows=1, n=1024, k=1024, group=128, zeros=False, dtype="bf16"),
        # an ordinary projection of a decode step (the benchmark layer's hidden size) for one token
        dict(name="w4 one row 8192x4096", op="w4", rows=1, n=8192, k=4096, group=128, zeros=False, dtype="bf16"),
        # a few sequences' rows through a ragged projection: odd output width, short groups, zero points
        dict(name="w4 13 rows 2311x4000", op="w4", rows=13, n=2311, k=4000, group=32, zeros=True, dtype="f16"),
        # 48 verify rows through the benchmark's LM head in 4 bits
        dict(name="w4 48 rows 129280x4096", op="w4", rows=48, n=129280, k=4096, group=64, zeros=True, dtype="bf16"),
        # one sequence's next token: the smallest append
        dict(name="append one token", op="append", seqs=1, max_rows=1, ragged=False, ctx=1000, heads=32, kv_heads=8,
             dim=128, rope=128, neox=True, page=64, block=16, dtype="bf16"),
        # a verify step: 8 sequences of 6 rows, rotated in part, larger scale blocks, rows that cross blocks and pages
        dict(name="append 8x6 verify rows", op="append", seqs=8, max_rows=6, ragged=False, ctx=32768, heads=40,
             kv_heads=10, dim=64, rope=32, neox=False, page=32, block=32, dtype="f16"),
        # prompts of uneven lengths (one of them empty) entering the cache together
        dict(name="append ragged prompts", op="append", seqs=6, max_rows=4096, ragged=True, ctx=300, heads=32,
             kv_heads=8, dim=128, rope=128, neox=True, page=64, block=16, dtype="bf16"),
        # one sequence early in its answer: the smallest attention
        dict(name="attend one token ctx 777", op="attend", seqs=1, max_rows=1, ragged=False, ctx=777, even=True,
             heads=32, kv_heads=8, dim=128, window=0, sink=False, page=64, block=16, dtype="bf16"),
        # the benchmark's 48 decode rows at contexts up to 8192, every length different
        dict(name="attend 48 rows ctx 8192", op="attend", seqs=48, max_rows=1, ragged=False, ctx=8192, even=False,
             heads=64, kv_heads=8, dim=128, window=0, sink=False, page=64, block=16, dtype="bf16"),
        # the benchmark's verify step: 8 sequences of 6 rows at context 32768
        dict(name="attend 8x6 rows ctx 32768", op="attend", seqs=8, max_rows=6, ragged=False, ctx=32768, even=True,
             heads=32, kv_heads=8, dim=128, window=0, sink=True, page=64, block=16, dtype="f16"),
        # a windowed layer with a head of its own for every query head, uneven rows a sequence
        dict(name="attend window 1000 dim 64", op="attend", seqs=21, max_rows=5, ragged=True, ctx=16384, even=False,
             heads=12, kv_heads=12, dim=64, window=1000, sink=False, page=16, block=16, dtype="bf16"),
        # four long contexts: a gigabyte of cache for four rows
        dict(name="attend 4 rows ctx 131072", op="attend", seqs=4, max_rows=1, ragged=False, ctx=131072, even=True,
             heads=64, kv_heads=8, dim=128, window=0, sink=False, page=128, block=64, dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(["w4", "append", "attend"])
        dtype = rng.choice(["bf16", "f16"])
        if op == "w4":
            group = rng.choice([32, 64, 128])
            c = dict(op=op, rows=log(1, 48), n=log(256, 65536), k=group * max(1, log(512, 16384) // group),
                     group=group, zeros=rng.random() < 0.5, dtype=dtype)
            if c["n"] * c["k"] > 129280 * 4096:
                continue
            return c
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 16])
        block = rng.choice([16, 32, 64])
        page = block * rng.choice([1, 2, 4])
        c = dict(op=op, seqs=log(1, 64), max_rows=1, ragged=rng.random() < 0.5, ctx=0, heads=heads,
                 kv_heads=kv_heads, dim=dim, page=page, block=block, dtype=dtype)
        if op == "append":
            c.update(max_rows=rng.choice([1, 6, log(2, 2048)]), ctx=log(1, 8192),
                     rope=rng.choice([0, dim // 2, dim]), neox=rng.random() < 0.5)
            if c["seqs"] * c["max_rows"] * (heads + kv_heads) * dim <= 10000 * 40 * 128:
                return c
        else:
            c.update(max_rows=rng.choice([1, 1, log(2, 8)]), ctx=log(1, 131072), even=rng.random() < 0.5,
                     window=rng.choice([0, 0, log(16, 4096)]), sink=rng.random() < 0.3)
            if c["seqs"] * c["ctx"] * kv_heads * dim <= 4 * 131072 * 8 * 128 \
                    and c["seqs"] * c["ctx"] * c["max_rows"] * heads * dim <= 8 * 6 * 32768 * 32 * 128:
                return c


def _lengths(case):
    """(rows of each sequence, tokens of each sequence with its rows): plain numbers that follow from the case alone."""
    rows, lens = [], []
    for s in range(case["seqs"]):
        u = (0.6180339887 * (s + 1)) % 1.0
        n = case["max_rows"]
        if case["ragged"]:
            n = 0 if s == 3 else max(1, int(round(n * u)))
        ctx = case["ctx"] if case.get("even") else max(1, int(case["ctx"] * (0.25 + 0.75 * ((0.7548776662 * (s + 1)) % 1.0))))
        rows.append(n)
        lens.append(max(n, ctx + (n if case["op"] == "append" else 0)))
    if not sum(rows):
        rows[0] = 1
        lens[0] = max(1, lens[0])
    return rows, lens


def _visible(case):
    """Per sequence the number of keys that any of its rows sees, and per row all (row, key) pairs."""
    rows, lens = _lengths(case)
    keys = pairs = 0
    for n, length in zip(rows, lens):
        if not n:
            continue
        w = case["window"] or length
        lo = max(0, length - n + 1 - w)
        keys += length - lo
        pairs += sum(min(length - n + j + 1, w) for j in range(n))
    return keys, pairs


def work(case):
    if case["op"] == "w4":
        m, n, k, g = case["rows"], case["n"], case["k"], case["group"]
        return dict(bytes=n * k // 2 + n * (k // g) * (3 if case["zeros"] else 2) + 2 * m * k + 2 * m * n,
                    flops=2 * m * n * k)
    rows, lens = _lengths(case)
    t, h, hk, d = sum(rows), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        blocks = sum(-(-length // case["block"]) - (length - n) // case["block"] for n, length in zip(rows, lens) if n)
        return dict(bytes=t * (hk * d * 2 * 3 + h * d * 4 + case["rope"] * 4) + 2 * blocks * hk,
                    flops=t * (hk + h) * (3 * case["rope"] + d))
    keys, pairs = _visible(case)
    return dict(bytes=keys * hk * 2 * d + 2 * hk * keys // case["block"] + 4 * t * h * d, flops=4 * pairs * h * d)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    def randint(lo, hi, shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=g, device=dev, dtype=dtype)

    st = dict(case=case)
    if case["op"] == "w4":
        m, n, k, grp = case["rows"], case["n"], case["k"], case["group"]
        st.update(x=randn(m, k), w=randint(0, 256, (n, k // 2), torch.uint8),
                  scales=(torch.rand((n, k // grp), generator=g, device=dev) * 0.02 + 0.002).to(dt),
                  zeros=randint(4, 13, (n, k // grp), torch.uint8) if case["zeros"] else None)
        return st
    rows, lens = _lengths(case)
    s, t = len(rows), sum(rows)
    h, hk, d, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], case["block"]
    width = -(-max(lens) // page)
    pages = sum(-(-x // page) for x in lens) + 3
    # the pages of the pool in no order, as a server's allocator leaves them; what lies behind a sequence points at page 0
    perm = (torch.randperm(pages - 1, generator=g, device=dev) + 1).to(torch.int32)
    table = torch.zeros((s, width), dtype=torch.int32, device=dev)
    at = 0
    for i, x in enumerate(lens):
        np_ = -(-x // page)
        table[i, :np_] = perm[at:at + np_]
        at += np_

    def cache():
        b = torch.empty((pages, hk, page, d), dtype=FP8, device=dev)
        step = max(1, (1 << 27) // (hk * page * d))
        for i in range(0, pages, step):
            b[i:i + step] = (randn(*b[i:i + step].shape, dtype=torch.float16) * 100).clamp_(-448, 448).to(FP8)
        return b.view(torch.uint8), randint(118, 122, (pages, hk, page // block), torch.uint8)

    kc, kcodes = cache()
    vc, vcodes = cache()
    cu = torch.tensor([sum(rows[:i]) for i in range(s + 1)], dtype=torch.int32, device=dev)
    st.update(k_cache=kc, v_cache=vc, k_codes=kcodes, v_codes=vcodes, table=table,
              lens=torch.tensor(lens, dtype=torch.int32, device=dev), cu=cu)
    if case["op"] == "append":
        # q, k and v as one projection leaves them, side by side in a row
        qkv = randn(t, (h + 2 * hk) * d)
        st.update(q=qkv[:, :h * d].view(t, h, d), k=qkv[:, h * d:(h + hk) * d].view(t, hk, d),
                  v=qkv[:, (h + hk) * d:].view(t, hk, d), cos_sin=None)
        if case["rope"]:
            r = case["rope"]
            ang = torch.arange(max(lens), device=dev, dtype=torch.float64)[:, None] \
                * 10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)
            st["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float()
    else:
        st.update(q=randn(t, h, d), scale=1.0 / math.sqrt(d),
                  sink=torch.randn((h,), generator=g, device=dev) if case["sink"] else None)
    if own:
        from sgl_amd_mono_b200.deepseek_v41.sm100a import paged

        st["kv"] = paged.PagedKV(kc, vc, kcodes, vcodes)
    return st


def run(st):
    op = st["case"]["op"]
    if own:
        return _run_own(st, op)
    return {"w4": _w4, "append": _append, "attend": _attend}[op](st)


def _cache_out(st, q):
    """The whole cache after an append, and the rotated queries: the bytes as the e4m3 values that they hold, the codes as
    the powers of two."""
    e8 = torch.float8_e8m0fnu
    return dict(k=st["k_cache"].view(FP8), v=st["v_cache"].view(FP8), k_scale=st["k_codes"].view(e8),
                v_scale=st["v_codes"].view(e8), q=q)


def _run_own(st, op):
    if op == "w4":
        from sgl_amd_mono_b200.deepseek_v41.sm100a import ops

        return ops.gemv_w4(st["x"], st["w"], st["scales"], st["zeros"])
    case = st["case"]
    cu = st["cu"] if case["max_rows"] > 1 or case["ragged"] else None  # None: one row a sequence
    if op == "append":
        q = st["kv"].append(st["k"], st["v"], lens=st["lens"], table=st["table"], cu_rows=cu, q=st["q"],
                            cos_sin=st["cos_sin"], neox=case["neox"])
        return _cache_out(st, q)
    return st["kv"].attend(st["q"], lens=st["lens"], table=st["table"], cu_rows=cu, scale=st["scale"],
                           window=case["window"], sink=st["sink"])


# ------------------------------------------------------------------ the plain forms
def _w4(st):
    w, s, z = st["w"], st["scales"].float(), st["zeros"]
    n, groups = s.shape
    v = torch.stack([w & 15, w >> 4], 2).view(n, groups, -1).float()
    v = (v - (8.0 if z is None else z.float()[:, :, None])) * s[:, :, None]
    return (st["x"].float() @ v.view(n, -1).T).to(st["x"].dtype)


def _positions(st):
    """(sequence of each row, its position, tokens that were there before) of all rows."""
    cu, lens = st["cu"].long(), st["lens"].long()
    seq = torch.searchsorted(cu[1:], torch.arange(st["q"].shape[0], device=cu.device), right=True)
    start = lens - (cu[1:] - cu[:-1])
    return seq, start[seq] + torch.arange(seq.shape[0], device=cu.device) - cu[seq], start


def _rotate(x, pos, cos_sin, neox):
    x = x.float()
    if cos_sin is None:
        return x
    r = cos_sin.shape[1]
    c, s = cos_sin[pos][:, None, :r // 2], cos_sin[pos][:, None, r // 2:]
    keep, y = x[..., :x.shape[-1] - r], x[..., x.shape[-1] - r:]
    a, b = (y[..., :r // 2], y[..., r // 2:]) if neox else (y[..., 0::2], y[..., 1::2])
    ra, rb = a * c - b * s, a * s + b * c
    return torch.cat([keep, torch.cat([ra, rb], -1) if neox else torch.stack([ra, rb], -1).flatten(-2)], -1)


def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _store(x, cache, codes, table, seq, pos, start, cu):
    """Rows x [T, heads, dim] (fp32) into their cache blocks."""
    pages, heads, page, dim = cache.shape
    per = codes.shape[2]
    block = page // per
    phys, off = table[seq, pos // page].long(), pos % page
    at = phys * per + off // block  # the row's block in the pool
    amax = torch.zeros((pages * per, heads), device=x.device).index_reduce_(0, at, x.abs().amax(-1), "amax")
    need = (amax.clamp_min(1e-4) / 448.0).view(torch.int32)
    need = ((need >> 23) & 255) + ((need & 0x7fffff) != 0).int()
    flat = codes.transpose(1, 2).reshape(pages * per, heads).int()
    older = torch.zeros(pages * per, dtype=torch.bool, device=x.device)
    older[at] = pos // block * block < start[seq]  # the same for all rows of a block
    new = torch.where(older[:, None], torch.maximum(flat, need), need)
    touched = torch.zeros_like(older)
    touched[at] = True
    new = torch.where(touched[:, None], new, flat)
    # a sequence's partly filled block: its older tokens move to the new scale
    live = (start % block != 0) & (cu[1:] > cu[:-1])
    sp, so = table[torch.arange(len(start), device=x.device), (start // page).clamp_max(table.shape[1] - 1)].long(), \
        start % page // block
    blocks = cache.view(pages, heads, per, block, dim)
    old = blocks[sp, :, so]  # [sequences, heads, block, dim]
    ratio = _pow2(flat[sp * per + so] - new[sp * per + so])
    moved = (old.view(FP8).float() * ratio[:, :, None, None]).to(FP8).view(torch.uint8)
    is_old = (torch.arange(block, device=x.device)[None] < (start % block)[:, None]) & live[:, None]
    blocks[sp, :, so] = torch.where(is_old[:, None, :, None], moved, old)
    y = (x * _pow2(127 - new[at])[:, :, None]).clamp(-448, 448)
    cache[phys, :, off] = y.to(FP8).view(torch.uint8)
    codes.copy_(new.to(torch.uint8).view(pages, per, heads).transpose(1, 2))


def _append(st):
    seq, pos, start = _positions(st)
    cs, neox, cu = st["cos_sin"], st["case"]["neox"], st["cu"]
    _store(_rotate(st["k"], pos, cs, neox), st["k_cache"], st["k_codes"], st["table"], seq, pos, start, cu)
    _store(st["v"].float(), st["v_cache"], st["v_codes"], st["table"], seq, pos, start, cu)
    return _cache_out(st, _rotate(st["q"], pos, cs, neox).to(st["q"].dtype))


def _dequant(cache, codes, table):
    """The pages of every sequence, [sequences, heads, keys, dim] fp32."""
    pages, heads, page, dim = cache.shape
    per = codes.shape[2]
    t = table.long()
    v = cache.view(FP8)[t].float().view(*t.shape, heads, per, page // per, dim)
    v *= _pow2(codes[t].int() - 127)[..., None, None]
    return v.view(*t.shape, heads, page, dim).transpose(1, 2).reshape(t.shape[0], heads, -1, dim)


def _attend(st):
    q, case = st["q"], st["case"]
    seq, pos, _ = _positions(st)
    k = _dequant(st["k_cache"], st["k_codes"], st["table"])
    s, hk, keys, d = k.shape
    t, h = q.shape[:2]
    j = torch.arange(t, device=q.device) - st["cu"].long()[seq]
    most = case["max_rows"]
    rows = torch.zeros((s, most, h, d), device=q.device)
    rows[seq, j] = q.float()
    rows = rows.view(s, most, hk, h // hk, d).transpose(1, 2).reshape(s, hk, -1, d)
    score = (rows @ k.transpose(2, 3) * st["scale"]).view(s, hk, most, h // hk, keys)
    del k
    last = torch.full((s, most), -1, device=q.device)
    last[seq, j] = pos
    i = torch.arange(keys, device=q.device)
    seen = i <= last[..., None]
    if case["window"]:
        seen &= i > last[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    if st["sink"] is not None:
        sink = st["sink"].view(1, hk, 1, h // hk, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (score - top).exp_()
    total = p.sum(-1, keepdim=True)
    if st["sink"] is not None:
        total = total + (sink - top).exp()
    v = _dequant(st["v_cache"], st["v_codes"], st["table"])
    o = (p.view(s, hk, -1, keys) @ v).view(s, hk, most, h // hk, d) / total.masked_fill(total == 0, 1.0)
    return o.transpose(1, 2).reshape(s, most, h, d)[seq, j].to(q.dtype)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "w4":
        x, w = st["x"].double(), st["w"]
        m, grp = case["rows"], case["group"]
        y = torch.empty((m, case["n"]), dtype=torch.float64, device=x.device)
        for a in range(0, case["n"], 8192):
            wa, sa = w[a:a + 8192], st["scales"][a:a + 8192].double()
            za = torch.full_like(sa, 8.0) if st["zeros"] is None else st["zeros"][a:a + 8192].double()
            acc = torch.zeros((m, wa.shape[0]), dtype=torch.float64, device=x.device)
            for half in (0, 1):  # even columns lie in the low nibbles
                part = ((wa >> (4 * half)) & 15).double()
                sel = torch.arange(half, case["k"], 2, device=x.device) // grp
                acc += x[:, half::2] @ ((part - za[:, sel]) * sa[:, sel]).T
            y[:, a:a + 8192] = acc
        return y
    rows, lens = _lengths(case)
    if case["op"] == "append":
        return _exact_append(case, st, rows, lens)
    d, rep = case["dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    at = 0
    for s, (n, length) in enumerate(zip(rows, lens)):
        ids = torch.arange(length, device=out.device)
        page, off = st["table"][s].long()[ids // case["page"]], ids % case["page"]
        for head in range(case["kv_heads"] if n else 0):
            def read(cache, codes):
                b = cache[page, head, off].view(FP8).double()
                return b * torch.exp2(codes[page, head, off // case["block"]].double() - 127)[:, None]

            k, v = read(st["k_cache"], st["k_codes"]), read(st["v_cache"], st["v_codes"])
            hs = slice(head * rep, head * rep + rep)
            for j in range(n):
                vis = length - n + j + 1
                lo = max(0, vis - case["window"]) if case["window"] else 0
                z = st["q"][at + j, hs].double() @ k[lo:vis].T * st["scale"]
                if st["sink"] is not None:
                    z = torch.cat([z, st["sink"][hs].double()[:, None]], 1)
                p = torch.softmax(z, 1)[:, :vis - lo]
                out[at + j, hs] = p @ v[lo:vis]
        at += n
    return out


def _exact_append(case, st, rows, lens):
    """Every block's scale, and the values over it before they are rounded to e4m3; what was there before in its bits."""
    r, d, page, block = case["rope"], case["dim"], case["page"], case["block"]
    if sum(rows) > 4096:
        return None

    def turn(x, pos):
        x = x.double().clone()
        if r:
            i = torch.arange(r // 2, device=x.device)
            a, b = (d - r + i, d - r // 2 + i) if case["neox"] else (d - r + 2 * i, d - r + 2 * i + 1)
            c, s = st["cos_sin"][pos, :r // 2].double(), st["cos_sin"][pos, r // 2:].double()
            xa, xb = x[..., a].clone(), x[..., b].clone()
            x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
        return x

    out, q = {}, torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for name in ("k", "v"):
        vals = st[name + "_cache"].view(FP8).double()
        codes = st[name + "_codes"].double()
        at = 0
        for s, (n, length) in enumerate(zip(rows, lens)):
            first = length - n
            for b0 in range(first // block * block, length if n else 0, block):
                pg, o = int(st["table"][s, b0 // page]), b0 % page
                new = [p for p in range(max(b0, first), min(b0 + block, length))]
                x = torch.stack([turn(st[name][at + p - first], p) if name == "k" else st[name][at + p - first].double()
                                 for p in new])  # [tokens, heads, dim]
                # float32 of the largest magnitude sets the code, as the cache's format says
                top = x.abs().amax((0, 2)).clamp_min(1e-4)
                code = torch.ceil(torch.log2(top / 448.0)) + 127
                was = codes[pg, :, o // block].clone()
                if b0 < first:
                    code = torch.maximum(code, was)
                    vals[pg, :, o:o + first - b0] *= torch.exp2(was - code)[:, None, None]
                codes[pg, :, o // block] = code
                for p, y in zip(new, x):
                    vals[pg, :, o + p - b0] = y * torch.exp2(127 - code)[:, None]
            if name == "k":
                for p in range(first, length):
                    q[at + p - first] = turn(st["q"][at + p - first], p)
            at += n
        out[name], out[name + "_scale"] = vals, torch.exp2(codes - 127)
    return dict(k=out["k"], v=out["v"], k_scale=out["k_scale"], v_scale=out["v_scale"], q=q)
