"""The grouped-query decode operators against their plain forms: 4-bit GEMV, paged append, attention."""

import math

import pytest
import torch

from oracle import gqa as G

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
FP8 = torch.float8_e4m3fn


def half_step(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------ 4-bit GEMV
def w4_case(M, N, K, group, zeros, dt, seed=0, ld=0):
    g = torch.Generator().manual_seed(seed + M + N + K)
    x = torch.randn(M, K + ld, generator=g).to(dt)[:, :K]
    w = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand(N, K // group, generator=g) * 0.02 + 1e-3).to(dt)
    s[::3] *= -1
    z = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    return x, w, s, z


def w4_check(y, x, w, s, z):
    wd = G.w4_dequant(w, s, z)
    ref, size = x.double() @ wd.T, x.double().abs() @ wd.abs().T
    # one rounding to the output type, and fp32 sums: a chain of at most K / 8 + 32 additions, each off
    # by at most a step (2^-23) of a partial sum that is no larger than sum |x w|
    tol = half_step(y.dtype) * ref.abs() + (x.shape[1] / 8 + 32) * 2.0 ** -23 * size
    if y.dtype == HF:
        tol = tol + 2.0 ** -25  # half of f16's smallest step
    off = ((y.to(x.device).double() - ref).abs() / tol).max().item()
    assert off <= 1, off


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group", [
    (1, 1, 32, 32), (1, 17, 64, 32), (2, 130, 96, 96), (1, 1024, 1024, 128), (5, 333, 416, 32), (8, 64, 2048, 64),
    (9, 100, 4000, 32), (16, 257, 1536, 512), (17, 96, 640, 128), (33, 1600, 4096, 128), (48, 70, 8192, 64),
    (48, 2311, 1056, 96)])
def test_w4_matches(M, N, K, group, zeros, dt):
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(M, N, K, group, zeros, dt)
    y = ops.gemv_w4(x.cuda(), w.cuda(), s.cuda(), None if z is None else z.cuda())
    w4_check(y, x, w, s, z)


@pytest.mark.parametrize("M,N,K,group,zeros,dt", [
    (17, 8192, 4096, 128, True, BF), (48, 8200, 4128, 32, True, HF), (33, 9000, 4096, 64, False, BF),
    (32, 70000, 640, 128, True, BF), (40, 300, 129984, 96, True, HF), (48, 33000, 1056, 32, True, BF),
    (20, 5000, 8192, 512, True, BF), (9, 20000, 2048, 64, True, HF), (1, 20001, 2304, 256, False, BF),
    (6, 9000, 4064, 32, True, BF), (9, 16500, 4096, 32, False, HF), (16, 2100, 32000, 64, True, BF),
    (13, 8200, 8256, 96, True, BF)])
def test_w4_large(M, N, K, group, zeros, dt):
    """Matrices that fill the GPU: many row tiles a CTA, tiles that lie in several CTAs' shares, over 16
    rows (over 8 where scales are many) the tensor-memory kernel; the plain form in fp64 on the GPU."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = (None if t is None else t.cuda() for t in w4_case(M, N, K, group, zeros, dt, seed=3))
    w4_check(ops.gemv_w4(x, w, s, z), x, w, s, z)


def test_w4_unaligned_scales_and_tiny_scales():
    """Scales and zeros that start anywhere, and scales near the ends of bf16's range."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = (t.cuda() for t in w4_case(5, 300, 1024, 64, True, BF, seed=4))
    sb, zb = torch.zeros(s.numel() + 1, dtype=BF, device="cuda"), torch.zeros(z.numel() + 3, dtype=torch.uint8, device="cuda")
    s1, z1 = sb[1:].view(s.shape), zb[3:].view(z.shape)
    s1.copy_(s)
    z1.copy_(z)
    assert torch.equal(ops.gemv_w4(x, w, s1, z1), ops.gemv_w4(x, w, s, z))
    for e in (-70, 70):
        st = (s.float() * 2.0 ** e).to(BF)
        w4_check(ops.gemv_w4(x, w, st, z), x, w, st, z)


@pytest.mark.parametrize("M,N,K,group", [(3, 40, 1024, 128), (48, 1000, 2304, 32), (7, 19, 160, 32), (11, 2100, 32000, 64),
                                         (20, 9000, 4096, 64)])
def test_w4_strides_and_neighbours(M, N, K, group):
    """Rows of x further apart than K, an output inside a wider buffer whose other values stay."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(M, N, K, group, True, BF, seed=5, ld=24)
    xd = torch.full((M, K + 24), float("nan"), dtype=BF, device="cuda")
    xd[:, :K] = x.cuda()
    buf = torch.full((M + 2, N + 11), 7.0, dtype=BF, device="cuda")
    ops.gemv_w4(xd[:, :K], w.cuda(), s.cuda(), z.cuda(), out=buf[1:M + 1, 3:N + 3])
    w4_check(buf[1:M + 1, 3:N + 3], x, w, s, z)
    buf[1:M + 1, 3:N + 3] = 7.0
    assert bool((buf == 7.0).all())


def test_w4_non_finite_stays_in_its_row_and_column():
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(4, 50, 512, 64, True, BF, seed=9)
    x[1, 100], x[2, 7] = float("inf"), float("nan")
    s[9, 3] = float("nan")
    y = ops.gemv_w4(x.cuda(), w.cuda(), s.cuda(), z.cuda()).cpu()
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1:3] = True
    want[:, 9] = True
    assert torch.equal(bad, want)


# ------------------------------------------------------------------ the paged cache
class Step:
    """A step over a paged cache: CPU tensors, and the same on the GPU."""

    def __init__(self, rows, lens, heads, kvh, dim, page, block, dt, seed=0, cu=True, tail=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dt, self.rows, self.page = g, dt, rows, page
        S = len(rows)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.cu = torch.tensor([sum(rows[:i]) for i in range(S + 1)], dtype=torch.int32) if cu else None
        T = sum(rows) + tail
        width = max(1, -(-max(max(lens), 1) // page)) + 1
        need = [max(0, -(-x // page)) for x in lens]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=g, dtype=torch.int32)
        self.table = torch.full((S, width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        shape, cshape = (pages, kvh, page, dim), (pages, kvh, page // block)
        self.k, self.v = (G.to_bytes(torch.randn(shape, generator=g) * 100) for _ in range(2))
        self.kc, self.vc = (torch.randint(117, 123, cshape, generator=g, dtype=torch.uint8) for _ in range(2))
        # q, k and v side by side in a row, as a projection leaves them
        qkv = torch.randn(T, (heads + 2 * kvh) * dim, generator=g).to(dt)
        self.qkv, self.heads, self.kvh, self.dim = qkv, heads, kvh, dim

    def split(self, qkv):
        h, kvh, d, T = self.heads, self.kvh, self.dim, qkv.shape[0]
        return (qkv[:, :h * d].view(T, h, d), qkv[:, h * d:(h + kvh) * d].view(T, kvh, d),
                qkv[:, (h + kvh) * d:].view(T, kvh, d))

    def cache(self):
        from sgl_amd_mono_b200.deepseek_v41.sm100a.paged import PagedKV
        return PagedKV(self.k.cuda(), self.v.cuda(), self.kc.cuda(), self.vc.cuda())

    def where(self):
        return dict(lens=self.lens.cuda(), table=self.table.cuda(), cu_rows=None if self.cu is None else self.cu.cuda())


def rope_table(n, r):
    ang = torch.arange(n)[:, None] * 10000.0 ** (-torch.arange(0, r, 2) / r)
    return torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()


def same_bytes(got, want):
    """Equal bytes, NaN of either sign and zeros of either sign alike."""
    a, b = got.cpu().view(FP8).float(), want.view(FP8).float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def run_append(st, rope=0, neox=False, with_q=True, in_place=False):
    kv = st.cache()
    qkv = st.qkv.cuda()
    q, k, v = st.split(qkv)
    cs = rope_table(int(st.lens.max().clamp_min(1)), rope) if rope else None
    got = kv.append(k, v, q=q if with_q else None, cos_sin=None if cs is None else cs.cuda(), neox=neox,
                    q_out=q if in_place else None, **st.where())
    qc, kc, vc = st.split(st.qkv)
    want_q = qc.clone() if in_place else None
    G.append(st.k, st.kc, kc, st.cu, st.lens, st.table, cs, neox)
    G.append(st.v, st.vc, vc, st.cu, st.lens, st.table)
    assert torch.equal(kv.k_codes.cpu(), st.kc) and torch.equal(kv.v_codes.cpu(), st.vc)
    assert same_bytes(kv.k, st.k) and same_bytes(kv.v, st.v)
    if not with_q:
        assert got is None
        return
    used = sum(st.rows)
    want_q = G.rotate_rows(qc, st.cu, st.lens, cs, neox, torch.zeros(qc.shape, dtype=st.dt))
    assert torch.equal(got.cpu()[:used], want_q[:used])
    if in_place:
        assert got.data_ptr() == q.data_ptr() and torch.equal(qkv[used:].cpu(), st.qkv[used:])


APPENDS = {
    "one token": dict(rows=[1], lens=[1], heads=4, kvh=1, dim=64, page=16, block=16, cu=False),
    "one token into an old block": dict(rows=[1], lens=[15], heads=4, kvh=2, dim=128, page=64, block=16, cu=False),
    "decode rows, one without tokens": dict(rows=[1, 1, 1, 1], lens=[17, 0, 64, 129], heads=2, kvh=2, dim=64, page=32,
                                            block=16, cu=False),
    "verify rows over blocks and pages": dict(rows=[6, 6, 6], lens=[18, 34, 70], heads=8, kvh=2, dim=128, page=32,
                                              block=32),
    "ragged, empty, padded": dict(rows=[3, 0, 40, 1, 0], lens=[3, 9, 77, 48, 0], heads=6, kvh=3, dim=64, page=48,
                                  block=48, tail=4),
    "prompt over pages": dict(rows=[150], lens=[163], heads=2, kvh=1, dim=256, page=64, block=16),
    "more rows than tokens": dict(rows=[5, 2], lens=[3, 1], heads=1, kvh=1, dim=64, page=16, block=16),
}


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("name", APPENDS)
def test_append_bits(name, dt):
    run_append(Step(dt=dt, seed=1, **APPENDS[name]))


@pytest.mark.parametrize("rope,neox", [(16, False), (64, True), (32, True), (64, False)])
@pytest.mark.parametrize("name", ["one token into an old block", "ragged, empty, padded", "prompt over pages"])
def test_append_rotates(name, rope, neox):
    run_append(Step(dt=BF, seed=2, **APPENDS[name]), rope=rope, neox=neox, in_place=neox)


def test_append_without_queries():
    run_append(Step(dt=BF, seed=3, **APPENDS["verify rows over blocks and pages"]), rope=64, with_q=False)


@pytest.mark.parametrize("big", [1.0, 64.0, 3e4])
def test_append_grows_the_scale(big):
    """Older bytes are rounded again to a larger scale, many of them into the subnormals and to zero."""
    st = Step([2, 1], [9, 30], 2, 2, 64, 16, 16, HF, seed=4)
    st.qkv[0] *= big
    st.qkv[2] = 0
    run_append(st)


def test_append_non_finite():
    st = Step([3, 2], [19, 33], 2, 2, 64, 16, 16, BF, seed=5)
    st.qkv[0, 130], st.qkv[1, 200], st.qkv[3, 300] = float("nan"), float("inf"), float("-inf")
    st.qkv[4, 128:256] = float("nan")
    run_append(st)


def test_append_bad_pages_and_positions():
    """Tokens without a page are skipped, and nothing else moves."""
    st = Step([20, 1, 1, 4], [40, 70, 33, 16], 2, 1, 64, 16, 16, BF, seed=6)
    st.table[0, 1], st.table[1, 4], st.table[2, 2] = -7, 1 << 30, st.k.shape[0]
    st.lens[3] = 1 << 20  # far past its table row
    run_append(st)


def test_append_one_by_one_and_together_hold_the_same_scale():
    """Tokens that arrive one at a time end in the codes of one append of all, and in values within
    what the extra roundings allow."""
    rows, dim = 37, 64
    one, all_ = (Step([rows], [rows], 2, 2, dim, 64, 16, BF, seed=7) for _ in range(2))
    a, b = one.cache(), all_.cache()
    _, k, v = one.split(one.qkv.cuda())
    where = all_.where()
    b.append(k, v, **where)
    for i in range(rows):
        a.append(k[i:i + 1], v[i:i + 1], lens=torch.tensor([i + 1], dtype=torch.int32, device="cuda"),
                 table=where["table"])
    assert torch.equal(a.k_codes, b.k_codes) and torch.equal(a.v_codes, b.v_codes)
    x, y = a.k.view(FP8).float(), b.k.view(FP8).float()
    # scales are powers of two: only values that end below e4m3's smallest normal (2^-6) were rounded
    # more than once, each time by at most half a step of 2^-9, at most 15 times and mostly to even
    used = one.table[0, :1].long()
    diff = (x - y).abs()[used.cuda()]
    assert bool((diff[y[used.cuda()].abs() > 2.0 ** -6 + 2.0 ** -9] == 0).all()) and diff.max().item() <= 2.0 ** -8


# ------------------------------------------------------------------ attention
def attn_tol(dt, ref, sizes):
    vabs, sabs, top, seen = sizes
    # the output's rounding; the weights' rounding to f16 (half a step, 2^-11 of each weight, and of
    # those too small for a normal f16 2^-32 of the largest times a byte of at most 448); the scores'
    # fp32 sums (dim terms, a step of 2^-23 each, twice: numerator and sum) and exponentials (2^-20)
    dim = ref.shape[-1]
    ds = (2 * (dim + 4) * 2.0 ** -23 * sabs + 2.0 ** -20 + seen * 2.0 ** -23)[..., None]
    tol = half_step(dt) * ref.abs() + (2.0 ** -11 + ds) * vabs + (seen * 2.0 ** -32 * 448 * top)[..., None] * 1.01
    return tol + 2.0 ** -24 if dt == HF else tol


def run_attend(st, window=0, sink=False, scale=None):
    scale = scale or 1 / math.sqrt(st.dim)
    sk = torch.randn(st.heads, generator=st.g) if sink else None
    kv = st.cache()
    T = st.qkv.shape[0]
    q = st.split(st.qkv)[0]
    qd = st.split(st.qkv.cuda())[0]
    out = torch.full((T, st.heads, st.dim), 5.0, dtype=st.dt, device="cuda")
    sk_d, where = None if sk is None else sk.cuda(), st.where()
    got = kv.attend(qd, scale=scale, window=window, sink=sk_d, out=out, **where)
    assert got is out
    ref, sizes = G.attend(q, st.k, st.v, st.kc, st.vc, st.cu, st.lens, st.table, scale, window, sk)
    used = sum(st.rows)
    # a table with room for long sequences, room for more rows: the same rows, their work split and joined
    wide = torch.full((len(st.rows), 4000), -1, dtype=torch.int32, device="cuda")
    wide[:, :st.table.shape[1]] = where["table"]
    more = torch.zeros((4000,) + qd.shape[1:], dtype=qd.dtype, device="cuda")
    split = torch.full_like(torch.cat([out, more]), 5.0)
    kv.attend(torch.cat([qd, more]), scale=scale, window=window, sink=sk_d, out=split,
              **{**where, "table": wide, "cu_rows": torch.arange(len(st.rows) + 1, dtype=torch.int32).cuda() if st.cu is None
                 else where["cu_rows"]})
    for o in (out, split):
        g = o.cpu().double()
        assert bool((g[used:] == 5.0).all()), "rows behind the last sequence moved"
        err, tol = (g[:used] - ref[:used]).abs(), attn_tol(st.dt, ref, sizes)[:used]
        nan = ref[:used].isnan()
        assert torch.equal(g[:used].isnan(), nan)
        assert bool((err <= tol)[~nan].all()), (err / tol.clamp_min(1e-30))[~nan].max().item()
    return out


ATTNS = {
    "one key": dict(rows=[1], lens=[1], heads=4, kvh=1, dim=64, page=16, block=16, cu=False),
    "one row": dict(rows=[1], lens=[777], heads=8, kvh=2, dim=128, page=64, block=16, cu=False),
    "no keys, one key, a tile, a tile and one": dict(rows=[1, 1, 1, 1, 1], lens=[0, 1, 16, 17, 129], heads=5, kvh=5,
                                                     dim=64, page=16, block=16, cu=False),
    "verify rows": dict(rows=[6, 6], lens=[300, 131], heads=8, kvh=2, dim=128, page=32, block=32),
    "ragged, empty, padded": dict(rows=[3, 0, 7, 1, 0], lens=[3, 9, 200, 48, 0], heads=12, kvh=4, dim=64, page=48,
                                  block=16, tail=3),
    "more rows than tokens": dict(rows=[5, 2], lens=[3, 1], heads=2, kvh=1, dim=64, page=16, block=16),
    "sixteen heads a key": dict(rows=[1, 2], lens=[260, 515], heads=16, kvh=1, dim=256, page=64, block=64),
    "a prompt's rows": dict(rows=[40, 1], lens=[40, 90], heads=6, kvh=2, dim=64, page=16, block=16),
    "three heads a key, wide": dict(rows=[2, 1], lens=[1100, 30], heads=9, kvh=3, dim=256, page=128, block=32),
}


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("name", ATTNS)
def test_attend_matches(name, dt):
    run_attend(Step(dt=dt, seed=11, **ATTNS[name]))


@pytest.mark.parametrize("window", [1, 5, 16, 100, 1000])
@pytest.mark.parametrize("name", ["one row", "ragged, empty, padded", "a prompt's rows", "verify rows"])
def test_attend_window(name, window):
    run_attend(Step(dt=BF, seed=12, **ATTNS[name]), window=window)


@pytest.mark.parametrize("name", ["no keys, one key, a tile, a tile and one", "verify rows", "sixteen heads a key"])
def test_attend_sink(name):
    run_attend(Step(dt=HF, seed=13, **ATTNS[name]), sink=True, window=40)


@pytest.mark.parametrize("code", [0, 60, 200])
def test_attend_extreme_scales(code):
    """Value scales at the ends of E8M0's range beside ordinary ones, in either order: the scores' sum
    counts every token, whatever its value's size."""
    for first in (False, True):
        st = Step([1], [32], 2, 1, 64, 16, 16, BF, seed=18)
        st.vc[st.table[0, 0 if first else 1].long()] = code
        if code > 127:  # values of 2^73 and f32 sums of them: keep the output finite
            st.v[st.table[0, 0 if first else 1].long()] = 0x38
        run_attend(st)


@pytest.mark.parametrize("spread", [0, 30])
def test_attend_uneven_scales(spread):
    """Blocks whose values differ by powers of two, and scores that differ by hundreds."""
    st = Step([4, 1], [700, 350], 8, 2, 64, 32, 16, BF, seed=14)
    st.vc += torch.randint(0, spread + 1, st.vc.shape, generator=st.g, dtype=torch.uint8)
    run_attend(st, scale=4.0)


def test_attend_rising_scores():
    """Every block's scores above all earlier ones: the running maximum moves at each."""
    st = Step([2], [400], 4, 1, 64, 16, 16, HF, seed=15)
    for i in range(25):
        st.kc[st.table[0, i].long()] = 110 + i // 2
    run_attend(st, scale=2.0)


def test_attend_masked_places_hold_anything():
    """NaN in keys, values, scales and pages that a row does not see leaves it untouched."""
    st = Step([3, 1], [37, 21], 4, 2, 64, 16, 16, BF, seed=16)
    pg = st.table.long()
    for c in (st.k, st.v):
        c[pg[0, 2], :, 5:] = 0x7f   # behind the first sequence
        c[pg[1, 1], :, 5:] = 0xff
    st.kc[pg[0, 2]], st.vc[pg[1, 1]] = 120, 121
    run_attend(st)
    # tokens 35 and 36 are the sequence's own later rows: row 0 does not see them
    st.v[pg[0, 2], 0, 3, 10], st.k[pg[0, 2], 1, 4, 3] = 0x7f, 0x7f
    out = run_attend(st)
    assert bool(torch.isfinite(out[0]).all()) and bool(out[1, 0, 10].isnan()) and bool(out[2, 2].isnan().all())
    # before a window
    st.v[pg[0, 0], :, 9] = 0x7f
    run_attend(st, window=20)


def test_attend_bad_pages_are_not_seen():
    st = Step([1, 2, 1], [70, 50, 33], 4, 2, 64, 16, 16, BF, seed=17)
    st.table[0, 1], st.table[1, 0], st.table[1, 3] = -1, 1 << 30, st.k.shape[0]
    st.table[2] = -5
    run_attend(st)
    st.lens[0] = 1 << 30  # past its table row: what the row holds is seen
    run_attend(st)


@pytest.mark.parametrize("heads,kvh", [(4, 2), (20, 1), (48, 2)])
def test_attend_many_sequences(heads, kvh):
    """More sequences than a CTA has threads, most of them without rows, through a table wider than its
    slice: the plan's walk over them."""
    g = torch.Generator().manual_seed(19)
    S = 700
    rows = [int(x) if i % 3 else 0 for i, x in enumerate(torch.randint(0, 3, (S,), generator=g))]
    lens = [int(x) for x in torch.randint(0, 60, (S,), generator=g)]
    lens[650], rows[650] = 900, 2
    st = Step(rows, lens, heads, kvh, 64, 16, 16, BF, seed=20)
    wide = torch.full((S, st.table.shape[1] + 5), 1 << 29, dtype=torch.int32)
    wide[:, :st.table.shape[1]] = st.table
    out = run_attend(st)
    kv, w = st.cache(), st.where()
    w["table"] = wide.cuda()[:, :st.table.shape[1]]
    used = sum(rows)
    again = kv.attend(st.split(st.qkv.cuda())[0], scale=1 / 8, **w)
    assert torch.equal(again[:used], out[:used])


def test_far_pages():
    """Pages whose bytes lie past 2^31: appended to and read as any other."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a.paged import PagedKV
    pages, page, kvh, dim = 70000, 64, 4, 128  # 2.3 GB of keys, as many of values
    big = PagedKV.empty(pages, page, kvh, dim)
    small = PagedKV.empty(8, page, kvh, dim)
    far = torch.tensor([[pages - 1, 3, 66000, 65537]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[1, 3, 6, 7]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(230, kvh, dim, generator=g, device="cuda").to(BF) for _ in range(2))
    cu = torch.tensor([0, 230], dtype=torch.int32, device="cuda")
    lens = torch.tensor([230], dtype=torch.int32, device="cuda")
    for kv, t in ((big, far), (small, near)):
        kv.append(k, v, lens=lens, table=t, cu_rows=cu)
    assert torch.equal(big.k[far[0].long()], small.k[near[0].long()])
    assert torch.equal(big.v_codes[far[0].long()], small.v_codes[near[0].long()])
    q = torch.randn(2, 8, dim, generator=g, device="cuda").to(BF)
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    a, b = (kv.attend(q, lens=lens, table=t, cu_rows=cu, scale=0.1) for kv, t in ((big, far), (small, near)))
    assert torch.equal(a, b) and bool(a.abs().max() > 0)


def test_empty_steps_and_streams():
    """No rows, no sequences; the calls on a side stream, two of them at once."""
    st = Step([3, 1], [40, 20], 4, 2, 64, 16, 16, BF, seed=22)
    kv = st.cache()
    q, k, v = st.split(st.qkv.cuda())
    w = st.where()
    none = dict(lens=w["lens"][:0], table=w["table"][:0])
    assert kv.attend(q[:0], scale=1.0, **none).shape == (0, 4, 64)
    assert kv.append(k[:0], v[:0], q=q[:0], **none).shape == (0, 4, 64)
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept = torch.full_like(q, 3.0)
    assert bool((kv.attend(q, scale=1.0, cu_rows=cu, out=kept, **none) == 3.0).all())
    ref = kv.attend(q, scale=0.125, **w)
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for _ in range(20):
        for s in side:
            with torch.cuda.stream(s):
                outs.append(kv.attend(q, scale=0.125, **w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_wrong_arguments_are_refused():
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    st = Step([1, 1], [20, 40], 4, 2, 64, 16, 16, BF, seed=23, cu=False)
    kv = st.cache()
    q, k, v = st.split(st.qkv.cuda())
    w = {k_: v_ for k_, v_ in st.where().items() if v_ is not None}
    cs = rope_table(64, 64).cuda()
    bad_append = [dict(k=k.float()), dict(v=v.half()), dict(k=k[:1]), dict(v=v[:, :1]), dict(q=q[:, :3]), dict(q_out=q),
                  dict(q=q, q_out=q[:1]), dict(cos_sin=cs.half()), dict(cos_sin=cs[:, :24].contiguous()),
                  dict(cos_sin=cs.cpu()), dict(lens=w["lens"].long()), dict(lens=w["lens"][:1]), dict(table=w["table"].cpu()),
                  dict(table=w["table"].t()), dict(cu_rows=w["lens"]), dict(k=k.transpose(0, 1)), dict(k=k[..., ::2])]
    for bad in bad_append:
        with pytest.raises(RuntimeError):
            kv.append(**{**dict(k=k, v=v), **w, **bad})
    bad_attend = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:1]), dict(out=q[:1]), dict(out=torch.empty_like(q).half()),
                  dict(window=-1), dict(sink=torch.zeros(3, device="cuda")), dict(sink=torch.zeros(4)), dict(q=q[0]),
                  dict(q=torch.empty(2, 4, 72, dtype=BF, device="cuda")[..., 4:68])]
    for bad in bad_attend:
        with pytest.raises(RuntimeError):
            kv.attend(**{**dict(q=q, scale=1.0), **w, **bad})
    x, wt, s, z = (t.cuda() for t in w4_case(3, 64, 256, 64, True, BF))
    bad_w4 = [dict(x=x.float()), dict(x=x[:, :128]), dict(x=x.repeat(20, 1)), dict(w=wt[:, :64]), dict(w=wt[:50]),
              dict(w=wt.t()), dict(scales=s.half()), dict(scales=s[:, :3]), dict(zeros=z[:, :2]), dict(zeros=z.int()),
              dict(out=torch.empty(3, 63, dtype=BF, device="cuda")), dict(out=torch.empty(64, 3, dtype=BF, device="cuda").t()),
              dict(x=x.t().contiguous().t()), dict(zeros=z.cpu())]
    for bad in bad_w4:
        with pytest.raises(RuntimeError):
            ops.gemv_w4(**{**dict(x=x, w=wt, scales=s, zeros=z), **bad})


def test_attend_long_context_splits():
    """One sequence over many work shares beside short ones, checked against the plain form in fp64 on
    the GPU."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a.paged import PagedKV
    g = torch.Generator(device="cuda").manual_seed(3)
    lens, page, kvh, heads, dim = [70001, 1, 3000], 64, 2, 10, 128
    pages = sum(-(-x // page) for x in lens) + 1
    kv = PagedKV.empty(pages, page, kvh, dim, block=32)
    for c in (kv.k, kv.v):
        c.copy_((torch.randn(c.shape, generator=g, device="cuda") * 100).clamp(-448, 448).to(FP8).view(torch.uint8))
    for c in (kv.k_codes, kv.v_codes):
        c.copy_(torch.randint(118, 122, c.shape, generator=g, device="cuda", dtype=torch.uint8))
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(3, -(-lens[0] // page), dtype=torch.int32, device="cuda")
    at = 0
    for i, x in enumerate(lens):
        table[i, :-(-x // page)] = perm[at:at + -(-x // page)]
        at += -(-x // page)
    q = torch.randn(3, heads, dim, generator=g, device="cuda").to(BF)
    out = kv.attend(q, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), table=table, scale=0.2)
    for i, x in enumerate(lens):
        p = torch.arange(x, device="cuda")
        pg, off = table[i].long()[p // page], p % page
        for h in range(heads):
            j = h // (heads // kvh)
            k = kv.k[pg, j, off].view(FP8).double() * torch.exp2(kv.k_codes[pg, j, off // 32].double() - 127)[:, None]
            v = kv.v[pg, j, off].view(FP8).double() * torch.exp2(kv.v_codes[pg, j, off // 32].double() - 127)[:, None]
            w = torch.softmax(k @ q[i, h].double() * 0.2, 0)
            ref = w @ v
            ds = 2 * (dim + 4) * 2.0 ** -23 * (k.abs() @ q[i, h].double().abs()).max() * 0.2 + 2.0 ** -20 + x * 2.0 ** -23
            tol = half_step(BF) * ref.abs() + (2.0 ** -11 + ds) * (w @ v.abs()) + x * 2.0 ** -32 * 448 * w.max() * 2.0 ** -5
            assert bool(((out[i, h].double() - ref).abs() <= tol).all()), (i, h)


# ------------------------------------------------------------------ together
def test_attention_block_step_by_step():
    """A grouped-query layer's attention block over a few steps, as a server runs it: 4-bit q/k/v
    projection, append with rotation, attention, 4-bit output projection, captured once in a CUDA
    graph and replayed with other rows, lengths and pages; every stage against its plain form on the
    stage's own inputs."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    from sgl_amd_mono_b200.deepseek_v41.sm100a.paged import PagedKV
    g = torch.Generator().manual_seed(21)
    hidden, heads, kvh, dim, page, block, S, per = 256, 4, 2, 64, 32, 16, 3, 2
    T = S * per
    _, wq, sq, zq = w4_case(1, (heads + 2 * kvh) * dim, hidden, 64, True, BF)
    _, wo, so, _ = w4_case(1, hidden, heads * dim, 128, False, BF)
    cs = rope_table(200, dim)
    kv = PagedKV.empty(20, page, kvh, dim, block=block)
    x = torch.zeros(T, hidden, dtype=BF, device="cuda")
    cu = torch.arange(0, T + 1, per, dtype=torch.int32, device="cuda")
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    table = torch.arange(S * 6, dtype=torch.int32, device="cuda").view(S, 6).clone()
    W = [t.cuda() for t in (wq, sq, zq, wo, so, cs)]

    def step():
        qkv = ops.gemv_w4(x, W[0], W[1], W[2])
        q = qkv[:, :heads * dim].view(T, heads, dim)
        k = qkv[:, heads * dim:(heads + kvh) * dim].view(T, kvh, dim)
        v = qkv[:, (heads + kvh) * dim:].view(T, kvh, dim)
        qr = kv.append(k, v, lens=lens, table=table, cu_rows=cu, q=q, cos_sin=W[5], neox=True)
        o = kv.attend(qr, lens=lens, table=table, cu_rows=cu, scale=0.125)
        return qkv, qr, o, ops.gemv_w4(o.view(T, -1), W[3], W[4])

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        outs = step()
    for t in (kv.k, kv.v, kv.k_codes, kv.v_codes):
        t.zero_()
    K, V, KC, VC = (t.cpu() for t in (kv.k, kv.v, kv.k_codes, kv.v_codes))
    now = torch.tensor([0, 30, 60], dtype=torch.int32)  # the cache starts as zeros that count as tokens
    for i in range(12):
        now += per
        tab = torch.randperm(20, generator=g, dtype=torch.int32)[:S * 6].view(S, 6) if i == 0 else tab
        x.copy_(torch.randn(T, hidden, generator=g).to(BF))
        lens.copy_(now)
        table.copy_(tab)
        graph.replay()
        qkv, qr, o, y = (t.cpu() for t in outs)
        w4_check(qkv, x.cpu(), wq, sq, zq)
        q, k, v = (qkv[:, :heads * dim].view(T, heads, dim), qkv[:, heads * dim:(heads + kvh) * dim].view(T, kvh, dim),
                   qkv[:, (heads + kvh) * dim:].view(T, kvh, dim))
        G.append(K, KC, k, cu.cpu(), now, tab, cs, True)
        G.append(V, VC, v, cu.cpu(), now, tab)
        assert torch.equal(kv.k_codes.cpu(), KC) and torch.equal(kv.v_codes.cpu(), VC)
        assert same_bytes(kv.k, K) and same_bytes(kv.v, V)
        assert torch.equal(qr, G.rotate_rows(q, cu.cpu(), now, cs, True, torch.zeros_like(qr)))
        ref, sizes = G.attend(qr, K, V, KC, VC, cu.cpu(), now, tab, 0.125)
        off = ((o.double() - ref).abs() / attn_tol(BF, ref, sizes)).max().item()
        assert off <= 1, off
        w4_check(y, o.reshape(T, -1), wo, so, None)
