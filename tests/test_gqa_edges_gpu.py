"""The grouped-query operators where their first tests do not reach: instances of the kernels that
other sizes choose, the ends of the accepted ranges, the precision of the attention's weights."""

import copy
import math

import pytest
import torch

from oracle import gqa as G
from test_gqa_gpu import BF, HF, Step, attn_tol, half_step, rope_table, run_append, run_attend, same_bytes, w4_case, w4_check

pytestmark = pytest.mark.gpu


def attend_both(st, scale, window=0, sink=None, rows_out=None):
    """The attention with the step's own table and with one so wide that the work is split and joined;
    the rows and with them the kernel's instance stay."""
    kv, where = st.cache(), st.where()
    q = st.split(st.qkv.cuda())[0]
    wide = torch.full((len(st.rows), 4000), -1, dtype=torch.int32, device="cuda")
    wide[:, :st.table.shape[1]] = where["table"]
    sink = None if sink is None else sink.cuda()
    return [kv.attend(q, scale=scale, window=window, sink=sink, **{**where, "table": t}).cpu()
            for t in (where["table"], wide)]


# (dim, query heads a kv head): with one row a sequence 8, 16, 24 and 32 columns together
INSTANCES = [(64, 4), (64, 12), (64, 20), (64, 32), (128, 8), (128, 12), (128, 20), (128, 32), (256, 5), (256, 16)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("dim,group", INSTANCES)
def test_attend_weights_keep_fp32(dim, group, dt):
    """The weights enter the second product with fp32's precision. Queries of one dim that is not zero
    make every score a single product, so nothing else is off by more than this bound:

    * an exponent: the score's rounding (1.5 steps of 2^-24 of at most 8), two additions of the
      references and scales (2^-24 of at most 32 each), as much once more for the sum, ex2's 2^-22
      where a weight, a term of the sum or a factor between references is made: 2^-17 in all
    * a weight: head and tail in f16 leave 2^-22 of it, and 2^-32 of the largest where the tail ends
    * fp32 sums: at most 3 tiles a warp, 17 additions for each product of head and of tail, then the
      joins of 12 warps and 4 pieces: 120 additions, each off by a step (2^-23) of sum p |v| at most
    * the factor and its quotient: 2^-22 of the value; and the output's rounding
    """
    st = Step([1, 1, 1, 1], [300, 40, 17, 0], 2 * group, 2, dim, 32, 16, dt, seed=31)
    q = st.split(st.qkv)[0]
    keep = q[..., 5].clone()
    q.zero_()
    q[..., 5] = keep
    ref, (vabs, sabs, top, seen) = G.attend(q, st.k, st.v, st.kc, st.vc, st.cu, st.lens, st.table, 1 / 16)
    assert sabs.max().item() * 1.4427 < 8
    tol = (half_step(dt) + 2.0 ** -22) * ref.abs() + (2.0 ** -17 + 2.0 ** -22 + 120 * 2.0 ** -23) * vabs \
        + (seen * 2.0 ** -32 * 448 * top)[..., None]
    tol = tol + 2.0 ** -25 if dt == HF else tol
    for o in attend_both(st, 1 / 16):
        off = ((o.double() - ref).abs() / tol.clamp_min(1e-30)).max().item()
        assert off <= 1, off


def test_a_snapshot_of_the_cache_is_its_own():
    """What is appended to a deep copy leaves the cache that it was taken of as it was."""
    st = Step([3, 1], [40, 20], 4, 2, 64, 16, 16, BF, seed=32)
    kv = st.cache()
    snap = copy.deepcopy(kv)
    q, k, v = st.split(st.qkv.cuda())
    w = st.where()
    before = kv.attend(q, scale=0.125, **w)
    snap.append(k, v, **w)
    for a, b in ((kv.k, st.k), (kv.v, st.v), (kv.k_codes, st.kc), (kv.v_codes, st.vc)):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(kv.attend(q, scale=0.125, **w), before)
    kv.append(k, v, **w)
    assert torch.equal(kv.k, snap.k) and torch.equal(kv.v_codes, snap.v_codes)
    assert torch.equal(kv.attend(q, scale=0.125, **w), snap.attend(q, scale=0.125, **w))


@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 8, (1 << 31) - 1])
@pytest.mark.parametrize("rows,lens", [([6, 2], [3, 2]), ([6, 1], [0, 1]), ([9, 3], [8, 50])])
def test_attend_windows_up_to_the_last(window, rows, lens):
    """A window that no sequence fills is none, with more rows than tokens too."""
    st = Step(rows, lens, 4, 2, 64, 16, 16, BF, seed=33)
    a, b = attend_both(st, 0.125)
    c, d = attend_both(st, 0.125, window=window)
    assert torch.equal(a, c) and torch.equal(b, d)
    ref, sizes = G.attend(st.split(st.qkv)[0], st.k, st.v, st.kc, st.vc, st.cu, st.lens, st.table, 0.125, window)
    assert bool(((c.double() - ref).abs() <= attn_tol(BF, ref, sizes)).all()) and bool(c.any())


def test_attend_negative_lengths_see_nothing():
    """A length below zero holds no token, whatever its size."""
    st = Step([2, 1, 3], [0, 20, 0], 4, 2, 64, 16, 16, BF, seed=34)
    st.lens[0], st.lens[2] = -5, -(1 << 31)
    for window in (0, 7, (1 << 31) - 1):
        for o in attend_both(st, 0.125, window=window):
            assert not bool(o[:2].any()) and not bool(o[3:].any()) and bool(o[2].any())


@pytest.mark.parametrize("M,N,K,group", [(1, 300, 1024, 64), (5, 9000, 512, 128), (12, 300, 2080, 32), (1, 64, 32768, 256),
                                         (20, 9000, 4096, 64)])
@pytest.mark.parametrize("e", [-100, -90, 90, 100, 126])
def test_w4_scales_to_the_ends_of_bf16(M, N, K, group, e):
    """Scales and activations whose products stay in range, each near an end of its own."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(M, N, K, group, True, BF, seed=35)
    s = s.float().clamp(-0.9, 0.9)
    s, x = (s * 2.0 ** e).to(BF), (x.float() * 2.0 ** max(-50, min(50, -e // 2))).to(BF)
    assert bool(torch.isfinite(s).all())
    w4_check(ops.gemv_w4(x.cuda(), w.cuda(), s.cuda(), z.cuda()), x, w, s, z)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,N,K,group", [(1, 300, 1024, 128), (5, 333, 416, 32), (13, 2311, 4000, 32), (48, 2311, 1056, 96),
                                         (20, 9000, 4096, 64)])
def test_w4_weights_at_their_zero_point(M, N, K, group, dt):
    """Rows and groups whose weights all equal the zero point: their terms are 0 within the contract's
    bound, sum |x| (n + z) |s| times the additions' steps."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(M, N, K, group, True, dt, seed=38)
    z2 = z[:, :, None].expand(-1, -1, group // 2).reshape(N, -1)
    at = (z2 | z2 << 4).to(torch.uint8)
    w[::3] = at[::3]
    w[1::3, :group // 2] = at[1::3, :group // 2]
    y = ops.gemv_w4(x.cuda(), w.cuda(), s.cuda(), z.cuda()).cpu().double()
    wd = G.w4_dequant(w, s, z)
    ref = x.double() @ wd.T
    assert bool((ref[:, ::3] == 0).all())
    n = torch.stack([w & 15, w >> 4], -1).reshape(N, -1, group).double()
    size = x.double().abs() @ ((n + z.double()[:, :, None]) * s.double().abs()[:, :, None]).reshape(N, -1).T
    tol = half_step(dt) * ref.abs() + (K / 8 + 32) * 2.0 ** -23 * size + (2.0 ** -25 if dt == HF else 0)
    off = ((y - ref).abs() / tol.clamp_min(1e-300)).max().item()
    assert off <= 1, off


@pytest.mark.parametrize("M,N,K,group", [(1, 300, 1024, 64), (12, 300, 2080, 32), (20, 9000, 4096, 64)])
@pytest.mark.parametrize("e", [-50, -64, -80])
def test_w4_small_activations(M, N, K, group, e):
    """Activations of 2^-50 and less: the sums keep an absolute 2^-80 a term (the smallest fp32 number,
    2^-149, times the 2^69 by which bf16 nibbles and activations are scaled)."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(M, N, K, group, True, BF, seed=39)
    x = (x.float() * 2.0 ** e).to(BF)
    y = ops.gemv_w4(x.cuda(), w.cuda(), s.cuda(), z.cuda()).cpu().double()
    wd = G.w4_dequant(w, s, z)
    ref, size = x.double() @ wd.T, x.double().abs() @ wd.abs().T
    zs = s.double().abs().sum(1) * group
    tol = half_step(BF) * ref.abs() + (K / 8 + 32) * 2.0 ** -23 * size + 17 * 2.0 ** -80 * zs
    off = ((y - ref).abs() / tol).max().item()
    assert off <= 1, off


def test_w4_takes_an_empty_step():
    """No rows give an empty output, as the cache's two operators take them."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = (t.cuda() for t in w4_case(3, 64, 256, 64, True, BF))
    y = ops.gemv_w4(x[:0], w, s, z)
    assert y.shape == (0, 64) and y.dtype == BF and y.is_cuda
    out = torch.empty(0, 64, dtype=BF, device="cuda")
    assert ops.gemv_w4(x[:0], w, s, z, out=out) is out
    for bad in (dict(w=w[:50]), dict(scales=s.half()), dict(zeros=z.int()), dict(out=torch.empty(3, 64, dtype=BF, device="cuda")),
                dict(x=x[:0].float())):
        with pytest.raises(RuntimeError):
            ops.gemv_w4(**{**dict(x=x[:0], w=w, scales=s, zeros=z), **bad})


@pytest.mark.parametrize("neox,in_place", [(False, True), (True, False)])
def test_append_prompts_take_four_heads_a_thread(neox, in_place):
    """Enough rows that a thread rotates four query heads, the last one of ten two; a sequence without
    rows and rows behind the last sequence."""
    rows = [1500, 0, 1701, 1, 700]
    st = Step(rows, [1500, 5, 1800, 40, 733], 10, 2, 128, 64, 16, BF, seed=36, tail=3)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert (sum(rows) + 3) * 10 * 128 // 16 >= sms * 2048
    kv, qkv = st.cache(), st.qkv.cuda()
    q, k, v = st.split(qkv)
    cs = rope_table(1800, 128)
    got = kv.append(k, v, q=q, cos_sin=cs.cuda(), neox=neox, q_out=q if in_place else None, **st.where())
    qc, kc, vc = st.split(st.qkv)
    G.append(st.k, st.kc, kc, st.cu, st.lens, st.table, cs, neox)
    G.append(st.v, st.vc, vc, st.cu, st.lens, st.table)
    assert torch.equal(kv.k_codes.cpu(), st.kc) and torch.equal(kv.v_codes.cpu(), st.vc)
    assert same_bytes(kv.k, st.k) and same_bytes(kv.v, st.v)
    used = sum(rows)
    want = G.rotate_rows(qc, st.cu, st.lens, cs, neox, torch.zeros(qc.shape, dtype=BF))
    assert torch.equal(got[:used].cpu(), want[:used])
    if in_place:
        assert torch.equal(qkv[used:].cpu(), st.qkv[used:]) and torch.equal(qkv[:, 10 * 128:].cpu(), st.qkv[:, 10 * 128:])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("code", [0, 1, 4, 8, 12])
def test_attend_small_values_everywhere(code, dim):
    """Every value under a scale near the smallest that E8M0 holds: bf16 outputs hold them still."""
    st = Step([1, 1], [300, 21], 2, 1, dim, 16, 16, BF, seed=37)
    st.vc.fill_(code)
    ref, sizes = G.attend(st.split(st.qkv)[0], st.k, st.v, st.kc, st.vc, st.cu, st.lens, st.table, 0.125)
    for o in attend_both(st, 0.125):
        # (and half a step of bf16 below its smallest normal number)
        assert bool(((o.double() - ref).abs() <= attn_tol(BF, ref, sizes) + 2.0 ** -134).all())


def test_scales_that_fp32_does_not_hold_are_refused():
    st = Step([1], [20], 4, 2, 64, 16, 16, BF, seed=46, cu=False)
    kv, w = st.cache(), st.where()
    q = st.split(st.qkv.cuda())[0]
    for scale in (1e39, -1e300, "1", None):
        for x, where in ((q, w), (q[:0], dict(lens=w["lens"][:0], table=w["table"][:0]))):
            with pytest.raises(RuntimeError, match="scale"):
                kv.attend(x, scale=scale, **where)
    assert torch.equal(kv.attend(q, scale=0.125, **w), kv.attend(q, scale=torch.tensor(0.125), **w))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("dim,group", INSTANCES)
def test_attend_every_instance_whole_and_split(dim, group, dt):
    st = Step([1, 1, 1, 1], [777, 0, 131, 16], group * 2, 2, dim, 32, 16, dt, seed=41)
    sink = torch.randn(st.heads, generator=st.g)
    for window, sk in ((0, None), (200, sink)):
        ref, sizes = G.attend(st.split(st.qkv)[0], st.k, st.v, st.kc, st.vc, st.cu, st.lens, st.table, dim ** -0.5, window, sk)
        for o in attend_both(st, dim ** -0.5, window, sk):
            assert bool(((o.double() - ref).abs() <= attn_tol(dt, ref, sizes)).all())


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows,heads,kvh", [([6, 6, 6], 8, 2), ([3, 0, 9], 8, 2), ([5, 5], 12, 4), ([2, 7, 3], 6, 1)])
def test_attend_verify_rows_split(rows, heads, kvh, dt):
    """Rows of several tokens over 9 to 32 columns, whole and split."""
    st = Step(rows, [500, 77, 260][:len(rows)], heads, kvh, 128, 32, 16, dt, seed=42)
    ref, sizes = G.attend(st.split(st.qkv)[0], st.k, st.v, st.kc, st.vc, st.cu, st.lens, st.table, 0.1)
    for o in attend_both(st, 0.1):
        assert bool(((o.double() - ref).abs() <= attn_tol(dt, ref, sizes)).all())


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group", [
    (48, 8200, 4096, 128), (33, 9000, 4096, 256), (32, 8200, 4096, 32), (17, 8300, 4224, 32), (1, 8192, 4096, 32),
    (8, 300, 8192, 32), (2, 5000, 16384, 128), (3, 200, 16384, 256), (4, 130, 32768, 64), (16, 200, 16384, 128)])
def test_w4_every_instance(M, N, K, group, zeros, dt):
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = (None if t is None else t.cuda() for t in w4_case(M, N, K, group, zeros, dt, seed=43))
    w4_check(ops.gemv_w4(x, w, s, z), x, w, s, z)


def test_w4_non_finite_stays_in_its_row_and_column_of_a_large_matrix():
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    x, w, s, z = w4_case(20, 9000, 4096, 64, True, BF, seed=44)
    x[1, 100], x[7, 4000] = float("inf"), float("nan")
    s[8999, 3] = float("nan")
    y = ops.gemv_w4(x.cuda(), w.cuda(), s.cuda(), z.cuda()).cpu()
    bad, want = ~torch.isfinite(y), torch.zeros(20, 9000, dtype=torch.bool)
    want[1], want[7], want[:, 8999] = True, True, True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("dim,rope", [(128, 128), (256, 256), (128, 64), (256, 16)])
def test_append_rotates_whole_and_part_heads(dim, rope, neox, dt):
    st = Step([3, 0, 20, 1], [40, 9, 77, 48], 6, 2, dim, 32, 16, dt, seed=45, tail=2)
    run_append(st, rope=rope, neox=neox, in_place=not neox)


@pytest.mark.parametrize("M,group,zeros,dt", [(1, 128, True, BF), (7, 64, False, HF), (20, 64, True, HF)])
def test_w4_weights_past_four_gigabytes(M, group, zeros, dt):
    """More weights than 32 bits of bytes: the last and the first rows against 64 bits."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    N, K = 530003, 16384
    assert N * K // 2 > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(47)
    w = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand(N, K // group, generator=g, device="cuda") * 0.02 + 1e-3).to(dt)
    z = torch.randint(0, 16, (N, K // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    x = torch.randn(M, K, generator=g, device="cuda").to(dt)
    y = ops.gemv_w4(x, w, s, z)
    for part in (slice(0, 600), slice(N // 2, N // 2 + 300), slice(N - 600, N)):
        w4_check(y[:, part], x, w[part], s[part], None if z is None else z[part])


def test_append_positions_past_the_angles_read_the_last_row():
    st = Step([3, 0, 20, 1], [40, 9, 77, 48], 6, 2, 128, 32, 16, BF, seed=48)
    cs = rope_table(45, 128)
    kv, w = st.cache(), st.where()
    q, k, v = st.split(st.qkv.cuda())
    got = kv.append(k, v, q=q, cos_sin=cs.cuda(), neox=True, **w)
    qc, kc, vc = st.split(st.qkv)
    G.append(st.k, st.kc, kc, st.cu, st.lens, st.table, cs, True)
    assert torch.equal(kv.k_codes.cpu(), st.kc) and same_bytes(kv.k, st.k)
    assert torch.equal(got.cpu(), G.rotate_rows(qc, st.cu, st.lens, cs, True, torch.zeros(qc.shape, dtype=BF)))


def test_calls_of_two_streams_and_two_graphs_at_once():
    """The large products, whose scratch and TMEM are a call's own, and the split attention: eager on two
    streams together, then two captured graphs replayed together."""
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    st = Step([1, 1], [3000, 70], 16, 2, 128, 32, 16, BF, seed=49)
    kv, where = st.cache(), st.where()
    q = st.split(st.qkv.cuda())[0]
    cases = [tuple(t.cuda() for t in w4_case(20, 9000, 4096, 64, True, BF, seed=s)) for s in (50, 51)]

    def calls(i):
        return ops.gemv_w4(*cases[i]), kv.attend(q, scale=0.05 * (i + 1), **where), ops.gemv_w4(*cases[1 - i])

    ref = [calls(0), calls(1)]
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(side):
            with torch.cuda.stream(s):
                got[i].append(calls(i))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in side]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g, stream=side[i]):
            got[i].append(calls(i))
    for _ in range(10):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for r, outs in zip(ref, got):
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(r, o))
    from sgl_amd_mono_b200.common import ext
    assert ext.lib().dsv41_device_error() == 0
