"""What the grouped-query operators refuse, and their plain forms' own properties (no GPU needed)."""

import ctypes
import math

import pytest
import torch

from oracle import gqa as G

EINVAL = -1


def _call(fn, a):
    from sgl_amd_mono_b200.common import ext
    f = getattr(ext.lib(), fn)
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
    return f(ctypes.byref(a), None)


# Valid but for one field each: an invalid argument is refused before anything is launched, so the
# pointers are never followed.
P = 1 << 20
W4 = dict(w=P, scales=P, zeros=0, x=P, y=P, M=4, N=64, K=256, group=64, x_ld=256, y_ld=64, f16=0, scratch=P, scratch_bytes=1 << 40)
PAGED = dict(T=4, seqs=2, heads=8, kv_heads=2, dim=64, f16=0, cu_rows=P, lens=P, table=P, table_ld=4, width=4,
             k_cache=P, v_cache=P, k_codes=P, v_codes=P, pages=9, page=32, block=16, q=P, q_ld=512)
APPEND = dict(PAGED, rope=32, neox=1, q_out=P, q_out_ld=512, k=P, k_ld=128, v=P, v_ld=128, cos_sin=P, rope_rows=10)
ATTN = dict(PAGED, out=P, out_ld=512, scale_f32=0, window=0, sink=0, scratch=P, scratch_bytes=1 << 40)

BAD_W4 = [dict(w=0), dict(w=P + 8), dict(scales=0), dict(scales=P + 1), dict(x=0), dict(x=P + 8), dict(y=0),
          dict(y=P + 1), dict(M=0), dict(M=49), dict(N=0), dict(N=1 << 40), dict(group=0), dict(group=48),
          dict(group=-64), dict(K=0), dict(K=320 + 16), dict(K=1 << 40), dict(x_ld=248), dict(x_ld=260), dict(y_ld=63),
          dict(f16=2)]
BAD_PAGED = [dict(T=-1), dict(T=1 << 30), dict(seqs=-1), dict(heads=0), dict(heads=7), dict(kv_heads=0), dict(dim=96),
             dict(dim=0), dict(f16=3), dict(lens=0), dict(lens=P + 2), dict(table=0), dict(table=P + 1),
             dict(cu_rows=P + 2), dict(cu_rows=0), dict(width=0), dict(table_ld=3), dict(width=1 << 30, table_ld=1 << 30),
             dict(pages=0), dict(pages=1 << 40), dict(block=8), dict(block=24), dict(block=0), dict(page=16, block=32),
             dict(page=48, block=32), dict(page=1 << 31), dict(k_cache=0), dict(v_cache=P + 8), dict(k_codes=0),
             dict(v_codes=0), dict(q=P + 8), dict(q_ld=504), dict(q_ld=516)]
BAD_APPEND = [dict(k=0), dict(v=0), dict(k=P + 2), dict(v_ld=120), dict(k_ld=132), dict(q_out=0), dict(q_out=P + 2),
              dict(q_out_ld=500), dict(rope=-16), dict(rope=80), dict(rope=24), dict(neox=2), dict(cos_sin=0),
              dict(cos_sin=P + 4), dict(rope_rows=0)]
BAD_ATTN = [dict(T=1 << 24, heads=1024, q_ld=1 << 20, out_ld=1 << 20), dict(q=0), dict(out=0), dict(out=P + 2), dict(out_ld=504), dict(window=-1), dict(window=1 << 31),
            dict(sink=P + 2)]


@pytest.mark.parametrize("bad", BAD_W4, ids=str)
def test_gemv_w4_refuses(bad):
    from sgl_amd_mono_b200.deepseek_v41.sm100a import abi
    from sgl_amd_mono_b200.common import ext
    a = abi.GemvW4Args(**{**W4, **bad})
    assert _call("dsv41_gemv_w4", a) == EINVAL
    with pytest.raises(ext.ExtError):
        ext.query("dsv41_gemv_w4_scratch_bytes", a)


@pytest.mark.parametrize("bad", BAD_PAGED + BAD_APPEND, ids=str)
def test_kv_append_refuses(bad):
    from sgl_amd_mono_b200.deepseek_v41.sm100a import abi
    assert _call("dsv41_kv_append", abi.KvAppendArgs(**{**APPEND, **bad})) == EINVAL


@pytest.mark.parametrize("bad", BAD_PAGED + BAD_ATTN, ids=str)
def test_paged_attn_refuses(bad):
    from sgl_amd_mono_b200.common import ext
    from sgl_amd_mono_b200.deepseek_v41.sm100a import abi
    a = abi.PagedAttnArgs(**{**ATTN, **bad})
    assert _call("dsv41_paged_attn", a) == EINVAL
    with pytest.raises(ext.ExtError):
        ext.query("dsv41_paged_attn_scratch_bytes", a)


@pytest.mark.parametrize("short", [dict(scratch=0), dict(scratch=P + 8), dict(scratch_bytes=-1)], ids=str)
def test_scratch_that_does_not_do_is_refused(short):
    from sgl_amd_mono_b200.common import ext
    from sgl_amd_mono_b200.deepseek_v41.sm100a import abi
    long = {**ATTN, "width": 1000, "table_ld": 1000}
    assert ext.query("dsv41_paged_attn_scratch_bytes", abi.PagedAttnArgs(**ATTN)) == 0
    assert ext.query("dsv41_paged_attn_scratch_bytes", abi.PagedAttnArgs(**long)) > 0
    assert _call("dsv41_paged_attn", abi.PagedAttnArgs(**{**long, **short})) == -3
    assert ext.query("dsv41_gemv_w4_scratch_bytes", abi.GemvW4Args(**{**W4, "M": 8})) == 0
    small = {**W4, "M": 48, "N": 8191, "K": 4096, "x_ld": 4096, "y_ld": 8192}
    assert ext.query("dsv41_gemv_w4_scratch_bytes", abi.GemvW4Args(**small)) == 0
    big = {**W4, "M": 48, "N": 8192, "K": 4096, "x_ld": 4096, "y_ld": 8192}
    assert ext.query("dsv41_gemv_w4_scratch_bytes", abi.GemvW4Args(**big)) > 0
    assert _call("dsv41_gemv_w4", abi.GemvW4Args(**{**big, **short})) == -3


def test_null_arguments_are_refused():
    from sgl_amd_mono_b200.common import ext
    for fn in ("dsv41_gemv_w4", "dsv41_kv_append", "dsv41_paged_attn"):
        f = getattr(ext.lib(), fn)
        f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
        assert f(None, None) == EINVAL


@pytest.mark.parametrize("empty", [dict(T=0), dict(seqs=0)])
def test_nothing_to_do_is_ok(empty):
    from sgl_amd_mono_b200.deepseek_v41.sm100a import abi
    assert _call("dsv41_kv_append", abi.KvAppendArgs(**{**APPEND, **empty})) == 0
    assert _call("dsv41_paged_attn", abi.PagedAttnArgs(**{**ATTN, **empty})) == 0


def test_wrappers_refuse_host_tensors_and_wrong_forms():
    from sgl_amd_mono_b200.deepseek_v41.sm100a import ops
    from sgl_amd_mono_b200.deepseek_v41.sm100a.paged import PagedKV
    kv = PagedKV.empty(4, 32, 2, 64, device="cpu")
    assert (kv.page, kv.block, kv.kv_heads, kv.dim) == (32, 16, 2, 64)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    lens, table = torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="current CUDA device"):
        kv.append(x, x, lens=lens, table=table)
    with pytest.raises(RuntimeError, match="current CUDA device"):
        kv.attend(x, lens=lens, table=table, scale=1.0)
    with pytest.raises(RuntimeError, match="current CUDA device"):
        ops.gemv_w4(x[0], torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="want matrices"):
        ops.gemv_w4(x, torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 1, dtype=torch.bfloat16))
    for bad in (dict(dim=96), dict(block=8), dict(page=40), dict(page=16, block=32)):
        with pytest.raises(RuntimeError, match="PagedKV"):
            PagedKV.empty(**{**dict(pages=4, page=32, kv_heads=2, dim=64, device="cpu"), **bad})
    u8 = torch.zeros(4, 2, 32, 64, dtype=torch.uint8)
    codes = torch.zeros(4, 2, 2, dtype=torch.uint8)
    for args in ((u8, u8[:3], codes, codes), (u8, u8, codes, codes[:, :1]), (u8.float(), u8, codes, codes),
                 (u8.transpose(1, 2), u8, codes, codes), (u8[0], u8, codes, codes)):
        with pytest.raises(RuntimeError, match="PagedKV"):
            PagedKV(*args)


def test_plain_append_is_within_half_a_step():
    """The plain form's values against 64 bits: e4m3 under the block's scale is off by at most half a
    step, 2^-4 of a normal value and 2^-10 scales of a smaller one."""
    g = torch.Generator().manual_seed(0)
    rows, dim = 40, 64
    cache, codes = torch.zeros(2, 1, 32, dim, dtype=torch.uint8), torch.zeros(2, 1, 2, dtype=torch.uint8)
    x = torch.randn(rows, 1, dim, generator=g).to(torch.bfloat16)
    ang = torch.arange(64)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2) / dim)
    cs = torch.cat([ang.cos(), ang.sin()], 1).float()
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    G.append(cache, codes, x, [0, rows], [rows], table, cs, True)
    for p in range(rows):
        a, b = x[p, 0, :32].double(), x[p, 0, 32:].double()
        c, s = cs[p, :32].double(), cs[p, 32:].double()
        want = torch.cat([a * c - b * s, a * s + b * c])
        pg, off = int(table[0, p // 32]), p % 32
        scale = 2.0 ** (int(codes[pg, 0, off // 16]) - 127)
        got = cache[pg, 0, off].view(G.FP8).double() * scale
        tol = torch.maximum(want.abs() * 2.0 ** -4, torch.tensor(scale * 2.0 ** -10)) + 2.0 ** -22
        assert bool(((got - want).abs() <= tol).all())
        assert want.abs().max() <= 448 * scale * (1 + 2.0 ** -20)


def test_plain_attention_masks():
    """Nothing visible gives zeros, a window of one key gives that key's value, and a sink takes its share."""
    g = torch.Generator().manual_seed(1)
    k, v = (G.to_bytes(torch.randn(2, 1, 16, 64, generator=g) * 50) for _ in range(2))
    codes = torch.full((2, 1, 1), 120, dtype=torch.uint8)
    q = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16)
    table = torch.tensor([[1], [0]], dtype=torch.int32)
    out, _ = G.attend(q, k, v, codes, codes, None, [0, 9], table, 0.1, window=1)
    assert bool((out[0] == 0).all())
    assert torch.equal(out[1, 0], v[0, 0, 8].view(G.FP8).double() * 2.0 ** -7)
    z = (k[0, 0, 8].view(G.FP8).double() * 2.0 ** -7 @ q[1].double().T) * 0.1
    sunk, _ = G.attend(q, k, v, codes, codes, None, [0, 9], table, 0.1, window=1, sink=torch.tensor([0.5, 0.5]))
    share = 1 / (1 + math.exp(0.5 - z[0].item()))
    assert torch.allclose(sunk[1, 0], out[1, 0] * share, rtol=1e-12)


def test_a_cache_stays_with_its_tensors():
    """Copies address their own tensors; tensors cannot be replaced, and a moved one is refused."""
    import copy
    import io

    from sgl_amd_mono_b200.deepseek_v41.sm100a import abi
    from sgl_amd_mono_b200.deepseek_v41.sm100a.paged import PagedKV

    def addresses(kv):
        both = [t.from_buffer_copy(b) for t, b in ((abi.KvAppendArgs, kv._append_args), (abi.PagedAttnArgs, kv._attend_args))]
        return [[getattr(a, n) for n in ("k_cache", "v_cache", "k_codes", "v_codes")] for a in both]

    def own(kv):
        return [[t.data_ptr() for t in (kv.k, kv.v, kv.k_codes, kv.v_codes)]] * 2

    kv = PagedKV.empty(4, 32, 2, 64, device="cpu")
    kv.k[1, 0, 2, 3] = 7
    buf = io.BytesIO()
    torch.save(kv, buf)
    deep, shallow, saved = copy.deepcopy(kv), copy.copy(kv), torch.load(io.BytesIO(buf.getvalue()), weights_only=False)
    for c in (kv, deep, shallow, saved):
        assert addresses(c) == own(c) and (c.pages, c.page, c.block, c.kv_heads, c.dim) == (4, 32, 16, 2, 64)
        assert int(c.k[1, 0, 2, 3]) == 7
    assert shallow.k is kv.k and len({c.k.data_ptr() for c in (kv, deep, saved)}) == 3
    for name in ("k", "v", "k_codes", "v_codes"):
        with pytest.raises(AttributeError):
            setattr(kv, name, getattr(deep, name))
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    where = dict(lens=torch.ones(1, dtype=torch.int32), table=torch.zeros(1, 1, dtype=torch.int32))
    args = abi.KvAppendArgs()
    kv._step(args, x, "k", where["lens"], where["table"], None)
    assert args.T == 1
    for name, t in (("k", kv.k), ("v_codes", kv.v_codes)):
        moved = copy.deepcopy(kv)
        getattr(moved, name).set_(t.clone())
        with pytest.raises(RuntimeError, match="moved"):
            moved._step(abi.KvAppendArgs(), x, "k", where["lens"], where["table"], None)
