"""The grouped-query decode operators in plain form (CPU): 4-bit products and attention in 64 bits,
the paged cache's append in the fp32 steps that its contract fixes bit for bit.

No counterpart in the reference; the formulas are those of the C header.
"""

from __future__ import annotations

import math

import torch

FP8 = torch.float8_e4m3fn


def w4_dequant(w: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None) -> torch.Tensor:
    """[N, K] fp64 of packed 4-bit values (even k in the low nibble)."""
    n, groups = scales.shape
    v = torch.stack([w & 15, w >> 4], -1).reshape(n, groups, -1).double()
    z = 8.0 if zeros is None else zeros.double()[:, :, None]
    return ((v - z) * scales.double()[:, :, None]).reshape(n, -1)


def rotate(x: torch.Tensor, pos: int, cos_sin: torch.Tensor | None, neox: bool) -> torch.Tensor:
    """[heads, dim] fp32 rotated at a position, every product and sum rounded in fp32."""
    x = x.float().clone()
    if cos_sin is None:
        return x
    r, d = cos_sin.shape[1], x.shape[-1]
    row = cos_sin[min(max(pos, 0), cos_sin.shape[0] - 1)]
    j = torch.arange(r // 2)
    a, b = (d - r + j, d - r // 2 + j) if neox else (d - r + 2 * j, d - r + 2 * j + 1)
    c, s = row[:r // 2], row[r // 2:]
    xa, xb = x[..., a], x[..., b]
    x[..., a], x[..., b] = xa * c - xb * s, xa * s + xb * c
    return x


def code_of(amax: torch.Tensor) -> torch.Tensor:
    """E8M0 code of the smallest power of two not below max(amax, 1e-4) / 448."""
    bits = (amax.clamp(1e-4, torch.finfo(torch.float32).max) / 448.0).view(torch.int32)
    return ((bits >> 23) & 255) + ((bits & 0x7fffff) != 0).int()


def pow2(e: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def to_bytes(x: torch.Tensor) -> torch.Tensor:
    return x.clamp(-448.0, 448.0).to(FP8).view(torch.uint8)


def spans(cu_rows, lens):
    """(sequence, its first row, its rows, its tokens) of every sequence that has rows."""
    cu = list(range(len(lens) + 1)) if cu_rows is None else [int(x) for x in cu_rows]
    return [(s, cu[s], cu[s + 1] - cu[s], int(lens[s])) for s in range(len(lens)) if cu[s + 1] > cu[s]]


def page_of(table, s: int, p: int, page: int, pages: int) -> int:
    if p < 0 or p // page >= table.shape[1]:
        return -1
    pg = int(table[s, p // page])
    return pg if 0 <= pg < pages else -1


def append(cache, codes, x, cu_rows, lens, table, cos_sin=None, neox=False) -> None:
    """Rows x [T, heads, dim] into cache [pages, heads, page, dim] u8 / codes [pages, heads, page / block]."""
    pages, _, page, _ = cache.shape
    block = page // codes.shape[2]
    for s, r0, n, length in spans(cu_rows, lens):
        first = length - n
        for b in range(max(first, 0) // block, -(-min(length, table.shape[1] * page) // block)):
            new = range(max(first, b * block, 0), min(length, (b + 1) * block))
            pg = page_of(table, s, b * block, page, pages)
            if pg < 0 or not len(new):
                continue
            y = torch.stack([rotate(x[r0 + p - first], p, cos_sin, neox) for p in new], 1)  # [heads, tokens, dim]
            amax = torch.nan_to_num(y.abs(), nan=0.0, posinf=math.inf).amax((1, 2))
            code = code_of(amax)
            o, old = b * block % page, new[0] - b * block
            if old:
                was = codes[pg, :, o // block].int()
                code = torch.maximum(code, was)
                part = cache[pg, :, o:o + old].view(FP8).float()
                cache[pg, :, o:o + old] = to_bytes(part * pow2((was - code).clamp_min(-140))[:, None, None])
            codes[pg, :, o // block] = code.to(torch.uint8)
            cache[pg, :, o + old:o + old + len(new)] = to_bytes(y * pow2(127 - code)[:, None, None])


def rotate_rows(q, cu_rows, lens, cos_sin, neox, out):
    """The rotated queries of every row that belongs to a sequence, rounded to out's type."""
    for _, r0, n, length in spans(cu_rows, lens):
        for j in range(n):
            out[r0 + j] = rotate(q[r0 + j], length - n + j, cos_sin, neox).to(out.dtype)
    return out


def attend(q, k, v, k_codes, v_codes, cu_rows, lens, table, scale, window=0, sink=None):
    """(out [T, heads, dim] fp64, an error bound's sizes per row and head: sum p |v| [.., dim], the
    largest |scale| sum |q||k|, the largest p times its value's scale, the keys seen)."""
    pages, kvh, page, dim = k.shape
    block = page // k_codes.shape[2]
    heads = q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    vabs, sabs = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64)
    top, seen = torch.zeros_like(sabs), torch.zeros_like(sabs)
    for s, r0, n, length in spans(cu_rows, lens):
        for j in range(n):
            vis = length - n + j + 1
            lo = max(0, vis - window) if window else 0
            keys = torch.arange(lo, max(lo, min(vis, table.shape[1] * page)))
            pg = table[s, keys // page].long()
            keys, pg = keys[(pg >= 0) & (pg < pages)], pg[(pg >= 0) & (pg < pages)]
            if not len(keys):
                continue
            off = keys % page
            for h in range(heads):
                g = h // (heads // kvh)
                kk = k[pg, g, off].view(FP8).double() * torch.exp2(k_codes[pg, g, off // block].double() - 127)[:, None]
                vs = torch.exp2(v_codes[pg, g, off // block].double() - 127)
                vv = v[pg, g, off].view(FP8).double() * vs[:, None]
                z = kk @ q[r0 + j, h].double() * scale
                if sink is not None:
                    z = torch.cat([z, sink[h].double().view(1)])
                p = torch.softmax(z, 0)[:len(keys)]
                out[r0 + j, h] = p @ vv
                vabs[r0 + j, h] = p @ vv.abs()
                sabs[r0 + j, h] = (kk.abs() @ q[r0 + j, h].double().abs()).max() * abs(scale)
                top[r0 + j, h] = (p * vs).max()
                seen[r0 + j, h] = len(keys)
    return out, (vabs, sabs, top, seen)
