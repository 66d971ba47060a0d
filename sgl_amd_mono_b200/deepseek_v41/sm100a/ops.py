"""Thin torch-facing wrappers of single C-ABI launches (tests and the runner use them)."""

from __future__ import annotations

import torch

from ...common import ext
from . import abi
from .paged import current_stream

W4_MAX_ROWS = 48  # of gemv_w4


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def gemv_fp8(x: torch.Tensor, w: torch.Tensor, codes: torch.Tensor, x_group_rows: int = 0,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 [M, N] = x (bf16 [M, >= K]) . dequant(W e4m3 [N, K], E8M0 128 x 128 codes)^T."""
    M, N, K = x.shape[0], w.shape[0], w.shape[1]
    y = out if out is not None else torch.empty(M, N, dtype=torch.float32, device=w.device)
    a = abi.GemvArgs(w=_ptr(w), codes=_ptr(codes), x=_ptr(x), y=_ptr(y), M=M, N=N, K=K,
                     x_ld=x.stride(0), x_group_rows=x_group_rows, scratch=0, scratch_bytes=0)
    need = ext.query("dsv41_gemv_fp8_scratch_bytes", a)
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device=w.device)
    a.scratch, a.scratch_bytes = _ptr(scratch), need
    ext.call("dsv41_gemv_fp8", a, _stream())
    return y


def gemv_w4(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, N] of x's type = x (bf16 or f16 [M, K], M from 0 to 48) . dequant(w)^T, with w 4-bit values
    [N, K / 2] (even k in the low nibble), read in place, minus ``zeros`` (u8 [N, K / group]; 8
    without them), times ``scales`` ([N, K / group] of x's type); group a multiple of 32. fp32 sums
    whose error goes by sum |x| (w + zero) |scale|; bf16 x below 2^63 in magnitude."""
    if x.dim() != 2 or w.dim() != 2 or scales.dim() != 2:
        raise RuntimeError(f"gemv_w4: x {tuple(x.shape)}, w {tuple(w.shape)}, scales {tuple(scales.shape)}: want matrices")
    dev, dtype = x.get_device(), x.dtype
    stream = current_stream(dev, "gemv_w4")
    (M, K), (N, groups), x_at, w_at = x.shape, scales.shape, x.data_ptr(), w.data_ptr()
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise RuntimeError(f"gemv_w4: x of {dtype}, want bfloat16 or float16")
    if M > W4_MAX_ROWS or not N or not groups or K % groups or K // groups % 32:
        raise RuntimeError(f"gemv_w4: {M} rows of {K} in {groups} groups, {N} outputs: at most {W4_MAX_ROWS} rows, groups "
                           "a multiple of 32")
    if w.shape != (N, K // 2) or w.dtype is not torch.uint8 or w.get_device() != dev or not w.is_contiguous() or w_at & 15:
        raise RuntimeError(f"gemv_w4: w {tuple(w.shape)} {w.dtype} on {w.device}: want contiguous, 16-byte aligned "
                           f"[{N}, {K // 2}] uint8 on {x.device}")
    if scales.dtype is not dtype or scales.get_device() != dev or not scales.is_contiguous():
        raise RuntimeError(f"gemv_w4: scales of {scales.dtype} on {scales.device}: want contiguous {dtype} on {x.device}")
    x_ld, one = x.stride()
    if M < 2:
        x_ld = K
    if one != 1 or x_ld & 7 or x_ld < K or x_at & 15:
        raise RuntimeError(f"gemv_w4: x strides {x.stride()} at {x_at:#x}: want contiguous rows a multiple of 8 values "
                           "apart, 16-byte aligned")
    a = abi.GemvW4Args(w_at, scales.data_ptr(), 0, x_at, 0, M, N, K, K // groups, x_ld, N, dtype is torch.float16)
    if zeros is not None:
        if zeros.shape != (N, groups) or zeros.dtype is not torch.uint8 or zeros.get_device() != dev \
                or not zeros.is_contiguous():
            raise RuntimeError(f"gemv_w4: zeros {tuple(zeros.shape)} {zeros.dtype} on {zeros.device}: want [{N}, {groups}] "
                               f"uint8 on {x.device}")
        a.zeros = zeros.data_ptr()
    if out is None:
        out = x.new_empty((M, N))
    else:
        y_ld, one = out.stride() if out.dim() == 2 else (0, 0)
        if M < 2:
            y_ld = N
        if out.shape != (M, N) or out.dtype is not dtype or out.get_device() != dev or (N > 1 and one != 1) or y_ld < N:
            raise RuntimeError(f"gemv_w4: out {tuple(out.shape)} {out.dtype} on {out.device} of strides {out.stride()}: "
                               f"want [{M}, {N}] {dtype} on {x.device}, contiguous rows")
        a.y_ld = y_ld
    if not M:
        return out
    a.y = out.data_ptr()
    if M > 8 and N * K >= 1 << 25:  # fewer rows and smaller matrices need no scratch
        need = ext.query("dsv41_gemv_w4_scratch_bytes", a)
        if need:
            scratch = w.new_empty((need,))
            a.scratch, a.scratch_bytes = scratch.data_ptr(), need
    ext.call("dsv41_gemv_w4", a, stream)
    return out
