"""Thin torch-facing wrappers of single C-ABI launches (tests and the runner use them)."""

from __future__ import annotations

import torch

from ...common import ext
from . import abi
from .paged import check_device

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
    """[M, N] of x's type = x (bf16 or f16 [M, K], M <= 48) . dequant(w)^T, with w 4-bit values
    [N, K / 2] (even k in the low nibble), read in place, minus ``zeros`` (u8 [N, K / group]; 8
    without them), times ``scales`` ([N, K / group] of x's type); group a multiple of 32."""
    if x.dim() != 2 or w.dim() != 2 or scales.dim() != 2:
        raise RuntimeError(f"gemv_w4: x {tuple(x.shape)}, w {tuple(w.shape)}, scales {tuple(scales.shape)}: want matrices")
    (M, K), N, groups = x.shape, w.shape[0], scales.shape[1]
    dev = x.device
    check_device(dev, "gemv_w4")
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float16:
        raise RuntimeError(f"gemv_w4: x of {x.dtype}, want bfloat16 or float16")
    if not 1 <= M <= W4_MAX_ROWS or not N or not groups or K % groups or K // groups % 32:
        raise RuntimeError(f"gemv_w4: {M} rows of {K} in {groups} groups, {N} outputs: at most {W4_MAX_ROWS} rows, groups "
                           "a multiple of 32")
    if w.shape[1] * 2 != K or w.dtype != torch.uint8 or w.device != dev or not w.is_contiguous() or w.data_ptr() % 16:
        raise RuntimeError(f"gemv_w4: w {tuple(w.shape)} {w.dtype} on {w.device}: want contiguous, 16-byte aligned "
                           f"[{N}, {K // 2}] uint8 on {dev}")
    if scales.shape[0] != N or scales.dtype != x.dtype or scales.device != dev or not scales.is_contiguous():
        raise RuntimeError(f"gemv_w4: scales {tuple(scales.shape)} {scales.dtype} on {scales.device}: want [{N}, groups] "
                           f"{x.dtype} on {dev}")
    if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != torch.uint8 or zeros.device != dev
                              or not zeros.is_contiguous()):
        raise RuntimeError(f"gemv_w4: zeros {tuple(zeros.shape)} {zeros.dtype} on {zeros.device}: want [{N}, {groups}] "
                           f"uint8 on {dev}")
    x_ld = x.stride(0) if M > 1 else -(-max(x.stride(0), K) // 8) * 8
    if x.stride(1) != 1 or x_ld % 8 or x_ld < K or _ptr(x) % 16:
        raise RuntimeError(f"gemv_w4: x strides {x.stride()} at {_ptr(x):#x}: want contiguous rows a multiple of 8 values "
                           "apart, 16-byte aligned")
    if out is None:
        out = torch.empty(M, N, dtype=x.dtype, device=dev)
    y_ld = out.stride(0) if M > 1 else N
    if out.shape != (M, N) or out.dtype != x.dtype or out.device != dev or (N > 1 and out.stride(1) != 1) or y_ld < N:
        raise RuntimeError(f"gemv_w4: out {tuple(out.shape)} {out.dtype} on {out.device}: want [{M}, {N}] {x.dtype}")
    a = abi.GemvW4Args(w=_ptr(w), scales=_ptr(scales), zeros=0 if zeros is None else _ptr(zeros), x=_ptr(x),
                       y=_ptr(out), M=M, N=N, K=K, group=K // groups, x_ld=x_ld, y_ld=y_ld, f16=x.dtype is torch.float16)
    need = ext.query("dsv41_gemv_w4_scratch_bytes", a)
    if need:
        scratch = torch.empty(need, dtype=torch.uint8, device=dev)
        a.scratch, a.scratch_bytes = _ptr(scratch), need
    ext.call("dsv41_gemv_w4", a, _stream())
    return out
