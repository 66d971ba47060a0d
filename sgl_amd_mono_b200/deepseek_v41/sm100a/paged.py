"""A paged 8-bit cache of grouped-query keys and values, and the two operators of a decode step on
it: the append of the step's rows (with the position rotation) and their attention.

``PagedKV`` wraps the cache's four tensors, which a server allocates once: keys and values
``[pages, kv_heads, page, dim]`` e4m3 bytes, and an E8M0 code per ``block`` consecutive tokens of a
head, ``[pages, kv_heads, page / block]``. Sequence ``s`` of a step holds ``lens[s]`` tokens on the
pages ``table[s]``; its rows are its last tokens. The rows ``[T, heads, dim]`` of all sequences lie
one after the other: ``cu_rows[s] .. cu_rows[s + 1]`` are sequence ``s``'s, or row ``s`` alone with
``cu_rows=None``. Everything a call needs stays on the device, so a call can be captured in a CUDA
graph with its lengths and pages changed between replays; a padded batch gives its unused
sequences no rows (or length 0). A ``PagedKV`` stays with the tensors that it was made of: they
cannot be replaced, a copy has tensors of its own, and calls are refused once one of them has moved
to other memory. Host-side argument errors raise ``RuntimeError``.
"""

from __future__ import annotations

import struct

import torch

from ...common import ext
from . import abi

DIMS = (64, 128, 256)
_F32, _U32 = struct.Struct("<f"), struct.Struct("<I")


def current_stream(device: int, name: str) -> int:
    """The current stream of CUDA device ``device``, which has to be the current device: the launch
    goes there. (torch's own short way to both, a tenth of the public calls' time.)"""
    if device < 0 or device != torch._C._cuda_getDevice():
        where = "the host" if device < 0 else f"cuda:{device}"
        raise RuntimeError(f"{name}: on {where}, which is not the current CUDA device")
    return torch._C._cuda_getCurrentRawStream(device)


class PagedKV:
    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor):
        if k.dim() != 4 or k_codes.dim() != 3:
            raise RuntimeError(f"PagedKV: keys {tuple(k.shape)}, codes {tuple(k_codes.shape)}; want "
                               "[pages, kv_heads, page, dim] and [pages, kv_heads, page / block]")
        pages, heads, page, dim = k.shape
        per = k_codes.shape[2]
        if dim not in DIMS or not pages or not heads or not per or page % per or page // per % 16 or not page:
            raise RuntimeError(f"PagedKV: pages {pages}, heads {heads}, page {page}, dim {dim}, {per} codes a page: "
                               f"dim in {DIMS}, tokens a code a multiple of 16")
        for t, name, shape in ((k, "keys", k.shape), (v, "values", k.shape),
                               (k_codes, "key codes", (pages, heads, per)), (v_codes, "value codes", (pages, heads, per))):
            if t.shape != tuple(shape) or t.element_size() != 1 or not t.is_contiguous() or t.device != k.device:
                raise RuntimeError(f"PagedKV: {name} {tuple(t.shape)} {t.dtype} on {t.device}: want contiguous bytes "
                                   f"{tuple(shape)} on {k.device}")
        self._tensors = (k, v, k_codes, v_codes)
        self._at = (k.data_ptr(), v.data_ptr(), k_codes.data_ptr(), v_codes.data_ptr())
        self.pages, self.kv_heads, self.page, self.dim, self.block = pages, heads, page, dim, page // per
        self._dev = k.get_device()
        cache = dict(zip(("k_cache", "v_cache", "k_codes", "v_codes"), self._at), kv_heads=heads, dim=dim, pages=pages,
                     page=page, block=self.block)
        self._append_args, self._attend_args = bytes(abi.KvAppendArgs(**cache)), bytes(abi.PagedAttnArgs(**cache))

    @classmethod
    def empty(cls, pages: int, page: int, kv_heads: int, dim: int, *, block: int = 16, device="cuda") -> "PagedKV":
        """A new cache of ``pages`` pages of ``page`` tokens."""
        if block < 16 or block % 16 or page % block:
            raise RuntimeError(f"PagedKV: page {page}, block {block}: block a multiple of 16, page of block")
        u8 = dict(dtype=torch.uint8, device=device)
        data, codes = (pages, kv_heads, page, dim), (pages, kv_heads, page // block)
        return cls(torch.zeros(data, **u8), torch.zeros(data, **u8), torch.zeros(codes, **u8),
                   torch.zeros(codes, **u8))

    # The calls' argument blocks hold the tensors' addresses, so the tensors are read-only attributes and
    # a copy (deepcopy, pickle) is made from its own.
    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_codes = property(lambda self: self._tensors[2])
    v_codes = property(lambda self: self._tensors[3])

    def __reduce__(self):
        return type(self), self._tensors

    # ------------------------------------------------------------ checks
    def _rows(self, x: torch.Tensor, name: str, rows: int, dtype: torch.dtype, heads: int) -> tuple[int, int]:
        """Check rows [rows, heads, dim] (a row's heads contiguous): their address and their stride."""
        dim, at = self.dim, x.data_ptr()
        if x.shape != (rows, heads, dim) or x.dtype is not dtype or x.get_device() != self._dev:
            raise RuntimeError(f"{name}: {tuple(x.shape)} {x.dtype} on {x.device}: want [{rows}, {heads}, {dim}] {dtype} "
                               f"on {self.k.device}")
        ld, head, one = x.stride()
        if rows < 2:
            ld = heads * dim
        if one != 1 or (head != dim and heads > 1) or ld & 7 or ld < heads * dim or at & 15:
            raise RuntimeError(f"{name}: strides {x.stride()} at {at:#x}: a row's heads have to be contiguous, rows a "
                               "multiple of 8 values apart and 16-byte aligned")
        return at, ld

    def _step(self, a, x: torch.Tensor, name: str, lens: torch.Tensor, table: torch.Tensor,
              cu_rows: torch.Tensor | None) -> tuple[int, torch.dtype]:
        """Check the step's tensors and fill in what the two calls share: (rows, their type)."""
        dev, i32, dtype = self._dev, torch.int32, x.dtype
        kt, vt, kc, vc = self._tensors
        if (kt.data_ptr(), vt.data_ptr(), kc.data_ptr(), vc.data_ptr()) != self._at:
            raise RuntimeError(f"{name}: a cache tensor has moved since the PagedKV was made of it; make another")
        if x.dim() != 3:
            raise RuntimeError(f"{name}: {tuple(x.shape)}: want [rows, heads, {self.dim}]")
        if dtype is not torch.bfloat16 and dtype is not torch.float16:
            raise RuntimeError(f"{name}: {dtype}, want bfloat16 or float16")
        rows = x.shape[0]
        if lens.dim() != 1 or lens.dtype is not i32 or lens.get_device() != dev or not lens.is_contiguous():
            raise RuntimeError(f"lens: {tuple(lens.shape)} {lens.dtype} on {lens.device}: want [sequences] int32 on "
                               f"{self.k.device}")
        seqs = lens.shape[0]
        if table.dim() != 2 or table.dtype is not i32 or table.get_device() != dev:
            raise RuntimeError(f"table: {tuple(table.shape)} {table.dtype} on {table.device}: want [{seqs}, pages] int32 "
                               f"on {self.k.device}")
        n, width = table.shape
        ld, one = table.stride()
        if n != seqs or not width or (one != 1 and width > 1) or (ld < width and seqs > 1):
            raise RuntimeError(f"table: {tuple(table.shape)} of strides {table.stride()}: want [{seqs}, pages] with "
                               "contiguous rows")
        if cu_rows is None:
            if seqs != rows:
                raise RuntimeError(f"{rows} rows for {seqs} sequences without cu_rows: one row a sequence")
        elif cu_rows.shape != (seqs + 1,) or cu_rows.dtype is not i32 or cu_rows.get_device() != dev \
                or not cu_rows.is_contiguous():
            raise RuntimeError(f"cu_rows: {tuple(cu_rows.shape)} {cu_rows.dtype} on {cu_rows.device}: want [{seqs + 1}] "
                               f"int32 on {self.k.device}")
        else:
            a.cu_rows = cu_rows.data_ptr()
        a.T, a.seqs, a.f16, a.lens, a.table = rows, seqs, dtype is torch.float16, lens.data_ptr(), table.data_ptr()
        a.width, a.table_ld = width, ld if seqs > 1 else width
        return rows, dtype

    # ------------------------------------------------------------ operators
    def append(self, k: torch.Tensor, v: torch.Tensor, *, lens: torch.Tensor, table: torch.Tensor,
               cu_rows: torch.Tensor | None = None, q: torch.Tensor | None = None,
               cos_sin: torch.Tensor | None = None, neox: bool = False,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Write the step's keys and values [T, kv_heads, dim] (bf16 or f16) into the cache as its
        sequences' last tokens; ``lens`` [sequences] int32 counts them already. With ``cos_sin``
        [positions, rope] fp32 (rope / 2 cos, then rope / 2 sin) the last ``rope`` dims of the keys,
        and of the queries ``q`` [T, heads, dim] where given, are rotated by their positions, in
        pairs (2j, 2j + 1) or, ``neox``, (j, j + rope / 2). Returns the rotated queries (``q_out``,
        which may be ``q``, or a new tensor), or None without ``q``; rows behind the last sequence are
        left as they were (unset in a new tensor). A sequence's pages must not be
        another's: two sequences that append to one block race."""
        stream = current_stream(self._dev, "PagedKV.append")
        a = abi.KvAppendArgs.from_buffer_copy(self._append_args)
        rows, dtype = self._step(a, k, "k", lens, table, cu_rows)
        heads = self.kv_heads
        a.k, a.k_ld = self._rows(k, "k", rows, dtype, heads)
        a.v, a.v_ld = self._rows(v, "v", rows, dtype, heads)
        if cos_sin is not None:
            if cos_sin.dim() != 2 or cos_sin.dtype is not torch.float32 or cos_sin.get_device() != self._dev \
                    or not cos_sin.is_contiguous() or not cos_sin.shape[0] or cos_sin.shape[1] % 16 \
                    or not 16 <= cos_sin.shape[1] <= self.dim or cos_sin.data_ptr() & 15:
                raise RuntimeError(f"cos_sin: {tuple(cos_sin.shape)} {cos_sin.dtype} on {cos_sin.device}: want "
                                   f"[positions, rope] fp32, rope a multiple of 16 up to {self.dim}")
            a.cos_sin = cos_sin.data_ptr()
            a.rope_rows, a.rope = cos_sin.shape
            a.neox = bool(neox)
        if q is not None:
            if q.dim() != 3 or not q.shape[1] or q.shape[1] % heads:
                raise RuntimeError(f"q: {tuple(q.shape)}: want [{rows}, heads, {self.dim}], heads a multiple of {heads}")
            heads = q.shape[1]
            a.q, a.q_ld = self._rows(q, "q", rows, dtype, heads)
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            a.q_out, a.q_out_ld = self._rows(q_out, "q_out", rows, dtype, heads)
        elif q_out is not None:
            raise RuntimeError("q_out without q")
        a.heads = heads
        if rows and a.seqs:
            ext.call("dsv41_kv_append", a, stream)
        return q_out

    def attend(self, q: torch.Tensor, *, lens: torch.Tensor, table: torch.Tensor, scale: float,
               cu_rows: torch.Tensor | None = None, window: int = 0, sink: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the rows q [T, heads, dim] (bf16 or f16) over the cache: row j of a
        sequence's n sees the tokens before ``lens[s] - n + j + 1`` (causal over the step's own
        rows), with ``window`` the last ``window`` of them; ``scale`` times q . k goes into the
        softmax, with ``sink`` [heads] fp32 as one more score without a value. A row that sees
        nothing gives zeros. Returns ``out`` (or a new tensor) [T, heads, dim]; rows behind the last
        sequence are left as they were (unset in a new tensor)."""
        stream = current_stream(self._dev, "PagedKV.attend")
        a = abi.PagedAttnArgs.from_buffer_copy(self._attend_args)
        rows, dtype = self._step(a, q, "q", lens, table, cu_rows)
        heads = q.shape[1]
        if not heads or heads % self.kv_heads:
            raise RuntimeError(f"q: {heads} heads over {self.kv_heads} key heads")
        a.heads = heads
        a.q, a.q_ld = self._rows(q, "q", rows, dtype, heads)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a.out, a.out_ld = self._rows(out, "out", rows, dtype, heads)
        if not 0 <= window < 1 << 31:
            raise RuntimeError(f"window {window}")
        a.window = window
        try:
            a.scale_f32 = _U32.unpack(_F32.pack(scale))[0]
        except (OverflowError, struct.error):
            raise RuntimeError(f"scale {scale}: want a number in fp32's range") from None
        if sink is not None:
            if sink.shape != (heads,) or sink.dtype is not torch.float32 or sink.get_device() != self._dev \
                    or not sink.is_contiguous():
                raise RuntimeError(f"sink: {tuple(sink.shape)} {sink.dtype} on {sink.device}: want [{heads}] fp32")
            a.sink = sink.data_ptr()
        if not rows or not a.seqs:
            return out
        need = ext.query("dsv41_paged_attn_scratch_bytes", a)
        if need:
            scratch = self.k.new_empty((need,))
            a.scratch, a.scratch_bytes = scratch.data_ptr(), need
        ext.call("dsv41_paged_attn", a, stream)
        return out
