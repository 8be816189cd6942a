"""The quantised KV cache over the C ABI: rows written into pages of 8- or 4-bit codes (or 16-bit
values), read back, attended to, and the accepted drafts of a tree kept.

The pages are what the codec takes: a dense pool of fp8 pages is a run of 16384-symbol blocks for
``EntropyAwareHuffmanSystem.encode_blocks``, and ``ParrallelHuffmanDecoder.decode_blocks_to``
decodes stored pages straight into a pool.  The reference names the operand formats
(reports/spec.md:22) and has no counterpart of these calls.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch

from . import _lib as L
from ._lib import check
from . import api
from .api import Context, _Module, default_context

_DTYPES = {torch.bfloat16: L.HF_DT_BF16, torch.float16: L.HF_DT_FP16, torch.float32: L.HF_DT_FP32}
# hf_kv_batch and hf_kv_query as bytes: a ctypes structure takes longer to fill than a small call runs
_BATCH = struct.Struct("=QQQqIIII")
_QUERY = struct.Struct("=QQQQqqqqIIIf")
assert _BATCH.size == C.sizeof(L.hf_kv_batch) and _QUERY.size == C.sizeof(L.hf_kv_query)
_POOL_DTYPES = {
    L.HF_KV_BF16: (torch.bfloat16,), L.HF_KV_FP16: (torch.float16,),
    L.HF_KV_FP8_E4M3: (torch.uint8, torch.float8_e4m3fn),
    L.HF_KV_FP8_E5M2: (torch.uint8, torch.float8_e5m2), L.HF_KV_FP4_E2M1: (torch.uint8,),
}


def _raw_stream(index: int) -> int:
    """hipStream_t of torch's current stream; building the Stream object takes as long as a third of a
    write call's launch (1.2 us)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _pool_strides(k: torch.Tensor) -> Tuple[int, int, int]:
    """Page, token and head stride of a pool in bytes.  The stride of a dimension of one says nothing and is
    replaced by a valid one; every other stays what it is, so that a pool whose rows lie on one another
    (an expanded tensor) is refused by the call and not taken for a dense one."""
    size = k.element_size()
    page, token, head = (n * size for n in k.stride()[:3])
    row = k.shape[3] * size
    if k.shape[2] == 1:
        head = row
    if k.shape[1] == 1:
        token = row
    if k.shape[0] == 1:
        page = max(token, head)
    return page, token, head


class KvCache(_Module):
    """Two page pools and their scales (include/huffhip.h has the layout and the arithmetic).

    ``k``, ``v``: [pages, page_size, heads, head_dim] of codes (uint8 or the float8 type; fp4: two
    codes a byte, so the last dimension is head_dim / 2) or of the 16-bit type, any strides with a
    contiguous last dimension, the same for both.  ``k_scale``, ``v_scale``: uint8 [pages, heads,
    head_dim / group, page_size], contiguous; None for a 16-bit cache.  The pools stay the
    caller's: the cache keeps them alive and never allocates, copies or clears them.

    Without ``ctx`` every call runs on torch's current stream of the pools' device (its default
    context, made at the first call there, which therefore cannot be a captured one).

    In every call ``table`` is int32 [batch, pages of a sequence], ``kv_len`` int32 [batch] (tokens
    of a sequence, the call's rows included) and ``cu`` int32 [batch + 1], the first row of each
    sequence; None: one row each.  They are read on the device, on the context's stream; what they
    say wrongly is reported by ``Context.sync``.  No call synchronises or copies to the host.
    With ``ctx`` they run on its stream, whatever the current one is: the tensors of a call are to be
    ready there, and its results are.
    The cache is for inference: rows, queries and outputs that need a gradient are refused while
    gradients are recorded.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None, fmt: int = L.HF_KV_FP8_E4M3,
                 ctx: Optional[Context] = None):
        super().__init__(ctx)
        if fmt not in _POOL_DTYPES:
            raise ValueError(f"unknown cache format {fmt}")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.device != v.device:
            raise ValueError("k and v: [pages, page_size, heads, head_dim], alike in shape, strides and device")
        if k.dtype not in _POOL_DTYPES[fmt] or v.dtype != k.dtype:
            raise TypeError(f"cache format {fmt} holds {_POOL_DTYPES[fmt]}, not {k.dtype}, {v.dtype}")
        if not k.is_cuda or k.stride(3) != 1:
            raise ValueError("the pools are device tensors with a contiguous last dimension")
        pages, page_size, heads, width = k.shape
        dim = 2 * width if fmt == L.HF_KV_FP4_E2M1 else width
        group = 0
        if fmt in (L.HF_KV_BF16, L.HF_KV_FP16):
            if k_scale is not None or v_scale is not None:
                raise ValueError("a 16-bit cache has no scales")
        else:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.uint8 or s.device != k.device or not s.is_contiguous() \
                        or s.dim() != 4 or s.shape[0] != pages or s.shape[1] != heads \
                        or s.shape[2] < 1 or dim % s.shape[2] or s.shape[3] != page_size \
                        or s.shape != k_scale.shape:
                    raise ValueError("scales: contiguous uint8 [pages, heads, head_dim / group, page_size]")
            group = dim // k_scale.shape[2]
        self.k, self.v, self.k_scale, self.v_scale, self.fmt = k, v, k_scale, v_scale, fmt
        self.heads, self.head_dim, self.group, self.page_size = heads, dim, group, page_size
        self._device, self._index = k.device, k.device.index
        if ctx is not None and ctx.device != self._index:
            raise ValueError(f"the pools are on {k.device}, the context on cuda:{ctx.device}")
        self._hold(k, v, k_scale, v_scale)
        self._need = {}  # scratch of hf_kv_attend by the sizes it depends on
        self._c = L.hf_kv_cache(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if group else 0,
            v_scale.data_ptr() if group else 0, pages, *_pool_strides(k), page_size, heads, dim, group, fmt, 0)

    @staticmethod
    def empty(pages: int, page_size: int, heads: int, head_dim: int, fmt: int = L.HF_KV_FP8_E4M3,
              group: Optional[int] = None, ctx: Optional[Context] = None) -> "KvCache":
        """A cache with dense pools of its own, cleared.  ``group``: elements of a row that share a
        scale (default: the largest power of two that divides head_dim)."""
        own, ctx = ctx, ctx if ctx is not None else default_context()
        dev = f"cuda:{ctx.device}"
        wide = fmt in (L.HF_KV_BF16, L.HF_KV_FP16)
        dtype = {L.HF_KV_BF16: torch.bfloat16, L.HF_KV_FP16: torch.float16}.get(fmt, torch.uint8)
        width = head_dim // 2 if fmt == L.HF_KV_FP4_E2M1 else head_dim
        if group is None:
            group = head_dim & -head_dim
        with torch.cuda.stream(ctx.stream):
            pools = [torch.zeros(pages, page_size, heads, width, dtype=dtype, device=dev) for _ in range(2)]
            scales = [None, None] if wide else [
                torch.full((pages, heads, head_dim // group, page_size), 127, dtype=torch.uint8, device=dev)
                for _ in range(2)]
        return KvCache(*pools, *scales, fmt=fmt, ctx=own)

    # -- arguments -------------------------------------------------------------------------------
    @property
    def ctx(self) -> Context:
        if self._ctx is not None:
            return self._ctx
        key = (self._index, _raw_stream(self._index))
        ctx = api._default_ctx.get(key)
        if ctx is None:
            stream = torch.cuda.current_stream(self._index)
            with torch.cuda.device(self._index):  # (the question is asked of the current device's stream)
                capturing = torch.cuda.is_current_stream_capturing()
            if capturing:
                raise RuntimeError("the captured stream has no context yet: give the cache one made before the "
                                   "capture (ctx=Context(stream=...)), or call once on that stream before it")
            ctx = api._default_ctx[key] = Context(self._index, stream)
        return ctx

    def _handle(self):
        return self.ctx.handle

    def _empty(self, *tensors):
        """Tensors (shape, dtype) that belong to the context's stream, where the kernels use them."""
        if self._ctx is None or _raw_stream(self._index) == self._ctx.stream.cuda_stream:
            return [torch.empty(shape, dtype=dtype, device=self._device) for shape, dtype in tensors]
        with torch.cuda.stream(self._ctx.stream):
            return [torch.empty(shape, dtype=dtype, device=self._device) for shape, dtype in tensors]

    def _hold(self, *tensors) -> None:
        """Tensors of a call that ran on another stream than the current one: dropped by the caller, their
        memory is not handed out again before the call is through with it."""
        if self._ctx is not None and _raw_stream(self._index) != self._ctx.stream.cuda_stream:
            for t in tensors:
                if t is not None:
                    t.record_stream(self._ctx.stream)

    def _ints(self, name: str, t: torch.Tensor, dim: int) -> torch.Size:
        shape = t.shape
        # (one entry may have any stride: a column of a wider list, for one sequence)
        if t.dtype != torch.int32 or len(shape) != dim or t.get_device() != self._index or \
                (shape[-1] > 1 and t.stride(-1) != 1 and t.numel()):
            raise ValueError(f"{name}: int32, {dim} dimension(s), contiguous rows, on the pools' device")
        return shape

    def _batch(self, table, kv_len, cu, rows: int, max_rows: int) -> bytes:
        batch, width = self._ints("table", table, 2)
        if self._ints("kv_len", kv_len, 1)[0] != batch:
            raise ValueError("kv_len: one length for every row of the table")
        offsets = 0
        if cu is None:
            if rows != batch:
                raise ValueError("without cu there is one row for each sequence")
        else:
            if self._ints("cu", cu, 1)[0] != batch + 1:
                raise ValueError("cu: batch + 1 row offsets")
            offsets = cu.data_ptr()
        if not 0 <= max_rows < 1 << 32:
            raise ValueError("a sequence's largest number of rows is a 32-bit number")
        return _BATCH.pack(offsets, kv_len.data_ptr(), table.data_ptr(), table.stride(0) if batch > 1 else width,
                           width, batch, rows, max_rows)

    def _rows(self, name: str, t: torch.Tensor, heads: int) -> Tuple[int, int, int]:
        """Pointer and strides of a row tensor."""
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or t.get_device() != self._index:
            raise ValueError(f"{name}: [rows, {heads}, {self.head_dim}] on the pools' device")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name}: bf16, fp16 or fp32, not {t.dtype}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} needs a gradient, and no call here records one: detach it, or call under "
                               "torch.no_grad()")
        row, head, one = t.stride()
        if one != 1 and t.numel():
            raise ValueError(f"{name}: the last dimension is contiguous")
        # (a stride of a dimension of one says nothing)
        if heads == 1:
            head = self.head_dim
        return t.data_ptr(), row if shape[0] > 1 else heads * head, head

    # -- calls -----------------------------------------------------------------------------------
    def write(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor,
              cu: Optional[torch.Tensor] = None) -> None:
        """``hf_kv_write``: quantise rows [rows, heads, head_dim] into the last places of their
        sequences.  Rows outside every sequence are not looked at."""
        if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
            raise ValueError("k and v: as many rows of the same type")
        pk, kr, kh = self._rows("k", k, self.heads)
        pv, vr, vh = self._rows("v", v, self.heads)
        b = self._batch(table, kv_len, cu, k.shape[0], 0)
        check(L.lib().hf_kv_write(self._handle(), C.addressof(self._c), b, pk, pv, kr, kh, vr, vh,
                                  _DTYPES[k.dtype]), "hf_kv_write")
        self._hold(k, v, table, kv_len, cu)

    def read(self, table: torch.Tensor, kv_len: torch.Tensor, cu: Optional[torch.Tensor] = None,
             rows: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``hf_kv_read``: the last rows of the sequences as (keys, values) of ``dtype``, [rows,
        heads, head_dim] (whole sequences: offsets that count their tokens).  ``rows`` is needed
        with ``cu``; rows outside every sequence are left as they are (``out``) or undefined."""
        if out is None:
            n = table.shape[0] if cu is None and rows is None else rows
            if n is None:
                raise ValueError("rows: how many the offsets of cu cover")
            if dtype not in _DTYPES:
                raise TypeError(f"bf16, fp16 or fp32, not {dtype}")
            out = self._empty(((n, self.heads, self.head_dim), dtype), ((n, self.heads, self.head_dim), dtype))
        k, v = out
        if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
            raise ValueError("out: as many rows of the same type")
        pk, kr, kh = self._rows("out[0]", k, self.heads)
        pv, vr, vh = self._rows("out[1]", v, self.heads)
        b = self._batch(table, kv_len, cu, k.shape[0], 0)
        check(L.lib().hf_kv_read(self._handle(), C.addressof(self._c), b, pk, pv, kr, kh, vr, vh,
                                 _DTYPES[k.dtype]), "hf_kv_read")
        self._hold(k, v, table, kv_len, cu)
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor,
               cu: Optional[torch.Tensor] = None, max_q: int = 1, mask: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, lse: bool = False, out: Optional[torch.Tensor] = None):
        """``hf_kv_attend``: attention of rows ``q`` [rows, query heads, head_dim] (bf16 or fp16),
        whose keys and values are in the cache already, over their sequences.  ``max_q``: rows a
        sequence has at most (host knowledge; with ``cu``).  ``mask``: int32 [rows, words], bit j of
        a row: it sees row j of its sequence (a tree's ancestors); None: causal.  ``scale``: default
        1 / sqrt(head_dim).  Returns the outputs, with ``lse`` (outputs, fp32 [rows, query heads]
        logarithms of the softmax sums)."""
        if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % self.heads or q.dtype == torch.float32:
            raise ValueError(f"q: [rows, a multiple of {self.heads}, {self.head_dim}], bf16 or fp16")
        rows, heads = q.shape[0], q.shape[1]
        pq, qr, qh = self._rows("q", q, heads)
        if cu is None:
            max_q = 1
        b = self._batch(table, kv_len, cu, rows, max_q)
        handle, cache, words, bits = self._handle(), C.addressof(self._c), 0, 0
        if mask is not None:
            shape = self._ints("mask", mask, 2)
            words = shape[1]
            if shape[0] != rows or not mask.is_contiguous():
                raise ValueError("mask: contiguous int32 [rows, words]")
            if 32 * words < min(max_q, rows):
                raise ValueError("mask: a bit for each of the max_q rows of a sequence")
            bits = mask.data_ptr()
        # The scratch is taken from torch's allocator for this call: another stream's call, or a
        # captured graph, has its own.
        sizes = (table.shape, rows, max_q, cu is None, heads)
        need = self._need.get(sizes)
        known = need is not None
        if not known:
            need = L.lib().hf_kv_attend_work_bytes(handle, cache, b, heads)
        wanted = [((need,), torch.uint8)]
        if lse:
            wanted.append(((rows, heads), torch.float32))
        if out is None:
            wanted.append((q.shape, q.dtype))
        elif out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out: the shape and type of q")
        got = self._empty(*wanted)
        work, sums = got[0], got[1] if lse else None
        if out is None:
            out = got[-1]
        po, orow, oh = self._rows("out", out, heads)
        query = _QUERY.pack(pq, po, sums.data_ptr() if lse else 0, bits, qr, qh, orow, oh, heads, words,
                            _DTYPES[q.dtype], self.head_dim ** -0.5 if scale is None else scale)
        check(L.lib().hf_kv_attend(handle, cache, b, query, work.data_ptr() if need else None, need),
              "hf_kv_attend")
        self._hold(q, table, kv_len, cu, mask, out)
        if not known:  # (of a call that was taken: what hf_kv_attend refuses needs no scratch)
            if len(self._need) >= 1000:
                self._need = {}
            self._need[sizes] = need
        return (out, sums) if lse else out

    def keep(self, table: torch.Tensor, kv_len: torch.Tensor, cu: Optional[torch.Tensor],
             path: torch.Tensor, path_len: torch.Tensor, rows: Optional[int] = None,
             new_len: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``hf_kv_keep``: of the sequences' last rows (drafts), keep those that ``path`` int32
        [batch, width] names in ascending order, ``path_len`` int32 [batch] of them; returns the
        sequences' new lengths (``new_len``: no part of the call's other lists).  ``rows``: rows that
        ``cu`` covers (default: any number)."""
        batch = table.shape[0]
        if self._ints("path", path, 2)[0] != batch or self._ints("path_len", path_len, 1)[0] != batch:
            raise ValueError("path and path_len: one row for each sequence")
        b = self._batch(table, kv_len, cu, batch if cu is None else 0x7FFFFFFF if rows is None else rows, 0)
        if new_len is None:
            new_len, = self._empty(((batch,), torch.int32))
        elif self._ints("new_len", new_len, 1)[0] != batch:
            raise ValueError("new_len: one length for each sequence")
        check(L.lib().hf_kv_keep(self._handle(), C.addressof(self._c), b, path.data_ptr(),
                                 path.stride(0) if batch > 1 else path.shape[1], path.shape[1],
                                 path_len.data_ptr(), new_len.data_ptr()), "hf_kv_keep")
        self._hold(table, kv_len, cu, path, path_len, new_len)
        return new_len
