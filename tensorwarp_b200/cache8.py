"""A key/value cache held in 8 bits, the append that fills it and the attention that reads it (``include/twm_serve.h``).

Tensors are torch CUDA tensors; every computation is a call into ``libtwmarlin.so`` on the given stream (the current one
if none), enqueued and not waited for.  A cache belongs to one layer and holds `seqs` sequences; where each of them
stands is the caller's, in device memory, so that a captured step serves every position.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from ._lib import TwmError, check
from .quantize import _require_cuda, _stream_ptr

BLOCK = 64                      # tokens that share a scale


def rope_table(positions: int, head_dim: int, base: float, device="cuda") -> torch.Tensor:
    """f32 [positions, head_dim]: cosines, then sines, of every position's rotation (angles in 64 bits)."""
    pair = torch.arange(head_dim // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * float(base) ** (-2.0 * pair / head_dim)
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


class Cache8:
    """The tensors of one layer's cache, as ``include/twm_serve.h`` lays them out."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k_tail: torch.Tensor, v_tail: torch.Tensor):
        _require_cuda(k, v, k_scale, v_scale, k_tail, v_tail)
        if k.dim() != 4:
            raise TwmError(_lib.TWM_EINVAL, "Cache8: k must be [sequences, heads, capacity, head_dim]")
        self.seqs, self.kv_heads, self.capacity, self.head_dim = k.shape
        scales, tail = (self.seqs, self.kv_heads, self.capacity // BLOCK), (self.seqs, self.kv_heads, 2, BLOCK, self.head_dim)
        for t, shape, dtypes in ((k, k.shape, (torch.float8_e4m3fn, torch.uint8)), (v, k.shape, (torch.float8_e4m3fn, torch.uint8)),
                                 (k_scale, scales, (torch.float32,)), (v_scale, scales, (torch.float32,)),
                                 (k_tail, tail, (torch.float16,)), (v_tail, tail, (torch.float16,))):
            if tuple(t.shape) != tuple(shape) or t.dtype not in dtypes or not t.is_contiguous() or t.device != k.device:
                raise TwmError(_lib.TWM_EINVAL, f"Cache8: expected a contiguous {dtypes[0]} tensor of {tuple(shape)} on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail = k, v, k_scale, v_scale, k_tail, v_tail
        self.device, self.index = k.device, k.get_device()
        self.desc = _lib.Cache8(self.seqs, self.kv_heads, self.head_dim, self.capacity, k.data_ptr(), v.data_ptr(), k_scale.data_ptr(),
                                v_scale.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr())
        self._ref = C.addressof(self.desc)

    @classmethod
    def empty(cls, seqs: int, capacity: int, kv_heads: int, head_dim: int, device="cuda") -> "Cache8":
        """Room for `capacity` tokens (rounded up to whole blocks) of each sequence."""
        capacity = -(-capacity // BLOCK) * BLOCK
        sides = []
        for _ in range(2):
            sides.append((torch.zeros((seqs, kv_heads, capacity, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                          torch.ones((seqs, kv_heads, capacity // BLOCK), dtype=torch.float32, device=device),
                          torch.zeros((seqs, kv_heads, 2, BLOCK, head_dim), dtype=torch.float16, device=device)))
        (k, ks, kt), (v, vs, vt) = sides
        return cls(k, v, ks, vs, kt, vt)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail))


class Workspace:
    """Scratch of ``attention``, for one call at a time."""

    def __init__(self, nbytes: int, device="cuda"):
        self.nbytes = max(int(nbytes), 16)
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        self.ptr, self.index = self.buf.data_ptr(), self.buf.get_device()

    @classmethod
    def for_cache(cls, cache: Cache8, num_heads: int, max_rows: int = 1) -> "Workspace":
        """Enough for calls of up to `max_rows` rows a sequence."""
        return cls(_lib.lib().twm_cache8_attention_bytes(cache._ref, num_heads, max_rows), cache.device)


def _refuse(where: str, cache: Cache8, wide: torch.Tensor, narrow: torch.Tensor, start: torch.Tensor, row_start: Optional[torch.Tensor],
            columns: int, out_columns: int) -> None:
    """Says what is wrong with a call's rows, which are not as they must be."""
    for t in (wide, narrow, start) if row_start is None else (wide, narrow, start, row_start):
        _require_cuda(t)
        if t.device != cache.device:
            raise TwmError(_lib.TWM_EINVAL, f"{where}: tensors of {t.device} with a cache of {cache.device}")
    if wide.dtype is not torch.float16 or narrow.dtype is not torch.float16 or wide.dim() != 2 or narrow.dim() != 2:
        raise TwmError(_lib.TWM_EINVAL, f"{where}: rows must be float16 matrices")
    if start.dtype is not torch.int32 or start.numel() != cache.seqs or not start.is_contiguous():
        raise TwmError(_lib.TWM_EINVAL, f"{where}: start must be int32 [{cache.seqs}]")
    if row_start is not None and (row_start.dtype is not torch.int32 or row_start.numel() != cache.seqs + 1 or not row_start.is_contiguous()):
        raise TwmError(_lib.TWM_EINVAL, f"{where}: row_start must be int32 [{cache.seqs + 1}]")
    raise TwmError(_lib.TWM_EINVAL, f"{where}: expected rows of {columns} and {out_columns} numbers, as many of both")


def _pointer(cache: Cache8, start: torch.Tensor, row_start: Optional[torch.Tensor]) -> Optional[int]:
    """Address of row_start (0: none); None if it or start is not what a call takes."""
    i32, index = torch.int32, cache.index
    if start.dtype is not i32 or start.get_device() != index or start.numel() != cache.seqs or not start.is_contiguous():
        return None
    if row_start is None:
        return 0
    if row_start.dtype is not i32 or row_start.get_device() != index or row_start.numel() != cache.seqs + 1 or not row_start.is_contiguous():
        return None
    return row_start.data_ptr()


def append(cache: Cache8, qkv: torch.Tensor, q_out: torch.Tensor, start: torch.Tensor, *, num_heads: int, row_start: Optional[torch.Tensor] = None,
           max_rows: int = 1, bias: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None,
           flags: int = 0) -> None:
    """qkv f16 [rows, (num_heads + 2 kv_heads) * head_dim]: queries out, rotated, to q_out [rows, num_heads * head_dim]; keys, rotated, and
    values to the cache.  start int32 [seqs]: tokens of each sequence before the call (< 0: not in the call); row_start int32
    [seqs + 1]: its rows among the call's, at most `max_rows` (None: one row a sequence).  rope: ``rope_table`` of the cache's capacity;
    bias f32 of a whole row.  q_out may be the columns of the queries in qkv, else it must not overlap them; a call without rows (row_start of zeros) does nothing."""
    # Once per layer and token, and as long as the call itself takes: sizes and strides are read at once, and the arguments packed by struct.
    d, index, f16 = cache.head_dim, cache.index, torch.float16
    columns, out_columns = (num_heads + 2 * cache.kv_heads) * d, num_heads * d
    size, ld, out_size, out_ld = qkv.size(), qkv.stride(), q_out.size(), q_out.stride()
    at = _pointer(cache, start, row_start)
    if (at is None or len(size) != 2 or len(out_size) != 2 or size[1] != columns or out_size[1] != out_columns or out_size[0] < size[0] or ld[1] != 1
            or out_ld[1] != 1 or qkv.dtype is not f16 or q_out.dtype is not f16 or qkv.get_device() != index or q_out.get_device() != index):
        _refuse("append", cache, qkv, q_out, start, row_start, columns, out_columns)
    if size[0] == 0 and at:
        return
    bias_at = rope_at = 0
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.numel() != columns or not bias.is_contiguous() or bias.get_device() != index:
            raise TwmError(_lib.TWM_EINVAL, "append: bias must be float32 of a whole row")
        bias_at = bias.data_ptr()
    if rope is not None:
        if rope.dtype is not torch.float32 or rope.numel() < cache.capacity * d or not rope.is_contiguous() or rope.get_device() != index:
            raise TwmError(_lib.TWM_EINVAL, "append: rope must be float32 [capacity, head_dim]")
        rope_at = rope.data_ptr()
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return append(cache, qkv, q_out, start, num_heads=num_heads, row_start=row_start, max_rows=max_rows, bias=bias, rope=rope, stream=stream, flags=flags)
    rows = size[0]
    q_ld, qkv_ld = (out_ld[0], ld[0]) if rows > 1 else (out_columns, columns)                # the stride of a single row says nothing
    args = _lib.pack_append_args(q_out.data_ptr(), q_ld, qkv.data_ptr(), qkv_ld, bias_at, rope_at, num_heads, rows, min(max_rows, rows) if at else max_rows, at,
                                 start.data_ptr())
    status = _lib.lib().twm_cache8_append(cache._ref, args, flags, _stream_ptr(stream))
    if status:
        check(status, "twm_cache8_append")


def attention(cache: Cache8, q: torch.Tensor, out: torch.Tensor, start: torch.Tensor, *, num_heads: int, row_start: Optional[torch.Tensor] = None,
              max_rows: int = 1, scale: Optional[float] = None, window: int = 0, workspace: Optional[Workspace] = None,
              stream: Optional[torch.cuda.Stream] = None, flags: int = 0) -> None:
    """Causal softmax attention of q f16 [rows, num_heads * head_dim] over the cache, which holds the rows' own keys and values already
    (``append`` with the same start and row_start); out like q.  scale: 1/sqrt(head_dim) if None; window: how many of the newest keys
    a row sees (0: all).  workspace: ``Workspace.for_cache``; without one the call makes its own.  out must not overlap q (refused); a
    call without rows (row_start of zeros) does nothing."""
    d, index, f16 = cache.head_dim, cache.index, torch.float16
    columns = num_heads * d
    size, ld, out_size, out_ld = q.size(), q.stride(), out.size(), out.stride()
    at = _pointer(cache, start, row_start)
    if (at is None or len(size) != 2 or len(out_size) != 2 or size[1] != columns or out_size[1] != columns or out_size[0] < size[0] or ld[1] != 1
            or out_ld[1] != 1 or q.dtype is not f16 or out.dtype is not f16 or q.get_device() != index or out.get_device() != index):
        _refuse("attention", cache, q, out, start, row_start, columns, columns)
    if size[0] == 0 and at:
        return
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return attention(cache, q, out, start, num_heads=num_heads, row_start=row_start, max_rows=max_rows, scale=scale, window=window,
                             workspace=workspace, stream=stream, flags=flags)
    if workspace is None:
        with torch.cuda.stream(stream):
            workspace = Workspace.for_cache(cache, num_heads, max_rows)
    elif workspace.index != index:
        raise TwmError(_lib.TWM_EINVAL, "attention: the workspace is on another device")
    rows = size[0]
    o_ld, q_ld = (out_ld[0], ld[0]) if rows > 1 else (columns, columns)                      # the stride of a single row says nothing
    args = _lib.pack_attention_args(out.data_ptr(), o_ld, q.data_ptr(), q_ld, num_heads, rows, min(max_rows, rows) if at else max_rows, window, at,
                                    start.data_ptr(), workspace.ptr, workspace.nbytes, 1.0 / math.sqrt(d) if scale is None else scale)
    status = _lib.lib().twm_cache8_attention(cache._ref, args, flags, _stream_ptr(stream))
    if status:
        check(status, "twm_cache8_attention")
