"""The decoder's K/V cache in 4 bits: writing rows, reading them back, attention over them.

Thin wrappers of madi_kv4_store / madi_kv4_load / madi_kv4_attn on torch CUDA tensors (format
and rules: include/madi_q8.h).  36 bytes hold the 64 elements of a (token, kv head), against
128 in f16 and 256 in f32.  Every call runs on the caller's current torch stream unless a
stream is given; for torch's default stream (handle 0) that is, as in the library's other calls,
the library stream, which runs in order with it unless madi_set_stream put another in its place.
A call takes nothing from the host but its arguments' addresses and can be captured in a CUDA
graph; positions and lengths are read on the device.

Errors: f32 attention is as near the exact result over the stored rows as plain f32 arithmetic;
f16 attention is that result rounded, calls of many rows with weights rounded to f16 besides, so
that the last bits of a row can depend on the rows and slots of its call.  Storing itself rounds every
element to one of 16 values: for normal rows attention is some 13 % (in norm) off that over
the rows themselves, more where scores spread widely (a third at a deviation of ten nats).

A token step's attention takes a few microseconds on the GPU, so the calls are kept short on
the host: structs are packed in one go, tensors are asked for their properties once.
"""
import contextlib
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import MADI_F16, MADI_F32

HEAD_DIM = 64
BLOCK_TOKENS = 64          # tokens per block
BLOCK_BYTES = 4608         # K and V of a block: codes and (c, d) of each
_DT = {torch.float32: MADI_F32, torch.float16: MADI_F16}
_U32 = (torch.int32, torch.uint32)
_current_device = getattr(torch._C, "_cuda_getDevice", None)       # absent in torch without CUDA
# the structs of include/madi_q8.h
_CACHE = struct.Struct("=Qiii4x").pack
_ROWS = struct.Struct("=QQQQqqii").pack
_QUERY = struct.Struct("=QQQQQqqqqiiii").pack


class Cache:
    """data: contiguous u8 [slots][kv_heads][ceil(max_tok / 64)][4608] on the library's
    device; max_tok: rows per slot that may be written and attended."""

    __slots__ = ("data", "slots", "kv_heads", "max_tok", "device", "_struct")

    def __init__(self, data: torch.Tensor, max_tok: int):
        sh = data.shape
        if data.dtype != torch.uint8 or len(sh) != 4 or sh[3] != BLOCK_BYTES or not data.is_contiguous():
            raise ValueError("data must be a contiguous u8 [slots][kv_heads][blocks][4608] tensor")
        if not 0 < max_tok <= 1 << 30 or sh[2] != (max_tok + BLOCK_TOKENS - 1) // BLOCK_TOKENS:
            raise ValueError(f"max_tok {max_tok} does not take {sh[2]} blocks of {BLOCK_TOKENS} tokens")
        self.data, self.max_tok = data, max_tok
        self.slots, self.kv_heads = sh[0], sh[1]
        self.device = data.get_device()             # -1: host memory, refused by the calls
        self._struct = _CACHE(data.data_ptr(), sh[0], sh[1], max_tok)

    @classmethod
    def empty(cls, slots: int, kv_heads: int, max_tok: int, device="cuda") -> "Cache":
        """A cache with no rows written."""
        if slots < 1 or kv_heads < 1 or max_tok < 1:
            raise ValueError(f"a cache of {slots} slots, {kv_heads} kv heads, {max_tok} tokens")
        blocks = (max_tok + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        return cls(torch.empty((slots, kv_heads, blocks, BLOCK_BYTES), dtype=torch.uint8, device=device), max_tok)


def _raw_stream(stream, c: Cache) -> int:
    if c.device < 0:
        raise ValueError("the cache is in host memory: the kernels need a CUDA device")
    if c.device != _current_device():
        raise ValueError(f"the cache is on {c.data.device}, which is not the current device")
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(c.device)
    return getattr(stream, "cuda_stream", stream)


def _on(stream):
    """Allocations and fills inside go to the stream the kernel runs on."""
    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(stream))


def _index(t: Optional[torch.Tensor], name: str, c: Cache) -> int:
    """Device pointer of a per-slot u32 / int32 vector (0: not given)."""
    if t is None:
        return 0
    if t.dtype not in _U32 or t.dim() != 1 or t.numel() != c.slots or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous u32 or int32 [{c.slots}] tensor")
    if t.get_device() != c.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {c.data.device}")
    return t.data_ptr()


def _layout(t: torch.Tensor, name: str, c: Cache, width: int) -> Tuple[int, int, int]:
    """(rows, slot stride, row stride) of an f32 or f16 [slots][rows][width] tensor, or of a
    [slots][width] one of one row per slot."""
    sh = t.shape
    dims = len(sh)
    if (dims != 3 and dims != 2) or sh[0] != c.slots or sh[dims - 1] != width or t.dtype not in _DT:
        raise ValueError(f"{name} must be an f32 or f16 [{c.slots}][rows][{width}] tensor, got {tuple(sh)} {t.dtype}")
    if t.get_device() != c.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {c.data.device}")
    st = t.stride()
    if st[dims - 1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if dims == 2:
        return 1, st[0] if sh[0] > 1 else width, width
    # a dimension of one element has no stride of its own
    row = st[1] if sh[1] > 1 else width
    return sh[1], st[0] if sh[0] > 1 else row * max(sh[1], 1), row


def _pair(k: torch.Tensor, v: torch.Tensor, names: str, c: Cache) -> Tuple[int, int, int]:
    lay = _layout(k, names, c, c.kv_heads * HEAD_DIM)
    if k.dim() != 3:
        raise ValueError(f"{names} must be a [slots][rows][kv_heads * 64] tensor")
    if v.shape != k.shape or v.dtype != k.dtype or (
            (v.stride() != k.stride() or v.get_device() != c.device) and
            _layout(v, "v" + names[1:], c, c.kv_heads * HEAD_DIM) != lay):
        raise ValueError(f"v{names[1:]} must match {names} in shape, type and strides")
    return lay


def store(cache: Cache, k: torch.Tensor, v: torch.Tensor, pos: Optional[torch.Tensor] = None,
          n: Optional[torch.Tensor] = None, stream=None) -> None:
    """Quantise rows into the cache: k / v f32 or f16 [slots][rows][kv_heads * 64] (rows may be
    strided); row i of slot s goes to cache row pos[s] + i (pos None: i), for i < n[s] (n None:
    all).  Rows at or past max_tok are dropped."""
    rows, slot, row = _pair(k, v, "k", cache)
    args = _ROWS(k.data_ptr(), v.data_ptr(), _index(pos, "pos", cache), _index(n, "n", cache), slot, row, _DT[k.dtype],
                 rows)
    rc = _lib.load().madi_kv4_store(cache._struct, args, _raw_stream(stream, cache))
    if rc:
        _lib.check(rc, "madi_kv4_store")


def load(cache: Cache, rows: int, pos: Optional[torch.Tensor] = None, n: Optional[torch.Tensor] = None,
         dtype: torch.dtype = torch.float16, k_out: Optional[torch.Tensor] = None,
         v_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read cache rows pos[s] .. pos[s] + rows - 1 back as (k, v), f32 or f16
    [slots][rows][kv_heads * 64].  Rows i >= n[s] and rows past max_tok are left as they were
    in k_out / v_out (zero where these are not given)."""
    if (k_out is None) != (v_out is None):
        raise ValueError("k_out and v_out go together")
    if k_out is None:
        if dtype not in _DT or rows < 0:
            raise ValueError(f"{rows} rows of {dtype} (f32 or f16)")
        with _on(stream):
            k_out = torch.zeros((cache.slots, rows, cache.kv_heads * HEAD_DIM), dtype=dtype, device=cache.data.device)
            v_out = torch.zeros_like(k_out)
    got, slot, row = _pair(k_out, v_out, "k_out", cache)
    if got != rows:
        raise ValueError(f"k_out holds {got} rows, not {rows}")
    args = _ROWS(k_out.data_ptr(), v_out.data_ptr(), _index(pos, "pos", cache), _index(n, "n", cache), slot, row,
                 _DT[k_out.dtype], rows)
    rc = _lib.load().madi_kv4_load(cache._struct, args, _raw_stream(stream, cache))
    if rc:
        _lib.check(rc, "madi_kv4_load")
    return k_out, v_out


def attn(q: torch.Tensor, cache: Cache, heads: int, pos: Optional[torch.Tensor] = None,
         lens: Optional[torch.Tensor] = None, n: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
         stream=None) -> torch.Tensor:
    """Attention over the cache.  q f32 or f16 [slots][heads * 64] (one query token per slot) or
    [slots][rows][heads * 64], finite and below 2^100; returns out like q.  Query row i of slot s attends cache rows
    0 .. pos[s] + i (pos: causal), or 0 .. lens[s] - 1 (lens), or all max_tok rows; no row to
    attend gives zeros.  Rows i >= n[s] are padding: left as they were in `out`."""
    rows, q_slot, q_row = _layout(q, "q", cache, heads * HEAD_DIM)
    if pos is not None and lens is not None:
        raise ValueError("pos (causal) and lens exclude one another")
    args = (_index(pos, "pos", cache), _index(lens, "lens", cache), _index(n, "n", cache))
    if out is None:
        with _on(stream):
            out = (torch.empty if n is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and type")
    if out.stride() == q.stride() and out.get_device() == cache.device:
        o_slot, o_row = q_slot, q_row
    else:
        _, o_slot, o_row = _layout(out, "out", cache, heads * HEAD_DIM)
    rc = _lib.load().madi_kv4_attn(cache._struct, _QUERY(q.data_ptr(), out.data_ptr(), *args, q_slot, q_row, o_slot,
                                                         o_row, _DT[q.dtype], heads, rows, 0),
                                   _raw_stream(stream, cache))
    if rc:
        _lib.check(rc, "madi_kv4_attn")
    return out
