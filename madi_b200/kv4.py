"""The decoder's K/V cache in 4 bits: writing rows, reading them back, attention over them.

Thin wrappers of madi_kv4_store / madi_kv4_load / madi_kv4_attn on torch CUDA tensors (format
and rules: include/madi_q8.h).  36 bytes hold the 64 elements of a (token, kv head), against
128 in f16 and 256 in f32.  Every call runs on the caller's current torch stream unless a
stream is given, takes nothing from the host but its arguments' addresses, and can be captured
in a CUDA graph; positions and lengths are read on the device.
"""
import contextlib
import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import MADI_F16, MADI_F32
from .q8 import _stream

HEAD_DIM = 64
BLOCK_TOKENS = 64          # tokens per block
BLOCK_BYTES = 4608         # K and V of a block: codes and (c, d) of each
_DT = {torch.float32: MADI_F32, torch.float16: MADI_F16}


@dataclass
class Cache:
    """data: contiguous u8 [slots][kv_heads][ceil(max_tok / 64)][4608] on the library's
    device; max_tok: rows per slot that may be written and attended."""
    data: torch.Tensor
    max_tok: int

    def __post_init__(self):
        d = self.data
        if d.dtype != torch.uint8 or d.dim() != 4 or d.shape[3] != BLOCK_BYTES or not d.is_contiguous():
            raise ValueError("data must be a contiguous u8 [slots][kv_heads][blocks][4608] tensor")
        if not 0 < self.max_tok <= 1 << 30 or d.shape[2] != (self.max_tok + BLOCK_TOKENS - 1) // BLOCK_TOKENS:
            raise ValueError(f"max_tok {self.max_tok} does not take {d.shape[2]} blocks of {BLOCK_TOKENS} tokens")

    @classmethod
    def empty(cls, slots: int, kv_heads: int, max_tok: int, device="cuda") -> "Cache":
        """A cache with no rows written."""
        if slots < 1 or kv_heads < 1 or max_tok < 1:
            raise ValueError(f"a cache of {slots} slots, {kv_heads} kv heads, {max_tok} tokens")
        blocks = (max_tok + BLOCK_TOKENS - 1) // BLOCK_TOKENS
        return cls(torch.empty((slots, kv_heads, blocks, BLOCK_BYTES), dtype=torch.uint8, device=device), max_tok)

    @property
    def slots(self) -> int:
        return self.data.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.data.shape[1]

    def handle(self) -> _lib.madi_kv4:
        return _lib.madi_kv4(self.data.data_ptr(), self.slots, self.kv_heads, self.max_tok)


def _device(c: Cache) -> None:
    if not c.data.is_cuda:
        raise ValueError(f"the cache is on {c.data.device}: the kernels need a CUDA device")


def _on(stream):
    """Allocations and fills inside go to the stream the kernel runs on."""
    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(stream))


def _index(t: Optional[torch.Tensor], name: str, c: Cache) -> Optional[int]:
    """Device pointer of a per-slot u32 / int32 vector."""
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.uint32) or t.shape != (c.slots,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous u32 or int32 [{c.slots}] tensor")
    if t.device != c.data.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {c.data.device}")
    return t.data_ptr()


def _strides(t: torch.Tensor, name: str, c: Cache, width: int) -> Tuple[int, int]:
    """(slot, row) strides of a [slots][rows][width] tensor."""
    if t.dim() != 3 or t.shape[0] != c.slots or t.shape[2] != width or t.dtype not in _DT:
        raise ValueError(f"{name} must be an f32 or f16 [{c.slots}][rows][{width}] tensor, got {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if t.device != c.data.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {c.data.device}")
    # a dimension of one element has no stride of its own
    row = t.stride(1) if t.shape[1] > 1 else width
    return (t.stride(0) if t.shape[0] > 1 else row * max(t.shape[1], 1)), row


def store(cache: Cache, k: torch.Tensor, v: torch.Tensor, pos: Optional[torch.Tensor] = None,
          n: Optional[torch.Tensor] = None, stream=None) -> None:
    """Quantise rows into the cache: k / v f32 or f16 [slots][rows][kv_heads * 64] (rows may be
    strided); row i of slot s goes to cache row pos[s] + i (pos None: i), for i < n[s] (n None:
    all).  Rows at or past max_tok are dropped."""
    w = cache.kv_heads * HEAD_DIM
    st = _strides(k, "k", cache, w)
    if v.shape != k.shape or v.dtype != k.dtype or _strides(v, "v", cache, w) != st:
        raise ValueError("v must match k in shape, type and strides")
    args = (_index(pos, "pos", cache), _index(n, "n", cache))
    _device(cache)
    h = cache.handle()
    _lib.check(_lib.load().madi_kv4_store(ctypes.byref(h), k.data_ptr(), v.data_ptr(), _DT[k.dtype], k.shape[1], *st,
                                          *args, _stream(stream)), "madi_kv4_store")


def load(cache: Cache, rows: int, pos: Optional[torch.Tensor] = None, n: Optional[torch.Tensor] = None,
         dtype: torch.dtype = torch.float16, k_out: Optional[torch.Tensor] = None,
         v_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Read cache rows pos[s] .. pos[s] + rows - 1 back as (k, v), f32 or f16
    [slots][rows][kv_heads * 64].  Rows i >= n[s] and rows past max_tok are left as they were
    in k_out / v_out (zero where these are not given)."""
    w = cache.kv_heads * HEAD_DIM
    if (k_out is None) != (v_out is None):
        raise ValueError("k_out and v_out go together")
    if k_out is None:
        if dtype not in _DT or rows < 0:
            raise ValueError(f"{rows} rows of {dtype} (f32 or f16)")
        with _on(stream):
            k_out = torch.zeros((cache.slots, rows, w), dtype=dtype, device=cache.data.device)
            v_out = torch.zeros_like(k_out)
    st = _strides(k_out, "k_out", cache, w)
    if k_out.shape[1] != rows:
        raise ValueError(f"k_out holds {k_out.shape[1]} rows, not {rows}")
    if v_out.shape != k_out.shape or v_out.dtype != k_out.dtype or _strides(v_out, "v_out", cache, w) != st:
        raise ValueError("v_out must match k_out in shape, type and strides")
    args = (_index(pos, "pos", cache), _index(n, "n", cache))
    _device(cache)
    h = cache.handle()
    _lib.check(_lib.load().madi_kv4_load(ctypes.byref(h), k_out.data_ptr(), v_out.data_ptr(), _DT[k_out.dtype], rows,
                                         *st, *args, _stream(stream)), "madi_kv4_load")
    return k_out, v_out


def attn(q: torch.Tensor, cache: Cache, heads: int, pos: Optional[torch.Tensor] = None,
         lens: Optional[torch.Tensor] = None, n: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
         stream=None) -> torch.Tensor:
    """Attention over the cache.  q f32 or f16 [slots][heads * 64] (one query token per slot) or
    [slots][rows][heads * 64]; returns out like q.  Query row i of slot s attends cache rows
    0 .. pos[s] + i (pos: causal), or 0 .. lens[s] - 1 (lens), or all max_tok rows; no row to
    attend gives zeros.  Rows i >= n[s] are padding: left as they were in `out`."""
    one = q.dim() == 2
    qv = q.unsqueeze(1) if one else q
    w = heads * HEAD_DIM
    qs = _strides(qv, "q", cache, w)
    if pos is not None and lens is not None:
        raise ValueError("pos (causal) and lens exclude one another")
    args = (_index(pos, "pos", cache), _index(lens, "lens", cache), _index(n, "n", cache))
    if out is None:
        with _on(stream):
            out = (torch.empty if n is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and type")
    os_ = _strides(out.unsqueeze(1) if one else out, "out", cache, w)
    _device(cache)
    h = cache.handle()
    _lib.check(_lib.load().madi_kv4_attn(ctypes.byref(h), q.data_ptr(), _DT[q.dtype], heads, qv.shape[1], *qs,
                                         *args, out.data_ptr(), *os_, _stream(stream)), "madi_kv4_attn")
    return out
