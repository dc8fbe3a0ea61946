"""Quantised, paged key/value cache on the HIP kernels, and attention that reads it.

* ``QuantizedKVCache.write``   -> ``mpq_kv_write``: keys and values are quantised as they are written
* ``QuantizedKVCache.read``    -> ``mpq_kv_read``: sequences read back
* ``QuantizedKVCache.attend``  -> ``mpq_kv_attend``: new tokens (a chunk of a prompt, or one a sequence) over the cache

Keys and values are held in ``mxfp4`` or ``mxfp8`` (:mod:`mpq_amd.mx`), in blocks of 32 along the head size.  A
sequence's tokens lie in pages that its row of the block table names; a token's slot is
``page * page_size + place in the page``.  No counterpart in the reference, which ends at the model's weights.

Tensors live on the ROCm device; there is no CPU path.  Nothing here waits for the device: tables, lengths and
slots stay there and are checked by the kernels, which leave out what lies outside the pool.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib, mx, ops

HEAD_SIZES = (64, 128)


def _over(cls, k_codes, k_scales, v_codes, v_scales, fmt, dtype) -> "QuantizedKVCache":
    """A copied or unpickled cache, with the addresses of its own tensors."""
    return cls.from_tensors(k_codes, k_scales, v_codes, v_scales, fmt=fmt, dtype=dtype)


class QuantizedKVCache:
    """A pool of ``num_pages`` pages of ``page_size`` tokens (a power of two from 16).

    ``k_codes`` (pages, heads, page, bytes of a token's codes) and ``k_scales`` (pages, heads, page, dim / 32) hold the
    keys token by token; ``v_codes`` (pages, heads, page / 4, dim / 8, 4, bytes of 8 codes) and ``v_scales``
    (pages, heads, page / 4, dim / 32, 4) the values in groups of four tokens, all uint8.  ``dtype`` (bfloat16 or
    float16) is the type of the keys, values and queries.  A cache keeps these for life (their contents may change):
    the calls hold their addresses."""

    _FIXED = frozenset(("k_codes", "k_scales", "v_codes", "v_scales", "fmt", "dtype", "device", "num_pages", "heads",
                        "page_size", "head_dim", "_f", "_call"))

    def __init__(self, num_pages: int, page_size: int, heads: int, head_dim: int, *, fmt: str = "mxfp8",
                 dtype: torch.dtype = torch.bfloat16, device: Union[str, torch.device] = "cuda") -> None:
        P, H, D = int(page_size), int(heads), int(head_dim)
        if int(num_pages) < 1 or H < 1:
            raise ValueError(f"the cache needs at least one page and one head, got {num_pages} and {heads}")
        if P < 16 or P > 65536 or P & (P - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 65536, got {page_size}")
        if D not in HEAD_SIZES:
            raise ValueError(f"head_dim must be one of {HEAD_SIZES}, got {head_dim}")
        wide = 2 if mx._fmt(fmt) == 0 else 1

        def new(*shape):
            return torch.zeros(int(num_pages), H, *shape, dtype=torch.uint8, device=device)

        self._set(new(P, D // wide), new(P, D // mx.BLOCK), new(P // 4, D // 8, 4, 8 // wide),
                  new(P // 4, D // mx.BLOCK, 4), fmt, dtype)

    @classmethod
    def from_tensors(cls, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                     v_scales: torch.Tensor, *, fmt: str = "mxfp8",
                     dtype: torch.dtype = torch.bfloat16) -> "QuantizedKVCache":
        """A cache over tensors that the caller allocated (used in place).  Where others filled them, NaN is a block's scale
        byte 255: codes 0x7f and 0xff of ``mxfp8`` under another scale byte are not supported (:meth:`attend` may let
        them reach rows that do not see them)."""
        self = cls.__new__(cls)
        self._set(k_codes, k_scales, v_codes, v_scales, fmt, dtype)
        return self

    def __setattr__(self, name: str, value) -> None:
        if name in self._FIXED:
            raise AttributeError(f"{name} of a cache is fixed; QuantizedKVCache.from_tensors makes one over other tensors")
        super().__setattr__(name, value)

    def __delattr__(self, name: str) -> None:
        if name in self._FIXED:
            raise AttributeError(f"{name} of a cache is fixed")
        super().__delattr__(name)

    def __reduce__(self):
        return _over, (type(self), self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.fmt, self.dtype)

    def _set(self, k_codes, k_scales, v_codes, v_scales, fmt, dtype) -> None:
        f = mx._fmt(fmt)
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        if k_codes.dim() != 4:
            raise ValueError(f"k_codes must be (pages, heads, page, bytes), got {tuple(k_codes.shape)}")
        N, H, P, width = k_codes.shape
        wide = 2 if f == 0 else 1
        D = width * wide
        if N < 1 or H < 1 or P < 16 or P > 65536 or P & (P - 1) or D not in HEAD_SIZES:
            raise ValueError(f"k_codes {tuple(k_codes.shape)} are no {fmt} cache: pages of a power of two from 16 "
                             f"tokens, head sizes {HEAD_SIZES}")
        shapes = ((N, H, P, width), (N, H, P, D // mx.BLOCK), (N, H, P // 4, D // 8, 4, 8 // wide),
                  (N, H, P // 4, D // mx.BLOCK, 4))
        tensors = (k_codes, k_scales, v_codes, v_scales)
        at = [t.data_ptr() for t in tensors]
        for i, t in enumerate(tensors):
            if t.shape != shapes[i] or t.dtype != torch.uint8 or not t.is_contiguous() or at[i] % 16:
                raise ValueError(f"{('k_codes', 'k_scales', 'v_codes', 'v_scales')[i]} must be a contiguous, 16-byte "
                                 f"aligned uint8 tensor of shape {shapes[i]}, got {t.dtype} {tuple(t.shape)}")
        self.__dict__.update(device=mx._on_device(*tensors), k_codes=k_codes, k_scales=k_scales, v_codes=v_codes,
                             v_scales=v_scales, fmt=fmt, dtype=dtype, num_pages=N, heads=H, page_size=P, head_dim=D,
                             _f=f, _call=(f, H, D, P, N, *at))

    def _tokens(self, t: torch.Tensor, name: str, heads: Optional[int] = None) -> torch.Tensor:
        """(tokens, heads, dim) with a contiguous last dimension."""
        if t.dim() != 3 or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{name} must be (tokens, {'heads' if heads is None else heads}, {self.head_dim}), got "
                             f"{tuple(t.shape)}")
        if t.dtype != self.dtype:
            raise ValueError(f"{name} must be {self.dtype}, got {t.dtype}")
        return t if t.stride(2) == 1 else t.contiguous()

    @staticmethod
    def _index(t: torch.Tensor, name: str, dtype: torch.dtype, n: int) -> torch.Tensor:
        if t.dtype != dtype or t.shape != (n,):
            raise ValueError(f"{name} must be a {dtype} tensor of shape ({n},), got {t.dtype} {tuple(t.shape)}")
        return t if t.is_contiguous() else t.contiguous()

    @staticmethod
    def _table(t: torch.Tensor) -> torch.Tensor:
        if t.dtype != torch.int32 or t.dim() != 2:
            raise ValueError(f"block_table must be a 2-D int32 tensor, got {t.dtype} {tuple(t.shape)}")
        return t if t.is_contiguous() else t.contiguous()

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise keys and values (tokens, heads, dim; any token and head strides) into ``slots`` (tokens, int64).
        A slot outside the pool (-1 for padding) is skipped.  The others must be distinct: two tokens written to one slot
        at once leave a mixture of both there (codes of one under scales of the other)."""
        k, v = self._tokens(k, "k", self.heads), self._tokens(v, "v", self.heads)
        if k.shape != v.shape:
            raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
        n = k.shape[0]
        slots = self._index(slots, "slots", torch.int64, n)
        dev = mx._on_device(self.k_codes, k, v, slots)
        if n:
            kt, kh, _ = k.stride()
            vt, vh, _ = v.stride()
            with ops.on_device(dev):
                _lib.check(_lib.load().mpq_kv_write(k.data_ptr(), v.data_ptr(), mx.DTYPES[self.dtype], n, kt, kh, vt, vh,
                                                    slots.data_ptr(), *self._call, ops.raw_stream(dev)),
                           "mpq_kv_write")

    def read(self, block_table: torch.Tensor, starts: torch.Tensor, total: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys and values (total, heads, dim) of the sequences in ``block_table`` (batch, pages; int32), one after the
        other: sequence i fills ``starts[i]`` to ``starts[i + 1]`` (batch + 1, int32) with its first positions.
        Tokens whose page the table does not name are zeros."""
        block_table = self._table(block_table)
        (B, W), total = block_table.shape, int(total)
        if total < 0 or (total and B == 0):
            raise ValueError(f"total must be the tokens of {B} sequences, got {total}")
        starts = self._index(starts, "starts", torch.int32, B + 1)
        dev = mx._on_device(self.k_codes, block_table, starts)
        k = torch.empty((total, self.heads, self.head_dim), dtype=self.dtype, device=dev)
        v = torch.empty((total, self.heads, self.head_dim), dtype=self.dtype, device=dev)
        if total:
            with ops.on_device(dev):
                _lib.check(_lib.load().mpq_kv_read(block_table.data_ptr(), B, W, starts.data_ptr(), total, *self._call,
                                                   k.data_ptr(), v.data_ptr(), mx.DTYPES[self.dtype],
                                                   ops.raw_stream(dev)), "mpq_kv_read")
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor,
               max_q: int, *, scale: Optional[float] = None, causal: bool = True, max_kv: Optional[int] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of the new tokens ``q`` (tokens, query heads, dim) over the cache that already holds them.

        Sequence i is the tokens ``q_starts[i]`` to ``q_starts[i + 1]`` (batch + 1, int32, in rising order; no sequence
        has more than ``max_q``) over the positions below ``kv_lens[i]`` (batch, int32) of its row of ``block_table``.
        Tokens before the first sequence, behind the last one (a batch padded to a captured size) or behind ``max_q``
        of their sequence see nothing. Query heads h * G to h * G + G - 1 read key/value head h. With ``causal`` the
        last new token sees every position, the one before it all but the last, and so on. ``scale`` defaults to
        ``dim ** -0.5``. ``max_kv`` is the longest length if the caller knows it (default: what the table can hold); the work
        is split by it. A row that sees nothing is 0. With ``return_lse`` the logarithm of each row's sum of
        exponentials (tokens, query heads; float32) comes too. A backward pass through the results raises (a given
        ``out`` is left out of it)."""
        q = self._tokens(q, "q")
        block_table = self._table(block_table)
        B, W = block_table.shape
        T, Hq, D = q.shape
        max_q, most = int(max_q), W * self.page_size
        if Hq < 1 or Hq % self.heads:
            raise ValueError(f"{Hq} query heads do not share {self.heads} key/value heads")
        kv_lens = self._index(kv_lens, "kv_lens", torch.int32, B)
        q_starts = self._index(q_starts, "q_starts", torch.int32, B + 1)
        if max_q < 0 or max_q * B < T:
            raise ValueError(f"{T} tokens do not fit {B} sequences of up to {max_q}")
        max_kv = most if max_kv is None else int(max_kv)
        if max_kv < 0 or max_kv > most:
            raise ValueError(f"max_kv must be between 0 and the table's {most} positions, got {max_kv}")
        dev = mx._on_device(self.k_codes, q, block_table, kv_lens, q_starts, out)
        fresh = out is None
        if fresh:
            out = torch.empty((T, Hq, D), dtype=self.dtype, device=dev)
        elif out.shape != q.shape or out.dtype != self.dtype or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {self.dtype} tensor of shape {(T, Hq, D)}")
        lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
        if T:
            lib = _lib.load()
            max_q = min(max_q, T)
            need = lib.mpq_kv_attend_workspace_size(T, B, max_q, max_kv, Hq, self.heads, D)
            ws = ops.workspace(need, dev) if need else None
            qt, qh, _ = q.stride()
            with ops.on_device(dev):
                _lib.check(lib.mpq_kv_attend(q.data_ptr(), mx.DTYPES[self.dtype], T, qt, qh, Hq, B,
                                             block_table.data_ptr(), W, kv_lens.data_ptr(), q_starts.data_ptr(), max_q,
                                             max_kv, *self._call, D ** -0.5 if scale is None else float(scale),
                                             1 if causal else 0, out.data_ptr(),
                                             None if lse is None else lse.data_ptr(),
                                             None if ws is None else ws.data_ptr(), need, ops.raw_stream(dev)),
                           "mpq_kv_attend")
        if q.requires_grad:
            out = mx._no_gradient("QuantizedKVCache.attend", out, q) if fresh else out
            lse = mx._no_gradient("QuantizedKVCache.attend", lse, q) if return_lse else None
        return (out, lse) if return_lse else out
