"""The 4-bit key/value cache of a decoder layer and the arrays of one step over it.

Counterparts in the reference: the quantised KV codecs (crates/velox-core/src/kv.rs) and the page
tables of its paged cache; format and layout are this library's own (include/velox_sm100.h): NVFP4
as in the weights, 4.5 bits per value."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .errors import ShapeError, Unsupported

HEAD_DIMS = (64, 128)
PAGE_SIZES = (16, 32, 64, 128)


class Kv4Cache:
    """K and V of one layer: ``storage`` is uint8 [pages, kv_heads, page_size / 16, 18 * head_dim].

    ``k_divisor`` / ``v_divisor`` play the part of an NVFP4 tensor's divisor: a group of 16 whose largest
    magnitude is a is stored with the scale e4m3(divisor * a / 6), so magnitudes from 6 * 2**-6 / divisor up to
    2688 / divisor keep the scale's full precision (16: from 0.006 to 168)."""

    __slots__ = ("_storage", "page_size", "head_dim", "kv_heads", "pages", "k_divisor", "v_divisor", "struct", "ref",
                 "device_index")

    def __init__(self, storage: torch.Tensor, page_size: int, head_dim: int, k_divisor: float = 16.0,
                 v_divisor: float = 16.0):
        if head_dim not in HEAD_DIMS or page_size not in PAGE_SIZES:
            raise Unsupported(f"4-bit cache: head_dim {head_dim} (of {HEAD_DIMS}), page_size {page_size} (of {PAGE_SIZES})")
        if storage.dtype != torch.uint8 or storage.dim() != 4 or not storage.is_contiguous():
            raise ShapeError("4-bit cache: expected contiguous uint8 [pages, kv_heads, page_size / 16, 18 * head_dim]")
        pages, kv_heads, blocks, width = storage.shape
        if blocks * 16 != page_size or width != 18 * head_dim or pages <= 0 or kv_heads <= 0:
            raise ShapeError(f"4-bit cache: storage {tuple(storage.shape)} for pages of {page_size} tokens, head_dim {head_dim}")
        if pages * page_size >= 1 << 31:
            raise Unsupported(f"4-bit cache: {pages} pages of {page_size} tokens pass 32-bit slots")
        if not (k_divisor > 0 and v_divisor > 0):
            raise ShapeError("4-bit cache: divisors are positive")
        self._storage, self.page_size, self.head_dim = storage, page_size, head_dim
        self.pages, self.kv_heads = pages, kv_heads
        self.k_divisor, self.v_divisor = float(k_divisor), float(v_divisor)
        self.struct = _lib.Kv4CacheStruct(storage.data_ptr(), pages, page_size, kv_heads, head_dim, self.k_divisor,
                                          self.v_divisor, 0)
        self.ref = C.byref(self.struct)
        self.device_index = storage.get_device()

    @property
    def storage(self) -> torch.Tensor:
        return self._storage

    @classmethod
    def alloc(cls, backend, pages: int, page_size: int, kv_heads: int, head_dim: int, k_divisor: float = 16.0,
              v_divisor: float = 16.0) -> "Kv4Cache":
        if head_dim not in HEAD_DIMS or page_size not in PAGE_SIZES:
            raise Unsupported(f"4-bit cache: head_dim {head_dim} (of {HEAD_DIMS}), page_size {page_size} (of {PAGE_SIZES})")
        storage = torch.zeros(pages, kv_heads, page_size // 16, 18 * head_dim, dtype=torch.uint8, device=backend.device)
        return cls(storage, page_size, head_dim, k_divisor, v_divisor)

    def bytes_per_token(self) -> int:
        return self.kv_heads * 18 * self.head_dim // 16


class Kv4Step:
    """What ``Sm100Backend.kv4_plan`` writes for one step: ``cu`` [requests + 1], ``kv_lens`` [requests],
    ``positions`` and ``slots`` [tokens], ``status`` [1], all int32 on the device."""

    __slots__ = ("_arrays", "requests", "tokens", "addresses")

    def __init__(self, backend, requests: int, tokens: int):
        if requests < 0 or tokens < 0:
            raise ShapeError(f"step of {requests} requests, {tokens} tokens")
        self.requests, self.tokens = requests, tokens
        # ..., status, and the word the blocks of a plan count themselves with
        self._arrays = tuple(torch.zeros(n, dtype=torch.int32, device=backend.device)
                             for n in (requests + 1, requests, tokens, tokens, 1, 1))
        self.addresses = tuple(t.data_ptr() for t in self._arrays)

    cu = property(lambda self: self._arrays[0])
    kv_lens = property(lambda self: self._arrays[1])
    positions = property(lambda self: self._arrays[2])
    slots = property(lambda self: self._arrays[3])
    status = property(lambda self: self._arrays[4])
    ticket = property(lambda self: self._arrays[5])


def rope_table(positions: int, rot: int, theta: float = 1e6, device: Optional[torch.device] = None) -> torch.Tensor:
    """[positions, rot] f32: rot/2 cosines and rot/2 sines of position * theta ** (-2i / rot), angles in f64 (in f32 a
    position of 100,000 is off by up to 0.004 radians)."""
    half = rot // 2
    inv = float(theta) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    a = torch.arange(positions, dtype=torch.float64, device=device).unsqueeze(1) * inv
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()
