"""Paged 4-bit cache of attention latents on the B200 library: quantise as it is written, read back.

A decoder layer with latent attention keeps one latent vector ``c`` and one rotary key ``k_rope`` a
token. Here a token's row holds ``c`` in 4 bits (every 64 values rotated by the normalised Hadamard
matrix, as the expert weights are, with one fp16 scale) and ``k_rope`` in fp16: 400 bytes for 512 + 64
values instead of 1152 in bf16. The byte layout is in ``include/vq2_b200.h``. The reference plugin leaves
attention and its cache to vLLM, so these entries have no counterpart there.
"""
from __future__ import annotations

import torch

from .. import _lib

MAX_LATENT, MAX_ROPE = 512, 64


def latent_row_bytes(latent_dim: int, rope_dim: int) -> int:
    """Bytes of one cached row; raises for dimensions the cache does not hold (latent_dim a multiple of
    64 up to 512, rope_dim a multiple of 8 up to 64, or 0)."""
    if not (0 < latent_dim <= MAX_LATENT and latent_dim % 64 == 0 and 0 <= rope_dim <= MAX_ROPE and rope_dim % 8 == 0):
        raise ValueError(f"vq2 latent cache: latent_dim {latent_dim} must be a multiple of 64 up to {MAX_LATENT} and "
                         f"rope_dim {rope_dim} a multiple of 8 up to {MAX_ROPE}")
    return (latent_dim // 2 + 2 * rope_dim + 2 * (latent_dim // 64) + 15) // 16 * 16


class LatentCache:
    """A paged latent cache: ``data`` u8 [pages, page_size, row_bytes], contiguous, on the GPU. Any
    page size >= 1. A slot is ``page * page_size + place``. ``LatentCache.alloc`` makes one. Another tensor may be assigned to
    ``data`` (a grown pool); it is checked like the first, and calls use it from then on. The dimensions stay."""

    __slots__ = ("_data", "_latent_dim", "_rope_dim", "args")

    def __init__(self, data: torch.Tensor, latent_dim: int, rope_dim: int):
        self._latent_dim, self._rope_dim = latent_dim, rope_dim
        self.data = data

    latent_dim = property(lambda self: self._latent_dim)
    rope_dim = property(lambda self: self._rope_dim)

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @data.setter
    def data(self, data: torch.Tensor):
        L, R = self._latent_dim, self._rope_dim
        rb = latent_row_bytes(L, R)
        if data.dtype != torch.uint8 or data.dim() != 3 or data.shape[2] != rb or not data.is_contiguous():
            raise ValueError(f"vq2 latent cache: contiguous uint8 [pages, page_size, {rb}] expected")
        if data.shape[0] < 1 or data.shape[1] < 1:
            raise ValueError("vq2 latent cache: at least one page of at least one row expected")
        # what the calls pass on: the pointer and the sizes of one and the same tensor
        self._data, self.args = data, _lib.Vq2LatentCache(data.data_ptr(), data.shape[0], data.shape[1], L, R)

    @classmethod
    def alloc(cls, pages: int, page_size: int, latent_dim: int, rope_dim: int, device="cuda") -> "LatentCache":
        data = torch.zeros(pages, page_size, latent_row_bytes(latent_dim, rope_dim), dtype=torch.uint8, device=device)
        return cls(data, latent_dim, rope_dim)


def _slots(slots: torch.Tensor):
    if slots.dim() != 1 or slots.dtype not in _lib.ID:
        raise ValueError("vq2 latent cache: slots must be int32 or int64 [N]")
    return slots if slots.is_contiguous() else slots.contiguous()


def _rows(x: torch.Tensor):
    """x [N, D] as rows the kernels can load 16 bytes at a time (a copy only where they cannot), and their stride."""
    if x.is_contiguous():                  # (of a single row the tensor's own stride may be anything)
        return x if x.data_ptr() % 16 == 0 else x.clone(), x.shape[1]
    s0, s1 = x.stride()
    if x.data_ptr() % 16 or s1 != 1 or s0 < x.shape[1] or s0 % 8:
        x = x.clone(memory_format=torch.contiguous_format)
        s0 = x.shape[1]
    return x, s0


def latent_cache_write(cache: LatentCache, c: torch.Tensor, k_rope: torch.Tensor | None, slots: torch.Tensor) -> None:
    """Quantise ``c`` [N, latent_dim] and ``k_rope`` [N, rope_dim] (bf16 / fp16 / fp32, rows may be strided;
    None where rope_dim is 0) into the cache rows ``slots`` [N] (int32 / int64; negative: skipped). A slot
    beyond the cache is skipped and reported by ``vq2_device_status``. Slots in one call must differ."""
    L, R = cache.latent_dim, cache.rope_dim
    dt = _lib.DT.get(c.dtype)
    if c.dim() != 2 or c.shape[1] != L or dt is None:
        raise ValueError(f"vq2 latent cache: c must be bf16 / fp16 / fp32 [N, {L}]")
    N = c.shape[0]
    if R and (k_rope is None or k_rope.shape != (N, R) or k_rope.dtype != c.dtype):
        raise ValueError(f"vq2 latent cache: k_rope must be [N, {R}] of c's dtype")
    slots = _slots(slots)
    if slots.shape[0] != N:
        raise ValueError("vq2 latent cache: one slot per row expected")
    _lib.require_cuda(cache.data)
    dev = cache.data.get_device()
    _lib.require_cuda(c, slots, device=dev)
    if R:
        _lib.require_cuda(k_rope, device=dev)
    if not N:
        return
    with _lib.on_device(dev):
        c, c_stride = _rows(c)
        rope_stride = 0
        if R:
            k_rope, rope_stride = _rows(k_rope)
        rc = _lib.lib().vq2_latent_cache_write(cache.args, c.data_ptr(), k_rope.data_ptr() if R else None, dt, c_stride, rope_stride,
                                               slots.data_ptr(), _lib.ID[slots.dtype], N, _lib.raw_stream(dev))
    _lib.check(rc, "vq2_latent_cache_write")


def latent_cache_read(cache: LatentCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The values that cache rows ``slots`` [N] stand for -> (c [N, latent_dim], k_rope [N, rope_dim]) of
    ``dtype`` (bf16 / fp16 / fp32): what the expanded form projects up for a cached prefix. A negative slot, or
    one beyond the cache (reported by ``vq2_device_status``), gives zeros. N < 2^27."""
    dt = _lib.DT.get(dtype)
    if dt is None:
        raise ValueError("vq2 latent cache: dtype must be bf16, fp16 or fp32")
    slots = _slots(slots)
    _lib.require_cuda(cache.data)
    dev = cache.data.get_device()
    _lib.require_cuda(slots, device=dev)
    N = slots.shape[0]
    c = torch.empty(N, cache.latent_dim, dtype=dtype, device=slots.device)
    k_rope = torch.empty(N, cache.rope_dim, dtype=dtype, device=slots.device)
    if N:
        with _lib.on_device(dev):
            rc = _lib.lib().vq2_latent_cache_read(cache.args, slots.data_ptr(), _lib.ID[slots.dtype], N, c.data_ptr(),
                                                  k_rope.data_ptr() or None, dt, _lib.raw_stream(dev))
        _lib.check(rc, "vq2_latent_cache_read")
    return c, k_rope
