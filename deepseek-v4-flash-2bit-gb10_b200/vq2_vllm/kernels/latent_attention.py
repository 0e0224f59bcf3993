"""Latent attention on the B200 library: the absorbed form over the paged 4-bit cache (decode) and the
expanded form over per-head keys and values (prompt chunks).

In latent attention all heads share one latent vector a token: keys are ``c @ W_uk[h]`` beside a shared
rotary key, values ``c @ W_uv[h]``. For a few new tokens the projections move to the query and the
result (``q_c = q_nope @ W_uk[h]^T``, ``o @ W_uv[h]``), and attention reads the latents themselves:
``latent_attention_decode``. For a prompt it is cheaper to project keys and values up once:
``latent_attention_prefill``. No counterpart in the reference plugin, which leaves attention to vLLM.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .latent_cache import MAX_ROPE, LatentCache

_DT = {torch.bfloat16: 0, torch.float16: 1}
MAX_HEAD_DIM = 128


def _i32(t: torch.Tensor, dim: int, what: str):
    if t.dim() != dim or t.dtype not in _lib.ID:
        raise ValueError(f"vq2 latent attention: {what} must be an int32 tensor of {dim} dimension(s)")
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


@functools.lru_cache(maxsize=1024)
def _prefill_workspace_size(B: int, heads: int, dv: int, max_q: int, Tq: int, Tk: int) -> int:
    return _lib.lib().vq2_latent_prefill_workspace_size(B, heads, dv, max_q, Tq, Tk)


@functools.lru_cache(maxsize=1024)
def _workspace_size(B: int, T: int, heads: int, L: int, R: int) -> int:
    return _lib.lib().vq2_latent_decode_workspace_size(B, T, heads, L, R)


def latent_attention_decode(q: torch.Tensor, cache: LatentCache, block_table: torch.Tensor, kv_len: torch.Tensor,
                            scale: float) -> torch.Tensor:
    """Absorbed form: q [B, T, heads, latent_dim + rope_dim] (bf16 / fp16; the T newest tokens of each
    sequence, whose rows are in the cache already), block_table int32 [B, max_pages] and kv_len int32 [B]
    on the GPU -> [B, T, heads, latent_dim] of q's dtype:

        out = sum_j softmax_j(scale * (q_c . c_j + q_r . r_j)) c_j,   j <= kv_len - T + t

    A sequence of length 0 (or a row that sees nothing) gives zeros; rows of the cache past kv_len are never
    used, whatever they hold. ``scale`` is positive. fp16 queries are held in two terms, which costs up to half as much
    time again as bf16. Three launches; nothing waits for the host: safe to capture in
    a CUDA graph. The kernel is chosen by the table's width, not by kv_len: a table cut to the longest sequence of the batch
    keeps short contexts on the one with less latency (64 rows of one sequence: 11 us on the device, 17 with a wide table)."""
    L, R = cache.latent_dim, cache.rope_dim
    if not scale > 0:
        raise ValueError("vq2 latent attention: scale must be positive")
    if q.dim() != 4 or q.dtype not in _DT or q.shape[3] != L + R:
        raise ValueError(f"vq2 latent attention: q must be bf16 or fp16 [B, T, heads, {L + R}]")
    B, T, heads, _ = q.shape
    block_table, kv_len = _i32(block_table, 2, "block_table"), _i32(kv_len, 1, "kv_len")
    if block_table.shape[0] != B or kv_len.shape[0] != B or block_table.shape[1] < 1:
        raise ValueError("vq2 latent attention: block_table [B, max_pages >= 1] and kv_len [B] expected")
    _lib.require_cuda(q)
    dev = q.get_device()
    _lib.require_cuda(cache.data, block_table, kv_len, device=dev)
    out = torch.empty(B, T, heads, L, dtype=q.dtype, device=q.device)
    if not out.numel():
        return out
    with _lib.on_device(dev):
        if q.data_ptr() % 16 or not q.is_contiguous():
            q = q.clone(memory_format=torch.contiguous_format)
        lib, stream = _lib.lib(), _lib.raw_stream(dev)
        ws = _lib.workspace(_workspace_size(B, T, heads, L, R), q.device, stream)
        k = cache.args
        a = _lib.Vq2LatentDecodeArgs(B, T, heads, L, R, k.page_size, block_table.shape[1], _DT[q.dtype], k.pages, scale, q.data_ptr(),
                                     k.data, block_table.data_ptr(), kv_len.data_ptr(), out.data_ptr())
        rc = lib.vq2_latent_decode(a, ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc, "vq2_latent_decode")
    return out


def _rows(x: torch.Tensor):
    """x [tokens, .., dim] as the kernels can read it, last dimension contiguous and the others in multiples of 16
    bytes (copied if not)."""
    st = x.stride()
    if st[-1] != 1 or min(st) < 1 or any(n % 8 for n in st[:-1]) or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def latent_attention_prefill(q: torch.Tensor, k_nope: torch.Tensor, k_rope: torch.Tensor | None, v: torch.Tensor,
                             cu_q: torch.Tensor, cu_k: torch.Tensor, max_q: int, scale: float) -> torch.Tensor:
    """Expanded form, causal, ragged batch: q [Tq, heads, nope + rope], k_nope [Tk, heads, nope], k_rope [Tk, rope]
    (shared by the heads; None where rope is 0), v [Tk, heads, dv], all bf16 or all fp16 (views with a
    contiguous last dimension are taken as they are) -> [Tq, heads, dv]. Sequence b has query rows
    cu_q[b] .. cu_q[b+1]-1 and key rows cu_k[b] .. cu_k[b+1]-1 (int32 [B+1] on the GPU): its keys are a prefix
    followed by the chunk's own, and query i sees keys up to i + keys - queries. ``max_q`` is the most query
    rows a sequence has; rows of ``q`` outside cu_q, or past max_q in their sequence, are left unset. A row that sees no
    key gives zeros. A NaN or an infinity in a value reaches every row that sees it, may reach earlier rows of its
    sequence whose block of 128 keys it is in (their weight for it is 0, and 0 times it is NaN), and no other sequence's. ``scale`` is
    positive. Dimensions are multiples of 8, nope and dv at most 128, rope at most 64."""
    if q.dtype not in _DT:
        raise ValueError("vq2 latent attention: q must be bf16 or fp16")
    if not scale > 0:
        raise ValueError("vq2 latent attention: scale must be positive")
    if q.dim() != 3 or k_nope.dim() != 3 or v.dim() != 3:
        raise ValueError("vq2 latent attention: q, k_nope and v must be [tokens, heads, dim]")
    Tq, heads, dq = q.shape
    Tk, _, dn = k_nope.shape
    dv = v.shape[2]
    if v.shape[:2] != k_nope.shape[:2] or k_nope.shape[1] != heads:
        raise ValueError("vq2 latent attention: k_nope and v must be [key tokens, heads, dim] with q's heads")
    R = dq - dn
    if not (0 < dn <= MAX_HEAD_DIM and 0 < dv <= MAX_HEAD_DIM and 0 <= R <= MAX_ROPE) or dn % 8 or dv % 8 or R % 8:
        raise ValueError(f"vq2 latent attention: nope {dn} and v {dv} must be multiples of 8 up to {MAX_HEAD_DIM}, rope {R} one up "
                         f"to {MAX_ROPE}")
    if R and (k_rope is None or k_rope.shape != (Tk, R)):
        raise ValueError(f"vq2 latent attention: k_rope must be [{Tk}, {R}]")
    if k_nope.dtype != q.dtype or v.dtype != q.dtype or (R and k_rope.dtype != q.dtype):
        raise ValueError("vq2 latent attention: q, k_nope, k_rope and v must have one dtype")
    cu_q, cu_k = _i32(cu_q, 1, "cu_q"), _i32(cu_k, 1, "cu_k")
    B = cu_q.shape[0] - 1
    if B < 0 or cu_k.shape[0] != B + 1 or max_q < 0:
        raise ValueError("vq2 latent attention: cu_q and cu_k [B + 1] and max_q >= 0 expected")
    _lib.require_cuda(q)
    dev = q.get_device()
    _lib.require_cuda(k_nope, v, cu_q, cu_k, *((k_rope,) if R else ()), device=dev)
    out = torch.empty(Tq, heads, dv, dtype=q.dtype, device=q.device)
    if not out.numel() or not B:
        return out
    with _lib.on_device(dev):
        q, k_nope, v = _rows(q), _rows(k_nope), _rows(v)
        if R:
            k_rope = _rows(k_rope)
        stream, nb = _lib.raw_stream(dev), _prefill_workspace_size(B, heads, dv, max_q, Tq, Tk)
        ws = _lib.workspace(nb, q.device, stream).data_ptr() if nb else None
        a = _lib.Vq2LatentPrefillArgs(B, heads, dn, R, dv, max_q, _DT[q.dtype], Tq, Tk, scale, q.stride(0), q.stride(1),
                                      k_nope.stride(0), k_nope.stride(1), v.stride(0), v.stride(1), k_rope.stride(0) if R else 0,
                                      q.data_ptr(), k_nope.data_ptr(), k_rope.data_ptr() if R else None, v.data_ptr(),
                                      cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), ws, nb)
        rc = _lib.lib().vq2_latent_prefill(a, stream)
    _lib.check(rc, "vq2_latent_prefill")
    return out
