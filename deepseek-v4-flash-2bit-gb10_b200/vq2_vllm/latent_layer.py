"""A decoder layer with latent attention over the 4-bit cache and vq2 routed experts, the way a serving loop
runs the two halves together.

    layer = LatentLayer.random(H=4096, heads=16, experts=synth.make_layer(...), ...)
    cache = LatentCache.alloc(pages, page_size, layer.L, layer.R)
    y = layer.prefill(x, positions, cache, slots, seq_slots, cu_q, cu_k, max_q)        # prompt chunks, ragged
    y = layer.decode(x, positions, cache, slots, block_table, kv_len)                  # T new tokens a sequence

Both write the new tokens' latents to the cache first and attend to what the cache then holds, so a prompt processed in
chunks, or continued token by token, sees the same keys and values throughout. Projections are plain
library products; attention, cache, router and experts are this package's kernels. The reference plugin serves the
experts only (vq2_vllm/__init__.py:197-218) and leaves the rest of the layer to vLLM.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .kernels.ds4_vq2_cuda import vq2_moe_grouped_wmma
from .kernels.latent_attention import latent_attention_decode, latent_attention_prefill
from .kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
from .kernels.router import router_topk
from .kernels.shared_expert import shared_expert_fused
from .kernels.vq2_kernel import vq2_moe_fused_10b
from .plugin import _WMMA_MIN

_ROUTER_MAX = 64          # tokens the router kernel takes at once


def rms_norm(x: torch.Tensor, gain: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * gain.float()).to(x.dtype)


def rotate_positions(x: torch.Tensor, positions: torch.Tensor, base: float = 10000.0) -> torch.Tensor:
    """Rotary position embedding of x [tokens, .., R]: pairs (i, i + R/2) turned by position * base^(-2 i / R)."""
    half = x.shape[-1] // 2
    freq = base ** (-torch.arange(half, device=x.device, dtype=torch.float32) / max(half, 1))
    angle = (positions.float()[:, None] * freq).reshape(positions.shape[0], *([1] * (x.dim() - 2)), half)
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1).to(x.dtype)


@dataclass
class LatentLayer:
    """Weights of one layer. w_q [H, heads * (nope + rope)], w_kv [H, L + R] (latent, then rotary key), w_uk
    [heads, nope, L] and w_uv [heads, L, dv] (up-projections of the latent), w_o [heads * dv, H], w_r bf16 [H, E],
    experts: the eight vq2 tensors in kernel order, shared: (w13, w2) of the shared expert or None."""
    heads: int
    L: int
    R: int
    nope: int
    dv: int
    norm_in: torch.Tensor
    norm_kv: torch.Tensor
    norm_ffn: torch.Tensor
    w_q: torch.Tensor
    w_kv: torch.Tensor
    w_uk: torch.Tensor
    w_uv: torch.Tensor
    w_o: torch.Tensor
    w_r: torch.Tensor
    topk: int
    experts: tuple
    shared: tuple | None = None

    @classmethod
    def random(cls, H: int, heads: int, experts: tuple, n_experts: int, topk: int, L: int = 512, R: int = 64, nope: int = 128,
               dv: int = 128, shared: tuple | None = None, seed: int = 0, device="cuda") -> "LatentLayer":
        g = torch.Generator(device=device).manual_seed(seed)
        w = lambda *s, fan: (torch.randn(*s, generator=g, device=device) * fan ** -0.5).bfloat16()  # noqa: E731
        one = lambda n: torch.ones(n, device=device, dtype=torch.bfloat16)  # noqa: E731
        return cls(heads, L, R, nope, dv, one(H), one(L), one(H), w(H, heads * (nope + R), fan=H), w(H, L + R, fan=H),
                   w(heads, nope, L, fan=L), w(heads, L, dv, fan=L), w(heads * dv, H, fan=heads * dv), w(H, n_experts, fan=H), topk,
                   experts, shared)

    @property
    def scale(self) -> float:
        return (self.nope + self.R) ** -0.5

    # -------------------------------------------------------------------------------- attention
    def _project(self, x, positions):
        """Normed input -> query [N, heads, nope + R], latent [N, L], rotary key [N, R] (positions applied)."""
        h = rms_norm(x, self.norm_in)
        q = (h @ self.w_q).view(-1, self.heads, self.nope + self.R)
        kv = h @ self.w_kv
        c, k_rope = rms_norm(kv[:, : self.L], self.norm_kv), kv[:, self.L:]
        if self.R:
            q = torch.cat((q[..., : self.nope], rotate_positions(q[..., self.nope:], positions)), -1)
            k_rope = rotate_positions(k_rope, positions)
        return q, c, k_rope

    def attend_prefill(self, x, positions, cache: LatentCache, slots, seq_slots, cu_q, cu_k, max_q):
        """Attention of prompt chunks (expanded form) -> [N, heads * dv]. slots [N]: the new tokens' cache rows;
        seq_slots [Tk]: the rows of every sequence from its start, prefix and chunk, in order (cu_k)."""
        q, c, k_rope = self._project(x, positions)
        latent_cache_write(cache, c, k_rope if self.R else None, slots)
        c_all, rope_all = latent_cache_read(cache, seq_slots, x.dtype)
        k_nope = torch.einsum("tl,hdl->thd", c_all, self.w_uk)
        v = torch.einsum("tl,hld->thd", c_all, self.w_uv)
        o = latent_attention_prefill(q, k_nope, rope_all if self.R else None, v, cu_q, cu_k, max_q, self.scale)
        return o.reshape(-1, self.heads * self.dv)

    def attend_decode(self, x, positions, cache: LatentCache, slots, block_table, kv_len):
        """Attention of T new tokens a sequence (absorbed form), x [B * T, H] sequence by sequence -> [B * T, heads * dv]."""
        q, c, k_rope = self._project(x, positions)
        latent_cache_write(cache, c, k_rope if self.R else None, slots)
        B = kv_len.shape[0]
        q_c = torch.einsum("thd,hdl->thl", q[..., : self.nope], self.w_uk)
        T = x.shape[0] // max(B, 1)
        o = latent_attention_decode(torch.cat((q_c, q[..., self.nope:]), -1).view(B, T, self.heads, self.L + self.R), cache,
                                    block_table, kv_len, self.scale)
        return torch.einsum("thl,hld->thd", o.view(-1, self.heads, self.L), self.w_uv).reshape(-1, self.heads * self.dv)

    # ---------------------------------------------------------------------------------- experts
    def feed_forward(self, x):
        """Router, routed experts and, where the layer has one, the shared expert -> fp32 [N, H]."""
        h = rms_norm(x, self.norm_ffn)
        N = h.shape[0]
        if not N:                              # a step without tokens
            return h.float()
        if N <= _ROUTER_MAX:
            ids, w = router_topk(h, self.w_r, self.topk)
        else:
            w, ids = torch.topk(torch.softmax(h.float() @ self.w_r.float(), -1), self.topk, dim=-1)
            ids = ids.int()
        if N < _WMMA_MIN:
            out = vq2_moe_fused_10b(h, ids, w, *self.experts)
        else:
            out = vq2_moe_grouped_wmma(h, ids, w, *self.experts)
        if self.shared is not None:
            w13, w2 = self.shared
            if N <= 8:
                out = shared_expert_fused(h, w13, w2, out=out)
            else:
                gate, up = (h @ w13.T).float().chunk(2, -1)
                out = out + ((torch.nn.functional.silu(gate) * up).to(h.dtype) @ w2.T).float()
        return out

    # ------------------------------------------------------------------------------------- layer
    def _finish(self, x, attended):
        x = x + attended @ self.w_o
        return (x.float() + self.feed_forward(x)).to(x.dtype)

    def prefill(self, x, positions, cache, slots, seq_slots, cu_q, cu_k, max_q):
        return self._finish(x, self.attend_prefill(x, positions, cache, slots, seq_slots, cu_q, cu_k, max_q))

    def decode(self, x, positions, cache, slots, block_table, kv_len):
        return self._finish(x, self.attend_decode(x, positions, cache, slots, block_table, kv_len))
