"""Latent attention where 16-bit probabilities and 32-bit logits run out of range: logits of any finite size, and rows whose
weight is nearly all on one key. Inputs are chosen so that the logits themselves are exact in 32 bits; what may differ from the
definition in 64 bits is then the rounding of the output and of the probabilities (tests/test_latent_gpu.py), and that of the
exponents: 2^-24 of a difference of logits, counted below 2^-18 for the differences that matter (up to 64)."""
import math

import pytest
import torch

from test_latent_gpu import DT, _check, _gen

pytestmark = pytest.mark.gpu


def _cu(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n,past", [(300, 0), (64, 4000)])            # whole and with the keys split
@pytest.mark.parametrize("dtype,e,f", [("bf16", 1, 1), ("bf16", 8, 2), ("bf16", 9, 9), ("bf16", 12, 11), ("bf16", 17, 17),
                                       ("bf16", 40, 40), ("f16", 1, 1), ("f16", 8, 2), ("f16", 9, 8), ("f16", 13, 8), ("f16", 15, 8)])
def test_prefill_over_logits_of_any_size(dtype, e, f, n, past):
    """Logits are multiples of 2^(e + f) up to 96 of them: beyond 2^24 a score times the scale rounds to whole powers of 2."""
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    dt, u = DT[dtype]
    g = _gen(e + f)
    for order in ("random", "rising", "falling"):
        q = torch.zeros(n, 2, 64, device="cuda")
        q[..., 0] = 2.0 ** e
        k = torch.zeros(n + past, 2, 64, device="cuda")
        k[..., 0] = torch.randint(-96, 97, (n + past, 2), generator=g, device="cuda") * 2.0 ** f
        if order != "random":
            k = k.sort(0, descending=order == "falling").values
        v = torch.randn(n + past, 2, 64, generator=g, device="cuda")
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
        cu_q, cu_k = _cu(0, n), _cu(0, n + past)
        out = latent_attention_prefill(q, k, None, v, cu_q, cu_k, n, 1.0)
        ref, absolute = O.prefill(q, k, None, v, cu_q, cu_k, 1.0)
        _check(out, ref, absolute, u, u, 2.0 ** -18, 64)


# ------------------------------------------------------------------------------- one key with nearly all the weight
# Probabilities in fp16 are held with their row's maximum at 2^7 or above (at most 2^15): above 2^-21 of it they round by 2^-11 of themselves,
# below by up to 2^-32 of it. The 2-norm counts both as independent (the values are), the first twice for good measure, and half a step
# of the output's smallest values.
@pytest.mark.parametrize("n,past", [(200, 0), (1000, 0), (64, 4000)])
@pytest.mark.parametrize("gap", [8, 10, 12, 14, 16, 18, 20])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prefill_beside_a_key_without_a_value(dtype, gap, n, past):
    """The first key is `gap` above the others' logits (e^gap times a weight) and its value is zero: the output is
    what the others leave."""
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    dt, u = DT[dtype]
    g = _gen(gap)
    S, scale, heads, d = n + past, 0.125, 2, 64
    q = torch.randn(n, heads, d, generator=g, device="cuda") * 0.3
    k = torch.randn(S, heads, d, generator=g, device="cuda")
    v = torch.randn(S, heads, d, generator=g, device="cuda").to(dt)
    q[..., 0], k[..., 0], k[0], v[0] = 8.0, 0.0, 0.0, 0.0
    k[0, :, 0] = gap
    q, k = q.to(dt), k.to(dt)
    out = latent_attention_prefill(q, k, None, v, _cu(0, n), _cu(0, S), n, scale).double()
    z = torch.einsum("ihd,jhd->hij", q.double(), k.double()) * scale
    hidden = torch.arange(S, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + past
    p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
    sums = lambda w, x: torch.einsum("hij,jhd->ihd", w, x)  # noqa: E731
    v = v.double()
    ref, absolute, square = sums(p, v), sums(p, v.abs()), sums(p * p, v * v).sqrt()
    seen = sums((~hidden).double().expand_as(p), v * v).sqrt()
    dz = d * 2.0 ** -23 * scale * 0.3 * 8 * 2 * 8 * 2                 # of the keys but the first: norms under 0.6 * 8 and 2 * 8
    tiny = 2.0 ** -32 if dtype == "f16" else 0.0
    bound = u * ref.norm() + 2 * u * square.norm() + (2 * dz / math.sqrt(d) + 1e-5) * absolute.norm() + tiny * seen.norm()
    bound += 2.0 ** -25 * math.sqrt(out.numel()) if dtype == "f16" else 0.0
    assert torch.isfinite(out).all()
    assert (out - ref).norm() <= bound, ((out - ref).norm() / bound).item()


@pytest.mark.parametrize("q_scale", [1e-3, 10.0, 100.0])
@pytest.mark.parametrize("qlens,prefix", [([333], [77]), ([140], [4000])])
def test_fp16_prefill_over_flat_and_peaked_rows(q_scale, qlens, prefix):
    from test_latent_gpu import _prefill_case
    _prefill_case(qlens, prefix, 3, 128, 64, 128, "f16", 71, q_scale=q_scale)


@pytest.mark.parametrize("n,past", [(1000, 0), (64, 4000)])
def test_fp16_prefill_rising_logits(n, past):
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    heads, S, g = 2, n + past, _gen(74)
    q = torch.randn(n, heads, 144, generator=g, device="cuda").half()
    kv = torch.randn(S, heads, 256, generator=g, device="cuda").half()
    kr = torch.zeros(S, 16, device="cuda")
    kr[:, 0] = torch.arange(S, device="cuda") / 4
    kr = kr.half()
    for sign in (1.0, -1.0):
        q[..., 128] = sign * 8.0
        out = latent_attention_prefill(q, kv[..., :128], kr, kv[..., 128:], _cu(0, n), _cu(0, S), n, 0.25)
        ref, absolute = O.prefill(q, kv[..., :128], kr, kv[..., 128:], _cu(0, n), _cu(0, S), 0.25)
        _check(out, ref, absolute, 2.0 ** -11, 2.0 ** -11, 144 * 2.0 ** -23 * 0.25 * 30 * (S / 4 + 50), 144)


# ------------------------------------------------------------------------------- absorbed form
def _unit_scale():
    """A scale whose product with log2(e), both in 32 bits, rounds to 1."""
    import numpy as np
    log2e = np.float32(1.4426950408889634)
    s = np.float32(1.0) / log2e
    for s in (s, np.nextafter(s, np.float32(0)), np.nextafter(s, np.float32(1))):
        if np.float32(s * log2e) == 1.0:
            return float(s)
    raise AssertionError("no such scale")


@pytest.mark.parametrize("heads", [16, 24, 64])                        # narrow kernel, 32 and 64 query rows a block
@pytest.mark.parametrize("dtype,e", [("bf16", 20), ("bf16", 24), ("bf16", 25), ("bf16", 26), ("bf16", 27), ("bf16", 29), ("f16", 20),
                                     ("f16", 24), ("f16", 25)])
def test_decode_over_logits_of_any_size(dtype, e, heads):
    """Logits of 2^e, in log2 units, that grow over a block's tiles by less than what raises the running maximum and by
    more, in multiples of what 32 bits resolve there (so that every sum of the two products behind a logit is exact)."""
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    from vq2_vllm.kernels.latent_cache import LatentCache
    dt, u = DT[dtype]
    L, R, n, g = 64, 8, 64 * 296 * 4, _gen(e)                       # 4 tiles a block, 8 in the wide kernels
    unit = max(4.0, 2.0 ** (e - 23))
    for step in (0, 1, 2, 3, 4, -1):
        c, kr = torch.randn(n, L, generator=g, device="cuda"), torch.zeros(n, R, device="cuda")
        kr[:, 0] = 2.0 ** 10
        kr[:, 1] = (7 + step * (torch.arange(n, device="cuda") // 64 % 4)) * unit / 4.0
        cache = LatentCache.alloc(n, 1, L, R)
        cache.data[:, 0] = O.pack_rows(c, kr)
        table = torch.arange(n, dtype=torch.int32, device="cuda")[None]
        q = torch.zeros(1, 1, heads, L + R, device="cuda")
        q[..., L], q[..., L + 1] = 2.0 ** (e - 10), 4.0
        q = q.to(dt)
        kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
        out = latent_attention_decode(q, cache, table, kv_len, _unit_scale())
        k = torch.cat(O.unpack_rows(cache.data[:, 0], L, R), 1)
        z = (q[0, 0].double() @ k.T) * math.log(2.0)
        p = torch.softmax(z, -1)
        _check(out, (p @ k[:, :L])[None, None], (p @ k[:, :L].abs())[None, None], u, 2.0 ** -11, 2.0 ** -18, L + R, True)
