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
