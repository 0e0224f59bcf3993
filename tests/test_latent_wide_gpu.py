"""Absorbed latent attention through its wide kernels (32 and 64 query rows a block), against the definition in 64 bits. A call goes
there where the block table has room for more tiles than the narrow kernel is meant for, so the tables here are
padded with columns that no length reaches. Tolerances: tests/test_latent_gpu.py."""
import math

import pytest
import torch

from test_latent_gpu import DT, _check, _gen

pytestmark = pytest.mark.gpu


def _widen(table, page, rows):
    """The table with columns for `rows` cached rows; those beyond a sequence's length are never looked at."""
    wide = torch.full((table.shape[0], -(-rows // page)), -1, dtype=torch.int32, device=table.device)
    wide[:, : table.shape[1]] = table
    return wide


# ------------------------------------------------------------------------------- rows that are not there
def _listed(n, seed, L=128, R=16):
    """n cached rows in single-row pages, in random order. A rotary value of 1 gives every row a logit of about -20 under
    the queries of `_queries`: a row that counted with logit 0 would take nearly all the weight."""
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_cache import LatentCache
    g = _gen(seed)
    cache = LatentCache.alloc(n + 3, 1, L, R)
    c, kr = torch.randn(n, L, generator=g, device="cuda"), torch.randn(n, R, generator=g, device="cuda")
    kr[:, 0] = 1.0
    table = torch.randperm(n, generator=g, device="cuda").int()[None] + 3
    cache.data[table[0].long(), 0] = O.pack_rows(c, kr)
    return cache, table


def _queries(T, heads, dt, seed, L=128, R=16):
    q = torch.randn(1, T, heads, L + R, generator=_gen(seed), device="cuda")
    q[..., L] = -200.0
    return q.to(dt)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,heads", [(1, 24), (2, 16), (1, 64), (3, 30)])
@pytest.mark.parametrize("n", [64 * 20, 64 * 31 + 17])
def test_rows_on_pages_outside_the_cache_are_masked_in_every_tile(dtype, T, heads, n):
    """A third of each tile's rows have no page, most of them the same rows as in the tiles next to it: a tile's mark must
    outlast the marking of the tile that follows it in the same place."""
    from oracle import latent_ref as O
    from vq2_vllm import _lib
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    lib, (dt, u) = _lib.lib(), DT[dtype]
    L, R, scale = 128, 16, 0.1
    cache, table = _listed(n, 3)
    q = _queries(T, heads, dt, 5)
    at = torch.arange(n, device="cuda")
    for k in range(8):
        g = _gen(100 + k)
        bad = (at % 64) % 3 == k % 3
        bad ^= torch.rand(n, generator=g, device="cuda") < 0.1
        listed = torch.where(bad, torch.where(at % 2 == 0, -1, cache.data.shape[0]).int(), table[0])[None]
        kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
        lib.vq2_device_status(1)
        out = latent_attention_decode(q, cache, _widen(listed, 1, 64 * 1600), kv_len, scale)
        assert lib.vq2_device_status(1) == 2
        c, kr = O.unpack_rows(cache.data[table[0].long(), 0], L, R)
        keys = torch.cat((c, kr), 1)
        z = (q[0].double().reshape(T * heads, -1) @ keys.T) * scale
        last = (n - T + torch.arange(T, device="cuda")).repeat_interleave(heads)
        z = z.masked_fill(bad[None] | (at[None] > last[:, None]), -math.inf)
        p = torch.softmax(z, -1)
        dz = (2.0 ** -11 + (L + R) * 2.0 ** -23) * scale * q.double().norm(dim=-1).max().item() * keys.norm(dim=1).max().item()
        _check(out, p @ c, p @ c.abs(), u, 2.0 ** -11, dz, L + R, True)


@pytest.mark.parametrize("T,heads", [(1, 24), (2, 16), (1, 64), (3, 30)])
def test_a_nan_row_is_not_forgotten_where_the_next_tiles_lack_it(T, heads):
    """A row with a non-finite scale whose places in the two tiles after it are empty: all who see it read NaN."""
    from vq2_vllm import _lib
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    n, L = 64 * 12 + 5, 128
    cache, table = _listed(n, 7)
    q = _queries(T, heads, torch.bfloat16, 9)
    kv_len = torch.tensor([n], dtype=torch.int32, device="cuda")
    for k in range(16):
        row = 64 * (k % 9) + (k * 37) % 64
        data = cache.data.clone()
        cache.data[table[0, row].long()] = 255
        listed = table.clone()
        listed[0, row + 64], listed[0, row + 128] = -1, -1
        wide = _widen(listed, 1, 64 * 1600)
        out = latent_attention_decode(q, cache, wide, kv_len, 0.1)
        assert out.isnan().all()
        cache.data.copy_(data)
        assert torch.isfinite(latent_attention_decode(q, cache, wide, kv_len, 0.1)).all()
    assert _lib.lib().vq2_device_status(1) == 2          # the missing pages
