"""Absorbed latent attention through its wide kernels (32 and 64 query rows a block), against the definition in 64 bits. A call goes
there where the block table has room for more tiles than the narrow kernel is meant for, so the tables here are
padded with columns that no length reaches. Tolerances: tests/test_latent_gpu.py."""
import math

import pytest
import torch

from test_latent_gpu import DT, _cache_for, _check, _dz, _gen

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


# ------------------------------------------------------------------------------- against the definition
def _wide(q, table, page, nq):
    """The table as wide as the kernel for `nq` query rows a block needs it, and a check that the call takes that one."""
    from vq2_vllm import _lib
    B, T, heads, _ = q.shape
    lib, dt = _lib.lib(), {torch.bfloat16: 0, torch.float16: 1}[q.dtype]
    rows = 64
    while lib.vq2_latent_decode_query_rows(B, T, heads, -(-rows // page), page, dt) == 16 and rows < 1 << 22:
        rows += 64
    table = _widen(table, page, max(rows, table.shape[1] * page))
    assert lib.vq2_latent_decode_query_rows(B, T, heads, table.shape[1], page, dt) == nq
    return table


def _case(lens, T, heads, L, R, page, dtype, seed, nq, q_scale=1.0, spread=1.0, scale=None):
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    dt, u = DT[dtype]
    cache, table, kv_len = _cache_for(lens, L, R, page, dt, seed, spread)
    q = (torch.randn(len(lens), T, heads, L + R, generator=_gen(seed + 1), device="cuda") * q_scale).to(dt)
    scale = (L // 4 + R) ** -0.5 if scale is None else scale
    table = _wide(q, table, page, nq)
    out = latent_attention_decode(q, cache, table, kv_len, scale)
    assert out.dtype == dt and out.shape == (len(lens), T, heads, L)
    ref, absolute = O.decode(q, cache.data, table, kv_len, scale, L, R)
    _check(out, ref, absolute, u, 2.0 ** -11, _dz(q, cache, table, kv_len, scale, L, R), L + R, True)
    return q, cache, table, kv_len, scale, out


SIZES = [
    # lens, T, heads, L, R, page
    ([1], 1, 17, 64, 0, 1),
    ([64], 1, 32, 512, 64, 64),                          # exactly one tile
    ([65, 63, 0, 1], 2, 16, 512, 64, 64),                # one over, one under, empty, one row
    ([2, 40, 3, 0, 200], 4, 5, 192, 8, 16),              # fewer rows than new tokens
    ([5000, 17], 1, 24, 448, 64, 1),                     # single-row pages
    ([1000, 900, 800], 3, 9, 320, 40, 7),
    ([20000], 1, 32, 512, 0, 64),                        # some 2 tiles a block
    ([70000, 3], 2, 16, 64, 16, 48),                     # 8 tiles a block, a block with both sequences
    ([129, 700, 0, 0, 31, 2000] * 4, 1, 20, 128, 16, 16),
]
MORE = [
    ([1], 1, 33, 64, 0, 1),
    ([64], 1, 64, 512, 64, 64),
    ([65, 63, 0, 1], 3, 64, 512, 64, 64),
    ([2, 40, 3, 0, 200], 7, 5, 192, 8, 16),
    ([5000, 17], 1, 65, 448, 64, 1),
    ([1000, 900, 800], 2, 96, 320, 40, 7),
    ([20000], 1, 64, 512, 0, 64),
    ([70000, 3], 2, 32, 64, 16, 48),
    ([129, 700, 0, 0, 31, 2000] * 4, 1, 40, 128, 16, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,T,heads,L,R,page", SIZES)
def test_up_to_32_query_rows(dtype, lens, T, heads, L, R, page):
    _case(lens, T, heads, L, R, page, dtype, sum(lens) + heads, 32)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,T,heads,L,R,page", MORE)
def test_more_than_32_query_rows(dtype, lens, T, heads, L, R, page):
    _case(lens, T, heads, L, R, page, dtype, sum(lens) + heads, 64 if dtype == "bf16" else 32)


@pytest.mark.parametrize("heads,nq", [(16, 32), (30, 64)])
@pytest.mark.parametrize("q_scale,spread,scale", [(20.0, 1.0, 0.1), (1e-3, 1.0, None), (1.0, 50.0, 1e-3), (300.0, 1.0, 1e-3),
                                                  (1.0, 0.02, 1.0)])
def test_peaked_flat_large_and_small_values(heads, nq, q_scale, spread, scale):
    _case([30777, 130], 2, heads, 512, 64, 64, "bf16", 21, nq, q_scale=q_scale, spread=spread, scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [16, 30])
@pytest.mark.parametrize("L", [64, 320])
def test_rising_and_falling_logits(dtype, heads, L):
    """Logits that rise from tile to tile, within a block's tiles too: O is rescaled each time."""
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    dt, u = DT[dtype]
    R, n, page, scale = 16, 64 * 148 * 5 + 9, 32, 0.5
    cache, table, kv_len = _cache_for([n], L, R, page, dt, 31)
    at = torch.arange(n, device="cuda")
    kr = torch.zeros(n, R, device="cuda")
    kr[:, 0] = (at % 1024).float() / 8
    cache.data.view(-1, cache.data.shape[2])[table[0, at // page].long() * page + at % page] = \
        O.pack_rows(torch.randn(n, L, generator=_gen(32), device="cuda"), kr)
    for sign in (1.0, -1.0):
        q = torch.randn(1, 2, heads, L + R, generator=_gen(33), device="cuda").to(dt)
        q[..., L] = sign * 4.0
        wide = _wide(q, table, page, 64 if dtype == "bf16" and heads == 30 else 32)
        out = latent_attention_decode(q, cache, wide, kv_len, scale)
        ref, absolute = O.decode(q, cache.data, wide, kv_len, scale, L, R)
        _check(out, ref, absolute, u, 2.0 ** -11, _dz(q, cache, wide, kv_len, scale, L, R), L + R, True)


@pytest.mark.parametrize("heads,nq", [(8, 32), (30, 64)])
def test_nan_reaches_only_its_readers(heads, nq):
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    cache, table, kv_len = _cache_for([300, 250], 128, 16, 64, torch.bfloat16, 51)
    q = torch.randn(2, 3, heads, 144, generator=_gen(52), device="cuda").bfloat16()
    table = _wide(q, table, 64, nq)
    before = latent_attention_decode(q, cache, table, kv_len, 0.1)
    cache.data[table[1, 3], 249 - 192] = 255                     # the newest row of sequence 1: its last token sees it
    out = latent_attention_decode(q, cache, table, kv_len, 0.1)
    assert torch.equal(out[0], before[0]) and torch.equal(out[1, :2], before[1, :2])
    assert out[1, 2].isnan().all() and torch.isfinite(before).all()


@pytest.mark.parametrize("heads,nq", [(24, 32), (64, 64)])
def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph(heads, nq):
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    q, cache, table, kv_len, scale, out = _case([30000, 300, 0, 1], 1, heads, 512, 64, 64, "bf16", 61, nq)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = latent_attention_decode(q, cache, table, kv_len, scale)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, again)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = latent_attention_decode(q, cache, table, kv_len, scale)
    kv_len.copy_(torch.tensor([4000, 0, 0, 1], dtype=torch.int32))        # lengths move between replays
    g.replay()
    assert torch.equal(got, latent_attention_decode(q, cache, table, kv_len, scale))
