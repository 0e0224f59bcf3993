"""Latent cache and latent attention kernels against their definitions in 64 bits (oracle/latent_ref.py).

Tolerances, derived from the number formats (u = unit roundoff of the output type: 2^-8 bf16, 2^-11 fp16):
  cache      bit-exact on inputs whose rotation is exact in fp32 (multiples of 1/16 up to 8); on others a
             group's error is at most 8 (s/2 + clamping at 7 when s was rounded down by up to 2^-8)
  attention  every output |err| <= u |out| + (P + 2 dz + 1e-5) A, with A = sum_j p_j |v_j|, P the rounding of
             the probabilities before the second product (2^-11 where they are fp16, 2^-8 where bf16)
             and dz the largest error of a logit: in the absorbed form the rotated query is rounded to
             fp16, dz <= 2^-11 scale |q| |k| (Cauchy-Schwarz); in the expanded form products are exact
             and only their fp32 sum rounds, dz <= D 2^-23 scale |q| |k|
             and in the 2-norm the same with dz / sqrt(D), as independent roundings add up. The absorbed form
             also sums in the rotated space and rotates back in fp32: a rotated sum rounds by at most 2^-22 of
             sum_j p_j |y_j| (y = H c), whose norm over a group of 64 is at most 8 times that of A, and
             the six butterfly stages by 6 2^-24 of it: together under 2^-16 |A| of the group."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check(out, ref, absolute, u, P, dz, D, rotated=False):
    turned = absolute.reshape(-1, 64).norm(dim=1).repeat_interleave(64) * 2.0 ** -16 if rotated else 0.0
    ref, absolute = ref.reshape(-1), absolute.reshape(-1)
    err = (out.double().reshape(-1) - ref).abs()
    assert torch.isfinite(out).all()
    bound = u * ref.abs() + (P + 2 * dz + 1e-5) * absolute + turned + 1e-7
    assert (err <= bound).all(), (err - bound).max().item()
    assert err.norm() <= u * ref.norm() + (P + 2 * dz / math.sqrt(D) + 1e-5) * absolute.norm() + 1e-7 * len(ref) ** 0.5


# ------------------------------------------------------------------------------------------ cache
def _pages(N, page, seed):
    pages = -(-N // page) + 2
    order = torch.randperm(pages, generator=_gen(seed), device="cuda")
    at = torch.arange(N, device="cuda")
    return pages, order[at // page] * page + at % page


@pytest.mark.parametrize("N,L,R,page", [(1, 64, 0, 1), (3, 512, 64, 64), (77, 448, 64, 16), (130, 192, 8, 48), (33, 320, 40, 7),
                                        (1000, 256, 32, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_write_is_bit_exact_where_the_rotation_is(N, L, R, page, dt):
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
    g = _gen(N + L)
    pages, slots = _pages(N, page, 1)
    cache = LatentCache.alloc(pages, page, L, R)
    cache.data.fill_(0xA5)
    before = cache.data.clone()
    c = (torch.randint(-128, 129, (N, L), generator=g, device="cuda").float() / 16).to(dt)
    c[0, :64] = 0                                               # a group of zeros
    kr = torch.randn(N, R, generator=g, device="cuda").to(dt)
    latent_cache_write(cache, c, kr, slots)
    flat = cache.data.view(pages * page, -1)
    assert torch.equal(flat[slots], O.pack_rows(c, kr))
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    assert torch.equal(flat[rest], before.view(pages * page, -1)[rest])         # nothing else was touched
    ref_c, ref_kr = O.unpack_rows(flat[slots], L, R)
    for out_dt in (torch.float32, dt):
        got_c, got_kr = latent_cache_read(cache, slots, out_dt)
        assert got_c.dtype == out_dt and got_c.shape == (N, L) and got_kr.shape == (N, R)
        # n s in fp32 is exact; the six butterfly stages and the cast round
        u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[out_dt]
        err = (got_c.double() - ref_c).abs()
        assert (err <= u * ref_c.abs() + 6 * 2.0 ** -24 * 64 * ref_c.abs().max() + 2.0 ** -25).all()
        assert torch.equal(got_kr, ref_kr.to(out_dt))


@pytest.mark.parametrize("scale", [1e-3, 1.0, 300.0])
def test_quantisation_error_is_within_half_a_step(scale):
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
    N, L = 200, 512
    c = torch.randn(N, L, generator=_gen(3), device="cuda") * scale
    cache = LatentCache.alloc(4, 64, L, 0)
    slots = torch.randperm(256, generator=_gen(4), device="cuda")[:N].int()
    latent_cache_write(cache, c, None, slots)
    got, _ = latent_cache_read(cache, slots, torch.float32)
    from oracle import latent_ref as O
    _, s = O.quantise(c)
    err = (got.double() - c.double()).reshape(N, L // 64, 64).norm(dim=-1)
    # |y - n s| <= s/2, or, for the largest values, 7 2^-8 s more where s was rounded down
    assert (err <= 8 * s * (0.5 + 7 * 2.0 ** -8) * 1.001).all()


def test_slots_that_are_skipped_and_extreme_values():
    from vq2_vllm import _lib
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
    lib = _lib.lib()
    lib.vq2_device_status(1)
    cache = LatentCache.alloc(2, 8, 64, 16)
    cache.data.fill_(7)
    c = torch.randn(5, 64, generator=_gen(5), device="cuda")
    kr = torch.randn(5, 16, generator=_gen(6), device="cuda")
    c[1, 5] = math.nan                       # makes its group NaN
    c[2] = 1e6                               # beyond 7 * 2048: saturates (one rotated value holds it all)
    kr[2, 0], kr[2, 1], kr[2, 2] = 1e6, -math.inf, math.nan
    latent_cache_write(cache, c, kr, torch.tensor([3, 4, 5, -1, -7], device="cuda"))
    assert lib.vq2_device_status(1) == 0
    got_c, got_kr = latent_cache_read(cache, torch.tensor([3, 4, 5, -1], device="cuda"), torch.float32)
    assert torch.isfinite(got_c[0]).all() and got_c[1].isnan().all() and torch.isfinite(got_c[2]).all()
    assert got_c[2].double().norm().item() == pytest.approx(7 * 2048, rel=1e-6)
    assert got_kr[2, 0] == 65504 and got_kr[2, 1] == -65504 and got_kr[2, 2].isnan()
    assert (got_c[3] == 0).all() and (got_kr[3] == 0).all()
    used = torch.zeros(16, dtype=torch.bool, device="cuda")
    used[[3, 4, 5]] = True
    assert (cache.data.view(16, -1)[~used] == 7).all()
    latent_cache_write(cache, c[:1], kr[:1], torch.tensor([16], device="cuda"))     # beyond the cache: reported
    assert lib.vq2_device_status(1) == 2 and (cache.data.view(16, -1)[~used] == 7).all()


def test_strided_rows():
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_write
    x = (torch.randint(-128, 129, (40, 600), generator=_gen(8), device="cuda").float() / 16).bfloat16()
    for c, kr in ((x[:, :512], x[:, 512:576]), (x[:, 4:516], x[:, 520:584]), (x[::2, :512], x[::2, 536:600])):
        cache = LatentCache.alloc(1, 40, 512, 64)
        latent_cache_write(cache, c, kr, torch.arange(c.shape[0], device="cuda"))
        assert torch.equal(cache.data[0, : c.shape[0]], O.pack_rows(c, kr))


# ------------------------------------------------------------------------------- absorbed form
def _cache_for(lens, L, R, page, dt, seed, spread=1.0):
    """A cache with the sequences' rows in scattered pages; every other slot holds bytes that read as NaN."""
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_cache import LatentCache
    g = _gen(seed)
    per = [-(-n // page) for n in lens]
    cache = LatentCache.alloc(sum(per) + 2, page, L, R)
    cache.data.fill_(255)
    order = torch.randperm(sum(per) + 2, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(1, max(per))), -1, dtype=torch.int32, device="cuda")
    done = 0
    for b, n in enumerate(lens):
        table[b, : per[b]] = order[done: done + per[b]]
        done += per[b]
        if n:
            at = torch.arange(n, device="cuda")
            c = torch.randn(n, L, generator=g, device="cuda").to(dt) * spread
            kr = torch.randn(n, R, generator=g, device="cuda").to(dt) * spread
            cache.data.view(-1, cache.data.shape[2])[table[b, at // page].long() * page + at % page] = O.pack_rows(c, kr)
    return cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _dz(q, cache, table, kv_len, scale, L, R):
    from oracle import latent_ref as O
    page, flat = cache.data.shape[1], cache.data.reshape(-1, cache.data.shape[2])
    k = 0.0
    for b in range(q.shape[0]):
        n = int(kv_len[b])
        if n > 0:
            at = torch.arange(n, device="cuda")
            c, kr = O.unpack_rows(flat[table[b, at // page].long() * page + at % page], L, R)
            k = max(k, torch.cat((c, kr), 1).norm(dim=1).max().item())
    return (2.0 ** -11 + (L + R) * 2.0 ** -23) * scale * q.double().norm(dim=-1).max().item() * k


def _decode_case(lens, T, heads, L, R, page, dtype, seed, q_scale=1.0, spread=1.0, scale=None):
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    dt, u = DT[dtype]
    cache, table, kv_len = _cache_for(lens, L, R, page, dt, seed, spread)
    q = (torch.randn(len(lens), T, heads, L + R, generator=_gen(seed + 1), device="cuda") * q_scale).to(dt)
    scale = (L // 4 + R) ** -0.5 if scale is None else scale
    out = latent_attention_decode(q, cache, table, kv_len, scale)
    assert out.dtype == dt and out.shape == (len(lens), T, heads, L)
    ref, absolute = O.decode(q, cache.data, table, kv_len, scale, L, R)
    _check(out, ref, absolute, u, 2.0 ** -11, _dz(q, cache, table, kv_len, scale, L, R), L + R, True)
    return q, cache, table, kv_len, scale, out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,T,heads,L,R,page", [
    ([1], 1, 1, 64, 0, 1),
    ([128], 1, 16, 512, 64, 64),                    # exactly one tile
    ([129, 127, 0, 1], 1, 16, 512, 64, 64),         # one over, one under, empty, one row
    ([300], 1, 64, 512, 64, 48),                    # pages that end inside a tile
    ([2, 40, 3, 0, 200], 3, 5, 192, 8, 16),         # fewer rows than new tokens; odd head count
    ([5000, 17], 1, 33, 448, 64, 1),                # single-row pages (a list of selected tokens), odd heads
    ([700], 4, 64, 256, 32, 128),
    ([1000, 900, 800], 2, 96, 320, 40, 7),
    ([20000], 1, 8, 512, 0, 64),                    # split over many blocks
])
def test_decode_matches_the_definition(dtype, lens, T, heads, L, R, page):
    _decode_case(lens, T, heads, L, R, page, dtype, seed=sum(lens) + heads)


def test_decode_many_sequences():
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 600, (200,), generator=g).tolist()
    _decode_case(lens, 1, 16, 512, 64, 64, "bf16", seed=11)


@pytest.mark.parametrize("q_scale,spread,scale", [(20.0, 1.0, 0.1), (1e-3, 1.0, None), (1.0, 50.0, 1e-3), (300.0, 1.0, 1e-3),
                                                  (1.0, 0.02, 1.0)])
def test_decode_over_peaked_flat_large_and_small_values(q_scale, spread, scale):
    _decode_case([777, 130], 2, 16, 512, 64, 64, "bf16", seed=21, q_scale=q_scale, spread=spread, scale=scale)


def test_decode_rising_logits():
    """Logits that rise from tile to tile, so that the running maximum moves every time."""
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    L, R, n = 128, 16, 1500
    cache, table, kv_len = _cache_for([n], L, R, 32, torch.bfloat16, 31)
    at = torch.arange(n, device="cuda")
    slots = table[0, at // 32].long() * 32 + at % 32
    c = torch.randn(n, L, generator=_gen(32), device="cuda")
    kr = torch.zeros(n, R, device="cuda")
    kr[:, 0] = at.float() / 8
    cache.data.view(-1, cache.data.shape[2])[slots] = O.pack_rows(c, kr)
    for sign in (1.0, -1.0):
        q = torch.randn(1, 2, 16, L + R, generator=_gen(33), device="cuda").bfloat16()
        q[..., L] = sign * 4.0
        out = latent_attention_decode(q, cache, table, kv_len, 0.5)
        ref, absolute = O.decode(q, cache.data, table, kv_len, 0.5, L, R)
        _check(out, ref, absolute, 2.0 ** -8, 2.0 ** -11, _dz(q, cache, table, kv_len, 0.5, L, R), L + R, True)


def test_decode_ignores_wrong_pages_and_says_so():
    from vq2_vllm import _lib
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    lib = _lib.lib()
    lib.vq2_device_status(1)
    cache, table, kv_len = _cache_for([200], 128, 16, 64, torch.bfloat16, 41)
    q = torch.randn(1, 1, 16, 144, generator=_gen(42), device="cuda").bfloat16()
    short = latent_attention_decode(q, cache, table, torch.tensor([192], dtype=torch.int32, device="cuda"), 0.1)
    assert lib.vq2_device_status(1) == 0
    for bad in (-1, cache.data.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 3] = bad                                            # rows 192 .. 199
        out = latent_attention_decode(q, cache, t, kv_len, 0.1)
        assert lib.vq2_device_status(1) == 2
        assert (out.float() - short.float()).abs().max() <= 2 ** -7 * short.float().abs().max()
    # a length beyond the table is clamped to it
    out = latent_attention_decode(q, cache, table[:, :3].contiguous(), torch.tensor([10 ** 9], dtype=torch.int32, device="cuda"), 0.1)
    assert lib.vq2_device_status(1) == 0
    assert (out.float() - short.float()).abs().max() <= 2 ** -7 * short.float().abs().max()


def test_decode_nan_reaches_only_its_readers():
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    cache, table, kv_len = _cache_for([300, 250], 128, 16, 64, torch.bfloat16, 51)
    q = torch.randn(2, 2, 4, 144, generator=_gen(52), device="cuda").bfloat16()
    cache.data[table[1, 3], 249 - 192] = 255                     # the newest row of sequence 1
    out = latent_attention_decode(q, cache, table, kv_len, 0.1)
    assert torch.isfinite(out[0]).all()
    assert torch.isfinite(out[1, 0]).all()                       # its first new token does not see that row
    assert out[1, 1].isnan().all()


def test_decode_repeats_bit_for_bit_on_another_stream_and_in_a_graph():
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    q, cache, table, kv_len, scale, out = _decode_case([5000, 300, 0, 1], 1, 64, 512, 64, 64, "bf16", 61)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = latent_attention_decode(q, cache, table, kv_len, scale)
        side = latent_attention_decode(q, cache, table, kv_len, scale)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, again) and torch.equal(out, side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = latent_attention_decode(q, cache, table, kv_len, scale)
    kv_len.copy_(torch.tensor([4000, 0, 0, 1], dtype=torch.int32))        # lengths move between replays
    g.replay()
    assert torch.equal(got, latent_attention_decode(q, cache, table, kv_len, scale))


# ------------------------------------------------------------------------------- expanded form
def _prefill_case(qlens, prefix, heads, dn, R, dv, dtype, seed, q_scale=1.0, views=True):
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    dt, u = DT[dtype]
    g = _gen(seed)
    klens = [n + p for n, p in zip(qlens, prefix)]
    cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    Tq, Tk = sum(qlens), sum(klens)
    q = (torch.randn(Tq, heads, dn + R, generator=g, device="cuda") * q_scale).to(dt)
    kv = torch.randn(Tk, heads, dn + dv, generator=g, device="cuda").to(dt)
    k_nope, v = kv[..., :dn], kv[..., dn:]
    if not views:
        k_nope, v = k_nope.contiguous(), v.contiguous()
    kr = torch.randn(Tk, R, generator=g, device="cuda").to(dt) if R else None
    scale = (dn + R) ** -0.5
    out = latent_attention_prefill(q, k_nope, kr, v, cu(qlens), cu(klens), max(qlens), scale)
    assert out.dtype == dt and out.shape == (Tq, heads, dv)
    ref, absolute = O.prefill(q, k_nope, kr, v, cu(qlens), cu(klens), scale)
    k = torch.cat((k_nope.double().flatten(0, 1), ) if kr is None else
                  (k_nope.double().flatten(0, 1), kr.double().repeat_interleave(heads, 0)), 1)
    dz = (dn + R) * 2.0 ** -23 * scale * q.double().norm(dim=-1).max().item() * (k.norm(dim=1).max().item() if len(k) else 0.0)
    _check(out, ref, absolute, u, u, dz, dn + R)
    return q, k_nope, kr, v, cu(qlens), cu(klens), scale, out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("qlens,prefix,heads,dn,R,dv", [
    ([1], [0], 1, 64, 0, 64),
    ([128], [0], 2, 128, 64, 128),
    ([129], [0], 2, 128, 64, 128),
    ([256], [0], 3, 128, 64, 128),
    ([257, 1, 0, 127], [0, 0, 0, 0], 2, 128, 64, 128),
    ([77, 300], [1000, 5], 4, 96, 32, 96),
    ([5, 600], [127, 129], 3, 64, 16, 128),
    ([1, 1, 1], [0, 500, 383], 16, 128, 64, 64),         # single tokens
    ([40], [0], 5, 72, 8, 40),
    ([200], [300], 2, 8, 0, 8),
    ([1100], [0], 2, 128, 64, 128),
])
def test_prefill_matches_the_definition(dtype, qlens, prefix, heads, dn, R, dv):
    _prefill_case(qlens, prefix, heads, dn, R, dv, dtype, seed=sum(qlens) + heads)


@pytest.mark.parametrize("q_scale", [1e-3, 10.0, 100.0])
def test_prefill_over_flat_and_peaked_rows(q_scale):
    _prefill_case([333], [77], 3, 128, 64, 128, "bf16", 71, q_scale=q_scale, views=False)


def test_prefill_rows_that_see_nothing():
    """More queries than keys: the first rows see no key and give zeros."""
    _prefill_case([300, 40], [-200, -40], 2, 128, 64, 128, "bf16", 72)


def test_prefill_keeps_sequences_apart():
    """NaN and infinities in one sequence's keys and values stay out of its neighbours' outputs."""
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    q, kn, kr, v, cu_q, cu_k, scale, out = _prefill_case([70, 90, 300], [0, 10, 0], 2, 128, 64, 128, "bf16", 73)
    kn, v, kr = kn.clone(), v.clone(), kr.clone()
    for t, bad in ((kn, math.nan), (v, math.inf), (kr, math.nan)):
        t[70:170] = bad
    got = latent_attention_prefill(q, kn, kr, v, cu_q, cu_k, 300, scale)
    assert torch.equal(got[:70], out[:70]) and torch.equal(got[160:], out[160:])
    assert got[70:160].isnan().all()


def test_prefill_rising_logits_and_graph():
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    n, heads = 1000, 2
    g = _gen(74)
    q = torch.randn(n, heads, 144, generator=g, device="cuda").bfloat16()
    kv = torch.randn(n, heads, 256, generator=g, device="cuda").bfloat16()
    kr = torch.zeros(n, 16, device="cuda")
    kr[:, 0] = torch.arange(n, device="cuda") / 4
    kr = kr.bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for sign in (1.0, -1.0):
        q[..., 128] = sign * 8.0
        out = latent_attention_prefill(q, kv[..., :128], kr, kv[..., 128:], cu, cu, n, 0.25)
        ref, absolute = O.prefill(q, kv[..., :128], kr, kv[..., 128:], cu, cu, 0.25)
        _check(out, ref, absolute, 2.0 ** -8, 2.0 ** -8, 144 * 2.0 ** -23 * 0.25 * 30 * 300, 144)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = latent_attention_prefill(q, kv[..., :128], kr, kv[..., 128:], cu, cu, n, 0.25)
    graph.replay()
    assert torch.equal(got, out)


# ------------------------------------------------------------------------------------ refusals
def test_refusals():
    from vq2_vllm.kernels.latent_attention import latent_attention_decode, latent_attention_prefill
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
    cache = LatentCache.alloc(2, 8, 128, 16)
    c, kr = torch.zeros(3, 128, device="cuda"), torch.zeros(3, 16, device="cuda")
    slots = torch.arange(3, device="cuda")
    with pytest.raises(ValueError):
        latent_cache_write(cache, c[:, :64], kr, slots)
    with pytest.raises(ValueError):
        latent_cache_write(cache, c, None, slots)
    with pytest.raises(ValueError):
        latent_cache_write(cache, c, kr, slots[:2])
    with pytest.raises(ValueError):
        latent_cache_write(cache, c, kr, slots.float())
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_cache_write(cache, c.cpu(), kr, slots)
    with pytest.raises(ValueError):
        latent_cache_read(cache, slots, torch.int8)
    q = torch.zeros(1, 1, 4, 144, device="cuda", dtype=torch.bfloat16)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for bad in (q.float(), q[..., :100], q[0]):
        with pytest.raises(ValueError):
            latent_attention_decode(bad, cache, table, n, 1.0)
    with pytest.raises(ValueError):
        latent_attention_decode(q, cache, table[:, :0], n, 1.0)
    with pytest.raises(ValueError):
        latent_attention_decode(q, cache, table.float(), n, 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_attention_decode(q, cache, table, n.cpu(), 1.0)
    assert latent_attention_decode(q[:0], cache, table[:0], n[:0], 1.0).shape == (0, 1, 4, 128)
    p = torch.zeros(4, 2, 144, device="cuda", dtype=torch.bfloat16)
    k, v, r = (torch.zeros(4, *s, device="cuda", dtype=torch.bfloat16) for s in ((2, 128), (2, 128), (16,)))
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    for args in ((p.float(), k, r, v), (p, k, None, v), (p, k, r.float(), v), (p, k[:, :1], r, v), (p, k, r[:3], v),
                 (p[..., :140], k, r[:, :12], v), (p, k[..., :64], r, v)):
        with pytest.raises(ValueError):
            latent_attention_prefill(*args, cu, cu, 4, 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_attention_prefill(p, k, r, v, cu.cpu(), cu, 4, 1.0)
    assert latent_attention_prefill(p[:0], k, r, v, cu * 0, cu, 0, 1.0).shape == (0, 2, 128)


# ------------------------------------------------------------------------------------ keys split over blocks
# The parts' sums are held and joined in fp32: a value takes at most 64 parts' factors and sums, 3 roundings of 2^-24 each, and its
# denominator the same, under 2^-16 of A in all: half of it beside the 1e-5 that the bound has for sums already. P is
# rounded relative to itself, whatever maximum it is held against, so its term does not change.
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("qlens,prefix,heads,dn,R,dv", [
    ([1], [5000], 1, 128, 64, 128),
    ([64], [4000], 3, 128, 64, 128),
    ([129], [3001], 2, 96, 32, 96),
    ([300], [2900], 4, 64, 0, 64),
    ([2000], [0], 1, 128, 64, 128),                     # blocks from one part to many
    ([1, 0, 200], [3000, 700, 9], 2, 128, 64, 72),      # one sequence far longer than the others
    ([5, 7], [6000, 0], 1, 64, 16, 128),
])
def test_prefill_with_split_keys(dtype, qlens, prefix, heads, dn, R, dv):
    from vq2_vllm import _lib
    klens = [n + p for n, p in zip(qlens, prefix)]
    assert _lib.lib().vq2_latent_prefill_workspace_size(len(qlens), heads, dv, max(qlens), sum(qlens), sum(klens)) > 0
    _prefill_case(qlens, prefix, heads, dn, R, dv, dtype, seed=sum(klens) + heads)


@pytest.mark.parametrize("q_scale", [1e-3, 10.0, 100.0])
def test_split_keys_over_flat_and_peaked_rows(q_scale):
    _prefill_case([140], [4000], 2, 128, 64, 128, "bf16", 81, q_scale=q_scale)


def test_split_keys_rows_that_see_nothing():
    """Rows before the first key give zeros, also where their block has keys in several parts."""
    out = _prefill_case([2400], [-100], 1, 128, 64, 128, "bf16", 82)[-1]
    assert not out[:100].any()


def test_split_keys_keep_nan_where_it_is_seen():
    """A NaN value reaches the rows that see it and, from another step, no other; a graph gives the same bits."""
    from vq2_vllm.kernels.latent_attention import latent_attention_prefill
    q, kn, kr, v, cu_q, cu_k, scale, out = _prefill_case([600], [2000], 2, 128, 64, 128, "bf16", 83)
    v = v.clone()
    v[2432] = math.nan                                  # the first key of a step; rows from 432 on see it
    got = latent_attention_prefill(q, kn, kr, v, cu_q, cu_k, 600, scale)
    assert torch.equal(got[:256], out[:256]) and got[432:].isnan().all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = latent_attention_prefill(q, kn, kr, v, cu_q, cu_k, 600, scale)
    graph.replay()
    assert torch.equal(again.nan_to_num(7.0), got.nan_to_num(7.0))


def test_prefill_without_workspace_agrees():
    """The C call without a workspace does not split and agrees to the roundings of the output and of P."""
    from vq2_vllm import _lib
    q, kn, kr, v, cu_q, cu_k, scale, out = _prefill_case([200], [3000], 2, 128, 64, 128, "f16", 84)
    whole = torch.empty_like(out)
    a = _lib.Vq2LatentPrefillArgs(1, 2, 128, 64, 128, 200, 1, len(q), len(v), scale, q.stride(0), q.stride(1), kn.stride(0), kn.stride(1),
                                  v.stride(0), v.stride(1), kr.stride(0), q.data_ptr(), kn.data_ptr(), kr.data_ptr(), v.data_ptr(),
                                  cu_q.data_ptr(), cu_k.data_ptr(), whole.data_ptr())
    assert _lib.lib().vq2_latent_prefill(a, torch.cuda.current_stream().cuda_stream) == 0
    assert (whole.double() - out.double()).norm() <= 4 * 2.0 ** -11 * out.double().norm()


def test_graphs_of_growing_sizes_keep_their_workspaces():
    """Graphs captured for growing batches replay right after the stream's workspace has grown past the first one's."""
    from vq2_vllm.kernels.latent_attention import latent_attention_decode
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_write
    g = _gen(91)
    cache = LatentCache.alloc(40, 64, 512, 64)
    latent_cache_write(cache, torch.randn(2560, 512, generator=g, device="cuda").bfloat16(),
                       torch.randn(2560, 64, generator=g, device="cuda").bfloat16(), torch.arange(2560, device="cuda"))
    made = []
    for B in (1, 8, 96):
        q = torch.randn(B, 1, 64, 576, generator=g, device="cuda").bfloat16()
        table = torch.stack([torch.randperm(40, generator=g, device="cuda") for _ in range(B)]).int()
        n = torch.randint(1, 2561, (B,), generator=g, device="cuda").int()
        want = latent_attention_decode(q, cache, table, n, 0.05)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = latent_attention_decode(q, cache, table, n, 0.05)
        made.append((graph, out, want, q, table, n))
    others = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(64)]       # takes any memory let go
    for graph, out, want, *_ in made:
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert all((t == 7.0).all() for t in others)


# ------------------------------------------------------------------------------------ fp16 queries
# In the 2-norm the fp16 form may err by the rounding of its output (that of ref.half(), measured on the same values) and by that of the
# probabilities, whose relative errors have the same distribution and average over the keys: together at most sqrt(2) of
# the first. The query's remainder beyond its second term (2^-14 of it at most) and the fp32 sums stay under the rest up to 1.5; a
# query rounded to fp16 alone gives 1.6 to 2.6.
@pytest.mark.parametrize("lens,T,heads,L,R,page", [
    ([236], 1, 3, 128, 64, 64),                     # 16 query rows a block
    ([4000, 1700], 1, 16, 512, 64, 64),
    ([90, 0, 33], 2, 5, 448, 0, 1),
    ([40000, 20000], 1, 24, 512, 64, 64),           # 32 query rows a block
    ([30000, 10000], 2, 64, 320, 32, 16),
    ([60000, 3], 1, 64, 64, 64, 128),
])
def test_fp16_decode_errs_like_its_output(lens, T, heads, L, R, page):
    from oracle import latent_ref as O
    q, cache, table, kv_len, scale, out = _decode_case(lens, T, heads, L, R, page, "f16", seed=sum(lens) + L)
    ref, _ = O.decode(q, cache.data, table, kv_len, scale, L, R)
    assert (out.double() - ref).norm() <= 1.5 * (ref.half().double() - ref).norm()
