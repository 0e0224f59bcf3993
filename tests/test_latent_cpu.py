"""Latent cache and latent attention without a GPU: the oracle's properties, the checks of arguments, and
the C entries' error codes (every call below fails its checks before it touches the device)."""
import ctypes

import pytest
import torch

from oracle import latent_ref as O


def test_rows_round_trip_and_sizes():
    from vq2_vllm import _lib
    from vq2_vllm.kernels.latent_cache import latent_row_bytes
    L_ = _lib.lib()
    for L in range(64, 513, 64):
        for R in range(0, 65, 8):
            assert O.row_bytes(L, R) == latent_row_bytes(L, R) == L_.vq2_latent_row_bytes(L, R)
    assert latent_row_bytes(512, 64) == 400
    for L, R in ((0, 0), (32, 0), (96, 0), (576, 0), (64, 4), (64, 72), (64, -8)):
        assert L_.vq2_latent_row_bytes(L, R) == 0
        with pytest.raises(ValueError):
            latent_row_bytes(L, R)


@pytest.mark.parametrize("L,R", [(64, 0), (192, 24), (512, 64)])
def test_oracle_quantisation_is_within_half_a_step_and_idempotent(L, R):
    g = torch.Generator().manual_seed(L)
    c, kr = torch.randn(20, L, generator=g), torch.randn(20, R, generator=g)
    rows = O.pack_rows(c, kr)
    assert rows.shape == (20, O.row_bytes(L, R))
    c1, kr1 = O.unpack_rows(rows, L, R)
    _, s = O.quantise(c)
    assert ((c1 - c).reshape(20, -1, 64).norm(dim=-1) <= 8 * s * (0.5 + 7 * 2.0 ** -8)).all()
    assert torch.equal(kr1, kr.half().double())


def test_oracle_attention_rotation_invariance():
    """q . c = (H q) . (H c) and the result rotates with the values: what the kernel relies on."""
    g = torch.Generator().manual_seed(1)
    q, c = torch.randn(3, 64, generator=g).double(), torch.randn(50, 64, generator=g).double()
    last = torch.full((3,), 49)
    h = O.hadamard()
    a, _ = O.attend(q, c, c, last, 0.2)
    b, _ = O.attend(q @ h, c @ h, c @ h, last, 0.2)
    assert (a - b @ h).abs().max() < 1e-12


def test_python_refusals_without_a_gpu():
    from vq2_vllm.kernels.latent_attention import latent_attention_decode, latent_attention_prefill
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
    with pytest.raises(ValueError):
        LatentCache(torch.zeros(2, 8, 96, dtype=torch.uint8), 128, 64)
    with pytest.raises(ValueError):
        LatentCache(torch.zeros(2, 8, 112, dtype=torch.int8), 128, 16)
    cache = LatentCache.alloc(2, 8, 128, 16, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_cache_write(cache, torch.zeros(1, 128), torch.zeros(1, 16), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_cache_read(cache, torch.zeros(1, dtype=torch.int64))
    i = torch.ones(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_attention_decode(torch.zeros(1, 1, 2, 144, dtype=torch.bfloat16), cache, i, i[0], 1.0)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        latent_attention_prefill(x, x, None, x, torch.tensor([0, 2]), torch.tensor([0, 2]), 2, 1.0)


def test_c_entries_reject_bad_arguments_without_a_gpu():
    from vq2_vllm import _lib
    L = _lib.lib()
    fake = 1 << 20
    cache = lambda data=fake, pages=4, page=8, lat=128, rope=16: _lib.Vq2LatentCache(data, pages, page, lat, rope)  # noqa: E731
    write = lambda k, c=fake, r=fake, dt=0, cs=128, rs=16, slots=fake, sd=0, n=3: \
        L.vq2_latent_cache_write(k, c, r, dt, cs, rs, slots, sd, n, None)  # noqa: E731
    assert write(None) == 1 and write(cache(data=None)) == 1 and write(cache(), c=None) == 1 and write(cache(), r=None) == 1
    assert write(cache(lat=96)) == 2 and write(cache(rope=12)) == 2 and write(cache(pages=0)) == 2 and write(cache(), cs=127) == 2
    assert write(cache(), n=-1) == 2 and write(cache(), rs=8) == 2
    assert write(cache(data=fake + 8)) == 3 and write(cache(), c=fake + 2) == 3
    assert write(cache(), dt=3) == 4 and write(cache(), sd=2) == 4
    assert write(cache(), n=0) == 0
    read = lambda k, slots=fake, sd=0, n=3, c=fake, r=fake, dt=0: L.vq2_latent_cache_read(k, slots, sd, n, c, r, dt, None)  # noqa: E731
    assert read(None) == 1 and read(cache(), slots=None) == 1 and read(cache(), c=fake + 4) == 3 and read(cache(), dt=-1) == 4
    assert read(cache(page=0)) == 2 and read(cache(), n=0) == 0

    def decode(ws=fake, nb=1 << 40, **kw):
        v = dict(B=1, T=1, heads=4, latent_dim=128, rope_dim=16, page_size=8, max_pages=2, dtype=0, pages=4, scale=1.0, q=fake, cache=fake,
                 block_table=fake, kv_len=fake, out=fake) | kw
        return L.vq2_latent_decode(_lib.Vq2LatentDecodeArgs(**v), ws, nb, None)
    assert L.vq2_latent_decode(None, fake, 1 << 20, None) == 1
    assert decode(q=None) == 1 and decode(kv_len=None) == 1
    assert decode(B=0) == 2 and decode(latent_dim=100) == 2 and decode(page_size=0) == 2 and decode(heads=-1) == 2
    assert decode(out=fake + 2) == 3 and decode(dtype=2) == 4 and decode(ws=None) == 5 and decode(nb=0) == 5
    assert L.vq2_latent_decode_workspace_size(0, 1, 1, 64, 0) == 0 and L.vq2_latent_decode_workspace_size(1, 1, 1, 64, 0) > 0

    def prefill(**kw):
        v = dict(B=1, heads=2, nope_dim=128, rope_dim=64, v_dim=128, max_q=4, dtype=0, total_q=4, total_k=4, scale=1.0, q_stride_t=384,
                 q_stride_h=192, k_stride_t=256, k_stride_h=128, v_stride_t=256, v_stride_h=128, r_stride_t=64, q=fake, k_nope=fake,
                 k_rope=fake, v=fake, cu_q=fake, cu_k=fake, out=fake) | kw
        return L.vq2_latent_prefill(ctypes.byref(_lib.Vq2LatentPrefillArgs(**v)), None)
    assert L.vq2_latent_prefill(None, None) == 1
    assert prefill(q=None) == 1 and prefill(k_rope=None) == 1 and prefill(cu_k=None) == 1
    assert prefill(nope_dim=136) == 2 and prefill(v_dim=4) == 2 and prefill(rope_dim=72) == 2 and prefill(B=0) == 2 and prefill(max_q=-1) == 2
    assert prefill(k_stride_h=127) == 2 and prefill(r_stride_t=4) == 2
    assert prefill(v=fake + 8) == 3 and prefill(dtype=2) == 4 and prefill(max_q=0) == 0


def test_a_captured_workspace_outlives_a_larger_one(monkeypatch):
    """A graph keeps the address of the workspace it was captured with: a later, larger call on the stream takes a new buffer
    and leaves that one alone. A buffer that no graph has is let go."""
    import weakref

    import torch
    from vq2_vllm import _lib
    monkeypatch.setattr(_lib, "_WS", {})
    capturing = True
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    dev, stream = torch.device("cpu"), -12345
    first = weakref.ref(_lib.workspace(1 << 20, dev, stream))
    again = weakref.ref(_lib.workspace(1 << 19, dev, stream))
    assert again() is first()
    capturing = False
    second = weakref.ref(_lib.workspace(1 << 21, dev, stream))
    assert first() is not None and second() is not first()
    _lib.workspace(1 << 22, dev, stream)
    assert second() is None and first() is not None


def test_which_decode_kernel_a_call_takes():
    """16 query rows a block for few rows or few tiles (counted by the table's width), else 32 or, in bf16, 64."""
    from vq2_vllm import _lib
    rows = _lib.lib().vq2_latent_decode_query_rows
    assert rows(64, 1, 16, 128, 64, 0) == 16 and rows(1, 1, 64, 5, 64, 0) == 16 and rows(1, 1, 64, 370, 64, 0) == 16
    assert rows(1, 1, 64, 371, 64, 0) == 64 and rows(1, 1, 64, 371, 64, 1) == 32 and rows(1, 1, 32, 1000, 64, 0) == 32
    assert rows(0, 1, 16, 8, 64, 0) == 0 and rows(1, 1, 16, 8, 64, 2) == 0 and rows(1, 1, 16, 1 << 30, 1 << 10, 0) == 0


def test_calls_use_the_tensor_that_the_cache_has_now():
    """A pool that is assigned anew is the one the calls point to; a tensor that does not fit is refused and changes nothing."""
    from vq2_vllm.kernels.latent_cache import LatentCache
    cache = LatentCache.alloc(2, 8, 128, 16, device="cpu")
    grown = torch.zeros(5, 16, 112, dtype=torch.uint8)
    cache.data = grown
    assert cache.data is grown
    assert (cache.args.data, cache.args.pages, cache.args.page_size) == (grown.data_ptr(), 5, 16)
    for bad in (torch.zeros(5, 16, 96, dtype=torch.uint8), grown[:, ::2], grown[:0], grown.char()):
        with pytest.raises(ValueError):
            cache.data = bad
    assert cache.data is grown and cache.args.data == grown.data_ptr()
    for name in ("latent_dim", "rope_dim"):          # the kernels' sizes were checked against them
        with pytest.raises(AttributeError):
            setattr(cache, name, 64)
    assert (cache.latent_dim, cache.rope_dim) == (128, 16)


def test_strides_of_rows():
    """What the write entry is given: rows on 16-byte boundaries, a stride of whole 16 bytes that is no less than the row. The stride
    that a tensor of one row happens to have does not count."""
    from vq2_vllm.kernels.latent_cache import _rows
    x = torch.randn(6, 577)
    one = torch.randn(600).as_strided((1, 512), (3, 1))
    for rows in (x[:1, :512], x[2:3, 1:513], x[3:4, 4:516], x[:, :512], x[:, 1:513], x[::2, :64], torch.randn(512, 1).T, torch.randn(512, 4).T,
                 one, torch.randn(6, 576)[:, :512], torch.randn(1, 512), torch.randn(512).expand(3, 512), torch.randn(4, 0)):
        got, stride = _rows(rows)
        assert torch.equal(got, rows) and got.data_ptr() % 16 == 0 and stride % 8 == 0 and stride >= rows.shape[1]
        assert got.numel() == 0 or torch.equal(torch.as_strided(got, rows.shape, (stride, 1)), rows) or rows.shape[0] == 1
