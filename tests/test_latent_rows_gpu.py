"""Single rows in whatever stride a slice leaves them: the same bytes in the cache as from rows of their own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width", [577, 579, 584, 1000])
def test_one_row_of_a_wider_tensor(dt, width):
    from oracle import latent_ref as O
    from vq2_vllm.kernels.latent_cache import LatentCache, latent_cache_read, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(width)
    x = (torch.randint(-128, 129, (3, width), generator=g, device="cuda").float() / 16).to(dt)
    cache = LatentCache.alloc(1, 8, 512, 64)
    at = torch.tensor([5], device="cuda")
    for c, kr in ((x[:1, :512], x[:1, 512:576]), (x[1:2, 1:513], x[2:3, :64]), (x[2:3, 8:520], x[1:2, 7:71]),
                  (x[0, :512].contiguous()[:, None].T, x[0, :64].contiguous()[:, None].T)):
        cache.data.zero_()
        latent_cache_write(cache, c, kr, at)
        assert torch.equal(cache.data[0, 5:6], O.pack_rows(c, kr)) and not cache.data[0, :5].any() and not cache.data[0, 6:].any()
        got, got_kr = latent_cache_read(cache, at, torch.float32)
        assert torch.equal(got_kr.half(), kr.half()) and got.shape == (1, 512)
