"""A step that has no tokens for this layer (an empty batch) gives an empty result and leaves the cache alone."""
import pytest
import torch

from test_latent_layer_gpu import H, _cache, _i32, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", [False, True])
def test_steps_without_tokens(shared):
    layer = _layer(shared)
    cache, slots, table = _cache(layer, 40)
    before = cache.data.clone()
    x, none = torch.empty(0, H, dtype=torch.bfloat16, device="cuda"), slots[:0]
    for y in (layer.prefill(x, none, cache, none, none, _i32(0), _i32(0), 0),
              layer.prefill(x, none, cache, none, none, _i32(0, 0), _i32(0, 0), 0),
              layer.prefill(x, none, cache, none, slots, _i32(0, 0), _i32(0, 40), 0),
              layer.decode(x, none, cache, none, table[:0], _i32()[:0])):
        assert y.shape == (0, H) and y.dtype == x.dtype
    assert torch.equal(cache.data, before)
