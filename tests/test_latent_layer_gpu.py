"""The decoder layer that runs latent cache, latent attention, router and routed experts together: a prompt in one
piece, in chunks over a cached prefix, and continued token by token has to give the same attention.

Tolerance: both forms attend to the same cached values; they differ in where bf16 rounds. Expanded: keys, values (after
a projection each), probabilities and the output; absorbed: the absorbed query, the output in latent space and its
projection. Each rounding is 2^-8 at most and 2^-9.8 in the mean square of its term; eight of them, with the logits'
errors (of the order of the logits' own size times 2^-9) acting through the softmax, stay under 8 * 2^-8 = 3.1e-2 in
the 2-norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H, HEADS, E, TOPK = 512, 6, 8, 2


def _layer(shared=False, L=256, R=32, seed=0):
    from vq2_vllm import synth
    from vq2_vllm.latent_layer import LatentLayer
    experts = synth.layer_args({k: v.cuda() for k, v in synth.make_layer(E, H, 256, seed=seed).items()})
    sh = None
    if shared:
        g = torch.Generator(device="cuda").manual_seed(3)
        sh = ((torch.randn(512, H, generator=g, device="cuda") * 0.04).bfloat16(), (torch.randn(H, 256, generator=g, device="cuda") * 0.06).bfloat16())
    return LatentLayer.random(H, HEADS, experts, E, TOPK, L=L, R=R, nope=64, dv=64, shared=sh, seed=seed)


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(layer, n, page=16, seed=5):
    from vq2_vllm.kernels.latent_cache import LatentCache
    pages = -(-n // page) + 2
    order = torch.randperm(pages, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    at = torch.arange(n, device="cuda")
    return LatentCache.alloc(pages, page, layer.L, layer.R), order[at // page] * page + at % page, order[: -(-n // page)].int()[None].contiguous()


def _close(a, b):
    a, b = a.double(), b.double()
    assert torch.isfinite(a).all()
    rel = ((a - b).norm() / b.norm()).item()
    assert rel <= 8 * 2.0 ** -8, rel


@pytest.mark.parametrize("L,R", [(256, 32), (512, 64), (64, 0)])
def test_chunks_and_steps_attend_as_the_whole_prompt_does(L, R):
    layer = _layer(L=L, R=R)
    n = 300
    x = torch.randn(n, H, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    pos = torch.arange(n, device="cuda")
    cache, slots, table = _cache(layer, n)
    whole = layer.attend_prefill(x, pos, cache, slots, slots, _i32(0, n), _i32(0, n), n)
    cache2, slots2, table2 = _cache(layer, n, seed=6)
    a, b = 130, 280                                      # a chunk, a second over its prefix, then steps of 1 and 3 tokens
    first = layer.attend_prefill(x[:a], pos[:a], cache2, slots2[:a], slots2[:a], _i32(0, a), _i32(0, a), a)
    second = layer.attend_prefill(x[a:b], pos[a:b], cache2, slots2[a:b], slots2[:b], _i32(0, b - a), _i32(0, b), b - a)
    _close(first, whole[:a])
    _close(second, whole[a:b])
    at = b
    for T in (1, 3, 1, 2, 4, 3, 3, 3):
        step = layer.attend_decode(x[at: at + T], pos[at: at + T], cache2, slots2[at: at + T], table2, _i32(at + T))
        _close(step, whole[at: at + T])
        at += T
    assert at == n


@pytest.mark.parametrize("shared", [False, True])
def test_layer_runs_both_halves(shared):
    """prefill and decode of the whole layer are their parts put together, and a captured step repeats."""
    from vq2_vllm.latent_layer import rms_norm
    layer = _layer(shared)
    n = 290                                              # the grouped prefill path of the experts
    x = torch.randn(n, H, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16()
    pos = torch.arange(n, device="cuda")
    cache, slots, table = _cache(layer, n + 8)
    y = layer.prefill(x, pos, cache, slots[:n], slots[:n], _i32(0, n), _i32(0, n), n)
    att = layer.attend_prefill(x, pos, cache, slots[:n], slots[:n], _i32(0, n), _i32(0, n), n)
    mid = x + att @ layer.w_o
    want = (mid.float() + layer.feed_forward(mid)).to(x.dtype)
    assert y.shape == x.shape and torch.isfinite(y).all()
    assert ((y.double() - want.double()).norm() / want.double().norm()).item() < 1e-2        # experts' atomics, one bf16 rounding
    assert rms_norm(x, layer.norm_in).dtype == torch.bfloat16
    new = torch.randn(3, H, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").bfloat16()
    args = (new, pos[:3] + n, cache, slots[n: n + 3], table, _i32(n + 3))
    out = layer.decode(*args)
    assert out.shape == new.shape and torch.isfinite(out).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer.decode(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = layer.decode(*args)
    graph.replay()
    assert ((again.double() - out.double()).norm() / out.double().norm()).item() < 1e-2
