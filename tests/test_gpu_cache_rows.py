"""Rows that the caches take."""
import pytest

from libero_hip import episodes, room

pytestmark = pytest.mark.gpu
OPTIONS = dict(kv_heads=2, head_dim=32, tokens=64, storage='bf16', page_tokens=16, block_tokens=16)


def caches():
    """(a cache, a ragged chunk of 1 and 3 tokens) of either kind."""
    import torch
    host, device = episodes.EpisodeCache(2, **OPTIONS), room.DeviceEpisodeCache(2, **OPTIONS)
    return ((host, host.extend([1, 3], [0, 1])),
            (device, device.extend(torch.tensor([1, 3], dtype=torch.int32, device='cuda'), rows=4, most=3)))


def test_padded_rows_are_refused(gpu_available):
    """Rows (worlds, most, heads, head_dim) for a ragged chunk: nothing is stored."""
    import torch
    from libero_hip.rotary import Rotary
    print('case padded rows', flush=True)
    turning = Rotary.make(32)
    for cache, chunk in caches():
        packed = torch.randn((4, 2, 32), device='cuda').bfloat16()
        cache.write(chunk, packed, packed)
        before = cache.layers[0].k.view(torch.int16).clone()           # bits: what no token has is not initialised
        for shape in ((2, 3, 2, 32), (2, 2, 2, 32)):     # with padding, and as many rows as there are tokens
            x = torch.ones(shape, dtype=torch.bfloat16, device='cuda')
            for call in (lambda: cache.write(chunk, x, x), lambda: cache.enter(chunk, turning, x, x, x), lambda: cache.attend(chunk, x),
                         lambda: cache.recall(chunk, x, top=1)):
                with pytest.raises(ValueError):
                    call()
        assert torch.equal(cache.layers[0].k.view(torch.int16), before)


def test_results_of_other_shapes_are_refused(gpu_available):
    import torch
    from libero_hip.rotary import Rotary
    print('case shapes of results', flush=True)
    cache, turning = room.DeviceEpisodeCache(2, **OPTIONS), Rotary.make(32)
    chunk = cache.extend(3)
    q = torch.randn((2, 3, 4, 32), device='cuda').bfloat16()
    k = torch.randn((2, 3, 2, 32), device='cuda').bfloat16()
    cache.enter(chunk, turning, q, k, k, out=torch.empty_like(q))
    out, lse = torch.full((3, 2, 4, 32), 7.0, dtype=torch.bfloat16, device='cuda'), torch.full((3, 2, 4), 7.0, device='cuda')
    for options in (dict(out=out), dict(lse=lse)):
        for call in (lambda: cache.attend(chunk, q, **options), lambda: cache.recall(chunk, q, top=1, **options)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        cache.enter(chunk, turning, q, k, k, out=out)
    assert bool((out == 7).all()) and bool((lse == 7).all())
