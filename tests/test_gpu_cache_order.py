"""The order of what DeviceEpisodeCache does on several streams."""
import pytest

from libero_hip import room

pytestmark = pytest.mark.gpu
OPTIONS = dict(kv_heads=2, head_dim=32, tokens=64, storage='bf16', page_tokens=16, block_tokens=16)


def test_rows_that_step_unevenly_on_another_stream(gpu_available):
    """Rows of a wider tensor, which are packed first: on the stream of the call, where they are made."""
    import torch
    print('case uneven rows', flush=True)
    made = {}
    for late in (False, True):
        cache = room.DeviceEpisodeCache(5, **OPTIONS)
        chunk = cache.extend(3)
        gen = torch.Generator('cuda').manual_seed(2)
        source = torch.randn((5, 4, 8, 32), generator=gen, device='cuda').bfloat16()
        wide = torch.zeros_like(source)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        options = {}
        if late:
            options['stream'] = side
            with torch.cuda.stream(side):
                torch.cuda._sleep(20_000_000)
                wide.copy_(source)
        else:
            wide.copy_(source)
        x = wide[:, :3]
        cache.write(chunk, x[:, :, :2], x[:, :, 2:4], **options)
        out = cache.attend(chunk, x[:, :, 4:], **options)
        torch.cuda.synchronize()
        made[late] = out, cache.layers[0].k[:5, :, :3].clone()
    for a, b in zip(made[False], made[True]):
        assert torch.equal(a, b)


