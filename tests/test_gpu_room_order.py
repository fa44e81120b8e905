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




@pytest.mark.parametrize('behind', ['changes', 'places'])
def test_places_follow_the_last_change(gpu_available, behind):
    """A chunk's places asked for on another stream than that of the changes before and after, whichever is behind."""
    import torch
    print('case places order', behind, flush=True)
    cache = room.DeviceEpisodeCache(5, **OPTIONS)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(6):
        if behind == 'changes':
            torch.cuda._sleep(20_000_000)
        chunk = cache.extend(3)
        with torch.cuda.stream(side):
            if behind == 'places':
                torch.cuda._sleep(20_000_000)
            world, position, slot = cache.places(chunk)
        cache.extend(2)
        torch.cuda.synchronize()
        assert position.tolist() == [[5 * i, 5 * i + 1, 5 * i + 2]] * 5
        assert world.tolist() == [[w] * 3 for w in range(5)]
        pages = cache.table[:, [5 * i // 16, (5 * i + 1) // 16, (5 * i + 2) // 16]]
        assert torch.equal(slot, pages * 16 + position % 16)
