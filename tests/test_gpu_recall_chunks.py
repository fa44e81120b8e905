"""Blocks for chunks that are longer than max_count."""
import pytest

from libero_hip import recall
from test_gpu_episodes import World, compare, queries
from test_gpu_recall import expected_blocks, listed_attention, summarised

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('most', [0, 1, 4, 39, 100])
def test_tokens_behind_max_count_are_seen(gpu_available, most):
    """Queries that see all of their world see its last blocks too, in chunks of one size that are longer than max_count."""
    import torch
    print('case behind max_count', most, flush=True)
    world = World([200, 331, 45], 2, 64, 64, 'bf16', seed=3)
    counts = [40, 40, 40]
    q, start = queries(counts, 4, 64, 'bf16')
    s = summarised(world, 16)
    x = q.cuda().view(3, 40, 4, 64)
    blocks = recall.select(s, x, top=1, near=1, causal=False, max_count=most)
    assert blocks.shape[3] == 2 + (max(most, 40) + 14) // 16
    got = blocks.cpu().numpy().reshape(120, 2, -1)
    for r, row in enumerate(expected_blocks(world, q, start, 16, 1, 1, 0, False)):
        for h, want in enumerate(row if r % 40 < most else [[], []]):
            assert got[r, h].tolist() == want + [-1] * (got.shape[2] - len(want)), (r, h)
    out = recall.recall(world.pages, x, blocks, block_tokens=16, causal=False)
    compare(out, None, listed_attention(world, q, start, got, 16, False), 'bf16')


def test_ragged_chunks_beyond_max_count(gpu_available):
    """Where the sizes are known on the device alone, a list has as many places as max_count tokens need: the first blocks of
    it, in their order."""
    import torch
    print('case ragged beyond max_count', flush=True)
    world = World([200, 331], 2, 64, 64, 'bf16', seed=3)
    q, start = queries([40, 3], 4, 64, 'bf16')
    s, at = summarised(world, 16), torch.from_numpy(start).cuda()
    for most, whole in ((4, False), (40, True), (None, True)):
        blocks = recall.select(s, q.cuda(), at, top=1, near=1, causal=False, max_count=most)
        got = blocks.cpu().numpy()
        for r, row in enumerate(expected_blocks(world, q, start, 16, 1, 1, 0, False)):
            for h, want in enumerate(row):
                if not whole and 4 <= r < 40:
                    want = []
                assert got[r, h].tolist() == (want + [-1] * 9)[:got.shape[2]], (most, r, h)
