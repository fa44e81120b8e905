"""Attention to listed blocks in tables that reach further than any world does."""
import numpy as np
import pytest

from libero_hip import episodes, recall
from test_gpu_episodes import World, compare, queries
from test_gpu_recall import listed_attention

pytestmark = pytest.mark.gpu


def sizes(world, tokens, heads, listed, block, longest):
    """The workspace of a call in which every world has tokens / worlds new ones."""
    import ctypes as ct
    s, n = world.pages.struct, len(world.lengths)
    rows = episodes.MxRows(4096, heads * s.head_dim, s.head_dim, heads, s.type)
    a = episodes.MxAttention(rows, rows, None, None, 0, tokens // n, 1, 0, 0.1, longest)
    chunk, m = episodes.MxChunk(None, tokens, tokens // n), episodes.MxSelection(4096, listed)
    return episodes.load().mx_recall_workspace(*(ct.byref(x) for x in (s, chunk, a, m)), block)


@pytest.mark.parametrize('longest', [0, 512, 64, 1, 2 ** 31 - 1])
def test_longest_is_a_hint(gpu_available, longest):
    """Right, wrong or not known: the results are the definition's, gathered or not."""
    import torch
    print('case recall longest', longest, flush=True)
    world = World([512, 400], 2, 64, 64, 'bf16', seed=4, width=1000)
    q, start = queries([200, 200], 4, 64, 'bf16')
    blocks = np.random.default_rng(3).integers(-1, 9, (400, 2, 12)).astype(np.int32)
    lse = torch.zeros((2, 200, 4), device='cuda')
    out = recall.recall(world.pages, q.cuda().view(2, 200, 4, 64), torch.from_numpy(blocks).cuda().view(2, 200, 2, 12), block_tokens=64,
                        longest=longest, lse=lse)
    compare(out, lse, listed_attention(world, q, start, blocks, 64, True), 'bf16')
    parts = 400 * 4 * (64 + 2) * 4
    if longest in (64, 512):
        assert sizes(world, 400, 4, 12, 64, longest) > 12 * parts          # gathered
    if not longest:
        assert sizes(world, 400, 4, 12, 64, longest) < 12 * parts


def test_caches_say_what_they_know(gpu_available):
    """A cache made for long episodes takes the same way for short ones as one made for those."""
    import torch
    print('case recall of a large cache', flush=True)
    made = []
    for tokens in (1024, 262144):
        cache = episodes.EpisodeCache(2, kv_heads=2, head_dim=64, tokens=tokens, pages=40, storage='bf16', page_tokens=64, block_tokens=64)
        gen = torch.Generator('cuda').manual_seed(1)
        chunk = cache.extend(600)
        q = torch.randn((2, 600, 4, 64), generator=gen, device='cuda').bfloat16()
        k, v = (torch.randn((2, 600, 2, 64), generator=gen, device='cuda').bfloat16() for _ in range(2))
        cache.write(chunk, k, v)
        made.append(cache.recall(chunk, q, top=4, near=2, first=1))
    assert torch.equal(*made)
    with pytest.raises(ValueError, match='longest'):
        cache.recall(chunk, q, top=4, longest=-1)
