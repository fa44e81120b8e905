"""Rows gathered by their blocks: ragged chunks whose sizes the host does not know, and lists that change meanwhile."""
import numpy as np
import pytest

from libero_hip import recall
from test_gpu_episodes import World, compare, queries
from test_gpu_recall import gathers, listed_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('counts', [[33, 0, 0, 31, 1, 64, 65, 0, 95, 2, 127, 32], [0, 0, 300, 0], [1] * 30 + [200]],
                         ids=['mixed', 'one', 'singles'])
def test_unknown_sizes(gpu_available, counts):
    """Chunks that begin anywhere in a word of marks, empty worlds among them; with the largest known, not known, and less."""
    import torch
    print('case gathered unknown', len(counts), flush=True)
    world = World([min(c + 130, 420) for c in counts], 2, 64, 64, 'bf16', seed=len(counts))
    q, start = queries(counts, 4, 64, 'bf16')
    tokens = int(sum(counts))
    assert gathers(world, counts, 4, 12, 64) and gathers(world, counts, 4, 12, 64, most=tokens)
    blocks = np.random.default_rng(1).integers(-1, 7, (tokens, 2, 12)).astype(np.int32)
    at, given = torch.from_numpy(start).cuda(), torch.from_numpy(blocks).cuda()
    lse = torch.zeros((tokens, 4), device='cuda')
    out = recall.recall(world.pages, q.cuda(), given, at, block_tokens=64, lse=lse)
    compare(out, lse, listed_attention(world, q, start, blocks, 64, True), 'bf16')
    assert torch.equal(out, recall.recall(world.pages, q.cuda(), given, at, block_tokens=64, max_count=max(counts)))
    # rows behind the last world's, and those beyond max_count, stay as they were
    more = torch.cat([q.cuda(), torch.ones((37, 4, 64), dtype=torch.bfloat16, device='cuda')])
    lists = torch.cat([given, torch.zeros((37, 2, 12), dtype=torch.int32, device='cuda')])
    target = torch.full_like(more, 7)
    recall.recall(world.pages, more, lists, at, block_tokens=64, max_count=70, out=target)
    kept = np.concatenate([np.arange(start[w], start[w] + min(c, 70)) for w, c in enumerate(counts)])
    left = np.setdiff1d(np.arange(tokens + 37), kept)
    assert bool((target[torch.from_numpy(left).cuda()] == 7).all())
    if gathers(world, counts + [37], 4, 12, 64, most=70):
        assert torch.equal(target[torch.from_numpy(kept).cuda()], out[torch.from_numpy(kept).cuda()])


def test_many_worlds(gpu_available):
    """A thousand worlds' ragged chunks over long tables: little more memory than the sums where the largest is not known."""
    import torch
    print('case gathered many worlds', flush=True)
    n, kv, dim, width = 1024, 8, 128, 128
    gen = torch.Generator('cuda').manual_seed(0)
    k, v = (torch.randn((4096, kv, 64, dim), generator=gen, device='cuda').bfloat16() for _ in range(2))
    from libero_hip import episodes
    table = torch.randint(0, 4096, (n, width), generator=gen, dtype=torch.int32, device='cuda')
    length = torch.randint(200, width * 64 + 1, (n,), generator=gen, dtype=torch.int32, device='cuda')
    pages = episodes.Pages(k, v, table, length)
    counts = torch.randint(0, 65, (n,), generator=gen, device='cuda')
    start = torch.zeros(n + 1, dtype=torch.int32, device='cuda')
    start[1:] = counts.cumsum(0)
    tokens = 32768
    q = torch.randn((tokens, kv, dim), generator=gen, device='cuda').bfloat16()
    blocks = torch.randint(0, 128, (tokens, kv, 19), generator=gen, dtype=torch.int32, device='cuda')
    made = []
    for most in (64, None):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        made.append(recall.recall(pages, q, blocks, start, block_tokens=64, max_count=most, out=torch.zeros_like(q)))
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - before < 1.2 * 2 ** 30
    assert torch.equal(*made) and bool(made[0][:int(start[-1])].any())


def test_lists_that_change(gpu_available):
    """Lists written from another stream while they are attended to: the call ends, and writes nothing but its results."""
    import torch
    print('case changing lists', flush=True)
    world = World([500, 310], 2, 64, 64, 'bf16', seed=5)
    q, start = queries([200, 130], 4, 64, 'bf16')
    assert gathers(world, [200, 130], 4, 12, 64)
    rng = np.random.default_rng(0)
    lists = [torch.from_numpy(rng.integers(-1, 8, (330, 2, 12)).astype(np.int32)).cuda() for _ in range(2)]
    given, at, side = lists[0].clone(), torch.from_numpy(start).cuda(), torch.cuda.Stream()
    whole = torch.full((3, 330, 4, 64), 7.0, dtype=torch.bfloat16, device='cuda')
    rows = q.cuda()
    torch.cuda.synchronize()
    for i in range(20):
        with torch.cuda.stream(side):
            for j in range(10):
                given.copy_(lists[j % 2])
        recall.recall(world.pages, rows, given, at, block_tokens=64, out=whole[1])
    torch.cuda.synchronize()
    assert bool((whole[0] == 7).all()) and bool((whole[2] == 7).all())
    out = recall.recall(world.pages, rows, lists[1], at, block_tokens=64)
    compare(out, None, listed_attention(world, q, start, lists[1].cpu().numpy(), 64, True), 'bf16')


def test_replays_with_other_chunks(gpu_available):
    """A captured call whose chunks and lengths change between replays: the same as the eager one."""
    import torch
    print('case gathered replays', flush=True)
    world = World([420] * 9, 2, 64, 64, 'bf16', seed=8)
    rng = np.random.default_rng(5)
    tokens, at = 500, torch.zeros(10, dtype=torch.int32, device='cuda')
    q = torch.randn((tokens, 4, 64), device='cuda').bfloat16()
    lists = torch.from_numpy(rng.integers(-1, 7, (tokens, 2, 12)).astype(np.int32)).cuda()
    out = torch.zeros_like(q)
    assert gathers(world, [tokens] + [0] * 8, 4, 12, 64)

    def call(to):
        return recall.recall(world.pages, q, lists, at, block_tokens=64, out=to)

    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for i in range(8):
        cuts = np.sort(rng.integers(0, tokens + 1, 8)) if i % 2 else np.repeat([0, 37, 400, tokens], 2)
        start = np.concatenate([[0], cuts, [tokens if i < 6 else max(cuts[-1], 450)]])
        at.copy_(torch.from_numpy(start.astype(np.int32)))
        world.pages.length.copy_(torch.from_numpy(rng.integers(0, 421, 9).astype(np.int32)))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = call(torch.full_like(out, 7))
        assert torch.equal(out, want), i
        assert bool((out[int(start[-1]):] == 7).all())


def test_chunks_without_rows(gpu_available):
    import torch
    from libero_hip import room
    print('case no new tokens', flush=True)
    cache = room.DeviceEpisodeCache(3, kv_heads=2, head_dim=32, tokens=64, storage='bf16', page_tokens=16, block_tokens=16)
    cache.extend(5)
    chunk = cache.extend(0)
    q, k = (torch.zeros((3, 0, h, 32), dtype=torch.bfloat16, device='cuda') for h in (4, 2))
    cache.write(chunk, k, k)
    for causal in (True, False):
        assert cache.recall(chunk, q, top=2, causal=causal).shape == q.shape and cache.attend(chunk, q, causal=causal).shape == q.shape
    assert [x.shape for x in cache.places(chunk)] == [(3, 0)] * 3
    none = cache.extend(torch.zeros(3, dtype=torch.int32, device='cuda'), rows=4)
    rows = torch.ones((4, 4, 32), dtype=torch.bfloat16, device='cuda')
    out = torch.full_like(rows, 7)
    cache.write(none, rows[:, :2], rows[:, :2])
    assert bool((cache.recall(none, rows, top=1, causal=False, out=out) == 7).all()) and cache.lengths.tolist() == [5] * 3
