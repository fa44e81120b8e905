"""Recall on the GPU against its definitions (tests/recall_reference.py): summaries and chosen blocks are whole numbers and
compared for equality, attention to them with the tolerances of tests/test_gpu_episodes.py."""
import math

import numpy as np
import pytest

from recall_reference import blocks_of, summary
from libero_hip import episodes, recall
from test_gpu_episodes import World, compare, queries

pytestmark = pytest.mark.gpu


def listed_attention(world, q, start, blocks, block, causal, scale=None):
    """(out, lse, sum p |v|) of the rows over the keys of their blocks (rows, kv, listed), each as often as it is listed."""
    q = q.double().numpy()
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, lse, size = np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(q.shape)
    kv = world.k[0].shape[1]
    group = q.shape[1] // kv
    for w in range(len(world.lengths)):
        length, count = int(world.lengths[w]), start[w + 1] - start[w]
        for r in range(start[w], start[w + 1]):
            p = length - count + r - start[w]
            high = 0 if p < 0 else min(p + 1, length) if causal else length
            for h in range(q.shape[1]):
                keys = np.array([t for b in blocks[r, h // group] if b >= 0 for t in range(b * block, min((b + 1) * block, high))], int)
                if not len(keys):
                    continue
                with np.errstate(all='ignore'):
                    s = scale * (world.k[w][keys, h // group] @ q[r, h])
                    top = s.max() if not np.isnan(s).any() else np.nan
                    if top == -np.inf:
                        continue
                    weight = np.exp(s - top)
                    v = world.v[w][keys, h // group]
                    out[r, h], size[r, h] = weight @ v / weight.sum(), weight @ np.abs(v) / weight.sum()
                    lse[r, h] = top + math.log(weight.sum())
    return out, lse, size


def expected_blocks(world, q, start, block, top, near, first, causal, most=2 ** 31):
    q = q.double().numpy()
    kv = world.k[0].shape[1]
    group = q.shape[1] // kv
    found = []
    for w in range(len(world.lengths)):
        length, count = int(world.lengths[w]), start[w + 1] - start[w]
        for i in range(count):
            r = start[w] + i
            found.append([blocks_of(q[r, h * group:(h + 1) * group], world.k[w][:, h], length - count + i, length, block, top, near, first,
                                    causal) if i < most else [] for h in range(kv)])
    return found


def summarised(world, block):
    """Summaries of all full blocks of all worlds, made in one call with whole histories as the chunk."""
    import torch
    s = recall.Summaries.make(world.pages, block)
    s.codes.fill_(99)
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(world.lengths)]).astype(np.int32)).cuda()
    recall.summarise(s, start, tokens=int(world.lengths.sum()))
    return s


def check(world, counts, heads, kind, block, top, near, first, causal=True, uniform=False, most=None, seed=1):
    import torch
    dim = world.pages.struct.head_dim
    q, start = queries(counts, heads, dim, kind, seed)
    s = summarised(world, block)
    options = dict(top=top, near=near, first=first, causal=causal)
    if uniform:
        x, at = q.cuda().view((len(counts), counts[0]) + q.shape[1:]), None
    else:
        x, at, options['max_count'] = q.cuda(), torch.from_numpy(start).cuda(), max(counts) if most is None else most
    blocks = recall.select(s, x, at, **options)
    assert blocks.shape[:-1] == x.shape[:-2] + (world.k[0].shape[1],)
    got = blocks.cpu().numpy().reshape(q.shape[0], -1, blocks.shape[-1])
    for r, row in enumerate(expected_blocks(world, q, start, block, top, near, first, causal)):
        for h, want in enumerate(row):
            assert got[r, h].tolist() == want + [-1] * (got.shape[2] - len(want)), (r, h)
    lse = torch.full(q.shape[:-1], 7.0, device='cuda')
    out = recall.recall(world.pages, x, blocks, at, block_tokens=block, causal=causal, lse=lse.view(x.shape[:-1]))
    compare(out, lse, listed_attention(world, q, start, got, block, causal), kind)
    return blocks


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]


# ------------------------------------------------------------------------------ summaries
@pytest.mark.parametrize('store', ['bf16', 'f16', 'fp8'])
@pytest.mark.parametrize('dim', [32, 64, 96, 128, 256])
@pytest.mark.parametrize('page,block', [(16, 16), (64, 16), (64, 32), (128, 128)])
def test_summaries(gpu_available, page, block, dim, store):
    """Chunks that complete no block, one and several: those are summarised, all others stay as they were."""
    import torch
    print('case summaries', page, block, dim, store, flush=True)
    lengths = [0, 1, block - 1, block, block + 1, 2 * block + 3, 5 * block, 5 * block + 1, 3 * block]
    counts = [0, 1, block - 1, 1, 1, block + 4, 2 * block, block + 1, 3 * block + 7]
    world = World(lengths, 3, dim, page, store, seed=dim)
    s = recall.Summaries.make(world.pages, block)
    s.codes.fill_(99)
    s.exponent.fill_(98)
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
    recall.summarise(s, start, tokens=sum(counts))
    codes, exponent = np.full(s.codes.shape, 99), np.full(s.exponent.shape, 98)
    for w, (length, count) in enumerate(zip(lengths, counts)):
        for b in range(max(length - count, 0) // block, length // block):
            at, inside = world.table[w, b * block // page], b * block % page // block
            for h in range(3):
                codes[at, h, inside], exponent[at, h, inside] = summary(world.k[w][b * block:(b + 1) * block, h])
    np.testing.assert_array_equal(s.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(s.exponent.cpu().numpy(), exponent)
    # the same number of tokens of every world
    for count in (1, 2 * block + 3):
        s.codes.fill_(99)
        recall.summarise(s, count=count)
        got = (s.codes != 99).any(-1).cpu().numpy()
        want = np.zeros(got.shape, bool)
        for w, length in enumerate(lengths):
            for b in range(max(length - count, 0) // block, length // block):
                want[world.table[w, b * block // page], :, b * block % page // block] = True
        np.testing.assert_array_equal(got, want)


def test_summaries_of_extremes(gpu_available):
    """Zeros, the smallest and largest keys, ties at half a code, infinities and NaN."""
    import torch
    print('case summary extremes', flush=True)
    world = World([160], 1, 64, 16, 'bf16', seed=3)
    k = world.k[0]
    k[:16] = 0
    k[16:32] *= 2.0 ** -60
    k[32:48] *= 2.0 ** 90
    k[48, 0, 7], k[64, 0, 8], k[80, 0, 9] = np.inf, np.nan, -np.inf
    k[81, 0, 9] = np.inf
    k[96:112] = 0
    k[96:112, 0, 0], k[96:112, 0, 1], k[96:112, 0, 2], k[96:112, 0, 3] = 127, 0.5, 1.5, -2.5
    k[112:128] = 3.3e38                                  # finite, and their sum is in 64 bits
    k[:] = torch.from_numpy(k).bfloat16().double().numpy()
    for t in range(160):
        world.pages.k[world.table[0, t // 16], :, t % 16] = torch.from_numpy(k[t]).cuda().bfloat16()
    s = summarised(world, 16)
    for b in range(10):
        c, e = summary(k[16 * b:16 * b + 16, 0])
        assert s.exponent[world.table[0, b], 0, 0].item() == e and s.codes[world.table[0, b], 0, 0].tolist() == c.tolist(), b
    assert (s.exponent == 255).sum().item() == 3


# ------------------------------------------------------------------------------ selection and attention
@pytest.mark.parametrize('kind,store', [('bf16', 'bf16'), ('f16', 'f16'), ('bf16', 'fp8'), ('f16', 'fp8')])
@pytest.mark.parametrize('dim', [32, 64, 96, 128, 256])
def test_single_tokens(gpu_available, dim, kind, store):
    """One new token of worlds of every length around the sizes of blocks, three query heads to a key head."""
    print('case recall single', dim, kind, store, flush=True)
    world = World(LENGTHS, 2, dim, 32, store, seed=dim)
    check(world, [1] * len(LENGTHS), 6, kind, 16, 3, 1, 0, uniform=True)
    check(world, [1] * len(LENGTHS), 6, kind, 32, 2, 2, 1, uniform=True)


@pytest.mark.parametrize('group', [1, 5, 16, 17, 40])
@pytest.mark.parametrize('store', ['bf16', 'fp8'])
def test_groups(gpu_available, group, store):
    """Query heads per key head below, at and above one tile's rows."""
    print('case recall group', group, store, flush=True)
    world = World([5, 164, 330], 2, 64, 16, store, seed=group)
    check(world, [1, 1, 1], 2 * group, 'bf16', 16, 4, 1, 1, uniform=True)
    check(world, [2, 3, 7], 2 * group, 'bf16', 16, 4, 1, 1)


@pytest.mark.parametrize('kind,store', [('bf16', 'bf16'), ('f16', 'fp8')])
@pytest.mark.parametrize('dim', [32, 96, 128])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('top,near,first', [(2, 1, 0), (0, 3, 2), (5, 2, 1), (64, 1, 0)])
def test_chunks(gpu_available, top, near, first, causal, dim, kind, store):
    """Ragged chunks: none, one, whole prompts; nothing chosen, everything chosen."""
    print('case recall chunk', dim, kind, store, causal, top, near, first, flush=True)
    lengths, counts = [0, 1, 9, 33, 64, 150, 200, 177, 240], [0, 1, 9, 5, 0, 40, 37, 1, 33]
    world = World(lengths, 2, dim, 32, store, seed=3 * dim + top)
    check(world, counts, 4, kind, 16, top, near, first, causal)


@pytest.mark.parametrize('page,block,length', [(16, 16, 9000), (64, 16, 36000), (256, 16, 140000), (4096, 512, 70000)])
def test_long_episodes(gpu_available, page, block, length):
    """Teams of one, four and sixteen waves, and more blocks than those hold at once; short worlds beside."""
    print('case recall long', page, block, length, flush=True)
    world = World([length, 77, length // 3, 0], 1, 32, page, 'bf16', seed=page)
    check(world, [1, 1, 1, 1], 2, 'bf16', block, 7, 2, 1, uniform=True)
    check(world, [2, 1, 3, 0], 2, 'bf16', block, 33, 1, 0)


def test_the_most_blocks(gpu_available):
    """As many as can be chosen, over several segments."""
    print('case recall most', flush=True)
    world = World([9000 * 16], 1, 32, 64, 'bf16', seed=1)
    check(world, [1], 1, 'bf16', 16, 1024, 1, 1)
    check(world, [1], 1, 'bf16', 16, 1023, 2, 3)


def test_equal_scores(gpu_available):
    """Of blocks with equal scores the earlier are chosen, in every team and across segments."""
    import torch
    print('case recall ties', flush=True)
    for length, page in ((1700, 16), (20000, 64), (140000, 256)):
        world = World([length], 1, 32, page, 'bf16', seed=2)
        s = recall.Summaries.make(world.pages, 16)
        s.exponent.fill_(127)
        q = torch.ones((1, 1, 2, 32), device='cuda').bfloat16()
        blocks = recall.select(s, q, top=5, near=1, first=1)[0, 0, 0].tolist()
        last = (length - 1) // 16
        assert blocks == [0, 1, 2, 3, 4, 5, last]
        best = [last // 2, last - 1, 7]
        for b in best:
            s.codes[world.table[0, b * 16 // page], 0, b * 16 % page // 16] = 1
        assert recall.select(s, q, top=5, near=1, first=1)[0, 0, 0].tolist() == [0, 1, 2] + sorted(best) + [last]
        # a block that is not finite stands above all
        s.exponent[world.table[0, 100 * 16 // page], 0, 100 * 16 % page // 16] = 255
        if page == 256:
            assert 100 in recall.select(s, q, top=1, near=1, first=0)[0, 0, 0].tolist()


def test_pages_that_are_not_there(gpu_available):
    """Table entries that name no page stand below all others, and their keys are not seen."""
    import torch
    print('case recall missing', flush=True)
    world = World([200], 1, 64, 16, 'bf16', seed=4)
    s = summarised(world, 16)
    q, start = queries([1], 2, 64, 'bf16')
    missing = (2, 5, 11)
    for i, b in enumerate(missing):
        world.pages.table[0, b] = (-1, 2 ** 31 - 1, s.codes.shape[0])[i]
    blocks = recall.select(s, q.cuda()[None], top=8, near=2, first=1)
    got = blocks[0, 0, 0].tolist()
    want = blocks_of(q[0].double().numpy(), world.k[0][:, 0], 199, 200, 16, 8, 2, 1, True, missing)
    assert got == want and 5 not in got and 11 in got
    out = recall.recall(world.pages, q.cuda()[None], blocks, block_tokens=16)
    seen = np.array([[[b for b in want if b not in missing]]])
    compare(out, None, listed_attention(world, q, start, seen, 16, True), 'bf16')
    blocks.fill_(2)
    assert not recall.recall(world.pages, q.cuda()[None], blocks, block_tokens=16).any()


@pytest.mark.parametrize('store', ['bf16', 'fp8'])
@pytest.mark.parametrize('listed', [3, 40, 700])
def test_lists_of_the_caller(gpu_available, listed, store):
    """Any order, gaps, numbers that are no block, blocks listed twice; short lists and lists that are split."""
    import torch
    print('case recall lists', listed, store, flush=True)
    rng = np.random.default_rng(listed)
    world = World([200, 0, 1500, 33], 2, 64, 64, store, seed=5)
    counts = [2, 0, 1, 3]
    q, start = queries(counts, 6, 64, 'bf16')
    blocks = rng.integers(-3, 100, (6, 2, listed)).astype(np.int32)
    blocks[0, 0, :] = -1
    blocks[1, 1, 0], blocks[1, 1, 1] = 2 ** 31 - 1, -2 ** 31
    blocks[2, 0, :] = 0
    valid = np.where(blocks < 1536 // 32, blocks, -1)
    at = torch.from_numpy(start).cuda()
    for causal in (True, False):
        lse = torch.zeros((6, 6), device='cuda')
        out = recall.recall(world.pages, q.cuda(), torch.from_numpy(blocks).cuda(), at, block_tokens=32, causal=causal, lse=lse)
        compare(out, lse, listed_attention(world, q, start, valid, 32, causal), 'bf16')
        again = recall.recall(world.pages, q.cuda(), torch.from_numpy(blocks).cuda(), at, block_tokens=32, causal=causal)
        assert torch.equal(out, again)


# 8-bit values have no infinity of their own
@pytest.mark.parametrize('bad,store', [(np.inf, 'bf16'), (-np.inf, 'bf16'), (np.nan, 'bf16'), (np.nan, 'fp8')])
def test_hidden_values_stay_hidden(gpu_available, bad, store):
    """An infinity or NaN in a key or value reaches the queries whose blocks hold it and who see it, and no others; what
    lies behind a world's last token is whatever was left there (here NaN)."""
    import torch
    print('case recall hidden', bad, store, flush=True)
    world = World([100, 90], 1, 64, 16, store, seed=6)
    world.v[0][40, 0, 5 if store != 'fp8' else slice(0, 32)] = bad
    world.v[1][89, 0, 6 if store != 'fp8' else slice(0, 32)] = bad
    for w, t in ((0, 40), (1, 89)):
        if store == 'fp8':
            world.pages.v_scale[world.table[w, t // 16], 0, t % 16, 0] = 255
        else:
            world.pages.v[world.table[w, t // 16], 0, t % 16] = torch.from_numpy(world.v[w][t, 0]).cuda().bfloat16()
    q, start = queries([3, 2], 2, 64, 'bf16')
    at = torch.from_numpy(start).cuda()
    for lists in ([0, 1, 6], [0, 2, 6], [5, 5, 2]):
        blocks = np.tile(np.array(lists, np.int32), (5, 1, 1))
        for causal in (True, False):
            out = recall.recall(world.pages, q.cuda(), torch.from_numpy(blocks).cuda(), at, block_tokens=16, causal=causal)
            compare(out, None, listed_attention(world, q, start, blocks, 16, causal), 'bf16')


def test_blocks_that_are_not_finite_are_seen(gpu_available):
    """A key that is NaN makes its block the first choice, and the result NaN, as in attention to everything."""
    import torch
    print('case recall nan key', flush=True)
    world = World([400], 1, 64, 16, 'bf16', seed=7)
    world.pages.k[world.table[0, 3], 0, 2, 1] = float('nan')
    q, _ = queries([1], 2, 64, 'bf16')
    s = summarised(world, 16)
    blocks = recall.select(s, q.cuda()[None], top=1)
    assert blocks[0, 0, 0].tolist() == [3, 24]
    assert bool(recall.recall(world.pages, q.cuda()[None], blocks, block_tokens=16).isnan().all())
    assert bool(episodes.attend(world.pages, q.cuda()[None]).isnan().all())


def test_queries_of_any_size(gpu_available):
    """Zeros, infinities, NaN and numbers beyond the scales in queries choose as defined."""
    print('case recall queries', flush=True)
    import torch
    world = World([500, 500, 500, 500, 500], 1, 64, 16, 'bf16', seed=8)
    q, start = queries([1] * 5, 3, 64, 'bf16')
    q[0] = 0
    q[1, 0, 3] = float('nan')
    q[2, 1, 4], q[2, 2, 5] = float('inf'), float('-inf')
    q[3] *= 2.0 ** 100
    q[4] *= 2.0 ** -60
    s = summarised(world, 16)
    got = recall.select(s, q.cuda()[:, None], top=4, near=2, first=1).cpu().numpy()
    for r, row in enumerate(expected_blocks(world, q, start, 16, 4, 2, 1, True)):
        assert got[r, 0, 0].tolist() == row[0], r


def test_rows_without_blocks(gpu_available):
    """Rows beyond the last world's or max_count, and before a world's first token: no blocks; their results are left as
    they were, or zeros where the row has a world."""
    import torch
    print('case recall no rows', flush=True)
    world = World([5, 200, 0], 1, 32, 16, 'bf16', seed=9)
    s = summarised(world, 16)
    q = torch.randn((3, 8, 2, 32), device='cuda').bfloat16()
    blocks = recall.select(s, q, top=2)
    assert bool((blocks[0, :3] == -1).all()) and bool((blocks[0, 3:, 0, 0] == 0).all()) and bool((blocks[2] == -1).all())
    out, lse = torch.full_like(q, 7), torch.full(q.shape[:-1], 7.0, device='cuda')
    recall.recall(world.pages, q, blocks, block_tokens=16, out=out, lse=lse)
    assert not out[0, :3].any() and not out[2].any() and bool(torch.isneginf(lse[0, :3]).all()) and bool(out[1].any())
    start = torch.tensor([0, 2, 6, 6], dtype=torch.int32, device='cuda')
    rows = q.view(24, 2, 32)[:9]
    blocks = recall.select(s, rows, start, top=2, max_count=3)
    assert bool((blocks[5:] == -1).all()) and not bool((blocks[:5] == -1).all(-1).any())
    out = torch.full_like(rows, 7)
    recall.recall(world.pages, rows, recall.select(s, rows, start, top=2), start, block_tokens=16, max_count=3, out=out)
    assert bool((out[5:] == 7).all()) and not bool((out[:5] == 7).all(-1).any())
    empty = recall.select(s, rows[:0], start, top=2)
    assert empty.shape == (0, 1, 3) and recall.recall(world.pages, rows[:0], empty, start, block_tokens=16).shape == (0, 2, 32)


@pytest.mark.parametrize('offset', [0, 1, 4])
def test_strides(gpu_available, offset):
    import torch
    print('case recall strides', offset, flush=True)
    world = World([133, 264, 100], 2, 64, 16, 'bf16', seed=11)
    q, start = queries([1, 5, 2], 4, 64, 'bf16')
    wide = torch.full((q.shape[0], 1000), float('nan'), dtype=torch.bfloat16, device='cuda')
    inside = wide.as_strided(q.shape, (1000, 80, 1), offset)
    inside.copy_(q)
    s, at = summarised(world, 16), torch.from_numpy(start).cuda()
    blocks = recall.select(s, inside, at, top=3)
    assert torch.equal(blocks, recall.select(s, q.cuda(), at, top=3))
    target = torch.zeros((q.shape[0], 3, 4, 72), dtype=torch.bfloat16, device='cuda')
    out = target[:, 1, :, offset:offset + 64]
    assert recall.recall(world.pages, inside, blocks, at, block_tokens=16, out=out) is out
    assert torch.equal(out, recall.recall(world.pages, q.cuda(), blocks, at, block_tokens=16))
    out.zero_()
    assert not target.any()


@pytest.mark.parametrize('listed', [12, 600])
def test_captured_calls_follow_the_lengths(gpu_available, listed):
    """summarise, select and recall in a HIP graph, with the keys split and not."""
    import torch
    print('case recall graph', listed, flush=True)
    world = World([9000, 880, 12000], 2, 64, 16, 'bf16', seed=13)
    p = world.pages
    final = p.length.clone()
    s = summarised(world, 16)
    q = torch.randn((3, 2, 4, 64), device='cuda').bfloat16()

    def step():
        recall.summarise(s, count=2)
        blocks = recall.select(s, q, top=listed)
        return blocks, recall.recall(p, q, blocks, block_tokens=16)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        p.length.copy_(final - 37 * i)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_other_stream(gpu_available):
    import torch
    print('case recall stream', flush=True)
    world = World([3000, 2500, 77], 2, 128, 64, 'fp8', seed=12)
    side = torch.cuda.Stream()
    q, start = queries([1, 1, 1], 8, 128, 'bf16')
    q, first = q.cuda(), torch.from_numpy(start).cuda()
    s = recall.Summaries.make(world.pages, 16)
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    recall.summarise(s, count=3000, stream=side)
    blocks = recall.select(s, q, first, top=30, stream=side)
    out = recall.recall(world.pages, q, blocks, first, block_tokens=16, stream=side)
    torch.cuda.synchronize()
    t = summarised(world, 16)
    assert torch.equal(blocks, recall.select(t, q, first, top=30))
    assert torch.equal(out, recall.recall(world.pages, q, blocks, first, block_tokens=16))


def test_offsets_beyond_32_bits(gpu_available):
    """Pages whose elements lie past 2^31 and 2^32: keys, values and summaries are found there."""
    import torch
    print('case recall far', flush=True)
    npage, page, dim = 33000, 64, 256
    k = torch.zeros((npage, 8, page, dim), dtype=torch.bfloat16, device='cuda')
    v = torch.zeros_like(k)
    ids = torch.tensor([[32999, 17000, 5, 32998, 16500, 8300, 32997]], dtype=torch.int32, device='cuda')
    length = torch.tensor([420], dtype=torch.int32, device='cuda')
    gen = torch.Generator('cuda').manual_seed(0)
    small = [torch.randn((7, 8, page, dim), generator=gen, device='cuda').bfloat16() for _ in range(2)]
    k[ids[0].long()], v[ids[0].long()] = small
    near = episodes.Pages(*small, torch.arange(7, dtype=torch.int32, device='cuda')[None].contiguous(), length)
    far = episodes.Pages(k, v, ids, length)
    q = torch.randn((1, 1, 16, dim), generator=gen, device='cuda').bfloat16()
    got = []
    for p in (near, far):
        s = recall.Summaries.make(p, 16)
        recall.summarise(s, count=420)
        blocks = recall.select(s, q, top=6, first=1)
        got.append((blocks, recall.recall(p, q, blocks, block_tokens=16)))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize('causal', [True, False])
def test_everything_chosen_is_attention(gpu_available, causal):
    """With room for all blocks, recall is attend: through the cache, over many steps."""
    import torch
    from libero_hip.rotary import Rotary
    print('case recall all', causal, flush=True)
    n, turning = 5, Rotary.make(64, layout='interleaved')
    c = episodes.EpisodeCache(n, kv_heads=2, head_dim=64, tokens=300, storage='bf16', page_tokens=32, block_tokens=16)
    rng = np.random.default_rng(0)
    for step in range(10):
        counts = rng.integers(0, 30, n)
        chunk = c.extend(counts, range(n)) if step % 2 else c.extend(int(counts[0]) + 1)
        q, k, v = (torch.randn(chunk.shape + (h, 64), device='cuda').bfloat16() for h in (6, 2, 2))
        x = c.enter(chunk, turning, q, k, v)
        a, b = c.attend(chunk, x, causal=causal), c.recall(chunk, x, top=40, near=2, first=1, causal=causal)
        # each is within 2^-8 (|out| + sum p |v|) / sqrt 3 or so of the same values
        assert (a.double() - b.double()).norm() <= 2.0 ** -7 * a.double().norm()
        # fewer blocks: what select and recall give by themselves
        got = c.recall(chunk, x, top=2, near=1, first=1, causal=causal)
        options = dict(causal=causal, max_count=chunk.count) if chunk.start is not None else dict(causal=causal)
        blocks = recall.select(c.summaries[0], x, chunk.start, top=2, near=1, first=1, **options)
        assert torch.equal(got, recall.recall(c.layers[0], x, blocks, chunk.start, block_tokens=16, **options))
        if step == 6:
            c.reset([1, 3])


def test_refusals(gpu_available):
    import torch
    print('case recall refusals', flush=True)
    world = World([50, 200], 2, 64, 32, 'bf16', seed=1)
    p, s = world.pages, recall.Summaries.make(world.pages, 16)
    q = torch.randn((2, 1, 4, 64), device='cuda').bfloat16()
    blocks = recall.select(s, q, top=2)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device='cuda')
    cache = episodes.EpisodeCache(2, kv_heads=1, head_dim=32, tokens=40, storage='bf16')
    other = episodes.EpisodeCache(2, kv_heads=1, head_dim=32, tokens=40, storage='bf16', block_tokens=16)
    rows = torch.randn((2, 1, 1, 32), device='cuda').bfloat16()
    bad = [lambda: recall.Summaries.make(p, 8), lambda: recall.Summaries.make(p, 64), lambda: recall.Summaries.make(p, 24),
           lambda: recall.Summaries(p, s.codes.float(), s.exponent), lambda: recall.Summaries(p, s.codes, s.exponent[:1]),
           lambda: recall.Summaries(p, s.codes.cpu(), s.exponent.cpu()), lambda: recall.summarise(s),
           lambda: recall.summarise(s, tokens=3), lambda: recall.summarise(s, start, count=1), lambda: recall.summarise(s, count=-1),
           lambda: recall.select(s, q, top=-1), lambda: recall.select(s, q, top=1025), lambda: recall.select(s, q, top=1, near=0),
           lambda: recall.select(s, q, top=1, first=-1), lambda: recall.select(s, q, top=1, near=4096),
           lambda: recall.select(s, q[:, :, :3], top=1), lambda: recall.select(s, q.half(), top=1),
           lambda: recall.select(s, q.float(), top=1), lambda: recall.select(s, q, start, top=1),
           lambda: recall.select(s, q, top=1, out=blocks), lambda: recall.select(s, q.clone().requires_grad_(), top=1),
           lambda: recall.recall(p, q, blocks, block_tokens=8), lambda: recall.recall(p, q, blocks, block_tokens=64),
           lambda: recall.recall(p, q, blocks.long(), block_tokens=16), lambda: recall.recall(p, q, blocks[:1], block_tokens=16),
           lambda: recall.recall(p, q, blocks[..., :0], block_tokens=16), lambda: recall.recall(p, q, blocks[:, :, :1], block_tokens=16),
           lambda: recall.recall(p, q, blocks.transpose(0, 1), block_tokens=16), lambda: recall.recall(p, q, blocks.cpu(), block_tokens=16),
           lambda: recall.recall(p, q, blocks, block_tokens=16, scale=float('inf')),
           lambda: recall.recall(p, q, blocks, block_tokens=16, scale=1e39),
           lambda: recall.recall(p, q, blocks, block_tokens=16, out=q.new_zeros((1, 1, 4, 64)).expand(2, 1, 4, 64)),
           lambda: recall.recall(p, q, blocks, block_tokens=16, lse=torch.zeros(3, device='cuda')),
           lambda: recall.recall(p, q.clone().requires_grad_(), blocks, block_tokens=16),
           lambda: cache.recall(cache.extend(1), rows, top=1), lambda: other.recall(other.extend(1), rows, top=1, scale=-1.0),
           lambda: episodes.EpisodeCache(2, kv_heads=1, head_dim=32, tokens=40, block_tokens=128)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('not refused', i)


# ------------------------------------------------------------------------------ rows that share blocks
def gathers(world, counts, heads, listed, block, most=None):
    """Whether the rows of such a call are gathered by their blocks: its workspace then has more than the parts' numbers."""
    import ctypes as ct
    import torch
    s = world.pages.struct
    tokens = int(np.sum(counts))
    start = torch.zeros(len(counts) + 1, dtype=torch.int32, device='cuda')
    chunk = episodes.MxChunk(start.data_ptr(), tokens, 0)
    kind = s.type if s.type != 3 else 1
    rows = episodes.MxRows(start.data_ptr(), heads * s.head_dim, s.head_dim, heads, kind)
    a = episodes.MxAttention(rows, rows, None, None, 0, max(counts) if most is None else most, 1, 0, 0.1, 0)
    m = episodes.MxSelection(start.data_ptr(), listed)
    need = episodes.load().mx_recall_workspace(*(ct.byref(x) for x in (s, chunk, a, m)), block)
    return need % (tokens * heads * (s.head_dim + 2) * 4) != 0


@pytest.mark.parametrize('kind,store', [('bf16', 'bf16'), ('f16', 'f16'), ('bf16', 'fp8'), ('f16', 'fp8')])
@pytest.mark.parametrize('dim,block,page,heads', [(32, 64, 64, 6), (64, 32, 32, 2), (96, 64, 128, 6), (128, 64, 64, 6),
                                                  (128, 128, 256, 4), (256, 64, 64, 6), (256, 128, 128, 2)])
def test_gathered_rows(gpu_available, dim, block, page, heads, kind, store):
    """Chunks of hundreds of tokens, whose rows are gathered by the blocks that they share: full and partial tiles, blocks of
    less than a step's keys, one step's and more; worlds of other lengths beside."""
    print('case gathered', dim, block, page, heads, kind, store, flush=True)
    world = World([700, 40, 0, 530], 2, dim, page, store, seed=dim + block)
    counts = [260, 40, 0, 97]
    assert gathers(world, counts, heads, 9, block)
    for causal in (True, False):
        check(world, counts, heads, kind, block, 4, 2, 3, causal)


@pytest.mark.parametrize('group', [1, 2, 5, 7, 8])
def test_gathered_groups(gpu_available, group):
    print('case gathered group', group, flush=True)
    world = World([600, 300], 3, 64, 128, 'bf16', seed=group)
    assert gathers(world, [150, 150], 3 * group, 4, 128)
    check(world, [150, 150], 3 * group, 'bf16', 128, 2, 1, 1, uniform=True)
    check(world, [150, 33], 3 * group, 'bf16', 128, 2, 1, 1, causal=False)


@pytest.mark.parametrize('store', ['bf16', 'fp8'])
def test_gathered_lists_of_the_caller(gpu_available, store):
    """Blocks listed twice, not at all, out of order, that are none; rows beyond max_count are left as they were."""
    import torch
    print('case gathered lists', store, flush=True)
    rng = np.random.default_rng(3)
    world = World([500, 310, 130], 2, 64, 64, store, seed=5)
    counts = [200, 0, 130]
    q, start = queries(counts, 4, 64, 'bf16')
    blocks = rng.integers(-2, 11, (330, 2, 12)).astype(np.int32)
    blocks[0, 0, :] = -1
    blocks[1, 1, :2] = 2 ** 31 - 1, -2 ** 31
    blocks[2, 0, :] = 0
    blocks[200:, 1, 5] = blocks[200:, 1, 4]
    assert gathers(world, counts, 4, 12, 64)
    valid = np.where(blocks < 8, blocks, -1)
    at = torch.from_numpy(start).cuda()
    for causal in (True, False):
        lse = torch.zeros((330, 4), device='cuda')
        given = torch.from_numpy(blocks).cuda()
        out = recall.recall(world.pages, q.cuda(), given, at, block_tokens=64, causal=causal, lse=lse)
        want = listed_attention(world, q, start, valid, 64, causal)
        compare(out, lse, want, 'bf16')
        assert torch.equal(out, recall.recall(world.pages, q.cuda(), given, at, block_tokens=64, causal=causal))
        target = torch.full_like(out, 7)
        recall.recall(world.pages, q.cuda(), given, at, block_tokens=64, causal=causal, max_count=150, out=target)
        assert bool((target[150:200] == 7).all())
        keep = np.r_[0:150, 200:330]
        compare(target[torch.from_numpy(keep).cuda()], None, [x[keep] for x in want], 'bf16')


@pytest.mark.parametrize('bad,store', [(np.inf, 'bf16'), (np.nan, 'bf16'), (np.nan, 'fp8')])
def test_gathered_hidden_values(gpu_available, bad, store):
    """An infinity or NaN in a value reaches the gathered rows that see it and no others."""
    import torch
    print('case gathered hidden', bad, store, flush=True)
    world = World([330, 290], 1, 64, 64, store, seed=6)
    for w, t in ((0, 40), (0, 300), (1, 289)):
        world.v[w][t, 0, 5 if store != 'fp8' else slice(0, 32)] = bad
        if store == 'fp8':
            world.pages.v_scale[world.table[w, t // 64], 0, t % 64, 0] = 255
        else:
            world.pages.v[world.table[w, t // 64], 0, t % 64] = torch.from_numpy(world.v[w][t, 0]).cuda().bfloat16()
    q, start = queries([160, 200], 2, 64, 'bf16')
    blocks = np.random.default_rng(0).integers(0, 6, (360, 1, 4)).astype(np.int32)
    assert gathers(world, [160, 200], 2, 4, 64)
    at = torch.from_numpy(start).cuda()
    for causal in (True, False):
        out = recall.recall(world.pages, q.cuda(), torch.from_numpy(blocks).cuda(), at, block_tokens=64, causal=causal)
        compare(out, None, listed_attention(world, q, start, blocks, 64, causal), 'bf16')


def test_gathered_pages_that_are_not_there(gpu_available):
    import torch
    print('case gathered missing', flush=True)
    world = World([400], 1, 64, 64, 'bf16', seed=7)
    world.pages.table[0, 1] = -1
    q, start = queries([200], 2, 64, 'bf16')
    blocks = np.tile(np.array([0, 1, 4, 6], np.int32), (200, 1, 1))
    assert gathers(world, [200], 2, 4, 64)
    out = recall.recall(world.pages, q.cuda(), torch.from_numpy(blocks).cuda(), torch.from_numpy(start).cuda(), block_tokens=64)
    blocks[..., 1] = -1
    compare(out, None, listed_attention(world, q, start, blocks, 64, True), 'bf16')


def test_gathered_in_batches_of_heads(gpu_available):
    """More parts than are kept at once: key heads in several batches, of which the last is smaller; and captured."""
    import torch
    print('case gathered batches', flush=True)
    n, kv, dim = 8192, 3, 64
    gen = torch.Generator('cuda').manual_seed(0)
    k, v = (torch.randn((n // 64, kv, 64, dim), generator=gen, device='cuda').bfloat16() for _ in range(2))
    p = episodes.Pages(k, v, torch.arange(n // 64, dtype=torch.int32, device='cuda')[None].contiguous(),
                       torch.tensor([n], dtype=torch.int32, device='cuda'))
    s = recall.Summaries.make(p, 64)
    recall.summarise(s, count=n)
    q = torch.randn((1, 4096, 4 * kv, dim), generator=gen, device='cuda').bfloat16()
    blocks = recall.select(s, q, top=21, near=1, first=1)

    def call():
        lse = torch.empty(q.shape[:-1], device='cuda')
        return recall.recall(p, q, blocks, block_tokens=64, lse=lse), lse

    out, lse = call()
    # a few rows at a time: few enough that they are not gathered
    for at in (0, 1000, 4090):
        some = torch.cat([q[:, at:at + 6]], 1).contiguous()
        short = episodes.Pages(k, v, p.table, torch.tensor([n - 4096 + at + 6], dtype=torch.int32, device='cuda'))
        few = torch.empty(some.shape[:-1], device='cuda')
        want = recall.recall(short, some, blocks[:, at:at + 6].contiguous(), block_tokens=64, lse=few)
        # both within 2^-8 of |out| and a little of sum p |v|, at most 2^-12, of the same
        torch.testing.assert_close(out[:, at:at + 6].float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -10)
        torch.testing.assert_close(lse[:, at:at + 6], few, rtol=2.0 ** -17, atol=2.0 ** -11)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        for a, b in zip(kept, call()):
            assert torch.equal(a, b)


@pytest.mark.parametrize('dim,kind,store', [(64, 'bf16', 'fp8'), (128, 'f16', 'f16'), (32, 'bf16', 'bf16')])
def test_many_short_lists(gpu_available, dim, kind, store):
    """Lists of few keys in thousands of worlds: one wave to a tile."""
    print('case recall short lists', dim, kind, store, flush=True)
    lengths = np.random.default_rng(dim).integers(0, 150, 1100)
    world = World(lengths, 2, dim, 16, store, seed=dim)
    check(world, [1] * 1100, 2, kind, 16, 3, 1, 1, uniform=True)


def test_two_graphs_side_by_side(gpu_available):
    """Two captured recalls, gathered and split, replayed at once on two streams: neither uses the other's memory."""
    import torch
    print('case recall two graphs', flush=True)
    made = []
    for seed, (lengths, count, top) in enumerate((([900, 700], 200, 4), ([20000, 9000], 1, 300))):
        world = World(lengths, 2, 64, 64, 'bf16', seed=30 + seed)
        s = summarised(world, 64 if count > 1 else 16)
        q = torch.randn((2, count, 4, 64), device='cuda').bfloat16()

        def call(world=world, s=s, q=q, top=top):
            blocks = recall.select(s, q, top=top)
            return recall.recall(world.pages, q, blocks, block_tokens=s.block_tokens)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        made.append((graph, got, q, call, torch.cuda.Stream()))
    for _ in range(4):
        for _, _, q, _, _ in made:
            q.normal_()
        want = [call() for _, _, _, call, _ in made]
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, _, _, _, side in made:
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, got, _, _, _), x in zip(made, want):
            assert torch.equal(got, x)
