"""Episode memory on the GPU at the limits of its arguments: lengths, windows, values and weights where the kernels'
numbers of keys, or their 16-bit operands, reach the end of their range.  References and tolerances are those of
test_gpu_episodes.py."""
import numpy as np
import pytest

from episode_reference import attention
from libero_hip import episodes
from test_gpu_episodes import World, check, compare, expected, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('count', [1, 3, 40])
@pytest.mark.parametrize('window', [1, 31, 64, 100, 2 ** 30, 2 ** 31 - 1])
def test_lengths_up_to_32_bits(gpu_available, window, count):
    """Worlds that say they are longer than their table reaches, up to 2^31 - 1 tokens: a window that lies beyond the table
    shows nothing, one that reaches back into it shows the tokens that are there."""
    import torch
    print('case lengths', window, count, flush=True)
    lengths = np.array([2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 31, 2 ** 31 - 66, 2 ** 30 + 5, 9000], np.int64)
    for dim, store, width in ((64, 'bf16', 2), (128, 'fp8', 2), (64, 'bf16', 512)):     # not split, and split
        world = World([32] * len(lengths), 2, dim, 16, store, seed=30, width=width)
        world.pages.length.copy_(torch.from_numpy(lengths.astype(np.int32)))
        q, start = queries([count] * len(lengths), 4, dim, 'bf16')
        qd = q.double().numpy()
        ref, ref_lse, size = np.zeros(qd.shape), np.full(qd.shape[:2], -np.inf), np.zeros(qd.shape)
        for w in range(len(lengths)):
            for i in range(count):
                low, row = max(0, lengths[w] - count + i - window + 1), w * count + i
                if low < 32:
                    ref[row], ref_lse[row], size[row] = (x[0] for x in attention(
                        qd[row:row + 1], world.k[w][low:], world.v[w][low:], 31 - low, False, 0, dim ** -0.5))
        assert np.isfinite(ref_lse).any() == (window >= 2 ** 30)
        for causal in (True, False):
            lse = torch.full(q.shape[:-1], 7.0, device='cuda')
            out = episodes.attend(world.pages, q.cuda(), torch.from_numpy(start).cuda(), causal=causal, window=window,
                                  max_count=count, lse=lse)
            compare(out, lse, (ref, ref_lse, size), 'bf16')


def hot_and_cold(world, hot, gap):
    """Queries of one value whose score (scale 1) is `gap` at each world's key `hot` and 0 at the others."""
    import torch
    for w in range(len(world.lengths)):
        world.k[w][:, :, 0] = 0
        world.k[w][hot[w], :, 0] = gap
    page = world.pages.k.shape[2]
    fp8 = world.pages.k.dtype == torch.float8_e4m3fn
    values = world.pages.k.view(torch.uint8) if fp8 else world.pages.k
    code = int(torch.tensor(float(gap)).to(torch.float8_e4m3fn).view(torch.uint8)) if fp8 else gap
    for w in range(len(world.lengths)):
        for t in range(world.lengths[w]):
            where = (int(world.table[w, t // page]), slice(None), t % page)
            values[where + (0,)] = code if t == hot[w] else 0
            if fp8:
                world.pages.k_scale[where + (0,)] = 127


def first_value(counts, heads, dim, kind):
    import torch
    q, start = queries(counts, heads, dim, kind)
    q.zero_()
    q[..., 0] = 1
    return q, torch.from_numpy(start).cuda()


@pytest.mark.parametrize('gap', [10, 14, 18])
@pytest.mark.parametrize('count', [1, 40])
@pytest.mark.parametrize('kind,store', [('f16', 'f16'), ('f16', 'fp8'), ('bf16', 'bf16')])
def test_small_weights_count(gpu_available, kind, store, count, gap):
    """One key outweighs all others but has a value of zero: the output is made of the others' weights alone, each
    exp(-gap) of the largest, which are operands of 16 bits as exact as any (float16: down to 2^-26 of the largest)."""
    import torch
    print('case small weights', kind, store, count, gap, flush=True)
    for dim, width in ((64, None), (128, 512)):
        world = World([600, 700], 1, dim, 16, store, seed=31, width=width)
        hot = [5, 640]
        hot_and_cold(world, hot, gap)
        if store == 'fp8':                         # values of one sign, 64 times as large: small weights add up
            world.pages.v.view(torch.uint8).bitwise_and_(0x7f)
            world.pages.v_scale.add_(torch.where(world.pages.v_scale < 255, 6, 0).to(torch.uint8))
        else:
            world.pages.v.abs_().mul_(64)
        for w in range(2):
            world.v[w] = np.abs(world.v[w]) * 64
            world.v[w][hot[w]] = 0
            world.pages.v.view(torch.uint8 if store == 'fp8' else world.pages.v.dtype)[
                int(world.table[w, hot[w] // 16]), :, hot[w] % 16] = 0
        q, start = first_value([count] * 2, 4, dim, kind)
        lse = torch.full(q.shape[:-1], 7.0, device='cuda')
        out = episodes.attend(world.pages, q.cuda(), start, scale=1.0, lse=lse, max_count=count)
        qd = q.double().numpy()
        want = [attention(qd[w * count:(w + 1) * count], world.k[w], world.v[w], int(world.lengths[w]) - count, True, 0, 1.0)
                for w in range(2)]
        compare(out, lse, [np.concatenate(x) for x in zip(*want)], kind)


@pytest.mark.parametrize('gap', [30, 120])
@pytest.mark.parametrize('count', [1, 40])
@pytest.mark.parametrize('dim,kind,store', [(32, 'f16', 'f16'), (64, 'bf16', 'bf16'), (64, 'bf16', 'fp8'), (96, 'f16', 'f16'),
                                            (128, 'f16', 'fp8'), (128, 'bf16', 'fp8'), (256, 'bf16', 'bf16'), (256, 'f16', 'fp8')])
def test_infinite_values_of_any_weight(gpu_available, dim, kind, store, count, gap):
    """An infinity among the values gives the queries that see it an infinity, and a NaN a NaN, also where the key's
    weight is beyond the reach of 16 bits or 32, before the keys that outweigh it and after, in their part and in others."""
    import torch
    print('case infinite values', dim, kind, store, count, gap, flush=True)
    for width in (None, 512):
        lengths = [300, 300, 700, 700, 2000, 90]
        hot, cold = [0, 299 - count, 640, 5, 100, 1], [200, 7, 9, 600, 1900, 2]
        world = World(lengths, 1, dim, 16, store, seed=32, width=width)
        hot_and_cold(world, hot, gap)
        for w in range(len(lengths)):
            at = (int(world.table[w, cold[w] // 16]), 0, cold[w] % 16)
            if store == 'fp8':                     # a block of scale 2^127, whose codes are 448 or -448
                world.v[w][cold[w], 0, :32] = np.inf
                world.v[w][cold[w], 0, 3] = -np.inf
                world.pages.v.view(torch.uint8)[at][:32] = 0x7e
                world.pages.v.view(torch.uint8)[at][3] = 0xfe
                world.pages.v_scale[at][0] = 254
            else:
                for d, x in ((3, -np.inf), (4, np.inf), (dim - 1, np.nan)):
                    world.v[w][cold[w], 0, d] = x
                    world.pages.v[at][d] = x
        q, start = first_value([count] * len(lengths), 3, dim, kind)
        for causal in (True, False):
            out = episodes.attend(world.pages, q.cuda(), start, scale=1.0, causal=causal, max_count=count)
            qd = q.double().numpy()
            want = [attention(qd[w * count:(w + 1) * count], world.k[w], world.v[w], int(world.lengths[w]) - count, causal, 0, 1.0)
                    for w in range(len(lengths))]
            compare(out, None, [np.concatenate(x) for x in zip(*want)], kind)


@pytest.mark.parametrize('most,count', [(1, 5), (3, 40), (40, 41), (60, 300)])
@pytest.mark.parametrize('width', [64, 512])
def test_fewer_rows_than_the_chunks_hold(gpu_available, width, most, count):
    """max_count below the chunks' size, keys split and not: the rows before it are computed, the others not touched."""
    import torch
    print('case fewer rows', width, most, count, flush=True)
    world = World([700, 301, 999], 2, 64, 16, 'bf16', seed=33, width=width)
    q, start = queries([count] * 3, 4, 64, 'bf16')
    want = expected(world, q, start)
    here = np.arange(3 * count) % count < most
    for ragged in (False, True):
        shape = (3 * count,) if ragged else (3, count)
        out = torch.full(shape + (4, 64), 9.0, dtype=torch.bfloat16, device='cuda')
        lse = torch.full(shape + (4,), 7.0, device='cuda')
        episodes.attend(world.pages, q.cuda().view(out.shape), torch.from_numpy(start).cuda() if ragged else None,
                        max_count=most, out=out, lse=lse)
        out, lse = out.cpu().view(q.shape), lse.cpu().view(q.shape[:-1])
        compare(out[here], lse[here], [x[here] for x in want], 'bf16')
        assert bool((out[~here] == 9).all()) and bool((lse[~here] == 7).all())


@pytest.mark.parametrize('store', ['bf16', 'fp8'])
@pytest.mark.parametrize('page', [16, 64])
def test_chunks_beyond_32_bits(gpu_available, page, store):
    """Chunks of many rows over pages whose elements lie past 2^31 and 2^32."""
    import torch
    print('case far chunks', page, store, flush=True)
    kv, dim = 4, 128
    npage = 9_000_000 // page                                  # 4.6e9 elements
    kind = {'bf16': torch.bfloat16, 'fp8': torch.float8_e4m3fn}[store]
    k, v = (torch.zeros((npage, kv, page, dim), dtype=kind, device='cuda') for _ in range(2))
    scales = [torch.zeros((npage, kv, page, 4), dtype=torch.uint8, device='cuda') for _ in range(2 if store == 'fp8' else 0)]
    held = -(-150 // page)
    ids = np.linspace(npage - 1, npage // 2, 2 * held).astype(np.int32).reshape(2, held)
    pages = episodes.Pages(k, v, torch.from_numpy(ids).cuda(), torch.tensor([150, 137], dtype=torch.int32, device='cuda'), *scales)
    x, y = (torch.randn((2, 137, kv, dim), device='cuda').bfloat16() for _ in range(2))
    episodes.write(pages, x, y)
    hk, hv = (g.double().cpu().numpy() for g in episodes.read(pages, count=137))
    if store == 'bf16':
        assert np.array_equal(hk, x.double().cpu().numpy()) and np.array_equal(hv, y.double().cpu().numpy())
    q, _ = queries([137, 137], 8, dim, 'bf16')
    lse = torch.empty((2, 137, 8), device='cuda')
    out = episodes.attend(pages, q.cuda().view(2, 137, 8, dim), lse=lse)
    pad = np.zeros((13, kv, dim))
    qd = q.double().numpy()
    want = [attention(qd[:137], np.concatenate([pad, hk[0]]), np.concatenate([pad, hv[0]]), 13, True, 0, dim ** -0.5),
            attention(qd[137:], hk[1], hv[1], 0, True, 0, dim ** -0.5)]
    compare(out, lse, [np.concatenate(z) for z in zip(*want)], 'bf16')


@pytest.mark.parametrize('count', [6, 40, 300])
@pytest.mark.parametrize('dim,kind,store', [(32, 'f16', 'f16'), (64, 'bf16', 'fp8'), (96, 'f16', 'f16'), (128, 'bf16', 'bf16'),
                                            (128, 'f16', 'fp8'), (256, 'f16', 'f16')])
def test_hidden_values_of_all_types(gpu_available, dim, kind, store, count):
    """Infinities and NaN in values reach the queries that see them and no others (tokens later in the chunk, tokens that
    have left the window), for every head size and type."""
    import torch
    print('case hidden values', dim, kind, store, count, flush=True)
    for causal, window in ((True, 0), (True, 9), (False, 11)):
        world = World([count, count + 21], 1, dim, 16, store, seed=34)
        for w, token, at, bad in ((0, count - 2, 5, np.nan), (1, 12, dim - 1, np.inf), (1, count // 2, 17, -np.inf)):
            where = (int(world.table[w, token // 16]), 0, token % 16)
            if store == 'fp8':                     # a block of NaN
                at = slice(at // 32 * 32, at // 32 * 32 + 32)
                world.v[w][token, 0, at] = np.nan
                world.pages.v_scale[where + (at.start // 32,)] = 255
            else:
                world.v[w][token, 0, at] = bad
                world.pages.v[where + (at,)] = bad
        check(world, [count, count], 3, kind, causal, window, seed=35)
        check(world, [count, count - 4], 3, kind, causal, window, uniform=False, seed=36)


@pytest.mark.parametrize('count', [1, 40])
@pytest.mark.parametrize('store', ['bf16', 'fp8'])
@pytest.mark.parametrize('dim', [64, 128])
def test_sums_beyond_32_bits(gpu_available, dim, store, count):
    """Finite values whose weighted sum passes 32 bits before it is divided: an infinity of their sign, or the value
    itself where the kernel's order of sums holds it, but nothing smaller."""
    import torch
    print('case sums beyond 32 bits', dim, store, count, flush=True)
    world = World([900, 700], 1, dim, 16, store, seed=37)
    if store == 'fp8':
        world.pages.v.view(torch.uint8).fill_(0x7e)             # 448 2^119
        world.pages.v_scale.fill_(246)
    else:
        world.pages.v.fill_(2.9e38)
    world.pages.v.view(torch.uint8 if store == 'fp8' else torch.int16)[..., dim // 2:] |= 0x80 if store == "fp8" else -32768
    q, start = first_value([count] * 2, 4, dim, 'bf16')
    q.zero_()
    out = episodes.attend(world.pages, q.cuda(), torch.from_numpy(np.array([0, count, 2 * count], np.int32)).cuda(),
                          max_count=count).float().cpu()
    assert bool((out[..., :dim // 2] > 2.8e38).all()) and bool((out[..., dim // 2:] < -2.8e38).all())
