"""Episode memory on the GPU against its definitions in 64 bits (tests/episode_reference.py).

Tolerances of attention, from the arithmetic (u: the type's unit roundoff, 2^-8 for bfloat16, 2^-11 for
float16): the result is rounded once (u |out|); the weights may be rounded to the type before they
multiply the values (u sum p|v|); everything else is in 32 bits, where scores of size 30 summed over up to
256 products and powers of two of them are within 2^-12 of their weight.  Element by element
|error| <= u |out| + (u + 2^-12) sum p|v|; and over all elements, where both roundings are spread evenly
(u / sqrt 3 each at most), the error's norm is within (sqrt(2/3) u + 2^-12) of sum p|v|'s.
Quantised values are powers of two times codes: they are compared for equality.
"""
import ctypes as ct
import math

import numpy as np
import pytest

from episode_reference import attention, quantised
from libero_hip import episodes

UNIT = {'bf16': 2.0 ** -8, 'f16': 2.0 ** -11}
pytestmark = pytest.mark.gpu


def dtype_of(name):
    import torch
    return {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32, 'fp8': torch.float8_e4m3fn}[name]


class World:
    """Pages filled with NaN wherever no token is, scattered over the pool; host copies of what is in them."""

    def __init__(self, lengths, kv, dim, page, store, seed=0, width=None, spare=3, kscale=1.0):
        import torch
        rng = np.random.default_rng(seed)
        self.lengths = np.asarray(lengths, np.int64)
        n = len(self.lengths)
        held = -(-self.lengths // page)
        width = int(max(1, held.max())) if width is None else width
        npage = int(held.sum()) + spare
        ids = rng.permutation(npage)
        self.table = np.full((n, width), -1, np.int32)
        at = 0
        for w in range(n):
            self.table[w, :held[w]] = ids[at:at + held[w]]
            at += held[w]
        self.k, self.v, values = [], [], {}
        for name in ('k', 'v'):
            if store == 'fp8':
                pool = np.full((npage, kv, page, dim), 0x7f, np.uint8)
                scales = np.full((npage, kv, page, dim // 32), 255, np.uint8)
            else:
                pool = np.full((npage, kv, page, dim), np.nan)
            for w in range(n):
                x = rng.standard_normal((int(self.lengths[w]), kv, dim)) * (kscale if name == 'k' else 1.0)
                x *= np.exp(0.5 * rng.standard_normal((kv, 1)))
                if store == 'fp8':
                    x, s = quantised(x)
                    per = 2.0 ** (s.astype(float) - 127).repeat(32, -1)
                    codes = torch.from_numpy(x / per).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
                else:
                    x = torch.from_numpy(x).to(dtype_of(store)).double().numpy()
                getattr(self, name).append(x)
                for t in range(len(x)):
                    where = (self.table[w, t // page], slice(None), t % page)
                    if store == 'fp8':
                        pool[where], scales[where] = codes[t], s[t]
                    else:
                        pool[where] = x[t]
            if store == 'fp8':
                values[name] = torch.from_numpy(pool).cuda().view(torch.float8_e4m3fn)
                values[name + '_scale'] = torch.from_numpy(scales).cuda()
            else:
                values[name] = torch.from_numpy(pool).cuda().to(dtype_of(store))
        self.pages = episodes.Pages(values['k'], values['v'], torch.from_numpy(self.table).cuda(),
                                    torch.from_numpy(self.lengths.astype(np.int32)).cuda(),
                                    values.get('k_scale'), values.get('v_scale'))


def queries(counts, heads, dim, kind, seed=1):
    import torch
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((int(np.sum(counts)), heads, dim))).to(dtype_of(kind))
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return x, start


def expected(world, q, start, causal=True, window=0, scale=None):
    q = q.double().numpy()
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    got = [attention(q[start[w]:start[w + 1]], world.k[w], world.v[w],
                     int(world.lengths[w] - (start[w + 1] - start[w])), causal, window, scale)
           for w in range(len(world.lengths))]
    return [np.concatenate(x) for x in zip(*got)]


def compare(out, lse, want, kind):
    ref, ref_lse, size = want
    out = out.double().cpu().numpy().reshape(ref.shape)
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(ref), np.isnan(out)), 'NaN in other places'
    assert np.array_equal(ref[~fine & ~np.isnan(ref)], out[~fine & ~np.isnan(ref)])
    u = UNIT[kind]
    error = np.abs(out[fine] - ref[fine])
    bound = (u * np.abs(ref) + (u + 2.0 ** -12) * size)[fine] + 2.0 ** -24
    assert np.all(error <= bound), (error / bound).max()
    assert np.linalg.norm(error) <= (math.sqrt(2 / 3) * u + 2.0 ** -12) * np.linalg.norm(size[fine]) + 1e-30
    if lse is not None:
        lse = lse.double().cpu().numpy().reshape(ref_lse.shape)
        assert np.array_equal(np.isinf(ref_lse), np.isinf(lse))
        real = np.isfinite(ref_lse)
        np.testing.assert_allclose(lse[real], ref_lse[real], rtol=2.0 ** -18, atol=2.0 ** -12)


def check(world, counts, heads, kind, causal=True, window=0, scale=None, uniform=False, most=None, seed=1):
    import torch
    dim = world.pages.struct.head_dim
    q, start = queries(counts, heads, dim, kind, seed)
    lse = torch.full(q.shape[:-1], 7.0, device='cuda')
    if uniform:
        shape = (len(counts), counts[0])
        out = episodes.attend(world.pages, q.cuda().reshape(shape + q.shape[1:]), causal=causal, window=window,
                              scale=scale, lse=lse.view(shape + (heads,)))
    else:
        out = episodes.attend(world.pages, q.cuda(), torch.from_numpy(start).cuda(), causal=causal, window=window,
                              scale=scale, lse=lse, max_count=most)
    compare(out, lse, expected(world, q, start, causal, window, scale), kind)


# ------------------------------------------------------------------------------ attention
LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize('kind,store', [('bf16', 'bf16'), ('f16', 'f16'), ('bf16', 'fp8'), ('f16', 'fp8')])
@pytest.mark.parametrize('dim', [32, 64, 96, 128, 256])
def test_single_tokens(gpu_available, dim, kind, store):
    """One new token of worlds of every length around the sizes of pages and tiles, three query heads to a key head."""
    print('case single', dim, kind, store, flush=True)
    world = World(LENGTHS, 2, dim, 32, store, seed=dim)
    check(world, [1] * len(LENGTHS), 6, kind, uniform=True)


@pytest.mark.parametrize('group', [1, 5, 16, 17, 40])
def test_groups(gpu_available, group):
    """Query heads per key head below, at and above one tile's rows."""
    print('case group', group, flush=True)
    world = World([5, 64, 130], 3, 64, 16, 'bf16', seed=group)
    check(world, [1, 1, 1], 3 * group, 'bf16', uniform=True)
    check(world, [2, 3, 7], 3 * group, 'bf16')


@pytest.mark.parametrize('kind,store', [('bf16', 'bf16'), ('f16', 'fp8')])
@pytest.mark.parametrize('dim', [32, 64, 96, 128, 256])
@pytest.mark.parametrize('causal,window', [(True, 0), (False, 0), (True, 7), (False, 40), (True, 100)])
def test_chunks(gpu_available, dim, kind, store, causal, window):
    """Ragged chunks: none, one, whole prompts, more rows than one tile; with and without window."""
    print('case chunk', dim, kind, store, causal, window, flush=True)
    lengths = [0, 1, 9, 33, 64, 150, 200, 77, 40]
    counts = [0, 1, 9, 5, 0, 150, 37, 1, 33]
    world = World(lengths, 2, dim, 16, store, seed=3 * dim + window)
    check(world, counts, 4, kind, causal, window)
    check(world, counts, 4, kind, causal, window, most=150)


@pytest.mark.parametrize('count', [2, 3, 16, 31, 64, 65, 129, 257])
def test_uniform_chunks(gpu_available, count):
    print('case uniform', count, flush=True)
    world = World([count, count + 1, count + 130], 1, 64, 64, 'bf16', seed=count)
    check(world, [count] * 3, 3, 'bf16', uniform=True)
    check(world, [count] * 3, 3, 'bf16', causal=False, uniform=True)
    check(world, [count] * 3, 3, 'bf16', window=65, uniform=True)


@pytest.mark.parametrize('kind,store', [('f16', 'f16'), ('bf16', 'fp8')])
@pytest.mark.parametrize('page,count', [(16, 17), (64, 33), (32, 70), (128, 140)])
def test_chunks_of_wide_heads(gpu_available, page, count, kind, store):
    """Heads of 256 values: pages on both sides of a step's keys, one part and several."""
    print('case wide heads', page, count, kind, store, flush=True)
    for width in (None, 2048 // page):
        world = World([count, 700, count + 31], 2, 256, page, store, seed=20 + count, width=width)
        check(world, [count] * 3, 4, kind, uniform=True)
        check(world, [count, 1, count - 1], 4, kind, causal=False, window=100)


@pytest.mark.parametrize('store', ['bf16', 'fp8'])
@pytest.mark.parametrize('page', [16, 64, 1024])
def test_long_keys_are_split(gpu_available, page, store):
    """Few rows over many keys: the work is split along the keys and joined; short worlds beside long ones."""
    print('case split', page, store, flush=True)
    world = World([5000, 3, 2049, 0], 1, 64, page, store, seed=page)
    check(world, [1, 1, 1, 1], 2, 'bf16', uniform=True)
    check(world, [5, 3, 20, 0], 2, 'bf16')
    check(world, [5, 3, 20, 0], 2, 'bf16', window=1500)
    check(world, [70, 1, 33, 0], 2, 'bf16', causal=False)


@pytest.mark.parametrize('dim,kind,store', [(32, 'f16', 'fp8'), (64, 'bf16', 'bf16'), (96, 'f16', 'f16'), (128, 'bf16', 'fp8'),
                                            (256, 'bf16', 'bf16')])
def test_parts_of_many_rows(gpu_available, dim, kind, store):
    """Thousands of rows whose keys are split, most parts without any: worlds far shorter than their table."""
    print('case parts', dim, kind, store, flush=True)
    world = World([150, 700, 0, 137], 2, dim, 16, store, seed=23, width=256)
    check(world, [130] * 4, 16, kind, uniform=True)
    check(world, [130, 261, 0, 137], 16, kind, window=300)
    check(world, [130, 129, 0, 5], 16, kind, causal=False)


@pytest.mark.parametrize('dim,kind,store', [(32, 'f16', 'f16'), (64, 'bf16', 'bf16'), (64, 'f16', 'fp8'), (96, 'bf16', 'fp8'),
                                            (128, 'bf16', 'bf16'), (256, 'bf16', 'fp8')])
def test_many_short_histories(gpu_available, dim, kind, store):
    """Thousands of tiles with few keys: none, one, some on both sides of a step's 32; one block of rows and two."""
    print('case short histories', dim, kind, store, flush=True)
    lengths = np.arange(264) % 67
    world = World(lengths, 8, dim, 16, store, seed=21)
    check(world, [1] * 264, 16, kind, uniform=True)
    check(world, (np.arange(264) % 4).tolist(), 24, kind, most=3)
    check(world, [8 if store == 'fp8' else 4] * 264, 24, kind, causal=False, window=35, uniform=True)


@pytest.mark.parametrize('longest', [1, 40, 300, 10 ** 9])
def test_longest_is_only_a_guide(gpu_available, longest):
    """Worlds longer than it says, in a table of any length, are seen whole."""
    import torch
    print('case longest', longest, flush=True)
    for lengths, kv in (([300, 0, 17], 1), (np.r_[np.arange(255) % 20, [130, 300, 64, 33, 1]], 8)):
        world = World(lengths, kv, 64, 16, 'bf16', seed=22, width=256)
        counts = [1] * len(lengths)
        q, start = queries(counts, 2 * kv, 64, 'bf16')
        lse = torch.full((len(counts), 1, 2 * kv), 7.0, device='cuda')
        out = episodes.attend(world.pages, q.cuda().unsqueeze(1), lse=lse, longest=longest)
        compare(out, lse, expected(world, q, start), 'bf16')


def test_rows_without_keys(gpu_available):
    """Empty worlds and chunks longer than their worlds: zeros and -inf, whatever the pages hold."""
    import torch
    print('case empty', flush=True)
    world = World([0, 0, 3, 40], 1, 64, 16, 'bf16', seed=5)
    for causal in (True, False):
        check(world, [1, 1, 1, 1], 2, 'bf16', causal=causal, uniform=True)
        check(world, [2, 0, 9, 70], 2, 'bf16', causal=causal)          # positions -6.. and -30..
        check(world, [2, 0, 9, 70], 2, 'bf16', causal=causal, window=2 ** 31 - 1)
        check(world, [2, 0, 9, 70], 2, 'bf16', causal=causal, window=20)
    q = torch.ones((0, 2, 64), dtype=torch.bfloat16, device='cuda')
    assert episodes.attend(world.pages, q, torch.zeros(5, dtype=torch.int32, device='cuda')).shape == (0, 2, 64)


def test_pages_that_are_not_there(gpu_available):
    """A table entry that names no page hides its tokens; lengths beyond the table end with it."""
    import torch
    print('case holes', flush=True)
    for hole in (-1, 10 ** 6, -2 ** 31):
        world = World([100, 64], 1, 64, 16, 'bf16', seed=6)
        world.pages.table[0, 2] = hole
        q, start = queries([3, 2], 2, 64, 'bf16')
        out = episodes.attend(world.pages, q.cuda(), torch.from_numpy(start).cuda())
        keep = np.r_[0:32, 48:100]
        qd = q.double().numpy()
        ref = [attention(qd[i:i + 1], world.k[0][:98 + i][keep[keep < 98 + i]], world.v[0][:98 + i][keep[keep < 98 + i]],
                         98 + i - 16, True, 0, 0.125) for i in range(3)]
        ref.append(attention(qd[3:5], world.k[1], world.v[1], 62, True, 0, 0.125))
        compare(out, None, [np.concatenate(x) for x in zip(*ref)], 'bf16')
    world = World([64, 30], 1, 64, 16, 'bf16', seed=7)
    world.pages.length[0] = 10 ** 9
    q, start = queries([1, 1], 2, 64, 'bf16')
    out = episodes.attend(world.pages, q.cuda().view(2, 1, 2, 64))
    compare(out, None, expected(world, q, start), 'bf16')


@pytest.mark.parametrize('count', [6, 40, 300])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_hidden_values_stay_hidden(gpu_available, count, bad):
    """An infinity or NaN in a key or value reaches the queries that see it, and no others: later tokens of the
    same chunk, tokens that have left the window."""
    import torch
    print('case hidden', count, bad, flush=True)
    for causal, window in ((True, 0), (True, 9), (False, 11)):
        world = World([count, count + 21], 1, 64, 16, 'bf16', seed=8)
        for w, token, name, at in ((0, count - 2, 'v', 5), (1, 12, 'v', 63), (1, count // 2, 'v', 17)):
            getattr(world, name)[w][token, 0, at] = bad
            getattr(world.pages, name)[world.table[w, token // 16], 0, token % 16, at] = bad
        check(world, [count, count], 2, 'bf16', causal, window)
    world = World([count, count + 21], 1, 64, 16, 'bf16', seed=9)
    world.k[0][count - 2, 0, 5] = bad
    world.pages.k[world.table[0, (count - 2) // 16], 0, (count - 2) % 16, 5] = bad
    q, start = queries([count, count], 2, 64, 'bf16')
    out = episodes.attend(world.pages, q.cuda(), torch.from_numpy(start).cuda()).double().cpu().numpy()
    ref, _, size = expected(world, q, start)
    seen = np.zeros(2 * count, bool)
    seen[count - 2:count] = True
    assert np.array_equal(np.isfinite(out[~seen]), np.ones_like(out[~seen], bool))
    compare(torch.from_numpy(out[~seen]), None, (ref[~seen], None, size[~seen]), 'bf16')


@pytest.mark.parametrize('count', [1, 40])
@pytest.mark.parametrize('page', [16, 64])
def test_quantised_values_beyond_float16(gpu_available, page, count):
    """8-bit pages hold magnitudes that float16 does not: as float16 values they are infinities of their sign, and
    so are the results of the queries that see them."""
    print('case beyond float16', page, count, flush=True)
    world = World([50, 300, 301], 1, 64, page, 'fp8', seed=18)
    for w, token in ((0, 5), (1, 101), (2, 299)):
        world.v[w][token, 0, :32] *= 2.0 ** 17
        world.pages.v_scale[world.table[w, token // page], 0, token % page, 0] += 17
    with np.errstate(over='ignore'):
        world.v = [x.astype(np.float16).astype(np.float64) for x in world.v]
    assert sum(np.isinf(x).sum() for x in world.v) > 30
    check(world, [count] * 3, 2, 'f16')


def test_scores_of_any_size(gpu_available):
    """Large scores of one sign, scale 0 and negative scale: the maximum is taken off first."""
    print('case scores', flush=True)
    world = World([40, 129, 700], 1, 64, 16, 'f16', seed=10, kscale=40.0)
    # a score's error is 2^-24 of the products' sum of sizes, some 64 * 40: well below the spread of the weights
    for scale in (0.0, 0.125, -0.125):
        check(world, [1, 1, 1], 3, 'f16', scale=scale, uniform=True)
        check(world, [20, 70, 129], 1, 'f16', scale=scale)


@pytest.mark.parametrize('offset', [0, 1, 4])
def test_strides(gpu_available, offset):
    """Queries as a part of a fused projection, at any alignment; results into a part of a wider tensor."""
    import torch
    print('case strides', offset, flush=True)
    for counts in ([1, 1, 1], [30, 40, 90]):
        world = World([33, 64, 100], 2, 64, 16, 'bf16', seed=11)
        q, start = queries(counts, 4, 64, 'bf16')
        wide = torch.full((q.shape[0], 1000), float('nan'), dtype=torch.bfloat16, device='cuda')
        inside = wide.as_strided(q.shape, (1000, 80, 1), offset)
        inside.copy_(q)
        target = torch.zeros((q.shape[0], 3, 4, 72), dtype=torch.bfloat16, device='cuda')
        out = target[:, 1, :, offset:offset + 64]
        got = episodes.attend(world.pages, inside, torch.from_numpy(start).cuda(), out=out)
        assert got is out
        compare(got, None, expected(world, q, start), 'bf16')
        target[:, 1, :, offset:offset + 64] = 0
        assert not target.any()


def test_other_stream_and_same_bits(gpu_available):
    """On a stream of its own, with other work around it; two calls give the same bits, split or not."""
    import torch
    print('case stream', flush=True)
    world = World([3000, 2500, 77], 2, 128, 64, 'fp8', seed=12)
    side = torch.cuda.Stream()
    for counts in ([1, 1, 1], [40, 3, 77]):
        q, start = queries(counts, 8, 128, 'bf16')
        q, first = q.cuda(), torch.from_numpy(start).cuda()
        side.wait_stream(torch.cuda.current_stream())
        a = episodes.attend(world.pages, q, first, stream=side)
        with torch.cuda.stream(side):
            b = episodes.attend(world.pages, q, first)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, b)
        compare(a, None, expected(world, q.cpu(), start), 'bf16')


@pytest.mark.parametrize('width,count', [(64, 1), (256, 1), (64, 30), (512, 30)])
def test_captured_calls_follow_the_lengths(gpu_available, width, count):
    """write and attend in a HIP graph, with the keys split (long tables) and not: replays with other lengths and
    rows give what eager calls give."""
    import torch
    print('case graph', width, count, flush=True)
    world = World([600, 80, 1000], 2, 64, 16, 'bf16', seed=13, width=width)
    p = world.pages
    final = p.length.clone()
    q = torch.randn((3, count, 4, 64), device='cuda').bfloat16()
    k, v = (torch.randn((3, count, 2, 64), device='cuda').bfloat16() for _ in range(2))
    out, lse = torch.empty_like(q), torch.empty((3, count, 4), device='cuda')
    episodes.write(p, k, v)
    episodes.attend(p, q, out=out, lse=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        episodes.write(p, k, v)
        episodes.attend(p, q, out=out, lse=lse)
    for step in range(4):
        p.length.copy_(final - 7 * step)
        k.normal_()
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse = out.clone(), lse.clone()
        x, y = episodes.read(p, count=count)
        assert torch.equal(x, k) and torch.equal(y, v)
        assert torch.equal(got, episodes.attend(p, q)) and bool(torch.isfinite(got_lse).all())


# ------------------------------------------------------------------------------ writing and reading
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('store', ['bf16', 'f16', 'fp8'])
@pytest.mark.parametrize('dim', [32, 96, 256])
def test_write_and_read(gpu_available, dim, store, kind):
    """Chunks of no, one and many tokens across pages: every slot of the chunk holds the rounded values, every
    other slot what it held, and reading returns the same."""
    import torch
    print('case write', dim, store, kind, flush=True)
    lengths, counts = [0, 1, 40, 17, 100, 33], [0, 1, 23, 17, 1, 2]
    rng = np.random.default_rng(dim)
    world = World(lengths, 3, dim, 16, store, seed=14)
    before = {n: getattr(world.pages, n).clone().view(torch.uint8) for n in ('k', 'v')}
    tokens = sum(counts)
    x = rng.standard_normal((2, tokens, 3, dim)) * np.exp(3 * rng.standard_normal((2, tokens, 3, 1)))
    x[:, 3, 1] = 0
    x[0, 4, 2, :32] = 448.0 * 2.0 ** rng.integers(-12, 1, 32)        # at the codes' limit, and just beyond
    x[0, 5, 2, :32] = 449.0 * 2.0 ** rng.integers(-12, 1, 32)
    x[1, 6, 0, :32] = (np.arange(32) - 16) / 16.0 * 3.4375 + 2.0 ** -9   # near ties
    x = torch.from_numpy(x).to(dtype_of(kind))
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
    episodes.write(world.pages, x[0].cuda(), x[1].cuda(), start)
    if store == 'fp8':
        want = [quantised(y.double().numpy())[0] for y in x]
    else:
        want = [y.to(dtype_of(store)).double().numpy() for y in x]
    for out in ('f32', 'bf16', 'f16'):
        got = episodes.read(world.pages, start, tokens=tokens, dtype=dtype_of(out))
        for g, y in zip(got, want):
            ref = torch.from_numpy(y).to(dtype_of('f32')).to(dtype_of(out))
            assert torch.equal(g.cpu(), ref)
    # untouched: everything but the chunk
    mine = np.zeros(before['k'].shape[:1] + before['k'].shape[2:3], bool)
    for w, (length, count) in enumerate(zip(lengths, counts)):
        for t in range(length - count, length):
            mine[world.table[w, t // 16], t % 16] = True
    keep = torch.from_numpy(~mine).cuda()
    for n in ('k', 'v'):
        after = getattr(world.pages, n).view(torch.uint8)
        assert torch.equal(after.transpose(1, 2)[keep], before[n].transpose(1, 2)[keep])


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_quantised_extremes(gpu_available, kind):
    """Zeros, the smallest and largest numbers, infinities and NaN in a block: the others are as always."""
    import torch
    print('case extremes', kind, flush=True)
    world = World([8], 1, 64, 16, 'fp8', seed=15)
    x = np.random.default_rng(0).standard_normal((8, 1, 64))
    x[0, 0, :32] = 0
    x[1, 0, :32] *= 2.0 ** -126
    x[2, 0, :32] *= 2.0 ** 125
    x[3, 0, 7], x[4, 0, 8], x[5, 0, 40] = np.inf, np.nan, -np.inf
    x[6, 0, :32] = 2.0 ** -149 if kind == 'f32' else 2.0 ** -133
    x[7, 0, :32] *= 2.0 ** -118
    x = torch.from_numpy(x).to(dtype_of(kind))
    episodes.write(world.pages, x.cuda().view(1, 8, 1, 64), x.cuda().view(1, 8, 1, 64))
    ref = torch.from_numpy(quantised(x.double().numpy())[0]).float()
    for got in episodes.read(world.pages, count=8, dtype=torch.float32):
        got = got.cpu().view(8, 1, 64)
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(ref))


def test_write_skips_what_has_no_place(gpu_available):
    import torch
    print('case no place', flush=True)
    world = World([5, 20, 0], 1, 32, 16, 'bf16', seed=16)
    world.pages.table[1, 1] = -1
    x = torch.randn((3, 8, 1, 32), device='cuda').bfloat16()
    episodes.write(world.pages, x, x)                 # world 0 has places for five, world 1 for its first four
    got, _ = episodes.read(world.pages, count=8)
    ref = torch.zeros_like(x)
    ref[0, 3:], ref[1, :4] = x[0, 3:], x[1, :4]
    assert torch.equal(got, ref)


@pytest.mark.parametrize('offset', [0, 3])
def test_write_strides(gpu_available, offset):
    """Keys and values as parts of a fused projection, at any alignment, 8-bit and 16-bit."""
    import torch
    print('case write strides', offset, flush=True)
    for store in ('bf16', 'fp8'):
        world = World([9, 30], 2, 64, 16, store, seed=17)
        fused = torch.randn((2, 9, 500), device='cuda').bfloat16()
        k = fused.as_strided((2, 9, 2, 64), (4500, 500, 70, 1), offset)
        v = fused.as_strided((2, 9, 2, 64), (4500, 500, 64, 1), 200 + offset)
        episodes.write(world.pages, k, v)
        got = episodes.read(world.pages, count=9)
        for g, x in zip(got, (k, v)):
            ref = x.cpu() if store == 'bf16' else torch.from_numpy(quantised(x.cpu().double().numpy())[0]).bfloat16()
            assert torch.equal(g.cpu(), ref)


def test_offsets_beyond_32_bits(gpu_available):
    """Pages whose elements lie past 2^31 and 2^32: written, read and attended to."""
    import torch
    print('case far pages', flush=True)
    npage, kv, page, dim = 70000, 4, 128, 128                  # 4.6e9 elements
    k, v = (torch.zeros((npage, kv, page, dim), dtype=torch.float8_e4m3fn, device='cuda') for _ in range(2))
    ks, vs = (torch.zeros((npage, kv, page, 4), dtype=torch.uint8, device='cuda') for _ in range(2))
    ids = [69999, 3, 40000, 33333]
    table = torch.tensor([ids[:2], ids[2:]], dtype=torch.int32, device='cuda')
    length = torch.tensor([200, 150], dtype=torch.int32, device='cuda')
    pages = episodes.Pages(k, v, table, length, ks, vs)
    x = torch.randn((2, 150, kv, dim), device='cuda').bfloat16()
    y = torch.randn((2, 150, kv, dim), device='cuda').bfloat16()
    episodes.write(pages, x, y)
    got = episodes.read(pages, count=150)
    for g, ref in zip(got, (x, y)):
        assert torch.equal(g.cpu(), torch.from_numpy(quantised(ref.cpu().double().numpy())[0]).bfloat16())
    q, start = queries([1, 1], 8, dim, 'bf16')
    out = episodes.attend(pages, q.cuda().view(2, 1, 8, dim))
    pad = np.zeros((50, kv, dim))
    hk, hv = (g.double().cpu().numpy() for g in got)
    ref = [attention(q[:1].double().numpy(), np.concatenate([pad, hk[0]]), np.concatenate([pad, hv[0]]), 199, True, 0,
                     dim ** -0.5),
           attention(q[1:].double().numpy(), hk[1], hv[1], 149, True, 0, dim ** -0.5)]
    compare(out, None, [np.concatenate(z) for z in zip(*ref)], 'bf16')


# ------------------------------------------------------------------------------ refusals
def test_refusals(gpu_available):
    import torch
    print('case refusals', flush=True)
    world = World([5, 20], 2, 64, 16, 'bf16', seed=18)
    p = world.pages
    q = torch.zeros((2, 1, 4, 64), dtype=torch.bfloat16, device='cuda')
    kv = q[:, :, :2]
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device='cuda')
    bad = [
        lambda: episodes.attend(p, q.float()), lambda: episodes.attend(p, q.half()), lambda: episodes.attend(p, q[..., :32]),
        lambda: episodes.attend(p, q[:, :, :3]), lambda: episodes.attend(p, q[:1]), lambda: episodes.attend(p, q.cpu()),
        lambda: episodes.attend(p, q[:, 0]), lambda: episodes.attend(p, q, start), lambda: episodes.attend(p, q[:, 0], start[:2]),
        lambda: episodes.attend(p, q[:, 0], start.long()), lambda: episodes.attend(p, q, window=-1),
        lambda: episodes.attend(p, q, scale=float('nan')), lambda: episodes.attend(p, q, out=q[:, :, :2]),
        lambda: episodes.attend(p, q, lse=torch.zeros((2, 1, 3), device='cuda')), lambda: episodes.attend(p, q, max_count=-1),
        lambda: episodes.attend(p, q, longest=-1),
        lambda: episodes.attend(p, torch.zeros((2, 1, 64, 4), dtype=torch.bfloat16, device='cuda').transpose(2, 3)),
        lambda: episodes.write(p, q, q), lambda: episodes.write(p, kv, kv.float()), lambda: episodes.write(p, kv, kv[:, :0]),
        lambda: episodes.write(p, kv.double(), kv.double()), lambda: episodes.read(p), lambda: episodes.read(p, start),
        lambda: episodes.read(p, count=1, dtype=torch.int32), lambda: episodes.read(p, start, count=1),
        lambda: episodes.Pages(p.k, p.v[:1], p.table, p.length), lambda: episodes.Pages(p.k.float(), p.v.float(), p.table, p.length),
        lambda: episodes.Pages(p.k[:, :, :12].contiguous(), p.v[:, :, :12].contiguous(), p.table, p.length),
        lambda: episodes.Pages(p.k[..., :48].contiguous(), p.v[..., :48].contiguous(), p.table, p.length),
        lambda: episodes.Pages(p.k.transpose(0, 1), p.v.transpose(0, 1), p.table, p.length),
        lambda: episodes.Pages(p.k, p.v, p.table.long(), p.length), lambda: episodes.Pages(p.k, p.v, p.table, p.length[:1]),
        lambda: episodes.Pages(p.k, p.v, p.table.cpu(), p.length), lambda: episodes.Pages(p.k, p.v, p.table, p.length, p.k, p.v),
        lambda: episodes.Pages(p.k.to(torch.float8_e4m3fn), p.v.to(torch.float8_e4m3fn), p.table, p.length),
        lambda: episodes.Pages(p.k.cpu(), p.v.cpu(), p.table.cpu(), p.length.cpu()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('not refused:', i)


def test_gradients_are_refused(gpu_available):
    """There is no backward pass: a result that silently had no gradient would train nothing."""
    import torch
    print('case gradients', flush=True)
    world = World([5, 20], 2, 64, 16, 'bf16', seed=19)
    q = torch.randn((2, 1, 4, 64), device='cuda').bfloat16().requires_grad_()
    kv = q[:, :, :2]
    for call in (lambda: episodes.attend(world.pages, q), lambda: episodes.write(world.pages, kv, kv)):
        with pytest.raises(ValueError, match='backward'):
            call()
    with torch.no_grad():
        out = episodes.attend(world.pages, q)
    assert not out.requires_grad and torch.equal(out, episodes.attend(world.pages, q.detach()))
