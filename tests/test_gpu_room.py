"""Room for tokens on the GPU against the books that a list of pages gives (tests/recall_reference.py): whole numbers, compared
for equality."""
import numpy as np
import pytest

from recall_reference import Books
from libero_hip import episodes, room

pytestmark = pytest.mark.gpu


def there(x):
    import torch
    return torch.from_numpy(np.array(x, order='C')).cuda()


class Rooms:
    """An empty room of the GPU and its books."""

    def __init__(self, nworld, width, npage, page, tokens=None, seed=0):
        free = np.random.default_rng(seed).permutation(npage).astype(np.int32)
        table, length = np.full((nworld, width), -1, np.int32), np.zeros(nworld, np.int32)
        self.room = room.Room(there(table), there(length), npage, page, there(free), there(np.array([npage, 0], np.int32)), tokens=tokens)
        self.books = Books(table, length, free, width * page if tokens is None else tokens, page)

    def change(self, count, over=None, rows=2 ** 31 - 1, uniform=False):
        n = len(self.books.length)
        want = self.books.change(np.broadcast_to(np.asarray(count, np.int64), n), over, rows)
        given = int(count) if uniform else there(np.broadcast_to(np.asarray(count, np.int32), n))
        start = room.make_room(self.room, given, None if over is None else there(over), rows=rows)
        np.testing.assert_array_equal(start.cpu().numpy(), want)
        self.same()
        return start

    def same(self):
        np.testing.assert_array_equal(self.room.table.cpu().numpy(), self.books.table)
        np.testing.assert_array_equal(self.room.length.cpu().numpy(), self.books.length)
        left, why = self.room.state.cpu().numpy()
        assert left == len(self.books.free) and why == self.books.why
        np.testing.assert_array_equal(self.room.free.cpu().numpy()[:left], self.books.free)


@pytest.mark.parametrize('nworld,page,width', [(1, 16, 5), (5, 16, 5), (17, 32, 3), (67, 16, 9), (300, 64, 4), (4096, 64, 3),
                                               (9000, 16, 2)])
def test_random_changes(gpu_available, nworld, page, width):
    """Worlds grow, shrink, end and are refused, in any mixture."""
    print('case room', nworld, page, width, flush=True)
    rng = np.random.default_rng(nworld)
    r = Rooms(nworld, width, max(3, nworld * width * 2 // 3), page, tokens=width * page - 3, seed=nworld)
    refused = 0
    for step in range(25 if nworld < 4000 else 10):
        before = r.books.why
        r.books.why = 0
        r.room.state[1] = 0
        over = rng.random(nworld) < rng.choice([0, 0.2, 1.0]) if rng.random() < 0.6 else None
        base = np.where(over, 0, r.books.length) if over is not None else r.books.length
        limit = width * page - 3 - base
        if rng.random() < 0.2:                       # some world may not fit
            limit = limit + (rng.random(nworld) < 0.02)
        count = (rng.random(nworld) * (limit + 1) * rng.choice([0.1, 0.5, 1.0])).astype(int)
        if rng.random() < 0.4:
            count = np.where(rng.random(nworld) < 0.5, -(rng.random(nworld) * (base + 1)).astype(int), count)
        rows = int(np.maximum(count, 0).sum()) - (rng.random() < 0.1)
        r.change(count, over, max(rows, 0))
        refused += r.books.why != 0
    assert refused < 25


def test_uniform_counts_and_reasons(gpu_available):
    print('case room reasons', flush=True)
    r = Rooms(6, 4, 9, 16, tokens=50)
    r.change(3, uniform=True)
    r.change(14, uniform=True)                       # a second page for three worlds only: refused
    assert r.books.why == 2
    r.change(13, uniform=True)
    r.change(-16, uniform=True)
    assert not r.books.length.any() and len(r.books.free) == 9
    r.change(-1, uniform=True)
    assert r.books.why == 3
    r.change([0, 51, 0, 0, 0, 0])
    r.change([0, 50, 0, 0, 0, 0], rows=49)
    assert r.books.why == 7
    r.change([0, 50, 0, 0, 0, 0], rows=50)
    r.change([0, 1, 0, 0, 0, 0])
    r.change([60, 0, 0, 0, 0, 0], np.array([False, True, False, False, False, False]))    # refused, but world 1 is empty
    assert not r.books.length.any() and len(r.books.free) == 9
    r.change(0, uniform=True)
    r.change(2 ** 31 - 1, uniform=True, rows=2 ** 31 - 1)
    r.change([-2 ** 31, 0, 0, 0, 0, 0])


def test_looking_ahead_leaves_no_trace(gpu_available):
    import torch
    print('case room ahead', flush=True)
    r = Rooms(100, 8, 500, 16)
    rng = np.random.default_rng(1)
    r.change(rng.integers(0, 60, 100))
    kept = [getattr(r.room, n).clone() for n in ('table', 'length', 'free', 'state')]
    count = rng.integers(0, 60, 100)
    r.change(count)
    r.change(-count)
    for n, x in zip(('table', 'length', 'free', 'state'), kept):
        assert torch.equal(getattr(r.room, n), x)


def test_lengths_and_states_out_of_range(gpu_available):
    """Tables that say nonsense are answered within their bounds: nothing outside of table and stack is touched."""
    import torch
    print('case room nonsense', flush=True)
    guard = 64
    pool = torch.full((3 * guard + 40 + 6,), 12345, dtype=torch.int32, device='cuda')
    table, free = pool[guard:guard + 40].view(4, 10), pool[2 * guard + 40:2 * guard + 46]
    table.fill_(-7)
    free.fill_(99)
    length = torch.tensor([2 ** 31 - 1, -5, 160, 3], dtype=torch.int32, device='cuda')
    for left in (0, 6, 2 ** 31 - 1, -2 ** 31):
        state = torch.tensor([left, 0], dtype=torch.int32, device='cuda')
        x = room.Room(table, length.clone(), 6, 16, free, state)
        for count, over in ((0, None), (1, None), (-3, None), (5, torch.ones(4, dtype=torch.bool, device='cuda'))):
            room.make_room(x, count, over)
        torch.cuda.synchronize()
        assert 0 <= int(state[0]) <= 6
    keep = torch.ones_like(pool, dtype=torch.bool)
    keep[guard:guard + 40] = False
    keep[2 * guard + 40:2 * guard + 46] = False
    assert bool((pool[keep] == 12345).all())


@pytest.mark.parametrize('nworld', [1, 7, 300])
def test_places(gpu_available, nworld):
    """World, position and slot of every row: ragged and even chunks, rows beyond the last world's, before the first token,
    without a page."""
    import torch
    print('case places', nworld, flush=True)
    rng = np.random.default_rng(nworld)
    page, width, npage = 16, 6, 6 * nworld
    table = rng.permutation(npage).reshape(nworld, width).astype(np.int32)
    table[rng.random((nworld, width)) < 0.1] = -1
    table[0, 0] = npage                              # names no page either
    length = rng.integers(0, 120, nworld).astype(np.int32)            # some beyond the table's reach
    x = room.Room(there(table), there(length), npage, page)

    def want(counts, tokens):
        out = np.full((3, tokens), -1)
        at = 0
        for w, c in enumerate(counts):
            for i in range(c):
                p = length[w] - c + i
                slot = -1
                if 0 <= p < width * page and 0 <= table[w, p // page] < npage:
                    slot = table[w, p // page] * page + p % page
                if at < tokens:
                    out[:, at] = w, max(p, -1), slot
                at += 1
        return out

    counts = rng.integers(0, 40, nworld)
    counts[-1] = 0
    start = there(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    for extra in (0, 5, -1):
        tokens = max(0, int(counts.sum()) + extra)
        got = room.places(x, start, tokens=tokens)
        assert all(g.dtype == torch.int32 for g in got)
        np.testing.assert_array_equal(torch.stack(got).cpu().numpy(), want(counts, tokens))
    for count in (0, 1, 33):
        got = room.places(x, count=count)
        assert got[0].shape == (nworld, count)
        np.testing.assert_array_equal(torch.stack(got).cpu().numpy().reshape(3, -1), want([count] * nworld, nworld * count))


@pytest.mark.parametrize('storage', ['bf16', 'fp8'])
def test_cache_on_the_device_equals_the_hosts(gpu_available, storage):
    """The same steps through EpisodeCache and DeviceEpisodeCache: the same attention, whatever pages the worlds have."""
    import torch
    print('case device cache', storage, flush=True)
    n = 9
    options = dict(kv_heads=2, head_dim=32, tokens=80, layers=2, storage=storage, page_tokens=16, block_tokens=16)
    host, device = episodes.EpisodeCache(n, **options), room.DeviceEpisodeCache(n, **options)
    rng = np.random.default_rng(0)
    for step in range(12):
        over = rng.random(n) < 0.2
        host.reset(np.flatnonzero(over))
        if step % 2:
            chunk, other = host.extend(3), device.extend(3, there(over))
            shape = (n, 3)
        else:
            counts = rng.integers(0, 6, n)
            chunk = host.extend(counts, range(n))
            other = device.extend(there(counts.astype(np.int32)), there(over), rows=int(counts.sum()), most=5)
            shape = chunk.shape
        q = torch.randn(shape + (4, 32), device='cuda').bfloat16()
        k, v = (torch.randn(shape + (2, 32), device='cuda').bfloat16() for _ in range(2))
        for layer in range(2):
            host.write(chunk, k, v, layer)
            device.write(other, k, v, layer)
            a, b = host.attend(chunk, q, layer), device.attend(other, q, layer)
            assert a.shape == b.shape
            torch.testing.assert_close(a, b, rtol=2.0 ** -7, atol=2.0 ** -7)      # two roundings of one value
            a, b = (c.recall(x, q, layer, top=1, near=2, first=1) for c, x in ((host, chunk), (device, other)))
            torch.testing.assert_close(a, b, rtol=2.0 ** -7, atol=2.0 ** -7)
        device.check()
        np.testing.assert_array_equal(host.lengths, device.lengths)
        assert host.free_pages == device.free_pages
        world, position, slot = device.places(other)
        assert world.shape == other.shape
        if step % 2:
            np.testing.assert_array_equal(position.cpu().numpy(), host.lengths[:, None] - 3 + np.arange(3))
    x, y = host.read(layer=1), device.read(layer=1)
    assert all(torch.equal(a, b) for a, b in zip(x[:2], y[:2])) and x[2].tolist() == y[2].tolist()
    device.reset()
    assert not device.lengths.any() and device.free_pages == device.pages


def test_refused_steps_do_nothing(gpu_available):
    """A step without room writes nothing, its attention computes nothing, and check() says so once."""
    import torch
    print('case refused step', flush=True)
    c = room.DeviceEpisodeCache(3, kv_heads=1, head_dim=32, tokens=20, storage='bf16', page_tokens=16, pages=5)
    k = torch.randn((3, 18, 1, 32), device='cuda').bfloat16()
    chunk = c.extend(16)
    c.write(chunk, k[:, :16], k[:, :16])
    chunk = c.extend(2)
    c.write(chunk, k[:, 16:], k[:, 16:])
    out = torch.full((3, 2, 2, 32), 7.0, dtype=torch.bfloat16, device='cuda')
    assert c.attend(chunk, torch.randn_like(out), out=out) is out and bool((out == 7).all())
    with pytest.raises(RuntimeError, match='free pages'):
        c.check()
    c.check()
    assert c.lengths.tolist() == [16, 16, 16]
    x, y, _ = c.read()
    assert torch.equal(x.view(3, 16, 1, 32), k[:, :16])
    c.take_back(3)
    c.extend(there(np.array([7, 0, 0], np.int32)), rows=7)
    c.check()
    assert c.lengths.tolist() == [20, 13, 13]
    c.extend(there(np.array([1, 0, 0], np.int32)), rows=1)
    with pytest.raises(RuntimeError, match='more tokens'):
        c.check()


def test_captured_steps(gpu_available):
    """A whole step in a HIP graph: worlds end and grow by tensors on the device, as in eager steps."""
    import torch
    from libero_hip.rotary import Rotary
    print('case captured step', flush=True)
    n = 7
    turning = Rotary.make(32)
    options = dict(kv_heads=1, head_dim=32, tokens=200, storage='bf16', page_tokens=16, block_tokens=16)
    caches = [room.DeviceEpisodeCache(n, **options) for _ in range(2)]
    q = torch.randn((n, 2, 4, 32), device='cuda').bfloat16()
    k, v = (torch.randn((n, 2, 1, 32), device='cuda').bfloat16() for _ in range(2))
    over = torch.zeros(n, dtype=torch.bool, device='cuda')

    def step(c):
        chunk = c.extend(2, over)
        x = c.enter(chunk, turning, q, k, v)
        return c.attend(chunk, x), c.recall(chunk, x, top=2, near=1, first=1), torch.stack(c.places(chunk))

    for c in caches:
        step(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    rng = np.random.default_rng(0)
    for i in range(60):
        over.copy_(there(rng.random(n) < 0.05))
        q.normal_()
        k.normal_()
        v.normal_()
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in got]
        want = step(caches[1])
        for a, b in zip(kept, want):
            assert torch.equal(a, b), i
        for name in ('table', 'length'):
            assert torch.equal(*(getattr(c, name) for c in caches))
        assert torch.equal(caches[0].room.state, caches[1].room.state)
    caches[0].check()
    assert caches[0].lengths.max() > 60


def test_other_stream(gpu_available):
    import torch
    print('case room stream', flush=True)
    r, other = (Rooms(40, 6, 200, 16) for _ in range(2))
    count = np.random.default_rng(0).integers(0, 50, 40).astype(np.int32)
    side = torch.cuda.Stream()
    given = there(count)
    side.wait_stream(torch.cuda.current_stream())
    start = room.make_room(r.room, given, stream=side)
    found = room.places(r.room, start, tokens=int(count.sum()), stream=side)
    torch.cuda.synchronize()
    first = room.make_room(other.room, given)
    assert torch.equal(start, first)
    for a, b in zip(found, room.places(other.room, first, tokens=int(count.sum()))):
        assert torch.equal(a, b)


def test_refusals(gpu_available):
    import torch
    print('case room refusals', flush=True)
    table, length = torch.zeros((3, 2), dtype=torch.int32, device='cuda'), torch.zeros(3, dtype=torch.int32, device='cuda')
    free, state = torch.zeros(6, dtype=torch.int32, device='cuda'), torch.zeros(2, dtype=torch.int32, device='cuda')
    x = room.Room(table, length, 6, 16, free, state)
    bad = [lambda: room.Room(table.long(), length, 6, 16), lambda: room.Room(table, length[:2], 6, 16), lambda: room.Room(table, length, 6, 24),
           lambda: room.Room(table, length, 0, 16), lambda: room.Room(table.cpu(), length, 6, 16), lambda: room.Room(table, length, 6, 16, free),
           lambda: room.Room(table, length, 5, 16, free, state), lambda: room.Room(table, length, 6, 16, free, state[:1]),
           lambda: room.Room(table, length, 6, 16, free, state, tokens=-1), lambda: room.Room(table.t(), length[:2], 6, 16),
           lambda: room.make_room(room.Room(table, length, 6, 16), 1), lambda: room.make_room(x, length.long()),
           lambda: room.make_room(x, length[:2]), lambda: room.make_room(x, 2 ** 31), lambda: room.make_room(x, 1, rows=-1),
           lambda: room.make_room(x, 1, length), lambda: room.make_room(x, 1, torch.zeros(2, dtype=torch.bool, device='cuda')),
           lambda: room.places(x), lambda: room.places(x, tokens=3), lambda: room.places(x, count=-1),
           lambda: room.places(x, length, tokens=3), lambda: room.places(x, torch.zeros(4, dtype=torch.int64, device='cuda'), tokens=3),
           lambda: room.places(x, count=2 ** 30)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('not refused', i)
    n = 131073
    many = room.Room(torch.zeros((n, 1), dtype=torch.int32, device='cuda'), torch.zeros(n, dtype=torch.int32, device='cuda'), 6, 16, free, state)
    with pytest.raises(ValueError, match='worlds'):
        room.make_room(many, 1)
    assert not length.any() and not state.any()


def test_wrong_calls_change_nothing(gpu_available):
    import torch
    print('case room wrong calls', flush=True)
    c = room.DeviceEpisodeCache(4, kv_heads=1, head_dim=32, tokens=50, storage='bf16', page_tokens=16)
    c.extend(5)
    before = [x.clone() for x in (c.table, c.length, c.room.state, c.room.free)]
    two = torch.full((4,), 2, dtype=torch.int32, device='cuda')
    for call in (lambda: c.extend(two), lambda: c.extend(-1), lambda: c.extend(1, rows=3), lambda: c.extend(1, most=1),
                 lambda: c.extend(two.long(), rows=8), lambda: c.extend(two, rows=-1), lambda: c.extend(two, rows=8, most=-1),
                 lambda: c.take_back(-1), lambda: c.reset(two), lambda: c.extend(1, two.bool()[:3]), lambda: c.extend(2 ** 31)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: c.extend(2.5), lambda: c.extend(two, rows=8.5), lambda: c.take_back(0.5)):
        with pytest.raises(TypeError):
            call()
    c.take_back(-two)                                # counts that are not to be: refused on the device
    with pytest.raises(RuntimeError, match='more new rows'):
        c.check()
    for x, y in zip((c.table, c.length, c.room.state, c.room.free), before):
        assert torch.equal(x, y)
    assert c.extend(np.int64(2)).shape == (4, 2) and c.lengths.tolist() == [7] * 4


@pytest.mark.parametrize('busy', ['changes', 'calls'])
def test_device_cache_streams_keep_their_order(gpu_available, busy):
    """Changes on one stream, calls and what the host reads on another, whichever is behind."""
    import torch
    print('case device cache order', busy, flush=True)
    gen = torch.Generator('cuda').manual_seed(3)
    rows = [[torch.randn((5, 3, h, 64), generator=gen, device='cuda').bfloat16() for h in (2, 2, 4)] for _ in range(5)]

    def play(side):
        c = room.DeviceEpisodeCache(5, kv_heads=2, head_dim=64, tokens=64, storage='bf16', page_tokens=16, pages=9, block_tokens=16)
        torch.cuda.synchronize()
        outs, lengths = [], []
        for i, (k, v, q) in enumerate(rows):
            if busy == 'calls' and side is not None:
                with torch.cuda.stream(side):
                    torch.cuda._sleep(20_000_000)
            if busy == 'changes':
                torch.cuda._sleep(20_000_000)
            over = torch.tensor([i == 3, False, i == 2, False, i == 3], device='cuda')
            chunk = c.extend(3, over)
            options = dict(stream=side) if side is not None else {}
            c.write(chunk, k, v, **options)
            outs += [c.attend(chunk, q, **options), c.recall(chunk, q, top=1, **options)]
            with torch.cuda.stream(side):
                lengths.append(c.lengths.tolist())
        torch.cuda.synchronize()
        return outs, lengths

    want, lengths = play(None)
    got, again = play(torch.cuda.Stream())
    assert lengths == again and lengths[3] == [3, 12, 6, 12, 3]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
