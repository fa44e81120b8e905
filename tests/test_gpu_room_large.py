"""Room and places of thousands of worlds, at and beyond the sizes where other ways to find them begin."""
import numpy as np
import pytest

from libero_hip import room
from test_gpu_room import Rooms, there

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('nworld', [1023, 1024, 1025, 4096, 20000])
@pytest.mark.parametrize('kind', ['single', 'ragged', 'sparse', 'first', 'last', 'empty'])
def test_places(gpu_available, nworld, kind):
    """Chunks of one token each, of several, of few worlds with many empty ones between, of one world alone, of none; rows
    beyond the last world's."""
    import torch
    print('case places large', nworld, kind, flush=True)
    rng = np.random.default_rng(nworld)
    page, width = 16, 4
    table = rng.permutation(width * nworld).reshape(nworld, width).astype(np.int32)
    table[rng.random((nworld, width)) < 0.05] = -1
    length = rng.integers(0, 80, nworld).astype(np.int32)          # some beyond the table's reach
    counts = np.zeros(nworld, int)
    if kind == 'single':
        counts[:] = 1
    elif kind == 'ragged':
        counts = rng.integers(0, 8, nworld)
    elif kind == 'sparse':
        counts[rng.random(nworld) < 0.003] = 700
    elif kind == 'first':
        counts[0] = 2500
    elif kind == 'last':
        counts[-1] = 2500
    x = room.Room(there(table), there(length), width * nworld, page)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    for extra in (0, 1500):
        tokens = int(start[-1]) + extra
        world = np.full(tokens, -1)
        world[:start[-1]] = np.repeat(np.arange(nworld), counts)
        there_is = world >= 0
        w = np.maximum(world, 0)
        position = length[w] - counts[w] + np.arange(tokens) - start[w]
        entry = np.clip(position // page, 0, width - 1)
        has = there_is & (position >= 0) & (position < page * width) & (table[w, entry] >= 0)
        want = [world, np.where(there_is, np.maximum(position, -1), -1), np.where(has, table[w, entry] * page + position % page, -1)]
        for a, b in zip(room.places(x, there(start), tokens=tokens), want):
            np.testing.assert_array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize('nworld', [1024, 1025, 16384, 131072])
def test_changes(gpu_available, nworld):
    """The most worlds that a change takes: some end, some grow, some give tokens back; refused, and restarted as a whole."""
    print('case room large', nworld, flush=True)
    rng = np.random.default_rng(nworld)
    page, width = 16, 3
    r = Rooms(nworld, width, 2 * nworld, page, seed=nworld)
    r.change(rng.integers(0, 25, nworld))
    assert not r.books.why
    over = rng.random(nworld) < 0.2
    base = np.where(over, 0, r.books.length)
    r.change(np.where(rng.random(nworld) < 0.5, rng.integers(0, 8, nworld), -(base // 2)), over)
    assert not r.books.why
    r.change(48 - np.where(over, 0, r.books.length), over)            # three pages for each: refused, but for `over`
    assert r.books.why == 2
    r.change(rng.integers(17, 33, nworld), np.ones(nworld, bool))     # two pages for each
    assert len(r.books.free) == 0
    r.change(0, np.ones(nworld, bool), uniform=True)
    assert len(r.books.free) == 2 * nworld


def test_totals_beyond_32_bits(gpu_available):
    """New rows of all worlds that sum up to more than 2^32: refused, whatever their low bits say."""
    print('case room totals', flush=True)
    n = 5000
    r = Rooms(n, 256, 4, 4096)
    r.change(2 ** 20, uniform=True, rows=2 ** 31 - 1)
    assert r.books.why == 6
