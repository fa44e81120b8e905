"""Host bookkeeping of EpisodeCache (on CPU tensors, no library call): pages given out and taken back."""
import numpy as np
import pytest
import torch

from libero_hip import episodes


class NoPages:
    """In the place of Pages, whose tensors have to be on the GPU."""

    def __init__(self, *tensors):
        self.tensors = tensors


def cache(monkeypatch, nworld=5, tokens=70, **options):
    monkeypatch.setattr(episodes, 'Pages', NoPages)
    return episodes.EpisodeCache(nworld, kv_heads=1, head_dim=32, tokens=tokens, page_tokens=16, device='cpu', **options)


def consistent(c):
    """Device copies equal the host's; every page has one owner or is free; worlds have the pages their tokens need."""
    np.testing.assert_array_equal(c.table.numpy(), c._table)
    np.testing.assert_array_equal(c.length.numpy(), c.lengths)
    held = c._table[c._table >= 0]
    everyone = np.concatenate([held, c._free[:c._left]])
    assert len(np.unique(everyone)) == len(everyone) == len(c._free)
    need = -(-c.lengths // c.page_tokens)
    np.testing.assert_array_equal(c._table >= 0, np.arange(c._table.shape[1]) < need[:, None])


def test_extend_and_reset(monkeypatch):
    rng = np.random.default_rng(0)
    c = cache(monkeypatch, pages=14)
    assert c.table.shape == (5, 5) and c.free_pages == 14
    refused = 0
    for _ in range(300):
        before = c.lengths.copy(), c._table.copy(), c.free_pages
        ids = None if rng.random() < 0.3 else rng.permutation(5)[:rng.integers(0, 6)]
        n = 5 if ids is None else len(ids)
        count = int(rng.integers(0, 9)) if rng.random() < 0.5 else rng.integers(0, 30, n)
        try:
            chunk = c.extend(count, ids)
        except (RuntimeError, ValueError):
            refused += 1
            np.testing.assert_array_equal(before[0], c.lengths)
            np.testing.assert_array_equal(before[1], c._table)
            assert before[2] == c.free_pages
            c.reset(rng.permutation(5)[:2])
        else:
            np.testing.assert_array_equal(c.lengths - before[0], chunk.counts)
            assert chunk.tokens == chunk.counts.sum() and chunk.count == chunk.counts.max()
            if chunk.start is None:
                assert len(set(chunk.counts)) == 1 and chunk.shape == (5, chunk.count)
            else:
                np.testing.assert_array_equal(chunk.start.numpy(), np.r_[0, np.cumsum(chunk.counts)])
                assert chunk.shape == (chunk.tokens,)
        consistent(c)
    assert 10 < refused < 200
    c.reset()
    consistent(c)
    assert c.free_pages == 14 and not c.lengths.any()


def test_refusals(monkeypatch):
    c = cache(monkeypatch)
    for bad in (lambda: c.extend(-1), lambda: c.extend(71), lambda: c.extend(1, 5), lambda: c.extend(1, [0, 0]),
                lambda: c.extend([1, 2]), lambda: c.reset(-1)):
        with pytest.raises(ValueError):
            bad()
    consistent(c)
    for options in (dict(storage='f32'), dict(tokens=0), dict(pages=0)):
        with pytest.raises(ValueError):
            cache(monkeypatch, **options)
    for name, value in (('head_dim', 48), ('page_tokens', 24), ('kv_heads', 0), ('layers', 0)):
        with pytest.raises(ValueError):
            episodes.EpisodeCache(2, **{**dict(kv_heads=1, head_dim=32, tokens=9, device='cpu'), name: value})
    assert c.extend(0).count == 0 and c.extend(3, []).tokens == 0


def test_layers_have_their_own_pages(monkeypatch):
    c = cache(monkeypatch, layers=3, storage='fp8')
    tensors = [p.tensors for p in c.layers]
    assert all(t[2] is c.table and t[3] is c.length and len(t) == 6 for t in tensors)
    assert len({t[i].data_ptr() for t in tensors for i in (0, 1, 4, 5)}) == 12
    assert tensors[0][0].shape == (25, 1, 16, 32) and tensors[0][4].shape == (25, 1, 16, 1)
    assert len(cache(monkeypatch, storage='bf16').layers[0].tensors) == 4
    assert torch.float8_e4m3fn == tensors[0][0].dtype
