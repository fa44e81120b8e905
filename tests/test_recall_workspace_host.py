"""How large the workspace of attention to listed blocks may become (no GPU is needed)."""
import ctypes as ct

import pytest

from libero_hip import episodes

GIB = 2 ** 30


def workspace(worlds, blocks, heads, kv, dim, tokens, listed, most, block=64, page=64, even=None):
    at = 4096
    pages = episodes.MxPages(at, at, None, None, at, at, worlds, 1000, blocks * block // page, kv, dim, page, 1)
    chunk = episodes.MxChunk(at, tokens, 0) if even is None else episodes.MxChunk(None, worlds * even, even)
    rows = episodes.MxRows(at, heads * dim, dim, heads, 1)
    attention = episodes.MxAttention(rows, rows, None, None, 0, most, 1, 0, 0.125)
    selection = episodes.MxSelection(at, listed)
    return episodes.load().mx_recall_workspace(*(ct.byref(x) for x in (pages, chunk, attention, selection)), block)


@pytest.mark.parametrize('worlds,blocks,heads,kv,dim,tokens,listed', [
    (1024, 128, 8, 8, 128, 32768, 19), (256, 1024, 8, 8, 64, 32768, 64), (256, 2048, 8, 8, 64, 65536, 64),
    (64, 512, 8, 8, 128, 16384, 19), (4096, 32, 4, 4, 64, 32768, 19), (1, 1024, 32, 8, 128, 2048, 19),
    (1, 16384, 8, 8, 128, 32768, 128), (3, 4096, 2, 2, 256, 32768, 256)])
def test_chunks_of_unknown_size(worlds, blocks, heads, kv, dim, tokens, listed):
    """Ragged chunks whose largest is not known take little more than those whose largest is, and what they take follows from
    the rows: the sums of a batch of key heads (1 GiB at most), 8 bytes to each row and entry, and of marks a bit for each
    row and block, rounded up to words for each world."""
    rows = tokens * heads
    marks = 4 * kv * blocks * (tokens // 32 + worlds)
    tiles = kv * (tokens * listed // (128 // (heads // kv)) + worlds * blocks)
    most = GIB + 8 * rows * listed + marks + tiles * (16 + 4 * 128 // (heads // kv)) + 4096
    assert workspace(worlds, blocks, heads, kv, dim, tokens, listed, tokens) <= most
    known = workspace(worlds, blocks, heads, kv, dim, tokens, listed, min(tokens, 2 * (tokens // worlds)))
    assert workspace(worlds, blocks, heads, kv, dim, tokens, listed, tokens) <= 1.01 * known + 4096


def test_marks_have_an_end():
    """No call asks for more than a few GiB, whatever the table could hold: then rows are not gathered."""
    for worlds, blocks in ((1, 2 ** 18), (16, 2 ** 16), (64, 2 ** 14), (1, 2 ** 14)):
        for tokens in (2048, 32768):
            for heads, kv, dim, listed in ((8, 8, 128, 128), (4, 4, 256, 256), (8, 2, 64, 64)):
                for block in (64, 256, 4096):
                    if blocks * block > 2 ** 30:
                        continue
                    need = workspace(worlds, blocks, heads, kv, dim, tokens, listed, tokens, block, max(block, 64))
                    assert need <= 4 * GIB, (worlds, blocks, tokens, heads, kv, dim, listed, block, need / GIB)
