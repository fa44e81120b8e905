"""What the episode memory's further operators refuse before any launch (no GPU is needed), against include/mx_episode.h, the
angles of rotary positions, and the definitions that the GPU tests compare with against independent facts."""
import ctypes as ct
import math

import numpy as np
import pytest

from recall_reference import Books, blocks_of, codes, summary, turned
from libero_hip import episodes
from libero_hip.rotary import Rotary

INVALID, DOMAIN, WORKSPACE = -1, -2, -5


class Call:
    """Arguments that pass every check but the last; with no rows (or for room, no workspace), so that nothing is launched."""

    def __init__(self):
        self.buffer = ct.create_string_buffer(4096)
        at = (ct.addressof(self.buffer) + 63) & ~63
        self.at = at
        self.pages = episodes.MxPages(at, at, None, None, at, at, 2, 4, 64, 2, 64, 64, 1)
        self.chunk = episodes.MxChunk(None, 0, 0)
        self.q = episodes.MxRows(at, 256, 64, 4, 1)
        self.out = episodes.MxRows(at, 256, 64, 4, 1)
        self.k = episodes.MxRows(at, 128, 64, 2, 1)
        self.v = episodes.MxRows(at, 128, 64, 2, 1)
        self.rotary = episodes.MxRotary(at, 64, 0, 1.0)
        self.summaries = episodes.MxSummaries(at, at, 32)
        self.selection = episodes.MxSelection(at, 8, 4, 2, 1, 1, 1)
        self.attention = episodes.MxAttention(self.q, self.out, None, None, 0, 1, 1, 0, 0.125)
        self.room = episodes.MxRoom(at, at, at, at, 2, 4, 8, 64, 256)
        self.change = episodes.MxRoomChange(None, None, at, None, 0, 1, 2)
        self.head_dim, self.tokens, self.period, self.block = 64, 0, 1, 32

    def rotate(self):
        return episodes.load().mx_rotate(ct.byref(self.rotary), ct.byref(self.q), ct.byref(self.out), self.head_dim, self.tokens,
                                         self.at, self.period, 0, 0, None)

    def enter(self):
        return episodes.load().mx_episode_enter(*(ct.byref(x) for x in (self.pages, self.chunk, self.rotary, self.q, self.out,
                                                                        self.k, self.v)), None)

    def update(self):
        return episodes.load().mx_room_update(ct.byref(self.room), ct.byref(self.change), None)

    def places(self):
        return episodes.load().mx_room_places(ct.byref(self.room), ct.byref(self.chunk), self.at, self.at, self.at, None)

    def summarise(self):
        return episodes.load().mx_episode_summarise(ct.byref(self.pages), ct.byref(self.chunk), ct.byref(self.summaries), None)

    def select(self):
        return episodes.load().mx_episode_select(*(ct.byref(x) for x in (self.pages, self.chunk, self.summaries, self.q,
                                                                         self.selection)), None)

    def recall(self):
        return episodes.load().mx_episode_recall(*(ct.byref(x) for x in (self.pages, self.chunk, self.attention, self.selection)),
                                                 self.block, None)

    def workspace(self):
        return episodes.load().mx_recall_workspace(*(ct.byref(x) for x in (self.pages, self.chunk, self.attention, self.selection)),
                                                   self.block)


def check(entry, code, change):
    c = Call()
    change(c)
    assert getattr(c, entry)() == code, entry


def setting(name, field, value):
    return lambda c: setattr(getattr(c, name), field, value)


def test_what_passes():
    for entry in ('rotate', 'enter', 'places', 'summarise', 'select', 'recall'):
        assert getattr(Call(), entry)() == 0, entry


@pytest.mark.parametrize('entry', ['enter', 'summarise', 'select', 'recall'])
def test_pages_and_chunks_are_checked(entry):
    for field, value, code in (('k', None, INVALID), ('table', None, INVALID), ('nworld', 0, INVALID), ('type', 0, INVALID),
                               ('head_dim', 48, DOMAIN), ('page_tokens', 48, DOMAIN), ('npage', 2 ** 26, DOMAIN)):
        check(entry, code, setting('pages', field, value))
    for tokens, count in ((3, 1), (-1, 0), (0, -1)):
        check(entry, INVALID, lambda c: setattr(c, 'chunk', episodes.MxChunk(None, tokens, count)))


def test_rotary_is_checked():
    for entry in ('rotate', 'enter'):
        for field, value in (('turn', None), ('width', 0), ('width', 63), ('width', 66)):
            check(entry, INVALID, setting('rotary', field, value))
        for row in ('q', 'out'):
            for field, value in (('type', 3), ('type', 7), ('heads', 0)):
                check(entry, INVALID, setting(row, field, value))
        check(entry, INVALID, setting('out', 'type', 2))
    check('rotate', DOMAIN, lambda c: setattr(c, 'head_dim', 1025))
    check('rotate', DOMAIN, lambda c: setattr(c, 'head_dim', 1))
    check('rotate', INVALID, lambda c: setattr(c, 'tokens', -1))

    def rows(c):
        c.tokens, c.period = 4, 0
    check('rotate', INVALID, rows)

    def nothing(c):
        c.tokens, c.q.data = 4, None
    check('rotate', INVALID, nothing)
    for field, value in (('heads', 3), ('type', 2)):
        check('enter', INVALID, setting('k', field, value))
        check('enter', INVALID, setting('v', field, value))


def test_room_is_checked():
    for entry in ('update', 'places'):
        for field, value, code in (('table', None, INVALID), ('length', None, INVALID), ('nworld', 0, INVALID), ('width', 0, INVALID),
                                   ('npage', 0, INVALID), ('tokens', -1, INVALID), ('page_tokens', 8, DOMAIN),
                                   ('page_tokens', 96, DOMAIN), ('npage', 2 ** 26, DOMAIN), ('width', 2 ** 25, DOMAIN)):
            check(entry, code, setting('room', field, value))
    check('update', INVALID, setting('room', 'free', None))
    check('update', INVALID, setting('room', 'state', None))
    check('update', INVALID, setting('change', 'rows', -1))
    check('update', DOMAIN, setting('room', 'nworld', 131073))
    check('places', INVALID, lambda c: setattr(c, 'chunk', episodes.MxChunk(None, 3, 1)))
    c = Call()
    c.room.nworld, c.room.npage = 2000, 9000
    need = episodes.load().mx_room_workspace(ct.byref(c.room))
    assert need >= 16 and c.update() == WORKSPACE
    c.change.workspace, c.change.workspace_bytes = c.at, need - 1
    assert c.update() == WORKSPACE
    c.change.workspace, c.change.workspace_bytes = c.at + 4, need
    assert c.update() == WORKSPACE


def test_recall_is_checked():
    for field, value, code in (('codes', None, INVALID), ('exponent', None, INVALID), ('block_tokens', 8, DOMAIN),
                               ('block_tokens', 48, DOMAIN), ('block_tokens', 128, DOMAIN)):
        check('summarise', code, setting('summaries', field, value))
        check('select', code, setting('summaries', field, value))
    for field, value, code in (('top', -1, INVALID), ('near', 0, INVALID), ('first', -1, INVALID), ('max_count', -1, INVALID),
                               ('width', 0, INVALID), ('width', 6, INVALID), ('top', 1025, DOMAIN), ('width', 4097, DOMAIN)):
        check('select', code, setting('selection', field, value))
    for field, value in (('heads', 3), ('heads', 0), ('type', 0), ('type', 2)):
        check('select', INVALID, setting('q', field, value))
    for value in (8, 48, 128):
        check('recall', DOMAIN, lambda c: setattr(c, 'block', value))
    check('recall', DOMAIN, setting('selection', 'width', 0))
    check('recall', DOMAIN, setting('selection', 'width', 4097))
    check('recall', INVALID, setting('attention', 'window', 5))

    def rows(c):
        c.chunk, c.selection.blocks = episodes.MxChunk(None, 2, 1), None
    check('recall', INVALID, rows)
    check('select', INVALID, rows)


def test_recall_workspace():
    """Long lists of few rows are split, into a workspace that has to be there."""
    c = Call()
    c.chunk = episodes.MxChunk(None, 2, 1)
    c.selection.width, c.pages.width = 400, 4096
    need = c.workspace()
    assert need > 0 and need % (2 * 4 * (64 + 2) * 4) == 0
    assert c.recall() == WORKSPACE
    c.selection.width = 2
    assert c.workspace() == 0


def test_angles():
    """The first pair turns by one radian; scalings divide what they should, and leave what they should."""
    turn, amplitude = Rotary.angles(64, base=10000.0)
    assert turn.shape == (32,) and turn[0] == 1.0 and amplitude == 1.0
    np.testing.assert_allclose(turn.numpy(), 10000.0 ** (-np.arange(32) / 32), rtol=1e-15)
    linear, _ = Rotary.angles(64, scaling='linear', factor=4.0)
    np.testing.assert_array_equal(linear.numpy(), turn.numpy() / 4)
    larger, _ = Rotary.angles(64, scaling='base', factor=4.0)
    assert larger[0] == 1.0
    np.testing.assert_allclose(larger[-1], turn[-1] / 4, rtol=1e-14)
    parts, amplitude = Rotary.angles(64, scaling='parts', factor=4.0, original=512)
    turns = 512 * turn.numpy() / (2 * math.pi)
    np.testing.assert_allclose(parts.numpy()[turns >= 32], turn.numpy()[turns >= 32], rtol=1e-15)
    np.testing.assert_allclose(parts.numpy()[turns <= 1], turn.numpy()[turns <= 1] / 4, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and np.all((parts.numpy() < turn.numpy())[between]) and np.all((parts.numpy() > turn.numpy() / 4)[between])
    assert amplitude == 0.1 * math.log(4.0) + 1
    for options in (dict(width=3), dict(width=0), dict(width=4, base=0.0), dict(width=4, scaling='other'),
                    dict(width=4, scaling='linear', factor=0.5), dict(width=2, scaling='base', factor=2.0),
                    dict(width=4, scaling='parts', factor=2.0), dict(width=4, scaling='parts', original=9, slow=3, fast=2)):
        with pytest.raises(ValueError):
            Rotary.angles(**options)


def test_reference_rotation():
    """A quarter turn swaps a pair; lengths stay, and turning back undoes it."""
    x = np.arange(1.0, 7.0).reshape(1, 1, 6)
    quarter = np.array([math.pi / 2, 0.0])
    np.testing.assert_allclose(turned(x, [1], quarter, 1.0, 'half')[0, 0], [-3, 2, 1, 4, 5, 6], atol=1e-15)
    np.testing.assert_allclose(turned(x, [1], quarter, 1.0, 'interleaved')[0, 0], [-2, 1, 3, 4, 5, 6], atol=1e-15)
    y = turned(x, [77], np.array([0.3, 1.7]), 2.0, 'half')
    np.testing.assert_allclose(np.linalg.norm(y[0, 0, :4]), 2 * np.linalg.norm(x[0, 0, :4]))
    np.testing.assert_allclose(turned(y, [77], np.array([0.3, 1.7]), 0.5, 'half', back=True), x)


def test_reference_codes_and_blocks():
    c, e = codes(np.array([[127.0, -63.5, 0.0], [127.5, 1.0, np.nan], [0.0, 0.0, 0.0], [np.inf, -1e30, 1.0], [2.0 ** -41 * 1.5, 0, 0]]))
    assert c.tolist() == [[127, -64, 0], [64, 0, 0], [0, 0, 0], [127, -127, 0], [1, 0, 0]] and e.tolist() == [0, 1, -40, 40, -40]
    assert summary(np.full((16, 2), 3.0))[0].tolist() == [96, 96] and summary(np.array([[np.inf, 1.0]]))[1] == 255
    k = np.zeros((170, 4))
    k[:, 0] = np.arange(170) // 16 % 5                    # blocks of 0 to 4
    q = np.array([[1.0, 0, 0, 0]])
    # own block 10 and the one before are near, 0 is first; of 1 .. 8 the largest are 4, then 3 before 8
    assert blocks_of(q, k, 169, 170, 16, 2, 2, 1, True) == [0, 3, 4, 9, 10]
    assert blocks_of(q, k, 169, 170, 16, 3, 2, 1, True) == [0, 3, 4, 8, 9, 10]
    assert blocks_of(-q, k, 169, 170, 16, 1, 1, 0, True) == [0, 10]
    assert blocks_of(q, k, 20, 170, 16, 1, 1, 1, True) == [0, 1]
    assert blocks_of(q, k, 20, 60, 16, 1, 1, 1, False) == [0, 1, 2, 3]
    assert blocks_of(q, k, -1, 170, 16, 1, 1, 1, True) == []


def test_reference_books():
    """Tokens taken back leave everything as it was; what does not fit changes nothing."""
    b = Books(np.full((2, 4), -1), np.zeros(2), range(6), 50, 16)
    assert b.change(np.array([17, 3])).tolist() == [0, 17, 20]
    assert b.table.tolist() == [[5, 4, -1, -1], [3, -1, -1, -1]] and b.free == [0, 1, 2]
    b.change(np.array([30, 20]))
    assert b.table.tolist() == [[5, 4, 2, -1], [3, 1, -1, -1]] and b.free == [0] and b.length.tolist() == [47, 23]
    b.change(np.array([-30, -20]))
    assert b.table.tolist() == [[5, 4, -1, -1], [3, -1, -1, -1]] and b.free == [0, 1, 2] and not b.why
    assert not b.change(np.array([34, 1])).any() and b.why == 1 and b.length.tolist() == [17, 3]
    b.change(np.array([5, 2]), np.array([True, False]))
    assert b.table.tolist() == [[5, -1, -1, -1], [3, -1, -1, -1]] and b.free == [0, 1, 2, 4]
