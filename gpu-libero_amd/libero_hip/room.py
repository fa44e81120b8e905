"""Room for new tokens on the GPU: tables, lengths and free pages change without the host.

:class:`libero_hip.episodes.EpisodeCache` keeps its books on the host.  Here they are on the device, so that a step whose
worlds end and grow as the device finds out can be captured as a whole:

* :func:`make_room` empties worlds, gives others room for new tokens, or takes tokens back;
* :func:`places` tells the world, position and slot of each of a chunk's rows;
* :class:`DeviceEpisodeCache` is the cache with both in the place of ``extend`` and ``reset`` on the host.

A change that does not fit is refused as a whole, and the reason stays in ``state`` until the host looks.  The operators
run on the current stream or ``stream``, as those of :mod:`libero_hip.episodes`, and can be captured into a HIP graph.  The
reference has no counterpart.
"""
from __future__ import annotations

import ctypes as ct

import numpy as np
import torch

from . import episodes
from .episodes import MxChunk, MxRoom, MxRoomChange, _PAGE_TOKENS, _captured, _check, _current, _on, _require

REFUSED = {1: 'a world would hold more tokens than it may, or fewer than none', 2: 'the free pages do not suffice',
           4: 'more new rows than there is space for'}
MOST_WORLDS = 131072


class Room:
    """The worlds' tables and lengths (see :class:`libero_hip.episodes.Pages`) and the pages that none of them has.

    ``table`` (nworld, pages of a world) and ``length`` (nworld,), ``free`` (npage,) and ``state`` (2,) are contiguous int32 on
    one GPU.  ``free[:state[0]]`` are the numbers of the free pages, the next one last; ``state[1]`` collects why changes were
    refused (:data:`REFUSED`), until the caller sets it to 0.  ``tokens``: the most of a world, by default what its table
    reaches.  :func:`places` needs neither ``free`` nor ``state``.  The tensors stay the caller's, and are held here."""

    __slots__ = ('table', 'length', 'free', 'state', 'struct', 'index', 'workspace')

    def __init__(self, table, length, npage, page_tokens, free=None, state=None, *, tokens=None):
        index = table.get_device()
        if not (index >= 0 and table.dtype == torch.int32 and table.dim() == 2 and table.numel() and table.is_contiguous()
                and length.dtype == torch.int32 and length.shape == table.shape[:1] and length.is_contiguous()
                and length.get_device() == index and page_tokens in _PAGE_TOKENS and npage > 0
                and npage * page_tokens < 2 ** 31 and table.shape[1] * page_tokens <= 2 ** 30):
            _require(page_tokens in _PAGE_TOKENS, 'page_tokens must be a power of two from 16 to 4096, got %s', page_tokens)
            _require(npage > 0 and npage * page_tokens < 2 ** 31 and table.dim() == 2 and table.shape[1] * page_tokens <= 2 ** 30,
                     'npage * page_tokens must be below 2^31 and the tokens of a table row at most 2^30')
            raise ValueError('table (nworld, pages of a world) and length (nworld,) must be contiguous int32 on one GPU')
        _require((free is None) == (state is None), 'free and state go together')
        if free is not None:
            _require(free.dtype == torch.int32 and free.shape == (npage,) and free.is_contiguous() and free.get_device() == index,
                     'free must be contiguous int32 of shape (npage,) on the table\'s device')
            _require(state.dtype == torch.int32 and state.shape == (2,) and state.is_contiguous() and state.get_device() == index,
                     'state must be contiguous int32 of shape (2,) on the table\'s device')
        reach = table.shape[1] * page_tokens
        tokens = reach if tokens is None else tokens
        _require(0 <= tokens < 2 ** 31, 'tokens must be a number of tokens, got %s', tokens)
        self.table, self.length, self.free, self.state, self.index = table, length, free, state, index
        self.struct = MxRoom(table.data_ptr(), length.data_ptr(), None if free is None else free.data_ptr(),
                             None if state is None else state.data_ptr(), table.shape[0], table.shape[1], npage, page_tokens, tokens)
        self.workspace = None             # bytes, once a change has asked

    @property
    def device(self):
        return self.table.device


def _away(room, stream):
    return stream is not None or torch.cuda.current_device() != room.index


def make_room(room, count, over=None, *, rows=None, stream=None):
    """Empty the worlds of ``over`` (bool, one to a world), then give every world room for ``count`` new tokens: a number, or
    int32 of shape (nworld,).  A negative count takes a world's last tokens back, as after looking ahead.  Returns ``start``
    (int32, nworld + 1), the chunk of the new tokens for :func:`libero_hip.episodes.write` and the others, whose rows are packed.

    Pages go to worlds in their order, the next free one first, and come back in the opposite one, so that tokens taken back
    leave tables and free pages as they were.  If a world would pass the room's tokens or fall below none, if the free
    pages do not suffice, or if there are more new tokens than ``rows`` (what the caller's tensors hold; for a tensor of counts
    as many as there may be), no world gets or gives back any token: ``start`` is all 0, so that nothing is written or
    computed, and ``room.state[1]`` says why.  The worlds of ``over`` are empty all the same.  Changes of one room from several
    streams are the caller's to order."""
    if _away(room, stream):
        tensors = (count if torch.is_tensor(count) else None, over, room.table, room.length, room.free, room.state)
        return _on(room.device, stream, tensors, lambda: make_room(room, count, over, rows=rows))
    s = room.struct
    _require(room.free is not None, 'the room has no free pages to change: give it free and state')
    _require(s.nworld <= MOST_WORLDS, 'at most %d worlds can change at once, got %d', MOST_WORLDS, s.nworld)
    change = MxRoomChange()
    if torch.is_tensor(count):
        _require(count.dtype == torch.int32 and count.shape == (s.nworld,) and count.is_contiguous()
                 and count.get_device() == room.index,
                 'count must be a number, or contiguous int32 of shape (nworld,) on the room\'s device')
        change.count = count.data_ptr()
        rows = 2 ** 31 - 1 if rows is None else rows
    else:
        _require(-2 ** 31 < count < 2 ** 31, 'count must be a number of tokens, got %s', count)
        change.each = count
        rows = min(s.nworld * max(count, 0), 2 ** 31 - 1) if rows is None else rows
    _require(0 <= rows < 2 ** 31, 'rows must be a number of rows, got %s', rows)
    if over is not None:
        _require(over.dtype in (torch.bool, torch.uint8) and over.shape == (s.nworld,) and over.is_contiguous()
                 and over.get_device() == room.index, 'over must be contiguous bool of shape (nworld,) on the room\'s device')
        change.over = over.data_ptr()
    lib, device = episodes._LIB or episodes.load(), room.table.device
    if room.workspace is None:
        room.workspace = lib.mx_room_workspace(ct.byref(s))
    start = torch.empty(s.nworld + 1, dtype=torch.int32, device=device)
    if room.workspace:
        workspace = torch.empty(room.workspace, dtype=torch.uint8, device=device)
        change.workspace, change.workspace_bytes = workspace.data_ptr(), room.workspace
    change.start, change.rows = start.data_ptr(), rows
    rc = lib.mx_room_update(ct.byref(s), ct.byref(change), _current(room.index))
    if rc:
        _check(rc, 'mx_room_update')
    return start


def places(room, start=None, *, count=None, tokens=None, stream=None):
    """(world, position, slot) of each of a chunk's rows, int32: ``(nworld, count)``, or packed ``(tokens,)`` with ``start``.
    The slot is ``page * page_tokens`` and the place in the page.  Rows that belong to no world have -1 for all, those
    before their world's first token -1 for position and slot, those without a page -1 for the slot."""
    if _away(room, stream):
        return _on(room.device, stream, (start, room.table, room.length), lambda: places(room, start, count=count, tokens=tokens))
    s = room.struct
    many, none = (count, tokens) if start is None else (tokens, count)
    _require(many is not None and none is None and many >= 0, 'give count (every world), or start and tokens')
    if start is None:
        _require(s.nworld * count < 2 ** 31, 'a chunk has fewer than 2^31 rows: %d worlds of %d', s.nworld, count)
        shape, chunk = (s.nworld, count), MxChunk(None, s.nworld * count, count)
    else:
        _require(start.dtype == torch.int32 and start.shape == (s.nworld + 1,) and start.is_contiguous()
                 and start.get_device() == room.index, 'start must be contiguous int32 of shape (nworld + 1,) on the room\'s device')
        _require(tokens < 2 ** 31, 'a chunk has fewer than 2^31 rows: %d', tokens)
        shape, chunk = (tokens,), MxChunk(start.data_ptr(), tokens, 0)
    rows = chunk.tokens
    step = rows if rows < 4096 else rows + -rows % 4          # many rows: each of the three is 16-byte aligned
    found = torch.empty((3, step), dtype=torch.int32, device=room.table.device)
    at = found.data_ptr()
    lib = episodes._LIB or episodes.load()
    rc = lib.mx_room_places(ct.byref(s), ct.byref(chunk), at, at + 4 * step, at + 8 * step, _current(room.index))
    if rc:
        _check(rc, 'mx_room_places')
    if step > rows:
        found = found[:, :rows]
    return (found if start is not None else found.unflatten(1, shape)).unbind(0)


class DeviceChunk:
    """New tokens of a :class:`DeviceEpisodeCache`: packed rows with ``start`` on the device.  ``tokens``: how many rows tensors
    have, ``count``: the most of a world; with one count for all worlds, rows may also be ``(nworld, count, heads, head_dim)``."""

    __slots__ = ('start', 'tokens', 'count', 'shape')
    longest, bounded = 0, True            # tokens and count hold for replays of captured calls too

    def __init__(self, start, tokens, count, shape):
        self.start, self.tokens, self.count, self.shape = start, tokens, count, shape


class DeviceEpisodeCache(episodes.Layers):
    """:class:`libero_hip.episodes.EpisodeCache` with its books on the device: worlds end, and grow, by tensors there, nothing is
    uploaded and nothing waits, and a whole step of :meth:`extend`, ``write``, ``enter``, ``attend`` and ``recall`` can be
    captured into a HIP graph.

    :meth:`extend` cannot raise where the memory is full: it then does nothing, its chunk has no rows, and :meth:`check`
    (which waits for the device) says so."""

    def __init__(self, nworld, *, kv_heads, head_dim, tokens, pages=None, **options):
        super().__init__(nworld, kv_heads=kv_heads, head_dim=head_dim, tokens=tokens, pages=pages, **options)
        free = torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        state = torch.tensor([self.pages, 0], dtype=torch.int32, device=self.device)
        self.room = Room(self.table, self.length, self.pages, self.page_tokens, free, state, tokens=self.tokens)

    def _change(self):
        if not _captured(None):               # replays are the caller's to order
            super()._change()

    def _change_done(self):
        if not _captured(None):
            super()._change_done()

    def extend(self, count=1, over=None, *, rows=None, most=None):
        """Empty the worlds of ``over``, then make room for new tokens of every world, as :func:`make_room`, and return their
        chunk.  ``count``: a number, or int32 on the device, with ``rows`` (how many rows the step's tensors have; those beyond the
        counts' sum belong to no world, and what is computed from them is not defined) and ``most`` (the most of one world,
        if known: rows of a world beyond it are not attended from, and without causality :meth:`recall` has room for the last blocks
        of ``most`` tokens only)."""
        if torch.is_tensor(count):
            _require(rows is not None, 'give rows with a tensor of counts')
            most = rows if most is None else most
            _require(0 <= most < 2 ** 31, 'most must be a number of tokens, got %s', most)
            shape = (rows,)
        else:
            _require(count >= 0, 'count must not be negative; take tokens back with take_back')
            _require(most is None and rows in (None, self.nworld * count), 'rows and most go with a tensor of counts')
            most, rows = count, self.nworld * count
            _require(rows < 2 ** 31, 'a chunk has fewer than 2^31 rows: %d worlds of %d', self.nworld, count)
            shape = (self.nworld, count)
        self._change()
        start = make_room(self.room, count, over, rows=rows)
        self._change_done()
        return DeviceChunk(start, rows, most, shape)

    def take_back(self, count):
        """The last ``count`` tokens of every world (a number, or int32 on the device, none negative) are gone, as if they had
        never been."""
        _require(torch.is_tensor(count) or count >= 0, 'count must not be negative')
        self._change()
        make_room(self.room, -count, rows=0)
        self._change_done()

    def reset(self, over=None):
        """Empties the worlds of ``over`` (bool on the device; None: all)."""
        self._change()
        if over is None:
            over = torch.ones(self.nworld, dtype=torch.bool, device=self.device)
        make_room(self.room, 0, over)
        self._change_done()

    def places(self, chunk):
        """:func:`places` of the chunk's rows, in the chunk's shape."""
        other = self._enter(None, chunk.start)
        found = places(self.room, chunk.start, tokens=chunk.tokens)
        self._leave(other)
        return tuple(x.view(chunk.shape) for x in found)

    def _seen(self, x):
        """A tensor's values after the last change, on the host."""
        other = self._enter(None)
        x = x.cpu()
        self._leave(other)
        return x

    def check(self):
        """Raises RuntimeError if a change was refused since the last call; waits for the device."""
        why = int(self._seen(self.room.state)[1])
        if why:
            self._change()
            self.room.state[1] = 0
            self._change_done()
            raise RuntimeError('episode memory: ' + '; '.join(text for bit, text in REFUSED.items() if why & bit))

    @property
    def free_pages(self):
        """How many pages are free; waits for the device."""
        return int(self._seen(self.room.state)[0])

    @property
    def lengths(self):
        """The worlds' tokens (numpy); waits for the device."""
        return self._seen(self.length).numpy().astype(np.int64)
