"""Recall: attention of a query to some blocks of its world's tokens, those that match it best among them.

A long episode is mostly beside the point: of its full blocks of tokens each query attends to the ``top`` whose summaries
match it best, to its latest ``near`` blocks and to the ``first`` ones, whatever the length.

* :func:`summarise` computes the summaries of the blocks that a chunk's tokens complete: the mean of a block's keys, in
  8-bit whole numbers with a power of two;
* :func:`select` chooses the blocks of each query and key head, by products of whole numbers, which are exact: the same blocks
  on any machine;
* :func:`recall` attends to the keys of listed blocks, chosen here or by the caller.

In a step they follow the chunk's :func:`libero_hip.episodes.write` or :func:`libero_hip.rotary.enter`.  They run on the current
stream or ``stream``, as those of :mod:`libero_hip.episodes`, can be captured into a HIP graph, and have no backward pass.
The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as ct
import math

import torch

from . import episodes
from .episodes import (ERR_WORKSPACE, MxAttention, MxRows, MxSelection, MxSummaries, _check, _chunk, _current, _elsewhere, _on, _output,
                       _require, _rows)

MOST_LISTED, MOST_TOP = 4096, 1024


class Summaries:
    """The summaries of one layer's keys: ``codes`` (npage, kv_heads, blocks of a page, head_dim) int8 and ``exponent`` (the
    same without head_dim) uint8, contiguous on the pages' device.  A page's blocks have
    ``block_tokens = page_tokens / blocks`` tokens, 16 at least.  The tensors stay the caller's, and are held here; they belong to the
    pages' slots, and are valid for the full blocks that :func:`summarise` has been called for since they were written."""

    __slots__ = ('pages', 'codes', 'exponent', 'block_tokens', 'struct')

    def __init__(self, pages, codes, exponent):
        s = pages.struct
        blocks = codes.shape[2] if codes.dim() == 4 else 0
        block = s.page_tokens // blocks if blocks else 0
        if not (codes.dtype == torch.int8 and exponent.dtype == torch.uint8 and codes.is_contiguous() and exponent.is_contiguous()
                and codes.get_device() == pages.index and exponent.get_device() == pages.index and block >= 16
                and block * blocks == s.page_tokens and not block & (block - 1)
                and codes.shape == (s.npage, s.kv_heads, blocks, s.head_dim) and exponent.shape == codes.shape[:3]):
            raise ValueError('summaries must be contiguous codes (npage, kv_heads, blocks of a page, head_dim) int8 and exponent '
                             '(without head_dim) uint8 on the pages\' device, with blocks of 16 tokens at least and a power of two')
        _require(not codes.data_ptr() & 15, 'codes must be 16-byte aligned')
        self.pages, self.codes, self.exponent, self.block_tokens = pages, codes, exponent, block
        self.struct = MxSummaries(codes.data_ptr(), exponent.data_ptr(), block)

    @classmethod
    def make(cls, pages, block_tokens):
        """Empty summaries for pages."""
        s = pages.struct
        _require(16 <= block_tokens <= s.page_tokens and not block_tokens & (block_tokens - 1),
                 'block_tokens must be a power of two from 16 to the pages\' %d, got %s', s.page_tokens, block_tokens)
        shape = (s.npage, s.kv_heads, s.page_tokens // block_tokens, s.head_dim)
        return cls(pages, torch.zeros(shape, dtype=torch.int8, device=pages.device),
                   torch.zeros(shape[:3], dtype=torch.uint8, device=pages.device))


def _held(pages, *others):
    return (pages.k, pages.v, pages.k_scale, pages.v_scale, pages.table, pages.length) + others


def summarise(summaries, start=None, *, count=None, tokens=None, stream=None):
    """The summaries of the blocks that the chunk's tokens complete, from the keys in the pages: the last ``count`` tokens of
    every world, or with ``start`` those of packed rows of ``tokens``.  Sums are in 64 bits; a block with a key that is not
    finite is marked, and then stands above all others, so that it is not passed over in silence."""
    pages = summaries.pages
    if _elsewhere(pages, stream):
        return _on(pages.device, stream, _held(pages, summaries.codes, summaries.exponent, start),
                   lambda: summarise(summaries, start, count=count, tokens=tokens))
    many, none = (count, tokens) if start is None else (tokens, count)
    _require(many is not None and none is None and many >= 0, 'give count (every world), or start and tokens')
    chunk = _chunk(pages, (pages.struct.nworld, count) if start is None else (tokens,), start)
    lib = episodes._LIB or episodes.load()
    rc = lib.mx_episode_summarise(ct.byref(pages.struct), ct.byref(chunk), ct.byref(summaries.struct), _current(pages.index))
    if rc:
        _check(rc, 'mx_episode_summarise')


def select(summaries, q, start=None, *, top, near=1, first=0, causal=True, max_count=None, out=None, stream=None):
    """The blocks that each of the chunk's queries attends to, per key head: int32 of shape (rows..., kv_heads, listed), in
    ascending order, -1 behind the last.

    A query at position p sees the tokens ``j <= p``, or with ``causal=False`` all of its world.  Of the blocks that hold any of
    them it gets the ``first`` ones, those from the ``near``-th up to its own on (``near=1``: its own; and what lies behind it), and of
    those between the ``top`` with the largest score, of equal ones the earlier.  The score is the largest, over the query heads
    of the key head, of the product of the query and the summary, both in 8-bit whole numbers with powers of two.
    ``max_count`` (with ``start``): the largest chunk of a world, if known; rows beyond it get no blocks.  ``listed`` is first +
    near + top, and with ``causal=False`` as many more as the tokens behind a query may need: those of the chunk, or with ``start``
    of ``max_count`` tokens.  Then, in a chunk that is longer all the same, no row's list has room for the last blocks of what it
    sees: they are left out.  ``out`` is written if given."""
    pages = summaries.pages
    if _elsewhere(pages, stream):
        return _on(pages.device, stream, _held(pages, summaries.codes, summaries.exponent, q, start, out),
                   lambda: select(summaries, q, start, top=top, near=near, first=first, causal=causal, max_count=max_count, out=out))
    s, shape = pages.struct, q.shape
    chunk = _chunk(pages, shape[:-2], start)
    rows = _rows(pages, q, shape, 'q')
    _queries(pages, q, rows)
    if max_count is None:
        max_count = chunk.tokens if start is not None else chunk.count
    _require(0 <= max_count < 2 ** 31 and 0 <= top <= MOST_TOP and near >= 1 and first >= 0,
             'max_count and first must not be negative, top at most %d and near at least 1', MOST_TOP)
    listed = first + near + top
    if not causal:                        # the blocks behind a query's own: of the whole chunk, whichever of its rows are left out
        listed += (max(max_count, chunk.count) + summaries.block_tokens - 2) // summaries.block_tokens
    _require(listed <= MOST_LISTED, 'at most %d blocks can be listed, got %d: give max_count, the largest chunk of a world, with start',
             MOST_LISTED, listed)
    shape = shape[:-2] + (s.kv_heads, listed)
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=q.device)
    else:
        _require(out.dtype == torch.int32 and out.shape == shape and out.is_contiguous() and out.get_device() == pages.index,
                 'out must be contiguous int32 of shape %s on the pages\' device', tuple(shape))
    m = MxSelection(out.data_ptr(), listed, top, near, first, max_count, 1 if causal else 0)
    lib = episodes._LIB or episodes.load()
    rc = lib.mx_episode_select(ct.byref(s), ct.byref(chunk), ct.byref(summaries.struct), ct.byref(rows), ct.byref(m),
                               _current(pages.index))
    if rc:
        _check(rc, 'mx_episode_select')
    return out


def _queries(pages, q, rows):
    s = pages.struct
    if not (rows.type == s.type or s.type == 3 and rows.type) or rows.heads < 1 or rows.heads % s.kv_heads:
        _require(rows.heads > 0 and rows.heads % s.kv_heads == 0, 'q has %d heads, not a multiple of the pages\' %d',
                 rows.heads, s.kv_heads)
        raise ValueError('q must be bfloat16 or float16, and of the pages\' type unless those are 8-bit: %s on %s'
                         % (q.dtype, pages.k.dtype))


def recall(pages, q, blocks, start=None, *, block_tokens, max_count=None, causal=True, scale=None, out=None, lse=None, longest=0,
           stream=None):
    """:func:`libero_hip.episodes.attend` over the keys of listed blocks: ``blocks`` (rows..., kv_heads, listed), contiguous
    int32, as :func:`select` returns or by the caller.  Block b holds the tokens from ``b * block_tokens`` on; of those the query sees
    what ``attend`` lets it see.  A block counts as often as it is listed, in any order; numbers that are no block of the
    world's table are left out.  A query that sees nothing gives zeros (and ``lse`` -inf).  ``longest``, as for ``attend``, says how to
    divide the work: without it the table's reach is taken for the worlds' tokens."""
    if _elsewhere(pages, stream):
        return _on(pages.device, stream, _held(pages, q, blocks, start, out, lse),
                   lambda: recall(pages, q, blocks, start, block_tokens=block_tokens, max_count=max_count, causal=causal, scale=scale,
                                  out=out, lse=lse, longest=longest))
    s, shape = pages.struct, q.shape
    chunk = _chunk(pages, shape[:-2], start)
    rows = _rows(pages, q, shape, 'q')
    _queries(pages, q, rows)
    if not (blocks.dtype == torch.int32 and blocks.dim() == len(shape) and blocks.shape[:-1] == shape[:-2] + (s.kv_heads,)
            and 0 < blocks.shape[-1] <= MOST_LISTED and blocks.is_contiguous() and blocks.get_device() == pages.index):
        raise ValueError('blocks must be contiguous int32 of shape (rows..., %d key heads, 1 to %d) on the pages\' device: %s'
                         % (s.kv_heads, MOST_LISTED, tuple(blocks.shape)))
    _require(16 <= block_tokens <= s.page_tokens and not block_tokens & (block_tokens - 1),
             'block_tokens must be a power of two from 16 to the pages\' %d, got %s', s.page_tokens, block_tokens)
    if scale is None:
        scale = s.head_dim ** -0.5
    if max_count is None:
        max_count = chunk.tokens if start is not None else chunk.count
    _require(0 <= max_count < 2 ** 31 and 0 <= longest < 2 ** 31 and math.isfinite(scale),
             'max_count and longest must be numbers of tokens and scale finite: %s, %s, %s', max_count, longest, scale)
    if out is None:
        out = q.new_empty(shape)
        to = MxRows(out.data_ptr(), rows.heads * s.head_dim, s.head_dim, rows.heads, rows.type)
    else:
        to = _rows(pages, _output(q, out), shape, 'out')
    a = MxAttention(rows, to, None, None, 0, max_count, 1 if causal else 0, 0, scale, longest)
    if lse is not None:
        _require(lse.dtype == torch.float32 and lse.shape == shape[:-1] and lse.is_contiguous()
                 and lse.get_device() == pages.index, 'lse must be contiguous float32 of q\'s shape without head_dim')
        a.lse = lse.data_ptr()
    m = MxSelection(blocks.data_ptr(), blocks.shape[-1])
    lib, raw = episodes._LIB or episodes.load(), _current(pages.index)
    refs = ct.byref(s), ct.byref(chunk), ct.byref(a), ct.byref(m), block_tokens
    rc = lib.mx_episode_recall(*refs, raw)
    if rc == ERR_WORKSPACE:               # the keys are split: found before any launch
        need = lib.mx_recall_workspace(*refs)
        workspace = torch.empty(need, dtype=torch.uint8, device=pages.device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
        rc = lib.mx_episode_recall(*refs, raw)
    if rc:
        _check(rc, 'mx_episode_recall')
    return out
