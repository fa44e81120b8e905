"""Episode memory: the keys and values of every world's running episode, and attention over them.

A policy that steps a batch of worlds keeps, per attention layer, the keys and values of the tokens that
each world's episode has brought so far (instruction, observations, actions).  The worlds of a batch share
pages of that memory: worlds differ in how far their episodes are, and a reset gives one world's pages back.

Operators (``include/mx_episode.h``, on the current stream or ``stream``; they can be captured into a HIP
graph, and read ``table``, ``length`` and ``start`` on the device).  ``stream`` does not wait for the current one, nor that for
it: the order is the caller's, as with any stream; tensors that are given may be dropped when the call returns, what it
returns belongs to ``stream``:

* :func:`write` stores a chunk's keys and values in the pages, in 16 bits or quantised to 8;
* :func:`read` returns them as the pages stand for them;
* :func:`attend` attends from the chunk's queries to all tokens of their worlds.

A chunk is the last tokens of each world's ``length``: ``(nworld, n, heads, head_dim)``, the same number
for every world, or packed rows ``(tokens, heads, head_dim)`` with ``start`` (int32, ``nworld + 1``): world
w has the rows ``start[w]:start[w + 1]``.

They are the memory of running episodes and have no backward pass: tensors whose gradients are being recorded, or that
carry a forward-mode tangent, are refused.

:class:`Pages` holds the tensors of one layer; :class:`EpisodeCache` keeps the pages of several layers, the
worlds' tables and lengths, and hands out pages.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as ct
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from . import native

SCALE_BLOCK = 32                      # values along head_dim that share a scale in 8-bit pages
HEAD_DIMS = (32, 64, 96, 128, 256)
ERR_WORKSPACE = -5
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3}
_PAGE_TOKENS = frozenset(1 << i for i in range(4, 13))
STORAGE = {'bf16': torch.bfloat16, 'f16': torch.float16, 'fp8': torch.float8_e4m3fn}

EXPORTS = ['mx_pages_bytes', 'mx_chunk_bytes', 'mx_rows_bytes', 'mx_attention_bytes', 'mx_episode_write',
           'mx_episode_read', 'mx_episode_attend', 'mx_episode_workspace',
           'mx_rotary_bytes', 'mx_rotate', 'mx_episode_enter',
           'mx_room_bytes', 'mx_room_change_bytes', 'mx_room_workspace', 'mx_room_update', 'mx_room_places',
           'mx_summaries_bytes', 'mx_selection_bytes', 'mx_episode_summarise', 'mx_episode_select', 'mx_episode_recall',
           'mx_recall_workspace']


class MxPages(ct.Structure):
    _fields_ = ([(n, ct.c_void_p) for n in ('k', 'v', 'k_scale', 'v_scale', 'table', 'length')]
                + [(n, ct.c_int32) for n in ('nworld', 'npage', 'width', 'kv_heads', 'head_dim', 'page_tokens', 'type')])


class MxChunk(ct.Structure):
    _fields_ = [('start', ct.c_void_p), ('tokens', ct.c_int32), ('count', ct.c_int32)]


class MxRows(ct.Structure):
    _fields_ = [('data', ct.c_void_p), ('token_stride', ct.c_int64), ('head_stride', ct.c_int64),
                ('heads', ct.c_int32), ('type', ct.c_int32)]


class MxAttention(ct.Structure):
    _fields_ = [('q', MxRows), ('out', MxRows), ('lse', ct.c_void_p), ('workspace', ct.c_void_p),
                ('workspace_bytes', ct.c_size_t), ('max_count', ct.c_int32), ('causal', ct.c_int32),
                ('window', ct.c_int32), ('scale', ct.c_float), ('longest', ct.c_int32)]


class MxRotary(ct.Structure):
    _fields_ = [('turn', ct.c_void_p), ('width', ct.c_int32), ('interleaved', ct.c_int32), ('amplitude', ct.c_double)]


class MxRoom(ct.Structure):
    _fields_ = ([(n, ct.c_void_p) for n in ('table', 'length', 'free', 'state')]
                + [(n, ct.c_int32) for n in ('nworld', 'width', 'npage', 'page_tokens', 'tokens')])


class MxRoomChange(ct.Structure):
    _fields_ = [('count', ct.c_void_p), ('over', ct.c_void_p), ('start', ct.c_void_p), ('workspace', ct.c_void_p),
                ('workspace_bytes', ct.c_size_t), ('each', ct.c_int32), ('rows', ct.c_int32)]


class MxSummaries(ct.Structure):
    _fields_ = [('codes', ct.c_void_p), ('exponent', ct.c_void_p), ('block_tokens', ct.c_int32)]


class MxSelection(ct.Structure):
    _fields_ = [('blocks', ct.c_void_p)] + [(n, ct.c_int32) for n in ('width', 'top', 'near', 'first', 'max_count', 'causal')]


_LIB = None


def load():
    """The library, with the episode memory's entry points bound and their structs' sizes checked."""
    global _LIB
    if _LIB is None:
        lib = native.load()
        for name, struct in (('pages', MxPages), ('chunk', MxChunk), ('rows', MxRows), ('attention', MxAttention),
                             ('rotary', MxRotary), ('room', MxRoom), ('room_change', MxRoomChange),
                             ('summaries', MxSummaries), ('selection', MxSelection)):
            f = getattr(lib, 'mx_%s_bytes' % name)
            f.restype = ct.c_size_t
            if f() != ct.sizeof(struct):
                raise ImportError('libmx_physics struct sizes differ from the Python mirror')
        lib.mx_episode_write.argtypes = lib.mx_episode_read.argtypes = [ct.c_void_p] * 5
        lib.mx_episode_attend.argtypes = [ct.c_void_p] * 4
        lib.mx_episode_workspace.argtypes = [ct.c_void_p] * 3
        lib.mx_episode_workspace.restype = ct.c_size_t
        lib.mx_rotate.argtypes = [ct.c_void_p] * 3 + [ct.c_int32] * 2 + [ct.c_void_p] + [ct.c_int32] * 3 + [ct.c_void_p]
        lib.mx_episode_enter.argtypes = [ct.c_void_p] * 8
        lib.mx_room_workspace.argtypes = [ct.c_void_p]
        lib.mx_room_update.argtypes = [ct.c_void_p] * 3
        lib.mx_room_places.argtypes = [ct.c_void_p] * 6
        lib.mx_episode_summarise.argtypes = [ct.c_void_p] * 4
        lib.mx_episode_select.argtypes = [ct.c_void_p] * 6
        lib.mx_episode_recall.argtypes = [ct.c_void_p] * 4 + [ct.c_int32, ct.c_void_p]
        lib.mx_recall_workspace.argtypes = [ct.c_void_p] * 4 + [ct.c_int32]
        lib.mx_room_workspace.restype = lib.mx_recall_workspace.restype = ct.c_size_t
        _LIB = lib
    return _LIB


def _require(ok, message, *args):
    if not ok:
        raise ValueError(message % args)


_REFUSED = {-1: 'arguments that do not fit', -2: 'sizes beyond its range (1024 query heads to a key head, 2^24 - 1 workgroups)'}


def _check(rc, what):
    """ValueError for what the library refuses, which it finds before any launch; RuntimeError for a failed launch."""
    if rc < 0:
        raise ValueError('%s: %s (%d)' % (what, _REFUSED.get(rc) or load().mx_error_string(rc).decode(), rc))
    native.check(rc, what)


class Pages:
    """One layer's pages and the worlds' tables into them.

    ``k``, ``v``: (npage, kv_heads, page_tokens, head_dim), bfloat16, float16, or float8_e4m3fn with
    ``k_scale``, ``v_scale``: (npage, kv_heads, page_tokens, head_dim / 32) uint8, the exponent of each
    block's scale (2^(byte - 127); 255: the block is NaN).  ``table``: (nworld, pages of a world) int32, token t of world w is in
    page ``table[w, t // page_tokens]``; ``length``: (nworld,) int32, the worlds' tokens.  page_tokens is a power
    of two from 16 to 4096, head_dim one of 32, 64, 96, 128, 256.  The tensors stay the caller's, and are
    held here."""

    __slots__ = ('k', 'v', 'table', 'length', 'k_scale', 'v_scale', 'struct', 'index')

    def __init__(self, k, v, table, length, k_scale=None, v_scale=None):
        # one condition for what is as it should be; what is not is named by _refuse_pages
        shape, tables, kind, index = k.shape, table.shape, _TYPES.get(k.dtype, 0), k.get_device()
        if not (kind and index >= 0 and len(shape) == 4 and len(tables) == 2 and v.shape == shape and v.dtype == k.dtype
                and shape[3] in HEAD_DIMS and shape[2] in _PAGE_TOKENS and shape[0] > 0 and 0 < shape[1] <= 1024
                and tables[0] > 0 and tables[1] > 0 and length.shape == tables[:1]
                and table.dtype == torch.int32 and length.dtype == torch.int32
                and shape[0] * shape[2] < 2 ** 31 and tables[1] * shape[2] <= 2 ** 30
                and v.get_device() == index and table.get_device() == index and length.get_device() == index
                and k.is_contiguous() and v.is_contiguous() and table.is_contiguous() and length.is_contiguous()
                and (k_scale is None and v_scale is None) == (kind != 3)):
            _refuse_pages(k, v, table, length, k_scale, v_scale)
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            raise ValueError('pages: the episode memory has no backward pass; give it detached tensors')
        at_k, at_v = k.data_ptr(), v.data_ptr()
        _require(not (at_k | at_v) & 15, 'pages must be 16-byte aligned')
        scale_k = scale_v = None
        if kind == 3:
            scales = shape[:3] + (shape[3] // SCALE_BLOCK,)
            for x in (k_scale, v_scale):
                if x is None or x.dtype != torch.uint8 or x.shape != scales or not x.is_contiguous() or x.get_device() != index:
                    raise ValueError('8-bit pages need contiguous uint8 scales of shape %s on their device' % (tuple(scales),))
            scale_k, scale_v = k_scale.data_ptr(), v_scale.data_ptr()
        self.k, self.v, self.table, self.length, self.k_scale, self.v_scale = k, v, table, length, k_scale, v_scale
        self.index = index
        self.struct = MxPages(at_k, at_v, scale_k, scale_v, table.data_ptr(), length.data_ptr(), tables[0], shape[0],
                              tables[1], shape[1], shape[3], shape[2], kind)

    @property
    def device(self):
        return self.k.device


def _refuse_pages(k, v, table, length, k_scale, v_scale):
    _require(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype,
             'k and v pages must have one shape (npage, kv_heads, page_tokens, head_dim) and type')
    _require(_TYPES.get(k.dtype, 0) > 0, 'pages must be bfloat16, float16 or float8_e4m3fn, got %s', k.dtype)
    npage, kv, tokens, dim = k.shape
    _require(dim in HEAD_DIMS, 'head_dim must be one of %s, got %d', HEAD_DIMS, dim)
    _require(tokens in _PAGE_TOKENS, 'page_tokens must be a power of two from 16 to 4096, got %d', tokens)
    _require(npage > 0 and 0 < kv <= 1024, 'pages need at least one page and 1 to 1024 heads')
    _require(table.dim() == 2 and table.dtype == torch.int32 and table.is_contiguous() and table.numel() > 0,
             'table must be contiguous int32 of shape (nworld, pages of a world)')
    _require(length.dtype == torch.int32 and length.shape == table.shape[:1] and length.is_contiguous(),
             'length must be contiguous int32 of shape (nworld,)')
    _require(npage * tokens < 2 ** 31 and table.shape[1] * tokens <= 2 ** 30,
             'npage * page_tokens must be below 2^31 and the tokens of a table row at most 2^30')
    _require(k.is_contiguous() and v.is_contiguous(), 'pages must be contiguous')
    _require((k_scale is None) == (v_scale is None) == (k.dtype != torch.float8_e4m3fn),
             '8-bit pages have scales for k and v, others have none')
    raise ValueError('pages, table and length must be on one GPU')


def _chunk(pages, shape, start):
    """MxChunk of rows of this shape (without heads and head_dim)."""
    nworld = pages.struct.nworld
    if start is None:
        if len(shape) != 2 or shape[0] != nworld:
            raise ValueError('rows must be (nworld, n, heads, head_dim), or packed (tokens, heads, head_dim) with start')
        _require(nworld * shape[1] < 2 ** 31, 'a chunk has fewer than 2^31 rows: %d worlds of %d', nworld, shape[1])
        return MxChunk(None, nworld * shape[1], shape[1])
    _require(len(shape) == 1, 'rows with start must be packed: (tokens, heads, head_dim)')
    _require(start.dtype == torch.int32 and start.shape == (nworld + 1,) and start.is_contiguous()
             and start.get_device() == pages.index, 'start must be contiguous int32 of shape (nworld + 1,) on the pages\' device')
    _require(shape[0] < 2 ** 31, 'a chunk has fewer than 2^31 rows: %d', shape[0])
    return MxChunk(start.data_ptr(), shape[0], 0)


def _rows(pages, x, shape, name):
    """MxRows of a tensor (..., heads, head_dim) whose token dimensions step evenly."""
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError('%s: the episode memory has no backward pass; call it under torch.no_grad() or on a detached tensor' % name)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError('%s: the episode memory has no derivatives; give it the primal of a dual tensor' % name)
    kind = _TYPES.get(x.dtype, 3)
    stride = x.stride()
    if kind == 3 or shape[-1] != pages.struct.head_dim or x.get_device() != pages.index or stride[-1] != 1:
        _require(kind < 3, '%s must be float32, bfloat16 or float16, got %s', name, x.dtype)
        _require(shape[-1] == pages.struct.head_dim, '%s has the wrong head_dim: %s', name, tuple(shape))
        _require(x.get_device() == pages.index, '%s must be on the pages\' device', name)
        _require(stride[-1] == 1, '%s must be contiguous along head_dim', name)
    token = stride[-3]
    if len(shape) == 4:
        if shape[1] == 1:
            token = stride[0]
        elif shape[0] > 1 and shape[1] > 1 and stride[0] != shape[1] * token:
            raise ValueError('%s: the rows of all worlds must step evenly' % name)
    return MxRows(x.data_ptr(), token, stride[-2], shape[-2], kind)


# the current stream's handle, without a Stream object around it where torch offers that
_current = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _elsewhere(pages, stream):
    """Whether a call has to change to the pages' device, or to a stream that is not the current one."""
    return stream is not None or torch.cuda.current_device() != pages.index


def _there(call, pages, stream, tensors, *args, **options):
    """``call`` on the pages' device and on ``stream``, which then holds the memory of what it was given: a caller may
    drop a tensor as soon as the call returns, long before ``stream`` comes to read it."""
    _require(stream is None or stream.device == pages.device, 'stream must be on the pages\' device')
    with torch.cuda.device(pages.device), torch.cuda.stream(stream):
        result = call(pages, *args, **options)
        if stream is not None:
            for x in (pages.k, pages.v, pages.k_scale, pages.v_scale, pages.table, pages.length) + tensors:
                if x is not None:
                    x.record_stream(stream)
    return result


def _on(device, stream, tensors, call):
    """``call()`` on a device and a stream, as :func:`_there`."""
    _require(stream is None or stream.device == device, 'stream must be on the tensors\' device')
    with torch.cuda.device(device), torch.cuda.stream(stream):
        result = call()
        if stream is not None:
            for x in tensors:
                if x is not None:
                    x.record_stream(stream)
    return result


def _overlap(a, b):
    """Whether the memory from a tensor's first element to its last meets another's."""
    if not a.numel() or not b.numel():
        return False
    first, second = a.data_ptr(), b.data_ptr()
    reach = [x.element_size() * (1 + sum((n - 1) * step for n, step in zip(x.shape, x.stride()))) for x in (a, b)]
    return first < second + reach[1] and second < first + reach[0]


def _output(like, out):
    """``out``, given for rows like ``like``, once it is checked."""
    _require(out.shape == like.shape and out.dtype == like.dtype, 'out must have the rows\' shape and type')
    _require(all(step or n < 2 for n, step in zip(like.shape, out.stride())), 'out has elements that share memory')
    return out


def write(pages, k, v, start=None, *, stream=None):
    """Store the chunk's keys and values (float32, bfloat16 or float16; any strides whose tokens step evenly
    and whose head_dim is contiguous).  8-bit pages take, per 32 values along head_dim, the least power of two
    at which all are within the codes' range, and round to nearest even; a block with an infinity or NaN
    is stored as NaN.  Chunk tokens without a place (a chunk longer than its world's length, a table entry
    that names no page) are left out."""
    if _elsewhere(pages, stream):
        return _there(write, pages, stream, (k, v, start), k, v, start)
    s, shape = pages.struct, k.shape
    if shape != v.shape or k.dtype != v.dtype or len(shape) < 3 or shape[-2] != s.kv_heads:
        raise ValueError('k and v must have one type and one shape, with %d heads: %s, %s' % (s.kv_heads, tuple(shape), tuple(v.shape)))
    chunk = _chunk(pages, shape[:-2], start)
    a, b = _rows(pages, k, shape, 'k'), _rows(pages, v, shape, 'v')
    rc = load().mx_episode_write(ct.byref(s), ct.byref(chunk), ct.byref(a), ct.byref(b), _current(pages.index))
    if rc:
        _check(rc, 'mx_episode_write')


def read(pages, start=None, *, count=None, tokens=None, dtype=torch.bfloat16, stream=None):
    """The chunk's keys and values: ``(nworld, count, kv_heads, head_dim)``, or packed ``(tokens, kv_heads,
    head_dim)`` with ``start``; each value rounded once to ``dtype``.  Tokens without a place read as zeros."""
    if _elsewhere(pages, stream):
        return _there(read, pages, stream, (start,), start, count=count, tokens=tokens, dtype=dtype)
    s = pages.struct
    kind = _TYPES.get(dtype, 3)
    _require(kind < 3, 'read returns float32, bfloat16 or float16')
    many, none = (count, tokens) if start is None else (tokens, count)
    _require(many is not None and none is None and many >= 0, 'give count (every world), or start and tokens')
    shape = (s.nworld, count) if start is None else (tokens,)
    chunk = _chunk(pages, shape, start)
    shape += (s.kv_heads, s.head_dim)
    k = torch.empty(shape, dtype=dtype, device=pages.device)
    v = torch.empty_like(k)
    step = s.kv_heads * s.head_dim
    a, b = (MxRows(x.data_ptr(), step, s.head_dim, s.kv_heads, kind) for x in (k, v))
    rc = load().mx_episode_read(ct.byref(s), ct.byref(chunk), ct.byref(a), ct.byref(b), _current(pages.index))
    if rc:
        _check(rc, 'mx_episode_read')
    return k, v


def attend(pages, q, start=None, *, max_count=None, causal=True, window=0, scale=None, out=None, lse=None,
           longest=0, stream=None):
    """Softmax attention of the chunk's queries over their worlds' tokens, with scores and sums in 32 bits; the
    probabilities that multiply the values are rounded to q's type, in two parts for few rows and in one for many (see
    ``include/mx_episode.h``).

    Query head h uses key head ``h // (heads / kv_heads)``.  The query at position p (of its world's tokens)
    sees the tokens ``j <= p``, or with ``causal=False`` all of them (a step's tokens see each other), and
    with ``window`` > 0 only those with ``j > p - window``.  ``scale``: 1 / sqrt(head_dim) by default.  A query
    that sees nothing gives zeros (and ``lse`` -inf).  ``q`` is bfloat16 or float16, the pages' type unless
    those are 8-bit.  ``max_count`` (with ``start``): the largest chunk of a world, if known; rows beyond it are
    not computed.  ``longest``: the most tokens that a world has, if known; it says how to divide the work, and worlds that
    are longer all the same only take longer.  ``out`` (like q) and ``lse`` (float32, q's shape without head_dim, contiguous) are written
    if given.  Returns out.  The same inputs give the same bits."""
    if _elsewhere(pages, stream):
        return _there(attend, pages, stream, (q, start, out, lse), q, start, max_count=max_count, causal=causal, window=window,
                      scale=scale, out=out, lse=lse, longest=longest)
    s, shape = pages.struct, q.shape
    chunk = _chunk(pages, shape[:-2], start)
    rows = _rows(pages, q, shape, 'q')
    if not (rows.type == s.type or s.type == 3 and rows.type) or rows.heads < 1 or rows.heads % s.kv_heads:
        _require(rows.heads > 0 and rows.heads % s.kv_heads == 0, 'q has %d heads, not a multiple of the pages\' %d',
                 rows.heads, s.kv_heads)
        raise ValueError('q must be bfloat16 or float16, and of the pages\' type unless those are 8-bit: %s on %s'
                         % (q.dtype, pages.k.dtype))
    if scale is None:
        scale = s.head_dim ** -0.5
    if max_count is None:
        max_count = chunk.tokens if start is not None else chunk.count
    if not (0 <= window < 2 ** 31 and 0 <= max_count < 2 ** 31 and 0 <= longest < 2 ** 31 and math.isfinite(scale)):
        raise ValueError('window (0: none), max_count and longest must be numbers of tokens and scale finite: %s, %s, %s, %s'
                         % (window, max_count, longest, scale))
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _require(out.shape == shape and out.dtype == q.dtype, 'out must have q\'s shape and type')
        _require(all(step or n < 2 for n, step in zip(shape, out.stride())), 'out has elements that share memory')
    a = MxAttention(rows, _rows(pages, out, shape, 'out'), None, None, 0, max_count, 1 if causal else 0, window, scale,
                    longest)
    if lse is not None:
        _require(lse.dtype == torch.float32 and lse.shape == shape[:-1] and lse.is_contiguous()
                 and lse.get_device() == pages.index, 'lse must be contiguous float32 of q\'s shape without head_dim')
        a.lse = lse.data_ptr()
    lib, refs, raw = _LIB or load(), (ct.byref(s), ct.byref(chunk), ct.byref(a)), _current(pages.index)
    rc = lib.mx_episode_attend(*refs, raw)
    if rc == ERR_WORKSPACE:               # the keys are split: found before any launch
        need = lib.mx_episode_workspace(*refs)
        workspace = torch.empty(need, dtype=torch.uint8, device=pages.device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
        rc = lib.mx_episode_attend(*refs, raw)
    if rc:
        _check(rc, 'mx_episode_attend')
    return out


def _captured(stream):
    """Whether what is put on this stream (None: the current one) goes into a graph."""
    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


class Chunk:
    """New tokens of an :class:`EpisodeCache`: of all its worlds the same number (``start`` None; rows are
    ``(nworld, count, heads, head_dim)``), or ``counts[w]`` of world w (rows ``(tokens, heads, head_dim)``, packed
    world by world, ``start`` on the device).  ``longest``: the most tokens that a world had with them."""

    __slots__ = ('counts', 'tokens', 'count', 'start', 'longest')

    def __init__(self, counts, start, longest=0):
        self.counts, self.start, self.longest = counts, start, longest
        self.tokens, self.count = int(counts.sum()), int(counts.max())

    @property
    def shape(self):
        """The rows' leading shape."""
        return (self.tokens,) if self.start is not None else (len(self.counts), self.count)


class Layers:
    """The pages of several layers, the worlds' tables and lengths, and the calls on them: what caches share whatever keeps
    their books.  See :class:`EpisodeCache`."""

    def __init__(self, nworld, *, kv_heads, head_dim, tokens, layers=1, storage='fp8', page_tokens=64, pages=None,
                 device='cuda:0', block_tokens=None):
        _require(storage in STORAGE, 'storage must be one of %s, got %s', sorted(STORAGE), storage)
        _require(nworld > 0 and tokens > 0 and layers > 0 and kv_heads > 0, 'nworld, tokens, layers and kv_heads must be positive')
        _require(head_dim in HEAD_DIMS, 'head_dim must be one of %s, got %s', HEAD_DIMS, head_dim)
        _require(16 <= page_tokens <= 4096 and not page_tokens & (page_tokens - 1),
                 'page_tokens must be a power of two from 16 to 4096, got %s', page_tokens)
        width = -(-tokens // page_tokens)
        pages = nworld * width if pages is None else int(pages)
        _require(pages > 0, 'pages must be positive, got %s', pages)
        device = torch.device(device)
        if device.type == 'cuda' and device.index is None:
            device = torch.device('cuda', torch.cuda.current_device())
        self.nworld, self.tokens, self.page_tokens, self.device, self.pages = nworld, int(tokens), page_tokens, device, pages
        self.table = torch.full((nworld, width), -1, dtype=torch.int32, device=device)
        self.length = torch.zeros(nworld, dtype=torch.int32, device=device)
        shape = (pages, kv_heads, page_tokens, head_dim)
        self.layers = []
        for _ in range(layers):
            k, v = (torch.empty(shape, dtype=STORAGE[storage], device=device) for _ in range(2))
            scales = [torch.empty(shape[:3] + (head_dim // SCALE_BLOCK,), dtype=torch.uint8, device=device)
                      for _ in range(2 if storage == 'fp8' else 0)]
            self.layers.append(Pages(k, v, self.table, self.length, *scales))
        self.summaries = None
        if block_tokens is not None:
            from . import recall
            self.summaries = [recall.Summaries.make(x, block_tokens) for x in self.layers]
        # the stream of the last change and its handle; once calls come from others too, an event after that change and
        # after the last call of each
        self._home, self._handle, self._changed, self._used = None, 0, None, {}
        if device.type == 'cuda':
            self._change()

    def _change(self):
        """Before table and length change: the current stream waits for the calls that read them elsewhere."""
        if self.device.type != 'cuda' or self._home is not None and not self._used and _current(self.device.index) == self._handle:
            return
        stream = torch.cuda.current_stream(self.device)
        for handle, event in self._used.items():
            if handle != stream.cuda_stream:
                stream.wait_event(event)
        self._used.clear()
        if self._home is not None and self._handle != stream.cuda_stream:
            stream.wait_stream(self._home)
        self._home, self._handle = stream, stream.cuda_stream

    def _change_done(self):
        if self._changed is not None:
            self._changed.record(self._home)

    def _enter(self, stream, start=None):
        """The stream of a call if that is not the last change's, for which it then waits."""
        if (_current(self.device.index) if stream is None else stream.cuda_stream) == self._handle:
            return None
        _require(stream is None or stream.device == self.device, 'stream must be on the cache\'s device')
        stream = torch.cuda.current_stream(self.device) if stream is None else stream
        if _captured(stream):
            return None
        if self._changed is None:
            self._changed = self._home.record_event()
        stream.wait_event(self._changed)
        if start is not None:
            start.record_stream(stream)
        return stream

    def _leave(self, stream):
        if stream is not None:
            event = self._used.get(stream.cuda_stream) or torch.cuda.Event()
            event.record(stream)
            self._used[stream.cuda_stream] = event

    def _ids(self, id):
        ids = np.arange(self.nworld) if id is None else np.atleast_1d(np.asarray(id, np.int64))
        if ids.ndim != 1 or np.any((ids < 0) | (ids >= self.nworld)) or len(np.unique(ids)) != len(ids):
            raise ValueError('invalid world ids')
        return ids

    @staticmethod
    def _packed(chunk, x, behind=2, stream=None):
        """Rows in the shape that the chunk's start wants; ``behind``: the dimensions of a row.  Only a chunk of which every
        world has the same number may come as (nworld, count, ...): of a ragged one such rows would be padded.  Rows that do
        not step evenly are copied, on the stream of the call."""
        if chunk.start is None or x.dim() == 1 + behind:
            return x
        _require(len(chunk.shape) == 2, 'rows of a ragged chunk must be packed: (tokens, heads, head_dim), got %s', tuple(x.shape))
        _require(x.dim() == 2 + behind and x.shape[:2] == chunk.shape, 'rows must be packed, or of shape (%d, %d, heads, head_dim), got %s',
                 *chunk.shape, tuple(x.shape))
        if stream is None:
            return x.flatten(0, 1)
        with torch.cuda.stream(stream):
            packed = x.flatten(0, 1)
        if packed.data_ptr() != x.data_ptr():
            x.record_stream(stream)
        return packed

    @staticmethod
    def _bounds(chunk, stream, options, *names):
        """What is known of the chunk, where replays of a captured call could not come with longer worlds, and larger
        chunks."""
        if getattr(chunk, 'bounded', False) or not _captured(stream):
            if chunk.start is not None:
                options.setdefault('max_count', chunk.count)
            if 'longest' in names:
                options.setdefault('longest', chunk.longest)

    def _summarise(self, chunk, layer, stream):
        if self.summaries is not None:
            from . import recall
            given = dict(count=chunk.count) if chunk.start is None else dict(tokens=chunk.tokens)
            recall.summarise(self.summaries[layer], chunk.start, stream=stream, **given)

    def write(self, chunk, k, v, layer=0, *, stream=None):
        """:func:`write` of the chunk's keys and values to a layer, and the summaries of the blocks that they complete."""
        other = self._enter(stream, chunk.start)
        k, v = (self._packed(chunk, x, stream=stream) for x in (k, v))
        write(self.layers[layer], k, v, chunk.start, stream=stream)
        self._summarise(chunk, layer, stream)
        self._leave(other)

    def enter(self, chunk, rotary, q, k, v, layer=0, *, out=None, stream=None):
        """:func:`libero_hip.rotary.enter` of the chunk's rows to a layer, as :meth:`write`; returns the queries, turned."""
        from . import rotary as operators
        other = self._enter(stream, chunk.start)
        given = None if out is None else self._packed(chunk, out)
        _require(given is None or given.data_ptr() == out.data_ptr(), 'out: the rows of all worlds must step evenly')
        shape, (q, k, v) = q.shape, (self._packed(chunk, x, stream=stream) for x in (q, k, v))
        turned = operators.enter(self.layers[layer], rotary, q, k, v, chunk.start, out=given, stream=stream)
        self._summarise(chunk, layer, stream)
        self._leave(other)
        return turned.view(shape) if out is None else out

    def attend(self, chunk, q, layer=0, **options):
        """:func:`attend` from the chunk's queries to a layer; options as there.  ``max_count`` and ``longest`` are the chunk's
        own, but not in a call that is captured: replays follow ``length`` and ``start``, whatever sizes they then have."""
        stream = options.get('stream')
        other = self._enter(stream, chunk.start)
        self._bounds(chunk, stream, options, 'longest')
        out = self._attended(chunk, q, options, lambda x: attend(self.layers[layer], x, chunk.start, **options))
        self._leave(other)
        return out

    def recall(self, chunk, q, layer=0, *, top, near=1, first=0, **options):
        """:func:`libero_hip.recall.select` of blocks for the chunk's queries and :func:`libero_hip.recall.recall` of them: attention
        whose cost does not grow with the episode.  The cache has to be made with ``block_tokens``.  ``max_count`` and ``longest`` as
        in :meth:`attend`; ``scale`` must not be negative, as the blocks of the largest scores are chosen."""
        from . import recall
        _require(self.summaries is not None, 'the cache has no summaries: make it with block_tokens')
        _require(options.get('scale') is None or options['scale'] >= 0, 'scale must not be negative, got %s', options.get('scale'))
        stream = options.get('stream')
        other = self._enter(stream, chunk.start)
        self._bounds(chunk, stream, options, 'longest')
        both = {x: options[x] for x in ('causal', 'max_count', 'stream') if x in options}

        def call(x):
            blocks = recall.select(self.summaries[layer], x, chunk.start, top=top, near=near, first=first, **both)
            return recall.recall(self.layers[layer], x, blocks, chunk.start, block_tokens=self.summaries[layer].block_tokens, **options)

        out = self._attended(chunk, q, options, call)
        self._leave(other)
        return out

    def _attended(self, chunk, q, options, call):
        """A call with queries, ``out`` and ``lse`` in the shape that the chunk's start wants, and its result in q's."""
        x = self._packed(chunk, q, stream=options.get('stream'))
        if x is q:
            return call(q)
        given = options.get('out')
        for name, behind in (('out', 2), ('lse', 1)):
            if options.get(name) is not None:
                y = self._packed(chunk, options[name], behind)
                _require(y.data_ptr() == options[name].data_ptr(), '%s: the rows of all worlds must step evenly', name)
                options[name] = y
        out = call(x)
        return given if given is not None else out.view(q.shape)

    def read(self, id=None, layer=0, *, dtype=torch.bfloat16, stream=None):
        """The keys and values of the worlds ``id`` (all by default) as a layer stands for them, packed in the order of
        the worlds, and the rows' starts (numpy, one more than ids): ``(k, v, starts)``."""
        ids = np.sort(self._ids(id))
        counts = np.zeros(self.nworld, np.int64)
        counts[ids] = self.lengths[ids]
        start = np.concatenate([[0], np.cumsum(counts)])
        other = self._enter(stream)
        k, v = read(self.layers[layer], torch.from_numpy(start.astype(np.int32)).to(self.device), tokens=int(start[-1]),
                    dtype=dtype, stream=stream)
        self._leave(other)
        return k, v, np.concatenate([start[ids], start[-1:]])


class EpisodeCache(Layers):
    """The episode memory of a batch of worlds, for a policy of ``layers`` attention layers, with its books on the host
    (:class:`libero_hip.room.DeviceEpisodeCache`: on the device).

    ``tokens``: the most tokens of one world.  ``pages``: how many pages of ``page_tokens`` tokens all worlds
    share (by default enough for every world at its longest; worlds in different phases of their episodes do
    with about half).  ``storage``: 'fp8' (quantised, a scale per 32 values), 'bf16' or 'f16'.

    ``block_tokens``: blocks of so many tokens are summarised as they are written, for :meth:`recall`.

    Each step, :meth:`extend` makes room for the new tokens; then, layer by layer, :meth:`write` (with positions:
    :meth:`enter`) stores their keys and values and :meth:`attend` (over long episodes: :meth:`recall`) attends from their
    queries.  :meth:`reset` empties worlds, as ``HipBatchEnv.reset(id)`` restarts them.  Tables and lengths live on the device (``table``, ``length``), with a
    copy on the host (``lengths``) that room is made by; pages are not cleared, their old contents are never read.

    :meth:`extend` and :meth:`reset` work on the current stream.  Calls on another one (``stream=``, or the current one then)
    wait for the last of them, and the next of them waits for those calls.  Calls among each other (:meth:`write` on one
    stream, :meth:`attend` on another) and their tensors are the caller's to order, and so are replays of a graph."""

    def __init__(self, nworld, *, kv_heads, head_dim, tokens, layers=1, storage='fp8', page_tokens=64, pages=None,
                 device='cuda:0', block_tokens=None):
        super().__init__(nworld, kv_heads=kv_heads, head_dim=head_dim, tokens=tokens, layers=layers, storage=storage,
                         page_tokens=page_tokens, pages=pages, device=device, block_tokens=block_tokens)
        pages, width = self.pages, self.table.shape[1]
        self.lengths = np.zeros(nworld, np.int64)
        self._table = np.full((nworld, width), -1, np.int32)
        self._free = np.arange(pages - 1, -1, -1, dtype=np.int32)     # a stack; its first _left are free
        self._left = pages

    @property
    def free_pages(self):
        return self._left

    def extend(self, count=1, id=None):
        """Makes room for ``count`` (a number, or one for each world of ``id``) new tokens of the worlds ``id`` (all by
        default) and returns their :class:`Chunk`.  Raises ValueError where a world would pass ``tokens`` and RuntimeError
        when the pages do not suffice; nothing has changed then."""
        ids = self._ids(id)
        new = np.broadcast_to(np.asarray(count, np.int64), ids.shape)
        _require(not np.any(new < 0), 'count must not be negative')
        before = self.lengths[ids]
        _require(not np.any(before + new > self.tokens), 'a world would hold more than %d tokens', self.tokens)
        first, last = -(-before // self.page_tokens), -(-(before + new) // self.page_tokens)
        need = last - first
        total = int(need.sum())
        if total > self._left:
            raise RuntimeError('episode memory: %d more pages needed, %d free' % (total, self._left))
        self._change()
        if total:
            world = np.repeat(ids, need)
            slot = np.repeat(first, need) + np.arange(total) - np.repeat(np.cumsum(need) - need, need)
            page = self._free[self._left - total:self._left][::-1].copy()
            self._left -= total
            self._table[world, slot] = page
            where = torch.from_numpy(world * self._table.shape[1] + slot).to(self.device)
            self.table.view(-1)[where] = torch.from_numpy(page).to(self.device)
        self.lengths[ids] += new
        longest = int(self.lengths.max())
        counts = np.zeros(self.nworld, np.int64)
        counts[ids] = new
        if len(ids) and len(ids) == self.nworld and np.all(new == new[0]):
            if new[0]:
                self.length.add_(int(new[0]))
            self._change_done()
            return Chunk(counts, None, longest)
        both = np.zeros(2 * self.nworld + 1, np.int32)                # one upload: the chunk's starts, the lengths
        both[1:self.nworld + 1] = np.cumsum(counts)
        both[self.nworld + 1:] = self.lengths
        both = torch.from_numpy(both).to(self.device)
        self.length.copy_(both[self.nworld + 1:])
        self._change_done()
        return Chunk(counts, both[:self.nworld + 1], longest)

    def reset(self, id=None):
        """Empties the worlds ``id`` (all by default); their pages are free again."""
        ids = self._ids(id)
        if not len(ids):
            return
        rows = self._table[ids]
        pages = rows[rows >= 0]
        self._free[self._left:self._left + len(pages)] = pages
        self._left += len(pages)
        self._table[ids] = -1
        self.lengths[ids] = 0
        self._change()
        where = torch.from_numpy(ids).to(self.device)
        self.table[where] = -1
        self.length[where] = 0
        self._change_done()
