"""Rotary positions: the pairs of a head's values turn by their row's place in the episode.

A row at position p has pair i of the first ``width`` values of each head turned by ``p * turn[i]`` (and multiplied by an
amplitude), so that the product of a query and a key depends on how far apart they are:

* :func:`rotate` turns rows by given positions; it can be differentiated, for training over whole episodes;
* :func:`enter` turns a chunk's queries and keys by their places in their worlds, and stores the keys, turned, and the values
  in the pages: one launch in the place of three in a policy's step.

:class:`Rotary` holds the angles.  The operators run on the current stream or ``stream``, as those of
:mod:`libero_hip.episodes`, and can be captured into a HIP graph.  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as ct
import math

import torch
from torch.autograd import forward_ad

from . import episodes
from .episodes import MxRotary, MxRows, _TYPES, _check, _chunk, _current, _elsewhere, _on, _output, _overlap, _require, _rows

LAYOUTS = ('half', 'interleaved')
SCALINGS = (None, 'linear', 'base', 'parts')


class Rotary:
    """How far each pair turns from one position to the next: ``turn`` (float64, one to a pair, on the GPU), in radians.

    ``layout``: pair i is the values (i, i + width / 2) of a head ('half'), or (2 i, 2 i + 1) ('interleaved'), with width
    twice the number of pairs; a head's values from ``width`` on do not turn.  ``amplitude`` multiplies the values that do.
    :meth:`make` computes the angles.  The tensor stays the caller's, and is held here."""

    __slots__ = ('turn', 'layout', 'amplitude', 'struct', 'index')

    def __init__(self, turn, *, layout='half', amplitude=1.0):
        if not (turn.dtype == torch.float64 and turn.dim() == 1 and turn.is_contiguous() and turn.get_device() >= 0
                and 0 < turn.shape[0] <= 512 and layout in LAYOUTS and math.isfinite(amplitude)):
            _require(layout in LAYOUTS, 'layout must be one of %s, got %s', LAYOUTS, layout)
            _require(math.isfinite(amplitude), 'amplitude must be finite, got %s', amplitude)
            raise ValueError('turn must be contiguous float64 of 1 to 512 angles on a GPU')
        _require(not turn.requires_grad, 'turn is not learned; give it detached')
        self.turn, self.layout, self.amplitude, self.index = turn, layout, float(amplitude), turn.get_device()
        self.struct = MxRotary(turn.data_ptr(), 2 * turn.shape[0], 1 if layout == 'interleaved' else 0, amplitude)

    @property
    def width(self):
        return self.struct.width

    @staticmethod
    def angles(width, *, base=10000.0, scaling=None, factor=1.0, original=None, slow=1.0, fast=32.0):
        """(angles in radians, amplitude): ``base ** (-2 i / width)`` for pair i, and for episodes ``factor`` times as long
        as the ``original`` positions that a policy was trained on

        * 'linear': all angles divided by factor, as if positions were that much closer;
        * 'base': a larger base, which leaves the first pair's angle and divides the last one's by factor;
        * 'parts': pairs that turn less than ``slow`` times within the original positions are divided by factor, those that
          turn more than ``fast`` times stay, those between go from one to the other in a straight line; the amplitude is then
          0.1 ln(factor) + 1, which makes scores sharper over more keys."""
        _require(width >= 2 and width % 2 == 0, 'width must be even and positive, got %s', width)
        _require(scaling in SCALINGS, 'scaling must be one of %s, got %s', SCALINGS, scaling)
        _require(math.isfinite(base) and base > 0, 'base must be positive, got %s', base)
        _require(math.isfinite(factor) and factor >= 1, 'factor must be 1 or more, got %s', factor)
        if scaling == 'base':
            _require(width > 2, 'a larger base needs more than one pair')
            base *= factor ** (width / (width - 2))
        turn = torch.tensor([base ** (-2.0 * i / width) for i in range(width // 2)], dtype=torch.float64)
        if scaling == 'linear':
            return turn / factor, 1.0
        if scaling != 'parts':
            return turn, 1.0
        _require(original is not None and original > 0, 'parts needs the original number of positions')
        _require(0 < slow < fast, 'slow must be positive and below fast')
        kept = ((original * turn / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        return turn * (kept + (1.0 - kept) / factor), 0.1 * math.log(factor) + 1.0

    @classmethod
    def make(cls, width, *, layout='half', amplitude=None, device='cuda:0', **options):
        """A Rotary with the angles of :meth:`angles` (its options) on a device; ``amplitude``: another than theirs."""
        turn, by = cls.angles(width, **options)
        return cls(turn.to(device), layout=layout, amplitude=by if amplitude is None else amplitude)


def _stepping(x, name):
    """MxRows of a tensor (tokens, heads, head_dim) or (batch, tokens, heads, head_dim) whose rows step evenly."""
    shape, stride = x.shape, x.stride()
    _require(len(shape) in (3, 4), '%s must be (tokens, heads, head_dim) or (batch, tokens, heads, head_dim): %s', name, tuple(shape))
    _require(_TYPES.get(x.dtype, 3) < 3, '%s must be float32, bfloat16 or float16, got %s', name, x.dtype)
    _require(stride[-1] == 1 or shape[-1] == 1, '%s must be contiguous along head_dim', name)
    token = stride[-3]
    if len(shape) == 4:
        if shape[1] == 1:
            token = stride[0]
        elif shape[0] > 1 and shape[1] > 1 and stride[0] != shape[1] * token:
            raise ValueError('%s: its rows must step evenly' % name)
    return MxRows(x.data_ptr(), token, stride[-2], shape[-2], _TYPES[x.dtype])


def _turn(rotary, x, positions, back, out):
    rows, shape = _stepping(x, 'x'), x.shape
    if out is None:
        out = x.new_empty(shape)
        to = MxRows(out.data_ptr(), shape[-2] * shape[-1], shape[-1], shape[-2], rows.type)
    else:
        to = _stepping(out, 'out')
    tokens = shape[0] if len(shape) == 3 else shape[0] * shape[1]
    _require(tokens < 2 ** 31, 'fewer than 2^31 rows can be turned at once: %s', tokens)
    if tokens and rows.heads:
        _launch(rotary, rows, to, shape[-1], tokens, positions, back)
    return out


def _launch(rotary, rows, to, head_dim, tokens, positions, back):
    lib = episodes._LIB or episodes.load()
    rc = lib.mx_rotate(ct.byref(rotary.struct), ct.byref(rows), ct.byref(to), head_dim, tokens, positions.data_ptr(),
                       positions.numel(), positions.dtype == torch.int64, back, _current(rotary.index))
    if rc:
        _check(rc, 'mx_rotate')


class _Rotate(torch.autograd.Function):
    """A rotation's gradient is the rotation back.  ``how``: (Rotary, positions, back), in one argument, and the gradient's
    rotation without the checks of the forward's, as all that autograd's own thread does is waited for (a short batch's
    forward and backward 89 -> 79 us)."""

    @staticmethod
    def forward(ctx, x, how):
        rotary, positions, back = how
        ctx.save_for_backward(positions, rotary.turn)
        ctx.how = rotary, back
        return _turn(rotary, x, positions, back, None)

    @staticmethod
    def backward(ctx, grad):
        positions, _ = ctx.saved_tensors                 # raises if one has changed
        rotary, back = ctx.how
        if not grad.is_contiguous():
            grad = grad.contiguous()
        if torch.is_grad_enabled():                      # a gradient of the gradient is wanted
            return _Rotate.apply(grad, (rotary, positions, not back)), None
        out = torch.empty_like(grad)
        heads, head_dim = grad.shape[-2:]
        token = heads * head_dim
        if grad.numel():
            kind = _TYPES[grad.dtype]
            _launch(rotary, MxRows(grad.data_ptr(), token, head_dim, heads, kind), MxRows(out.data_ptr(), token, head_dim, heads, kind),
                    head_dim, grad.numel() // token, positions, not back)
        return out, None


def rotate(rotary, x, positions, *, back=False, out=None, stream=None):
    """Rows turned by their positions: x (tokens, heads, head_dim) or (batch, tokens, heads, head_dim) in float32, bfloat16 or
    float16, any strides whose rows step evenly and whose head_dim is contiguous; ``positions`` int32 or int64, contiguous, one
    to a row, or (tokens,) for all of a batch.  Cosines and sines are computed in 64 bits and rounded to 32, the values turned in
    32 and rounded once.

    ``back`` turns by the negative angles (with the same amplitude): that is the gradient, which autograd takes where x
    requires one; its own gradient is a rotation again.  A backward pass is captured as that of torch's own operations: where
    an eager graph of the same leaves still lives, torch cannot (give the capture leaves of its own, ``x.detach()``, or drop
    that graph first).  ``out``, like x and apart from it, is written if given, where no gradient is recorded.  Returns out."""
    shape = x.shape
    if not (x.get_device() == rotary.index and len(shape) in (3, 4) and rotary.struct.width <= shape[-1]
            and positions.dtype in (torch.int32, torch.int64) and positions.is_contiguous()
            and positions.get_device() == rotary.index and positions.shape in (shape[:-2], shape[-3:-2])):
        _require(x.get_device() == rotary.index, 'x must be on the device of the angles')
        _require(x.dim() in (3, 4) and rotary.struct.width <= x.shape[-1],
                 'x must be (..., tokens, heads, head_dim) with a head_dim of at least the %d values that turn: %s',
                 rotary.struct.width, tuple(x.shape))
        raise ValueError('positions must be contiguous int32 or int64 on x\'s device, one to a row, or of shape (tokens,)')
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError('x: there is no forward-mode derivative; rotate the tangent itself')
    recorded = x.requires_grad and torch.is_grad_enabled()
    if out is not None:
        _require(not recorded and not (out.requires_grad and torch.is_grad_enabled()),
                 'out cannot be given where gradients are recorded')
        _require(out.get_device() == rotary.index and not _overlap(x, out), 'out must be on x\'s device, and apart from x')
        _output(x, out)
    if stream is not None or torch.cuda.current_device() != rotary.index:
        return _on(x.device, stream, (x, positions, rotary.turn, out), lambda: rotate(rotary, x, positions, back=back, out=out))
    return _Rotate.apply(x, (rotary, positions, bool(back))) if recorded else _turn(rotary, x, positions, bool(back), out)


def enter(pages, rotary, q, k, v, start=None, *, out=None, stream=None):
    """Turn the chunk's queries and keys by their positions in their worlds (see :mod:`libero_hip.episodes`), store the keys
    and values in the pages, as :func:`libero_hip.episodes.write` does, and return the queries: q, k, v of one type (float32,
    bfloat16 or float16), any strides whose tokens step evenly and whose head_dim is contiguous.  Keys are rounded once,
    into the pages.  ``out``, like q and apart from q, k and v, is written if given; rows that belong to no world are left out.
    To be followed by :func:`libero_hip.episodes.attend` of what it returns."""
    if _elsewhere(pages, stream):
        tensors = (q, k, v, start, out, rotary.turn, pages.k, pages.v, pages.k_scale, pages.v_scale, pages.table, pages.length)
        return _on(pages.device, stream, tensors, lambda: enter(pages, rotary, q, k, v, start, out=out))
    s, shape = pages.struct, k.shape
    if shape != v.shape or k.dtype != v.dtype or len(shape) < 3 or shape[-2] != s.kv_heads:
        raise ValueError('k and v must have one type and one shape, with %d heads: %s, %s' % (s.kv_heads, tuple(shape), tuple(v.shape)))
    if q.dtype != k.dtype or q.shape[:-2] != shape[:-2]:
        raise ValueError('q must have the keys\' type and rows: %s, %s and %s, %s' % (q.dtype, k.dtype, tuple(q.shape), tuple(shape)))
    if rotary.index != pages.index or rotary.struct.width > s.head_dim:
        raise ValueError('the angles must be on the pages\' device, and no more than half of head_dim: %d' % (rotary.struct.width // 2))
    chunk = _chunk(pages, shape[:-2], start)
    a, b, c = _rows(pages, q, q.shape, 'q'), _rows(pages, k, shape, 'k'), _rows(pages, v, shape, 'v')
    _require(a.heads > 0, 'q has no heads')
    if out is None:
        out = q.new_empty(q.shape)
        to = MxRows(out.data_ptr(), a.heads * s.head_dim, s.head_dim, a.heads, a.type)
    else:
        _require(not (_overlap(out, q) or _overlap(out, k) or _overlap(out, v)), 'out must be apart from q, k and v')
        to = _rows(pages, _output(q, out), q.shape, 'out')
    lib = episodes._LIB or episodes.load()
    rc = lib.mx_episode_enter(ct.byref(s), ct.byref(chunk), ct.byref(rotary.struct), ct.byref(a), ct.byref(to), ct.byref(b),
                              ct.byref(c), _current(pages.index))
    if rc:
        _check(rc, 'mx_episode_enter')
    return out
