"""Episode memory, host side: the C entry points' checks (made before any launch, so no GPU is needed) against
include/mx_episode.h, and the definitions that the GPU tests compare with against independent facts."""
import ctypes as ct
import re
from pathlib import Path

import numpy as np
import pytest

from episode_reference import attention, e4m3, quantised
from libero_hip import episodes

HEADER = Path(__file__).resolve().parents[1] / 'include' / 'mx_episode.h'
INVALID, DOMAIN, WORKSPACE = -1, -2, -5


def test_exports():
    text = re.sub(r'/\*.*?\*/', '', HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r'^[a-z_ ]+[ *]+(mx_[a-z0-9_]+)\(', text, flags=re.M)))
    assert names == sorted(episodes.EXPORTS)
    lib = episodes.load()
    for name in names:
        assert hasattr(lib, name), name
    assert 'workspace' in lib.mx_error_string(WORKSPACE).decode()


class Call:
    """Arguments that pass every check but the last, an attention workspace that is missing."""

    def __init__(self):
        self.buffer = ct.create_string_buffer(4096)
        at = (ct.addressof(self.buffer) + 63) & ~63
        self.pages = episodes.MxPages(at, at, None, None, at, at, 2, 4, 64, 2, 64, 64, 1)
        self.chunk = episodes.MxChunk(None, 2, 1)
        self.k = episodes.MxRows(at, 128, 64, 2, 1)
        self.v = episodes.MxRows(at, 128, 64, 2, 1)
        rows = episodes.MxRows(at, 256, 64, 4, 1)
        self.attention = episodes.MxAttention(rows, rows, None, None, 0, 1, 1, 0, 0.125)
        self.at = at

    def write(self):
        return episodes.load().mx_episode_write(ct.byref(self.pages), ct.byref(self.chunk), ct.byref(self.k),
                                                ct.byref(self.v), None)

    def read(self):
        return episodes.load().mx_episode_read(ct.byref(self.pages), ct.byref(self.chunk), ct.byref(self.k),
                                               ct.byref(self.v), None)

    def attend(self):
        return episodes.load().mx_episode_attend(ct.byref(self.pages), ct.byref(self.chunk), ct.byref(self.attention), None)

    def workspace(self):
        return episodes.load().mx_episode_workspace(ct.byref(self.pages), ct.byref(self.chunk), ct.byref(self.attention))


@pytest.mark.parametrize('field,value,code', [
    ('k', None, INVALID), ('v', None, INVALID), ('table', None, INVALID), ('length', None, INVALID),
    ('nworld', 0, INVALID), ('npage', 0, INVALID), ('width', 0, INVALID), ('kv_heads', 0, INVALID),
    ('type', 0, INVALID), ('type', 3, INVALID), ('type', 9, INVALID), ('head_dim', 48, DOMAIN), ('head_dim', 512, DOMAIN),
    ('page_tokens', 8, DOMAIN), ('page_tokens', 48, DOMAIN), ('page_tokens', 8192, DOMAIN), ('npage', 2 ** 26, DOMAIN),
    ('width', 2 ** 24 + 1, DOMAIN), ('kv_heads', 2000, DOMAIN)])
def test_pages_are_checked(field, value, code):
    for entry in ('write', 'read', 'attend'):
        c = Call()
        setattr(c.pages, field, value)
        assert getattr(c, entry)() == code, entry
    c = Call()
    c.pages.k += 8
    assert c.attend() == INVALID


def test_rows_and_chunks_are_checked():
    lib = episodes.load()
    assert lib.mx_episode_attend(None, None, None, None) == INVALID
    assert lib.mx_episode_workspace(None, None, None) == 0
    for change in (lambda c: setattr(c.chunk, 'tokens', 3), lambda c: setattr(c.chunk, 'tokens', -1),
                   lambda c: setattr(c.chunk, 'count', -1)):
        for entry in ('write', 'read', 'attend'):
            c = Call()
            change(c)
            assert getattr(c, entry)() == INVALID
    for change in (lambda c: setattr(c.k, 'heads', 3), lambda c: setattr(c.k, 'data', None), lambda c: setattr(c.k, 'type', 3),
                   lambda c: setattr(c.k, 'type', 2), lambda c: setattr(c.v, 'data', c.at + 1)):
        for entry in ('write', 'read'):
            c = Call()
            change(c)
            assert getattr(c, entry)() == INVALID
    for change in (lambda a: setattr(a.q, 'heads', 3), lambda a: setattr(a.out, 'heads', 2), lambda a: setattr(a.q, 'type', 2),
                   lambda a: setattr(a.q, 'type', 0), lambda a: setattr(a.q, 'data', None), lambda a: setattr(a, 'window', -1),
                   lambda a: setattr(a, 'max_count', -1), lambda a: setattr(a, 'scale', float('inf'))):
        c = Call()
        change(c.attention)
        assert c.attend() == INVALID
    for entry in ('write', 'read', 'attend'):           # no rows: nothing to do
        c = Call()
        c.chunk.tokens = c.chunk.count = 0
        c.k.data = c.v.data = c.attention.q.data = None
        assert getattr(c, entry)() == 0


def test_more_workgroups_than_a_launch_holds():
    """Threads of a launch are counted in 32 bits, so 2^24 - 1 workgroups of 256 are the most."""
    c = Call()
    c.pages.nworld, c.pages.kv_heads, c.pages.page_tokens, c.pages.width = 1 << 21, 8, 16, 1
    rows = episodes.MxRows(c.at, 512, 64, 8, 1)
    c.attention.q = c.attention.out = rows
    c.chunk.tokens = c.pages.nworld
    assert c.workspace() == 0 and c.attend() == DOMAIN
    c = Call()                                            # 64 tokens to a workgroup are the most
    c.pages.kv_heads = c.k.heads = c.v.heads = 1
    c.chunk = episodes.MxChunk(c.at, 2 ** 31 - 1, 0)
    assert c.write() == DOMAIN and c.read() == DOMAIN


def test_workspace():
    """A long table and few rows are split along the keys, into a workspace that has to be there."""
    c = Call()
    c.pages.width = 4096
    need = c.workspace()
    assert need > 0 and need % (2 * 4 * (64 + 2) * 4) == 0      # parts of tokens x heads rows, of two numbers more
    assert c.attend() == WORKSPACE
    c.attention.workspace, c.attention.workspace_bytes = c.at, need - 1
    assert c.attend() == WORKSPACE
    c.attention.workspace, c.attention.workspace_bytes = c.at + 8, need
    assert c.attend() == WORKSPACE
    c.pages.width = 1
    assert c.workspace() == 0


def test_reference_quantisation():
    """All 256 codes are their own nearest values; between neighbours the nearer one, at the middle the even one."""
    codes = np.array([s * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
                      for s in (1, -1) for e in range(16) for m in range(8) if not (e == 15 and m == 7)])
    np.testing.assert_array_equal(e4m3(codes), codes)
    up = np.unique(np.abs(codes))
    middle = (up[1:] + up[:-1]) / 2
    even = np.where(np.arange(len(up) - 1) % 2 == 0, up[:-1], up[1:])
    np.testing.assert_array_equal(e4m3(middle), even)
    np.testing.assert_array_equal(e4m3(middle * (1 + 1e-9)), up[1:])
    np.testing.assert_array_equal(e4m3(middle * (1 - 1e-9)), up[:-1])
    x = np.random.default_rng(0).standard_normal((40, 64)) * 10.0 ** np.arange(-20, 20)[:, None]
    y, scale = quantised(x)
    # a value is off by 2^-4 of itself, or half the smallest step of a block whose largest is within a factor of two of 448
    assert np.all(np.abs(y - x) <= np.maximum(np.abs(x) / 16, 2.0 ** (scale.repeat(32, 1) - 127.0) * 2.0 ** -10))
    assert np.all(np.abs(x).reshape(40, 2, 32).max(-1) > 224 * 2.0 ** (scale - 127.0))


def test_reference_attention():
    """Equal scores average the visible values; a window of one returns the token's own value; a query before the
    first token sees nothing."""
    rng = np.random.default_rng(1)
    v = rng.standard_normal((6, 2, 4))
    q, k = rng.standard_normal((3, 4, 4)), np.zeros((6, 2, 4))
    out, lse, _ = attention(q, k, v, 3, True, 0, 1.0)
    for i in range(3):
        np.testing.assert_allclose(out[i, 2], v[:4 + i, 1].mean(0))
        np.testing.assert_allclose(lse[i], np.log(4 + i))
    np.testing.assert_allclose(attention(q, k, v, 3, True, 1, 1.0)[0][1, 0], v[4, 0])
    np.testing.assert_allclose(attention(q, k, v, 3, False, 0, 1.0)[0][0, 3], v[:, 1].mean(0))
    out, lse, _ = attention(q, k, v, -2, True, 0, 1.0)
    assert not out[:2].any() and np.all(np.isneginf(lse[:2])) and np.isfinite(lse[2]).all()


def test_workspace_of_the_rows_that_are_computed():
    """Chunks longer than max_count: the parts are of the computed rows, whatever the chunks hold beside them."""
    c = Call()
    c.pages.width = 4096
    need = c.workspace()                                        # one token of each of two worlds
    c.chunk.count, c.chunk.tokens = 2 ** 17, 2 ** 18
    assert c.workspace() == need
    c.attention.max_count = 3
    assert c.workspace() > 0 and c.workspace() % (2 * 3 * 4 * (64 + 2) * 4) == 0


def test_scales_are_finite_in_base_two():
    """The kernels take the scale times log2(e): 3e38 would become an infinity there, and scores of 0 NaN."""
    for scale in (3e38, -3e38, float('inf'), float('nan')):
        c = Call()
        c.attention.scale = scale
        assert c.attend() == INVALID and c.workspace() == 0
    c = Call()
    c.pages.width, c.attention.scale = 4096, 2.3e38
    assert c.attend() == WORKSPACE
