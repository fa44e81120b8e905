"""What a policy asks of its episode memory besides writing, reading and attending to all of it, as cases to time.

Three groups of operators, in the order in which a step of the policy calls them:

* room on the GPU (``room``): the worlds' page tables, lengths and the free pages change in one call, new tokens in
  and restarted worlds emptied, and every new row learns its world, position and slot;
* rotary positions (``rotate``, ``enter``): queries and keys turn by their place in the episode, for a training batch with
  the gradient, or on the way into the pages;
* recall (``recall``): of a long episode a query attends to the blocks of tokens whose summaries match it best, its latest
  blocks and its first ones.  The blocks that the step's tokens complete are summarised, blocks are selected, and
  attended to.

Worlds reset one by one, so their lengths are spread over the whole range and their pages lie in any order.  The lengths
and chunk sizes of a case follow from the case alone; the seed decides which world has which, where the pages lie, and all
values.
"""
from __future__ import annotations

import math
import sys
from functools import lru_cache
from pathlib import Path

import numpy as np
import torch

own = False

DEVICE = 'cuda:0'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}
BLOCK = 32          # values that share one scale in 8-bit pages
LARGEST = 448.0     # the largest 8-bit value
MOST = 127          # the largest code of a summary
POWER = 40          # the largest exponent of a summary's or a query's scale, and the least one's negative


def listed():
    return [
        # episodes as a training batch, read out of the memory: forward and gradient
        dict(name='rotate bf16 x16', do='rotate', batch=16, tokens=1024, heads=16, dim=64, width=64, layout='half',
             input='bf16', last=1023, base=10000.0),
        # two short pieces in single precision from far along, part of an odd head, neighbours turned together: latency
        dict(name='rotate f32 x2 far', do='rotate', batch=2, tokens=33, heads=3, dim=80, width=20, layout='interleaved',
             input='f32', last=1 << 24, base=500000.0),
        # each control step of the largest contact batch: one token per world, into the quantised memory
        dict(name='enter fp8 x4096', do='enter', worlds=4096, heads=16, kv=4, dim=64, width=64, layout='half',
             input='bf16', store='fp8', page=64, length=1024, count=1, base=10000.0),
        # demonstrations taken in as prompts of very different lengths, half of each head turned
        dict(name='enter f16 x67 ragged', do='enter', worlds=67, heads=12, kv=4, dim=96, width=48, layout='interleaved',
             input='f16', store='fp8', page=64, length=1024, count=501, ragged=True, base=10000.0),
        # whole prompts, positions stretched beyond those that the policy was trained on: bound by memory
        dict(name='enter bf16 x4 prompt', do='enter', worlds=4, heads=32, kv=8, dim=128, width=128, layout='half',
             input='bf16', store='bf16', page=64, length=4096, count=4096, base=10000.0, factor=8.0, original=512),
        # some worlds of a small batch look ahead by a few tokens and take them back: launches are all
        dict(name='room x67 ahead', do='room', worlds=67, page=16, tokens=512, length=300, count=9, ragged=True),
        # every world of the largest batch restarts with its own instruction and demonstration
        dict(name='room x4096 restart', do='room', worlds=4096, page=64, tokens=1024, length=1024, restart=True),
        # two worlds a few steps into their episodes, a head for each: latency again
        dict(name='recall bf16 x2', do='recall', worlds=2, heads=8, kv=8, dim=64, input='bf16', store='bf16', page=16,
             block=16, length=200, count=1, top=4, near=2, first=1),
        # each control step of a contact batch late in its episodes, from the quantised memory
        dict(name='recall fp8 x1024', do='recall', worlds=1024, heads=16, kv=4, dim=64, input='bf16', store='fp8', page=64,
             block=64, length=8192, count=1, top=8, near=2, first=1),
        # two very long episodes: few rows, the summaries are long
        dict(name='recall bf16 x2 long', do='recall', worlds=2, heads=32, kv=8, dim=128, input='bf16', store='bf16',
             page=256, block=64, length=131072, count=1, top=32, near=4, first=1),
        # a step's observation tokens, which see each other; ragged, odd sizes
        dict(name='recall f16 x67 chunk', do='recall', worlds=67, heads=12, kv=4, dim=96, input='f16', store='f16', page=32,
             block=32, length=2500, count=13, ragged=True, causal=False, top=6, near=3, first=2),
        # a long prompt behind a long episode: each token selects for itself
        dict(name='recall bf16 x1 prompt', do='recall', worlds=1, heads=32, kv=8, dim=128, input='bf16', store='bf16',
             page=64, block=64, length=65536, count=2048, top=16, near=2, first=1),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over the logarithm, odd ones among them."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        case = _drawn(rng)
        if _cost(case) <= 1.0:
            return case


def _drawn(rng):
    do = rng.choice(('rotate', 'enter', 'enter', 'room', 'recall', 'recall', 'recall'))
    if do == 'rotate':
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        tokens = _log(rng, 1, 16384)
        return dict(do=do, batch=_log(rng, 1, 64), tokens=tokens, heads=rng.choice((1, 2, 3, 8, 16, 32)), dim=dim,
                    width=rng.choice((dim, dim, dim // 2, 20)), layout=rng.choice(('half', 'interleaved')),
                    input=rng.choice(('f32', 'bf16', 'f16')), last=_log(rng, tokens, 1 << 24),
                    base=rng.choice((10000.0, 500000.0)))
    if do == 'room':
        case = dict(do=do, worlds=_log(rng, 1, 4096), page=rng.choice((16, 32, 64, 128, 256)), length=_log(rng, 1, 16384))
        case['tokens'] = case['length'] + _log(rng, 1, 1024)
        if rng.random() < 0.4:
            case['restart'] = True
        else:
            case['count'] = 1 if rng.random() < 0.4 else _log(rng, 1, case['length'])
            case['ragged'] = rng.random() < 0.5
        return case
    kv = rng.choice((1, 2, 3, 4, 8))
    page = rng.choice((16, 32, 64, 128, 256))
    case = dict(do=do, worlds=_log(rng, 1, 4096), kv=kv, heads=kv * rng.choice((1, 1, 2, 3, 4, 8)),
                dim=rng.choice((32, 64, 96, 128)), page=page, length=_log(rng, 1, 131072))
    case['input'] = rng.choice(('bf16', 'bf16', 'f16') if do == 'recall' else ('bf16', 'f16', 'f32'))
    case['store'] = rng.choice(('fp8', case['input'] if case['input'] != 'f32' else 'bf16'))
    case['count'] = 1 if rng.random() < 0.5 else _log(rng, 1, min(case['length'], 4096))
    if case['count'] > 1 and case['worlds'] > 1 and rng.random() < 0.5:
        case['ragged'] = True
    if do == 'enter':
        case.update(width=rng.choice((case['dim'], case['dim'], case['dim'] // 2)), base=rng.choice((10000.0, 500000.0)),
                    layout=rng.choice(('half', 'interleaved')))
        if rng.random() < 0.3:
            case.update(factor=float(rng.choice((2, 8, 32))), original=rng.choice((512, 4096)))
        return case
    case.update(block=min(page, rng.choice((16, 32, 64, 128))), top=_log(rng, 1, 64), near=rng.choice((1, 2, 3, 8)),
                first=rng.choice((0, 1, 2)))
    if rng.random() < 0.3:
        case['causal'] = False
    return case


def _cost(case):
    """A bound on what a case takes and holds, as a share of the largest listed ones."""
    if case['do'] == 'rotate':
        return case['batch'] * case['tokens'] * case['heads'] * case['dim'] / (16 * 1024 * 16 * 64)
    if case['do'] == 'room':
        return case['worlds'] * max(case['length'], case.get('count', 0)) / (4096 * 1024)
    held = case['worlds'] * case['length'] * case['kv'] * case['dim']
    rows = case['worlds'] * case['count']
    if case['do'] == 'enter':
        return max(rows * (case['heads'] + 2 * case['kv']) * case['dim'] / (4 * 4096 * 48 * 128), held / (4096 * 1024 * 4 * 64))
    keys = case['block'] * (case['top'] + case['near'] + case['first'] + (0 if case.get('causal', True) else case['count'] // case['block'] + 1))
    blocks = case['length'] / case['block'] + 1
    return max(held / (1024 * 8192 * 4 * 64), rows * keys * case['kv'] * case['dim'] / (2048 * 19 * 64 * 8 * 128),
               rows * blocks * case['heads'] / (2048 * 1024 * 32))


# ---------------------------------------------------------------------------- sizes and inputs
@lru_cache(maxsize=64)
def _sizes(worlds, length, count, ragged):
    """(new tokens, tokens in all) of each world, from the case alone."""
    i = np.arange(worlds)
    new = np.full(worlds, count, np.int64)
    if ragged:                    # 0 .. count, in an order that has nothing to do with the lengths'
        new = np.floor(((i * 0.6180339887498949 + 0.5) % 1.0) * (count + 1)).astype(np.int64)
        new[0] = count
    past = np.floor((i + 0.5) / worlds * (length - count + 1)).astype(np.int64)
    return new, past + new


def _case_sizes(case):
    if case.get('restart'):       # all tokens of all worlds are new
        _, total = _sizes(case['worlds'], case['length'], 0, False)
        return total, total
    if case['do'] == 'room':      # none of the new tokens is there yet
        new, _ = _sizes(case['worlds'], case['tokens'], case['count'], bool(case.get('ragged')))
        past = _sizes(case['worlds'], min(case['length'], case['tokens'] - case['count']), 0, False)[1]
        return new, past + new
    return _sizes(case['worlds'], case['length'], case['count'], bool(case.get('ragged')))


def _listed_blocks(case):
    """How many blocks a query's list has room for."""
    own_blocks = 0 if case.get('causal', True) else (case['count'] + case['block'] - 2) // case['block']
    return case['first'] + case['near'] + case['top'] + own_blocks


def _frequencies(case):
    """How far each pair of values turns from one position to the next, in radians (64 bits), and the factor of the
    turned values.  With a factor for long contexts, pairs that turn less than once within the original positions turn
    slower by it, those that turn more than 32 times as before, those between in between."""
    pair = np.arange(case['width'] // 2)
    turn = case['base'] ** (-2.0 * pair / case['width'])
    factor = case.get('factor')
    if not factor:
        return turn, 1.0
    turns = case['original'] * turn / (2 * math.pi)
    kept = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return turn * (kept + (1.0 - kept) / factor), 0.1 * math.log(factor) + 1.0


def _quantise(x):
    """8-bit codes and scale exponents of x, whose last axis is a whole number of blocks: the scale of a
    block is the least power of two (2^-117 at least) at which no value passes the largest 8-bit one."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    fraction, exponent = torch.frexp(b.abs().amax(-1, keepdim=True))     # amax = fraction * 2^exponent, fraction < 1
    e = (exponent - 9 + (fraction > LARGEST / 512)).clamp(min=-117)
    e = torch.where(fraction == 0, torch.full_like(e, -117), e)
    codes = (b * torch.exp2(-e.float())).to(torch.float8_e4m3fn).flatten(-2)
    return codes, (e.squeeze(-1) + 127).to(torch.uint8)


def _values(codes, scale):
    """The values that 8-bit codes (as bytes) and scale exponents stand for, in 32 bits."""
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, BLOCK))
    return (x * torch.exp2(scale.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _codes(x):
    """Whole numbers up to 127 and exponents e, x about codes * 2^e along the last axis: the least e from -40 to 40 at
    which none passes 127, rounded to nearest even.  x in 64 bits and finite."""
    fraction, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(fraction == 0, torch.full_like(exponent, -POWER), exponent - 7 + (fraction > MOST / 128))
    e = e.clamp(-POWER, POWER)
    codes = torch.round(x * torch.exp2(-e.double())).clamp(-MOST, MOST)
    return codes.to(torch.int8), e.squeeze(-1)


def _tables(case, rng, total, width, spare):
    """Pages of all worlds, in any order among each other, and the numbers of the pages that none has."""
    held = -(-total // case['page'])
    npage = int(held.sum()) + spare
    ids = rng.permutation(npage).astype(np.int32)
    table = np.full((case['worlds'], width), -1, np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = ids[spare:]
    return table, npage, ids[:spare]


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    if case['do'] == 'rotate':
        return _prepare_rotate(case, gen, rng)
    if case['do'] == 'room':
        return _prepare_room(case, rng)
    n, kv, dim, page = case['worlds'], case['kv'], case['dim'], case['page']
    dtype = TYPES[case['input']]
    new, total = _case_sizes(case)
    order = rng.permutation(n)
    new, total = new[order], total[order]
    table, npage, _ = _tables(case, rng, total, max(1, -(-case['length'] // page)), 3)

    # keys have channels of very different size, and some heads look closer than others
    def made(shape, spread):
        x = torch.randn(shape, generator=gen, device=DEVICE)
        if spread:
            x *= torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device=DEVICE))
        return x

    state = dict(case=case, page=page, npage=npage, table=torch.from_numpy(table).to(DEVICE),
                 length=torch.from_numpy(total.astype(np.int32)).to(DEVICE), start=None, k_scale=None, v_scale=None)
    block = case.get('block', page)
    for name in ('k', 'v'):
        x = made((npage, kv, page, dim), name == 'k')
        if case['do'] == 'recall' and name == 'k':     # neighbouring tokens are about the same things
            x.view(npage, kv, page // block, block, dim).add_(
                0.5 * torch.randn((npage, kv, page // block, 1, dim), generator=gen, device=DEVICE))
        if case['store'] == 'fp8':
            state[name], state[name + '_scale'] = _quantise(x)
        else:
            state[name] = x.to(TYPES[case['store']])
        del x
    tokens = int(new.sum())
    if case.get('ragged'):
        start = np.zeros(n + 1, np.int32)
        start[1:] = np.cumsum(new)
        state['start'] = torch.from_numpy(start).to(DEVICE)
    rows = (tokens,) if case.get('ragged') else (n, case['count'])
    state['tokens'], state['most'] = tokens, int(new.max())
    state['q'] = made(rows + (case['heads'], dim), False).to(dtype)
    if case['do'] == 'enter':
        state['new_k'] = made(rows + (kv, dim), True).to(dtype)
        state['new_v'] = made(rows + (kv, dim), False).to(dtype)
        turn, state['amplitude'] = _frequencies(case)
        state['turn'] = torch.from_numpy(turn).to(DEVICE)
    else:                                              # the summaries of all that was there before, and of later blocks
        shape = (npage, kv, page // block, dim)        # what their pages' earlier owners left
        state['codes'] = torch.empty(shape, dtype=torch.int8, device=DEVICE)
        state['exponent'] = torch.empty(shape[:3], dtype=torch.uint8, device=DEVICE)
        for at in range(0, npage, 4096):
            x = _stored(state, 'k', slice(at, at + 4096)).unflatten(2, (-1, block)).double().mean(3)
            codes, e = _codes(x)
            state['codes'][at:at + 4096], state['exponent'][at:at + 4096] = codes, (e + 127).to(torch.uint8)
    return state


def _prepare_rotate(case, gen, rng):
    shape = (case['batch'], case['tokens'], case['heads'], case['dim'])
    x, grad = (torch.randn(shape, generator=gen, device=DEVICE).to(TYPES[case['input']]) for _ in range(2))
    # pieces of episodes: each begins anywhere and goes on from there
    first = rng.integers(0, max(1, case['last'] - case['tokens'] + 1) + 1, case['batch'])
    positions = torch.from_numpy((first[:, None] + np.arange(case['tokens'])).astype(np.int64)).to(DEVICE)
    turn, amplitude = _frequencies(case)
    return dict(case=case, x=x.requires_grad_(), grad=grad, positions=positions, amplitude=amplitude,
                turn=torch.from_numpy(turn).to(DEVICE))


def _prepare_room(case, rng):
    n, page = case['worlds'], case['page']
    new, total = _case_sizes(case)
    order = rng.permutation(n)
    new, total = new[order], total[order]
    past = total if case.get('restart') else total - new
    width = -(-case['tokens'] // page)
    spare = 5 + int((-(-total // page)).sum() - (-(-past // page)).sum())
    table, npage, left = _tables(case, rng, past, width, spare)
    free = np.full(npage, -1, np.int32)
    free[:spare] = left

    def there(x):
        return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(DEVICE)

    return dict(case=case, page=page, npage=npage, table=there(table), length=there(past), free=there(free),
                state=there([spare, 0]), new=there(new), back=there(-new), tokens=int(new.sum()),
                over=torch.ones(n, dtype=torch.bool, device=DEVICE) if case.get('restart') else None)


# ---------------------------------------------------------------------------- the framework's operators
@lru_cache(maxsize=None)
def _library():
    path = str(Path.cwd() / 'gpu-libero_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    from libero_hip import episodes, recall, room, rotary
    return episodes, recall, room, rotary


def _own(s):
    episodes, recall, room, rotary = _library()
    case = s['case']
    if case['do'] == 'rotate':
        turning = rotary.Rotary(s['turn'], layout=case['layout'], amplitude=s['amplitude'])
        out = rotary.rotate(turning, s['x'], s['positions'])
        return out.detach(), torch.autograd.grad(out, s['x'], s['grad'])[0]
    if case['do'] == 'room':
        worlds = room.Room(s['table'], s['length'], s['npage'], s['page'], s['free'], s['state'], tokens=case['tokens'])
        start = room.make_room(worlds, s['new'], s['over'], rows=s['tokens'])
        maps = room.places(worlds, start, tokens=s['tokens'])
        if s['over'] is None:
            room.make_room(worlds, s['back'])
        return (start, *maps, s['table'], s['length'], s['free'], s['state'])
    pages = episodes.Pages(s['k'], s['v'], s['table'], s['length'], s['k_scale'], s['v_scale'])
    if case['do'] == 'enter':
        turning = rotary.Rotary(s['turn'], layout=case['layout'], amplitude=s['amplitude'])
        out = rotary.enter(pages, turning, s['q'], s['new_k'], s['new_v'], s['start'])
        if s['start'] is None:
            return (out, *episodes.read(pages, count=case['count'], dtype=s['q'].dtype))
        return (out, *episodes.read(pages, s['start'], tokens=s['tokens'], dtype=s['q'].dtype))
    summaries = recall.Summaries(pages, s['codes'], s['exponent'])
    if s['start'] is None:
        recall.summarise(summaries, count=case['count'])
    else:
        recall.summarise(summaries, s['start'], tokens=s['tokens'])
    causal = case.get('causal', True)
    blocks = recall.select(summaries, s['q'], s['start'], top=case['top'], near=case['near'], first=case['first'],
                           causal=causal, max_count=s['most'])
    out = recall.recall(pages, s['q'], blocks, s['start'], block_tokens=case['block'], causal=causal, max_count=s['most'])
    return blocks, out, s['codes'], s['exponent']


# ---------------------------------------------------------------------------- the plain forms
def _tokens_at(s, start, new, tokens):
    """World and position of every packed token."""
    at = torch.arange(tokens, device=DEVICE)
    if start is None:
        world, place = at // new, at % new
        return world, s['length'].long()[world] - new + place
    start = start.long()
    world = torch.searchsorted(start[1:], at, right=True)
    return world, s['length'].long()[world] - (start[1:] - start[:-1])[world] + at - start[world]


def _stored(s, name, page):
    """The values of pages, in 32 bits."""
    if s['k_scale'] is None:
        return s[name][page].float()
    return _values(s[name].view(torch.uint8)[page], s[name + '_scale'][page])


def _turned(x, positions, turn, amplitude, width, layout, back=False):
    """x (rows, heads, dim) with each pair of its first `width` values turned by its row's position, in 32 bits."""
    angle = positions.double()[:, None, None] * turn
    cos, sin = (torch.cos(angle) * amplitude).float(), (torch.sin(angle) * amplitude).float()
    sin = -sin if back else sin
    y = x.float()
    half = width // 2
    if layout == 'half':
        a, b = y[..., :half], y[..., half:width]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., width:]], -1)
    a, b = y[..., 0:width:2], y[..., 1:width:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), y[..., width:]], -1)


def _plain_rotate(s):
    case = s['case']
    positions = s['positions'].flatten()
    x, grad = s['x'].detach().flatten(0, 1), s['grad'].flatten(0, 1)
    out = _turned(x, positions, s['turn'], s['amplitude'], case['width'], case['layout'])
    back = _turned(grad, positions, s['turn'], s['amplitude'], case['width'], case['layout'], True)
    return out.to(x.dtype).view(s['x'].shape), back.to(x.dtype).view(s['x'].shape)


def _plain_enter(s):
    case = s['case']
    world, position = _tokens_at(s, s['start'], case['count'], s['tokens'])
    page, slot = s['table'].long()[world, position // s['page']], position % s['page']
    turned = (position, s['turn'], s['amplitude'], case['width'], case['layout'])
    out = _turned(s['q'].flatten(0, -3), *turned).to(s['q'].dtype).view(s['q'].shape)
    return (out, _put(s, 'k', page, slot, _turned(s['new_k'].flatten(0, -3), *turned)),
            _put(s, 'v', page, slot, s['new_v'].flatten(0, -3)))


def _put(s, name, page, slot, x):
    """Stores rows and returns them as the pages then stand for them."""
    if s['k_scale'] is not None:
        codes, scale = _quantise(x)
        s[name].view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
        s[name + '_scale'][page, :, slot] = scale
        x = _values(s[name].view(torch.uint8)[page, :, slot], s[name + '_scale'][page, :, slot])
    else:
        s[name][page, :, slot] = x.to(s[name].dtype)
        x = s[name][page, :, slot].float()
    shape = s['new_' + name].shape
    return x.to(s['new_' + name].dtype).view(shape)


def _plain_make_room(s, new, over):
    """The pages of restarted worlds and of tokens taken back go onto the stack of free pages, those of new tokens come off
    it; the rows' starts."""
    page, table, length, free = s['page'], s['table'], s['length'].long(), s['free']
    new = new.long()
    base = torch.where(over, 0, length) if over is not None else length
    after = base + new
    held, kept, need = -(-length // page), -(-torch.minimum(base, after) // page), -(-after // page)
    column = torch.arange(table.shape[1], device=DEVICE)
    given = (column >= kept[:, None]) & (column < held[:, None])           # back to the stack, the last one first
    taken = (column >= kept[:, None]) & (column < need[:, None])
    left = s['state'][0].long() + given.sum()
    place = torch.where(given, left - torch.cumsum(given.flatten(), 0).view(given.shape), s['npage'])
    stack = torch.nn.functional.pad(free, (0, 1))
    free.copy_(stack.scatter_(0, place.flatten(), table.flatten())[:-1])
    place = left - torch.cumsum(taken.flatten(), 0).view(taken.shape)
    table.copy_(torch.where(taken, free[place.clamp(0, s['npage'] - 1)], torch.where(given, -1, table)))
    s['state'][0] = left - taken.sum()
    s['length'].copy_(after)
    start = torch.zeros(length.numel() + 1, dtype=torch.int32, device=DEVICE)
    start[1:] = torch.cumsum(new.clamp(min=0), 0)
    return start


def _plain_room(s):
    start = _plain_make_room(s, s['new'], s['over'])
    world, position = _tokens_at(s, start, 0, s['tokens'])
    slot = s['table'].long()[world, position // s['page']] * s['page'] + position % s['page']
    maps = world.int(), position.int(), slot.int()
    if s['over'] is None:
        _plain_make_room(s, s['back'], None)
    return (start, *maps, s['table'], s['length'], s['free'], s['state'])


def _plain_summarise(s):
    """Means of the keys of the blocks that the chunk completes."""
    case = s['case']
    block, n = case['block'], case['worlds']
    length = s['length'].long()
    new = torch.full_like(length, case['count']) if s['start'] is None else (s['start'][1:] - s['start'][:-1]).long()
    number = (length - new)[:, None] // block + torch.arange((s['most'] - 1) // block + 1, device=DEVICE)
    world, _ = torch.nonzero((number + 1) * block <= length[:, None], as_tuple=True)
    number = number[(number + 1) * block <= length[:, None]]
    page, inside = s['table'].long()[world, number * block // s['page']], number * block % s['page'] // block
    slots = inside[:, None] * block + torch.arange(block, device=DEVICE)
    if s['k_scale'] is None:
        x = s['k'][page[:, None], :, slots]
    else:
        x = _values(s['k'].view(torch.uint8)[page[:, None], :, slots], s['k_scale'][page[:, None], :, slots])
    codes, e = _codes(x.double().mean(1))
    s['codes'][page, :, inside] = codes
    s['exponent'][page, :, inside] = (e + 127).to(torch.uint8)


def _plain_select(s, world, position):
    """The blocks of every row and key head, in order, -1 behind the last: (rows, kv, listed)."""
    case = s['case']
    block, n, kv, heads = case['block'], case['worlds'], case['kv'], case['heads']
    per = s['page'] // block
    table = s['table'].long().clamp(min=0)
    codes = s['codes'][table].permute(0, 2, 1, 3, 4).flatten(2, 3)         # (worlds, kv, blocks, dim)
    power = torch.exp2(s['exponent'][table].permute(0, 2, 1, 3).flatten(2).float() - 127.0)
    number = torch.arange(table.shape[1] * per, device=DEVICE)
    q, e = _codes(s['q'].flatten(0, -3).double())
    # the chunks side by side, padded to the longest
    place = torch.arange(s['most'], device=DEVICE)
    if s['start'] is None:
        row = torch.arange(n, device=DEVICE)[:, None] * s['most'] + place
    else:
        row = (s['start'][:-1].long()[:, None] + place).clamp(max=s['tokens'] - 1)
    rows = q.float()[row].view(n, s['most'], kv, heads // kv, -1).permute(0, 2, 1, 3, 4).flatten(2, 3)
    # products of whole numbers, exact in 32 bits
    dots = torch.matmul(rows, codes.float().transpose(2, 3)).view(n, kv, s['most'], heads // kv, -1)
    e = torch.exp2(e.float())[row].view(n, s['most'], kv, heads // kv).transpose(1, 2)
    scores = (dots * e[..., None]).amax(3) * power[:, :, None]
    if s['start'] is None:
        scores = scores.transpose(1, 2).reshape(s['tokens'], kv, -1)
    else:
        scores = scores.transpose(1, 2)[world, torch.arange(s['tokens'], device=DEVICE) - s['start'].long()[world]]
    high = position + 1 if case.get('causal', True) else s['length'].long()[world]
    own_block = (position // block)[:, None]
    listed_one = (number < case['first']) | (number > own_block - case['near'])
    is_one = number * block < high[:, None]
    scores = scores.masked_fill((listed_one | ~is_one)[:, None], -math.inf)
    best = torch.sort(scores, dim=-1, descending=True, stable=True)            # equal ones in their order
    best_scores, best_number = best.values[..., :case['top']], best.indices[..., :case['top']]
    chosen = torch.zeros(scores.shape, dtype=torch.bool, device=DEVICE)
    chosen.scatter_(2, best_number, best_scores > -math.inf)
    chosen |= (listed_one & is_one)[:, None]
    found = torch.where(chosen, number, number.numel()).sort(-1).values[..., :_listed_blocks(case)]
    found = torch.where(found < number.numel(), found, -1).int()
    return torch.nn.functional.pad(found, (0, _listed_blocks(case) - found.shape[-1]), value=-1)


def _plain_recall(s):
    case = s['case']
    block, kv, heads, dim = case['block'], case['kv'], case['heads'], case['dim']
    _plain_summarise(s)
    world, position = _tokens_at(s, s['start'], case['count'], s['tokens'])
    blocks = _plain_select(s, world, position)
    high = position + 1 if case.get('causal', True) else s['length'].long()[world]
    key = (blocks.long()[..., None] * block + torch.arange(block, device=DEVICE)).flatten(2)     # (rows, kv, keys)
    seen = (blocks >= 0).repeat_interleave(block, 2) & (key < high[:, None, None])
    key = key.clamp(min=0)
    page, slot = s['table'].long()[world[:, None, None], key // s['page']].clamp(min=0), key % s['page']
    head = torch.arange(kv, device=DEVICE)[None, :, None]

    def held(name):
        if s['k_scale'] is None:
            return s[name][page, head, slot].float()
        return _values(s[name].view(torch.uint8)[page, head, slot], s[name + '_scale'][page, head, slot])

    rows = s['q'].flatten(0, -3).float().view(s['tokens'], kv, heads // kv, dim)
    scores = torch.matmul(rows, held('k').transpose(2, 3)) * (1.0 / math.sqrt(dim))
    scores = scores.masked_fill(~seen[:, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights, held('v')) / weights.sum(-1, keepdim=True)
    return blocks.view(s['q'].shape[:-2] + blocks.shape[1:]), out.to(s['q'].dtype).view(s['q'].shape), s['codes'], s['exponent']


def run(state):
    if own:
        return _own(state)
    do = state['case']['do']
    if do == 'rotate':
        return _plain_rotate(state)
    if do == 'enter':
        return _plain_enter(state)
    if do == 'room':
        return _plain_room(state)
    return _plain_recall(state)


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case['do'] == 'rotate':
        values = case['batch'] * case['tokens'] * case['heads'] * case['dim']
        turned = values * case['width'] / case['dim']
        return dict(bytes=4.0 * values * SIZE[case['input']] + 8.0 * case['batch'] * case['tokens'], flops=6.0 * turned)
    new, total = _case_sizes(case)
    tokens = int(new.sum())
    if case['do'] == 'room':
        # per world its count, its length in and out and the rows' start; per page that changes hands a table entry in or out
        # and a place of the stack; per row its three numbers, and the page that it lies in
        past = total if case.get('restart') else total - new
        held, before = -(-total // case['page']), -(-past // case['page'])
        changed = int((held + before).sum()) if case.get('restart') else 2 * int((held - before).sum())
        touched = int((held - (total - new) // case['page']).sum())
        return dict(bytes=case['worlds'] * (17.0 if case.get('restart') else 28.0) + 8.0 * changed + 12.0 * tokens
                    + 4.0 * touched, flops=0.0)
    kv, dim = case['kv'], case['dim']
    entry = dim * SIZE[case['store']] if case['store'] != 'fp8' else dim + dim // BLOCK     # one key of one head, stored
    row = kv * dim * SIZE[case['input']]
    queries = tokens * case['heads'] * dim * SIZE[case['input']]
    if case['do'] == 'enter':      # queries in and out; keys and values in, their entries out, the entries in, the values out
        turned = tokens * (case['heads'] + kv) * case['width']
        return dict(bytes=2.0 * queries + 2.0 * tokens * (2 * row + 2 * kv * entry), flops=3.0 * turned)
    block = case['block']
    lists = _listed_blocks(case)
    nbytes, flops = 2.0 * queries + 4.0 * tokens * kv * lists, 0.0
    for count, length in zip(new.tolist(), total.tolist()):
        if not count:
            continue
        position = np.arange(length - count, length)
        at = position // block                                      # the query's own block
        high = position + 1 if case.get('causal', True) else np.full(count, length)
        scored = np.maximum(0, at - case['near'] + 1 - case['first'])
        first = np.minimum(case['first'], np.maximum(0, at - case['near'] + 1))
        late = high - np.maximum(0, at - case['near'] + 1) * block  # keys from the first near block on
        keys = late + (np.minimum(scored, case['top']) + first) * block
        done = length // block - (length - count) // block          # blocks that the chunk completes
        nbytes += kv * (done * (block * entry + dim + 1) + int(scored.max()) * (dim + 1))
        nbytes += 2.0 * kv * entry * min(int(keys.sum()), length)   # keys that several queries see are read once
        flops += 2.0 * dim * case['heads'] * int(scored.sum()) + 4.0 * dim * case['heads'] * int(keys.sum())
    return dict(bytes=nbytes, flops=flops)


# ---------------------------------------------------------------------------- the definitions, in 64 bits
def _stored64(x, store):
    """What new values stand for once they are stored."""
    if store != 'fp8':
        return x.to(TYPES[store]).double()
    shape = x.shape
    x = x.double().reshape(-1, BLOCK)
    most = x.abs().max(1, keepdim=True).values
    power = torch.full_like(most, -117.0)
    held = most > 0
    least = torch.ceil(torch.log2(most[held] / LARGEST))
    # the logarithm's rounding may be one off at powers of two: settle it by the definition
    least = torch.where(LARGEST * torch.exp2(least - 1) >= most[held], least - 1, least)
    least = torch.where(LARGEST * torch.exp2(least) < most[held], least + 1, least)
    power[held] = least.clamp(min=-117.0)
    y = x * torch.exp2(-power)
    grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(min=-6.0) - 3.0)
    return (torch.round(y / grid) * grid * torch.exp2(power)).reshape(shape)


def _turned64(x, positions, s, back=False):
    """Pairs as complex numbers times amplitude * e^(i position turn)."""
    case, y = s['case'], x.detach().double().clone()
    half = case['width'] // 2
    one, two = (slice(0, half), slice(half, 2 * half)) if case['layout'] == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    angle = positions.double()[..., None, None] * s['turn'] * (-1 if back else 1)
    z = torch.complex(y[..., one], y[..., two]) * torch.polar(torch.full_like(angle, s['amplitude']), angle)
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _codes64(x):
    """Whole numbers and the power of two that they count, by the definition."""
    most = x.abs().amax(-1, keepdim=True)
    power = torch.ceil(torch.log2(most.clamp(min=1e-300) / MOST))
    power = torch.where(MOST * torch.exp2(power - 1) >= most, power - 1, power)
    power = torch.where(MOST * torch.exp2(power) < most, power + 1, power).clamp(-POWER, POWER)
    return torch.round(x / torch.exp2(power)).clamp(-MOST, MOST), power.squeeze(-1)


def _recall64(case, rows, position, k, v, codes, power):
    """One world's rows over its keys and values (kv, tokens, dim) with the summaries of its blocks."""
    block, kv, length, full, count = case['block'], case['kv'], k.shape[1], codes.shape[1], rows.shape[0]
    rows = rows.view(count, kv, -1, case['dim'])
    q, e = _codes64(rows)
    marks = (torch.einsum('nkgd,kbd->nkgb', q, codes) * torch.exp2(e)[..., None]).amax(2) * torch.exp2(power)
    number = torch.arange(-(-length // block), device=DEVICE)
    high = position + 1 if case.get('causal', True) else torch.full_like(position, length)
    always = (number[None] > (position // block)[:, None] - case['near']) | (number < case['first'])
    rest = ~always[:, :full] & (number[:full] * block < high[:, None])
    order = torch.argsort(torch.where(rest[:, None], marks, -math.inf), dim=-1, descending=True, stable=True)[..., :case['top']]
    picked = torch.zeros(marks.shape, dtype=torch.bool, device=DEVICE).scatter_(2, order, True) & rest[:, None]
    sees = always[:, None].repeat(1, kv, 1)
    sees[..., :full] |= picked
    sees = sees.repeat_interleave(block, 2)[..., :length] & (torch.arange(length, device=DEVICE) < high[:, None])[:, None]
    scores = torch.einsum('nkgd,ktd->nkgt', rows, k) / math.sqrt(case['dim'])
    weights = torch.softmax(torch.where(sees[:, :, None], scores, -math.inf), -1)
    return torch.einsum('nkgt,ktd->nkgd', weights, v).reshape(count, case['heads'], case['dim'])


def exact(case, seed):
    if case['do'] == 'room':                               # whole numbers alone
        return None
    s = prepare(case, seed)
    if case['do'] == 'rotate':
        return _turned64(s['x'], s['positions'], s), _turned64(s['grad'], s['positions'], s, True)
    n, total = case['worlds'], s['length'].tolist()
    begins = s['start'].tolist() if s['start'] is not None else [i * case['count'] for i in range(n + 1)]
    if case['do'] == 'enter':
        position = torch.cat([torch.arange(total[w] - (begins[w + 1] - begins[w]), total[w], device=DEVICE) for w in range(n)])
        position = position.view(s['q'].shape[:-2])
        k = _turned64(s['new_k'], position, s)
        return (_turned64(s['q'], position, s), _stored64(k, case['store']),
                _stored64(s['new_v'], case['store']))
    page, block, kv, heads, dim = case['page'], case['block'], case['kv'], case['heads'], case['dim']
    if s['tokens'] * kv > 40000:                           # one row and head at a time: too many
        return None
    out = []
    for w in range(n):
        count, length = begins[w + 1] - begins[w], total[w]
        if not count:
            continue
        ids = s['table'][w, :-(-length // page)].long()
        k, v = ((_values(s[name].view(torch.uint8)[ids], s[name + '_scale'][ids]) if s['k_scale'] is not None else s[name][ids])
                .double().transpose(0, 1).reshape(kv, -1, dim)[:, :length] for name in ('k', 'v'))
        full = length // block
        codes, power = _codes64(k[:, :full * block].reshape(kv, full, block, dim).sum(2) / block)
        rows = s['q'].reshape(-1, heads, dim)[begins[w]:begins[w + 1]].double()
        position = torch.arange(length - count, length, device=DEVICE)
        for at in range(0, count, 64):                     # some rows at a time: the scores are large
            out.append(_recall64(case, rows[at:at + 64], position[at:at + 64], k, v, codes, power))
    out = torch.cat(out).view(s['q'].shape) if out else s['q'].double()
    return None, out, None, None
