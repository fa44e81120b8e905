"""Rotary positions on the GPU against their definition in 64 bits (tests/recall_reference.py).

Tolerance, from the arithmetic: sine and cosine, times the amplitude, are rounded once to 32 bits (2^-24), a product and the sum
round once more each (2^-24): three of the four that are allowed for.  With pairs (a, b): |error| <= amplitude (|a| + |b|) 2^-22 + u |y|, u the unit
roundoff of the result, and for float16 half its smallest step, 2^-25.  Positions whose angle passes 2^24 add the angle's own rounding in 64 bits, three
of 2^-53 each.
"""
import numpy as np
import pytest

from recall_reference import turned
from libero_hip import episodes, rotary
from test_gpu_episodes import World, dtype_of

UNIT = {'f32': 2.0 ** -24, 'bf16': 2.0 ** -8, 'f16': 2.0 ** -11}
pytestmark = pytest.mark.gpu


def sizes(x, half, layout, amplitude):
    """amplitude (|a| + |b|) of the pair that each value belongs to."""
    size = np.zeros(x.shape)
    one, two = (slice(0, half), slice(half, 2 * half)) if layout == 'half' else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    size[..., one] = size[..., two] = abs(amplitude) * (np.abs(x[..., one]) + np.abs(x[..., two]))
    return size


def bound(x, want, turning, positions, kind):
    turn = turning.turn.cpu().numpy()
    angle = np.abs(np.asarray(positions, np.float64)).max(initial=0) * np.abs(turn).max()
    size = sizes(x, len(turn), turning.layout, turning.amplitude)
    return size * (2.0 ** -22 + 3 * 2.0 ** -53 * angle) + UNIT[kind] * np.abs(want) + (2.0 ** -25 if kind == 'f16' else 2.0 ** -126)


def compare(got, x, positions, turning, kind, back=False):
    x = x.double().cpu().numpy()
    want = turned(x, positions, turning.turn.cpu().numpy(), turning.amplitude, turning.layout, back)
    error = np.abs(got.detach().double().cpu().numpy().reshape(want.shape) - want)
    limit = bound(x, want, turning, positions, kind)
    assert np.all(error <= limit), (error / limit).max()


def made(shape, kind, seed=0):
    import torch
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape)).to(dtype_of(kind)).cuda()


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('dim,width', [(64, 64), (128, 128), (256, 256), (96, 48), (80, 20), (32, 2), (7, 6), (1024, 1024), (2, 2)])
def test_rotate(gpu_available, dim, width, kind, layout):
    """Whole and partial heads, odd sizes; positions of both signs, near and far, in both whole types."""
    import torch
    print('case rotate', dim, width, kind, layout, flush=True)
    turning = rotary.Rotary.make(width, layout=layout, amplitude=1.25)
    x = made((37, 3, dim), kind, dim)
    p = np.concatenate([np.arange(20), [-1, -77, 1000, 65535, 65536, 10 ** 6, 2 ** 24 + 1, 2 ** 30, 2 ** 31 - 1, -2 ** 31],
                        np.random.default_rng(1).integers(-5000, 5000, 7)])
    for whole in (torch.int32, torch.int64):
        positions = torch.from_numpy(p).to(whole).cuda()
        got = rotary.rotate(turning, x, positions)
        assert got.shape == x.shape and got.dtype == x.dtype
        compare(got, x, p, turning, kind)
        compare(rotary.rotate(turning, x, positions, back=True), x, p, turning, kind, back=True)
        assert torch.equal(got[..., width:], x[..., width:])


@pytest.mark.parametrize('kind,offset', [('f32', 0), ('bf16', 0), ('bf16', 1), ('f16', 4), ('f32', 3)])
def test_strides_and_batches(gpu_available, kind, offset):
    """Rows inside a wider tensor at any alignment, positions for a whole batch or one to a row, results into a part of a
    tensor whose rest stays."""
    import torch
    print('case strides', kind, offset, flush=True)
    turning = rotary.Rotary.make(32)
    base = made((4 * 9 * 200 + 8,), kind)
    x = base[offset:].as_strided((4, 9, 3, 48), (9 * 200, 200, 56, 1))
    row = torch.arange(9, dtype=torch.int32, device='cuda') * 5
    target = torch.zeros((4, 9, 2, 3, 50), dtype=x.dtype, device='cuda')
    out = target[:, :, 1, :, offset % 3:offset % 3 + 48]
    got = rotary.rotate(turning, x, row, out=out)
    assert got is out
    compare(got, x.reshape(36, 3, 48), row.cpu().numpy().tolist() * 4, turning, kind)
    each = torch.randint(0, 1000, (4, 9), device='cuda')
    got = rotary.rotate(turning, x, each)
    compare(got, x.reshape(36, 3, 48), each.flatten().cpu().numpy(), turning, kind)
    out.zero_()
    assert not target.any()
    one = rotary.rotate(turning, x[:, :1], row[:1])
    compare(one, x[:, 0], [0] * 4, turning, kind)


def test_empty(gpu_available):
    import torch
    turning = rotary.Rotary.make(32)
    for shape in ((0, 2, 32), (3, 0, 32), (2, 0, 2, 32), (0, 5, 2, 32)):
        x = torch.empty(shape, device='cuda')
        p = torch.zeros(shape[:-2], dtype=torch.int32, device='cuda')
        assert rotary.rotate(turning, x, p).shape == x.shape


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_gradient(gpu_available, layout):
    """Against the formula and against differences in 64 bits; of a leaf, of a part of a tensor, and twice."""
    import torch
    print('case gradient', layout, flush=True)
    turning = rotary.Rotary.make(24, layout=layout, amplitude=0.75)
    p = np.array([0, 3, 1000, 5, 2, 99])
    positions = torch.from_numpy(p).cuda()
    wide = made((6, 3, 2, 32), 'f32').requires_grad_()
    x = wide[:, 1]
    weight = made((6, 2, 32), 'f32', 1)
    out = rotary.rotate(turning, x, positions)
    grad, = torch.autograd.grad((out * weight).sum(), wide)
    compare(grad[:, 1], weight, p, turning, 'f32', back=True)
    assert not grad[:, 0].any() and not grad[:, 2].any()
    # differences: the rotation is linear, so that they are exact but for the rounding of the definition's 64 bits
    base, step = x.detach().double().cpu().numpy(), np.zeros((6, 2, 32))
    rng = np.random.default_rng(2)
    for _ in range(20):
        at = rng.integers(6), rng.integers(2), rng.integers(32)
        step[at] = 1.0
        args = p, turning.turn.cpu().numpy(), turning.amplitude, layout
        difference = ((turned(base + step, *args) - turned(base - step, *args)) / 2 * weight.double().cpu().numpy()).sum()
        # a sum of two products of at most |weight|'s pair
        assert abs(grad[:, 1][at].item() - difference) <= 2.0 ** -21 * np.abs(weight[at[0], at[1]].cpu().numpy()).max() * 2
        step[at] = 0.0
    # the gradient's gradient is a rotation again
    out = rotary.rotate(turning, x, positions)
    cotangent = weight.clone().requires_grad_()
    first, = torch.autograd.grad(out, x, cotangent, create_graph=True)
    second, = torch.autograd.grad(first, cotangent, weight)
    compare(second, weight, p, turning, 'f32')
    # positions that change in between are found
    out = rotary.rotate(turning, x, positions)
    positions.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(out, x, weight)
    positions.sub_(1)
    # no rows, a batch of one token, a cotangent of other strides
    for shape in ((0, 2, 32), (3, 0, 2, 32)):
        y = torch.empty(shape, device='cuda', requires_grad=True)
        at = torch.zeros(shape[:-2], dtype=torch.int32, device='cuda')
        grad, = torch.autograd.grad(rotary.rotate(turning, y, at), y, torch.empty(shape, device='cuda'))
        assert grad.shape == shape
    y, c = made((6, 1, 2, 32), 'f32').requires_grad_(), made((6, 2, 32, 1), 'f32', 3).permute(0, 3, 1, 2)
    grad, = torch.autograd.grad(rotary.rotate(turning, y, positions.view(6, 1), back=True), y, c)
    compare(grad[:, 0], c[:, 0], p, turning, 'f32')
    c = made((2, 6, 32), 'f32', 4).transpose(0, 1)
    grad, = torch.autograd.grad(rotary.rotate(turning, x, positions), x, c)
    compare(grad, c, p, turning, 'f32', back=True)
    # an expanded cotangent, in 16 bits
    y = made((6, 2, 32), 'bf16').requires_grad_()
    rotary.rotate(turning, y, positions).sum().backward()
    compare(y.grad, torch.ones_like(y), p, turning, 'bf16', back=True)


def test_captured_and_other_streams(gpu_available):
    """Forward and backward in a HIP graph, replayed with other rows and positions; on a stream of its own, whose memory
    stays."""
    import torch
    print('case rotate graph', flush=True)
    turning = rotary.Rotary.make(64)
    x, w = made((5, 40, 4, 64), 'bf16'), made((5, 40, 4, 64), 'bf16', 1)
    positions = torch.arange(40, device='cuda')

    def both(x):
        x = x.detach().requires_grad_()
        out = rotary.rotate(turning, x, positions)
        return out.detach(), torch.autograd.grad(out, x, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(x)
    for step in range(3):
        x.normal_()
        w.normal_()
        positions.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, both(x)):
            assert torch.equal(a, b)
    y = rotary.rotate(turning, x.clone(), positions.clone(), stream=side)
    junk = [torch.full_like(x, 7) for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(y, rotary.rotate(turning, x, positions))
    del junk


def chunk(kind, heads, kv, dim, counts, seed):
    import torch
    n = int(np.sum(counts))
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
    return [made((n, h, dim), kind, seed + i) for i, h in enumerate((heads, kv, kv))] + [start]


LENGTHS, COUNTS = [0, 1, 40, 17, 100, 33], [0, 1, 23, 17, 1, 2]


def positions_of(lengths, counts):
    return np.concatenate([np.arange(l - c, l) for l, c in zip(lengths, counts)])


@pytest.mark.parametrize('layout,part', [('half', 1), ('interleaved', 1), ('half', 2), ('interleaved', 2)])
@pytest.mark.parametrize('kind,store', [('bf16', 'bf16'), ('f16', 'f16'), ('f32', 'bf16'), ('f32', 'f16'), ('bf16', 'fp8'),
                                        ('f16', 'fp8'), ('f32', 'fp8')])
@pytest.mark.parametrize('dim', [32, 64, 96, 128, 256])
def test_enter(gpu_available, dim, kind, store, layout, part):
    """Ragged chunks: the queries and the keys are turned, the keys and the values stored, and nothing else touched."""
    import torch
    print('case enter', dim, kind, store, layout, part, flush=True)
    world, other = (World(LENGTHS, 3, dim, 16, store, seed=14) for _ in range(2))
    turning = rotary.Rotary.make(dim // part, layout=layout, scaling='parts', factor=4.0, original=64, slow=0.5, fast=4.0)
    q, k, v, start = chunk(kind, 5, 3, dim, COUNTS, dim)
    p = positions_of(LENGTHS, COUNTS)
    out = rotary.enter(world.pages, turning, q, k, v, start)
    compare(out, q, p, turning, kind)
    # keys in 32 bits, rounded once by the write that is there: the same bits
    whole = rotary.rotate(turning, k.float(), torch.from_numpy(p).cuda())
    episodes.write(other.pages, whole, v.float(), start)
    for name in ('k', 'v', 'k_scale', 'v_scale'):
        a, b = (getattr(x.pages, name) for x in (world, other))
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
    compare(whole, k.float(), p, turning, 'f32')


@pytest.mark.parametrize('worlds,kind,store', [(1, 'bf16', 'bf16'), (70, 'bf16', 'fp8'), (257, 'f32', 'fp8'), (300, 'f16', 'f16')])
def test_enter_single_tokens(gpu_available, worlds, kind, store):
    import torch
    print('case enter single', worlds, kind, store, flush=True)
    lengths = 1 + np.random.default_rng(worlds).integers(0, 60, worlds)
    world = World(lengths, 2, 64, 16, store, seed=15)
    turning = rotary.Rotary.make(64)
    q, k, v, start = chunk(kind, 8, 2, 64, [1] * worlds, 3)
    four = [x.view(worlds, 1, -1, 64) for x in (q, k, v)]
    out = rotary.enter(world.pages, turning, *four)
    compare(out.view(q.shape), q, lengths - 1, turning, kind)
    packed = rotary.enter(world.pages, turning, q, k, v, start)
    assert torch.equal(out.view(q.shape), packed)
    got = episodes.read(world.pages, count=1, dtype=torch.float32)[1]
    if store != 'fp8':
        assert torch.equal(got.view(v.shape), v.to(dtype_of(store)).float())


def test_enter_without_a_place(gpu_available):
    """Chunks longer than their world, pages that are not there, rows behind the last world's: left as they were."""
    import torch
    print('case enter no place', flush=True)
    world = World([5, 20, 0], 1, 32, 16, 'bf16', seed=16)
    world.pages.table[1, 1] = -1
    before = world.pages.k.clone()
    turning = rotary.Rotary.make(32)
    q, k, v = (made((3, 8, 1, 32), 'bf16', i) for i in range(3))
    out = rotary.enter(world.pages, turning, q, k, v)
    compare(out.view(24, 1, 32), q.view(24, 1, 32), np.concatenate([np.arange(n - 8, n) for n in (5, 20, 0)]), turning, 'bf16')
    got = episodes.read(world.pages, count=8)[0]
    assert not got[0, :3].any() and not got[1, 4:].any() and not got[2].any()
    keep = np.ones(before.shape[:1] + before.shape[2:3], bool)
    keep[world.table[0, 0], :5] = False
    keep[world.table[1, 0], 12:] = False
    keep = torch.from_numpy(keep).cuda()
    assert torch.equal(world.pages.k.transpose(1, 2)[keep].view(torch.int16), before.transpose(1, 2)[keep].view(torch.int16))
    start = torch.tensor([0, 2, 4, 4], dtype=torch.int32, device='cuda')
    target = torch.full((9, 1, 32), 7.0, dtype=torch.bfloat16, device='cuda')
    rotary.enter(world.pages, turning, q.view(24, 1, 32)[:9], k.view(24, 1, 32)[:9], v.view(24, 1, 32)[:9], start, out=target)
    assert bool((target[4:] == 7).all()) and not bool((target[:4] == 7).all())


@pytest.mark.parametrize('offset', [0, 1, 4])
def test_enter_strides(gpu_available, offset):
    """Queries, keys and values as parts of a fused projection, at any alignment."""
    import torch
    print('case enter strides', offset, flush=True)
    worlds = [World([33, 64, 100], 2, 64, 16, 'fp8', seed=11) for _ in range(2)]
    turning = rotary.Rotary.make(64)
    fused = made((3, 21, 600), 'bf16')
    q, k, v = (fused.as_strided((3, 21, h, 64), (21 * 600, 600, 66, 1), offset + at) for h, at in ((4, 0), (2, 264), (2, 400)))
    target = torch.zeros((3, 21, 4, 70), dtype=torch.bfloat16, device='cuda')
    out = target[..., offset:offset + 64]
    rotary.enter(worlds[0].pages, turning, q, k, v, out=out)
    want = rotary.enter(worlds[1].pages, turning, q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(out, want)
    for name in ('k', 'v', 'k_scale', 'v_scale'):
        assert torch.equal(*(getattr(w.pages, name).view(torch.uint8) for w in worlds))


def test_enter_captured(gpu_available):
    """enter and attend in a HIP graph follow the lengths."""
    import torch
    print('case enter graph', flush=True)
    world = World([60, 80, 100], 2, 64, 16, 'bf16', seed=13)
    p = world.pages
    final = p.length.clone()
    turning = rotary.Rotary.make(64, layout='interleaved')
    q, k, v = (torch.randn((3, 2, h, 64), device='cuda').bfloat16() for h in (4, 2, 2))
    rotary.enter(p, turning, q, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = episodes.attend(p, rotary.enter(p, turning, q, k, v))
    for step in range(3):
        p.length.copy_(final - 7 * step)
        k.normal_()
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        kept = got.clone()
        assert torch.equal(kept, episodes.attend(p, rotary.enter(p, turning, q, k, v)))


def test_scores_depend_on_distance(gpu_available):
    """Attention of the last token to a memory moved along by any number of tokens is the same."""
    import torch
    print('case distance', flush=True)
    turning = rotary.Rotary.make(64)
    q, k = made((1, 1, 64), 'f32'), made((1, 1, 64), 'f32', 1)
    scores = [(rotary.rotate(turning, q, torch.tensor([p + 13], device='cuda')) * rotary.rotate(turning, k, torch.tensor([p], device='cuda'))).sum()
              for p in (0, 1, 500, 65536)]
    # two rotations, each within 2^-22 of |a| + |b|, and a sum of 64 products
    limit = 4 * 2.0 ** -21 * (q.abs().sum() * k.abs().max()).item()
    assert max(abs(s - scores[0]).item() for s in scores) <= limit


def test_refusals(gpu_available):
    import torch
    print('case rotary refusals', flush=True)
    turning = rotary.Rotary.make(64)
    x, p = made((4, 2, 64), 'f32'), torch.zeros(4, dtype=torch.int32, device='cuda')
    bad = [lambda: rotary.Rotary(torch.zeros(3, device='cuda')), lambda: rotary.Rotary(torch.zeros(3, dtype=torch.float64)),
           lambda: rotary.Rotary(turning.turn, layout='other'), lambda: rotary.Rotary(turning.turn, amplitude=float('nan')),
           lambda: rotary.Rotary(turning.turn[::2]), lambda: rotary.Rotary(turning.turn.clone().requires_grad_()),
           lambda: rotary.rotate(turning, x[..., :32], p), lambda: rotary.rotate(turning, x, p[:3]),
           lambda: rotary.rotate(turning, x, p.float()), lambda: rotary.rotate(turning, x.double(), p),
           lambda: rotary.rotate(turning, x.cpu(), p), lambda: rotary.rotate(turning, x, p.cpu()),
           lambda: rotary.rotate(turning, x, p, out=x), lambda: rotary.rotate(turning, x, p, out=x.bfloat16()),
           lambda: rotary.rotate(turning, x, p, out=x.new_zeros((1, 2, 64)).expand(4, 2, 64)),
           lambda: rotary.rotate(turning, x.transpose(1, 2), p), lambda: rotary.rotate(turning, x[0], p),
           lambda: rotary.rotate(turning, x.view(2, 2, 2, 64).transpose(0, 1), p.view(2, 2)),
           lambda: rotary.rotate(turning, x.clone().requires_grad_(), p, out=torch.empty_like(x))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('not refused', i)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(ValueError, match='forward-mode'):
            rotary.rotate(turning, fwd.make_dual(x, x), p)
    world = World([5, 20], 1, 64, 16, 'bf16', seed=1)
    q, k = made((2, 1, 4, 64), 'bf16'), made((2, 1, 1, 64), 'bf16')
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device='cuda')
    bad = [lambda: rotary.enter(world.pages, turning, q.float(), k, k), lambda: rotary.enter(world.pages, turning, q[:1], k, k),
           lambda: rotary.enter(world.pages, turning, q, q, q), lambda: rotary.enter(world.pages, turning, q, k, k, start),
           lambda: rotary.enter(world.pages, rotary.Rotary.make(128), q, k, k),
           lambda: rotary.enter(world.pages, turning, q, k, k, out=q), lambda: rotary.enter(world.pages, turning, q[:, :, :0], k, k),
           lambda: rotary.enter(world.pages, turning, q.clone().requires_grad_(), k, k),
           lambda: rotary.enter(world.pages, turning, q, k, k, out=q[:1]), lambda: rotary.enter(world.pages, turning, q.cpu(), k.cpu(), k.cpu())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print('not refused', i)


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_sines_are_rounded_once(gpu_available, layout):
    """Turned units are the amplitude's cosines and sines: within half a step of 32 bits, whatever the amplitude, the angle in
    64 bits to within 2^-36 of an eighth of a turn and three roundings of its own."""
    import torch
    print('case sines', layout, flush=True)
    turn = torch.from_numpy(np.random.default_rng(5).uniform(0.0, 7.0, 64))
    p = np.concatenate([np.arange(70), [1 << 12, -(1 << 12), 99999, 1 << 20]])
    turning = rotary.Rotary(turn.cuda(), layout=layout, amplitude=0.1 * np.log(8.0) + 1.0)
    x = torch.zeros((len(p), 1, 128), device='cuda')
    x[..., :64] = 1.0
    if layout == 'interleaved':
        x = x.view(len(p), 1, 2, 64).transpose(2, 3).reshape(len(p), 1, 128).contiguous()
    got = rotary.rotate(turning, x, torch.from_numpy(p).cuda()).double().cpu().numpy()
    want = turned(x.double().cpu().numpy(), p, turn.numpy(), turning.amplitude, layout)
    angle = np.abs(p).astype(np.float64)[:, None, None] * 7.0
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + turning.amplitude * (2.0 ** -36 + 4 * 2.0 ** -53 * (angle + 1)))
