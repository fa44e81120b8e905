"""The arithmetic of rotary positions, bit for bit: two products and their sum, each rounded to 32 bits, from sines and cosines
rounded once to 32, then one rounding to what the rows are stored in.

The sines and cosines are the framework's own, read out by turning the pair (1, 0): 1 c - 0 s and 1 s + 0 c are exact.  torch
on the CPU computes each operation by itself, so nothing is fused there."""
import pytest

from libero_hip import episodes, rotary
from test_gpu_episodes import World, dtype_of

pytestmark = pytest.mark.gpu


def halves(width, layout):
    return (slice(0, width // 2), slice(width // 2, width)) if layout == 'half' else (slice(0, width, 2), slice(1, width, 2))


def turned(turning, x, positions, back=False):
    """x (rows, heads, dim) in float32, turned as stated above, on the CPU."""
    import torch
    one, two = halves(turning.width, turning.layout)
    unit = torch.zeros((len(positions), 1, turning.width), device='cuda')
    unit[..., one] = 1.0
    unit = rotary.rotate(turning, unit, positions, back=back).cpu()
    c, s = unit[..., one], unit[..., two]
    x = x.float().cpu()
    y, a, b = x.clone(), x[..., one], x[..., two]
    y[..., one] = a * c - b * s
    y[..., two] = a * s + b * c
    return y


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('dim,width', [(128, 128), (96, 48), (80, 20), (7, 6)])
def test_rotate_bits(gpu_available, dim, width, kind, layout):
    import torch
    print('case rotate bits', dim, width, kind, layout, flush=True)
    gen = torch.Generator('cuda').manual_seed(dim)
    turning = rotary.Rotary.make(width, layout=layout, amplitude=1.2079)
    x = torch.randn((700, 3, dim), generator=gen, device='cuda').to(dtype_of(kind))
    positions = torch.randint(0, 1 << 20, (700,), generator=gen, device='cuda')
    for back in (False, True):
        got = rotary.rotate(turning, x, positions, back=back).cpu()
        assert torch.equal(got, turned(turning, x, positions, back).to(x.dtype))


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('store', ['bf16', 'f16', 'fp8'])
@pytest.mark.parametrize('kind', ['f32', 'bf16', 'f16'])
def test_entered_bits(gpu_available, kind, store, layout):
    """Millions of keys, so that those that lie next to a border of the pages' type are among them: float32 rows into 16 bits are
    where a fused product shows (one key in 50000, in float16 one in 8700)."""
    import torch
    print('case enter bits', kind, store, layout, flush=True)
    n, kv, dim, width, page = 1500, 8, 128, 128, 64
    gen = torch.Generator('cuda').manual_seed(1)
    turning = rotary.Rotary.make(width, layout=layout)
    world, other = (World([0], kv, dim, page, store, spare=-(-n // page), width=-(-n // page)) for _ in range(2))
    for x in (world, other):
        x.pages.table.copy_(torch.arange(x.pages.table.numel(), dtype=torch.int32).view(1, -1))
        x.pages.length.fill_(n)
    for seed in range(3):
        q = torch.randn((1, n, 2, dim), generator=gen, device='cuda').to(dtype_of(kind))
        k, v = (torch.randn((1, n, kv, dim), generator=gen, device='cuda').to(dtype_of(kind)) for _ in range(2))
        out = rotary.enter(world.pages, turning, q, k, v)
        positions = torch.arange(n, device='cuda')
        assert torch.equal(out[0].cpu(), turned(turning, q[0], positions).to(q.dtype))
        want = turned(turning, k[0], positions)
        got = episodes.read(world.pages, count=n, dtype=torch.float32)
        if store == 'fp8':                           # quantised as write does
            episodes.write(other.pages, want[None].cuda(), v.float())
            assert all(torch.equal(a, b) for a, b in zip(got, episodes.read(other.pages, count=n, dtype=torch.float32)))
        else:
            assert torch.equal(got[0][0].cpu(), want.to(dtype_of(store)).float())
            assert torch.equal(got[1][0].cpu(), v[0].cpu().float().to(dtype_of(store)).float())
