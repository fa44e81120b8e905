"""How the episode memory's calls are made on the GPU: what is refused and with which error, streams of the caller's
and of the cache, and what a call may be captured with."""
import pytest

from libero_hip import episodes
from test_gpu_episodes import World

pytestmark = pytest.mark.gpu


def test_refusals_of_the_library_are_value_errors(gpu_available):
    """Arguments that only the library refuses: more than 1024 query heads to a key head, a scale that is finite in
    64 bits and not in 32, more workgroups than a launch counts."""
    import torch
    print('case library refusals', flush=True)
    p = World([5, 20], 1, 32, 16, 'bf16', seed=40).pages
    q = torch.zeros((2, 1, 1025, 32), dtype=torch.bfloat16, device='cuda')
    with pytest.raises(ValueError, match='1024 query heads'):
        episodes.attend(p, q)
    assert not episodes.attend(p, q[:, :, :1024], scale=1.0).isnan().any()
    with pytest.raises(ValueError, match='do not fit'):
        episodes.attend(p, q[:, :, :4], scale=1e39)
    n = 2 ** 21
    pages = torch.zeros((1, 8, 16, 32), dtype=torch.bfloat16, device='cuda')
    p = episodes.Pages(pages, pages, torch.zeros((n, 1), dtype=torch.int32, device='cuda'),
                       torch.ones(n, dtype=torch.int32, device='cuda'))
    with pytest.raises(ValueError, match='workgroups'):
        episodes.attend(p, pages[:1, :, :1].transpose(1, 2).expand(n, 1, 8, 32))


def delayed(cycles=200_000_000):
    """A stream that is busy for about a tenth of a second."""
    import torch
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(cycles)
    return side


def filled(shape, dtype):
    """Allocations of the current stream that take whatever memory has been given back."""
    import torch
    return [torch.full(shape, 77, dtype=dtype, device='cuda') for _ in range(3)]


def test_tensors_may_be_dropped_after_a_call_on_another_stream(gpu_available):
    """What a call on a stream of its own reads is kept for it, though the caller drops it and allocates anew."""
    import torch
    print('case dropped tensors', flush=True)
    world = World([700, 301], 2, 64, 16, 'bf16', seed=41)
    p = world.pages
    q = torch.randn((70, 4, 64), device='cuda').bfloat16()
    kv = [torch.randn((70, 2, 64), device='cuda').bfloat16() for _ in range(2)]
    start = torch.tensor([0, 30, 70], dtype=torch.int32, device='cuda')
    episodes.write(p, *kv, start)
    want = episodes.attend(p, q, start)
    episodes.write(p, kv[0] * 0, kv[1] * 0, start)
    q2, first, k2, v2 = q.clone(), start.clone(), kv[0].clone(), kv[1].clone()
    torch.cuda.synchronize()
    side = delayed()
    episodes.write(p, k2, v2, first, stream=side)
    del k2, v2
    read = episodes.read(p, first, tokens=70, stream=side)
    out = episodes.attend(p, q2, first, stream=side)
    del q2, first
    junk = filled((70, 2, 64), torch.bfloat16), filled((70, 4, 64), torch.bfloat16), filled((3,), torch.int32)
    assert not side.query()                        # the calls were still to come
    torch.cuda.synchronize()
    assert torch.equal(read[0], kv[0]) and torch.equal(read[1], kv[1]) and torch.equal(out, want)
    del junk


def test_cache_reads_on_another_stream(gpu_available):
    """The rows' starts that EpisodeCache.read uploads itself stay whole until the stream has read them."""
    import torch
    print('case cache read elsewhere', flush=True)
    c = episodes.EpisodeCache(6, kv_heads=2, head_dim=64, tokens=100, storage='bf16', page_tokens=16)
    chunk = c.extend([50, 1, 20, 0, 100, 37], range(6))
    k = torch.randn((chunk.tokens, 2, 64), device='cuda').bfloat16()
    c.write(chunk, k, -k)
    torch.cuda.synchronize()
    side = delayed()
    x, y, starts = c.read([0, 2, 5], stream=side)
    junk = filled((7,), torch.int32)
    assert not side.query()
    torch.cuda.synchronize()
    want = torch.cat([k[0:50], k[51:71], k[171:208]])
    assert torch.equal(x, want) and torch.equal(y, -want) and starts.tolist() == [0, 50, 70, 107]
    del junk


@pytest.mark.parametrize('given', [True, False])
@pytest.mark.parametrize('busy', ['calls', 'changes', 'both'])
def test_cache_calls_and_changes_keep_their_order(gpu_available, busy, given):
    """Tables and lengths change on one stream, calls run on another: each sees the worlds as they were when it was
    called, whichever stream is behind, with pages that go from world to world."""
    import contextlib
    import torch
    print('case cache order', busy, given, flush=True)
    n, heads, steps = 5, 4, 6
    gen = torch.Generator('cuda').manual_seed(8)
    rows = [[torch.randn((n, 3, 2, 64), generator=gen, device='cuda').bfloat16() for _ in range(2)]
            + [torch.randn((n, 3, heads, 64), generator=gen, device='cuda').bfloat16()] for _ in range(steps)]

    def play(side):
        c = episodes.EpisodeCache(n, kv_heads=2, head_dim=64, tokens=64, storage='bf16', page_tokens=16, pages=9)
        c.table.add_(0), c.length.add_(0)
        torch.cuda.synchronize()
        outs = []
        for i, (k, v, q) in enumerate(rows):
            if side is not None and busy != 'changes':
                with torch.cuda.stream(side):
                    torch.cuda._sleep(20_000_000)
            if side is not None and busy != 'calls':
                torch.cuda._sleep(20_000_000)
            chunk = c.extend(3)
            with contextlib.nullcontext() if given or side is None else torch.cuda.stream(side):
                options = dict(stream=side) if given else {}
                c.write(chunk, k, v, **options)
                outs.append(c.attend(chunk, q, **options))
            if i == 2:
                c.reset([0, 3, 4])
            if i == 3:
                c.reset()
        torch.cuda.synchronize()                     # calls among each other are the caller's to order
        x, y, starts = c.read()
        return outs + [x, y], starts

    want, starts = play(None)
    got, again = play(torch.cuda.Stream())
    assert starts.tolist() == again.tolist() == [0, 6, 12, 18, 24, 30]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_streams_of_other_devices_are_refused(gpu_available):
    """A stream of another GPU was passed over for the current one without a word."""
    import types
    import torch
    print('case stream of another device', flush=True)
    other = types.SimpleNamespace(device=torch.device('cuda', 1), cuda_stream=1234567)
    c = episodes.EpisodeCache(2, kv_heads=2, head_dim=64, tokens=10, storage='bf16')
    chunk, p = c.extend(1), c.layers[0]
    q = torch.zeros((2, 1, 2, 64), dtype=torch.bfloat16, device='cuda')
    for call in (lambda: episodes.write(p, q, q, stream=other), lambda: episodes.read(p, count=1, stream=other),
                 lambda: episodes.attend(p, q, stream=other), lambda: c.write(chunk, q, q, stream=other),
                 lambda: c.attend(chunk, q, stream=other), lambda: c.read(stream=other)):
        with pytest.raises(ValueError, match='device'):
            call()


def test_tangents_are_refused(gpu_available):
    """A result without the tangent that its inputs had would be a derivative of zero."""
    import torch
    from torch.autograd import forward_ad
    print('case tangents', flush=True)
    p = World([5, 20], 2, 64, 16, 'bf16', seed=42).pages
    q = torch.randn((2, 1, 4, 64), device='cuda').bfloat16()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: episodes.attend(p, dual), lambda: episodes.write(p, q[:, :, :2], dual[:, :, :2]),
                     lambda: episodes.attend(p, q, out=forward_ad.make_dual(q.clone(), q))):
            with pytest.raises(ValueError, match='dual'):
                call()
        assert torch.equal(episodes.attend(p, forward_ad.unpack_dual(dual).primal), episodes.attend(p, q))


def test_pages_with_gradients_are_refused(gpu_available):
    """Keys or values that are being trained would get no gradient from attend."""
    import torch
    print('case pages with gradients', flush=True)
    p = World([5, 20], 2, 64, 16, 'bf16', seed=43).pages
    trained = torch.nn.Parameter(p.v.clone())
    for k, v in ((p.k, trained), (trained, p.v)):
        with pytest.raises(ValueError, match='backward'):
            episodes.Pages(k, v, p.table, p.length)
    episodes.Pages(p.k, trained.detach(), p.table, p.length)
    with torch.no_grad():
        episodes.Pages(p.k, trained, p.table, p.length)


def test_rows_beyond_32_bits_are_refused(gpu_available):
    """2^32 rows were counted as none: nothing was written, and the call returned as if it had."""
    import torch
    print('case rows beyond 32 bits', flush=True)
    p = World([5, 20], 2, 64, 16, 'bf16', seed=44).pages
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device='cuda')
    x = torch.zeros((1, 1, 2, 64), dtype=torch.bfloat16, device='cuda')
    for n in (2 ** 30, 2 ** 31):
        with pytest.raises(ValueError, match='rows'):
            episodes.write(p, x.expand(2, n, 2, 64), x.expand(2, n, 2, 64))
        with pytest.raises(ValueError, match='rows'):
            episodes.write(p, x[0].expand(2 * n, 2, 64), x[0].expand(2 * n, 2, 64), start)
        with pytest.raises(ValueError, match='rows'):
            episodes.read(p, count=n)
        with pytest.raises(ValueError, match='rows'):
            episodes.attend(p, x.expand(2, n, 2, 64))


def test_captured_attention_follows_larger_chunks(gpu_available):
    """A graph of the cache's ragged attention, replayed with rows dealt to the worlds in other numbers than those it
    was captured with: all rows are computed."""
    import torch
    print('case captured chunks', flush=True)
    for heads, counts in ((2, [1, 5, 2]), (4, [10, 50, 30])):
        c = episodes.EpisodeCache(3, kv_heads=2, head_dim=64, tokens=200, storage='bf16', page_tokens=16)
        total = sum(counts)
        past = c.extend(100)
        c.write(past, *(torch.randn(past.shape + (2, 64), device='cuda').bfloat16() for _ in range(2)))
        chunk = c.extend(counts)
        c.write(chunk, *(torch.randn((total, 2, 64), device='cuda').bfloat16() for _ in range(2)))
        q = torch.randn((total, heads, 64), device='cuda').bfloat16()
        out = torch.empty_like(q)
        c.attend(chunk, q, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.attend(chunk, q, out=out)
        for new in (counts, [total - 2, 1, 1], [0, 0, total], [0, total, 0]):
            chunk.start.copy_(torch.tensor([0, new[0], new[0] + new[1], total], dtype=torch.int32))
            out.fill_(9)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, episodes.attend(c.layers[0], q, chunk.start))


def test_results_that_share_memory_are_refused(gpu_available):
    """An expanded out: rows would overwrite each other, the last one to come winning."""
    import torch
    print('case shared out', flush=True)
    p = World([5, 20], 2, 64, 16, 'bf16', seed=45).pages
    q = torch.randn((2, 1, 4, 64), device='cuda').bfloat16()
    for out in (torch.zeros_like(q[:1]).expand(2, 1, 4, 64), torch.zeros_like(q[:, :, :1]).expand(2, 1, 4, 64)):
        with pytest.raises(ValueError, match='share'):
            episodes.attend(p, q, out=out)
    out = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device='cuda').as_strided((2, 1, 4, 64), (256, 0, 64, 1))
    assert torch.equal(episodes.attend(p, q, out=out), episodes.attend(p, q))


def test_captured_on_the_stream_that_is_given(gpu_available):
    """Calls with stream= that go into a graph on that stream, of the operators and of the cache: replays give what
    eager calls give, and memory that was dropped since is not the graph's."""
    import torch
    print('case captured stream', flush=True)
    side = torch.cuda.Stream()
    c = episodes.EpisodeCache(3, kv_heads=2, head_dim=64, tokens=2000, storage='fp8')
    past = c.extend([900, 40, 1500])
    c.write(past, *(torch.randn(past.shape + (2, 64), device='cuda').bfloat16() for _ in range(2)))
    chunk = c.extend(2)
    k, v = (torch.randn((3, 2, 2, 64), device='cuda').bfloat16() for _ in range(2))
    q = torch.randn((3, 2, 4, 64), device='cuda').bfloat16()
    outs = [torch.empty_like(q) for _ in range(2)]

    def calls():
        c.write(chunk, k, v, stream=side)
        c.attend(chunk, q, out=outs[0], stream=side)
        episodes.attend(c.layers[0], q, out=outs[1], stream=side)

    torch.cuda.synchronize()
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls()
    for _ in range(3):
        for x in (k, v, q):
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        junk = filled((3, 2, 4, 64), torch.bfloat16)
        want = episodes.attend(c.layers[0], q)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    del junk
