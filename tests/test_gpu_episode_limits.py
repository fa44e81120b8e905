"""Episode memory on the GPU at the limits of its arguments: lengths, windows, values and weights where the kernels'
numbers of keys, or their 16-bit operands, reach the end of their range.  References and tolerances are those of
test_gpu_episodes.py."""
import numpy as np
import pytest

from episode_reference import attention
from libero_hip import episodes
from test_gpu_episodes import World, compare, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('count', [1, 3, 40])
@pytest.mark.parametrize('window', [1, 31, 64, 100, 2 ** 30, 2 ** 31 - 1])
def test_lengths_up_to_32_bits(gpu_available, window, count):
    """Worlds that say they are longer than their table reaches, up to 2^31 - 1 tokens: a window that lies beyond the table
    shows nothing, one that reaches back into it shows the tokens that are there."""
    import torch
    print('case lengths', window, count, flush=True)
    lengths = np.array([2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 31, 2 ** 31 - 66, 2 ** 30 + 5, 9000], np.int64)
    for dim, store, width in ((64, 'bf16', 2), (128, 'fp8', 2), (64, 'bf16', 512)):     # not split, and split
        world = World([32] * len(lengths), 2, dim, 16, store, seed=30, width=width)
        world.pages.length.copy_(torch.from_numpy(lengths.astype(np.int32)))
        q, start = queries([count] * len(lengths), 4, dim, 'bf16')
        qd = q.double().numpy()
        ref, ref_lse, size = np.zeros(qd.shape), np.full(qd.shape[:2], -np.inf), np.zeros(qd.shape)
        for w in range(len(lengths)):
            for i in range(count):
                low, row = max(0, lengths[w] - count + i - window + 1), w * count + i
                if low < 32:
                    ref[row], ref_lse[row], size[row] = (x[0] for x in attention(
                        qd[row:row + 1], world.k[w][low:], world.v[w][low:], 31 - low, False, 0, dim ** -0.5))
        assert np.isfinite(ref_lse).any() == (window >= 2 ** 30)
        for causal in (True, False):
            lse = torch.full(q.shape[:-1], 7.0, device='cuda')
            out = episodes.attend(world.pages, q.cuda(), torch.from_numpy(start).cuda(), causal=causal, window=window,
                                  max_count=count, lse=lse)
            compare(out, lse, (ref, ref_lse, size), 'bf16')
