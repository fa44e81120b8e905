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
