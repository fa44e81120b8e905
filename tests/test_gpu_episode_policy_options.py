"""The example policy with positions, recall and tables on the device, in the loop with the environment."""
import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT / 'examples') not in sys.path:
    sys.path.insert(0, str(ROOT / 'examples'))
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('options', [dict(positions=True), dict(recall=1), dict(positions=True, recall=2, on_device=True)])
def test_rollout_with_options(gpu_available, options):
    from episode_policy import rollout
    print('case rollout', options, flush=True)
    actions, lengths, spent = rollout('c1', 6, steps=12, **options)
    assert actions.shape == (6, 7) and np.isfinite(actions).all() and np.abs(actions).max() <= 1
    assert np.all(lengths % 3 == 0) and lengths.max() <= 36 and np.all(spent > 0)


def test_tables_on_the_device_change_nothing(gpu_available):
    """The same tokens through both caches: the same actions, but for the order in which pages lie."""
    import torch
    from episode_policy import EpisodePolicy
    print('case policy on the device', flush=True)
    made = [EpisodePolicy(5, 22, tokens=80, storage='bf16', positions=True, recall=2, on_device=x) for x in (False, True)]
    gen = torch.Generator('cuda').manual_seed(3)
    actions = torch.zeros((5, 7), device='cuda')
    for step in range(20):
        observed = torch.randn((5, 22), generator=gen, device='cuda')
        a, b = (p.step(observed, actions) for p in made)
        assert torch.equal(a, b)
        actions = a
        if step % 6 == 5:
            for p in made:
                p.reset([step // 6, 4])
    assert made[0].cache.lengths.tolist() == made[1].cache.lengths.tolist()
