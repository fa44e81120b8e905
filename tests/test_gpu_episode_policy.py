"""EpisodeCache and the example policy on the GPU: a step's results against a recomputation of the whole episode
from the tokens themselves, with worlds that restart at different steps; and the rollout with the environment."""
import math
import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT / 'examples') not in sys.path:
    sys.path.insert(0, str(ROOT / 'examples'))
pytestmark = pytest.mark.gpu


def test_policy_remembers_its_episode(gpu_available):
    """In 16-bit storage the memory holds each token's keys and values exactly, so one layer's attention equals that
    over the episode's own keys and values, kept here in a list that a restart empties."""
    import torch
    from episode_policy import EpisodePolicy
    print('case policy', flush=True)
    n, width = 5, 22
    policy = EpisodePolicy(n, width, tokens=60, layers=2, storage='bf16', pages=14)
    kept = [[[] for _ in range(n)] for _ in policy.layers]
    calls = []
    attend, write = policy.cache.attend, policy.cache.write

    def keep(chunk, k, v, layer=0):
        for w in range(n):
            kept[layer][w].append((k[w].double().cpu().numpy(), v[w].double().cpu().numpy()))
        write(chunk, k, v, layer)

    def checked(chunk, q, layer=0, **options):
        out = attend(chunk, q, layer, **options)
        calls.append((layer, q.double().cpu().numpy(), out.double().cpu().numpy()))
        return out

    policy.cache.write, policy.cache.attend = keep, checked
    gen = torch.Generator('cuda').manual_seed(3)
    actions = torch.zeros((n, 7), device='cuda')
    u = 2.0 ** -8
    for step in range(9):
        actions = policy.step(torch.randn((n, width), generator=gen, device='cuda'), actions)
        assert actions.shape == (n, 7) and bool((actions.abs() <= 1).all())
        for layer, q, out in calls:
            for w in range(n):
                k, v = (np.concatenate(x) for x in zip(*kept[layer][w]))
                for h in range(q.shape[2]):
                    s = q[w, :, h] @ k[:, h // 4].T / math.sqrt(32)
                    p = np.exp(s - s.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    ref, size = p @ v[:, h // 4], p @ np.abs(v[:, h // 4])
                    # one rounding of the result, one of the weights, the rest in 32 bits
                    assert np.all(np.abs(out[w, :, h] - ref) <= u * np.abs(ref) + (u + 2.0 ** -12) * size)
        calls.clear()
        for w in ([1], [], [0, 3], [2], [])[step % 5]:
            policy.reset(w)
            for layer in kept:
                layer[w] = []
    np.testing.assert_array_equal(policy.cache.lengths, [3 * len(kept[0][w]) for w in range(n)])


def test_read_back_by_world(gpu_available):
    """read() of some worlds returns their tokens in the worlds' order, after restarts have scattered the pages."""
    import torch
    from libero_hip.episodes import EpisodeCache
    print('case read by world', flush=True)
    rng = np.random.default_rng(5)
    c = EpisodeCache(6, kv_heads=2, head_dim=64, tokens=100, storage='bf16', page_tokens=16, pages=30, layers=2)
    kept = [[] for _ in range(6)]
    for _ in range(12):
        ids = rng.permutation(6)[:4]
        counts = rng.integers(0, 12, 4)
        if np.any(c.lengths[ids] + counts > 100) or rng.random() < 0.2:
            c.reset(ids[:2])
            for w in ids[:2]:
                kept[w] = []
            continue
        chunk = c.extend(counts, ids)
        for layer in range(2):
            k = torch.randn(chunk.shape + (2, 64), device='cuda').bfloat16()
            c.write(chunk, k, -k, layer)
        start = chunk.start.tolist() if chunk.start is not None else None
        for w in range(6):
            kept[w].append(k[start[w]:start[w + 1]] if start else k[w])
    k, v, starts = c.read([4, 1, 2], 1)
    for i, w in enumerate([1, 2, 4]):
        want = torch.cat(kept[w]) if kept[w] else k[:0]
        assert torch.equal(k[starts[i]:starts[i + 1]], want) and torch.equal(v[starts[i]:starts[i + 1]], -want)


def test_rollout_with_the_environment(gpu_available):
    from episode_policy import rollout
    print('case rollout', flush=True)
    actions, lengths, spent = rollout('c1', 6, steps=5)
    assert actions.shape == (6, 7) and np.isfinite(actions).all() and np.abs(actions).max() <= 1
    assert np.all(lengths % 3 == 0) and lengths.max() <= 15 and np.all(spent > 0)
