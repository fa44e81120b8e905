"""A policy that remembers its episode, in the loop of the batch environment.

Every control step each world contributes a few tokens (joint state, objects, the last action), which see
each other and all tokens of the world's episode so far: the layers' keys and values stay in an
``EpisodeCache``, so a step computes its new tokens only.  Worlds restart one by one; the same ids empty the
memory.  Weights are random: the example shows the calls, not a trained policy.  With ``--positions`` queries and keys turn
by their place in the episode, with ``--recall N`` a token attends to the N blocks that match it best and the latest ones
instead of to all, with ``--device`` the worlds' tables are kept on the GPU.

    python examples/episode_policy.py --config c3 --worlds 256 --steps 20
"""
import argparse
import sys
import time
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / 'gpu-libero_amd'))
from libero_hip.environment import HipBatchEnv      # noqa: E402
from libero_hip.episodes import EpisodeCache        # noqa: E402
from libero_hip.room import DeviceEpisodeCache      # noqa: E402
from libero_hip.rotary import Rotary                # noqa: E402


class EpisodePolicy:
    """A small attention policy: ``step(observed, actions)`` appends a step's tokens and returns actions in [-1, 1]."""

    def __init__(self, nworld, observed_width, *, tokens, width=256, heads=8, kv_heads=2, head_dim=32, layers=2,
                 storage='fp8', pages=None, seed=0, device='cuda:0', positions=False, recall=None, on_device=False):
        gen = torch.Generator(device).manual_seed(seed)

        def matrix(rows, columns):
            return (torch.randn((rows, columns), generator=gen, device=device) * rows ** -0.5).bfloat16()

        half = observed_width // 2
        self.parts = ((0, half), (half, observed_width))           # of the observation: a token each
        self.embed = [matrix(stop - begin, width) for begin, stop in self.parts] + [matrix(7, width)]
        self.layers = [dict(q=matrix(width, heads * head_dim), kv=matrix(width, 2 * kv_heads * head_dim),
                            out=matrix(heads * head_dim, width), up=matrix(width, 2 * width), down=matrix(2 * width, width))
                       for _ in range(layers)]
        self.head = matrix(width, 7)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.tokens_per_step = len(self.embed)
        self.turning = Rotary.make(head_dim, device=device) if positions else None
        self.recall = recall                                       # how many blocks of 16 tokens to choose
        self.on_device = on_device
        self.cache = (DeviceEpisodeCache if on_device else EpisodeCache)(
            nworld, kv_heads=kv_heads, head_dim=head_dim, tokens=tokens, layers=layers, storage=storage, pages=pages,
            device=device, block_tokens=None if recall is None else 16)

    @staticmethod
    def norm(x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def step(self, observed, actions):
        """observed (nworld, width) and the last actions (nworld, 7), on the device -> actions (nworld, 7)."""
        inputs = [observed[:, begin:stop] for begin, stop in self.parts] + [actions]
        x = torch.stack([a.bfloat16() @ m for a, m in zip(inputs, self.embed)], 1)
        chunk = self.cache.extend(self.tokens_per_step)
        n, t = x.shape[:2]
        for i, w in enumerate(self.layers):
            y = self.norm(x)
            kv = (y @ w['kv']).view(n, t, 2, self.kv_heads, self.head_dim)
            q = (y @ w['q']).view(n, t, self.heads, self.head_dim)
            if self.turning is None:
                self.cache.write(chunk, kv[:, :, 0], kv[:, :, 1], i)
            else:
                q = self.cache.enter(chunk, self.turning, q, kv[:, :, 0], kv[:, :, 1], i)
            if self.recall is None:
                seen = self.cache.attend(chunk, q, i, causal=False)
            else:
                seen = self.cache.recall(chunk, q, i, top=self.recall, near=2, first=1, causal=False)
            x = x + seen.view(n, t, -1) @ w['out']
            x = x + torch.nn.functional.gelu(self.norm(x) @ w['up']) @ w['down']
        return torch.tanh(self.norm(x[:, -1]) @ self.head).float()

    def reset(self, id=None):
        if self.on_device and id is not None:
            over = np.zeros(self.cache.nworld, bool)
            over[id] = True
            id = torch.from_numpy(over).to(self.cache.device)
        self.cache.reset(id)


def rollout(config='c3', worlds=256, steps=20, storage='fp8', seed=0, **options):
    """Steps the environment with the policy, restarting about a tenth of the worlds each step; returns the
    actions of the last step, the tokens held by each world, and the seconds per step of policy and physics."""
    rng = np.random.default_rng(seed)
    with HipBatchEnv(config, worlds, seed=seed) as env:
        policy = EpisodePolicy(worlds, env.observer.plan.width, tokens=3 * steps, storage=storage, seed=seed, **options)
        actions = torch.zeros((worlds, 7), device='cuda')
        spent = np.zeros(2)
        for _ in range(steps):
            begin = time.perf_counter()
            actions = policy.step(env.observer.observed, actions)
            host = actions.cpu().numpy()
            middle = time.perf_counter()
            env.step(host)
            spent += middle - begin, time.perf_counter() - middle
            over = np.flatnonzero(rng.random(worlds) < 0.1)
            if len(over):
                env.reset(over)
                policy.reset(over)
                actions[torch.from_numpy(over).cuda()] = 0
        return host, policy.cache.lengths.copy(), spent / steps


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument('--config', default='c3')
    parser.add_argument('--worlds', type=int, default=256)
    parser.add_argument('--steps', type=int, default=20)
    parser.add_argument('--storage', default='fp8', choices=('fp8', 'bf16'))
    parser.add_argument('--positions', action='store_true')
    parser.add_argument('--recall', type=int, metavar='N')
    parser.add_argument('--device', action='store_true')
    args = parser.parse_args()
    _, lengths, (policy_s, physics_s) = rollout(args.config, args.worlds, args.steps, args.storage, positions=args.positions,
                                                recall=args.recall, on_device=args.device)
    print('%d worlds, %d steps: policy %.2f ms, environment %.2f ms a step; %d to %d tokens held'
          % (args.worlds, args.steps, 1e3 * policy_s, 1e3 * physics_s, lengths.min(), lengths.max()))
