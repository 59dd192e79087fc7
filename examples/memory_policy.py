"""A policy with a memory per world, acting in and trained on the character-rig worlds.

    python examples/memory_policy.py [--worlds 4096] [--steps 32] [--updates 4] [--dtype bfloat16]

The rig's worlds are partially observed: the policy sees the pot's pose and velocity and 16 rays, not the hammer. Each
world's memory is advanced one token per world step while it acts (goib2d.delta_step_), emptied when the world resets,
and the recorded rollout goes through the same memory as one sequence when it trains (goib2d.delta_rule, with its
gradient); the update clips the gradient by its global norm (goib2d.clip_grads_). Policy gradient (REINFORCE) on how
far the pot gets to the right; the policy is small and untuned - the example shows the calls, not a learned climb.
"""
import argparse
import sys
import time
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "getting-over-it-rl_b200"))
import goib2d  # noqa: E402
from goib2d import api, configs  # noqa: E402

POT, RAYS, RAY_LENGTH, FALLEN = 1, 16, 8.0, -5.0


class MemoryPolicy(nn.Module):
    """observation -> encoder -> (q, k, v, gates) -> memory -> the two joints' action means"""

    def __init__(self, inputs=6 + RAYS, hidden=128, heads=2, channels=32, actions=2):
        super().__init__()
        self.heads, self.channels = heads, channels
        self.encode = nn.Sequential(nn.Linear(inputs, hidden), nn.Tanh())
        self.token = nn.Linear(hidden, heads * (3 * channels + 2))
        self.act = nn.Linear(hidden + heads * channels, actions)

    def memory(self, worlds, device):
        return torch.zeros(worlds, self.heads, self.channels, self.channels, device=device)

    def tokens(self, x):
        """(encoded, q, k, v, log decay, write strength) of observations (..., inputs)"""
        e = self.encode(x)
        h, c = self.heads, self.channels
        q, k, v, g, b = self.token(e).split((h * c, h * c, h * c, h, h), -1)
        q, k = (nn.functional.normalize(y.unflatten(-1, (h, c)), dim=-1) for y in (q, k))
        return e, q, k, v.unflatten(-1, (h, c)), -nn.functional.softplus(g - 2), torch.sigmoid(b)

    def step(self, x, memory, reset):
        """Acting: one token per world, the memory updated in place."""
        e, *token = self.tokens(x)
        o = goib2d.delta_step_(memory, *token, reset=reset)
        return self.act(torch.cat((e, o.flatten(-2)), -1))

    def forward(self, x, memory, reset):
        """Training: rollouts (worlds, steps, inputs) from the memory that they began with."""
        e, *token = self.tokens(x)
        o, _ = goib2d.delta_rule(*token, state=memory, reset=reset)
        return self.act(torch.cat((e, o.flatten(-2)), -1))


def rollout(engine, scene, state, start, policy, memory, reset, steps, std, dtype):
    """Act for `steps` world steps. reset: the worlds that were reset before the first one. Returns (observations, actions,
    resets, rewards, action means), each (worlds, steps, ...), and the worlds that were reset after the last one."""
    falls = torch.zeros(memory.shape[0], dtype=torch.int32, device="cuda")
    seen, done, acted, rewards, means = [], [], [], [], []
    for _ in range(steps):
        body = engine.observe(state, [POT])[:, 0]
        rays = engine.raycast(state, POT, RAYS, RAY_LENGTH)
        x = torch.cat((body * 0.1, rays), -1).to(dtype)
        with torch.no_grad():
            mean = policy.step(x, memory, reset)
        action = mean.float() + std * torch.randn_like(mean, dtype=torch.float32)
        engine.step_(state, scene.settings, configs.DT, 1, action.contiguous())
        after = engine.observe(state, [POT])[:, 0]
        before = falls.clone()
        engine.reset_below(state, start, POT, FALLEN, falls)
        seen.append(x), done.append(reset), acted.append(action), means.append(mean)
        rewards.append(after[:, 0] - body[:, 0])
        reset = falls > before
    return (*(torch.stack(y, 1) for y in (seen, acted, done, rewards, means)), reset)


def train(worlds=4096, steps=32, updates=4, dtype=torch.bfloat16, seed=0, std=0.5, max_norm=0.5, lr=1e-3, log=print):
    torch.manual_seed(seed)
    scene, model, state, _, _ = configs.spawn_batch("c1", worlds, seed, seeded=True)
    start = goib2d.world.map_state(lambda x: x.clone(), state)
    engine = api.Engine(model, state.bodies.type.shape[1], scene.action_joints, scene.action_scale)
    policy = MemoryPolicy().cuda().to(dtype)
    optimiser = torch.optim.Adam(policy.parameters(), lr=lr, eps=1e-4)
    memory, fell = policy.memory(worlds, "cuda"), torch.zeros(worlds, dtype=torch.bool, device="cuda")
    results = []
    try:
        for update in range(updates):
            t = time.perf_counter()
            first = memory.clone()
            x, action, reset, reward, acted, fell = rollout(engine, scene, state, start, policy, memory, fell, steps, std, dtype)
            to_go = reward.flip(1).cumsum(1).flip(1)
            advantage = (to_go - to_go.mean(0)) / (to_go.std() + 1e-6)
            mean = policy(x, first, reset)
            replayed = float((mean.detach().float() - acted.float()).norm() / acted.float().norm())
            loss = (((action - mean.float()) ** 2).sum(-1) / (2 * std * std) * advantage).mean()
            optimiser.zero_grad(set_to_none=True)
            loss.backward()
            norm = goib2d.clip_grads_([p.grad for p in policy.parameters()], max_norm)
            optimiser.step()
            results.append({"reward": float(reward.sum(1).mean()), "loss": float(loss.detach()), "norm": float(norm),
                            "replayed": replayed})
            log(f"update {update}: reward {results[-1]['reward']:.4f}, gradient norm {results[-1]['norm']:.3f}, replay within "
                f"{replayed:.1e} of the acting pass, {time.perf_counter() - t:.2f} s")
    finally:
        engine.close()
    return policy, results


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--worlds", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--updates", type=int, default=4)
    ap.add_argument("--dtype", choices=("float32", "bfloat16"), default="bfloat16")
    a = ap.parse_args()
    train(a.worlds, a.steps, a.updates, getattr(torch, a.dtype))
