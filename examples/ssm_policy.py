"""Trains the state-space policy on a small memory task and rolls it out step by step.

Each episode shows a cue at its first step only; the reward is for naming it at every later step, so the policy has to carry it
in its state. Episodes end at random, in the middle of the trained segments too.

    python examples/ssm_policy.py [--updates N] [--envs B] [--steps T] [--f32]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from pufferlean_amd import device as D  # noqa: E402
from pufferlean_amd.ssm_policy import SSMPolicy  # noqa: E402

CUES = 4


def rollout(policy, B, T, state, first, cue, seed):
    """T steps of B environments: the minibatch's columns, and what carries over to the next rollout."""
    cols = dict(obs=[], act=[], logp=[], val=[], rew=[], done=[])
    for t in range(T):
        cue = torch.where(first > 0, torch.randint(0, CUES, (B,), device="cuda"), cue)
        obs = torch.zeros(B, CUES + 1, device="cuda")
        obs.scatter_(1, torch.where(first > 0, cue, CUES)[:, None], 1.0)
        out = policy.step(obs, state, first)
        act, logp, val = D.sample_actions(out, CUES, rng_state=(seed * T + t) * B * 0x9E3779B97F4A7C15)
        rew = (act == cue).float()
        done = (torch.rand(B, device="cuda") < 0.1).float()
        for k, v in dict(obs=obs, act=act, logp=logp, val=val, rew=rew, done=done).items():
            cols[k].append(v)
        first = done
    return {k: torch.stack(v) for k, v in cols.items()}, first, cue


def train(updates=30, B=256, T=32, dtype=torch.bfloat16, say=print):
    torch.manual_seed(1)
    policy = SSMPolicy(CUES + 1, CUES, width=64, inner=64, states=16, ffn=96, layers=1, dtype=dtype)
    state = policy.state(B)
    first, cue = torch.ones(B, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda")
    reward = []
    for u in range(updates):
        start = [(h.clone(), None if w is None else w.clone()) for h, w in state]
        first0 = first.clone()
        c, first, cue = rollout(policy, B, T, state, first, cue, u + 1)
        adv, ret = D.vtrace(c["rew"], c["val"], c["done"], variant=1, boot=torch.zeros(B, device="cuda"), gamma=0.5, clamp=False)
        g = policy.ppo_grad(c["obs"], c["act"], D.adv_normalize(adv), ret, c["logp"], done=c["done"], first=first0, state=start)
        policy.update(g, lr=0.01, scale=1.0 / (T * B))
        reward.append(float(c["rew"].mean()))
        if u % 10 == 0 or u == updates - 1:
            say(f"update {u}: mean reward {reward[-1]:.3f} (chance {1 / CUES:.2f})")
    return policy, reward


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--updates", type=int, default=60)
    ap.add_argument("--envs", type=int, default=256)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--f32", action="store_true")
    a = ap.parse_args()
    train(a.updates, a.envs, a.steps, torch.float32 if a.f32 else torch.bfloat16)
