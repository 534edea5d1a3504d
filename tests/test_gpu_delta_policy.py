"""The delta-rule policy: single steps against whole segments, its gradient against the model in 64 bits, rollouts and training."""
import os
import sys

import numpy as np
import pytest
import torch

import delta_layer_ref as R
import policy_layer_ref as P
from pufferlean_amd import device as D
from pufferlean_amd import rng
from pufferlean_amd.delta_policy import DeltaPolicy

pytestmark = pytest.mark.gpu
T, B, OBS, A = 21, 6, 7, 3


def cu(seed, *shape):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape)).float().cuda()


def columns():
    done = torch.from_numpy(rng.bernoulli(2, T * B, 0.15).reshape(T, B)).float().cuda()
    first = torch.from_numpy(rng.bernoulli(3, B, 0.5)).float().cuda()
    return cu(1, T, B, OBS), done, first


def carried(policy):
    return [0.3 * cu(10 + i, B, policy.heads, policy.K, policy.V) for i in range(policy.layers)]


def reference(policy, p, obs, done, first, state):
    """The head outputs from 64-bit leaves p."""
    r = obs.reshape(T * B, -1) @ p["enc"].T + p["enc_b"]
    add = scale = None
    for i in range(policy.layers):
        n, r = R.rms(r, p[f"{i}.n1w"], add, scale)
        q, k, v, z, a, b = (n @ p[f"{i}.in"].T).view(T, B, -1).split(policy.parts, dim=-1)
        y, _ = R.delta(dict(q=q.unflatten(-1, (policy.key_heads, policy.K)), k=k.unflatten(-1, (policy.key_heads, policy.K)),
                            v=v.unflatten(-1, (policy.heads, policy.V)), a=a, b=b, A=-torch.exp(p[f"{i}.A_log"]), dt_bias=p[f"{i}.dt_bias"]),
                       None, done, first, state[i])
        o, _ = R.rms(y.reshape(T * B, -1), p[f"{i}.ow"], gate=z.reshape(T * B, -1), groups=policy.heads)
        n, r = R.rms(r, p[f"{i}.n2w"], o @ p[f"{i}.out"].T, p[f"{i}.s1"])
        add, scale = P.ffn(n, p[f"{i}.ffn_in"], p[f"{i}.ffn_out"], policy.act_fn), p[f"{i}.s2"]
    return R.rms(r, p["nw"], add, scale)[0] @ p["head"].T + p["head_b"]


def policy_of(dtype):
    p = DeltaPolicy(OBS, A, width=24, heads=4, key_heads=2, K=8, V=12, ffn=36, layers=2, dtype=dtype, seed=5)
    for i, (k, v) in enumerate(sorted(p.p.items())):
        if v.dim() == 1:  # no norm or scale of one, no bias of zero
            v += 0.2 * cu(100 + i, *v.shape)
    return p


# fp32: some ten operators in a row, each within 2e-5 of its own definition. bf16: each residual block rounds its own few
# results by 2^-8 at most, and those of two layers meet in the head.
@pytest.mark.parametrize("dtype,bar", [(torch.float32, 2e-4), (torch.bfloat16, 12 * R.BF16)])
def test_steps_follow_the_segment(gpu, dtype, bar):
    policy = policy_of(dtype)
    obs, done, first = columns()
    s1, s2 = carried(policy), carried(policy)
    out = policy.forward(obs, done, first, s1)
    f = first
    for t in range(T):
        y = policy.step(obs[t].contiguous(), s2, f)
        assert P.rel(y, out[t]) <= bar, t
        f = done[t].contiguous()
    for h1, h2 in zip(s1, s2):
        assert P.rel(h1, h2) <= bar


def test_gradient_in_fp32(gpu):
    policy = policy_of(torch.float32)
    obs, done, first = columns()
    out, saved = policy.forward(obs, done, first, carried(policy), save=True)
    dout = cu(4, T, B, A + 1)
    g = policy.backward(saved, dout)
    p = {k: P.leaf(v) for k, v in policy.p.items()}
    host = lambda t: t.double().cpu()
    ref = reference(policy, p, host(obs), host(done), host(first), [host(h) for h in carried(policy)])
    assert P.rel(out.view(T * B, -1), ref) <= 2e-4
    grads = torch.autograd.grad(ref, list(p.values()), host(dout).view(T * B, -1))
    assert set(g) == set(p)
    for k, r in zip(p, grads):
        assert P.rel(g[k], r) <= 1e-3, k


def test_bf16_gradient_points_the_same_way(gpu):
    obs, done, first = columns()
    dout = cu(4, T, B, A + 1)
    gs = []
    for dtype in (torch.float32, torch.bfloat16):
        policy = policy_of(dtype)
        _, saved = policy.forward(obs, done, first, carried(policy), save=True)
        gs.append(policy.backward(saved, dout))
    for k in gs[0]:
        a, b = gs[0][k].double().flatten(), gs[1][k].double().flatten()
        assert float(a @ b / (a.norm() * b.norm())) > 0.98, k


def test_rollout_step_draws_from_its_own_logits(gpu):
    policy = policy_of(torch.float32)
    obs, _, first = columns()
    s1, s2 = carried(policy), carried(policy)
    u = torch.linspace(0, 0.99, B, device="cuda")
    act, logp, val = policy.act(obs[0], s1, u, first, temperature=0.7)
    out = policy.step(obs[0], s2, first)
    assert torch.equal(val, out[:, A])
    lp = torch.log_softmax(out[:, :A].double() / 0.7, 1)
    assert (logp.double() - lp.gather(1, act[:, None].long())[:, 0]).abs().max() < 1e-5
    assert torch.equal(act.long(), (lp.exp().cumsum(1) > u[:, None].double()).int().argmax(1))
    best, lp, _ = policy.act(obs[1], s1, u, top_k=1)
    assert torch.equal(best.long(), policy.step(obs[1], s2)[:, :A].argmax(1)) and not lp.any()


def test_example_runs_and_steps_its_weights(gpu):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import delta_policy as example
    policy, reward = example.train(updates=3, B=32, T=8, say=lambda *_: None)
    fresh = DeltaPolicy(example.CUES + 1, example.CUES, width=64, heads=2, K=32, V=32, ffn=96, layers=1)
    assert len(reward) == 3 and all(v.isfinite().all() for v in policy.p.values())
    assert all(not torch.equal(v, fresh.p[k]) for k, v in policy.p.items())
