"""The state-space policy: single steps against whole segments, its gradient against the model in 64 bits, and training."""
import os
import sys

import numpy as np
import pytest
import torch

import policy_layer_ref as R
from pufferlean_amd import device as D
from pufferlean_amd import rng
from pufferlean_amd.ssm_policy import SSMPolicy

pytestmark = pytest.mark.gpu
T, B, OBS, A = 21, 6, 7, 3


def cu(seed, *shape):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape)).float().cuda()


def columns():
    done = torch.from_numpy(rng.bernoulli(2, T * B, 0.15).reshape(T, B)).float().cuda()
    first = torch.from_numpy(rng.bernoulli(3, B, 0.5)).float().cuda()
    return cu(1, T, B, OBS), done, first


def carried(policy):
    return [(cu(10 + i, B, policy.C, policy.N), cu(20 + i, B, policy.K - 1, policy.C)) for i in range(policy.layers)]


def reference(policy, p, obs, done, first, state):
    """The head outputs from 64-bit leaves p."""
    x = obs.reshape(T * B, -1) @ p["enc"].T + p["enc_b"]
    for i in range(policy.layers):
        n = R.layer_norm(x, p[f"{i}.n1w"], p[f"{i}.n1b"])
        c = (n @ p[f"{i}.in"].T).view(T, B, -1).split(policy.parts, dim=-1)
        q = dict(zip(("x", "z", "delta", "Bm", "Cm"), c), A=-torch.exp(p[f"{i}.A_log"]), D=p[f"{i}.D"],
                 dt_bias=p[f"{i}.dt_bias"], conv_w=p[f"{i}.conv_w"], conv_b=p[f"{i}.conv_b"])
        y, _, _ = R.scan(q, 1, done, first, state[i][0], state[i][1])
        x = x + y.reshape(T * B, -1) @ p[f"{i}.out"].T
        n = R.layer_norm(x, p[f"{i}.n2w"], p[f"{i}.n2b"])
        x = x + R.ffn(n, p[f"{i}.ffn_in"], p[f"{i}.ffn_out"], policy.act)
    return R.layer_norm(x, p["nw"], p["nb"]) @ p["head"].T + p["head_b"]


def policy_of(dtype):
    return SSMPolicy(OBS, A, width=24, inner=40, states=8, ffn=36, layers=2, dtype=dtype, seed=5)


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
        assert R.rel(y, out[t]) <= bar, t
        f = done[t].contiguous()
    for (h1, w1), (h2, w2) in zip(s1, s2):
        assert R.rel(h1, h2) <= bar and R.rel(w1, w2) <= bar


def test_gradient_in_fp32(gpu):
    policy = policy_of(torch.float32)
    obs, done, first = columns()
    out, saved = policy.forward(obs, done, first, carried(policy), save=True)
    dout = cu(4, T, B, A + 1)
    g = policy.backward(saved, dout)
    p = {k: R.leaf(v) for k, v in policy.p.items()}
    host = lambda t: t.double().cpu()
    ref = reference(policy, p, host(obs), host(done), host(first), [(host(h), host(w)) for h, w in carried(policy)])
    assert R.rel(out.view(T * B, -1), ref) <= 2e-4
    grads = torch.autograd.grad(ref, list(p.values()), host(dout).view(T * B, -1))
    assert set(g) == set(p)
    for k, r in zip(p, grads):
        assert R.rel(g[k], r) <= 5e-4, k


def test_policy_without_taps(gpu):
    """No convolution: its bias is no part of the model, so the gradient leaves it where it is. Bars as above."""
    policy = SSMPolicy(OBS, A, width=24, inner=40, states=8, taps=0, ffn=36, layers=2, dtype=torch.float32, seed=5)
    obs, done, first = columns()
    out, saved = policy.forward(obs, done, first, save=True)
    dout = cu(4, T, B, A + 1)
    g = policy.backward(saved, dout)
    p = {k: R.leaf(v) for k, v in policy.p.items()}
    host = lambda t: t.double().cpu()
    ref = reference(policy, p, host(obs), host(done), host(first), [(None, None)] * policy.layers)
    assert R.rel(out.view(T * B, -1), ref) <= 2e-4
    used = [k for k in p if "conv" not in k]
    for k, r in zip(used, torch.autograd.grad(ref, [p[k] for k in used], host(dout).view(T * B, -1))):
        assert R.rel(g[k], r) <= 5e-4, k
    policy.update(g)
    for i in range(policy.layers):
        assert not g[f"{i}.conv_b"].any() and not policy.p[f"{i}.conv_b"].any()


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


def test_example_learns_the_cue(gpu):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import ssm_policy as example
    _, reward = example.train(updates=30, say=lambda *_: None)
    assert reward[0] < 0.4 and np.mean(reward[-3:]) > 0.6  # chance is 0.25
