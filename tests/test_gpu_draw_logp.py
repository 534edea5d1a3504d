"""The log-probability of a draw whose share is small. The masses are whole numbers of 2^-bits of the largest, with few digits near one
unit, but logp is formed from the logit: (logit - largest) / temperature minus the logarithm of what is left. Each of A masses is off by at
most half a unit, so the logarithm of their sum, which is one at least, by A 2^-(bits + 1) (2^-23 at 2^20 entries, the widest), and the result is
rounded to fp32: 2^-24 of it."""
import math

import pytest
import torch

import delta_layer_ref as R
from pufferlean_amd import device as D

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def bits(A):
    return min(51, 62 - math.ceil(math.log2(A)))


def check(x, u, **par):
    act, logp = D.sample_filtered(x, u, **par)
    xs, un = x.double().cpu().numpy(), u.double().cpu().numpy()
    for i in range(len(un)):
        a, lp, _ = R.filtered(xs[i], un[i], **{k: v for k, v in par.items()})
        assert int(act[i]) == a, (i, int(act[i]), a)
        err = abs(float(logp[i]) - lp)
        assert err <= 2.0 ** -24 * abs(lp) + xs.shape[1] * 2.0 ** -(bits(xs.shape[1]) + 1), (i, float(logp[i]), lp)
    return act, logp


def rows(A, dt, low, at=0):
    """The largest logit, one far below it in front, and others that weigh less than half a unit."""
    x = torch.full((8, A), -100.0, device="cuda")
    x[:, A // 2] = 0.75
    x[:, at] = 0.75 - torch.tensor([(low - 0.37 * i) * math.log(2) for i in range(8)], device="cuda")
    return x.to(dt)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("A", [3, 18, 64, 200, 1000, 5000, 20000, 60001, 1 << 20])
@pytest.mark.parametrize("par", [dict(), dict(top_k=2), dict(temperature=0.5)])
def test_masses_of_a_few_units(gpu, A, par, dt):
    t = par.get("temperature", 1.0)
    act, _ = check(rows(A, dt, (bits(A) - 2) * t), torch.zeros(8, device="cuda"), **par)
    assert act.tolist() == [0] * 8


@pytest.mark.parametrize("A", [18, 1000, 5000, 60001, 1 << 20])
def test_behind_top_p_and_min_p(gpu, A):
    x = rows(A, F32, 20)
    act, _ = check(x, torch.zeros(8, device="cuda"), top_p=1 - 2.0 ** -24)
    assert act.tolist() == [0] * 8
    act, _ = check(x, torch.zeros(8, device="cuda"), min_p=2.0 ** -21)
    assert act.tolist() == [0] * 8


@pytest.mark.parametrize("A", [18, 1000, 5000, 60001])
def test_infinite_and_extreme_logits(gpu, A):
    x = torch.full((4, A), -100.0, device="cuda")
    x[0, 1], x[0, A - 1] = float("inf"), float("inf")
    x[1, 1] = 3e38
    x[2, 2], x[2, 5] = -3e38, -3e38
    x[2, 0] = x[2, 1] = x[2, 3] = x[2, 4] = -float("inf")
    x[2, 6:] = -float("inf")
    x[3] = 0
    u = torch.full((4,), 0.75, device="cuda")
    for par in (dict(), dict(top_k=2), dict(temperature=1e30), dict(temperature=float("inf")), dict(temperature=1e-30)):
        act, logp = D.sample_filtered(x, u, **par)
        assert act[0] == A - 1 and abs(float(logp[0]) + math.log(2)) <= 1e-7
        assert act[2] == 5 and abs(float(logp[2]) + math.log(2)) <= 1e-7
        n = min(2, A) if par.get("top_k") else A
        assert abs(float(logp[3]) + math.log(n)) <= 2.0 ** -24 * math.log(n) + 1e-7
    act, logp = D.sample_filtered(x, u)
    assert act[1] == 1 and logp[1] == 0
