"""The draw from filtered logits against the definition, a sorted row in 64 bits. The index has to be equal; a row whose u or
p is within 1e-9 of a border is left out. The log-probability is a 64-bit value rounded to fp32: 2^-24, and the masses'
unit of 2^-45 of the largest, over the mass drawn (of the order of 1e-6 at least here): 3e-8."""
import numpy as np
import pytest
import torch

import delta_layer_ref as R
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
NAN, INF = float("nan"), float("inf")


def cu(seed, *shape, scale=1.0, dtype=F32):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", dtype)


def numbers(seed, N):
    return torch.from_numpy(rng.randf(seed, N, 0, 1)).float().cuda().clamp(max=1 - 2.0 ** -24)


def check(logits, u, **par):
    act, logp = D.sample_filtered(logits, u, **par)
    x, un = logits.double().cpu().numpy(), u.double().cpu().numpy()
    at = {k: (v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(len(un), v)) for k, v in par.items()}
    skipped = 0
    for i in range(len(un)):
        row = {k: (int(v[i]) if k == "top_k" else np.float32(v[i])) for k, v in at.items()}
        a, lp, near = R.filtered(x[i], un[i], **row)
        if near < 1e-9:
            skipped += 1
            continue
        assert int(act[i]) == a, (i, int(act[i]), a, row, un[i])
        assert float(logp[i]) == lp or abs(float(logp[i]) - lp) <= 1e-7 * abs(lp) + 1e-7, (i, float(logp[i]), lp)
    assert skipped <= len(un) // 20
    return act, logp


def mixed(N, seed=20):
    pick = rng.randf(seed, 4 * N, 0, 1).reshape(4, N)
    val = rng.randf(seed + 1, 4 * N, 0, 1).reshape(4, N)
    f = lambda v, dt=torch.float32: torch.from_numpy(v).to("cuda", dt)
    return dict(temperature=f(np.where(pick[0] < 0.1, 0.0, 0.3 + 1.5 * val[0])),
                top_k=f(np.where(pick[1] < 0.4, 0, 1 + val[1] * 40), torch.int32),
                top_p=f(np.where(pick[2] < 0.3, 1.0, 0.05 + 0.95 * val[2])),
                min_p=f(np.where(pick[3] < 0.5, 0.0, 0.3 * val[3])))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("A", [1, 2, 3, 18, 63, 64, 65, 200, 256, 257, 1000, 1024, 1025, 2048, 2100, 5003, 20000, 60001])
def test_sizes(gpu, A, dt):
    N = 60 if A <= 1024 else 12
    x = cu(1, N, A, scale=2.0, dtype=dt)
    x[torch.from_numpy(rng.bernoulli(3, N * A, 0.2).reshape(N, A)).bool().cuda()] = -INF
    check(x, numbers(2, N), **mixed(N))


@pytest.mark.parametrize("A", [50, 3000, 50001])
@pytest.mark.parametrize("par", [dict(), dict(temperature=0.7), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.1), dict(top_k=7, top_p=0.5),
                                 dict(temperature=0.0), dict(top_p=0.0), dict(top_k=1), dict(top_k=10 ** 6), dict(top_k=300, top_p=0.9), dict(top_p=1.0, min_p=1.0),
                                 dict(min_p=5.0), dict(temperature=-1.0), dict(temperature=NAN, top_p=NAN, min_p=NAN), dict(top_k=-3), dict(temperature=1e-30),
                                 dict(temperature=1e30, top_p=0.3001)])
def test_one_filter_at_a_time(gpu, par, A):
    N = 20 if A < 10000 else 6
    check(cu(1, N, A, scale=3.0), numbers(2, N), **par)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("A", [16, 700, 4096, 50000])
def test_equal_logits(gpu, A, dt):
    """A few values, so that every threshold is among equals; of these the lower indices stay."""
    N = 40 if A < 10000 else 12
    x = (cu(1, N, A) * 1.5).round().to(dt)
    x[0] = 0.25
    x[1], x[1, ::2] = 0.0, -0.0
    check(x, numbers(2, N), **mixed(N))
    x = torch.zeros(4, A, device="cuda", dtype=dt)
    u = torch.tensor([0.0, 0.49, 0.51, 1 - 2.0 ** -24], device="cuda")
    act, logp = D.sample_filtered(x, u, top_k=8)
    assert act.tolist() == [0, 3, 4, 7] and torch.allclose(logp.cpu(), torch.tensor(-np.log(8.0)).float())
    act, _ = D.sample_filtered(x, u, top_p=0.25)
    assert act.tolist() == [0, int(float(u[1]) * A / 4), int(float(u[2]) * A / 4), A // 4 - 1]  # u as it is in fp32
    act, logp = D.sample_filtered(x, u, temperature=0.0)
    assert act.tolist() == [0] * 4 and not logp.any()


@pytest.mark.parametrize("A", [5, 130, 2000, 9000, 50000])
def test_special_logits(gpu, A):
    x = cu(1, 8, A)
    x[0] = -INF
    x[1] = NAN
    x[2] = -INF
    x[2, A - 1] = -1e30
    x[3, ::2] = NAN
    x[4, 1] = INF
    x[5, 1], x[5, A - 2] = INF, INF
    x[6] = 3e38
    x[6, 0] = -3e38
    x[7] = torch.finfo(F32).min
    x[7, 3] = 0
    for u in (0.0, 0.3, 0.8):
        for par in (dict(), dict(top_k=2), dict(top_p=0.6), dict(temperature=0.0), dict(min_p=0.5)):
            act, logp = check(x, torch.full((8,), u, device="cuda"), **par)
            assert act[:2].tolist() == [-1, -1] and (logp[:2] == -INF).all()


def test_numbers_at_the_borders(gpu):
    """u of 0 takes the first that is left, the largest u below 1 the last."""
    x = torch.tensor([[-INF, 1.0, 0.5, 2.0, -INF]], device="cuda").expand(2, 5)
    act, _ = D.sample_filtered(x.contiguous(), torch.tensor([0.0, 1 - 2.0 ** -24], device="cuda"))
    assert act.tolist() == [1, 3]


def test_shares_follow_the_masses(gpu):
    """100,000 draws on an even grid of u: each entry as often as its share, to the grid."""
    N, A = 100000, 7
    row = cu(1, 1, A)
    u = (torch.arange(N, device="cuda") + 0.5) / N
    act, logp = D.sample_filtered(row.expand(N, A), u, temperature=0.8)
    share = torch.softmax(row[0].double() / 0.8, 0).cpu()
    assert (torch.bincount(act.long(), minlength=A).cpu() / N - share).abs().max() <= 2 / N
    assert (logp.double().cpu() - share.log()[act.long().cpu()]).abs().max() <= 1e-6


@pytest.mark.parametrize("A", [30, 3000, 49153])
def test_strides_outputs_and_numbers_for_all(gpu, A):
    wide = cu(1, 10, A + 9, dtype=BF)
    x = wide[:, 3:A + 3]
    u = numbers(2, 10)
    par = mixed(10)
    act, logp = torch.full((10,), 7, dtype=torch.int32, device="cuda"), torch.empty(10, device="cuda")
    a, b = D.sample_filtered(x, u, act=act, logp=logp, **par)
    assert a is act and b is logp
    a2, b2 = D.sample_filtered(x.contiguous(), u, **par)
    assert torch.equal(a, a2) and torch.equal(b, b2)
    one = D.sample_filtered(x, u, temperature=0.5, top_k=4)
    all_ = D.sample_filtered(x, u, temperature=torch.full((10,), 0.5, device="cuda"), top_k=torch.full((10,), 4, dtype=torch.int32, device="cuda"))
    assert torch.equal(one[0], all_[0])
    assert D.sample_filtered(x[:0], u[:0])[0].shape == (0,)


@pytest.mark.parametrize("A", [100, 5000, 49152])
def test_captured(gpu, A):
    x, u, par = cu(1, 30, A), numbers(2, 30), mixed(30)
    act, logp = D.sample_filtered(x, u, **par)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = D.sample_filtered(x, u, **par)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], act) and torch.equal(out[1], logp)
        D.sample_filtered(x.flip(1).contiguous(), u, **par)
        torch.cuda.synchronize()


def test_the_widest_rows(gpu):
    """2^20 entries in sixteen blocks, and the same rows in one block each where there are more than 128 of them."""
    A = 1 << 20
    x, u = cu(1, 2, A, scale=2.0), numbers(2, 130)
    for par in (dict(), dict(temperature=0.8, top_k=700, top_p=0.9, min_p=1e-3), dict(top_p=0.7)):
        check(x, u[:2], **par)
        act, logp = D.sample_filtered(x[:1].expand(130, A), u, **par)
        few = [D.sample_filtered(x[:1].expand(65, A), u[i:i + 65], **par) for i in (0, 65)]
        assert torch.equal(act, torch.cat([f[0] for f in few])) and torch.equal(logp, torch.cat([f[1] for f in few]))
