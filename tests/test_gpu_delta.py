"""The gated delta rule, its gradient and its single step against the definition in 64 bits.

Bars (relative 2-norms). Every step contracts the state, so an error made in it does not grow later on. fp32: a result passes
some eight sums of up to 128 products, each within 128 roundings of 2^-24 (8e-6) at the very worst and a tenth of that
when they do not all go the same way: 1e-5. bf16: values that the kernel holds in fp32 enter its products as two
bf16 within 2^-17 of them, and up to eight such products follow each other: 6e-5; bf16 results add their one rounding. The
decay's gradients are differences of three sums that may cancel; they get ten times as much. dq = r (d - q^ <q^, d>), with r the
factor to unit length and d the unit row's gradient, and dk likewise, may cancel down to the norm's eps (a row of one element: to the
last digit), so their error is measured against these two terms."""
import numpy as np
import pytest
import torch

import delta_layer_ref as R
from policy_layer_ref import leaf, rel
from pufferlean_amd import _lib as L
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
BAR = {F32: 1e-5, BF: 6e-5}


def cu(seed, *shape, scale=1.0, dtype=F32):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", dtype)


def flags(seed, p, *shape):
    return torch.from_numpy(rng.bernoulli(seed, int(np.prod(shape)), p).reshape(shape)).float().cuda()


def inputs(T, B, Hk, H, K, V, dt, seed=1, layout="columns"):
    parts = [Hk * K, Hk * K, H * V, H, H]
    if layout == "columns":  # slices of one projection, time-major
        cols = cu(seed, T, B, sum(parts), dtype=dt).split(parts, dim=-1)
    elif layout == "odd":  # the same, every row one element further
        cols = cu(seed, T, B, sum(parts) + 1, dtype=dt)[..., 1:].split(parts, dim=-1)
    elif layout == "batch":  # batch-major
        cols = cu(seed, B, T, sum(parts), dtype=dt).transpose(0, 1).split(parts, dim=-1)
    else:
        cols = [c.contiguous() for c in cu(seed, T, B, sum(parts), dtype=dt).split(parts, dim=-1)]
    q, k, v, a, b = cols
    return dict(q=q.unflatten(-1, (Hk, K)), k=k.unflatten(-1, (Hk, K)), v=v.unflatten(-1, (H, V)), a=a, b=b,
                A=-(0.2 + cu(seed + 1, H).abs()), dt_bias=cu(seed + 2, H) - 2)


def host(t):
    return None if t is None else t.double().cpu()


def close(x, ref, bar, what):
    """Within the bar of it, a bf16 tensor within one rounding more."""
    got = rel(x, ref)
    assert got <= bar + (R.BF16 if x.dtype == BF else 0.0), (what, got)


def norm_terms(x, u, d):
    """The size of the two terms whose difference is the gradient of a row x with the unit row u and its gradient d."""
    with torch.no_grad():
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)
        return float((r * (d.abs() + (u * (u * d).sum(-1, keepdim=True)).abs())).norm())


def through_norm(x, ref, size, bar, what):
    err = float((host(x) - ref).norm())
    assert err <= bar * size + (R.BF16 * float(ref.norm()) if x.dtype == BF else 0.0), (what, err, size, float(ref.norm()))


def check(p, done=None, first=None, h0=None, scale=None, with_dh=True, seed=50):
    T, B, H, V = p["v"].shape
    K, dt = p["q"].shape[-1], p["q"].dtype
    bar = BAR[dt]
    dy = cu(seed, T, B, H, V, dtype=dt)
    dh = cu(seed + 1, B, H, K, V) if with_dh else None
    ref = {n: leaf(t) for n, t in p.items() if t is not None}
    h0r = leaf(h0) if h0 is not None else torch.zeros(B, H, K, V, dtype=torch.float64, requires_grad=True)
    units = {}
    yr, hr = R.delta(ref, scale, host(done), host(first), h0r, units)
    obj = (yr * host(dy)).sum() + (0 if dh is None else (hr * host(dh)).sum())
    grads = dict(zip(list(ref) + ["h0"], torch.autograd.grad(obj, [*ref.values(), h0r], allow_unused=True, retain_graph=True)))
    size = {n: norm_terms(ref[n], u, d) for (n, u), d in zip(units.items(), torch.autograd.grad(obj, list(units.values())))}
    h = torch.empty(B, H, K, V, device="cuda")
    args, kw = [p[n] for n in "qkvabA"], dict(dt_bias=p.get("dt_bias"), scale=scale, done=done, first=first)
    y, saved = D.delta_scan(*args, h0=h0, h_out=h, save=True, **kw)
    close(y, yr, bar, "y")
    close(h, hr, bar, "h")
    dh0 = torch.empty(B, H, K, V, device="cuda")
    g = D.delta_scan_grad(*args, saved, dy, dh=dh, dh0=dh0, **kw)
    for n in ref:
        assert g["d" + n].shape == p[n].shape and g["d" + n].dtype == p[n].dtype
        if n in size:
            through_norm(g["d" + n], grads[n], size[n], bar, "d" + n)
        else:
            close(g["d" + n], grads[n], bar * (10 if n in ("a", "A", "dt_bias") else 1), "d" + n)
    close(dh0, grads["h0"] if grads["h0"] is not None else torch.zeros_like(hr), bar, "dh0")
    return y, h, g, dh0


SIZES = [  # T, B, Hk, H, K, V
    (1, 1, 1, 1, 1, 1), (1, 3, 1, 2, 8, 16), (2, 2, 2, 2, 16, 8), (15, 2, 1, 1, 24, 41), (16, 2, 1, 3, 32, 32), (17, 2, 1, 1, 33, 7),
    (31, 2, 2, 2, 64, 64), (32, 1, 1, 2, 64, 40), (33, 2, 1, 2, 40, 64), (48, 1, 1, 1, 65, 96), (64, 2, 1, 1, 128, 128), (65, 1, 1, 2, 128, 3),
    (97, 1, 1, 1, 5, 127), (130, 2, 2, 4, 16, 16)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("T,B,Hk,H,K,V", SIZES)
def test_sizes(gpu, T, B, Hk, H, K, V, dt):
    p = inputs(T, B, Hk, H, K, V, dt)
    check(p, flags(3, 0.1, T, B), flags(4, 0.5, B), cu(5, B, H, K, V, scale=0.3))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("p_done", [0.0, 0.004, 0.05])
@pytest.mark.parametrize("T,B,Hk,H,K,V", [(300, 2, 1, 1, 16, 24), (530, 1, 1, 2, 64, 33), (515, 1, 1, 1, 100, 128), (767, 1, 1, 1, 33, 64)])
def test_long_sequences(gpu, T, B, Hk, H, K, V, p_done, dt):
    """In segments of time, with and without an episode's start in each."""
    p = inputs(T, B, Hk, H, K, V, dt)
    p["A"] *= 0.05  # states that outlive a segment
    check(p, flags(3, p_done, T, B), flags(4, 0.5, B), cu(5, B, H, K, V, scale=0.3))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("layout", ["odd", "batch", "packed"])
def test_layouts(gpu, layout, dt):
    p = inputs(70, 3, 2, 4, 32, 48, dt, layout=layout)
    check(p, flags(3, 0.1, 70, 3), flags(4, 0.5, 3), cu(5, 3, 4, 32, 48))


@pytest.mark.parametrize("dt", [F32, BF])
def test_nothing_optional(gpu, dt):
    p = inputs(40, 2, 1, 2, 24, 20, dt)
    p.pop("dt_bias")
    y, _, g, _ = check(p, with_dh=False)
    assert "ddt_bias" not in g
    check(p, scale=2.5)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("p_done", [0.5, 1.0])
def test_many_episodes(gpu, p_done, dt):
    """Starts in every place of a chunk; every step its own episode, the gradient of whose decay is zero."""
    p = inputs(67, 3, 1, 2, 16, 24, dt)
    _, _, g, dh0 = check(p, flags(3, p_done, 67, 3), flags(4, 0.5, 3), cu(5, 3, 2, 16, 24))
    if p_done == 1.0:
        assert not g["da"][1:].any()


@pytest.mark.parametrize("dt", [F32, BF])
def test_hard_gates(gpu, dt):
    """Decays from none to all at once, write strengths from none to all, equal keys, keys and queries of zero."""
    p = {n: t.clone() for n, t in inputs(80, 2, 1, 2, 32, 32, dt).items()}
    p["A"] = torch.tensor([-30.0, -0.001], device="cuda")
    p["a"][::7] = 60
    p["a"][3::7] = -60
    p["b"][::5] = 40
    p["b"][2::5] = -40
    p["k"][10:20] = p["k"][10].clone()
    p["k"][30:33] = 0
    p["q"][33:36] = 0
    check(p, h0=cu(5, 2, 2, 32, 32))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("name", ["q", "k", "v", "a", "b", "dy"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("T", [70, 410])
def test_an_episode_does_not_see_the_one_before(gpu, T, name, value, dt):
    """Non-finite values in steps 0..9 and 45..49; the episodes of steps 10..44 and from 50 on give what they give alone."""
    B, H, K, V = 2, 2, 16, 24
    p = {n: t.clone() for n, t in inputs(T, B, 1, H, K, V, dt).items()}
    dy = cu(50, T, B, H, V, dtype=dt)
    done = torch.zeros(T, B, device="cuda")
    done[[9, 44, 49]] = 1
    clean = [slice(10, 45), slice(50, T)]
    x = dict(p, dy=dy)[name]
    x[4, :, ..., 0] = value
    x[47] = value
    h0 = torch.full((B, H, K, V), float("nan"), device="cuda")
    h = torch.empty_like(h0)
    args = [p[n] for n in "qkvabA"]
    y, saved = D.delta_scan(*args, dt_bias=p["dt_bias"], done=done, h0=h0, h_out=h, save=True)
    g = D.delta_scan_grad(*args, saved, dy, dt_bias=p["dt_bias"], done=done)
    for i, s in enumerate(clean):
        ref = {n: leaf(t[s] if t.dim() > 1 else t) for n, t in p.items()}
        units = {}
        yr, hr = R.delta(ref, units=units)
        close(y[s], yr, BAR[dt], "y")
        names = ["q", "k", "v", "a", "b"]
        grads = torch.autograd.grad(yr, [ref[n] for n in names] + [units["q"], units["k"]], host(dy[s]))
        for j, n in enumerate(names):
            if n in units:
                through_norm(g["d" + n][s], grads[j], norm_terms(ref[n], units[n], grads[5 + j]), BAR[dt], (i, n))
            else:
                close(g["d" + n][s], grads[j], BAR[dt] * (10 if n == "a" else 1), (i, n))
        if i == 1:
            close(h, hr, BAR[dt], "h")


@pytest.mark.parametrize("dt", [F32, BF])
def test_a_state_that_first_clears_may_hold_anything(gpu, dt):
    T, B = 40, 3
    p = inputs(T, B, 1, 2, 16, 16, dt)
    first = torch.tensor([1.0, 0.0, 1.0], device="cuda")
    h0 = cu(5, B, 2, 16, 16)
    a = D.delta_scan(*[p[n] for n in "qkvabA"], first=first, h0=h0)
    h0[0] = float("inf")
    h0[2] = float("nan")
    assert torch.equal(a, D.delta_scan(*[p[n] for n in "qkvabA"], first=first, h0=h0))
    h = h0.clone()
    y = D.delta_step(*[p[n][0] for n in "qkvab"], p["A"], h, first=first)
    assert y.isfinite().all() and h.isfinite().all()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("Hk,H,K,V", [(1, 1, 1, 1), (1, 2, 8, 4), (2, 4, 32, 32), (1, 3, 24, 41), (2, 2, 64, 64), (1, 1, 33, 16), (1, 1, 17, 13),
                                      (1, 2, 128, 128), (1, 1, 127, 63), (1, 2, 100, 20), (1, 1, 128, 96)])
@pytest.mark.parametrize("layout", ["columns", "odd"])
def test_steps_follow_the_sequence(gpu, Hk, H, K, V, dt, layout):
    """Each step within a bar of the definition, the state carried from one to the next."""
    T, B = 5, 6
    p = inputs(T, B, Hk, H, K, V, dt, layout=layout)
    done, first = flags(3, 0.3, T, B), flags(4, 0.5, B)
    h = cu(5, B, H, K, V)
    yr, hr = R.delta({n: host(t) for n, t in p.items()}, None, host(done), host(first), host(h))
    f = first
    for t in range(T):
        y = D.delta_step(*[p[n][t] for n in "qkvab"], p["A"], h, dt_bias=p["dt_bias"], first=f)
        close(y, yr[t], BAR[dt], t)
        f = done[t].contiguous()
    close(h, hr, BAR[dt], "h")


@pytest.mark.parametrize("T", [40, 600])
def test_state_in_place_and_rows_left_alone(gpu, T):
    B, H, K, V = 2, 2, 16, 24
    p = inputs(T, B, 1, H, K, V, BF)
    args = [p[n] for n in "qkvabA"]
    h0, h = cu(5, B, H, K, V), torch.empty(B, H, K, V, device="cuda")
    y = D.delta_scan(*args, h0=h0, h_out=h)
    wide = torch.full((T + 3, B, H, V + 8), 7.0, device="cuda", dtype=BF)
    h1 = h0.clone()
    D.delta_scan(*args, h0=h1, h_out=h1, out=wide[:T, :, :, 3:V + 3])
    assert torch.equal(wide[:T, :, :, 3:V + 3], y) and torch.equal(h, h1)
    assert (wide[T:] == 7).all() and (wide[..., :3] == 7).all() and (wide[..., V + 3:] == 7).all()


@pytest.mark.parametrize("T", [90, 500])
def test_whole_and_in_parts(gpu, T):
    """A sequence in two calls, the state and its gradient handed over, is the sequence in one."""
    B, H, K, V = 2, 2, 32, 24
    p = inputs(T, B, 2, H, K, V, F32)
    done, dy = flags(3, 0.05, T, B), cu(6, T, B, H, V)
    args = lambda s: [p[n][s] for n in "qkvab"] + [p["A"]]
    kw = dict(dt_bias=p["dt_bias"])
    y, saved = D.delta_scan(*args(slice(0, T)), done=done, save=True, **kw)
    g = D.delta_scan_grad(*args(slice(0, T)), saved, dy, done=done, **kw)
    one, two, h = slice(0, 37), slice(37, T), torch.empty(B, H, K, V, device="cuda")
    y1, s1 = D.delta_scan(*args(one), done=done[one].contiguous(), h_out=h, save=True, **kw)
    first = done[36].contiguous()
    y2, s2 = D.delta_scan(*args(two), done=done[two].contiguous(), first=first, h0=h, save=True, **kw)
    assert rel(torch.cat([y1, y2]), y) <= 2 * BAR[F32]
    dh = torch.empty_like(h)
    g2 = D.delta_scan_grad(*args(two), s2, dy[two].contiguous(), done=done[two].contiguous(), first=first, dh0=dh, **kw)
    g1 = D.delta_scan_grad(*args(one), s1, dy[one].contiguous(), done=done[one].contiguous(), dh=dh, dh0=dh, **kw)
    for n in "qkvab":
        assert rel(torch.cat([g1["d" + n], g2["d" + n]]), g["d" + n]) <= 2 * BAR[F32] * (10 if n == "a" else 1), n
    for n in ("dA", "ddt_bias"):
        assert rel(g1[n] + g2[n], g[n]) <= 20 * BAR[F32]


def test_gradient_against_differences(gpu):
    """Along one direction a parameter: central differences of the fp32 forward, sums in 64 bits. A step of 2^-7 leaves an error
    of its square (6e-5) times third derivatives of the order of the gradient, and 1e-5 of the objective's terms over it: 1 %."""
    T, B, Hk, H, K, V = 37, 3, 1, 2, 16, 24
    p = {n: t.clone() for n, t in inputs(T, B, Hk, H, K, V, F32).items()}
    done, dy = flags(3, 0.1, T, B), cu(6, T, B, H, V)
    f = lambda q: float((D.delta_scan(*[q[n] for n in "qkvabA"], dt_bias=q["dt_bias"], done=done).double() * dy.double()).sum())
    args = [p[n] for n in "qkvabA"]
    _, saved = D.delta_scan(*args, dt_bias=p["dt_bias"], done=done, save=True)
    g = D.delta_scan_grad(*args, saved, dy, dt_bias=p["dt_bias"], done=done)
    for n in p:
        d = g["d" + n] / g["d" + n].norm() * (p[n].numel() ** 0.5 * 0.3 if p[n].dim() > 1 else 0.3)
        e = 2.0 ** -7
        got = (f(dict(p, **{n: p[n] + e * d})) - f(dict(p, **{n: p[n] - e * d}))) / (2 * e)
        want = float((g["d" + n].double() * d.double()).sum())
        assert abs(got - want) <= 0.01 * abs(want), (n, got, want)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("T", [100, 700])
def test_same_call_same_bits(gpu, T, dt):
    p = inputs(T, 9, 2, 4, 32, 32, dt)
    dy, done = cu(6, T, 9, 4, 32, dtype=dt), flags(3, 0.1, T, 9)
    args = [p[n] for n in "qkvabA"]
    runs = []
    for _ in range(2):
        y, saved = D.delta_scan(*args, dt_bias=p["dt_bias"], done=done, save=True)
        runs.append(dict(D.delta_scan_grad(*args, saved, dy, dt_bias=p["dt_bias"], done=done), y=y))
    for n in runs[0]:
        assert torch.equal(runs[0][n], runs[1][n]), n


def test_no_sequences(gpu):
    p = inputs(5, 0, 1, 2, 8, 8, F32)
    args = [p[n] for n in "qkvabA"]
    y, saved = D.delta_scan(*args, dt_bias=p["dt_bias"], save=True)
    g = D.delta_scan_grad(*args, saved, torch.empty_like(y), dt_bias=p["dt_bias"])
    assert y.shape == (5, 0, 2, 8) and not g["dA"].any() and not g["ddt_bias"].any()
    p = inputs(1, 0, 1, 2, 8, 8, F32)
    assert D.delta_step(*[p[n][0] for n in "qkvab"], p["A"], torch.empty(0, 2, 8, 8, device="cuda")).shape == (0, 2, 8)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("T", [50, 400])
def test_captured(gpu, T, dt):
    """Forward, gradient and a step in one graph on a stream of its own, replayed between eager work."""
    B, Hk, H, K, V = 4, 1, 2, 32, 32
    p = inputs(T, B, Hk, H, K, V, dt)
    dy, h = cu(6, T, B, H, V, dtype=dt), cu(5, B, H, K, V)
    args = [p[n] for n in "qkvabA"]

    def work(state):
        y, saved = D.delta_scan(*args, h0=state, h_out=state, save=True)
        g = D.delta_scan_grad(*args, saved, dy)
        return dict(g, y=y, step=D.delta_step(*[p[n][0] for n in "qkvab"], p["A"], state))

    eager, states = [], h.clone()
    for _ in range(3):
        eager.append({n: t.clone() for n, t in work(states).items()})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = h.clone()
    with torch.cuda.stream(side):
        work(state)
        state.copy_(h)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = work(state)
    torch.cuda.synchronize()
    state.copy_(h)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for n, t in out.items():
            assert torch.equal(t, eager[i][n]), (i, n)
        work(h.clone())
        torch.cuda.synchronize()
    assert torch.equal(state, states)


def test_more_sequences_than_a_launch_has_blocks(gpu):
    """2^20 blocks go on to further sequences: copies of 64, compared with them."""
    B, K, V, T = 2 ** 20 + 70, 8, 4, 3
    p = inputs(T, 64, 1, 1, K, V, BF, layout="packed")
    far = {n: (t if t.dim() == 1 else t.repeat(1, -(-B // 64), *[1] * (t.dim() - 2))[:, :B].contiguous()) for n, t in p.items()}
    dy = cu(6, T, 64, 1, V, dtype=BF)
    outs = []
    for q, d in ((p, dy), (far, dy.repeat(1, -(-B // 64), 1, 1)[:, :B].contiguous())):
        args = [q[n] for n in "qkvabA"]
        y, saved = D.delta_scan(*args, save=True)
        g = D.delta_scan_grad(*args, saved, d)
        outs.append(dict(y=y, dq=g["dq"], dk=g["dk"], dv=g["dv"], da=g["da"], db=g["db"]))
    for n in outs[0]:
        a, b = outs
        assert torch.equal(b[n][:, -70:-6], a[n].roll(-(B - 70) % 64, 1)) and torch.equal(b[n][:, :64], a[n]), n
