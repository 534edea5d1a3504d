"""The selective state-space scan, its gradient and its single step against the recurrence in 64 bits.

Bars, relative 2-norm: a state after t steps carries at most t times the rounding of a decay and an update, about three
errors of 2^-24, so 70 steps stay under 1.3e-5 and 2e-5 holds for every fp32 result here (200 steps: 4e-5); bf16 results
add their one rounding."""
import numpy as np
import pytest
import torch

import policy_layer_ref as R
from pufferlean_amd import _lib as L
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
FP32 = 2e-5
NAMES = ("x", "delta", "Bm", "Cm", "z", "A", "D", "dt_bias", "conv_w", "conv_b")


def cu(seed, *shape, scale=1.0, dtype=torch.float32):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", dtype)


def place(t, layout):
    """[T, B, n] in one of the layouts a caller may hold."""
    if layout == "packed":
        return t.contiguous()
    if layout == "batch":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    T, B, n = t.shape
    buf = torch.full((T, B, n + 5), 3.0, device="cuda", dtype=t.dtype)
    buf[..., 1:n + 1] = t
    return buf[..., 1:n + 1]


def inputs(T, B, C, N, G=1, K=4, dt=torch.float32, gate=True, done=True, carry=True, layout="packed", extras=True):
    s = dict(x=cu(1, T, B, C, dtype=dt), delta=cu(2, T, B, C, scale=0.7, dtype=dt), Bm=cu(3, T, B, G * N, dtype=dt),
             Cm=cu(4, T, B, G * N, dtype=dt), z=cu(5, T, B, C, dtype=dt) if gate else None)
    s = {k: None if v is None else place(v, layout) for k, v in s.items()}
    s["A"] = -torch.exp(cu(6, C, N, scale=0.7))
    s["D"] = cu(7, C) if extras else None
    s["dt_bias"] = cu(8, C) - 2 if extras else None
    s["conv_w"] = cu(9, C, K, scale=0.6) if K else None
    s["conv_b"] = cu(10, C, scale=0.3) if K and extras else None
    c = dict(groups=G)
    c["done"] = torch.from_numpy(rng.bernoulli(11, T * B, 0.15).reshape(T, B)).float().cuda() if done else None
    c["first"] = torch.from_numpy(rng.bernoulli(12, B, 0.4)).float().cuda() if carry else None
    c["h0"] = cu(13, B, C, N) if carry else None
    c["win0"] = cu(14, B, K - 1, C) if carry and K > 1 else None
    return s, c


def forward(s, c, **kw):
    T, B, C = s["x"].shape
    h = torch.full((B, C, s["A"].shape[1]), 9.0, device="cuda")
    K = 0 if s["conv_w"] is None else s["conv_w"].shape[1]
    win = torch.full((B, K - 1, C), 9.0, device="cuda") if K > 1 else None
    rest = {k: s[k] for k in ("D", "z", "dt_bias", "conv_w", "conv_b")}
    y, saved = D.ssm_scan(s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], h_out=h, win_out=win, save=True, **rest, **c, **kw)
    return y, h, win, saved


def backward(s, c, saved, dy, **kw):
    rest = {k: s[k] for k in ("D", "z", "dt_bias", "conv_w", "conv_b")}
    cc = {k: v for k, v in c.items() if k != "h0"}
    return D.ssm_scan_grad(s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], saved, dy, **rest, **cc, **kw)


def reference(s, c, dy=None):
    p = {k: R.leaf(s[k]) for k in NAMES}
    host = {k: None if v is None or k == "groups" else v.double().cpu() for k, v in c.items()}
    host["groups"] = c["groups"]
    y, h, win = R.scan(p, **host)
    if dy is None:
        return y, h, win
    have = [k for k in NAMES if p[k] is not None]
    g = torch.autograd.grad(y, [p[k] for k in have], dy.double().cpu())
    return y, h, win, {"d" + k: v for k, v in zip(have, g)}


def check(s, c, bar=FP32, layout="packed"):
    dt = s["x"].dtype
    out = bar + (R.BF16 if dt == torch.bfloat16 else 0.0)
    dy = place(cu(20, *s["x"].shape, dtype=dt), layout)
    y, h, win, saved = forward(s, c)
    g = backward(s, c, saved, dy)
    yr, hr, wr, gr = reference(s, c, dy)
    assert R.rel(y, yr) <= out and R.rel(h, hr) <= bar
    if win is not None:
        assert torch.equal(win.double().cpu(), wr.detach())
    assert set(g) == set(gr)
    for k in g:
        assert R.rel(g[k], gr[k]) <= (out if g[k].dtype == dt and k in ("dx", "ddelta", "dBm", "dCm", "dz") else bar), k
    return y, h, win, g


@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 16, 31, 33, 64, 70])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_lengths(gpu, T, dt):
    check(*inputs(T, 3, 20, 5, dt=dt))


@pytest.mark.parametrize("N", [1, 3, 4, 7, 8, 13, 16, 17, 24, 32, 33, 64])
def test_states(gpu, N):
    check(*inputs(19, 2, 70, N))
    check(*inputs(19, 2, 70, N, G=2, dt=torch.bfloat16))


@pytest.mark.parametrize("K", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("done", [True, False])
def test_taps_gates_and_ends(gpu, K, gate, done):
    check(*inputs(45, 3, 33, 6, K=K, gate=gate, done=done, carry=done, extras=gate))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [9, 70])
def test_bias_without_taps(gpu, T, dt):
    """Without taps u is x: a bias of the convolution changes nothing, and its gradient is zero."""
    s, c = inputs(T, 2, 40, 4, K=0, dt=dt)
    dy = cu(20, T, 2, 40, dtype=dt)
    y, h, _, saved = forward(s, c)
    ref = backward(s, c, saved, dy)
    for w in (None, torch.empty(40, 0, device="cuda")):
        sb = dict(s, conv_w=w, conv_b=cu(10, 40))
        yb, hb, _, kept = forward(sb, c)
        g = backward(sb, c, kept, dy)
        assert torch.equal(yb, y) and torch.equal(hb, h)
        assert g["dconv_b"].shape == (40,) and not g["dconv_b"].any()
        for k in ref:
            assert torch.equal(g[k], ref[k]), k


@pytest.mark.parametrize("C,G", [(1, 1), (64, 1), (65, 1), (128, 2), (130, 2), (300, 3), (520, 1), (600, 1), (1100, 2)])
def test_channels_and_groups(gpu, C, G):
    check(*inputs(11, 2, C, 8, G=G, dt=torch.bfloat16))


@pytest.mark.parametrize("layout", ["batch", "slice"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_layouts(gpu, layout, dt):
    a = check(*inputs(37, 4, 40, 16, dt=dt, layout=layout), layout=layout)
    b = check(*inputs(37, 4, 40, 16, dt=dt))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for k in a[3]:
        assert torch.equal(a[3][k], b[3][k]), k


def test_outputs_into_slices(gpu):
    s, c = inputs(21, 3, 24, 4)
    dy = cu(20, 21, 3, 24)
    y, h, win, saved = forward(s, c)
    ref = backward(s, c, saved, dy)
    buf = torch.full((21, 3, 24 * 3 + 8 + 2), 5.0, device="cuda")
    dx, dz, dd, dB, dC = buf[..., 1:-1].split([24, 24, 24, 4, 4], dim=-1)
    backward(s, c, saved, dy, dx=dx, dz=dz, ddelta=dd, dBm=dB, dCm=dC)
    for k, t in dict(dx=dx, dz=dz, ddelta=dd, dBm=dB, dCm=dC).items():
        assert torch.equal(t, ref[k]), k
    assert torch.all(buf[..., 0] == 5) and torch.all(buf[..., -1] == 5)


def test_many_sequences_and_long_ones(gpu):
    check(*inputs(9, 60, 72, 16, dt=torch.bfloat16))
    check(*inputs(200, 2, 24, 4), bar=4e-5)


@pytest.mark.parametrize("T,N,K,carry,dt", [(13, 5, 3, True, torch.float32), (21, 16, 4, True, torch.bfloat16), (8, 4, 4, False, torch.float32)])
def test_blocks_of_several_sequences(gpu, T, N, K, carry, dt):
    """4500 sequences are more than the gradient's blocks run at a time (2048 of 64 channels), so a block goes on to its next
    ones; in parts of 1500 it has one. A sequence's own outputs are the same bit for bit. The parameters' sums are over the same
    terms in another order: chains of under 3000 additions that round by 2^-24 each, independently."""
    s, c = inputs(T, 4500, 16, N, K=K, dt=dt, carry=carry)
    dy = cu(20, T, 4500, 16, dtype=dt)
    y, h, _, saved = forward(s, c)
    g = backward(s, c, saved, dy)
    sums = {}
    for b in range(0, 4500, 1500):
        part = slice(b, b + 1500)
        sp = {k: v[:, part] if k in ("x", "delta", "Bm", "Cm", "z") and v is not None else v for k, v in s.items()}
        cp = {k: v if v is None or k == "groups" else v[:, part].contiguous() if k == "done" else v[part].contiguous()
              for k, v in c.items()}
        yp, hp, _, kept = forward(sp, cp)
        gp = backward(sp, cp, kept, dy[:, part].contiguous())
        assert torch.equal(yp, y[:, part]) and torch.equal(hp, h[part])
        for k, v in gp.items():
            if k in ("dx", "ddelta", "dBm", "dCm", "dz"):
                assert torch.equal(v, g[k][:, part]), k
            else:
                sums[k] = sums.get(k, 0) + v.double()
    assert sums and set(sums) | {"dx", "ddelta", "dBm", "dCm", "dz"} == set(g)
    for k, v in sums.items():
        assert R.rel(g[k], v) <= 2e-5, k


# (T, C, N, G, K, dtype, gate) of three sequences that both directions cut into chunks of 32 steps: whole last chunks and ones of
# 1 to 7 steps, every number of taps, groups, several wavefronts and blocks of channels, any number of states.
CHUNKED = [(160, 20, 16, 1, 4, torch.float32, True), (150, 70, 16, 1, 4, torch.float32, True), (129, 40, 16, 1, 4, torch.bfloat16, True),
           (129, 40, 16, 1, 3, torch.float32, True), (161, 96, 16, 2, 4, torch.bfloat16, True), (130, 33, 16, 1, 4, torch.float32, False),
           (131, 66, 16, 2, 2, torch.float32, True), (135, 20, 16, 1, 1, torch.float32, True), (200, 70, 16, 1, 0, torch.bfloat16, True),
           (290, 24, 4, 1, 4, torch.float32, True), (210, 90, 7, 1, 2, torch.bfloat16, False), (140, 130, 24, 2, 3, torch.bfloat16, True),
           (150, 300, 16, 1, 4, torch.bfloat16, True), (134, 40, 64, 1, 4, torch.float32, True)]


def chunked(T, C, N, G, K, dt, gate, B=3):
    """Half of the channels decay slowly, so that what a chunk starts from shows to its end; episodes end on and around the
    chunks' borders, at the last step, and in one sequence never."""
    s, c = inputs(T, B, C, N, G=G, K=K, dt=dt, gate=gate)
    s["A"][::2] *= 0.05
    c["done"].zero_()
    for b, steps in enumerate(((31, 95, T - 1), (28, 30, 32, 62, 63, 127))):
        c["done"][list(steps), b] = 1.0
    return s, c


@pytest.mark.parametrize("T,C,N,G,K,dt,gate", CHUNKED)
def test_chunks_of_time(gpu, T, C, N, G, K, dt, gate):
    # the bar of the head of this file for T steps
    check(*chunked(T, C, N, G, K, dt, gate), bar=max(FP32, 3 * T * 2.0 ** -24))


@pytest.mark.parametrize("K", [1, 2, 3, 4])
def test_chunks_carry_in_place(gpu, K):
    """h_out and win_out may be h0 and win0, where the first chunk reads what the last one writes; and two calls that hand the
    state on are one."""
    s, c = chunked(300, 40, 16, 1, K, torch.float32, True)
    y, h, win, _ = forward(s, c)
    rest = {k: s[k] for k in ("D", "z", "dt_bias", "conv_w", "conv_b")}
    hs, ws = c["h0"].clone(), None if K < 2 else c["win0"].clone()
    own = {k: v for k, v in c.items() if k not in ("h0", "win0")}
    yp = D.ssm_scan(s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], h0=hs, win0=ws, h_out=hs, win_out=ws, **rest, **own)
    assert torch.equal(yp, y) and torch.equal(hs, h) and (K < 2 or torch.equal(ws, win))
    hs, ws, first = c["h0"].clone(), None if K < 2 else c["win0"].clone(), c["first"]
    for t in (0, 150):
        part = {k: v[t:t + 150] if k in ("x", "delta", "Bm", "Cm", "z") else v for k, v in s.items()}
        rest = {k: part[k] for k in ("D", "z", "dt_bias", "conv_w", "conv_b")}
        done = c["done"][t:t + 150].contiguous()
        yp = D.ssm_scan(part["x"], part["delta"], s["A"], part["Bm"], part["Cm"], done=done, first=first, h0=hs, win0=ws,
                        h_out=hs, win_out=ws, **rest)
        assert R.rel(yp, y[t:t + 150]) <= 2 * 3 * 300 * 2.0 ** -24
        first = done[-1].contiguous()
    assert R.rel(hs, h) <= 2 * 3 * 300 * 2.0 ** -24 and (K < 2 or torch.equal(ws, win))


def test_chunks_keep_non_finite_values_in_their_episode(gpu):
    """Infinities and NaN in the first and the last chunk; the episode between them is the same bit for bit."""
    T, lo, hi = 150, 40, 101
    s, c = chunked(T, 40, 16, 1, 4, torch.float32, True)
    c["done"].zero_()
    c["done"][[lo - 1, hi - 1]] = 1.0
    bad = {k: v.clone() if k in ("x", "delta", "Bm", "Cm", "z") else v for k, v in s.items()}
    bad["x"][20], bad["x"][lo - 1], bad["x"][hi] = float("inf"), float("inf"), float("-inf")
    bad["Bm"][25], bad["Cm"][140], bad["z"][hi] = float("nan"), float("inf"), float("nan")
    dy = cu(20, T, 3, 40)
    y, h, _, saved = forward(s, c)
    g = backward(s, c, saved, dy)
    yb, hb, _, kept = forward(bad, c)
    gb = backward(bad, c, kept, dy)
    assert torch.isfinite(y).all() and not torch.isfinite(yb[:lo]).all() and not torch.isfinite(yb[hi:]).all()
    assert torch.equal(yb[lo:hi], y[lo:hi])
    for k in ("dx", "ddelta", "dBm", "dCm", "dz"):
        assert torch.equal(gb[k][lo:hi], g[k][lo:hi]), k


def test_chunks_in_a_graph(gpu):
    s, c = chunked(150, 72, 16, 1, 4, torch.bfloat16, True)
    dy = cu(20, 150, 3, 72, dtype=torch.bfloat16)

    def both():
        y, h, win, saved = forward(s, c)
        return [y, h, win, *backward(s, c, saved, dy).values()]
    ref = [t.clone() for t in both()]
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st), torch.cuda.graph(g, stream=st):
        out = both()
    torch.cuda.current_stream().wait_stream(st)
    for _ in range(3):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ref, out))
        assert all(torch.equal(p, q) for p, q in zip(ref, both()))


def test_every_step_ends_an_episode(gpu):
    s, c = inputs(40, 2, 16, 4, K=4)
    c["done"].fill_(1.0)
    c["first"].fill_(1.0)
    check(s, c)


def test_state_carried_over_calls(gpu):
    """One call over 50 steps equals five of 10 with the state handed on in place, ends of episodes included."""
    s, c = inputs(50, 3, 40, 8, carry=True)
    y, h, win, _ = forward(s, c)
    hs, ws, first = c["h0"].clone(), c["win0"].clone(), c["first"]
    for t in range(0, 50, 10):
        part = {k: v[t:t + 10] if k in ("x", "delta", "Bm", "Cm", "z") else v for k, v in s.items()}
        rest = {k: part[k] for k in ("D", "z", "dt_bias", "conv_w", "conv_b")}
        done = c["done"][t:t + 10].contiguous()
        yp = D.ssm_scan(part["x"], part["delta"], s["A"], part["Bm"], part["Cm"], done=done, first=first, h0=hs, win0=ws,
                        h_out=hs, win_out=ws, **rest)
        assert R.rel(yp, y[t:t + 10]) <= FP32
        first = done[-1].contiguous()
    assert R.rel(hs, h) <= FP32 and torch.equal(ws, win)


@pytest.mark.parametrize("T", [12, 60])
def test_non_finite_values_stay_in_their_episode(gpu, T):
    s, c = inputs(T, 2, 20, 4, K=3)
    c["done"].zero_()
    c["done"][T // 2 - 1] = 1.0
    cut = T // 2
    bad = {k: v.clone() if k in ("x", "delta", "Bm", "Cm", "z") and v is not None else v for k, v in s.items()}
    bad["x"][cut - 1] = float("inf")
    bad["Bm"][cut - 2] = float("nan")
    c["h0"][:] = float("nan")
    c["first"].fill_(1.0)
    y, h, win, saved = forward(s, c)
    yb, hb, wb, sb = forward(bad, c)
    assert torch.isfinite(y).all()  # the carried state was cleared
    assert torch.equal(yb[cut:], y[cut:]) and torch.equal(hb, h) and torch.equal(wb, win)
    dy = cu(20, T, 2, 20)
    g, gb = backward(s, c, saved, dy), backward(bad, c, sb, dy)
    for k in ("dx", "ddelta", "dBm", "dCm", "dz"):
        assert torch.equal(gb[k][cut:], g[k][cut:]), k


def test_unused_taps_do_not_see_infinities(gpu):
    s, c = inputs(20, 1, 8, 2, K=2, done=False, carry=False)
    s["x"][3] = float("inf")
    y, *_ = forward(s, c)
    assert torch.isfinite(y[:3]).all()
    yr, *_ = reference(s, c)
    bad = ~torch.isfinite(yr[5:])
    assert torch.equal(bad, ~torch.isfinite(y[5:]).cpu())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_extreme_time_steps(gpu, dt):
    """delta far below and above: decays of one and of zero, without a NaN."""
    s, c = inputs(40, 2, 16, 4, dt=dt)
    s["delta"][::3] = -200.0
    s["delta"][1::3] = 60.0
    check(s, c, bar=4e-5)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K", [(1, 4), (4, 0), (5, 4), (8, 2), (12, 4), (16, 4), (17, 1), (32, 3), (64, 4)])
def test_step(gpu, dt, N, K):
    s, c = inputs(3, 7, 50, N, K=K, dt=dt, G=2, done=False)
    yr, hr, wr = reference(s, c)
    h, win = c["h0"].clone(), None if K < 2 else c["win0"].clone()
    rest = {k: s[k] for k in ("D", "dt_bias", "conv_w", "conv_b")}
    for t in range(3):
        y = D.ssm_step(s["x"][t], s["delta"][t], s["A"], s["Bm"][t], s["Cm"][t], h, win, z=s["z"][t], groups=2,
                       first=c["first"] if t == 0 else None, **rest)
        assert R.rel(y, yr[t]) <= FP32 + (R.BF16 if dt == torch.bfloat16 else 0)
    assert R.rel(h, hr) <= FP32
    if win is not None:
        assert torch.equal(win.double().cpu(), wr.detach())


def test_step_clears_non_finite_state(gpu):
    s, c = inputs(1, 4, 30, 8, done=False)
    c["first"].fill_(1.0)
    h, win = torch.full_like(c["h0"], float("nan")), torch.full_like(c["win0"], float("inf"))
    rest = {k: s[k] for k in ("D", "dt_bias", "conv_w", "conv_b")}
    y = D.ssm_step(s["x"][0], s["delta"][0], s["A"], s["Bm"][0], s["Cm"][0], h, win, z=s["z"][0], first=c["first"], **rest)
    assert torch.isfinite(y).all() and torch.isfinite(h).all() and torch.isfinite(win).all()


def test_no_sequences(gpu):
    s, c = inputs(4, 1, 12, 4, done=False, carry=False)
    e = {k: v[:, :0] if k in ("x", "delta", "Bm", "Cm", "z") else v for k, v in s.items()}
    y, h, win, saved = forward(e, dict(groups=1))
    g = backward(e, dict(groups=1), saved, e["x"])
    assert y.shape == (4, 0, 12) and all(not v.any() for k, v in g.items())


def test_offsets_past_32_bits(gpu):
    """Steps 2^30 elements apart: the third lies past 2^31."""
    T, B, C, N = 4, 1, 16, 4
    s, c = inputs(T, B, C, N, done=False)
    buf = torch.empty(3 * 2 ** 30 + 64, device="cuda", dtype=torch.float32)
    far = buf.as_strided((T, B, C), (2 ** 30, C, 1))
    far.copy_(s["x"])
    y, *_ = forward(s, c)
    yf, *_ = forward(dict(s, x=far), c)
    assert torch.equal(y, yf)


def test_more_threads_than_a_launch_has(gpu):
    """A group of one channel takes a wavefront, and 2^26 wavefronts are more than one row of a launch has. Copies of 4096 sequences,
    and eight of their own at the end."""
    n, B, C, N = 4096, 2 ** 20 + 8, 64, 1
    s, c = inputs(1, n + 8, C, N, G=C, K=2, done=False)
    ref = forward(s, c)
    far = lambda t, d: torch.cat([t.narrow(d, 0, n).repeat(*(B // n if i == d else 1 for i in range(t.dim()))), t.narrow(d, n, 8)], d)
    sf = {k: far(v, 1) if k in ("x", "delta", "Bm", "Cm", "z") else v for k, v in s.items()}
    cf = dict(c, first=far(c["first"], 0), h0=far(c["h0"], 0), win0=far(c["win0"], 0))
    got = forward(sf, cf)
    for a, b, d in zip(got[:3], ref[:3], (1, 0, 0)):
        assert torch.equal(a, far(b, d))
    dy = cu(20, 1, n + 8, C)
    gr, gg = backward(s, c, ref[3], dy), backward(sf, cf, got[3], far(dy, 1))
    for k in ("dx", "ddelta", "dBm", "dCm", "dz"):
        assert torch.equal(gg[k], far(gr[k], 1)), k


def test_more_parameter_sums_than_a_launch_has(gpu):
    """2^24 channels of 60 states have over 2^30 parameters, four threads each. Channels of one group are their own but for dB and dC,
    so the first and the last ones are those of a small call."""
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("needs 50 GB")
    C, n = 2 ** 24, 128
    s, c = inputs(1, 1, n, 60, done=False, carry=False)
    dy = cu(20, 1, 1, n)
    _, _, _, saved = forward(s, c)
    ref = backward(s, c, saved, dy)
    chans = dict(x=-1, delta=-1, z=-1, A=0, D=0, dt_bias=0, conv_w=0, conv_b=0)
    far = lambda t, d: t.repeat(*(C // n if i == d % t.dim() else 1 for i in range(t.dim())))
    sf = {k: far(v, chans[k]) if k in chans else v for k, v in s.items()}
    rest = {k: sf[k] for k in ("D", "z", "dt_bias", "conv_w", "conv_b")}
    _, saved = D.ssm_scan(sf["x"], sf["delta"], sf["A"], sf["Bm"], sf["Cm"], save=True, **rest)
    got = backward(sf, c, saved, far(dy, -1))
    for k in ("dA", "dD", "ddt_bias", "dconv_w", "dconv_b"):
        assert torch.equal(got[k][:n], ref[k]) and torch.equal(got[k][-n:], ref[k]) and torch.equal(got[k][C // 2:C // 2 + n], ref[k]), k
    del sf, rest, saved, got
    torch.cuda.empty_cache()
    L.call("ph_release_scratch")


def test_gradient_against_differences(gpu):
    s, c = inputs(40, 2, 24, 4)
    dy = cu(20, 40, 2, 24)
    y, h, win, saved = forward(s, c)
    g = backward(s, c, saved, dy)
    e = 2.0 ** -8
    for i, k in enumerate(NAMES):
        v = cu(30 + i, *s[k].shape, scale=float(s[k].abs().mean()))
        f = [float((forward(dict(s, **{k: s[k] + m * e * v}), c)[0].double() * dy.double()).sum()) for m in (1, -1)]
        want, size = float((g["d" + k] * v).sum()), float(g["d" + k].norm() * v.norm())
        # the difference's own error: e^2 of a third derivative, and 2^-24 / e of |y| |dy|
        assert abs((f[0] - f[1]) / (2 * e) - want) <= 2e-3 * (abs(want) + 0.1 * size) + 2e-5 * float(y.norm() * dy.norm()), k


def test_same_twice_and_on_another_stream(gpu):
    s, c = inputs(70, 5, 100, 16, dt=torch.bfloat16)
    dy = cu(20, 70, 5, 100, dtype=torch.bfloat16)

    def both():
        y, h, win, saved = forward(s, c)
        return [y, h, win, *backward(s, c, saved, dy).values()]
    a = both()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b = both()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graph_replays(gpu):
    s, c = inputs(70, 3, 72, 16, dt=torch.bfloat16)
    dy = cu(20, 70, 3, 72, dtype=torch.bfloat16)

    def both():
        y, h, win, saved = forward(s, c)
        return [y, h, win, *backward(s, c, saved, dy).values()]
    ref = [t.clone() for t in both()]
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st), torch.cuda.graph(g, stream=st):
        out = both()
    torch.cuda.current_stream().wait_stream(st)
    for _ in range(3):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ref, out))
        (torch.ones(1000, device="cuda") * 2).sum().item()


@pytest.mark.parametrize("T,C,G", [(21, 24, 1), (70, 66, 2), (70, 300, 1)])
def test_gradients_left_out(gpu, T, C, G):
    """Each gradient may be left out; the others stay the same. With whole sequences and with chunks of time, with one block of
    channels and with two."""
    s, c = inputs(T, 3, C, 16, G=G, dt=torch.bfloat16)
    dy = cu(20, T, 3, C, dtype=torch.bfloat16)
    _, _, _, saved = forward(s, c)
    ref = backward(s, c, saved, dy)
    a = D._ssm_args(True, s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"], s["dt_bias"], s["conv_w"], s["conv_b"], G, c["done"],
                    c["first"], None, c["win0"])[0]
    acts, pars = ("dx", "dz", "ddelta", "dBm", "dCm"), ("dA", "dD", "ddt_bias", "dconv_w", "dconv_b")
    sets = [set(ref) - {k} for k in ref] + [{k} for k in ref] + [set()]
    for keep in sets:
        out = {k: torch.full_like(ref[k], 7.0) for k in keep}
        ptr = lambda k: out[k].data_ptr() if k in out else 0
        g = D._SSM_GRADS.pack(*map(ptr, acts), *(n for k in acts for n in ref[k].stride()[:2]), *map(ptr, pars))
        L.call("ph_ssm_scan_grad", a, saved.data_ptr(), dy.data_ptr(), dy.stride(0), dy.stride(1), g, D._stream())
        for k in keep:
            assert torch.equal(out[k], ref[k]), (k, keep)


def test_refusals(gpu):
    s, c = inputs(6, 2, 12, 4, done=False, carry=False)
    call = lambda **kw: forward({**s, **{k: v for k, v in kw.items() if k in s}}, {**c, **{k: v for k, v in kw.items() if k not in s}})
    call()
    with pytest.raises(TypeError):
        call(x=s["x"].double())
    with pytest.raises(ValueError):
        call(delta=s["delta"].bfloat16())
    with pytest.raises(ValueError):
        call(Bm=s["Bm"][..., :3])
    with pytest.raises(ValueError):
        call(A=s["A"].t().contiguous().t())
    with pytest.raises(ValueError):
        call(groups=5)
    with pytest.raises(ValueError):
        call(done=torch.zeros(2, 6, device="cuda"))
    with pytest.raises(ValueError):
        call(h0=torch.zeros(2, 12, 5, device="cuda"))
    with pytest.raises(ValueError):
        call(x=s["x"].transpose(0, 2))
    with pytest.raises(L.PufferHipError, match="N = 65"):
        D.ssm_scan(s["x"], s["delta"], torch.ones(12, 65, device="cuda"), torch.ones(6, 2, 65, device="cuda"),
                   torch.ones(6, 2, 65, device="cuda"))
    with pytest.raises(L.PufferHipError, match="K = 5"):
        call(conv_w=torch.ones(12, 5, device="cuda"))
    with pytest.raises(L.PufferHipError, match="no steps"):
        D.ssm_scan(s["x"][:0], s["delta"][:0], s["A"], s["Bm"][:0], s["Cm"][:0])
    y, h, win, saved = call()
    with pytest.raises(ValueError):
        backward(s, c, saved[:-1], y)
    with pytest.raises(ValueError):
        D.ssm_step(s["x"][0], s["delta"][0], s["A"], s["Bm"][0], s["Cm"][0], h, None, conv_w=s["conv_w"])
