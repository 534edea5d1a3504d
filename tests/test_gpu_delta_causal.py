"""The gated delta rule: no step sees a later one, whatever that holds. Steps in front of a value that is not finite, and the columns of V
that it does not enter, give what they give without it, within the bars of the clean sequence (two results, each within its bar)."""
import pytest
import torch

from policy_layer_ref import rel
from pufferlean_amd import device as D
from test_gpu_delta import BAR, BF, F32, cu, flags, inputs
import delta_layer_ref as R

pytestmark = pytest.mark.gpu


def scan(p, h0, done=None):
    h = torch.empty_like(h0)
    return D.delta_scan(*[p[n] for n in "qkvabA"], dt_bias=p["dt_bias"], done=done, h0=h0, h_out=h), h


def same(x, clean, what):
    bar = 2 * BAR[x.dtype] + (2 * R.BF16 if x.dtype == BF else 0)
    assert x.isfinite().all(), what
    assert rel(x, clean) <= bar, (what, rel(x, clean))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("T,at", [(1, 0), (30, 29), (33, 1), (70, 5), (70, 40), (70, 63), (410, 17), (410, 300)])
@pytest.mark.parametrize("K,V", [(16, 24), (64, 64), (100, 72)])
def test_steps_in_front(gpu, K, V, T, at, value, dt):
    """One value in one sequence and, for v, one column: from its step on y may be anything there."""
    B, H = 2, 2
    clean = {n: t.clone() for n, t in inputs(T, B, 1, H, K, V, dt).items()}
    h0 = cu(5, B, H, K, V)
    y0, hc = scan(clean, h0)
    for name in "kvab" if value != value else "kv":
        p = {n: t.clone() for n, t in clean.items()}
        p[name][at, 1, ..., V // 2 if name == "v" else 0] = value  # of every head
        y, h = scan(p, h0)
        same(y[:, 0], y0[:, 0], (name, "another sequence"))
        if at:
            same(y[:at], y0[:at], (name, "steps in front"))
        heads = slice(1, None) if name in "ab" else slice(0, 0) if name == "k" else slice(None)
        if name == "v":
            cols = torch.arange(V) != V // 2
            same(y[..., cols], y0[..., cols], (name, "other columns"))
            same(h[..., cols], hc[..., cols], (name, "other columns of the state"))
            assert not h[1, :, :, V // 2].isfinite().any()
        elif name in "ab":
            same(y[:, :, heads], y0[:, :, heads], (name, "other heads"))
            assert not h[1, 0].isfinite().any()
        else:
            assert not h[1].isfinite().any()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("p_done", [0.0, 0.05])
def test_values_at_many_steps(gpu, p_done, dt):
    """Columns that end at steps of their own, between episodes that clear them: each is finite up to there and again behind."""
    T, B, H, K, V = 200, 1, 2, 32, 48
    clean = {n: t.clone() for n, t in inputs(T, B, 2, H, K, V, dt).items()}
    done, h0 = flags(3, p_done, T, B), cu(5, B, H, K, V)
    y0, _ = scan(clean, h0, done)
    p = {n: t.clone() for n, t in clean.items()}
    at = torch.arange(V, device="cuda") * 37 % T
    p["v"][at, 0, 0, torch.arange(V, device="cuda")] = float("nan")
    p["v"][at, 0, 1, torch.arange(V, device="cuda")] = float("-inf")
    y, _ = scan(p, h0, done)
    ends = torch.cat([torch.zeros(1, device="cuda"), done[:-1, 0]]).cumsum(0)  # episodes
    hit = (torch.arange(T, device="cuda")[:, None] >= at) & (ends[:, None] == ends[at])  # [T, V]
    for h in range(H):
        x = y[:, 0, h]
        assert not x[hit].isfinite().any()
        assert x[~hit].isfinite().all()
        same(x[~hit], y0[:, 0, h][~hit], h)


@pytest.mark.parametrize("dt", [F32, BF])
def test_a_query_is_its_own_step_s(gpu, dt):
    T, B, H, K, V = 70, 2, 2, 32, 24
    clean = {n: t.clone() for n, t in inputs(T, B, 1, H, K, V, dt).items()}
    h0 = cu(5, B, H, K, V)
    y0, hc = scan(clean, h0)
    clean["q"][21, 1] = float("nan")
    clean["q"][40, :, :, 3] = float("inf")
    y, h = scan(clean, h0)
    assert torch.equal(h, hc)
    rest = torch.ones(T, B, dtype=torch.bool, device="cuda")
    rest[21, 1], rest[40] = False, False
    assert torch.equal(y[rest], y0[rest]) and not y[~rest].isfinite().any()


@pytest.mark.parametrize("dt", [F32, BF])
def test_a_decay_that_grows_past_fp32_stays_in_its_episode(gpu, dt):
    T, B, H, K, V = 90, 2, 2, 32, 24
    clean = {n: t.clone() for n, t in inputs(T, B, 1, H, K, V, dt).items()}
    clean["A"] = torch.full((H,), 0.01, device="cuda")  # 0.1 % a step otherwise
    done, h0 = torch.zeros(T, B, device="cuda"), cu(5, B, H, K, V)
    done[[11, 40, 47]] = 1
    y0, hc = scan(clean, h0, done)
    p = {n: t.clone() for n, t in clean.items()}
    p["a"][4:9] = 20000  # e^200 a step
    p["a"][43:46] = 20000
    y, h = scan(p, h0, done)
    same(h, hc, "h")
    for s in (slice(0, 4), slice(12, 41), slice(48, T)):
        if s.start:
            same(y[s], y0[s], s)
    assert not y[8].isfinite().any() and not y[46].isfinite().any()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("name,value", [("q", 3e19), ("k", 3e19), ("v", 3e38), ("dy", 3e38), ("b", float("nan")), ("a", float("nan")), ("a", 20000.0)])
@pytest.mark.parametrize("T,K,V", [(70, 16, 24), (410, 16, 24), (70, 64, 64), (70, 100, 128)])
def test_what_overflows_stays_in_its_episode(gpu, T, K, V, name, value, dt):
    """Finite values whose sums or squares pass fp32's range, gates that are none, and a decay that grows: y and the gradients of the
    episodes of steps 10..44 and from 50 on are those without them."""
    B, H = 2, 2
    clean = dict(inputs(T, B, 1, H, K, V, dt), dy=cu(50, T, B, H, V, dtype=dt))
    clean["A"] = torch.full((H,), 0.01 if value == 20000.0 else -0.4, device="cuda")
    done, h0 = torch.zeros(T, B, device="cuda"), cu(5, B, H, K, V)
    done[[9, 44, 49]] = 1

    def run(p):
        args = [p[n] for n in "qkvabA"]
        y, saved = D.delta_scan(*args, dt_bias=p["dt_bias"], done=done, h0=h0, save=True)
        return dict(D.delta_scan_grad(*args, saved, p["dy"], dt_bias=p["dt_bias"], done=done), y=y)

    want = run(clean)
    p = {n: t.clone() for n, t in clean.items()}
    p[name][2:7], p[name][46] = value, value
    got = run(p)
    for s in (slice(10, 45), slice(50, T)):
        for n in ("y", "dq", "dk", "dv", "da", "db"):
            bar = 2 * BAR[dt] * (10 if n == "da" else 1) + (2 * R.BF16 if dt == BF else 0)
            assert got[n][s].isfinite().all() and rel(got[n][s], want[n][s]) <= bar, (n, s)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("name", ["q", "k"])
def test_rows_too_long_for_fp32_are_none_in_scan_and_step(gpu, name, dt):
    """Not rows of zero: their unit rows could not be told."""
    B, H, K, V = 3, 2, 16, 24
    p = {n: t.clone() for n, t in inputs(1, B, 1, H, K, V, dt).items()}
    p[name][0, 1] = 3e19
    h0 = cu(5, B, H, K, V)
    y, h = scan(p, h0)
    step = h0.clone()
    ys = D.delta_step(*[p[n][0] for n in "qkvab"], p["A"], step, dt_bias=p["dt_bias"])
    for out, state in ((y[0], h), (ys, step)):
        assert not out[1].isfinite().any() and out[[0, 2]].isfinite().all()
        assert state[[0, 2]].isfinite().all() and state[1].isfinite().any() == (name == "q")
