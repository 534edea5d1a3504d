"""The gated delta rule on bf16 inputs keeps fp32's precision up to the one rounding of what leaves in bf16.

Inputs are exact, so an fp32 result differs from the 64-bit definition by the roundings of fp32 alone. A sum of n products of either
sign rounds partial sums of up to its own size: sqrt(n / 2) roundings of 0.4 * 2^-24 in the mean square, 2e-7 for n = 128. A state passes four
such sums, and factors (a decay, two norms, a write strength) of some 2^-23 each, and every step contracts it, so errors of earlier
chunks fade: 6e-7, and 1e-6 is the bar. A value held in two bf16 is off by 2^-17 / sqrt(3), twice to four times that bar. dA and
ddt_bias add one term per step, itself a sum of four such parts; they are measured against the root of the terms' squares: 2e-6.

A bf16 result that is off by e before its rounding rounds to the other side with probability e / ulp and then differs by an ulp, at
most 2^-7 of it, from the rounded 64-bit value: the squares add up to e |x| 2^-7, and their root, relative, to sqrt(e 2^-7). With
e = 1e-6 that is 9e-5. So this is asked of tensors of 40,000 elements and more, in which one of them does not count."""
import pytest
import torch

import delta_layer_ref as R
from policy_layer_ref import leaf, rel
from pufferlean_amd import device as D
from test_gpu_delta import cu, flags, host, inputs

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
STATE, TERMS = 1e-6, 2e-6
FLIPS = (1e-6 / 128) ** 0.5

# short sequences of each padded size, with tiles left out, two value heads to a key head; long ones in segments of time
CASES = [(64, 24, 4, 4, 32, 32), (70, 24, 1, 2, 24, 20), (96, 16, 2, 2, 64, 64), (64, 16, 1, 2, 40, 64), (64, 12, 1, 2, 128, 128), (70, 12, 2, 2, 100, 72),
         (1100, 1, 1, 2, 32, 32), (1024, 1, 1, 2, 64, 64), (700, 1, 1, 1, 128, 128)]


def forward(p, done, first, h0):
    h = torch.empty_like(h0)
    y, saved = D.delta_scan(*[p[n] for n in "qkvabA"], dt_bias=p["dt_bias"], done=done, first=first, h0=h0, h_out=h, save=True)
    return y, h, saved


def case(T, B, Hk, H, K, V):
    p = inputs(T, B, Hk, H, K, V, BF)
    if T > 256:
        p["A"] *= 0.05  # states that outlive a segment
    return p, flags(3, 0.01, T, B), flags(4, 0.3, B), cu(5, B, H, K, V, scale=0.3)


def rounded(x, ref, bar, what):
    """The bf16 tensor x against the 64-bit values rounded once."""
    assert x.dtype == BF
    got = rel(x, ref.to(BF).double())
    assert got <= bar, (what, got)


@pytest.mark.parametrize("T,B,Hk,H,K,V", CASES)
def test_outputs(gpu, T, B, Hk, H, K, V):
    p, done, first, h0 = case(T, B, Hk, H, K, V)
    y, h, _ = forward(p, done, first, h0)
    yr, hr = R.delta({n: host(t) for n, t in p.items()}, None, host(done), host(first), host(h0))
    assert rel(h, hr) <= STATE, rel(h, hr)
    rounded(y, yr, FLIPS, "y")


@pytest.mark.parametrize("T,B,Hk,H,K,V", CASES)
def test_gradients(gpu, T, B, Hk, H, K, V):
    p, done, first, h0 = case(T, B, Hk, H, K, V)
    dy, dh = cu(50, T, B, H, V, dtype=BF), cu(51, B, H, K, V)
    ref = {n: leaf(t) for n, t in p.items()}
    wide = {n: host(p[n]).expand(T, B, H).clone().requires_grad_(True) for n in ("A", "dt_bias")}  # a step's own
    h0r = leaf(h0)
    yr, hr = R.delta({**ref, **wide}, None, host(done), host(first), h0r)
    names = list("qkv")
    got = torch.autograd.grad((yr * host(dy)).sum() + (hr * host(dh)).sum(), [ref[n] for n in names] + [wide["A"], wide["dt_bias"], h0r])
    grads = dict(zip(names + ["A", "dt_bias", "h0"], got))
    _, _, saved = forward(p, done, first, h0)
    dh0 = torch.empty_like(h0)
    g = D.delta_scan_grad(*[p[n] for n in "qkvabA"], saved, dy, dt_bias=p["dt_bias"], done=done, first=first, dh=dh, dh0=dh0)
    found = {"h0": rel(dh0, grads["h0"])}
    for n in ("A", "dt_bias"):
        found[n] = float((host(g["d" + n]) - grads[n].sum((0, 1))).norm() / grads[n].norm())
    for n in names:
        found[n] = rel(g["d" + n], grads[n].to(BF).double())
    bars = dict(h0=STATE, A=TERMS, dt_bias=TERMS, v=FLIPS, q=FLIPS, k=FLIPS * 2 ** 0.5)  # dk: the sum of two such parts
    over = {n: x for n, x in found.items() if x > bars[n]}
    assert not over, (over, found)
