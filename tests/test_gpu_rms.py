"""RMS normalisation with its residual sum and gate, and the gradient, against the definition in 64 bits.

Bars: sums of at most 32 values a lane and 8 folds keep a row's statistics within 40 roundings of 2^-24 (2.4e-6), the gate's
exponential and quotient add four: 3e-6; the columns' sums add rows in runs of up to a few hundred, 1e-5. bf16 results
add their one rounding. A column's sum may cancel: each addition rounds a partial sum, and partial sums of terms of either sign are
of the size of sqrt(sum of squares), so errors are measured against that where it is the larger. dx is the difference of terms that may cancel, so its error is measured against them."""
import numpy as np
import pytest
import torch

import delta_layer_ref as R
from policy_layer_ref import leaf, rel
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
ROW, COL = 3e-6, 1e-5
F32, BF = torch.float32, torch.bfloat16
FORMS = {"plain": (), "add": ("add",), "scale": ("add", "scale"), "gate": ("gate",), "all": ("add", "scale", "gate")}


def cu(seed, *shape, scale=1.0, dtype=F32):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", dtype)


def laid(x, off):
    if not off:
        return x
    M, C = x.shape
    buf = torch.full((M, C + 5), 7.0, device="cuda", dtype=x.dtype)
    buf[:, off:C + off] = x
    return buf[:, off:C + off]


def case(M, C, dt, form, groups=1, off=0, w=True):
    k = dict(x=laid(cu(1, M, C, dtype=dt), off), w=1 + cu(2, C // groups, scale=0.2) if w else None)
    if "add" in FORMS[form]:
        k["add"] = laid(cu(3, M, C, dtype=dt), off)
    if "scale" in FORMS[form]:
        k["scale"] = 0.5 + cu(4, C, scale=0.3)
    if "gate" in FORMS[form]:
        k["gate"] = laid(cu(5, M, C, scale=2.0, dtype=dt), off)
    return k


def check(k, groups=1, with_dres=True, eps=1e-6):
    x, w = k["x"], k["w"]
    M, C = x.shape
    kw = {n: k.get(n) for n in ("add", "scale", "gate")}
    dout, dres = cu(6, M, C, dtype=x.dtype), cu(7, M, C, dtype=x.dtype) if with_dres else None
    out, res, rstd = D.rms_norm(x, w, groups=groups, eps=eps, **kw)
    g = D.rms_norm_grad(x, w, rstd, dout, dres=dres, groups=groups, eps=eps, **kw)
    one = BF if x.dtype == BF else None
    bar = R.BF16 if one else 0.0
    ref = {n: leaf(t) for n, t in k.items() if t is not None}
    o, r = R.rms(ref["x"], ref.get("w"), ref.get("add"), ref.get("scale"), ref.get("gate"), groups, eps)
    obj = (o * dout.double().cpu()).sum() + (0 if dres is None else (r * dres.double().cpu()).sum())
    grads = dict(zip(ref, torch.autograd.grad(obj, list(ref.values()))))
    assert rel(out, o) <= ROW + bar
    assert (res is None) == ("add" not in k) and (res is None or rel(res, r) <= ROW + bar)
    assert set(g) == {"d" + n for n in ref}
    with torch.no_grad():  # the terms of dx
        z = ref.get("gate")
        gn = dout.double().cpu() * (1 if z is None else z / (1 + torch.exp(-z)))
        gn = (gn.view(M, groups, -1) * (1 if w is None else ref["w"]))
        n, _ = R.rms(r, groups=groups, eps=eps)
        n, rs = n.view(M, groups, -1), rstd.double().cpu()[..., None]
        dw_size = 0.0 if w is None else float((gn / ref["w"] * n).norm())
        terms = rs * (gn.abs() + (n * (gn * n).mean(-1, keepdim=True)).abs())
        size = float((terms.reshape(M, C) + (0 if dres is None else dres.double().cpu().abs())).norm())
    for m in ("x", "add"):
        if m in ref:
            s = size if m == "x" or "scale" not in ref else size * float(ref["scale"].abs().max())
            assert float((g["d" + m].double().cpu() - grads[m]).norm()) <= 3 * ROW * s + bar * float(grads[m].norm()), m
    if "gate" in ref:
        assert rel(g["dgate"], grads["gate"]) <= 3 * ROW + bar
    if w is not None:
        assert float((g["dw"].double().cpu() - grads["w"]).norm()) <= COL * max(float(grads["w"].norm()), dw_size)
    if "scale" in ref:
        assert float((g["dscale"].double().cpu() - grads["scale"]).norm()) <= COL * max(float(grads["scale"].norm()), size * float(ref["add"].norm()) / (M * C) ** 0.5)
    return out, res, g


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 9, 31, 64, 96, 128, 203, 256, 512, 640, 1000, 1024, 2040, 2048, 2049, 4096])
@pytest.mark.parametrize("form", list(FORMS))
def test_widths(gpu, form, C, dt):
    check(case(5, C, dt, form))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("M,C,form", [(1, 64, "all"), (1, 4100, "all"), (130, 203, "scale"), (9000, 128, "all"), (4097, 203, "gate"), (1500, 1024, "scale"), (70, 5001, "all"),
                                      (40, 4200, "gate"), (300, 2048, "all")])
def test_rows(gpu, M, C, form, dt):
    check(case(M, C, dt, form))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("groups,C", [(2, 16), (3, 21), (4, 256), (8, 512), (5, 205), (16, 16), (2, 8200), (3, 3 * 520)])
@pytest.mark.parametrize("form", ["plain", "add", "gate"])
def test_groups(gpu, groups, C, form, dt):
    check(case(67, C, dt, form, groups), groups)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("off", [1, 4])
@pytest.mark.parametrize("C", [96, 203, 600])
def test_strided_rows(gpu, C, off, dt):
    a = check(case(67, C, dt, "all", off=off))
    b = check(case(67, C, dt, "all"))
    assert rel(a[0], b[0]) <= COL + (R.BF16 if dt == BF else 0)
    out, res = (torch.full((67, C + 5), 7.0, device="cuda", dtype=dt) for _ in range(2))
    k = case(67, C, dt, "all", off=off)
    D.rms_norm(k["x"], k["w"], add=k["add"], scale=k["scale"], gate=k["gate"], out=out[:, 2:C + 2], res=res[:, 2:C + 2])
    for t in (out, res):
        assert (t[:, :2] == 7).all() and (t[:, C + 2:] == 7).all() and not (t[:, 2:C + 2] == 7).all()


@pytest.mark.parametrize("dt", [F32, BF])
def test_without_weights_or_dres(gpu, dt):
    check(case(33, 96, dt, "all", w=False), with_dres=False)
    check(case(33, 96, dt, "plain", w=False))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [203, 512, 4100])
def test_in_place(gpu, C, dt):
    """out over the gate, res over x; dx over dout, dadd over add, dgate over the gate."""
    k = case(40, C, dt, "all")
    kw = {n: k[n] for n in ("add", "scale", "gate")}
    out, res, rstd = D.rms_norm(k["x"], k["w"], **kw)
    dout, dres = cu(6, 40, C, dtype=dt), cu(7, 40, C, dtype=dt)
    g = D.rms_norm_grad(k["x"], k["w"], rstd, dout, dres=dres, **kw)
    c = {n: t.clone() for n, t in k.items()}
    o2, r2, _ = D.rms_norm(c["x"], c["w"], add=c["add"], scale=c["scale"], gate=c["gate"], out=c["gate"], res=c["x"])
    assert torch.equal(out, o2) and torch.equal(res, r2)
    c = {n: t.clone() for n, t in k.items()}
    d = dout.clone()
    g2 = D.rms_norm_grad(c["x"], c["w"], rstd, d, dres=dres, add=c["add"], scale=c["scale"], gate=c["gate"], dx=d, dadd=c["add"], dgate=c["gate"])
    for n in g:
        assert torch.equal(g[n], g2[n]), n


def test_a_row_does_not_see_another(gpu):
    """Rows of zeros, infinities and NaN next to others."""
    k = case(8, 256, BF, "all")
    ref = D.rms_norm(k["x"], k["w"], add=k["add"], scale=k["scale"], gate=k["gate"])[0]
    k["x"][2], k["x"][5] = float("nan"), float("inf")
    k["x"][6] = 0
    k["add"][6] = 0
    out, _, rstd = D.rms_norm(k["x"], k["w"], add=k["add"], scale=k["scale"], gate=k["gate"])
    for i in (0, 1, 3, 4, 7):
        assert torch.equal(out[i], ref[i])
    assert not out[6].any() and rel(rstd[6], torch.tensor([1e3])) < 1e-6


def test_no_rows(gpu):
    x, w = torch.empty(0, 24, device="cuda"), torch.ones(24, device="cuda")
    out, res, rstd = D.rms_norm(x, w, add=x, scale=w)
    g = D.rms_norm_grad(x, w, rstd, x, add=x, scale=w, dw=torch.ones(24, device="cuda"), dscale=torch.ones(24, device="cuda"))
    assert out.shape == (0, 24) and not g["dw"].any() and not g["dscale"].any()


def test_gradient_against_differences(gpu):
    """Central differences of the fp32 forward with a step of 2^-7: its square, 6e-5, and 3e-6 over the step: 1 %."""
    k = case(9, 40, F32, "all")
    dout, dres = cu(6, 9, 40), cu(7, 9, 40)

    def f(c):
        out, res, _ = D.rms_norm(c["x"], c["w"], add=c["add"], scale=c["scale"], gate=c["gate"])
        return float((out.double() * dout + res.double() * dres).sum())

    rstd = D.rms_norm(k["x"], k["w"], add=k["add"], scale=k["scale"], gate=k["gate"])[2]
    g = D.rms_norm_grad(k["x"], k["w"], rstd, dout, dres=dres, add=k["add"], scale=k["scale"], gate=k["gate"])
    for n in k:
        d = g["d" + n] / g["d" + n].norm()
        e = 2.0 ** -7
        got = (f(dict(k, **{n: k[n] + e * d})) - f(dict(k, **{n: k[n] - e * d}))) / (2 * e)
        want = float((g["d" + n].double() * d.double()).sum())
        assert abs(got - want) <= 0.01 * abs(want), n


def test_captured(gpu):
    k = case(3000, 203, BF, "all")
    kw = {n: k[n] for n in ("add", "scale", "gate")}
    dout = cu(6, 3000, 203, dtype=BF)

    def work():
        out, res, rstd = D.rms_norm(k["x"], k["w"], **kw)
        return dict(D.rms_norm_grad(k["x"], k["w"], rstd, dout, dres=res, **kw), out=out)

    eager = {n: t.clone() for n, t in work().items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = work()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for n in eager:
            assert torch.equal(out[n], eager[n]), n
        work()
        torch.cuda.synchronize()
