"""Layer normalisation and its gradient against the definition in 64 bits.

Bars: fp32 sums of at most 32 values per lane and 6 folds keep a row's statistics within 38 rounding errors of 2^-24
(2.3e-6); the columns' sums add rows in runs of up to a few hundred, 1e-5. bf16 results add their one rounding. dx is the
difference of three terms that may cancel (two columns: to the last digit), so its error is measured against them."""
import numpy as np
import pytest
import torch

import policy_layer_ref as R
from pufferlean_amd import _lib as L
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
ROW, COL = 3e-6, 1e-5


def cu(seed, *shape, scale=1.0, dtype=torch.float32):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", dtype)


def laid(x, layout):
    if layout == "packed":
        return x.clone()
    M, C = x.shape
    buf = torch.full((M, C + 3), 7.0, device="cuda", dtype=x.dtype)
    buf[:, 1:C + 1] = x
    return buf[:, 1:C + 1]


def case(M, C, dt, layout="packed", affine=True, offset=0.0):
    x = laid((cu(1, M, C) + offset).to(dt), layout)
    dy = laid(cu(2, M, C, dtype=dt), layout)
    w = 1 + cu(3, C, scale=0.2) if affine else None
    b = cu(4, C, scale=0.2) if affine else None
    return x, dy, w, b


def check(x, dy, w, b, row=ROW, col=COL):
    out = R.BF16 if x.dtype == torch.bfloat16 else 0.0
    y, mean, rstd = D.layer_norm(x, w, b)
    dx, dw, db = D.layer_norm_grad(x, w, mean, rstd, dy)
    xr, wr, br = R.leaf(x), R.leaf(w), R.leaf(b)
    one = torch.ones(x.shape[1], dtype=torch.float64, requires_grad=True)
    zero = torch.zeros(x.shape[1], dtype=torch.float64, requires_grad=True)
    wr, br = one if wr is None else wr, zero if br is None else br
    yr = R.layer_norm(xr, wr, br)
    gx, gw, gb = torch.autograd.grad(yr, (xr, wr, br), dy.double().cpu())
    assert R.rel(y, yr) <= row + out
    with torch.no_grad():
        n, g, r = R.layer_norm(xr, None, None), dy.double().cpu() * wr, rstd.double().cpu()[:, None]
        terms = (r * (g.abs() + g.mean(1, keepdim=True).abs() + (n * (g * n).mean(1, keepdim=True)).abs())).norm()
    assert float((dx.double().cpu() - gx).norm()) <= 3 * row * float(terms) + out * float(gx.norm())
    if x.shape[1] > 1:  # of a row of one column n is zero, and so is dw
        assert R.rel(dw, gw) <= col
    assert R.rel(db, gb) <= col
    return y, dx, dw, db


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 9, 31, 64, 96, 128, 203, 255, 256, 512, 640, 1000, 1024, 2040, 2048])
@pytest.mark.parametrize("M", [1, 3, 33, 130])
def test_widths(gpu, M, C, dt):
    check(*case(M, C, dt))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C", [(5, 2049), (70, 4096), (3, 5001)])
def test_wide_rows(gpu, M, C, dt):
    # three passes over the row, 256 threads adding up to 20 values each: 20 + 8 folds
    check(*case(M, C, dt))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C", [(9000, 128), (4097, 203), (20011, 64), (1500, 1024)])
def test_many_rows(gpu, M, C, dt):
    check(*case(M, C, dt))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("affine", [True, False])
def test_strided_rows_and_no_affine(gpu, dt, affine):
    x, dy, w, b = case(300, 96, dt, "strided", affine)
    got = check(x, dy, w, b)
    again = check(x.clone(), dy.clone(), w, b)
    for a, c in zip(got, again):  # the layout changes no value of a row; column sums keep their order
        assert R.rel(a, c) <= COL
    out = torch.full((300, 99), 7.0, device="cuda", dtype=dt)
    D.layer_norm(x, w, b, out=out[:, 1:97])
    assert torch.all(out[:, 0] == 7) and torch.all(out[:, 97:] == 7)


def test_more_wide_rows_than_a_launch_has_blocks(gpu):
    """2^24 rows of a block of 256 threads each are more than one launch takes. Copies of 64 rows, and eight of their own at the end;
    the sums over the rows are too long for a bar of theirs and left out."""
    M, C = 2 ** 24 + 8, 2049
    if torch.cuda.mem_get_info()[0] < 150e9:
        pytest.skip("needs 140 GB")
    x, dy, w, b = case(72, C, torch.bfloat16)
    y, mean, rstd = D.layer_norm(x, w, b)
    dx, _, _ = D.layer_norm_grad(x, w, mean, rstd, dy)
    far, g = (torch.empty(M, C, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for t, v in ((far, x), (g, dy)):
        t[:2 ** 24].view(2 ** 18, 64, C).copy_(v[:64])
        t[2 ** 24:] = v[64:]
    check = lambda t, v: [(t[:2 ** 24].view(2 ** 18, 64, C)[i::2 ** 14] == v[:64]).all().item() for i in (0, 1, 2 ** 14 - 1)] + [torch.equal(t[2 ** 24:], v[64:])]
    stats = [torch.empty(M, device="cuda") for _ in range(2)]
    D.layer_norm(far, w, b, out=far, mean=stats[0], rstd=stats[1])
    assert all(check(far, y))
    assert torch.equal(stats[0][-8:], mean[64:]) and torch.equal(stats[1][-8:], rstd[64:])
    far[:2 ** 24].view(2 ** 18, 64, C).copy_(x[:64])
    far[2 ** 24:] = x[64:]
    L.call("ph_layer_norm_grad", L.PH_BF16, far.data_ptr(), C, g.data_ptr(), C, M, C, w.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(),
           g.data_ptr(), C, None, None, D._stream())
    assert all(check(g, dx))
    del far, g
    torch.cuda.empty_cache()


def test_large_offset_keeps_its_digits(gpu):
    # the mean is 1000 times the deviation: x itself holds 2^-24 * 1000 of a deviation, and so does the mean
    x, dy, w, b = case(64, 512, torch.float32, offset=1000.0)
    check(x, dy, w, b, row=3e-4, col=3e-4)


def test_constant_and_non_finite_rows(gpu):
    x, dy, w, b = case(8, 64, torch.float32)
    x[1] = 2.5
    x[3, 5] = float("nan")
    x[5, 7] = float("inf")
    y, mean, rstd = D.layer_norm(x, w, b)
    assert torch.equal(y[1], b) and torch.isnan(y[3]).all() and torch.isnan(y[5]).all()
    good = [0, 1, 2, 4, 6, 7]
    assert torch.isfinite(y[good]).all()
    dx, _, _ = D.layer_norm_grad(x, w, mean, rstd, dy)
    assert torch.isfinite(dx[good]).all() and torch.isnan(dx[3]).all()


def test_no_rows(gpu):
    x = torch.empty(0, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    y, mean, rstd = D.layer_norm(x, w)
    dx, dw, db = D.layer_norm_grad(x, w, mean, rstd, x, dw=torch.ones(16, device="cuda"))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and not dw.any() and not db.any()


def test_in_place(gpu):
    x, dy, w, b = case(100, 96, torch.bfloat16)
    y, mean, rstd = D.layer_norm(x, w, b)
    dx, _, _ = D.layer_norm_grad(x, w, mean, rstd, dy)
    g = dy.clone()
    D.layer_norm_grad(x, w, mean, rstd, g, dx=g)
    assert torch.equal(g, dx)
    D.layer_norm(x, w, b, out=x)
    assert torch.equal(x, y)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("into", ["dy", "x"])
@pytest.mark.parametrize("M,C", [(130, 96), (130, 203), (600, 2048), (3, 2049), (130, 2049), (600, 4096)])
def test_gradient_into_its_inputs(gpu, M, C, into, dt):
    """dx may be dy or x: nothing is read from either after it has been written, the columns' sums neither. Rows of every form, and
    one block's as well as several blocks' sums."""
    x, dy, w, b = case(M, C, dt)
    _, mean, rstd = D.layer_norm(x, w, b)
    ref = D.layer_norm_grad(x, w, mean, rstd, dy)
    got = D.layer_norm_grad(x, w, mean, rstd, dy, dx=dy if into == "dy" else x)
    for k, a, g in zip(("dx", "dw", "db"), ref, got):
        assert torch.equal(a, g), k


def test_gradient_against_differences(gpu):
    x, dy, w, b = case(40, 96, torch.float32)
    y, mean, rstd = D.layer_norm(x, w, b)
    dx, dw, db = D.layer_norm_grad(x, w, mean, rstd, dy)
    f = lambda x, w, b: float((D.layer_norm(x, w, b)[0].double() * dy.double()).sum())
    vx, vw, vb = cu(11, 40, 96), cu(12, 96), cu(13, 96)
    e = 2.0 ** -7  # difference error e^2, rounding 2^-24 / e of |y| |dy|
    for args, want in (((vx, 0, 0), (dx * vx).sum()), ((0, vw, 0), (dw * vw).sum()), ((0, 0, vb), (db * vb).sum())):
        d = (f(x + e * args[0], w + e * args[1], b + e * args[2]) - f(x - e * args[0], w - e * args[1], b - e * args[2])) / (2 * e)
        scale = float(vx.norm() * dx.norm()) * 0.05 + abs(float(want))
        assert abs(d - float(want)) <= 2e-3 * scale


def test_same_twice_and_on_another_stream(gpu):
    x, dy, w, b = case(5000, 203, torch.float32)
    a = check(x, dy, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, mean, rstd = D.layer_norm(x, w, b)
        c = (y, *D.layer_norm_grad(x, w, mean, rstd, dy))
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_graph_replays(gpu):
    x, dy, w, b = case(3000, 128, torch.bfloat16)
    ref = check(x, dy, w, b)
    y, mean, rstd = torch.empty_like(x), torch.empty(3000, device="cuda"), torch.empty(3000, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty(128, device="cuda"), torch.empty(128, device="cuda")
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        D.layer_norm(x, w, b, out=y, mean=mean, rstd=rstd)
        D.layer_norm_grad(x, w, mean, rstd, dy, dx=dx, dw=dw, db=db)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        for t in (y, dx, dw, db):
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ref, (y, dx, dw, db)))
        (torch.ones(1000, device="cuda") * 2).sum().item()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C", [(3, 96), (600, 96), (130, 203), (130, 2049)])
def test_results_left_out(gpu, M, C, dt):
    """The statistics, dw and db may each be left out; the others stay the same."""
    x, dy, w, b = case(M, C, dt)
    ref = D.layer_norm(x, w, b)
    code = L.PH_F32 if dt is torch.float32 else L.PH_BF16
    y = torch.full_like(x, 7.0)
    L.call("ph_layer_norm", code, x.data_ptr(), C, M, C, w.data_ptr(), b.data_ptr(), 1e-5, y.data_ptr(), C, None, None, D._stream())
    assert torch.equal(y, ref[0])
    grads = D.layer_norm_grad(x, w, ref[1], ref[2], dy)
    for keep in range(4):
        out = [torch.full_like(dy, 7.0)] + [torch.full_like(w, 7.0) if keep >> i & 1 else None for i in range(2)]
        p = [None if t is None else t.data_ptr() for t in out]
        L.call("ph_layer_norm_grad", code, x.data_ptr(), C, dy.data_ptr(), C, M, C, w.data_ptr(), ref[1].data_ptr(), ref[2].data_ptr(),
               p[0], C, p[1], p[2], D._stream())
        for a, g in zip(out, grads):
            assert a is None or torch.equal(a, g), keep


def test_refusals(gpu):
    x = torch.ones(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    with pytest.raises(TypeError):
        D.layer_norm(x.double(), w)
    with pytest.raises(ValueError):
        D.layer_norm(x, w[:4])
    with pytest.raises(ValueError):
        D.layer_norm(x, w.bfloat16())
    with pytest.raises(ValueError):
        D.layer_norm(x.t(), None)  # rows are not contiguous
    with pytest.raises(ValueError):
        D.layer_norm(x, w, out=torch.ones(4, 8, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        D.layer_norm(x.cpu(), None)
    lib = L.lib()
    p = x.data_ptr()
    assert lib.ph_layer_norm(L.PH_F64, p, 8, 4, 8, None, None, 1e-5, p, 8, None, None, None) == L.PH_ERR_ARG
    assert lib.ph_layer_norm(L.PH_F32, p, 7, 4, 8, None, None, 1e-5, p, 8, None, None, None) == L.PH_ERR_ARG
    assert lib.ph_layer_norm(L.PH_F32, p, 8, 4, 0, None, None, 1e-5, p, 8, None, None, None) == L.PH_ERR_ARG
    assert lib.ph_layer_norm(L.PH_F32, None, 8, 4, 8, None, None, 1e-5, p, 8, None, None, None) == L.PH_ERR_ARG
    assert lib.ph_layer_norm(L.PH_F32, p, 8, 4, 8, None, None, -1.0, p, 8, None, None, None) == L.PH_ERR_ARG
    assert lib.ph_layer_norm_grad(L.PH_F32, p, 8, p, 8, 4, 8, None, None, None, p, 8, None, None, None) == L.PH_ERR_ARG
    assert lib.ph_layer_norm_grad(L.PH_F32, p, 8, p, 8, 4, 8, None, p, p, p, 4, None, None, None) == L.PH_ERR_ARG
