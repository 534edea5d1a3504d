"""The gated feed-forward block and its gradient against the definition in 64 bits.

Bars, relative 2-norm. fp32: sums of up to K products round K^0.5 times 2^-24 of their size, under 1e-5 for the sizes here.
bf16: the operands are exact and the sums fp32, so what is lost are the roundings of stored values (h, the projections, the
projections' gradients, the result), at most 2^-8 each; up to three of them meet in a result. Each rounds one term of a sum
by itself, so errors are measured against the root of the sum of the terms' squares, which a sum that cancels falls below."""
import numpy as np
import pytest
import torch

import policy_layer_ref as R
from pufferlean_amd import _lib as L
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
BARS = {torch.float32: 1e-5, torch.bfloat16: 3 * R.BF16}


def cu(seed, *shape, scale=1.0, dtype=torch.float32):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", dtype)


def case(M, Dm, F, dt):
    return (cu(1, M, Dm, dtype=dt), cu(2, 2 * F, Dm, scale=Dm ** -0.5, dtype=dt), cu(3, Dm, F, scale=F ** -0.5, dtype=dt),
            cu(4, M, Dm, dtype=dt))


def check(x, wi, wo, dy, act="silu", dw_dtype=None):
    bar = BARS[x.dtype]
    y, saved = D.gated_ffn(x, wi, wo, act=act, save=True)
    assert R.rel(D.gated_ffn(x, wi, wo, act=act), y) <= bar
    dx, dwi, dwo = D.gated_ffn_grad(x, wi, wo, saved, dy, act=act, dw_dtype=dw_dtype)
    xr, ir, outr = R.leaf(x), R.leaf(wi), R.leaf(wo)
    yr = R.ffn(xr, ir, outr, act)
    gx, gi, go = torch.autograd.grad(yr, (xr, ir, outr), dy.double().cpu())
    with torch.no_grad():
        a = (xr @ ir[0::2].T).requires_grad_(True)
        v = (xr @ ir[1::2].T).requires_grad_(True)
        with torch.enable_grad():
            h = R.glu(a, v, act)
        da, dv = torch.autograd.grad(h, (a, v), dy.double().cpu() @ outr)
        dab2 = torch.stack([da, dv], -1).reshape(len(x), -1) ** 2
    for got, ref, terms in ((y, yr, (h ** 2) @ (outr ** 2).T), (dx, gx, dab2 @ ir ** 2), (dwi, gi, dab2.T @ xr ** 2),
                            (dwo, go, (dy.double().cpu() ** 2).T @ h ** 2)):
        size = max(float(terms.detach().sum().sqrt()), float(ref.norm()))
        assert float((got.double().cpu() - ref).norm()) <= bar * size
    return y, dx, dwi, dwo


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,Dm,F", [(1, 64, 96), (2, 8, 8), (3, 7, 5), (8, 512, 344), (16, 128, 128), (17, 96, 203), (33, 203, 64),
                                    (64, 64, 1), (65, 1, 33), (130, 264, 520), (300, 128, 688)])
def test_sizes(gpu, M, Dm, F, act, dt):
    check(*case(M, Dm, F, dt), act)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,Dm,F", [(4096, 128, 344), (3001, 200, 333), (2048, 512, 1024)])
def test_many_rows(gpu, M, Dm, F, dt):
    check(*case(M, Dm, F, dt))


# (M, D, F, dtype) whose products with the units in the epilogue take the larger tiles, with ragged rows, columns and sums, and the
# tiles of the units and of their gradient
LARGE = [(16500, 40, 1000, torch.bfloat16, "256", "256"), (16500, 40, 520, torch.bfloat16, "256x128", "128"),
         (33000, 24, 536, torch.bfloat16, "256x128", "256x128"), (1500, 72, 1400, torch.bfloat16, "128", "128"),
         (5000, 40, 1668, torch.float32, "128", "128"), (2000, 24, 4100, torch.float32, "128", "128")]


@pytest.mark.parametrize("M,Dm,F,dt,units,grad", LARGE)
def test_large_tiles(gpu, M, Dm, F, dt, units, grad):
    check(*case(M, Dm, F, dt))


@pytest.mark.parametrize("M,F", [(16500, 1000), (16500, 520), (1500, 1400)])
def test_kept_pairs_of_large_tiles(gpu, M, F):
    """As test_kept_pairs; of tens of millions of values |v| stays under 6."""
    x, wi, wo, _ = case(M, 64, F, torch.bfloat16)
    _, (pf, h) = D.gated_ffn(x, wi, wo, save=True)
    row = pf.cpu().contiguous().view(torch.uint8).numpy().reshape(M, 6 * F)
    b = np.zeros((M, 2 * F, 4), np.uint8)
    b[..., 2:] = row[:, :4 * F].reshape(M, 2 * F, 2)
    b[..., 1] = row[:, 4 * F:]
    got = torch.from_numpy(b.view(np.float32)[..., 0]).double()
    a, v = (x.double().cpu() @ wi.double().cpu()[k::2].T for k in (0, 1))
    s = 1 / (1 + torch.exp(-a))
    ref = torch.stack([v * s * (1 + a * (1 - s)), a * s], -1).reshape(M, -1)
    assert ((got - ref).abs() <= 2.0 ** -15 * ref.abs() + 1.5e-4).all()
    assert R.rel(h, a * s * v) <= R.BF16 + 1e-5


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,Dm,F", [(1, 64, 96), (8, 512, 344), (16, 128, 128), (17, 96, 203), (33, 203, 64), (64, 64, 96), (40, 7, 5)])
def test_few_rows_round_once(gpu, M, Dm, F, act):
    """Up to 64 rows y and dx are rounded once, by 2^-8 of their own size at most. What enters the second products keeps 16 bits (a
    share 2^-16 of each term), of dx also the pairs (2^-15); the fp32 sums' own error, 2^-24 of up to 512 terms each way, is
    within another 2^-16 of the terms."""
    x, wi, wo, dy = case(M, Dm, F, torch.bfloat16)
    y, saved = D.gated_ffn(x, wi, wo, act=act, save=True)
    assert torch.equal(D.gated_ffn(x, wi, wo, act=act), y)
    dx, _, _ = D.gated_ffn_grad(x, wi, wo, saved, dy, act=act)
    x, wi, wo, dy = (t.double().cpu() for t in (x, wi, wo, dy))
    a, v = ((x @ wi[k::2].T).requires_grad_(True) for k in (0, 1))
    h = R.glu(a, v, act)
    da, dv = torch.autograd.grad(h, (a, v), dy @ wo)
    h, dab = h.detach(), torch.stack([da, dv], -1).reshape(M, -1)
    for got, l, r, eps in ((y, h, wo.T, 2 * 2.0 ** -16), (dx, dab, wi, 4 * 2.0 ** -16)):
        assert ((got.double().cpu() - l @ r).abs() <= 2.0 ** -8 * (l @ r).abs() + eps * (l.abs() @ r.abs())).all()


def test_few_rows_keep_infinities(gpu):
    """An infinite unit is no NaN in the product that follows, and neither is the largest finite one."""
    bf = dict(device="cuda", dtype=torch.bfloat16)
    x, wi, wo = torch.zeros(2, 8, **bf), torch.zeros(16, 8, **bf), torch.zeros(8, 8, **bf)
    x[0, 0] = x[1, 1] = 1.0
    wi[0, 0] = wi[1, 0] = 2.0 ** 70  # unit 0 of row 0 is 2^140, past fp32
    wi[2, 1], wi[3, 1] = 2.0 ** 64, 2.0 ** 64 * (1 - 2.0 ** -8)  # unit 1 of row 1 is 2^128 (1 - 2^-8), the largest bf16
    wo[0, 0], wo[1, 1], wo[2, 1] = 1.0, 0.5, 0.25
    y = D.gated_ffn(x, wi, wo)
    top = 2.0 ** 127 * (1 - 2.0 ** -8)
    assert y[0, 0] == float("inf") and torch.equal(y[1, :3], torch.tensor([0.0, top, top / 2], **bf))


def test_fp32_weight_gradients_of_bf16(gpu):
    x, wi, wo, dy = case(700, 128, 264, torch.bfloat16)
    _, _, dwi, dwo = check(x, wi, wo, dy, dw_dtype=torch.float32)
    assert dwi.dtype == dwo.dtype == torch.float32


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_strided_rows(gpu, dt, off):
    x, wi, wo, dy = case(200, 128, 96, dt)
    ref = check(x, wi, wo, dy)

    def wide(t):
        buf = torch.full((200, 128 + 16), 5.0, device="cuda", dtype=dt)
        buf[:, off:off + 128] = t
        return buf[:, off:off + 128]
    got = check(wide(x), wi, wo, wide(dy))
    for a, b in zip(ref, got):
        assert R.rel(a, b) <= BARS[dt]
    out = torch.full((200, 144), 5.0, device="cuda", dtype=dt)
    D.gated_ffn(x, wi, wo, out=out[:, off:off + 128])
    assert R.rel(out[:, off:off + 128], ref[0]) <= BARS[dt]
    assert torch.all(out[:, :off] == 5) and torch.all(out[:, off + 128:] == 5)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("into", ["dy", "x"])
@pytest.mark.parametrize("M,Dm,F", [(8, 64, 96), (40, 203, 33), (300, 128, 96), (300, 203, 64), (2100, 64, 96)])
def test_gradient_into_its_inputs(gpu, M, Dm, F, into, dt):
    """dx may be dy or x: the weights' gradients read neither after it has been written."""
    x, wi, wo, dy = case(M, Dm, F, dt)
    _, saved = D.gated_ffn(x, wi, wo, save=True)
    ref = D.gated_ffn_grad(x, wi, wo, saved, dy)
    got = D.gated_ffn_grad(x, wi, wo, saved, dy, dx=dy if into == "dy" else x)
    for k, a, g in zip(("dx", "dw_in", "dw_out"), ref, got):
        assert torch.equal(a, g), k


def test_more_copies_than_a_launch_has_blocks(gpu):
    """2^24 tiles of rows of seven columns that are padded are more than one launch takes. Copies of 4096 rows, and 40 of their own
    at the end; against a smaller call, each within its bar."""
    M = 2 ** 29
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 50 GB")
    x, wi, wo, _ = case(4136, 7, 8, torch.bfloat16)
    ref = D.gated_ffn(x, wi, wo)
    far = torch.empty(M + 40, 7, device="cuda", dtype=torch.bfloat16)
    far[:M].view(M // 4096, 4096, 7).copy_(x[:4096])
    far[M:] = x[4096:]
    y = D.gated_ffn(far, wi, wo)
    assert R.rel(y[M:], ref[4096:]) <= 2 * BARS[torch.bfloat16] and R.rel(y[:4096], ref[:4096]) <= 2 * BARS[torch.bfloat16]
    v = y[:M].view(M // 4096, 4096 * 7)
    for part in v.split(2 ** 14):
        assert (part == v[0]).all()
    del far, y, v
    torch.cuda.empty_cache()
    L.call("ph_release_scratch")


def test_saturated_gates(gpu):
    """Gates far on both sides: the activation is the identity or zero, and its gradient finite."""
    x, wi, wo, dy = case(40, 64, 48, torch.float32)
    wi[0::4] *= 60.0
    wi[0::8] *= -1.0
    for act in ("silu", "gelu"):
        check(x, wi, wo, dy, act)


def test_non_finite_rows_stay_theirs(gpu):
    x, wi, wo, dy = case(70, 64, 96, torch.bfloat16)
    ref = D.gated_ffn(x, wi, wo)
    x[13] = float("nan")
    x[40, 3] = float("inf")
    y = D.gated_ffn(x, wi, wo)
    ok = [i for i in range(70) if i not in (13, 40)]
    assert torch.equal(y[ok], ref[ok]) and not torch.isfinite(y[13]).any()


def test_no_rows(gpu):
    x, wi, wo, dy = case(1, 16, 24, torch.bfloat16)
    x = dy = x[:0]
    y, saved = D.gated_ffn(x, wi, wo, save=True)
    dx, dwi, dwo = D.gated_ffn_grad(x, wi, wo, saved, dy)
    assert y.shape == (0, 16) and dx.shape == (0, 16) and not dwi.any() and not dwo.any()


def test_gradient_against_differences(gpu):
    x, wi, wo, dy = case(50, 32, 40, torch.float32)
    y, saved = D.gated_ffn(x, wi, wo, save=True)
    grads = D.gated_ffn_grad(x, wi, wo, saved, dy)
    f = lambda *a: float((D.gated_ffn(*a).double() * dy.double()).sum())
    e = 2.0 ** -7
    for i, g in enumerate(grads):
        base = [x, wi, wo]
        v = cu(20 + i, *base[i].shape, scale=float(base[i].abs().mean()))
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + e * v, base[i] - e * v
        want, size = float((g * v).sum()), float(g.norm() * v.norm())
        assert abs((f(*up) - f(*dn)) / (2 * e) - want) <= 2e-3 * (abs(want) + 0.1 * size)


def test_same_twice_and_on_another_stream(gpu):
    x, wi, wo, dy = case(1500, 136, 344, torch.bfloat16)
    a = check(x, wi, wo, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, saved = D.gated_ffn(x, wi, wo, save=True)
        b = (y, *D.gated_ffn_grad(x, wi, wo, saved, dy))
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("M", [8, 2000])
def test_graph_replays(gpu, M):
    x, wi, wo, dy = case(M, 128, 344, torch.bfloat16)
    check(x, wi, wo, dy)

    def both():
        y, saved = D.gated_ffn(x, wi, wo, save=True)
        return [y, D.gated_ffn(x, wi, wo), *D.gated_ffn_grad(x, wi, wo, saved, dy)]
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


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M", [8, 130, 4096])
def test_kept_pairs(gpu, M, act):
    """bf16 keeps the first 24 bits of v act'(a) and act(a): cut off at 2^-15 of the value, not rounded at 2^-9. The fp32 sums of
    64 exact products (of about 5 in all) are off by 2e-5 at most, which a pair takes up to 4 times (|v| under 5)."""
    Dm, F = 64, 96
    x, wi, wo, _ = case(M, Dm, F, torch.bfloat16)
    _, (pf, _) = D.gated_ffn(x, wi, wo, act=act, save=True)
    row = pf.cpu().contiguous().view(torch.uint8).numpy().reshape(M, 6 * F)
    b = np.zeros((M, 2 * F, 4), np.uint8)
    b[..., 2:] = row[:, :4 * F].reshape(M, 2 * F, 2)
    b[..., 1] = row[:, 4 * F:]
    got = b.view(np.float32)[..., 0].astype(np.float64)
    a, v = (x.double() @ wi.double()[k::2].T for k in (0, 1))
    a = a.cpu().requires_grad_(True)
    f = R.glu(a, torch.ones_like(a), act)
    p = torch.autograd.grad(f.sum(), a)[0] * v.cpu()
    ref = torch.stack([p, f.detach()], -1).reshape(M, -1).numpy()
    assert (np.abs(got - ref) <= 2.0 ** -15 * np.abs(ref) + 1e-4).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,Dm,F", [(8, 64, 96), (40, 203, 33), (300, 203, 64), (2100, 64, 96)])
def test_gradients_left_out(gpu, M, Dm, F, dt):
    """Each of dx, dw_in and dw_out may be left out; the others stay the same."""
    x, wi, wo, dy = case(M, Dm, F, dt)
    _, saved = D.gated_ffn(x, wi, wo, save=True)
    ref = D.gated_ffn_grad(x, wi, wo, saved, dy)
    pf, h = saved
    code = L.PH_F32 if dt is torch.float32 else L.PH_BF16
    for keep in range(1, 8):
        out = [torch.full_like(t, 7.0) if keep >> i & 1 else None for i, t in enumerate(ref)]
        p = [None if t is None else t.data_ptr() for t in out]
        L.call("ph_ffn_grad", code, L.PH_ACT_SILU, M, Dm, F, x.data_ptr(), Dm, wi.data_ptr(), wo.data_ptr(), pf.data_ptr(), h.data_ptr(),
               dy.data_ptr(), Dm, p[0], Dm, code, p[1], p[2], D._stream())
        for a, b in zip(out, ref):
            assert a is None or torch.equal(a, b), keep


def test_refusals(gpu):
    x, wi, wo, dy = case(4, 16, 24, torch.float32)
    with pytest.raises(TypeError):
        D.gated_ffn(x.half(), wi, wo)
    with pytest.raises(ValueError):
        D.gated_ffn(x, wi[:-2], wo)
    with pytest.raises(ValueError):
        D.gated_ffn(x, wi.bfloat16(), wo)
    with pytest.raises(ValueError):
        D.gated_ffn(x, wi, wo, act="relu")
    with pytest.raises(ValueError):
        D.gated_ffn(x, wi, wo.t().contiguous().t())
    y, saved = D.gated_ffn(x, wi, wo, save=True)
    with pytest.raises(ValueError):
        D.gated_ffn_grad(x, wi, wo, saved, dy[:2])
    with pytest.raises(L.PufferHipError):
        D.gated_ffn_grad(x, wi, wo, saved, dy, dw_dtype=torch.bfloat16)
    lib = L.lib()
    p = x.data_ptr()
    assert lib.ph_ffn(L.PH_F64, 0, 4, 16, 24, p, 16, p, p, None, None, p, 16, None) == L.PH_ERR_ARG
    assert lib.ph_ffn(L.PH_F32, 2, 4, 16, 24, p, 16, p, p, None, None, p, 16, None) == L.PH_ERR_ARG
    assert lib.ph_ffn(L.PH_F32, 0, 4, 16, 24, p, 15, p, p, None, None, p, 16, None) == L.PH_ERR_ARG
    assert lib.ph_ffn(L.PH_F32, 0, 4, 16, 24, p, 16, p, p, p, None, p, 16, None) == L.PH_ERR_ARG
    assert lib.ph_ffn(L.PH_F32, 0, 4, 0, 24, p, 16, p, p, None, None, p, 16, None) == L.PH_ERR_ARG
