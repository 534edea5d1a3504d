"""Outputs of the delta-rule layer's calls that share elements with an input or another output are refused before anything runs on
a GPU; columns of one buffer that lie between each other are not the same elements."""
import ctypes as C

import pytest

from pufferlean_amd import _lib as L

AT = 1 << 20  # addresses that are never read
T, B, Hk, H, K, V = 3, 4, 1, 2, 8, 16
W = 2 * Hk * K + 3 * H * V + 2 * H  # columns [q | k | v | out | out | a | b], fp32
Q, KC, VC = 0, Hk * K, 2 * Hk * K
Y, Z = VC + H * V, VC + 2 * H * V
AC = Z + H * V


def args(**kw):
    at = lambda c: AT + 4 * c
    a = L.DeltaArgs(dtype=L.PH_F32, T=T, B=B, Hk=Hk, H=H, K=K, V=V, q=at(Q), k=at(KC), v=at(VC), a=at(AC), b=at(AC + H), A=AT // 2, scale=1.0)
    for n in "qkv":
        setattr(a, n + "_t", B * W), setattr(a, n + "_b", W), setattr(a, n + "_h", dict(q=K, k=K, v=V)[n])
    for n in "ab":
        setattr(a, n + "_t", B * W), setattr(a, n + "_b", W)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def refused(status, text):
    assert status == L.PH_ERR_ARG and text in L.lib().ph_last_error().decode(), L.lib().ph_last_error()


def scan(y, h_out=None, keep=None, strides=(B * W, W, V), **kw):
    return L.lib().ph_delta_scan(C.byref(args(**kw)), y, *strides, h_out, keep, None)


FAR, STATE = 8 * AT, B * H * K * V * 4


@pytest.mark.parametrize("y,strides", [(AT + 4 * (VC + 1), None), (AT + 4 * (VC - 1), None), (AT + 4 * (VC - V * H + 1), None), (AT + 4 * (VC + W), None),
                                       (AT + 4 * (AC - 1), None), (AT // 2 - 4, (1000, 100, 50)), (AT - 4 * B * W * (T - 1) + 4 * Q, None)])
def test_y_over_an_input(y, strides):
    refused(scan(y, strides=strides or (B * W, W, V)), "y may not be an input or share elements")


@pytest.mark.parametrize("strides", [(B * W, W, V - 1), (0, W, V), (B * W, 0, V), (W, W, V), (3 * W + 10, W, V)])
def test_y_over_itself(strides):
    refused(scan(FAR, strides=strides), "twice")


@pytest.mark.parametrize("h_out,keep,h0", [(FAR - 4, None, FAR), (FAR + STATE - 4, None, FAR), (AT + 4 * Y, None, None), (AT, None, None), (None, AT + 4 * Y, None),
                                          (None, FAR, FAR), (FAR, FAR + 4, None)])
def test_states(h_out, keep, h0):
    refused(scan(AT + 4 * Y, h_out=h_out, keep=keep, h0=h0), "h_out or the kept states")


def test_step():
    lib, a = L.lib(), args(T=1)
    refused(lib.ph_delta_step(C.byref(a), AT + 4 * (VC + 1), W, V, FAR, None), "y may not be")
    refused(lib.ph_delta_step(C.byref(a), AT + 4 * Y, W, V, AT + 4 * Y, None), "the state shares")
    refused(lib.ph_delta_step(C.byref(a), FAR + STATE - 4, W, V, FAR, None), "the state shares")


def grads(**kw):
    g = L.DeltaGrads()
    for n, c in dict(dict(q=Q, k=KC, v=VC, a=AC, b=AC + H), **kw).items():
        setattr(g, "d" + n, None if c is None else 4 * AT + 4 * c)
    for n in "qkv":
        setattr(g, f"d{n}_t", B * W), setattr(g, f"d{n}_b", W), setattr(g, f"d{n}_h", dict(q=K, k=K, v=V)[n])
    for n in "ab":
        setattr(g, f"d{n}_t", B * W), setattr(g, f"d{n}_b", W)
    return g


def grad(g, dy=AT + 4 * Y, dh=None, keep=FAR):
    return L.lib().ph_delta_scan_grad(C.byref(args()), keep, dy, B * W, W, V, dh, C.byref(g), None)


@pytest.mark.parametrize("kw", [dict(k=KC - 1), dict(v=VC - 1), dict(a=AC + 1), dict(b=Q), dict(v=W + Q), dict(b=AC - 1)])
def test_gradients_over_one_another(kw):
    refused(grad(grads(**kw)), "two gradients")


def test_gradients_over_inputs():
    for dy in (4 * AT, 4 * AT + 4 * (VC - 1), 4 * AT + 4 * AC):
        refused(grad(grads(), dy=dy), "may not be an input")
    refused(grad(grads(), keep=4 * AT + 4 * (Y - 1)), "may not be an input")
    g = grads()
    g.dh0 = FAR + 4
    refused(grad(g, dh=FAR, keep=16 * AT), "may not be an input")
    g.dh0 = FAR
    refused(grad(g, keep=FAR - 4), "may not be an input")
    g.dv_h = V - 1
    refused(grad(g, keep=16 * AT), "twice")


def rms(**kw):
    a = L.RmsArgs(dtype=L.PH_BF16, M=5, C=8, G=1, x=AT, ldx=24, add=AT + 16, ldadd=24, gate=AT + 32, ldgate=24, eps=1e-6)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_rms():
    lib, a = L.lib(), rms()
    for out, ld, res, ldres in ((AT + 2, 24, FAR, 8), (AT - 2, 24, FAR, 8), (AT, 48, FAR, 8), (AT + 48, 24, FAR, 8), (FAR, 8, AT + 14, 24), (FAR, 8, AT + 64, 24)):
        refused(lib.ph_rms_norm(C.byref(a), out, ld, res, ldres, None, None), "with an input that it is not")
    refused(lib.ph_rms_norm(C.byref(a), FAR, 8, FAR + 14, 16, None, None), "out and res")
    refused(lib.ph_rms_norm(C.byref(rms(w=FAR + 4)), FAR, 8, 2 * FAR, 8, None, None), "with an input that it is not")
    refused(lib.ph_rms_norm(C.byref(a), FAR, 8, 2 * FAR, 8, FAR + 4, None), "with an input that it is not")
    for kw, text in ((dict(dx=FAR, dadd=FAR + 2), "two gradients"), (dict(dx=AT + 2), "with an input that it is not"), (dict(dadd=4 * AT + 4), "with an input that it is not"),
                     (dict(dgate=2 * FAR - 4), "with an input that it is not")):
        g = L.RmsGrads(lddx=8, lddadd=8, lddgate=8, **kw)
        refused(lib.ph_rms_norm_grad(C.byref(a), 2 * FAR, 4 * AT, 8, None, 0, C.byref(g), None), text)


def test_draw():
    lib = L.lib()
    call = lambda act, logp, u=2 * AT, k=None: lib.ph_sample_filtered(L.PH_F32, AT, 10, 6, 8, u, None, k, None, None, act, logp, None)
    refused(call(AT + 4, FAR), "with the logits")
    refused(call(AT - 4, FAR), "with the logits")
    refused(call(FAR, AT + 4 * 57), "with the logits")
    refused(call(FAR, 2 * AT + 4), "lies across")
    refused(call(2 * AT - 4, FAR), "lies across")
    refused(call(FAR, 2 * FAR, k=FAR + 4), "lies across")
    refused(call(FAR, FAR + 20), "act and logp")


@pytest.mark.gpu
def test_columns_between_the_inputs(gpu):
    """Outputs in columns of the inputs' own buffer give what they give elsewhere."""
    import torch

    from pufferlean_amd import device as D
    from test_gpu_delta import cu
    t, b, h, w = 50, 3, 2, 16
    cols = cu(1, t, b, 5 * h * w + 2 * h, dtype=torch.bfloat16)
    q, k, v, y, z, a, s = cols.split([h * w] * 5 + [h, h], dim=-1)
    q, k, v, y, z = (x.unflatten(-1, (h, w)) for x in (q, k, v, y, z))
    A = -cu(2, h).abs()
    want, saved = D.delta_scan(q, k, v, a, s, A, save=True)
    assert D.delta_scan(q, k, v, a, s, A, out=y) is y and torch.equal(y, want)
    dv = D.delta_scan_grad(q, k, v, a, s, A, saved, y)["dv"]
    assert torch.equal(D.delta_scan_grad(q, k, v, a, s, A, saved, y, dv=z)["dv"], dv) and torch.equal(z, dv)
    n = D.rms_norm(q[:, :, 0].flatten(0, 1))[0]
    out = v[:, :, 1].flatten(0, 1)
    D.rms_norm(q[:, :, 0].flatten(0, 1), out=out)
    assert torch.equal(out, n)
