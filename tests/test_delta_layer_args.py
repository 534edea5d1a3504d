"""Checks of the delta-rule policy layer's calls that come before anything runs on a GPU."""
import ctypes as C

import pytest
import torch

from pufferlean_amd import _lib as L
from pufferlean_amd import device as D

T, B, Hk, H, K, V = 2, 3, 1, 2, 8, 4


def delta(*lead, **kw):
    f = lambda *s: torch.zeros(*lead, *s)
    a = dict(q=f(Hk, K), k=f(Hk, K), v=f(H, V), a=f(H), b=f(H), A=torch.zeros(H))
    a.update(kw)
    return [a[n] for n in "qkvabA"]


@pytest.fixture
def no_call(monkeypatch):
    """A refused call does not reach the library."""
    def call(name, *a):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(D.L, "call", call)


@pytest.mark.parametrize("lead", [(), (B,), (1, T, B)])
def test_scan_takes_sequences(no_call, lead):
    with pytest.raises(ValueError, match=r"q must be \[T, B, Hk, K\]"):
        D.delta_scan(*delta(*lead))
    with pytest.raises(ValueError, match=r"q must be \[T, B, Hk, K\]"):
        D.delta_scan_grad(*delta(*lead), torch.zeros(4), torch.zeros(*lead, H, V))


@pytest.mark.parametrize("lead", [(), (T, B)])
def test_step_takes_one_step(no_call, lead):
    with pytest.raises(ValueError, match=r"q must be \[B, Hk, K\]"):
        D.delta_step(*delta(*lead), torch.zeros(B, H, K, V))


def test_tensors_on_the_host(no_call):
    for call in (lambda: D.delta_scan(*delta(T, B)), lambda: D.delta_step(*delta(B), torch.zeros(B, H, K, V)),
                 lambda: D.rms_norm(torch.zeros(3, 4)), lambda: D.sample_filtered(torch.zeros(3, 4), torch.zeros(3))):
        with pytest.raises(ValueError, match="on the current GPU"):
            call()


def test_types(no_call):
    for dt in (torch.float16, torch.float64, torch.int32):
        with pytest.raises(TypeError):
            D.delta_scan(*delta(T, B, q=torch.zeros(T, B, Hk, K, dtype=dt)))
        with pytest.raises(TypeError):
            D.rms_norm(torch.zeros(3, 4, dtype=dt))
        with pytest.raises(TypeError):
            D.sample_filtered(torch.zeros(3, 4, dtype=dt), torch.zeros(3))


def test_groups(no_call):
    for g in (0, -1, 3):
        with pytest.raises(ValueError, match="groups"):
            D.rms_norm(torch.zeros(3, 4), groups=g)


# ---- the library's own checks: they come before any use of the device ---------------------------------
NZ = 4096  # an address that is not NULL and never read


def delta_args(**kw):
    a = L.DeltaArgs(dtype=L.PH_F32, T=2, B=3, Hk=1, H=2, K=8, V=4, q=NZ, k=2 * NZ, v=3 * NZ, a=NZ, b=NZ, A=NZ, scale=1.0)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def refused(status, text):
    assert status == L.PH_ERR_ARG and text in L.lib().ph_last_error().decode(), L.lib().ph_last_error()


@pytest.mark.parametrize("kw,text", [(dict(dtype=L.PH_F64), "dtype"), (dict(K=129), "heads of K"), (dict(V=0), "heads of K"), (dict(V=129), "heads of K"),
                                     (dict(Hk=0), "key heads"), (dict(H=3, Hk=2), "key heads"), (dict(H=1, Hk=2), "key heads"),
                                     (dict(B=1 << 25), "out of range"), (dict(T=(1 << 30) + 1), "out of range"), (dict(T=0), "no steps"),
                                     (dict(q=None), "missing"), (dict(A=None), "missing"), (dict(scale=float("nan")), "scale")])
def test_scan_refuses(kw, text):
    lib, a = L.lib(), delta_args(**kw)
    refused(lib.ph_delta_scan(C.byref(a), 9 * NZ, 1, 1, 1, None, None, None), text)
    refused(lib.ph_delta_scan_grad(C.byref(a), NZ, 9 * NZ, 1, 1, 1, None, C.byref(L.DeltaGrads()), None), text)


def test_scan_refuses_outputs():
    lib, a = L.lib(), delta_args()
    refused(lib.ph_delta_scan(None, NZ, 1, 1, 1, None, None, None), "arguments missing")
    refused(lib.ph_delta_scan(C.byref(a), None, 1, 1, 1, None, None, None), "y missing")
    for y in (a.q, a.k, a.v):
        refused(lib.ph_delta_scan(C.byref(a), y, 1, 1, 1, None, None, None), "y may not be")
        refused(lib.ph_delta_step(C.byref(delta_args(T=1)), y, 1, 1, NZ, None), "y may not be")
    g = L.DeltaGrads(dv=5 * NZ)
    refused(lib.ph_delta_scan_grad(C.byref(a), None, NZ, 1, 1, 1, None, C.byref(g), None), "kept states missing")
    refused(lib.ph_delta_scan_grad(C.byref(a), NZ, 5 * NZ, 1, 1, 1, None, C.byref(g), None), "may not be an input")
    refused(lib.ph_delta_scan_grad(C.byref(a), NZ, 5 * NZ, 1, 1, 1, None, C.byref(L.DeltaGrads(dq=a.q)), None), "may not be an input")
    refused(lib.ph_delta_step(C.byref(delta_args(T=2)), 9 * NZ, 1, 1, NZ, None), "a single step")
    refused(lib.ph_delta_step(C.byref(delta_args(T=1)), 9 * NZ, 1, 1, None, None), "state missing")


def rms_args(**kw):
    a = L.RmsArgs(dtype=L.PH_BF16, M=3, C=8, G=1, x=NZ, ldx=8, eps=1e-6)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,text", [(dict(dtype=L.PH_I32), "dtype"), (dict(C=0), "columns"), (dict(G=3), "groups"), (dict(G=0), "groups"), (dict(ldx=7), "stride"),
                                     (dict(scale=NZ), "a scale needs"), (dict(scale=NZ, add=NZ, ldadd=8, G=2), "a scale needs"),
                                     (dict(add=NZ, ldadd=4), "stride"), (dict(gate=NZ, ldgate=0), "stride"), (dict(eps=-1.0), "eps"),
                                     (dict(M=(1 << 30) + 1), "rows"), (dict(x=None), "missing")])
def test_rms_refuses(kw, text):
    lib, a = L.lib(), rms_args(**kw)
    refused(lib.ph_rms_norm(C.byref(a), 2 * NZ, 8, None, 0, None, None), text)
    refused(lib.ph_rms_norm_grad(C.byref(a), NZ, NZ, 8, None, 0, C.byref(L.RmsGrads()), None), text)


def test_rms_refuses_outputs():
    lib, a = L.lib(), rms_args(add=2 * NZ, ldadd=8, gate=3 * NZ, ldgate=8)
    refused(lib.ph_rms_norm(C.byref(a), NZ, 8, NZ, 8, None, None), "out and res")
    refused(lib.ph_rms_norm(C.byref(a), NZ, 7, None, 0, None, None), "stride")
    for kw in (dict(dx=NZ, dadd=NZ), dict(dx=NZ, dgate=NZ), dict(dadd=NZ, dgate=NZ)):
        g = L.RmsGrads(lddx=8, lddadd=8, lddgate=8, **kw)
        refused(lib.ph_rms_norm_grad(C.byref(a), NZ, NZ, 8, None, 0, C.byref(g), None), "two gradients")


@pytest.mark.parametrize("kw,text", [(dict(dtype=L.PH_F64), "dtype"), (dict(A=0), "entries"), (dict(A=(1 << 20) + 1), "entries"), (dict(ld=3), "stride"),
                                     (dict(x=None), "missing"), (dict(u=None), "missing"), (dict(act=None), "missing")])
def test_draw_refuses(kw, text):
    k = dict(dtype=L.PH_F32, x=NZ, ld=1 << 21, N=3, A=4, u=NZ, act=NZ)
    k.update(kw)
    refused(L.lib().ph_sample_filtered(k["dtype"], k["x"], k["ld"], k["N"], k["A"], k["u"], None, None, None, None, k["act"], None, None), text)


def test_scan_refuses_what_it_would_overwrite():
    lib, a = L.lib(), delta_args(a=6 * NZ, b=7 * NZ)
    for y in (a.a, a.b):
        refused(lib.ph_delta_scan(C.byref(a), y, 1, 1, 1, None, None, None), "y may not be")
        refused(lib.ph_delta_step(C.byref(delta_args(T=1, a=6 * NZ, b=7 * NZ)), y, 1, 1, NZ, None), "y may not be")
    for kw in (dict(da=a.a), dict(db=a.a), dict(da=a.b), dict(dk=a.b)):
        refused(lib.ph_delta_scan_grad(C.byref(a), NZ, 5 * NZ, 1, 1, 1, None, C.byref(L.DeltaGrads(**kw)), None), "may not be an input")
    for kw in (dict(dq=9 * NZ, dk=9 * NZ), dict(dk=9 * NZ, dv=9 * NZ), dict(da=9 * NZ, db=9 * NZ), dict(dv=9 * NZ, da=9 * NZ)):
        refused(lib.ph_delta_scan_grad(C.byref(a), NZ, 5 * NZ, 1, 1, 1, None, C.byref(L.DeltaGrads(**kw)), None), "two gradients")
