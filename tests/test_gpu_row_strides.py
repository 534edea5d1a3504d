"""bf16 products of operands whose rows lie far apart: an offset within a tile of 256 rows passes 31 bits. Sizes are such that
packed operands take the kernels of large tiles."""
import numpy as np
import pytest
import torch

import policy_layer_ref as R
from pufferlean_amd import device as D
from pufferlean_amd import rng

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def cu(seed, *shape, scale=1.0):
    return torch.from_numpy(rng.normal(seed, int(np.prod(shape))).reshape(shape) * scale).float().to("cuda", BF)


def far(stride, *ts):
    """The matrices side by side in rows `stride` apart; the rest of the buffer is never touched."""
    M, n = len(ts[0]), sum(t.shape[1] for t in ts)
    buf = torch.empty((M - 1) * stride + n, device="cuda", dtype=BF)
    out, at = [], 0
    for t in ts:
        v = buf[at:].as_strided(t.shape, (stride, 1))
        v.copy_(t)
        out.append(v)
        at += t.shape[1]
    return out


@pytest.mark.parametrize("stride", [2 ** 23, 2 ** 23 + 8, 2 ** 24])
@pytest.mark.parametrize("swap", [False, True])
def test_gemm(gpu, stride, swap):
    """fp32 sums of 16 exact products; the result is rounded once."""
    x, w = cu(1, 300, 16), cu(2, 32768, 16)
    f, = far(stride, x)
    y = D.gemm(*((w, f) if swap else (f, w)), trans_b=True, out_dtype=BF)
    ref = x.double() @ w.double().t()
    assert R.rel(y, ref.t() if swap else ref) <= R.BF16 + 1e-5


@pytest.mark.parametrize("stride", [2 ** 23, 2 ** 23 + 8])
def test_gated_ffn(gpu, stride):
    """Packed and far apart the same operands, each result within its bar (three roundings) of the exact one."""
    x, dy, wi, wo = cu(1, 2048, 16), cu(2, 2048, 16), cu(3, 2 * 8192, 16, scale=0.25), cu(4, 16, 8192, scale=2.0 ** -6.5)
    fx, fdy = far(stride, x, dy)
    res = []
    for a, g in ((x, dy), (fx, fdy)):
        y, saved = D.gated_ffn(a, wi, wo, save=True)
        res.append((y, *D.gated_ffn_grad(a, wi, wo, saved, g)))
    for p, q in zip(*res):
        assert R.rel(q, p) <= 6 * R.BF16
