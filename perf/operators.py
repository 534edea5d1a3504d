"""The operators of a state-space policy layer: layer normalisation, the selective state-space scan with its short
causal convolution (sequences, their gradient, and single tokens), and the gated feed-forward block.

``listed()`` names the cases whose time counts, ``draw(rng)`` makes more of the same ranges, ``prepare`` builds what a
program holds before the call, ``run`` is one pass, ``work`` the bytes and operations that no implementation can
avoid, and ``exact`` the outputs from the definitions in 64 bits. ``own`` chooses between the plain form (elementary
torch operations in fp32, rounded once at the end) and the library's kernels.

Sequences are time-major, [T, B, ...], as everywhere in this library; the inputs of the scan are column slices of one
projection's output, [x | z | delta | B | C], as the layer in front of it leaves them.
"""
from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # normalisation of one rollout step of a few environments, small policy (latency)
        dict(name="norm_48x128_f32", kind="norm", M=48, C=128, dtype="f32", train=False),
        # ragged rows and columns, both directions
        dict(name="norm_train_6699x203_f32", kind="norm", M=6699, C=203, dtype="f32", train=True),
        # a whole minibatch of 4096 segments x 64 steps at width 512, both directions
        dict(name="norm_train_262144x512", kind="norm", M=262144, C=512, dtype="bf16", train=True),
        # a long prompt of a few sequences: the recurrence alone would leave the chip idle
        dict(name="scan_8192x2_c512", kind="scan", T=8192, B=2, C=512, N=16, G=1, K=4, dtype="bf16", gate=True,
             done=False, train=False),
        # a minibatch of short segments with episode ends, both directions (the largest call)
        dict(name="scan_train_64x2048_c512", kind="scan", T=64, B=2048, C=512, N=16, G=1, K=4, dtype="bf16", gate=True,
             done=True, train=True),
        # odd everything in fp32, no gate, three taps
        dict(name="scan_train_33x203_c96_f32", kind="scan", T=33, B=203, C=96, N=5, G=1, K=3, dtype="f32", gate=False,
             done=True, train=True),
        # long sequences in training, two groups of B and C
        dict(name="scan_train_2048x8_c384", kind="scan", T=2048, B=8, C=384, N=16, G=2, K=4, dtype="bf16", gate=True,
             done=True, train=True),
        # one environment step of the rollout, the state carried in fp32
        dict(name="step_4096_c512", kind="step", B=4096, C=512, N=16, G=1, K=4, dtype="bf16", gate=True),
        # a few environments of a small policy (latency)
        dict(name="step_48_c128_f32", kind="step", B=48, C=128, N=8, G=1, K=4, dtype="f32", gate=True),
        # single tokens through the feed-forward block
        dict(name="ffn_8x512x1376", kind="ffn", M=8, D=512, F=1376, dtype="bf16", act="silu", train=False),
        # odd sizes in fp32, both directions
        dict(name="ffn_train_6699x203x531_f32", kind="ffn", M=6699, D=203, F=531, dtype="f32", act="gelu", train=True),
        # a minibatch of 1024 segments x 64 steps at width 512, both directions
        dict(name="ffn_train_65536x512x1376", kind="ffn", M=65536, D=512, F=1376, dtype="bf16", act="silu", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _even(rng, v):
    """Two draws in three have the multiples of eight that a policy's widths are; the others are odd."""
    return max(8, v // 8 * 8) if rng.random() < 0.67 else v | 1


def draw(rng):
    kind = rng.choice(["norm", "norm", "scan", "scan", "scan", "step", "ffn", "ffn"])
    dt = rng.choice(["bf16", "bf16", "f32"])
    if kind == "norm":
        c = dict(kind=kind, M=_log(rng, 1, 262144), C=_even(rng, _log(rng, 8, 2048)), dtype=dt,
                 train=rng.random() < 0.7)
        while c["M"] * c["C"] > 1 << 27:
            c["M"] //= 2
        return c
    if kind == "scan":
        G = rng.choice([1, 1, 2])
        c = dict(kind=kind, T=_log(rng, 2, 8192), B=_log(rng, 1, 2048), C=G * _even(rng, _log(rng, 16, 640) // G), G=G,
                 N=rng.choice([4, 7, 8, 16, 16, 16, 24, 32]), K=rng.choice([0, 2, 3, 4, 4]), dtype=dt,
                 gate=rng.random() < 0.7, done=rng.random() < 0.5, train=rng.random() < 0.6)
        while c["T"] * c["B"] * c["C"] * c["N"] > 1 << 29:
            big = "T" if c["T"] > c["B"] else "B"
            c[big] = (c[big] + 1) // 2
        return c
    if kind == "step":
        G = rng.choice([1, 1, 2])
        return dict(kind=kind, B=_log(rng, 1, 4096), C=G * _even(rng, _log(rng, 16, 512) // G), G=G,
                    N=rng.choice([4, 7, 8, 16, 16]), K=rng.choice([0, 3, 4, 4]), dtype=dt, gate=rng.random() < 0.7)
    c = dict(kind=kind, M=_log(rng, 1, 65536), D=_even(rng, _log(rng, 16, 1024)), F=_even(rng, _log(rng, 16, 1400)),
             dtype=dt, act=rng.choice(["silu", "silu", "gelu"]), train=rng.random() < 0.6)
    cap = 65536 * 512 * 1376 // (1 if dt == "bf16" else 8)
    while c["M"] * c["D"] * c["F"] > cap:
        c["M"] //= 2
    return c


# ---- inputs ------------------------------------------------------------------------------------------
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DT[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = dict(case=case)
    if case["kind"] == "norm":
        M, C = case["M"], case["C"]
        # residual-stream rows: their own offset and scale
        s["x"] = (normal(M, C) * (0.5 + uniform(M, 1)) + normal(M, 1, scale=0.3)).to(dt)
        s["w"], s["b"] = 1 + normal(C, scale=0.1), normal(C, scale=0.1)
        if case["train"]:
            s["dy"] = normal(M, C, dtype=dt)
        return s
    if case["kind"] == "ffn":
        M, D, F = case["M"], case["D"], case["F"]
        s["x"] = normal(M, D, dtype=dt)
        s["w_in"] = normal(2 * F, D, scale=1 / math.sqrt(D), dtype=dt)  # rows 2j, 2j+1: gate and value of unit j
        s["w_out"] = normal(D, F, scale=1 / math.sqrt(F), dtype=dt)
        if case["train"]:
            s["dy"] = normal(M, D, dtype=dt)
        return s
    B, C, N, G, K = case["B"], case["C"], case["N"], case["G"], case["K"]
    T = case.get("T", 1)
    lead = (T, B) if case["kind"] == "scan" else (B,)
    parts = [C, C if case["gate"] else 0, C, G * N, G * N]
    cols = normal(*lead, sum(parts), dtype=dt).split(parts, dim=-1)
    s["x"], s["z"], s["delta"], s["Bm"], s["Cm"] = cols
    if not case["gate"]:
        s["z"] = None
    s["A"] = -(1 + torch.arange(N, device="cuda", dtype=torch.float32)) * (0.8 + 0.4 * uniform(C, 1))
    s["D"] = 1 + normal(C, scale=0.1)
    dt0 = torch.exp(uniform(C) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))  # time steps of 1e-3 to 1e-1
    s["dt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
    s["conv_w"] = normal(C, K, scale=1 / math.sqrt(K)) if K else None
    s["conv_b"] = normal(C, scale=0.1) if K else None
    s["h"] = normal(B, C, N, scale=0.2)
    s["win"] = normal(B, K - 1, C) if K > 1 else None
    s["done"] = (uniform(T, B) < 0.05).float() if case.get("done") else None
    s["first"] = (uniform(B) < 0.1).float()
    if case.get("train"):
        s["dy"] = normal(T, B, C, dtype=dt)
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)[case["kind"]](s, case)


def _own_norm(s, case):
    from pufferlean_amd import device as D
    y, mean, rstd = D.layer_norm(s["x"], s["w"], s["b"])
    if not case["train"]:
        return y
    dx, dw, db = D.layer_norm_grad(s["x"], s["w"], mean, rstd, s["dy"])
    return dict(y=y, dx=dx, dw=dw, db=db)


def _own_ffn(s, case):
    from pufferlean_amd import device as D
    if not case["train"]:
        return D.gated_ffn(s["x"], s["w_in"], s["w_out"], act=case["act"])
    y, saved = D.gated_ffn(s["x"], s["w_in"], s["w_out"], act=case["act"], save=True)
    dx, dw_in, dw_out = D.gated_ffn_grad(s["x"], s["w_in"], s["w_out"], saved, s["dy"], act=case["act"])
    return dict(y=y, dx=dx, dw_in=dw_in, dw_out=dw_out)


def _scan_args(s):
    return dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], conv_w=s["conv_w"], conv_b=s["conv_b"], groups=s["case"]["G"])


def _own_scan(s, case):
    from pufferlean_amd import device as D
    h, win = torch.empty_like(s["h"]), None if s["win"] is None else torch.empty_like(s["win"])
    kw = dict(_scan_args(s), done=s["done"], first=s["first"])
    out = D.ssm_scan(s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], h0=s["h"], win0=s["win"], h_out=h, win_out=win,
                     save=case["train"], **kw)
    if not case["train"]:
        return dict(y=out, h=h, win=win)
    y, saved = out
    x, z = s["x"], s["z"]
    # the gradients go where the projection's backward pass reads them: one buffer of the same columns
    T, B, C = x.shape
    parts = [C, C if z is not None else 0, C, s["Bm"].shape[-1], s["Cm"].shape[-1]]
    dx, dz, dd, dB, dC = torch.empty(T, B, sum(parts), device=x.device, dtype=x.dtype).split(parts, dim=-1)
    grads = D.ssm_scan_grad(x, s["delta"], s["A"], s["Bm"], s["Cm"], saved, s["dy"], win0=s["win"], dx=dx, ddelta=dd,
                            dBm=dB, dCm=dC, dz=dz if z is not None else None, **kw)
    return dict(y=y, h=h, win=win, **grads)


def _own_step(s, case):
    from pufferlean_amd import device as D
    y = D.ssm_step(s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], s["h"], s["win"], first=s["first"],
                   **_scan_args(s))
    return dict(y=y, h=s["h"], win=s["win"])


def _norm(x, w, b, eps=1e-5):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return d * r, r


def _plain_norm(s, case):
    n, r = _norm(s["x"], s["w"], s["b"])
    dt = s["x"].dtype
    y = (n * s["w"] + s["b"]).to(dt)
    if not case["train"]:
        return y
    dy = s["dy"].float()
    dn = dy * s["w"]
    dx = r * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
    return dict(y=y, dx=dx.to(dt), dw=(dy * n).sum(0), db=dy.sum(0))


def _act(a, kind):
    """The activation and its derivative."""
    if kind == "silu":
        g = 1 / (1 + torch.exp(-a))
        return a * g, g * (1 + a * (1 - g))
    p = 0.5 * (1 + torch.erf(a / math.sqrt(2)))
    return a * p, p + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)


def _plain_ffn(s, case):
    dt = s["x"].dtype
    x, wi, wo = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    ab = x @ wi.t()
    a, b = ab[:, 0::2], ab[:, 1::2]
    v, dv = _act(a, case["act"])
    h = v * b
    y = (h @ wo.t()).to(dt)
    if not case["train"]:
        return y
    dy = s["dy"].float()
    dh = dy @ wo
    dab = torch.stack([dh * b * dv, dh * v], dim=-1).reshape(ab.shape)
    return dict(y=y, dx=(dab @ wi).to(dt), dw_in=(dab.t() @ x).to(dt), dw_out=(dy.t() @ h).to(dt))


def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first axis, by doubling."""
    n = 1
    while n < a.shape[0]:
        b = torch.cat([b[:n], b[n:] + a[n:] * b[:-n]])
        a = torch.cat([a[:n], a[n:] * a[:-n]])
        n *= 2
    return b


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _taps(s, x, keep, K):
    """The K inputs that each step's convolution sees, [K, T, B, C], and whether each is of the same episode."""
    T = x.shape[0]
    hist = torch.cat([s["win"].float().transpose(0, 1), x]) if K > 1 else x
    k = torch.cat([keep.new_ones(K - 1, *keep.shape[1:]), keep])
    back = torch.stack([k[K - 1 - j:K - 1 - j + T] for j in range(K)])  # [j]: keep of step t - j
    same = torch.cat([torch.ones_like(back[:1]), torch.cumprod(back, 0)[:-1]]).flip(0)  # tap i is K-1-i steps back
    return torch.stack([hist[i:i + T] for i in range(K)]), same, hist


def _plain_scan(s, case):
    K, N, G, dt = case["K"], case["N"], case["G"], s["x"].dtype
    x, delta = s["x"].float(), s["delta"].float()
    T, B, C = x.shape
    start = torch.cat([s["first"][None], s["done"][:-1] if s["done"] is not None else s["first"].new_zeros(T - 1, B)])
    keep = (1 - start)[:, :, None]
    # the short convolution
    if K:
        taps, same, hist = _taps(s, x, keep, K)
        w = s["conv_w"].t()[:, None, None, :]
        c = (taps * same * w).sum(0) + s["conv_b"]
        gc = 1 / (1 + torch.exp(-c))
        u = c * gc
    else:
        u = x
    # the scan
    step = _softplus(delta + s["dt_bias"])
    per = C // G

    def heads(m):  # [T, B, G*N] -> [T, B, C, N]
        return m.float().reshape(T, B, G, 1, N).expand(T, B, G, per, N).reshape(T, B, C, N)

    Bm, Cm = heads(s["Bm"]), heads(s["Cm"])
    a = torch.exp(step[..., None] * s["A"])
    ak = a * keep[..., None]
    du_in = (step * u)[..., None] * Bm
    du_in[0] += ak[0] * s["h"]
    h = _linear_scan(ak, du_in)
    o = (h * Cm).sum(-1) + s["D"] * u
    if s["z"] is not None:
        z = s["z"].float()
        gz = 1 / (1 + torch.exp(-z))
        y = o * z * gz
    else:
        y = o
    out = dict(y=y.to(dt), h=h[-1].contiguous(), win=None)
    if K > 1:
        k = torch.cat([keep.new_ones(K - 1, B, 1), keep])[T:]
        tail = torch.cat([k[1:].flip(0).cumprod(0).flip(0), torch.ones_like(k[:1])])
        out["win"] = (hist[T:] * tail).transpose(0, 1).contiguous()
    if not case["train"]:
        return out
    dy = s["dy"].float()
    do = dy
    if s["z"] is not None:
        do = dy * z * gz
        out["dz"] = (dy * o * gz * (1 + z * (1 - gz))).to(dt)
    nxt = torch.cat([ak[1:], torch.zeros_like(ak[:1])])
    g = _linear_scan(nxt.flip(0), (do[..., None] * Cm).flip(0)).flip(0)
    prev = torch.cat([s["h"][None], h[:-1]])
    q = g * ak * prev
    gB = (g * Bm).sum(-1)
    out["dBm"] = (g * (step * u)[..., None]).reshape(T, B, G, per, N).sum(3).reshape(T, B, G * N).to(dt)
    out["dCm"] = (h * do[..., None]).reshape(T, B, G, per, N).sum(3).reshape(T, B, G * N).to(dt)
    out["dA"] = (q * step[..., None]).sum((0, 1))
    out["dD"] = (do * u).sum((0, 1))
    ddt = ((q * s["A"]).sum(-1) + u * gB) / (1 + torch.exp(-(delta + s["dt_bias"])))
    out["ddelta"], out["ddt_bias"] = ddt.to(dt), ddt.sum((0, 1))
    du = step * gB + s["D"] * do
    if not K:
        out["dx"] = du.to(dt)
        return out
    dc = du * gc * (1 + c * (1 - gc))
    out["dconv_w"] = (dc * taps * same).sum((1, 2)).t().contiguous()
    out["dconv_b"] = dc.sum((0, 1))
    dt_taps = dc * same * w
    pad = torch.nn.functional.pad
    dx = torch.stack([pad(dt_taps[i][K - 1 - i:], (0, 0, 0, 0, 0, K - 1 - i))[:T] if T > K - 1 - i else
                      torch.zeros_like(dc) for i in range(K)]).sum(0)
    out["dx"] = dx.to(dt)
    return out


def _plain_step(s, case):
    K, N, G, dt = case["K"], case["N"], case["G"], s["x"].dtype
    x = s["x"].float()
    B, C = x.shape
    keep = (1 - s["first"])[:, None]
    if K > 1:
        hist = torch.cat([s["win"] * keep[..., None], x[:, None]], 1)
        c = (hist * s["conv_w"].t()).sum(1) + s["conv_b"]
        s["win"].copy_(hist[:, 1:])
    elif K:
        c = x * s["conv_w"][:, 0] + s["conv_b"]
    u = c / (1 + torch.exp(-c)) if K else x
    step = _softplus(s["delta"].float() + s["dt_bias"])
    Bm, Cm = (m.float().reshape(B, G, 1, N).expand(B, G, C // G, N).reshape(B, C, N) for m in (s["Bm"], s["Cm"]))
    h = torch.exp(step[..., None] * s["A"]) * (s["h"] * keep[..., None]) + (step * u)[..., None] * Bm
    s["h"].copy_(h)
    y = (h * Cm).sum(-1) + s["D"] * u
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1 + torch.exp(-z))
    return dict(y=y.to(dt), h=s["h"], win=s["win"])


_run_own = dict(norm=_own_norm, ffn=_own_ffn, scan=_own_scan, step=_own_step)
_run_plain = dict(norm=_plain_norm, ffn=_plain_ffn, scan=_plain_scan, step=_plain_step)


# ---- the least that each pass needs -------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "norm":
        n = case["M"] * case["C"]
        # forward: x in, y out; backward: dy in, dx out (x again counts as the same input)
        return dict(bytes=n * e * (4 if case["train"] else 2) + 16 * case["C"], flops=n * (18 if case["train"] else 7))
    if case["kind"] == "ffn":
        M, D, F = case["M"], case["D"], case["F"]
        if not case["train"]:
            return dict(bytes=e * (2 * M * D + 3 * F * D), flops=6 * M * D * F)
        return dict(bytes=e * (4 * M * D + 6 * F * D), flops=18 * M * D * F)
    B, C, N, G, K = case["B"], case["C"], case["N"], case["G"], case["K"]
    T = case.get("T", 1)
    row = C * (3 + (1 if case["gate"] else 0)) + 2 * G * N  # x, delta, y (z) and B, C
    state = 8 * B * C * N + 8 * B * max(0, K - 1) * C
    par = 4 * C * (N + K + 3)
    n = T * B * C
    if not case.get("train"):
        # per state: the decay's argument and exponential, input, update, output
        return dict(bytes=T * B * row * e + state + par, flops=n * (7 * N + 2 * K + 12))
    # backward: dy in; dx, ddelta, (dz), dB, dC out; per state twice the forward's and the recomputed state
    back = C * (3 + (1 if case["gate"] else 0)) + 2 * G * N
    return dict(bytes=T * B * (row + back) * e + state + 2 * par, flops=n * (28 * N + 8 * K + 40))


# ---- the definitions in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return dict(norm=_exact_norm, ffn=_exact_ffn, scan=_exact_scan, step=_exact_step)[case["kind"]](s, case)


def _leaf(t):
    return None if t is None else t.detach().double().clone().requires_grad_(True)


def _exact_norm(s, case):
    x, w, b = _leaf(s["x"]), _leaf(s["w"]), _leaf(s["b"])
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    y = (x - mean) * torch.rsqrt(var + 1e-5) * w + b
    if not case["train"]:
        return y.detach()
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return dict(y=y.detach(), dx=gx, dw=gw, db=gb)


def _exact_ffn(s, case):
    x, wi, wo = _leaf(s["x"]), _leaf(s["w_in"]), _leaf(s["w_out"])
    gate, value = x @ wi[0::2].t(), x @ wi[1::2].t()
    gate = gate * torch.sigmoid(gate) if case["act"] == "silu" else gate * torch.special.ndtr(gate)
    y = (gate * value) @ wo.t()
    if not case["train"]:
        return y.detach()
    gx, gi, go = torch.autograd.grad(y, (x, wi, wo), s["dy"].double())
    return dict(y=y.detach(), dx=gx, dw_in=gi, dw_out=go)


def _sequence(p, T, K, N, G, done, first):
    """The recurrence step by step; p: the 64-bit leaves, time-major."""
    B, C = p["x"].shape[1:]
    h, win, ys = p["h"], [p["win"][:, i] for i in range(K - 1)] if K > 1 else [], []
    for t in range(T):
        new = first if t == 0 else (done[t - 1] if done is not None else None)
        if new is not None:
            alive = (1 - new)[:, None]
            h, win = h * alive[..., None], [v * alive for v in win]
        u = p["x"][t]
        if K:
            seen = win + [u]
            c = p["conv_b"] + sum(v * p["conv_w"][:, i] for i, v in enumerate(seen))
            u, win = c * torch.sigmoid(c), seen[1:]
        d = torch.nn.functional.softplus(p["delta"][t] + p["dt_bias"], threshold=1000.0)
        Bt, Ct = (p[k][t].view(B, G, N).repeat_interleave(C // G, dim=1) for k in ("Bm", "Cm"))
        h = torch.exp(d.unsqueeze(-1) * p["A"]) * h + (d * u).unsqueeze(-1) * Bt
        y = (h * Ct).sum(-1) + p["D"] * u
        if p["z"] is not None:
            y = y * p["z"][t] * torch.sigmoid(p["z"][t])
        ys.append(y)
    return torch.stack(ys), h, torch.stack(win, 1) if win else None


_LEAVES = ("x", "delta", "Bm", "Cm", "z", "A", "D", "dt_bias", "conv_w", "conv_b")


def _exact_scan(s, case):
    if case["T"] > 16384 or (case["train"] and case["T"] * case["B"] * case["C"] * case["N"] > 1 << 30):
        return None
    p = {k: _leaf(s[k]) if case["train"] else (None if s[k] is None else s[k].double()) for k in _LEAVES}
    p["h"], p["win"] = s["h"].double(), None if s["win"] is None else s["win"].double()
    y, h, win = _sequence(p, case["T"], case["K"], case["N"], case["G"],
                          None if s["done"] is None else s["done"].double(), s["first"].double())
    out = dict(y=y.detach(), h=h.detach(), win=None if win is None else win.detach())
    if case["train"]:
        have = [k for k in _LEAVES if p[k] is not None]
        out.update(zip(("d" + k for k in have), torch.autograd.grad(y, [p[k] for k in have], s["dy"].double())))
    return out


def _exact_step(s, case):
    p = {k: None if s[k] is None else s[k].double() for k in _LEAVES}
    for k in ("x", "delta", "Bm", "Cm", "z"):
        p[k] = None if p[k] is None else p[k][None]
    p["h"], p["win"] = s["h"].double(), None if s["win"] is None else s["win"].double()
    y, h, win = _sequence(p, 1, case["K"], case["N"], case["G"], None, s["first"].double())
    return dict(y=y[0], h=h, win=win)
