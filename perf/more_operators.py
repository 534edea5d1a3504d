"""The operators of a delta-rule policy layer: the gated delta rule (sequences, their gradient, and single tokens), RMS
normalisation fused with the residual sum in front of it or the gate behind it, and the draw from filtered logits.

``listed()`` names the cases whose time counts, ``draw(rng)`` makes more of the same ranges, ``prepare`` builds what a
program holds before the call, ``run`` is one pass, ``work`` the bytes and operations that no implementation can
avoid, and ``exact`` the outputs from the definitions in 64 bits. ``own`` chooses between the plain form (elementary
torch operations in fp32, the draw's masses in fp64, rounded once at the end) and the library's kernels.

Sequences are time-major, [T, B, ...], as everywhere in this library; the inputs of the delta rule are column slices of one
projection's output, [q | k | v | a | b], as the layer in front of it leaves them.
"""
from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # a minibatch of short segments with episode ends at width 512, both directions (the largest call)
        dict(name="delta_train_64x2048_h8x64", kind="delta", T=64, B=2048, Hk=8, H=8, K=64, V=64, dtype="bf16", done=True,
             train=True),
        # long sequences in training, two value heads to a key head
        dict(name="delta_train_2048x8_h4x128", kind="delta", T=2048, B=8, Hk=2, H=4, K=128, V=128, dtype="bf16", done=True,
             train=True),
        # odd everything in fp32, three value heads to a key head
        dict(name="delta_train_33x203_h3_f32", kind="delta", T=33, B=203, Hk=1, H=3, K=24, V=41, dtype="f32", done=True,
             train=True),
        # a long prompt of a few sequences: one block per sequence and head would leave the chip idle
        dict(name="delta_8192x2_h8x64", kind="delta", T=8192, B=2, Hk=8, H=8, K=64, V=64, dtype="bf16", done=False,
             train=False),
        # one environment step of the rollout, the state carried in fp32
        dict(name="delta_step_4096_h8x64", kind="step", B=4096, Hk=8, H=8, K=64, V=64, dtype="bf16"),
        # a few environments of a small policy (latency)
        dict(name="delta_step_48_h2x32_f32", kind="step", B=48, Hk=2, H=2, K=32, V=32, dtype="f32"),
        # one rollout step of a few environments: residual sum and norm (latency)
        dict(name="rms_48x128_f32", kind="rms", M=48, G=1, C=128, dtype="f32", add=True, scale=False, gate=False,
             train=False),
        # the residual stream of a minibatch of 4096 segments x 64 steps at width 512, with a scale per column
        dict(name="rms_train_262144x512", kind="rms", M=262144, G=1, C=512, dtype="bf16", add=True, scale=True, gate=False,
             train=True),
        # behind the delta rule: each head's output normalised and gated
        dict(name="rms_train_131072x8x64_gate", kind="rms", M=131072, G=8, C=512, dtype="bf16", add=False, scale=False,
             gate=True, train=True),
        # the actions of one rollout step of a few environments, some of them not allowed (latency)
        dict(name="draw_48x18_f32", kind="draw", N=48, A=18, dtype="f32", masked=True),
        # a large action set
        dict(name="draw_4096x1000_f32", kind="draw", N=4096, A=1000, dtype="f32", masked=True),
        # a vocabulary
        dict(name="draw_64x131072", kind="draw", N=64, A=131072, dtype="bf16", masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _even(rng, v):
    """Two draws in three have the multiples of eight that a policy's widths are; the others are odd."""
    return max(8, v // 8 * 8) if rng.random() < 0.67 else v | 1


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "step", "rms", "rms", "draw", "draw"])
    dt = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("delta", "step"):
        Hk, rep = rng.choice([1, 1, 2, 2, 4, 8]), rng.choice([1, 1, 1, 2, 3])
        c = dict(kind=kind, Hk=Hk, H=Hk * rep, K=min(128, _even(rng, _log(rng, 8, 128))),
                 V=min(128, _even(rng, _log(rng, 8, 128))), dtype=dt)
        if kind == "step":
            return dict(c, B=_log(rng, 1, 4096 // max(1, c["H"] // 8)))
        c.update(T=_log(rng, 2, 8192), B=_log(rng, 1, 2048), done=rng.random() < 0.6, train=rng.random() < 0.6)
        if c["train"]:
            c["T"] = min(c["T"], 4096)
        while c["T"] * c["B"] * c["H"] * c["K"] * c["V"] > (1 << 32 if dt == "bf16" else 1 << 30):
            big = "T" if c["T"] > c["B"] else "B"
            c[big] = (c[big] + 1) // 2
        return c
    if kind == "rms":
        form = rng.choice(["add", "scale", "gate", "heads", "all"])
        G = rng.choice([2, 4, 8]) if form == "heads" else 1
        c = dict(kind=kind, M=_log(rng, 1, 262144), G=G, C=G * _even(rng, _log(rng, 8, 2048) // G), dtype=dt,
                 add=form in ("add", "scale", "all"), scale=form in ("scale", "all"), gate=form in ("gate", "heads", "all"),
                 train=rng.random() < 0.7)
        while c["M"] * c["C"] > 1 << 27:
            c["M"] //= 2
        return c
    c = dict(kind=kind, N=_log(rng, 1, 8192), A=_log(rng, 2, 131072), dtype=dt, masked=rng.random() < 0.5)
    while c["N"] * c["A"] > 1 << 23:
        c["N"] //= 2
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
    if case["kind"] == "rms":
        M, C = case["M"], case["C"]
        s["x"] = (normal(M, C) * (0.5 + uniform(M, 1))).to(dt)
        s["add"] = normal(M, C, scale=0.5, dtype=dt) if case["add"] else None
        s["scale"] = 0.5 + normal(C, scale=0.1) if case["scale"] else None
        s["gate"] = normal(M, C, dtype=dt) if case["gate"] else None
        s["w"] = 1 + normal(C // case["G"], scale=0.1)
        if case["train"]:
            s["dout"] = normal(M, C, dtype=dt)
            s["dres"] = normal(M, C, dtype=dt) if case["add"] else None  # what comes down the residual stream
        return s
    if case["kind"] == "draw":
        N, A = case["N"], case["A"]
        s["logits"] = normal(N, A, scale=2.0, dtype=dt)
        if case["masked"]:  # actions that are not allowed; a row in fifty has none
            s["logits"].masked_fill_((uniform(N, A) < 0.3) | (uniform(N, 1) < 0.02), -math.inf)
        s["u"] = uniform(N)
        pick = uniform(4, N)
        s["temperature"] = torch.where(pick[0] < 0.1, 0.0, 0.5 + uniform(N))  # one row in ten is greedy
        s["top_k"] = torch.where(pick[1] < 0.5, 0, (uniform(N) * min(A, 64)).long() + 1).int()
        s["top_p"] = torch.where(pick[2] < 0.3, 1.0, 0.7 + 0.3 * uniform(N))
        s["min_p"] = torch.where(pick[3] < 0.5, 0.0, 0.1 * uniform(N))
        return s
    Hk, H, K, V = case["Hk"], case["H"], case["K"], case["V"]
    T, B = case.get("T", 1), case["B"]
    lead = (T, B) if case["kind"] == "delta" else (B,)
    parts = [Hk * K, Hk * K, H * V, H, H]
    q, k, v, s["a"], s["b"] = normal(*lead, sum(parts), dtype=dt).split(parts, dim=-1)
    s["q"], s["k"], s["v"] = q.unflatten(-1, (Hk, K)), k.unflatten(-1, (Hk, K)), v.unflatten(-1, (H, V))
    s["A"] = -(1 + 15 * uniform(H))
    dt0 = torch.exp(uniform(H) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))  # time steps of 1e-3 to 1e-1
    s["dt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
    s["h"] = normal(B, H, K, V, scale=0.2)
    s["done"] = (uniform(T, B) < 0.05).float() if case.get("done") else None
    s["first"] = (uniform(B) < 0.1).float()
    if case.get("train"):
        s["dy"] = normal(T, B, H, V, dtype=dt)
    return s


# ---- one pass ----------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)[case["kind"]](s, case)


def _own_delta(s, case):
    from pufferlean_amd import device as D
    ins = (s["q"], s["k"], s["v"], s["a"], s["b"], s["A"])
    kw = dict(dt_bias=s["dt_bias"], done=s["done"], first=s["first"])
    h = torch.empty_like(s["h"])
    out = D.delta_scan(*ins, h0=s["h"], h_out=h, save=case["train"], **kw)
    if not case["train"]:
        return dict(y=out, h=h)
    y, saved = out
    # the gradients go where the projection's backward pass reads them: one buffer of the same columns
    T, B, Hk, K = s["q"].shape
    H, V = s["v"].shape[2:]
    parts = [Hk * K, Hk * K, H * V, H, H]
    dq, dk, dv, da, db = torch.empty(T, B, sum(parts), device=y.device, dtype=y.dtype).split(parts, dim=-1)
    grads = D.delta_scan_grad(*ins, saved, s["dy"], dq=dq.unflatten(-1, (Hk, K)), dk=dk.unflatten(-1, (Hk, K)),
                              dv=dv.unflatten(-1, (H, V)), da=da, db=db, **kw)
    return dict(y=y, h=h, **grads)


def _own_step(s, case):
    from pufferlean_amd import device as D
    y = D.delta_step(s["q"], s["k"], s["v"], s["a"], s["b"], s["A"], s["h"], dt_bias=s["dt_bias"], first=s["first"])
    return dict(y=y, h=s["h"])


def _own_rms(s, case):
    from pufferlean_amd import device as D
    kw = dict(add=s["add"], scale=s["scale"], gate=s["gate"], groups=case["G"])
    out, res, rstd = D.rms_norm(s["x"], s["w"], **kw)
    o = dict(out=out, res=res)
    if case["train"]:
        o.update(D.rms_norm_grad(s["x"], s["w"], rstd, s["dout"], dres=s["dres"], **kw))
    return o


def _own_draw(s, case):
    from pufferlean_amd import device as D
    act, logp = D.sample_filtered(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                  min_p=s["min_p"])
    return dict(act=act, logp=logp)


QK_EPS = 1e-6


def _unit(x):
    """Rows of unit length, and the factors that made them so."""
    r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) + QK_EPS)
    return x * r, r


def _unit_grad(n, r, d):
    return r * (d - n * (n * d).sum(-1, keepdim=True))


def _heads(x, H):
    """Rows of key heads for every value head."""
    return x.repeat_interleave(H // x.shape[-2], dim=-2)


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _gates(s):
    arg = s["a"].float() + s["dt_bias"]
    sp = _softplus(arg)
    return arg, sp, torch.exp(s["A"] * sp), 1 / (1 + torch.exp(-s["b"].float()))


def _plain_delta(s, case):
    dt, H, Hk, K = s["q"].dtype, case["H"], case["Hk"], case["K"]
    T, B = s["q"].shape[:2]
    qn, qr = _unit(s["q"].float())
    kn, kr = _unit(s["k"].float())
    q, k, v = _heads(qn, H), _heads(kn, H), s["v"].float()
    arg, sp, al, be = _gates(s)
    keep = torch.ones(T, B, device=v.device)
    keep[0] -= s["first"]
    if s["done"] is not None:
        keep[1:] -= s["done"][:-1]
    scale, train = K ** -0.5, case["train"]
    S, states, errs, y = s["h"], [], [], torch.empty_like(v)
    for t in range(T):
        if train:
            states.append(S)
        S = S * (al[t] * keep[t][:, None])[..., None, None]
        e = v[t] - (S * k[t][..., None]).sum(-2)
        if train:
            errs.append(e)
        S = S + k[t][..., None] * (be[t][..., None] * e)[..., None, :]
        y[t] = scale * (S * q[t][..., None]).sum(-2)
    out = dict(y=y.to(dt), h=S)
    if not train:
        return out
    dy = s["dy"].float()
    dS = torch.zeros_like(S)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dal, dbe = torch.empty_like(al), torch.empty_like(be)
    for t in reversed(range(T)):
        prev = states.pop()
        dec = (al[t] * keep[t][:, None])[..., None, None]
        e, w = errs.pop(), be[t][..., None]
        d = scale * dy[t]
        dq[t] = (S * d[..., None, :]).sum(-1)
        dS = dS + q[t][..., None] * d[..., None, :]
        du = (dS * k[t][..., None]).sum(-2)  # of the written value be e
        dbe[t] = (du * e).sum(-1)
        de = w * du
        dv[t] = de
        P = prev * dec
        dk[t] = (dS * (w * e)[..., None, :]).sum(-1) - (P * de[..., None, :]).sum(-1)
        dS = dS - k[t][..., None] * de[..., None, :]
        dal[t] = (dS * prev).sum((-1, -2)) * keep[t][:, None]
        dS = dS * dec
        S = prev
    group = (T, B, Hk, H // Hk, K)
    out["dq"] = _unit_grad(qn, qr, dq.view(group).sum(3)).to(dt)
    out["dk"] = _unit_grad(kn, kr, dk.view(group).sum(3)).to(dt)
    out["dv"] = dv.to(dt)
    dsp = dal * al
    out["dA"] = (dsp * sp).sum((0, 1))
    da = dsp * s["A"] / (1 + torch.exp(-arg))
    out["da"], out["ddt_bias"] = da.to(dt), da.sum((0, 1))
    out["db"] = (dbe * be * (1 - be)).to(dt)
    return out


def _plain_step(s, case):
    H, K = case["H"], case["K"]
    q, k, v = _heads(_unit(s["q"].float())[0], H), _heads(_unit(s["k"].float())[0], H), s["v"].float()
    _, _, al, be = _gates(s)
    S = s["h"] * (al * (1 - s["first"])[:, None])[..., None, None]
    e = v - (S * k[..., None]).sum(-2)
    s["h"].copy_(S + k[..., None] * (be[..., None] * e)[..., None, :])
    return dict(y=(K ** -0.5 * (s["h"] * q[..., None]).sum(-2)).to(s["q"].dtype), h=s["h"])


RMS_EPS = 1e-6


def _plain_rms(s, case):
    dt, G = s["x"].dtype, case["G"]
    M, C = s["x"].shape
    x = s["x"].float()
    if s["add"] is not None:
        add = s["add"].float()
        x = x + (add if s["scale"] is None else add * s["scale"])
    rows = x.view(M, G, C // G)
    r = 1 / torch.sqrt((rows * rows).mean(-1, keepdim=True) + RMS_EPS)
    n = rows * r
    o = (n * s["w"]).view(M, C)
    if s["gate"] is not None:
        z = s["gate"].float()
        sg = 1 / (1 + torch.exp(-z))
        out = dict(out=(o * z * sg).to(dt))
    else:
        out = dict(out=o.to(dt))
    out["res"] = x.to(dt) if s["add"] is not None else None
    if not case["train"]:
        return out
    do = s["dout"].float()
    if s["gate"] is not None:
        out["dgate"] = (do * o * sg * (1 + z * (1 - sg))).to(dt)
        do = do * z * sg
    do = do.view(M, G, C // G)
    out["dw"] = (do * n).sum((0, 1))
    dn = do * s["w"]
    dx = (r * (dn - n * (dn * n).mean(-1, keepdim=True))).view(M, C)
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    out["dx"] = dx.to(dt)
    if s["add"] is not None:
        out["dadd"] = (dx if s["scale"] is None else dx * s["scale"]).to(dt)
        if s["scale"] is not None:
            out["dscale"] = (dx * add).sum(0)
    return out


def _plain_draw(s, case):
    """The filters in the order of falling logits (the lower index first), the draw in the order of the indices. Masses in
    64 bits: a draw next to a border may not depend on how they were added."""
    x = s["logits"].double()
    N, A = x.shape
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    best = v[:, :1]
    greedy = s["temperature"] == 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    e = torch.where(v == best, 1.0, torch.exp((v - best) / t)).masked_fill(v == -math.inf, 0.0)
    rank = torch.arange(A, device=x.device)[None]
    k = torch.where((s["top_k"] <= 0) | greedy, torch.where(greedy, 1, A), s["top_k"]).long()[:, None]
    e = e * (rank < k)
    total = e.sum(1, keepdim=True)
    p = s["top_p"].double()[:, None]
    before = torch.cumsum(e, 1) - e
    e = e * ((before < p * total) | (p >= 1) | (rank == 0))
    e = e * (e >= s["min_p"].double()[:, None])
    w = torch.zeros_like(e).scatter_(1, order, e)
    run_sum = torch.cumsum(w, 1)
    total = run_sum[:, -1:]
    hit = (run_sum > s["u"].double()[:, None] * total) & (w > 0)
    last = A - 1 - (w > 0).flip(1).int().argmax(1)
    act = torch.where(hit.any(1), hit.int().argmax(1), last)
    none = best[:, 0] == -math.inf
    logp = torch.log(w.gather(1, act[:, None]) / total)[:, 0]
    return dict(act=torch.where(none, -1, act).int(), logp=torch.where(none, -math.inf, logp).float())


_run_own = dict(delta=_own_delta, step=_own_step, rms=_own_rms, draw=_own_draw)
_run_plain = dict(delta=_plain_delta, step=_plain_step, rms=_plain_rms, draw=_plain_draw)


# ---- the least that each pass needs -------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "rms":
        n = case["M"] * case["C"]
        fwd = 2 + (2 if case["add"] else 0) + (1 if case["gate"] else 0)  # x, out; add, res; gate
        back = 0
        if case["train"]:  # dout, dx; dres (and dadd where it is not dx); dgate
            back = 2 + (1 if case["add"] else 0) + (1 if case["scale"] else 0) + (1 if case["gate"] else 0)
        return dict(bytes=n * e * (fwd + back) + 4 * case["C"], flops=n * (20 if case["train"] else 6))
    if case["kind"] == "draw":
        # each logit read once; an exponential and a few comparisons and sums for each
        return dict(bytes=case["N"] * (case["A"] * e + 28), flops=case["N"] * case["A"] * 8)
    Hk, H, K, V = case["Hk"], case["H"], case["K"], case["V"]
    rows = case.get("T", 1) * case["B"]
    token = 2 * Hk * K + 2 * H * V + 2 * H  # q, k; v, y; a, b
    state = 8 * case["B"] * H * K * V
    # per element of the state: decay, what it holds under k, the update, the output
    f = 7
    if case.get("train"):
        token += 2 * Hk * K + 2 * H * V + 2 * H  # dy in, dq, dk, dv, da, db out
        f = 25  # the state again, and twice the forward's products
    return dict(bytes=rows * token * e + state, flops=rows * H * K * V * f)


# ---- the definitions in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return dict(delta=_exact_delta, step=_exact_step, rms=_exact_rms, draw=_exact_draw)[case["kind"]](s, case)


def _leaf(t):
    return None if t is None else t.detach().double().clone().requires_grad_(True)


def _recurrence(p, H, first, done, h):
    """The rule step by step with matrix products; p: 64-bit leaves, time-major."""
    T, B, Hk, K = p["q"].shape
    qs, ks = (torch.nn.functional.pad(p[n], (0, 1), value=math.sqrt(QK_EPS)) for n in ("q", "k"))
    qs, ks = ((p[n] / m.norm(dim=-1, keepdim=True)) for n, m in (("q", qs), ("k", ks)))
    g = p["A"] * torch.nn.functional.softplus(p["a"] + p["dt_bias"], threshold=1000.0)
    be = torch.sigmoid(p["b"])
    rep, ys = H // Hk, []
    for t in range(T):
        new = first if t == 0 else (None if done is None else done[t - 1])
        if new is not None:
            h = h * (1 - new)[:, None, None, None]
        q, k = (m[t].unsqueeze(2).expand(B, Hk, rep, K).reshape(B, H, 1, K) for m in (qs, ks))
        h = h * torch.exp(g[t])[:, :, None, None]
        u = be[t][:, :, None, None] * (p["v"][t].unsqueeze(2) - torch.matmul(k, h))
        h = h + k.transpose(-1, -2).contiguous() * u
        ys.append(torch.matmul(q, h).squeeze(2) / math.sqrt(K))
    return torch.stack(ys), h


_LEAVES = ("q", "k", "v", "a", "b", "A", "dt_bias")


def _exact_delta(s, case):
    train, H = case["train"], case["H"]
    if case["T"] > 16384:
        return None
    first, done, h0 = s["first"].double(), None if s["done"] is None else s["done"].double(), s["h"].double()
    # some sequences at a time: the graph of a slice holds a few states a step
    per_seq = case["T"] * H * case["K"] * case["V"] * 8 * (4 if train else 0) + 1
    n = max(1, min(case["B"], int(16e9 // per_seq)))
    if train and -(-case["B"] // n) * case["T"] > 20000:
        return None
    parts = []
    for i in range(0, case["B"], n):
        sl = slice(i, i + n)
        p = {k: s[k] if s[k].dim() == 1 else s[k][:, sl] for k in _LEAVES}
        p = {k: _leaf(v) if train else v.double() for k, v in p.items()}
        y, h = _recurrence(p, H, first[sl], None if done is None else done[:, sl], h0[sl])
        out = dict(y=y.detach(), h=h.detach())
        if train:
            out.update(zip(("d" + k for k in _LEAVES),
                           torch.autograd.grad(y, list(p.values()), s["dy"][:, sl].double())))
        parts.append(out)
    join = {"h": lambda v: torch.cat(v), "dA": lambda v: sum(v), "ddt_bias": lambda v: sum(v)}
    return {k: join.get(k, lambda v: torch.cat(v, 1))([o[k] for o in parts]) for k in parts[0]}


def _exact_step(s, case):
    p = {k: s[k].double() if s[k].dim() == 1 else s[k].double()[None] for k in _LEAVES}
    y, h = _recurrence(p, case["H"], s["first"].double(), None, s["h"].double())
    return dict(y=y[0], h=h)


def _exact_rms(s, case):
    M, C = s["x"].shape
    G = case["G"]
    x, add, scale, gate, w = (_leaf(s[k]) for k in ("x", "add", "scale", "gate", "w"))
    r = x if add is None else (x + add if scale is None else torch.addcmul(x, add, scale))
    rows = r.reshape(M * G, C // G)
    n = math.sqrt(C // G) * rows / torch.sqrt(rows.square().sum(1, keepdim=True) + RMS_EPS * (C // G))
    o = (n * w).reshape(M, C)
    if gate is not None:
        o = o * gate * torch.sigmoid(gate)
    out = dict(out=o.detach(), res=None if add is None else r.detach())
    if not case["train"]:
        return out
    obj = (o * s["dout"].double()).sum()
    if s["dres"] is not None:
        obj = obj + (r * s["dres"].double()).sum()
    have = [(k, t) for k, t in (("dgate", gate), ("dw", w), ("dx", x), ("dadd", add), ("dscale", scale)) if t is not None]
    out.update(zip((k for k, _ in have), torch.autograd.grad(obj, [t for _, t in have])))
    return out


def _exact_draw(s, case):
    """Row by row on the host: what the filters leave as a set of indices."""
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    par = {k: s[k].cpu().numpy() for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    N, A = x.shape
    act, logp = np.full(N, -1, np.int32), np.full(N, -np.inf)
    for i in range(N):
        row = x[i]
        top = row.max()
        if top == -np.inf:
            continue
        if par["temperature"][i] == 0:
            act[i], logp[i] = int(row.argmax()), 0.0
            continue
        mass = np.exp((row - top) / float(par["temperature"][i]))
        left = np.lexsort((np.arange(A), -row))
        left = left[mass[left] > 0]
        if 0 < par["top_k"][i] < left.size:
            left = left[:par["top_k"][i]]
        if par["top_p"][i] < 1:
            got = np.cumsum(mass[left])
            left = left[:int(np.searchsorted(got, float(par["top_p"][i]) * got[-1])) + 1]
        left = np.sort(left[mass[left] >= float(par["min_p"][i])])
        got = np.cumsum(mass[left])
        at = min(int(np.searchsorted(got, float(par["u"][i]) * got[-1], side="right")), left.size - 1)
        act[i] = left[at]
        logp[i] = np.log(mass[left[at]] / got[-1])
    return dict(act=torch.from_numpy(act), logp=torch.from_numpy(logp))
