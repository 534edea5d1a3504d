"""The delta-rule policy layer's operators from their definitions, in 64 bits on the host; gradients by torch's automatic
differentiation of the loop over the steps."""
import numpy as np
import torch

BF16 = 2.0 ** -8  # one rounding of a bf16 result, relative


def unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def delta(p, scale=None, done=None, first=None, h0=None, units=None):
    """p: q, k [T, B, Hk, K], v [T, B, H, V], a, b [T, B, H], A, and maybe dt_bias, all float64. A cleared state is a new zero
    tensor. Returns y [T, B, H, V] and the state [B, H, K, V]; units (a dict) receives the unit rows."""
    q, k, v = unit(p["q"]), unit(p["k"]), p["v"]
    if units is not None:
        units.update(q=q, k=k)
    T, B, Hk, K = q.shape
    H, V = v.shape[2:]
    q, k = (m.repeat_interleave(H // Hk, dim=2) for m in (q, k))
    arg = p["a"] if p.get("dt_bias") is None else p["a"] + p["dt_bias"]
    al = torch.exp(p["A"] * torch.logaddexp(arg, torch.zeros_like(arg)))
    be = 1 / (1 + torch.exp(-p["b"]))
    seqs = []
    for b in range(B):
        S = torch.zeros(H, K, V, dtype=torch.float64) if h0 is None else h0[b]
        ys = []
        for t in range(T):
            if (first is not None and first[b] != 0) if t == 0 else (done is not None and done[t - 1, b] != 0):
                S = torch.zeros(H, K, V, dtype=torch.float64)
            S = al[t, b][:, None, None] * S
            e = be[t, b][:, None] * (v[t, b] - (S * k[t, b][:, :, None]).sum(1))
            S = S + k[t, b][:, :, None] * e[:, None, :]
            ys.append((K ** -0.5 if scale is None else scale) * (S * q[t, b][:, :, None]).sum(1))
        seqs.append((torch.stack(ys), S))
    return torch.stack([s[0] for s in seqs], 1), torch.stack([s[1] for s in seqs])


def rms(x, w=None, add=None, scale=None, gate=None, groups=1, eps=1e-6):
    r = x
    if add is not None:
        r = x + (add if scale is None else add * scale)
    M, C = r.shape
    g = r.view(M, groups, C // groups)
    n = g / torch.sqrt((g * g).mean(-1, keepdim=True) + eps)
    o = (n if w is None else n * w).reshape(M, C)
    return (o if gate is None else o * gate / (1 + torch.exp(-gate))), r


def filtered(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One row of float64 logits: (index, log-probability, how near u or p was to a border, relative to the total)."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    t, p, m = (d if v is None or np.isnan(v) else float(v) for v, d in ((temperature, 1.0), (top_p, 1.0), (min_p, 0.0)))
    t = t if t >= 0 else 1.0
    if x.max() == -np.inf:
        return -1, -np.inf, 1.0
    order = np.lexsort((np.arange(len(x)), -x))  # by falling logit, of equal ones by index
    order = order[x[order] > -np.inf]
    if t == 0 or p <= 0:
        return int(order[0]), 0.0, 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        mass = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / t))
    if top_k is not None and top_k > 0:
        order = order[:top_k]
    near = 1.0
    if p < 1:
        got = np.cumsum(mass[order])
        if len(set(x[order])) > 1:
            near = float(np.abs(got - p * got[-1]).min() / got[-1])
        order = order[:1 + int(np.sum(got[:-1] < p * got[-1]))]
    order = np.sort(order[mass[order] >= min(m, 1.0)])
    got = np.cumsum(mass[order])
    act = int(order[np.argmax(got > u * got[-1])])
    return act, float(np.log(mass[act] / got[-1])), near
