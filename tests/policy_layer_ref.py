"""The state-space policy layer's operators from their definitions, in 64 bits on the host, step by step; gradients by
torch's automatic differentiation of these loops."""
import torch

# relative 2-norm bars. bf16 results are fp32 results rounded once, by at most half a unit of eight significant bits: the
# unit of 1.x is 2^-7, half of it 2^-8.
BF16 = 2.0 ** -8


def rel(x, ref):
    x, ref = x.detach().double().cpu(), ref.detach().double().cpu()
    assert x.shape == ref.shape, (x.shape, ref.shape)
    n = ref.norm()
    return float((x - ref).norm() / n) if n > 0 else float((x - ref).norm())


def leaf(t):
    return None if t is None else t.detach().double().cpu().clone().requires_grad_(True)


def layer_norm(x, w, b, eps=1e-5):
    mu = x.mean(1, keepdim=True)
    n = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
    if w is not None:
        n = n * w
    return n if b is None else n + b


def glu(a, v, act):
    return (a / (1 + torch.exp(-a)) if act == "silu" else 0.5 * a * (1 + torch.erf(a / 2 ** 0.5))) * v


def ffn(x, w_in, w_out, act):
    return glu(x @ w_in[0::2].T, x @ w_in[1::2].T, act) @ w_out.T


def scan(p, groups=1, done=None, first=None, h0=None, win0=None):
    """p: x, delta, Bm, Cm [T, B, .], A, and maybe z, D, dt_bias, conv_w, conv_b, all float64. A cleared state is a new
    zero tensor, so that nothing of the episode before reaches it. Returns y, the state and the window."""
    x, A, cw = p["x"], p["A"], p.get("conv_w")
    T, B, C = x.shape
    N, K = A.shape[1], 0 if cw is None else cw.shape[1]
    seqs = []
    for b in range(B):
        h = torch.zeros(C, N, dtype=torch.float64) if h0 is None else h0[b]
        win = [torch.zeros(C, dtype=torch.float64)] * max(0, K - 1) if win0 is None else list(win0[b])
        ys = []
        for t in range(T):
            if (first is not None and first[b] != 0) if t == 0 else (done is not None and done[t - 1, b] != 0):
                h, win = torch.zeros(C, N, dtype=torch.float64), [torch.zeros(C, dtype=torch.float64)] * max(0, K - 1)
            u = x[t, b]
            if K:
                seen = win + [u]
                c = sum(seen[k] * cw[:, k] for k in range(K))
                if p.get("conv_b") is not None:
                    c = c + p["conv_b"]
                u, win = c / (1 + torch.exp(-c)), seen[1:]
            v = p["delta"][t, b] if p.get("dt_bias") is None else p["delta"][t, b] + p["dt_bias"]
            d = torch.logaddexp(v, torch.zeros_like(v))
            Bt = p["Bm"][t, b].view(groups, 1, N).expand(groups, C // groups, N).reshape(C, N)
            Ct = p["Cm"][t, b].view(groups, 1, N).expand(groups, C // groups, N).reshape(C, N)
            h = torch.exp(d[:, None] * A) * h + (d * u)[:, None] * Bt
            y = (h * Ct).sum(1)
            if p.get("D") is not None:
                y = y + p["D"] * u
            if p.get("z") is not None:
                y = y * p["z"][t, b] / (1 + torch.exp(-p["z"][t, b]))
            ys.append(y)
        seqs.append((torch.stack(ys), h, torch.stack(win) if win else torch.zeros(0, C, dtype=torch.float64)))
    return torch.stack([s[0] for s in seqs], 1), torch.stack([s[1] for s in seqs]), torch.stack([s[2] for s in seqs])
