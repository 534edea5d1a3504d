"""A recurrent actor-critic policy of state-space layers over the library's device operators.

Each layer is two residual blocks on rows of width H: normalisation, one projection to [x | z | delta | B | C], the selective
scan with its short convolution, a projection back; then normalisation and the gated feed-forward block. An encoder in front,
a normalisation and one head of A logits and the value behind. Time-major [T, B] columns, as the trainer's: `ppo_grad`
runs a minibatch of whole segments forward and backward, `step` one environment step with the carried state.

Weights are fp32 masters; products and activations run in bf16 (or fp32), the scan's parameters, the normalisations and all
states in fp32. Matrices are stepped by Muon, vectors by Nesterov momentum, as the other policies' are.
"""
from __future__ import annotations

import math

import torch

from . import _lib as L
from . import device as D


class SSMPolicy:
    """Parameters (a dict of fp32 tensors on `device`, key -> tensor) and the passes over them."""

    def __init__(self, obs, actions, *, width=128, inner=128, states=16, taps=4, ffn=344, layers=2, act="silu",
                 dtype=torch.bfloat16, device="cuda", seed=0):
        self.obs, self.A, self.H, self.C, self.N, self.K, self.F = obs, actions, width, inner, states, taps, ffn
        self.layers, self.act, self.dtype = layers, act, dtype
        self.parts = [inner, inner, inner, states, states]  # x, z, delta, B, C
        g = torch.Generator().manual_seed(seed)

        def mat(r, c, scale=1.0):
            return (torch.randn(r, c, generator=g) * (scale / math.sqrt(c))).to(device)

        p = dict(enc=mat(width, obs), enc_b=torch.zeros(width, device=device))
        for i in range(layers):
            dt = torch.exp(torch.rand(inner, generator=g) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
            p.update({f"{i}.n1w": torch.ones(width, device=device), f"{i}.n1b": torch.zeros(width, device=device),
                      f"{i}.in": mat(sum(self.parts), width), f"{i}.out": mat(width, inner),
                      f"{i}.A_log": torch.log(1 + torch.arange(states).float()).repeat(inner, 1).to(device),
                      f"{i}.D": torch.ones(inner, device=device),
                      f"{i}.dt_bias": (dt + torch.log(-torch.expm1(-dt))).to(device),
                      f"{i}.conv_w": (torch.randn(inner, taps, generator=g) / math.sqrt(taps)).to(device),
                      f"{i}.conv_b": torch.zeros(inner, device=device),
                      f"{i}.n2w": torch.ones(width, device=device), f"{i}.n2b": torch.zeros(width, device=device),
                      f"{i}.ffn_in": mat(2 * ffn, width), f"{i}.ffn_out": mat(width, ffn)})
        p.update(nw=torch.ones(width, device=device), nb=torch.zeros(width, device=device),
                 head=mat(actions + 1, width, 0.1), head_b=torch.zeros(actions + 1, device=device))
        self.p = {k: v.contiguous() for k, v in p.items()}
        self.mom = {k: torch.zeros_like(v) for k, v in self.p.items()}

    # ---- pieces ------------------------------------------------------------------------------------
    def _math(self):
        return "bf16" if self.dtype is torch.bfloat16 else "f32"

    def _weights(self):
        """The matrices that the products read, in the compute dtype."""
        if self.dtype is torch.float32:
            return self.p
        w = dict(self.p)
        for k, v in self.p.items():
            if v.dim() == 2 and not k.endswith(("A_log", "conv_w", "enc", "head")):
                w[k] = D.convert(v, self.dtype)
        return w

    def _nt(self, x, w, out_dtype=None, aux=None):
        """x w^T (+ aux)."""
        epi = dict(epilogue=L.PH_EPI_AXPBY, aux=aux, alpha=1.0, beta=1.0) if aux is not None else {}
        return D.gemm(x, w, trans_b=True, out_dtype=out_dtype or self.dtype, math=self._math(), **epi)

    def _scan_args(self, w, i, cols, done, first):
        x, z, d, Bm, Cm = cols.split(self.parts, dim=-1)
        args = (x, d, -torch.exp(w[f"{i}.A_log"]), Bm, Cm)
        return args, dict(D=w[f"{i}.D"], z=z, dt_bias=w[f"{i}.dt_bias"], conv_w=w[f"{i}.conv_w"], conv_b=w[f"{i}.conv_b"],
                          first=first, **({} if done is None else dict(done=done)))

    def _encode(self, obs):
        return D.gemm(obs, self.p["enc"], trans_b=True, out_dtype=self.dtype, math=self._math(), epilogue=L.PH_EPI_BIAS,
                      bias=self.p["enc_b"])

    def _head(self, x):
        return D.gemm(x, self.p["head"], trans_b=True, out_dtype=torch.float32, math=self._math(), epilogue=L.PH_EPI_BIAS,
                      bias=self.p["head_b"])

    # ---- rollout -----------------------------------------------------------------------------------
    def state(self, B):
        """The cleared state of B environments: per layer (h, window)."""
        dev = self.p["enc"].device
        return [(torch.zeros(B, self.C, self.N, device=dev), torch.zeros(B, self.K - 1, self.C, device=dev) if self.K > 1 else None)
                for _ in range(self.layers)]

    def step(self, obs, state, first=None):
        """One environment step: obs fp32 [B, obs], the state updated in place (cleared first where first[b] is set).
        Returns the head outputs fp32 [B, A + 1] (logits, value)."""
        w = self._weights()
        x = self._encode(obs)
        for i, (h, win) in enumerate(state):
            n, _, _ = D.layer_norm(x, w[f"{i}.n1w"], w[f"{i}.n1b"])
            args, kw = self._scan_args(w, i, self._nt(n, w[f"{i}.in"]), None, first)
            x = self._nt(D.ssm_step(*args, h, win, **kw), w[f"{i}.out"], aux=x)
            n, _, _ = D.layer_norm(x, w[f"{i}.n2w"], w[f"{i}.n2b"])
            x = x + D.gated_ffn(n, w[f"{i}.ffn_in"], w[f"{i}.ffn_out"], act=self.act)
        return self._head(D.layer_norm(x, w["nw"], w["nb"])[0])

    # ---- training ----------------------------------------------------------------------------------
    def forward(self, obs, done=None, first=None, state=None, save=False):
        """Whole segments: obs fp32 [T, B, obs], done fp32 [T, B] (step t ends an episode), first fp32 [B], state as
        `state` gives it (updated in place; None: cleared, not returned). Returns the head outputs [T, B, A + 1], with
        save=True also what `backward` needs."""
        T, B, _ = obs.shape
        w, tape = self._weights(), []
        x = self._encode(obs.reshape(T * B, -1))
        for i in range(self.layers):
            x0 = x
            n1, m1, r1 = D.layer_norm(x, w[f"{i}.n1w"], w[f"{i}.n1b"])
            cols = self._nt(n1, w[f"{i}.in"]).view(T, B, -1)
            args, kw = self._scan_args(w, i, cols, done, first)
            h, win = state[i] if state is not None else (None, None)
            win0 = None if win is None else win.clone()  # the gradient's: the scan overwrites the carried one
            out = D.ssm_scan(*args, h0=h, win0=win, h_out=h, win_out=win, save=save, **kw)
            s, kept = out if save else (out, None)
            x1 = self._nt(s.view(T * B, -1), w[f"{i}.out"], aux=x0)
            n2, m2, r2 = D.layer_norm(x1, w[f"{i}.n2w"], w[f"{i}.n2b"])
            f = D.gated_ffn(n2, w[f"{i}.ffn_in"], w[f"{i}.ffn_out"], act=self.act, save=save)
            x = x1 + (f[0] if save else f)
            if save:
                tape.append((x0, n1, m1, r1, args, kw, kept, win0, s, x1, n2, m2, r2, f[1]))
        nf, mf, rf = D.layer_norm(x, w["nw"], w["nb"])
        out = self._head(nf).view(T, B, -1)
        return (out, (obs, w, tape, x, nf, mf, rf)) if save else out

    def _tn(self, a, b):
        """a^T b in fp32: a weight's gradient."""
        return D.gemm(a, b, trans_a=True, out_dtype=torch.float32, math=self._math())

    def backward(self, saved, dout):
        """Gradient of sum(dout * outputs), dout fp32 [T, B, A + 1]: a dict like the parameters'."""
        obs, w, tape, x, nf, mf, rf = saved
        T, B, _ = dout.shape
        g, rows = {}, T * B
        dout = dout.reshape(rows, -1)
        g["head"], g["head_b"] = self._tn(dout, nf.float()), D.colsum(dout)
        dn = D.gemm(dout, self.p["head"], out_dtype=self.dtype, math=self._math())
        dx, g["nw"], g["nb"] = D.layer_norm_grad(x, w["nw"], mf, rf, dn)
        for i in reversed(range(self.layers)):
            x0, n1, m1, r1, args, kw, kept, win0, s, x1, n2, m2, r2, kf = tape[i]
            dn, g[f"{i}.ffn_in"], g[f"{i}.ffn_out"] = D.gated_ffn_grad(n2, w[f"{i}.ffn_in"], w[f"{i}.ffn_out"], kf, dx,
                                                                       act=self.act, dw_dtype=torch.float32)
            dn, g[f"{i}.n2w"], g[f"{i}.n2b"] = D.layer_norm_grad(x1, w[f"{i}.n2w"], m2, r2, dn)
            dx = dx + dn
            g[f"{i}.out"] = self._tn(dx, s.view(rows, -1))
            ds = D.gemm(dx, w[f"{i}.out"], out_dtype=self.dtype, math=self._math()).view(T, B, -1)
            dcols = torch.empty(T, B, sum(self.parts), device=dx.device, dtype=self.dtype)
            ddx, dz, dd, dB, dC = dcols.split(self.parts, dim=-1)
            gs = D.ssm_scan_grad(*args, kept, ds, win0=win0, dx=ddx, dz=dz, ddelta=dd, dBm=dB, dCm=dC, **kw)
            g[f"{i}.A_log"] = gs["dA"] * args[2]  # A = -exp(A_log)
            for k, n in (("D", "dD"), ("dt_bias", "ddt_bias"), ("conv_w", "dconv_w"), ("conv_b", "dconv_b")):
                g[f"{i}.{k}"] = gs[n]
            dcols = dcols.view(rows, -1)
            g[f"{i}.in"] = self._tn(dcols, n1)
            dn = D.gemm(dcols, w[f"{i}.in"], out_dtype=self.dtype, math=self._math())
            dn, g[f"{i}.n1w"], g[f"{i}.n1b"] = D.layer_norm_grad(x0, w[f"{i}.n1w"], m1, r1, dn)
            dx = dx + dn
        dx = dx.float()
        g["enc"], g["enc_b"] = self._tn(dx, obs.reshape(rows, -1)), D.colsum(dx)
        return g

    def ppo_grad(self, obs, act, adv, ret, old, ov=None, *, done=None, first=None, state=None, vf_coef=0.5, ent_coef=0.01,
                 clip_eps=0.2, vf_clip=0.0, losses=None):
        """Gradient of the clipped PPO objective (ascent sign, summed over the rows) of one minibatch of segments, as a dict
        like the parameters'. act int32, adv, ret, old (and ov) fp32, all [T, B]."""
        out, saved = self.forward(obs, done, first, state, save=True)
        T, B, W = out.shape
        rows = out.view(T * B, W)
        dout = torch.empty_like(rows)
        D.ppo_grad(rows[:, :self.A], rows[:, self.A], act.reshape(-1), adv.reshape(-1), ret.reshape(-1), old.reshape(-1),
                   None if ov is None else ov.reshape(-1), vf_coef=vf_coef, ent_coef=ent_coef, clip_eps=clip_eps, vf_clip=vf_clip,
                   dlogits=dout[:, :self.A], dvalues=dout[:, self.A], losses=losses)
        return self.backward(saved, dout.view(T, B, W))

    def update(self, grads, *, lr=0.015, scale=1.0, math="bf16"):
        """Muon on every matrix of a product, Nesterov momentum on the rest, in place."""
        for k, p in self.p.items():
            g = grads[k].contiguous()
            if p.dim() == 2 and not k.endswith(("A_log", "conv_w")):
                D.muon_mat(p, g, self.mom[k], gscale=scale, lr=lr, math=math)
            else:
                D.stepvec(p, g, self.mom[k], gscale=scale, lr=lr)
        D.ns_status()
