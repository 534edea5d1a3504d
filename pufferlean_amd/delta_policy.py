"""A recurrent actor-critic policy of delta-rule layers over the library's device operators.

Each layer is two residual blocks on rows of width H: RMS normalisation fused with the residual sum in front of it, one projection to
[q | k | v | z | a | b], the gated delta rule, its heads' outputs normalised and gated by z, a projection back; then the gated
feed-forward block. What a block adds to the residual stream is scaled per column. An encoder in front, a normalisation and one head of
A logits and the value behind. Columns, weights, precision and updates are as in the state-space policy; `act` draws the actions of
a rollout step from the filtered logits.
"""
from __future__ import annotations

import math

import torch

from . import device as D
from .ssm_policy import SSMPolicy


class DeltaPolicy(SSMPolicy):
    """Parameters (a dict of fp32 tensors on `device`, key -> tensor) and the passes over them. `heads` value heads of key and value
    widths K and V share `key_heads` heads of queries and keys."""

    def __init__(self, obs, actions, *, width=128, heads=4, key_heads=None, K=32, V=32, ffn=344, layers=2, act="silu",
                 dtype=torch.bfloat16, device="cuda", seed=0):
        key_heads = heads if key_heads is None else key_heads
        self.obs, self.A, self.H, self.heads, self.key_heads, self.K, self.V, self.F = obs, actions, width, heads, key_heads, K, V, ffn
        self.layers, self.act_fn, self.dtype = layers, act, dtype
        self.parts = [key_heads * K, key_heads * K, heads * V, heads * V, heads, heads]  # q, k, v, z, a, b
        g = torch.Generator().manual_seed(seed)

        def mat(r, c, scale=1.0):
            return (torch.randn(r, c, generator=g) * (scale / math.sqrt(c))).to(device)

        def ones(n):
            return torch.ones(n, device=device)

        p = dict(enc=mat(width, obs), enc_b=torch.zeros(width, device=device))
        for i in range(layers):
            dt = torch.exp(torch.rand(heads, generator=g) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
            p.update({f"{i}.n1w": ones(width), f"{i}.in": mat(sum(self.parts), width), f"{i}.A_log": torch.log(1 + 15 * torch.rand(heads, generator=g)).to(device),
                      f"{i}.dt_bias": (dt + torch.log(-torch.expm1(-dt))).to(device), f"{i}.ow": ones(V), f"{i}.out": mat(width, heads * V),
                      f"{i}.s1": ones(width), f"{i}.n2w": ones(width), f"{i}.ffn_in": mat(2 * ffn, width), f"{i}.ffn_out": mat(width, ffn),
                      f"{i}.s2": ones(width)})
        p.update(nw=ones(width), head=mat(actions + 1, width, 0.1), head_b=torch.zeros(actions + 1, device=device))
        self.p = {k: v.contiguous() for k, v in p.items()}
        self.mom = {k: torch.zeros_like(v) for k, v in self.p.items()}

    # ---- pieces ------------------------------------------------------------------------------------
    def _cols(self, cols):
        """q, k, v by heads, z as rows, a, b: views of the projection's columns [..., sum(parts)]."""
        q, k, v, z, a, b = cols.split(self.parts, dim=-1)
        hk, hv = (self.key_heads, self.K), (self.heads, self.V)
        return q.unflatten(-1, hk), k.unflatten(-1, hk), v.unflatten(-1, hv), z.reshape(-1, z.shape[-1]) if z.dim() == 2 else z.flatten(0, 1), a, b

    def _rule(self, w, i):
        return -torch.exp(w[f"{i}.A_log"]), dict(dt_bias=w[f"{i}.dt_bias"])

    # ---- rollout -----------------------------------------------------------------------------------
    def state(self, B):
        """The cleared state of B environments, per layer."""
        return [torch.zeros(B, self.heads, self.K, self.V, device=self.p["enc"].device) for _ in range(self.layers)]

    def step(self, obs, state, first=None):
        """One environment step: obs fp32 [B, obs], the state updated in place (cleared first where first[b] is set).
        Returns the head outputs fp32 [B, A + 1] (logits, value)."""
        w = self._weights()
        r, add, scale = self._encode(obs), None, None
        for i, h in enumerate(state):
            n, res, _ = D.rms_norm(r, w[f"{i}.n1w"], add=add, scale=scale)
            r = r if res is None else res
            q, k, v, z, a, b = self._cols(self._nt(n, w[f"{i}.in"]))
            A, kw = self._rule(w, i)
            o = D.delta_step(q, k, v, a, b, A, h, first=first, **kw)
            g, _, _ = D.rms_norm(o.view(len(o), -1), w[f"{i}.ow"], gate=z, groups=self.heads)
            n, r, _ = D.rms_norm(r, w[f"{i}.n2w"], add=self._nt(g, w[f"{i}.out"]), scale=w[f"{i}.s1"])
            add, scale = D.gated_ffn(n, w[f"{i}.ffn_in"], w[f"{i}.ffn_out"], act=self.act_fn), w[f"{i}.s2"]
        return self._head(D.rms_norm(r, w["nw"], add=add, scale=scale)[0])

    def act(self, obs, state, u, first=None, **filters):
        """One rollout step: the actions drawn from the numbers u (fp32 [B]) with sample_filtered's filters, their
        log-probabilities and the values, each [B]."""
        out = self.step(obs, state, first)
        act, logp = D.sample_filtered(out[:, :self.A], u, **filters)
        return act, logp, out[:, self.A]

    # ---- training ----------------------------------------------------------------------------------
    def forward(self, obs, done=None, first=None, state=None, save=False):
        """Whole segments: obs fp32 [T, B, obs], done fp32 [T, B] (step t ends an episode), first fp32 [B], state as
        `state` gives it (updated in place; None: cleared, not returned). Returns the head outputs [T, B, A + 1], with
        save=True also what `backward` needs."""
        T, B, _ = obs.shape
        w, tape = self._weights(), []
        r, add, scale = self._encode(obs.reshape(T * B, -1)), None, None
        for i in range(self.layers):
            x1, add1, scale1 = r, add, scale
            n1, res, rs1 = D.rms_norm(r, w[f"{i}.n1w"], add=add, scale=scale)
            r = r if res is None else res
            q, k, v, z, a, b = self._cols(self._nt(n1, w[f"{i}.in"]).view(T, B, -1))
            A, kw = self._rule(w, i)
            kw.update(done=done, first=first)
            h = None if state is None else state[i]
            out = D.delta_scan(q, k, v, a, b, A, h0=h, h_out=h, save=save, **kw)
            o, kept = out if save else (out, None)
            o = o.view(T * B, -1)
            g, _, rs2 = D.rms_norm(o, w[f"{i}.ow"], gate=z, groups=self.heads)
            y = self._nt(g, w[f"{i}.out"])
            x3 = r
            n2, r, rs3 = D.rms_norm(r, w[f"{i}.n2w"], add=y, scale=w[f"{i}.s1"])
            f = D.gated_ffn(n2, w[f"{i}.ffn_in"], w[f"{i}.ffn_out"], act=self.act_fn, save=save)
            add, kf = f if save else (f, None)
            scale = w[f"{i}.s2"]
            if save:
                tape.append((x1, add1, scale1, n1, rs1, (q, k, v, a, b, A), kw, kept, o, z, rs2, g, x3, y, n2, rs3, kf))
        nf, _, rsf = D.rms_norm(r, w["nw"], add=add, scale=scale)
        out = self._head(nf).view(T, B, -1)
        return (out, (obs, w, tape, r, add, scale, nf, rsf)) if save else out

    def backward(self, saved, dout):
        """Gradient of sum(dout * outputs), dout fp32 [T, B, A + 1]: a dict like the parameters'."""
        obs, w, tape, r, add, scale, nf, rsf = saved
        T, B, _ = dout.shape
        g, rows = {}, T * B
        dout = dout.reshape(rows, -1)
        g["head"], g["head_b"] = self._tn(dout, nf.float()), D.colsum(dout)
        dn = D.gemm(dout, self.p["head"], out_dtype=self.dtype, math=self._math())
        d = D.rms_norm_grad(r, w["nw"], rsf, dn, add=add, scale=scale)
        g["nw"] = d["dw"]
        for i in reversed(range(self.layers)):
            x1, add1, scale1, n1, rs1, ins, kw, kept, o, z, rs2, gated, x3, y, n2, rs3, kf = tape[i]
            g[f"{i}.s2"] = d["dscale"]
            dn, g[f"{i}.ffn_in"], g[f"{i}.ffn_out"] = D.gated_ffn_grad(n2, w[f"{i}.ffn_in"], w[f"{i}.ffn_out"], kf, d["dadd"],
                                                                       act=self.act_fn, dw_dtype=torch.float32)
            d = D.rms_norm_grad(x3, w[f"{i}.n2w"], rs3, dn, dres=d["dx"], add=y, scale=w[f"{i}.s1"])
            g[f"{i}.n2w"], g[f"{i}.s1"] = d["dw"], d["dscale"]
            g[f"{i}.out"] = self._tn(d["dadd"], gated)
            dg = D.gemm(d["dadd"], w[f"{i}.out"], out_dtype=self.dtype, math=self._math())
            dcols = torch.empty(T, B, sum(self.parts), device=dg.device, dtype=self.dtype)
            dq, dk, dv, dz, da, db = self._cols(dcols)
            do = D.rms_norm_grad(o, w[f"{i}.ow"], rs2, dg, gate=z, groups=self.heads, dgate=dz)
            g[f"{i}.ow"] = do["dw"]
            gs = D.delta_scan_grad(*ins, kept, do["dx"].view(T, B, self.heads, self.V), dq=dq, dk=dk, dv=dv, da=da, db=db, **kw)
            g[f"{i}.A_log"], g[f"{i}.dt_bias"] = gs["dA"] * ins[5], gs["ddt_bias"]  # A = -exp(A_log)
            dcols = dcols.view(rows, -1)
            g[f"{i}.in"] = self._tn(dcols, n1)
            dn = D.gemm(dcols, w[f"{i}.in"], out_dtype=self.dtype, math=self._math())
            d = D.rms_norm_grad(x1, w[f"{i}.n1w"], rs1, dn, dres=d["dx"], add=add1, scale=scale1)
            g[f"{i}.n1w"] = d["dw"]
        dx = d["dx"].float()
        g["enc"], g["enc_b"] = self._tn(dx, obs.reshape(rows, -1)), D.colsum(dx)
        return g
