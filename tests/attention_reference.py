"""Attention and its gradients from the definition in 64 bits, with a bound of what the kernels' arithmetic may be off by."""
from __future__ import annotations

import math

import torch

HALF = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # half a step, relative


def visible(B, Sq, Sk, causal, window, lengths, device):
    i = torch.arange(Sq, device=device)[:, None] + (Sk - Sq)
    j = torch.arange(Sk, device=device)[None]
    see = torch.ones((B, 1, Sq, Sk), dtype=torch.bool, device=device)
    if causal:
        see = see & (j <= i)
    if window:
        see = see & (j > i - window)
    if lengths is not None:
        see = see & (j < lengths.long()[:, None, None, None])
    return see


def reference(q, k, v, d_o=None, causal=False, window=None, key_lengths=None, mask=None, scale=None):
    """-> {name: (values, bound)} for o, lse and, with ``d_o``, dq, dk, dv.

    The bound counts roundings.  u = 2^-24 throughout; with bf16 tensors h = 2^-8 for every probability and every score's gradient
    that is rounded for the products, and for the stored output that delta = rowsum(dO O) is taken from:
      score      x: D products and sums, the scale, the mask, the subtraction of the maximum, the change to base 2
      probability p: its score's error, exp2 (2^-21), the sum of n terms and its rounding, (h)
      output     o: sum of n terms p v"""
    dt, u = q.dtype, 2.0 ** -24
    h = HALF[dt] if dt == torch.bfloat16 else 0.0
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    see = visible(B, Sq, Sk, causal, window, key_lengths, q.device).expand(B, Hq, Sq, Sk)
    if key_lengths is not None:                                  # what lies behind the lengths does not exist
        gone = (torch.arange(Sk, device=q.device)[None] >= key_lengths.long()[:, None])[:, None, :, None]
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    Q, K, V = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    x = scale * Q @ K.mT
    xe = scale * (Q.abs() @ K.abs().mT) * (D + 4) * u
    if mask is not None:
        m = mask.expand(B, Hq, Sq, Sk)
        if m.dtype == torch.bool:
            see = see & m
        else:
            see = see & (m != -math.inf)
            low = m.double().masked_fill(m == -math.inf, 0.0)
            # the sum is taken in fp32: next to a mask of the type's lowest value nothing of the product is left
            big = low.abs() > 1e30
            x = torch.where(big, low, x + low)
            xe = torch.where(big, torch.zeros_like(xe), xe + u * low.abs())
    x = x.masked_fill(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    base = top.masked_fill(top == -math.inf, 0.0)
    e = (x - base).exp()
    total = e.sum(-1, keepdim=True)
    some = total > 0
    p = e / total.masked_fill(~some, 1.0)
    lse = (base + total.masked_fill(~some, 1.0).log()).masked_fill(~some, -math.inf)
    n = float(Sk)
    gap = (x - base).masked_fill(~see, 0.0).abs()
    xe = xe.masked_fill(~see, 0.0)
    pe = 2 * (xe + 4 * u * gap) + (p * 2 * (xe + 4 * u * gap)).sum(-1, keepdim=True) + 2.0 ** -20 + (n / 32 + 40) * u     # relative; sums run in up to n / 32 steps
    pe = pe.masked_fill(~see, 0.0).clamp_max(2.0)
    o = p @ V
    oe = (p * (pe + h)) @ V.abs() + (n / 8 + 160) * u * (p @ V.abs())
    out = {"o": (o, oe * (1 + HALF[dt]) + HALF[dt] * o.abs() + 2.0 ** -126),
           "lse": (lse[..., 0], (xe.amax(-1) + 4 * u * base[..., 0].abs() + 2.0 ** -18 + u * lse[..., 0].abs().nan_to_num(0.0, posinf=0.0)) + 0.0)}
    if d_o is None:
        return out
    g = d_o.double()
    dp = g @ V.mT
    dpe = (g.abs() @ V.abs().mT) * (D + 4) * u
    delta = (g * o).sum(-1, keepdim=True)
    deltae = (g.abs() * out["o"][1]).sum(-1, keepdim=True) + (g.abs() * o.abs()).sum(-1, keepdim=True) * (D + 4) * u
    ds = p * (dp - delta)
    dse = p * pe * (dp - delta).abs() + p * (1 + pe) * (dpe + deltae + 2 * u * (dp.abs() + delta.abs()))
    dse = dse + (h + 2 * u) * (ds.abs() + dse)

    def shared(t):
        return t.view(B, Hkv, G, Sk, D).sum(2)
    many = (G * max(Sq, Sk) / 8 + 160) * u
    for name, val, err in (("dq", scale * ds @ K, scale * (dse @ K.abs() + many * ((ds.abs() + dse) @ K.abs()))),
                           ("dk", shared(scale * ds.mT @ Q), shared(scale * (dse.mT @ Q.abs() + many * ((ds.abs() + dse).mT @ Q.abs())))),
                           ("dv", shared(p.mT @ g), shared((p * (pe + h)).mT @ g.abs() + many * (p.mT @ g.abs())))):
        out[name] = (val, err * (1 + HALF[dt]) + (HALF[dt] + 4 * u) * val.abs() + 2.0 ** -126)
    return out


def check(name, got, want, bound, norm=None):
    """Every value within its bound; with ``norm`` also the relative 2-norm of the whole."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine]), name
    err = (got[fine] - want[fine]).abs()
    worst = float((err - bound[fine]).max()) if err.numel() else 0.0
    assert worst <= 0.0, (name, worst, float((err / bound[fine].clamp_min(1e-300)).max()))
    if norm is not None and err.numel() and float(want[fine].norm()) > 0:
        rel = float(err.norm() / want[fine].norm())
        assert rel <= norm, (name, rel)
