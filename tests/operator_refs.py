"""Plain 64-bit forms of grouped routing, 4-bit experts and the 8-bit RMSNorm, for tests.

They run on any device, straight from the operators' definitions."""

import math

import torch

NEG = -math.inf


def route(logits, K, *, scoring, select_bias=None, num_groups=1, topk_groups=1, group_score="max", renormalize=True,
          scale=1.0):
    """(weights fp64 [T,K], ids int64 [T,K])."""
    l = logits.double()
    T, E = l.shape
    s = torch.softmax(l, 1) if scoring == "softmax" else torch.sigmoid(l)
    c = s.clone() if select_bias is None else s + select_bias.double()
    c = torch.where(torch.isnan(c), NEG, c)
    if num_groups > 1:
        per = E // num_groups
        top = torch.topk(c.view(T, num_groups, per), 2 if group_score == "top2" else 1).values.sum(-1)
        top = torch.where(torch.isnan(top), NEG, top)
        best = torch.sort(top, dim=1, descending=True, stable=True).indices[:, :topk_groups]
        kept = torch.zeros(T, num_groups, dtype=torch.bool, device=l.device).scatter_(1, best, True)
        c = torch.where(kept.repeat_interleave(per, 1), c, NEG)
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :K]
    w = torch.gather(s, 1, ids)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total < 1e-20, 1e-20, total)
    return w * scale, ids


def act(kind, g):
    if kind == "silu":
        return g * torch.sigmoid(g)
    if kind == "gelu":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def dequantise(codes, scales, group):
    """codes [S, N, K/2] uint8, scales [S, N, ceil(K/group)] -> fp64 [S, N, K]."""
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
    return q * scales.double().repeat_interleave(group, -1)[..., : q.shape[-1]]


def experts(x, w1, w2, weights, ids, activation, *, shared_y=None, shared_scale=None, residual=None):
    """(out fp64 [T,H] unrounded, bound fp64 [T,H]) for dequantised fp64 w1 [E,2I,H], w2 [E,H,I].

    bound: how far a kernel may be that sums in fp32 and rounds the gated activation h and the output
    to x's dtype.  With u = eps / 2 of that dtype, per product of n terms an fp32 sum is off by at most
    n * 2^-23 * sum|terms| (twice the textbook bound: tensor cores may truncate), so
      |dg| <= eg = H 2^-23 |x||Wg|, likewise eu;  |dh| <= 1.2 eg (|u| + eu) + |a| eu + (u + 2^-16) |h| + tiny
    (|act'| < 1.2; 2^-16: the activation's own fp32 error; tiny: half a subnormal step of fp16),
    |dy| <= |dh||W2| + I 2^-23 |h||W2|, and the output adds u |out|."""
    T, H = x.shape
    E, I = w2.shape[0], w2.shape[2]
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        xe, wk = x[t].double(), weights[t, k].double()[:, None]
        gu, mag = xe @ w1[e].T, xe.abs() @ w1[e].abs().T
        g, up = gu[:, :I], gu[:, I:]
        a = act(activation, g)
        eg, eu = H * 2.0 ** -23 * mag[:, :I], H * 2.0 ** -23 * mag[:, I:]
        h = a * up
        dh = 1.2 * eg * (up.abs() + eu) + a.abs() * eu + (u + 2.0 ** -16) * h.abs() + tiny
        out.index_add_(0, t, wk * (h @ w2[e].T))
        bound.index_add_(0, t, wk.abs() * ((dh + I * 2.0 ** -23 * h.abs()) @ w2[e].abs().T))
    if shared_y is not None:
        out += shared_y.double() * (1 if shared_scale is None else shared_scale.double()[:, None])
    if residual is not None:
        out += residual.double()
    return out, bound * 1.01 + (u + 2.0 ** -20) * out.abs() + 32 * 2.0 ** -24 * (out.abs() + bound) + tiny


def norm(x, weight, *, residual=None, bias=None, eps=1e-6):
    """(r in x's dtype, z fp64)."""
    r = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    d = r.double()
    z = d / torch.sqrt(d.pow(2).mean(1, keepdim=True) + eps) * weight.double()
    return r, z if bias is None else z + bias.double()
