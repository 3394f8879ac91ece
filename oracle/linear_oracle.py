"""CPU checker of linear attention with a decay for each head: the recurrence in 64 bits, its gradients by autograd, and the sums of
absolute values that bound what rounding can do to each result."""
from __future__ import annotations

import torch


def spans(q, cu):
    """(batch row, first token, length) of every sequence."""
    if cu is None:
        return [(b, 0, q.shape[1]) for b in range(q.shape[0])]
    c = cu.tolist()
    return [(0, a, e - a) for a, e in zip(c, c[1:])]


def recurrent(q, k, v, g, scale, s0=None, cu=None):
    """o [B,T,Hv,dv] and final states [N,Hv,dk,dv] in 64 bits; differentiable.  g: [B,T,Hv], [Hv] or None."""
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    rep = Hv // Hk
    q, k, v = q.double().repeat_interleave(rep, 2), k.double().repeat_interleave(rep, 2), v.double()
    a = torch.ones(B, T, Hv, dtype=torch.float64) if g is None else torch.exp(g.double().expand(B, T, Hv))
    o = [[None] * T for _ in range(B)]
    finals = []
    for n, (b, t0, length) in enumerate(spans(q, cu)):
        M = torch.zeros(Hv, dk, dv, dtype=torch.float64) if s0 is None else s0[n].double()
        for t in range(t0, t0 + length):
            M = a[b, t, :, None, None] * M + k[b, t, :, :, None] * v[b, t, :, None, :]
            o[b][t] = scale * torch.einsum("hkv,hk->hv", M, q[b, t])
        finals.append(M)
    zero = torch.zeros(Hv, dv, dtype=torch.float64)
    out = torch.stack([torch.stack([x if x is not None else zero for x in row]) if row else torch.zeros(0, Hv, dv, dtype=torch.float64) for row in o])
    return out, torch.stack(finals) if finals else torch.zeros(0, Hv, dk, dv, dtype=torch.float64)


def magnitudes(q, k, v, g, scale, s0=None, cu=None):
    """The same with every term's absolute value."""
    return recurrent(q.abs(), k.abs(), v.abs(), g, abs(scale), None if s0 is None else s0.abs(), cu)


def gradients(q, k, v, g, scale, s0, cu, d_o, d_final):
    """(dq, dk, dv, dg, ds0) in 64 bits, None where there is no input."""
    leaves = {n: (None if x is None else x.detach().double().requires_grad_(True)) for n, x in dict(q=q, k=k, v=v, g=g, s0=s0).items()}
    o, final = recurrent(leaves["q"], leaves["k"], leaves["v"], leaves["g"], scale, leaves["s0"], cu)
    loss = (o * d_o.double()).sum()
    if d_final is not None:
        loss = loss + (final * d_final.double()).sum()
    used = [x for x in leaves.values() if x is not None]
    got = iter(torch.autograd.grad(loss, used, allow_unused=True))
    return tuple(None if x is None else next(got) for x in leaves.values())
