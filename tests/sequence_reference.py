"""Attention, its position buckets and layer norm from their definitions in 64 bits, with the size of the terms that every
output sums (what a rounding error can be relative to): test infrastructure."""
import math

import torch


def bucket(dist, buckets, max_distance, both):
    """Bucket of a distance (int): the far buckets' borders compared in whole numbers."""
    side = buckets // 2 if both else buckets
    n = abs(dist) if both else max(-dist, 0)
    E = side // 2
    far = side - E
    if n < E:
        b = n
    else:
        n = min(n, max_distance)
        b = E
        while b < side - 1 and n ** far * E ** (b - E + 1) >= max_distance ** (b - E + 1) * E ** far:
            b += 1
    return b + side if both and dist > 0 else b


def places(B, H, Lq, Lk, causal=False, lengths=None, mask=None, starts=None, start=None):
    """allowed [B, H, Lq, Lk] and distances [B, Lq, Lk] (CPU)."""
    j = torch.arange(Lk)
    first = torch.full((B,), Lk - Lq if start is None else start) if starts is None else starts.long().cpu()
    pos = first.view(B, 1) + torch.arange(Lq)
    dist = j.view(1, 1, Lk) - pos.unsqueeze(-1)
    ok = torch.ones(B, H, Lq, Lk, dtype=torch.bool)
    if lengths is not None:
        ok &= j.view(1, 1, 1, Lk) < lengths.long().cpu().view(B, 1, 1, 1)
    if causal:
        ok &= (dist <= 0).unsqueeze(1)
    if mask is not None:
        ok &= (mask.cpu() != 0)
    return ok, dist


def attention(q, k, v, ok, scale, dout=None, bias=None):
    """q [B,H,Lq,d], k, v [B,Hk,Lk,d] in any type; ok as above; bias [B,H,Lq,Lk] fp64 or None.  Returns a dict of fp64 tensors:
    out, and with dout dq, dk, dv, ds; and under "mag" the same names' sums of absolute terms."""
    dev = q.device
    B, H, Lq, d = q.shape
    Hk, Lk = k.shape[1], k.shape[2]
    G = H // Hk
    ok = ok.to(dev)
    seen = ok.any(2).view(B, Hk, G, Lk).any(2)                   # keys that some query sees: the others are not part of anything
    q, k, v = (x.detach().double() for x in (q, k, v))
    k, v = (torch.where(seen.unsqueeze(-1), x, torch.zeros_like(x)) for x in (k, v))
    ke, ve = (x.repeat_interleave(G, 1) for x in (k, v))
    s = q @ ke.transpose(2, 3) * scale
    smax = (q.abs() @ ke.abs().transpose(2, 3) * scale).amax().item() if s.numel() else 0.0
    if bias is not None:
        s = s + bias
        smax += bias.abs().amax().item() if bias.numel() else 0.0
    s = s.masked_fill(~ok, -math.inf)
    some = ok.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1), torch.zeros_like(s)) if Lk else s
    r = {"out": p @ ve, "smax": smax, "mag": {"out": p @ ve.abs()}}
    if dout is None:
        return r
    do = dout.detach().double()
    dp = do @ ve.transpose(2, 3)
    delta = (do * r["out"]).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    size = p * (do.abs() @ ve.abs().transpose(2, 3) + (do.abs() * r["mag"]["out"]).sum(-1, keepdim=True))
    group = lambda x: x.view(B, Hk, G, Lk, d).sum(2)
    r.update(dq=ds @ ke * scale, dk=group(ds.transpose(2, 3) @ q * scale), dv=group(p.transpose(2, 3) @ do), ds=ds)
    r["mag"].update(dq=size @ ke.abs() * scale, dk=group(size.transpose(2, 3) @ q.abs() * scale), dv=group(p.transpose(2, 3) @ do.abs()), ds=size)
    return r


def bias_of(table, dist, buckets, max_distance, both):
    """[B,H,Lq,Lk] from table [buckets, H], and the buckets [B,Lq,Lk]."""
    lo, hi = int(dist.min()), int(dist.max())
    lut = torch.tensor([bucket(x, buckets, max_distance, both) for x in range(lo, hi + 1)])
    at = lut[dist - lo]
    return table.detach().double()[at.to(table.device)].permute(0, 3, 1, 2), at


def table_grad(ds, at, buckets):
    """sum of ds [B,H,Lq,Lk] over the places of each bucket: [buckets, H]"""
    at = at.to(ds.device)
    return torch.stack([(ds * (at == b).unsqueeze(1)).sum((0, 2, 3)) for b in range(buckets)])


def tolerance(name, r, dtype, d, terms):
    """Bound of |computed - exact| per element, before the final rounding, from the sums of absolute terms:
    fp32 rounding of a score is at most (d + 4) half steps of its terms' sum, twice that is a probability's (numerator and
    denominator), a sum of n terms adds n half steps; in 16 bits the second product's left factor is rounded once
    (out, dv: p; dq, dk: ds, whose delta comes from the rounded output: a second one)."""
    u32, ut = 2.0 ** -24, (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0)
    rounds = 2 if name in ("dq", "dk", "ds") else 1
    rel = 2 * (d + 4) * u32 * max(r["smax"], 1.0) + (terms + d + 16) * u32 + rounds * ut
    return rel * r["mag"][name]


def check(name, got, r, dtype, d, terms):
    ref = r[name]
    assert got.shape == ref.shape and got.dtype == dtype, (name, got.shape, got.dtype)
    if not ref.numel():
        return
    limit = tolerance(name, r, dtype, d, terms) + torch.finfo(dtype).eps / 2 * ref.abs() * 1.01 + 1e-30
    err = (got.detach().double() - ref).abs()
    assert torch.isfinite(got).all(), f"{name} not finite"
    worst = (err / limit).amax().item()
    assert worst <= 1.0, f"{name}: {worst:.3g} times the bound, max err {err.amax().item():.3e}"
