"""Plain attention with capped scores, a bias by distance and key spans in 64 bits (any device), from the
definition: the checks of the scored attention tests. And the masks that those tests use."""
from __future__ import annotations

import torch

MASKS = ("causal", "full", "prefix", "docs", "window", "ragged", "nothing")


def spans_of(mask: str, b: int, s: int, seed: int = 0):
    """(start, end) int32 (b, s), or None for the masks that need none."""
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(s).expand(b, s)
    start, end = torch.zeros(b, s, dtype=torch.int64), i + 1
    if mask in ("causal", "full"):
        return None
    if mask == "prefix":    # row 0 without a prefix, the last row all of it
        p = torch.randint(0, s + 1, (b, 1), generator=g)
        p[0], p[-1] = 0 if b > 1 else s // 2, s if b > 1 else s // 2
        end = torch.maximum(end, p)
    elif mask == "docs":    # documents that see themselves whole, then padding that sees nothing
        cuts = torch.sort(torch.randint(0, s + 1, (b, 5), generator=g), dim=1).values
        used = s - s // 5
        for r in range(b):
            edges = [0, *[int(c) for c in cuts[r] if 0 < c < used], used]
            start, end = start.clone(), end.clone()
            for a, z in zip(edges, edges[1:]):
                start[r, a:z], end[r, a:z] = a, z
            start[r, used:] = end[r, used:] = used
    elif mask == "window":
        start = (i - max(1, s // 6)).clamp(min=0)
    elif mask == "ragged":  # any two bounds that do not decrease: some queries see nothing, in the middle too
        start = torch.sort(torch.randint(0, s + 1, (b, s), generator=g), dim=1).values
        end = torch.sort(torch.randint(0, s + 1, (b, s), generator=g), dim=1).values
    elif mask == "nothing":
        start, end = torch.zeros(b, s, dtype=torch.int64), torch.zeros(b, s, dtype=torch.int64)
    return start.to(torch.int32).contiguous(), end.to(torch.int32).contiguous()


def visible(mask: str, spans, b: int, s: int, device="cpu") -> torch.Tensor:
    j = torch.arange(s, device=device)
    if spans is not None:
        return (j >= spans[0].to(device)[..., None]) & (j < spans[1].to(device)[..., None])
    see = j[None, :] <= j[:, None] if mask == "causal" else torch.ones(s, s, dtype=torch.bool, device=device)
    return see.expand(b, s, s)


def attention(q, k, v, d_o, *, scale, see, softcap=None, slopes=None, d_terms=False):
    """(o, dq, dk, dv) in 64 bits; `see` (b, s, s).

    `d_terms`: also what an error of D = rowsum(dO o O) does to dq and dk, for D formed from an O whose probabilities
    and values were each rounded by a relative u: |delta D_i| <= u sum_d |dO| (|O| + P |V|), and, as
    dS = P (dP - D) (1 - tanh^2), delta dq_i = scale delta D_i sum_j P (1 - tanh^2) k_j and
    delta dk_j = scale sum_i P (1 - tanh^2) delta D_i q_i. Bounds of both, for u = 1. (dS is a difference that all but
    cancels where one probability is nearly 1, so dq and dk have no relative bound without this term.)"""
    b, hq, s, dh = q.shape
    hkv = k.shape[1]
    q, k, v, d_o = (x.double() for x in (q, k, v, d_o))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    tq, tk = torch.zeros_like(q), torch.zeros_like(k)
    i = torch.arange(s, device=q.device)
    away = (i[:, None] - i[None, :]).abs().double()
    for r in range(b):
        for h in range(hq):
            kv = h // (hq // hkv)
            x = scale * (q[r, h] @ k[r, kv].T)
            bend = torch.ones_like(x)
            if softcap is not None:
                bend = 1 - torch.tanh(x / softcap) ** 2
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * away
            top = torch.where(see[r], x, -torch.inf).amax(1, keepdim=True).clamp(min=-1e300)
            p = torch.where(see[r], torch.exp(x - top), 0.0)
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            o[r, h] = p @ v[r, kv]
            dp = d_o[r, h] @ v[r, kv].T
            ds = torch.where(see[r], p * (dp - (d_o[r, h] * o[r, h]).sum(1, keepdim=True)) * bend, 0.0)
            dq[r, h] = scale * (ds @ k[r, kv])
            dk[r, kv] += scale * (ds.T @ q[r, h])
            dv[r, kv] += p.T @ d_o[r, h]
            off = (d_o[r, h].abs() * (o[r, h].abs() + p @ v[r, kv].abs())).sum(1, keepdim=True)
            tq[r, h] = scale * off * ((p * bend) @ k[r, kv]).abs()
            tk[r, kv] += scale * ((p * bend * off).T @ q[r, h].abs())
    return (o, dq, dk, dv, tq, tk) if d_terms else (o, dq, dk, dv)


def inputs(b, hq, hkv, s, dh, dtype, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    def normal(h, x=1.0):
        return (torch.randn(b, h, s, dh, generator=g) * x).to(dtype)
    return normal(hq, std), normal(hkv), normal(hkv), normal(hq)


def slopes_of(hq: int) -> torch.Tensor:
    return 2.0 ** (-8.0 * torch.arange(1, hq + 1) / hq)


def off(a: torch.Tensor, want: torch.Tensor) -> float:
    return float((a.detach().double().cpu() - want.double().cpu()).norm())


def rel(a: torch.Tensor, want: torch.Tensor) -> float:
    """2-norm of the difference over that of `want` (the difference's itself where `want` is all zeros)."""
    a, want = a.detach().double().cpu(), want.double().cpu()
    norm = float(want.norm())
    off = float((a - want).norm())
    return off / norm if norm else off
