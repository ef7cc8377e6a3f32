"""The preference and policy losses in 64 bits, sequence by sequence, from their definitions."""
from __future__ import annotations

import math

import pytest
import torch


def sequences(shape, offsets, mask):
    """The indices of the tokens that count, of each sequence."""
    n = math.prod(shape)
    if offsets is None:
        t = shape[1]
        ranges = [(r * t, (r + 1) * t) for r in range(shape[0])]
    else:
        o = [int(x) for x in offsets]
        ranges = list(zip(o, o[1:]))
    keep = [True] * n if mask is None else [bool(x) for x in mask.reshape(-1).cpu()]
    return [[t for t in range(a, z) if keep[t]] for a, z in ranges]


def preference(nll, ref, *, offsets=None, mask=None, beta=0.1, kind="sigmoid", label_smoothing=0.0, reduction="mean", ct=None):
    """(loss, chosen, rejected, d_nll); ct: the loss's cotangent."""
    x, r = nll.detach().double().cpu().reshape(-1), ref.detach().double().cpu().reshape(-1)
    seqs = sequences(tuple(nll.shape), offsets, mask)
    pairs = len(seqs) // 2
    g = [sum(float(r[t] - x[t]) for t in s) / (max(1, len(s)) if kind == "ipo" else 1) for s in seqs]
    loss, slope = [], []
    for p in range(pairs):
        d = beta * (g[p] - g[pairs + p])
        if kind == "sigmoid":
            soft = lambda y: max(y, 0.0) + math.log1p(math.exp(-abs(y)))  # noqa: E731
            loss.append((1 - label_smoothing) * soft(-d) + label_smoothing * soft(d))
            slope.append(label_smoothing - (1 / (1 + math.exp(d)) if d < 700 else 0.0))
        elif kind == "hinge":
            loss.append(max(0.0, 1 - d))
            slope.append(-1.0 if d < 1 else 0.0)
        else:
            loss.append((d / beta - 0.5 / beta) ** 2)
            slope.append(2 * (d / beta - 0.5 / beta) / beta)
    loss = torch.tensor(loss, dtype=torch.float64)
    total = {"none": loss, "mean": loss.mean(), "sum": loss.sum()}[reduction]
    ct = torch.ones_like(total) if ct is None else ct.detach().double().cpu()
    up = (ct if reduction == "none" else ct.expand(pairs)) / (pairs if reduction == "mean" else 1)
    grad = torch.zeros_like(x)
    for k, s in enumerate(seqs):
        p, sign = k % pairs, -1.0 if k < pairs else 1.0
        share = 1 / max(1, len(s)) if kind == "ipo" else 1.0
        if s:
            grad[torch.tensor(s)] = sign * slope[p] * beta * share * float(up[p])
    g = torch.tensor(g, dtype=torch.float64) * beta
    return total, g[:pairs], g[pairs:], grad.reshape(nll.shape)


def policy(nll, old, adv, *, ref_nll=None, offsets=None, mask=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
           reduction="token", ct=None):
    """(loss, kl, clip_fraction, d_nll)."""
    x, o = nll.detach().double().cpu().reshape(-1), old.detach().double().cpu().reshape(-1)
    seqs = sequences(tuple(nll.shape), offsets, mask)
    a = adv.detach().double().cpu().reshape(-1)
    per_token = adv.shape == nll.shape
    r = None if ref_nll is None else ref_nll.detach().double().cpu().reshape(-1)
    loss, slope = torch.zeros_like(x), torch.zeros_like(x)
    kl, clipped, count = 0.0, 0, sum(map(len, seqs))
    filled = sum(1 for s in seqs if s)
    weight = torch.zeros_like(x)
    for k, s in enumerate(seqs):
        for t in s:
            at = float(a[t] if per_token else a[k])
            u = math.exp(float(o[t] - x[t]))
            c = min(max(u, 1 - clip_low), 1 + clip_high)
            out = c * at < u * at
            loss[t] = -min(u * at, c * at)
            slope[t] = 0.0 if out else u * at
            clipped += out
            if r is not None:
                d = float(x[t] - r[t])
                kl += math.expm1(d) - d
                if kl_coef:
                    loss[t] += kl_coef * (math.expm1(d) - d)
                    slope[t] += kl_coef * math.expm1(d)
            weight[t] = {"token": 1 / count, "sequence": 1 / (len(s) * filled), "none": 1.0}[reduction]
    if reduction == "none":
        total = loss.reshape(nll.shape)
        up = torch.ones_like(x) if ct is None else ct.detach().double().cpu().reshape(-1)
    else:
        total, up = (loss * weight).sum(), torch.full_like(x, 1.0 if ct is None else float(ct))
    n = max(1, count)
    return (total, torch.tensor(kl / n, dtype=torch.float64), torch.tensor(clipped / n, dtype=torch.float64),
            (slope * weight * up).reshape(nll.shape))


def tensors(shape, seed, std=1.0):
    """nll, old_nll, ref_nll: losses near each other, as of models that were the same some steps ago."""
    g = torch.Generator().manual_seed(seed)
    nll = torch.randn(shape, generator=g).abs() * 2
    return nll, nll + 0.2 * std * torch.randn(shape, generator=g), nll + 0.4 * std * torch.randn(shape, generator=g)


def layout(name, seqs, t, seed):
    """(shape, offsets, mask) of `seqs` sequences of about t tokens."""
    g = torch.Generator().manual_seed(seed + 100)
    if name == "batch":
        return (seqs, t), None, None
    if name == "masked":
        m = torch.rand((seqs, t), generator=g) < 0.6
        m[-1] = False   # a sequence without a token that counts
        return (seqs, t), None, m
    n = seqs * t
    cuts = torch.sort(torch.randint(0, n + 1, (seqs - 1,), generator=g)).values
    if name == "packed":
        return (n,), torch.cat([torch.tensor([0]), cuts, torch.tensor([n])]), None
    # tokens of no sequence before, behind; an empty sequence; a mask as well
    o = torch.cat([torch.tensor([2]), (cuts + 2).clamp(max=n + 2), torch.tensor([n + 2])])
    o[1] = o[0]
    return (n + 7,), o, torch.rand((n + 7,), generator=g) < 0.8


LAYOUTS = ("batch", "masked", "packed", "gaps")


def check_infinite(place, **kw):
    """Losses and gradients where a ratio is infinite or 0; `place` puts a tensor where `kw`'s impl wants it."""
    from mlx_train_perf import policy_loss, preference_loss

    inf = math.inf
    # the rejected answer (then the chosen one) has a token that the policy rules out
    for nll, want, slope in (([[1.0, 2.0], [1.0, inf]], 0.0, 0.0), ([[1.0, inf], [1.0, 2.0]], inf, 0.1)):
        x = place(torch.tensor(nll)).requires_grad_(True)
        r = preference_loss(x, place(torch.ones(2, 2)), **kw)
        (d,) = torch.autograd.grad(r.loss, x)
        assert float(r.loss.detach()) == want
        assert torch.allclose(d.double().cpu(), torch.tensor([[slope] * 2, [-slope] * 2], dtype=torch.float64), atol=1e-9)
    # old = inf: a ratio of infinity; advantages that clip it, drop it and leave it. nll = inf: a ratio of 0
    old = torch.tensor([[inf, inf, inf, 1.0, 1.0, 1.0]])
    nll = torch.tensor([[1.0, 1.0, 1.0, inf, inf, inf]])
    adv = torch.tensor([[1.0, 0.0, -1.0, 1.0, 0.0, -1.0]])
    x = place(nll).requires_grad_(True)
    r = policy_loss(x, place(old), place(adv), reduction="none", **kw)
    (d,) = torch.autograd.grad(r.loss, x, torch.ones_like(r.loss))
    assert r.loss.detach().tolist()[0] == pytest.approx([-1.2, 0.0, inf, 0.0, 0.0, 0.8])
    assert d.tolist()[0] == [0.0, 0.0, -inf, 0.0, 0.0, 0.0]
    assert float(r.clip_fraction) == pytest.approx(2 / 6)
