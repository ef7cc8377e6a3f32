"""Inputs, expected values in 64 bits and error bounds for the tests of token scoring and distillation.

Hidden states and weights are whole multiples of a unit, so that every logit is exact in fp32 in any order of summation: what
is left to bound is the statistics' arithmetic. u = 2^-24 is half a step of fp32 at 1, r half a step of bf16 (2^-8).
- x = z log2(e) / t - max: one rounding, |x| below 64, so e^x is off by 64 ln2 u and the exponential's own 2 u; sums run in
  chains of at most V / 8 + 64 terms: a sum's relative error is `stat` = (V / 8 + 256) u, and log s is off by that. lse and a
  log probability (below 32 in size) add 4 roundings of 32 u.
- the entropy is log s - (sum e x) / s, the second term below 64 with the relative errors of both sums: 64 * 2 stat more.
- a gradient by a logit, p (alpha + beta x) or a listed column's: p is off by stat + 128 u of itself, the factors (below 64
  times the incoming gradient) by 256 u of that; bf16 products round it by r. The products sum V (or N) terms in fp32."""
from __future__ import annotations

import math

import torch

from mlx_train_perf import DenseHead, QuantizedHead

U, R = 2.0 ** -24, 2.0 ** -8
TAIL = 1e-6


def grid(g, *shape, unit=1 / 32, limit=127):
    return (torch.randn(*shape, generator=g) / unit).round().clamp(-limit, limit) * unit


def make(n, d, v, *, head="dense", dtype="bf16", seed=0):
    """(hidden, head, weights in fp64) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp64": torch.float64}[dtype]
    size = 2.0 ** round(math.log2(2 / math.sqrt(d)))
    hidden = grid(g, n, d).to(dt)
    if head == "q4":
        words = torch.randint(-2 ** 31, 2 ** 31, (v, d // 8), generator=g).to(torch.int32)
        scales = size / 4 * 2.0 ** torch.randint(-1, 2, (v, d // 64), generator=g)
        q = torch.stack([(words >> (4 * i)) & 15 for i in range(8)], -1).reshape(v, d).double()
        w = (q - 8) * scales.double().repeat_interleave(64, 1)
        return hidden, QuantizedHead(w_q=words, scales=scales.bfloat16(), biases=(-8 * scales).bfloat16()), w
    w = grid(g, v, d) * size
    return hidden, DenseHead(weight=w.to(dt), trainable=head == "trainable"), w.double()


def to(head, device):
    if isinstance(head, DenseHead):
        w = head.weight.to(device)
        return DenseHead(weight=w.requires_grad_(head.trainable), trainable=head.trainable)
    return QuantizedHead(w_q=head.w_q.to(device), scales=head.scales.to(device), biases=head.biases.to(device))


def stat(v):
    return (v / 8 + 256) * U


def logits(hidden, w, live):
    return (torch.where(live[:, None], hidden.double(), 0.0) @ w.T).requires_grad_(True)


def score(z, targets, live, temperature, top):
    """(logprobs, entropy, top_logprobs, top_ids) of logits z."""
    n, v = z.shape
    e = torch.exp(z / temperature - (z / temperature).amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    logp = z / temperature - torch.logsumexp(z / temperature, 1, keepdim=True)
    entropy = torch.where(live, -(p * logp).sum(1), 0.0)
    logprobs = None
    if targets is not None:
        y = torch.where(live, targets, 0)
        logprobs = torch.where(live, logp[torch.arange(n), y], 0.0)
    zd = z.detach()
    # ranks: by value, then by index
    order = sorted_ids(zd)[:, :top]
    ids = torch.where(live[:, None], order, -1)
    best = torch.where(live[:, None], logp.detach().gather(1, order), -math.inf)
    return logprobs, entropy, best, ids


def sorted_ids(z):
    ids = torch.empty(z.shape, dtype=torch.int64)
    for i, row in enumerate(z.tolist()):
        ids[i] = torch.tensor(sorted(range(len(row)), key=lambda j: (-row[j], j)))
    return ids


def teacher_list(n, v, k, *, seed=0, renormalize=False, holes=True):
    """(ids, log probabilities, mask): shorter lists, empty and repeated slots, rows without any, and rows that are masked."""
    g = torch.Generator().manual_seed(seed + 7)
    ids = torch.stack([torch.randperm(max(v, k), generator=g)[:k] % v for _ in range(n)])
    lp = torch.log_softmax(2 * torch.randn(n, k, generator=g), 1)
    if renormalize:
        lp = lp + 3
    else:
        lp = lp + torch.log(0.5 + 0.499 * torch.rand(n, 1, generator=g))
    mask = torch.ones(n, dtype=torch.bool)
    if holes:
        for i in range(n):
            if i % 4 == 1 and k > 1:
                ids[i, k // 2:] = -1
            if i % 4 == 2:
                lp[i, k - 1] = -math.inf
            if i % 4 == 3 and k > 2:
                ids[i, k - 1] = ids[i, 0]
            if i % 7 == 5:
                ids[i] = -1
        mask[1::3] = False
        lp[~mask] = math.nan
    return ids, lp.float(), mask


def distill(z, ids, lp, mask, *, kind, beta, temperature, renormalize, reduction):
    """The loss of logits z, row by row over the outcomes that count."""
    logp = torch.log_softmax(z / temperature, 1)
    losses = []
    for i in range(z.shape[0]):
        seen = {}
        if mask is None or mask[i]:
            for slot, y in enumerate(ids[i].tolist()):
                if 0 <= y < z.shape[1] and lp[i, slot] != -math.inf and y not in seen:
                    seen[y] = lp[i, slot].double()
        if not seen:
            losses.append(None)
            continue
        t = torch.stack(list(seen.values()))
        q = logp[i, list(seen)]
        if renormalize:
            t = torch.log_softmax(t / temperature, 0)
        rq, rt = (lift(1 - a.exp().sum()) for a in (q, t))
        q = torch.cat([q, rq.log()[None]])
        if renormalize:
            t = torch.cat([t, torch.tensor([-math.inf], dtype=torch.float64)])
        else:
            t = torch.cat([t, rt.log()[None]])
        losses.append({"forward": lambda: kl(t, q), "reverse": lambda: kl(q, t),
                       "jsd": lambda: jsd(t, q, beta)}[kind]())
    live = torch.tensor([x is not None for x in losses])
    loss = torch.stack([z.new_zeros(()) if x is None else x for x in losses])
    if reduction == "mean":
        loss = loss.sum() / live.sum().clamp(min=1)
    elif reduction == "sum":
        loss = loss.sum()
    return loss, live


def lift(rest):
    return rest + (rest.clamp(min=TAIL) - rest).detach()


def kl(a, b):
    keep = a != -math.inf
    return (a[keep].exp() * (a[keep] - b[keep])).sum()


def jsd(t, q, beta):
    m = (beta * t.exp() + (1 - beta) * q.exp()).log()
    return beta * kl(t, m) + (1 - beta) * kl(q, m)


def gradient_bounds(g, p, extra, hidden, w, want_dw, dtype, halves):
    """(dL/dhidden, its bound, dL/dw, its bound) of a gradient g by the logits with the probabilities p; extra: the size of what
    its factors are made of, per row. halves: g goes into the products as two bf16 numbers, so half a step of the second, which is at
    most half a step of the first, is lost."""
    n, v = g.shape
    off = (stat(v) + 512 * U) * (p * extra[:, None]) + (stat(v) + 512 * U) * g.abs()
    off = off + ((R * R if halves else R) if dtype == "bf16" else U) * g.abs()
    half = R if dtype == "bf16" else U
    dh, dh_sum = g @ w, g.abs() @ w.abs()
    out = [dh, off @ w.abs() + v * U * dh_sum + half * dh.abs() + 1e-12]
    if want_dw:
        dw, dw_sum = g.T @ hidden, g.abs().T @ hidden.abs()
        out += [dw, off.T @ hidden.abs() + (2 * n if halves else n) * U * dw_sum + half * dw.abs() + 1e-12]
    else:
        out += [None, None]
    return out


def within(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.detach().double()
    same = (got == want) | ((got - want).abs() <= bound)
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} off, worst by {float(((got - want).abs() / bound).nan_to_num(nan=9e9).max()):.3g} bounds"
