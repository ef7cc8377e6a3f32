"""GPU: scored attention at the ends of its range, against the plain form in 64 bits: biases far larger than the scores,
caps that all scores exceed.

Tolerances beside those of test_gpu_scored_attention.py (BAR, and U for D, which its `_scored.attention` explains): the
bias of a key is slope times its distance less that of the row's highest bias, a whole number, so its rounding counts by
the bias within reach of that key alone: 4 roundings (bias, score, L, their difference) of 2^-24 of it."""
from __future__ import annotations

import pytest
import torch

from tests import _scored as S

pytestmark = pytest.mark.gpu

BAR = {torch.bfloat16: 1e-2, torch.float32: 2e-5}
U = {torch.bfloat16: 2 ** -8, torch.float32: 2e-6}


def _form(q, k, v, d_o, *, scale, see, away, cap=None, slopes=None):
    """(o, dq, dk, dv), then the bounds of what a relative error of O does to dq and dk (through D), and of what an absolute
    error of 1 - tanh^2 does, each for an error of 1. q, d_o (hq, s, dh), k, v (hkv, w, dh); see, away (s, w)."""
    q, k, v, d_o = (x.double() for x in (q, k, v, d_o))
    o, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    tq, tk, bq, bk = (torch.zeros_like(x) for x in (q, k, q, k))
    for h in range(q.shape[0]):
        n = h // (q.shape[0] // k.shape[0])
        x = scale * (q[h] @ k[n].T)
        bend = torch.ones_like(x)
        if cap is not None:
            bend = 1 / torch.cosh(x / cap) ** 2
            x = cap * torch.tanh(x / cap)
        if slopes is not None:
            x = x - float(slopes[h]) * away
        x = torch.where(see, x, -torch.inf)
        p = torch.where(see, torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e300)), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        o[h] = p @ v[n]
        gap = torch.where(see, d_o[h] @ v[n].T - (d_o[h] * o[h]).sum(1, keepdim=True), 0.0)
        ds = p * gap * bend
        dq[h] = scale * (ds @ k[n])
        dk[n] += scale * (ds.T @ q[h])
        dv[n] += p.T @ d_o[h]
        off = (d_o[h].abs() * (o[h].abs() + p @ v[n].abs())).sum(1, keepdim=True)
        tq[h] = scale * off * ((p * bend) @ k[n]).abs()
        tk[n] += scale * ((p * bend * off).T @ q[h].abs())
        bq[h] = scale * ((p * gap.abs()) @ k[n].abs())
        bk[n] += scale * ((p * gap.abs()).T @ q[h].abs())
    return (o, dq, dk, dv), {"dq": (tq, bq), "dk": (tk, bk)}


def _compare(got, want, terms, dtype, bar, bend=0.0):
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(a).all(), name
        more = 0.0
        if name in terms:
            t, b = terms[name]
            more = U[dtype] * float(t.norm()) + bend * float(b.norm())
        assert float((a.double() - w).norm()) <= bar * float(w.norm()) + more, (name, S.rel(a, w), more / float(w.norm()))


def _step(q, k, v, d_o, **kw):
    from mlx_train_perf.attention import flash_attention

    qs = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = flash_attention(*qs, **kw)
    return [o.detach(), *torch.autograd.grad(o, qs, d_o)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap", [None, 20.0, 100.0])
@pytest.mark.parametrize("dh", [64, 96, 128])
def test_keys_far_away(dh, cap, dtype):
    """Every query sees the row's first 16 keys, up to 60000 positions before it, under biases of up to 240000 (of which
    fp32 steps are 2^-7 to 2^-6) that differ by at most 4 * 16 within a row: fp32 4 * 64 * 2^-24 = 1.5e-5 on top, and sums
    of 60000 terms sqrt(60000) * 2^-24 = 1.5e-5."""
    from mlx_train_perf.attention import SpanMask

    hq, hkv, s, w = 4, 2, 60003, 16
    print(f"[far] dh={dh} cap={cap} {dtype}", flush=True)
    q, k, v, d_o = (x.cuda() for x in S.inputs(1, hq, hkv, s, dh, dtype, dh, std=3.0))
    slopes = torch.tensor([4.0, -4.0, -0.5, 0.3])
    zero = torch.zeros(1, s, dtype=torch.int32, device="cuda")
    got = _step(q, k, v, d_o, scale=dh ** -0.5, softcap=cap, slopes=slopes.cuda(), spans=SpanMask(start=zero, end=zero + w))
    away = (torch.arange(s, device="cuda")[:, None] - torch.arange(w, device="cuda")).abs().double()
    want, terms = _form(q[0], k[0, :, :w], v[0, :, :w], d_o[0], scale=dh ** -0.5, see=away >= 0, away=away, cap=cap, slopes=slopes)
    for x in got[2:]:
        assert not x[:, :, w:].any()
    got = [x[0] if n < 2 else x[0, :, :w] for n, x in enumerate(got)]
    _compare(got, want, terms, dtype, BAR[dtype] + (3e-5 if dtype == torch.float32 else 0.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("mask", "cap"), [("causal", None), ("full", None), ("behind", None), ("causal", 30.0), ("behind", 30.0)])
def test_steep_slopes_on_long_rows(mask, cap, dtype):
    """Slopes of hundreds below 0 over 12000 positions, biases of up to 6e6: nearly all of a row is one far key. `behind`: a
    window that ends 700 positions before its query, at slopes of either sign. A key beside the highest differs by the slope
    itself, 4 * 500 * 2^-24 = 1.2e-4, of a probability of e^-40 at most where slopes are steep."""
    from mlx_train_perf.attention import SpanMask

    hq, hkv, s, dh = 4, 2, 12011, 64
    print(f"[steep] {mask} cap={cap} {dtype}", flush=True)
    q, k, v, d_o = (x.cuda() for x in S.inputs(1, hq, hkv, s, dh, dtype, 5))
    slopes = torch.tensor([-500.0, -300.0, -0.01, 100.0 if mask == "behind" else -1.0])
    i = torch.arange(s, device="cuda")
    spans = None
    see = i[:, None] >= i[None] if mask == "causal" else torch.ones(s, s, dtype=torch.bool, device="cuda")
    if mask == "behind":
        start, end = (i - 900).clamp(min=0), (i - 700).clamp(min=0)
        see = (i[None] >= start[:, None]) & (i[None] < end[:, None])
        spans = SpanMask(start=start.to(torch.int32)[None], end=end.to(torch.int32)[None])
    got = _step(q, k, v, d_o, scale=dh ** -0.5, causal=mask == "causal", softcap=cap, slopes=slopes.cuda(), spans=spans)
    away = (i[:, None] - i[None]).abs().double()
    want, terms = _form(q[0], k[0], v[0], d_o[0], scale=dh ** -0.5, see=see, away=away, cap=cap, slopes=slopes)
    # sums of up to 12011 terms: 110 * 2^-24 = 7e-6, within the bar's own 20 of 400
    _compare([x[0] for x in got], want, terms, dtype, BAR[dtype])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize(("cap", "std"), [(0.5, 30.0), (3.0, 30.0), (3.0, 8.0), (20.0, 100.0)])
@pytest.mark.parametrize("dh", [64, 96, 128])
def test_gradients_of_scores_above_the_cap(dh, cap, std, biased, dtype):
    """Where scores exceed the cap, 1 - tanh^2 is the small difference of numbers near 1: off by 2^-21 at most. bf16 kernels:
    v = -1 / (1 + e) with its sum, reciprocal and exponential within 2^-24 of 1 each and a factor 4 behind v + v^2; fp32: tanhf
    within 2 ulp, 2^-23, twice that in its square. What that does to dq and dk is bounded by sums of P |dP - D| |k| and |q|."""
    hq, hkv, s = 2, 1, 190
    q, k, v, d_o = (x.cuda() for x in S.inputs(1, hq, hkv, s, dh, dtype, 12, std))
    slopes = torch.tensor([0.2, -0.05]) if biased else None
    got = _step(q, k, v, d_o, scale=dh ** -0.5, softcap=cap, slopes=None if slopes is None else slopes.cuda())
    i = torch.arange(s, device="cuda")
    away = (i[:, None] - i[None]).abs().double()
    want, terms = _form(q[0], k[0], v[0], d_o[0], scale=dh ** -0.5, see=i[:, None] >= i[None], away=away, cap=cap, slopes=slopes)
    # fp32: scores reach 4 std, of which 2^-24 (100: 2.4e-5) is also an error of x in the derivative's 2 x / cap
    more = 0.0 if dtype == torch.bfloat16 else 4 * std * 2 ** -24 * (1 + 2 / cap)
    _compare([x[0] for x in got], want, terms, dtype, BAR[dtype] + more, bend=2 ** -21)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("mask", "cap"), [("causal", None), ("full", None), ("ragged", None), ("window", 20.0), ("causal", 20.0), ("full", 90.0)])
def test_logarithms_count_from_the_highest_bias(mask, cap, dtype):
    """L of the C entry points is that of the scores less the highest bias of a row's visible keys, +inf where it sees none.
    Scores of up to 2^5 in four roundings, 4 * 2^5 * 2^-24 = 8e-6, the logarithm's own, and 2^-22 of a cap: 5e-5 is twice that.
    bf16 kernels: a tile's biases are slope * c, c < 64, and a term of the tile: the product begins from the former (one
    rounding), adds up over dh / 16 = 4 steps, is multiplied and added to the latter, itself rounded (2), and L once: 8
    roundings of at most 2^-24 of up to 64 * |slope|."""
    from mlx_train_perf.attention.api import scored_forward

    hq, hkv, s, dh = 4, 2, 301, 64
    q, k, v, _ = (x.cuda() for x in S.inputs(1, hq, hkv, s, dh, dtype, 8))
    slopes = torch.tensor([0.3, -0.3, -5.0, 60.0])
    spans = S.spans_of(mask, 1, s, 4)
    start, end = (None, None) if spans is None else (t.cuda() for t in spans)
    _, lse, _, _ = scored_forward(q, k, v, slopes.cuda(), start, end, scale=dh ** -0.5, causal=mask == "causal", softcap=cap or 0.0)
    see = S.visible(mask, spans, 1, s, "cuda")[0]
    i = torch.arange(s, device="cuda")
    away = (i[:, None] - i[None]).abs().double()
    for h in range(hq):
        x = dh ** -0.5 * (q[0, h].double() @ k[0, h // 2].double().T)
        if cap is not None:
            x = cap * torch.tanh(x / cap)
        bias = torch.where(see, -float(slopes[h]) * away, -torch.inf)
        want = torch.logsumexp(x + bias, 1) - bias.amax(1)
        seen = see.any(1)
        assert torch.isposinf(lse[0, h, ~seen]).all()
        steps = 8 * 64 * abs(float(slopes[h])) * 2 ** -24 if dtype == torch.bfloat16 else 0.0
        assert float((lse[0, h].double() - want)[seen].abs().max()) <= 5e-5 + steps, h
