"""Scoring where logits are rounded (ordinary random numbers, not tests/_scoring.py's grid), and rows that are no numbers among
others."""
from __future__ import annotations

import math

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, QuantizedHead, _native, token_logprobs
from mlx_train_perf.core import scoring

pytestmark = pytest.mark.gpu


def _random(n, d, v, *, head, dtype, seed=0, size=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    hidden = torch.randn(n, d, generator=g, device="cuda").to(dt)
    if head == "q4":
        w_q = torch.randint(-2 ** 31, 2 ** 31, (v, d // 8), generator=g, device="cuda").to(torch.int32)
        scales = (size / math.sqrt(d) / 5 * (1 + torch.rand(v, d // 64, generator=g, device="cuda"))).bfloat16()
        return hidden, QuantizedHead(w_q=w_q, scales=scales, biases=(-7.5 * scales.float()).bfloat16())
    return hidden, DenseHead(weight=(torch.randn(v, d, generator=g, device="cuda") * (size / math.sqrt(d))).to(dt), trainable=False)


def _logits(hidden, head, top):
    """(the logits as a forward keeps them, its alternatives)."""
    lib, x = _native.load(), scoring._inputs(hidden, head)
    n = hidden.shape[0]
    z = torch.empty(n, int(lib.mtp_score_logits_ld(x.v)), dtype=torch.float32, device="cuda")
    _, _, top_lp, top_ids, lse, _ = scoring._score_forward(x, None, -100, top, 1.0, z)
    return z[:, :x.v], top_lp, top_ids, lse


@pytest.mark.parametrize(("n", "d", "v", "top", "head", "dtype"), [
    (1400, 64, 50001, 20, "dense", "bf16"), (1400, 72, 50001, 3, "dense", "bf16"), (1400, 192, 50001, 128, "q4", "bf16"),
    (700, 1536, 100003, 8, "dense", "bf16"), (1400, 64, 50001, 20, "dense", "fp32"), (1400, 33, 50001, 2, "dense", "fp32"),
    (1400, 512, 50001, 16, "q4", "fp32")])
@pytest.mark.parametrize("staged", [True, False])
def test_groups_formed_again_have_the_forwards_bits(n, d, v, top, head, dtype, staged, monkeypatch):
    """Alternatives of logits that are not kept are those of the same forward when a caller keeps them, value by value."""
    if not staged:
        if head != "q4":
            pytest.skip("a dense head is not staged")
        monkeypatch.setenv("MTP_LCE_STAGE_HEAD", "0")
    hidden, hd = _random(n, d, v, head=head, dtype=dtype)
    z, lp, ids, _ = _logits(hidden, hd, top)
    value, want = torch.sort(z, dim=1, descending=True, stable=True)
    assert torch.equal(ids, want[:, :top])
    got = token_logprobs(hidden, hd, top=top)
    assert torch.equal(got.top_ids, ids) and torch.equal(got.top_logprobs, lp)


@pytest.mark.parametrize(("n", "v", "dtype"), [(5, 3000, "bf16"), (100, 3000, "bf16"), (300, 3000, "bf16"), (40, 3000, "fp32"), (300, 3000, "fp32")])
def test_near_certain_targets(n, v, dtype):
    """Targets that have all but 1e-1 to 1e-7 of the mass. A logit of d terms has an error of d u |h||w|: log p, and 1 - p in the
    gradient at the target, are off by that and by the logarithm's rounding at the size of a logit."""
    d = 64
    hidden, hd = _random(n, d, v, head="dense", dtype=dtype, seed=n)
    y = torch.arange(n, device="cuda") * 7 % v
    w = hd.weight.double()
    gap = torch.linspace(8, 24, n, device="cuda").double()
    mine = w[y] * (gap / w[y].square().sum(1))[:, None]
    h = (hidden.double() * 0.5 + mine).to(hidden.dtype).requires_grad_(True)
    z = (h.detach().double() @ w.T).requires_grad_(True)
    logp = torch.log_softmax(z, 1).gather(1, y[:, None])[:, 0]
    size = (h.detach().double().abs() @ w.abs().T).amax(1)
    off = 2 * d * S.U * size + S.stat(v) + 8 * S.U * (z.detach().abs().amax(1) + 1)
    got = token_logprobs(h, hd, y)
    assert float(logp.detach().max()) > -2e-5
    assert bool(((got.logprobs.double() - logp).abs() <= off).all())
    (gz,) = torch.autograd.grad(logp.sum(), z)
    (dh,) = torch.autograd.grad(got.logprobs.sum(), h)
    p = torch.softmax(z.detach(), 1)
    hot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    g_off = off[:, None] * (hot + 2 * p * (1 - hot)) + (S.R if dtype == "bf16" else S.U) * gz.abs()
    half = S.R if dtype == "bf16" else S.U
    want = gz @ w
    bound = g_off @ w.abs() + v * S.U * (gz.abs() @ w.abs()) + half * want.abs() + 1e-12
    assert bool(((dh.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [5, 16, 40, 64, 100, 128, 140])
@pytest.mark.parametrize("top", [0, 7])
def test_rows_that_are_no_numbers_leave_the_others(n, top, dtype):
    """NaN and infinities in the first, the last and a middle row: every other row is as without them."""
    hidden, hd = _random(n, 64, 1000, head="dense", dtype=dtype, seed=n)
    y = torch.arange(n, device="cuda")
    want = token_logprobs(hidden, hd, y, top=top)
    bad = hidden.clone()
    bad[0], bad[-1, 0], bad[n // 2, 3] = math.nan, math.inf, -math.inf
    got = token_logprobs(bad, hd, y, top=top)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[[0, n // 2, n - 1]] = False
    assert int(keep.sum()) == n - 3 and bool(torch.isnan(got.entropy[~keep]).all())
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, want, strict=True))
