"""Scoring and distillation at high temperatures over vocabularies whose last tile is partly empty, at one tile or more a
split: a lane may have met nothing but columns past the head's end."""
from __future__ import annotations

import _scoring as S
import pytest
import torch

from mlx_train_perf import distillation_loss, token_logprobs

pytestmark = pytest.mark.gpu

# n, V (few tokens; tiles), temperature
_CALLS = [(n, v, t) for n, v in ((3, 97), (70, 129), (140, 97), (140, 129), (140, 300)) for t in (100.0, 200.0, 400.0, 1000.0)]
_CALLS.append((140, 32003, 200.0))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize(("n", "v", "temperature"), _CALLS)
@pytest.mark.parametrize("top", [0, 4])
def test_scoring(n, v, top, dtype, temperature):
    """Near to even: the entropy is log V but for little, so its bound is that of a sum of p log p with |log p| below 16."""
    hidden, hd, w = S.make(n, 64, v, head="trainable", dtype=dtype, seed=n)
    hd = S.to(hd, "cuda")
    h = hidden.cuda().requires_grad_(True)
    y = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(n))
    got = token_logprobs(h, hd, y.cuda(), top=top, temperature=temperature)
    live = torch.ones(n, dtype=torch.bool)
    z = S.logits(hidden, w, live)
    logprobs, entropy, _, _ = S.score(z, y, live, temperature, 0)
    off = S.stat(v) + 256 * S.U
    S.within(got.logprobs, logprobs, off, "logprobs")
    S.within(got.entropy, entropy, off + 128 * S.stat(v), "entropy")
    if top:
        value, ids = torch.sort(z.detach(), dim=1, descending=True, stable=True)
        assert torch.equal(got.top_ids.cpu(), ids[:, :top])
        S.within(got.top_logprobs, torch.log_softmax(z.detach() / temperature, 1).gather(1, ids[:, :top]), off, "top_logprobs")
    a, b = torch.randn(2, n, generator=torch.Generator().manual_seed(n + 1))
    (gz,) = torch.autograd.grad((logprobs * a.double() + entropy * b.double()).sum(), z)
    grad = torch.autograd.grad((got.logprobs, got.entropy), (h, hd.weight), (a.cuda(), b.cuda()))
    p = torch.softmax(z.detach() / temperature, 1)
    dh, dh_off, dw, dw_off = S.gradient_bounds(gz, p, (a.abs() + 64 * b.abs()).double() / temperature, hidden.double(), w, True, dtype, n <= 128)
    S.within(grad[0], dh, dh_off, "d_hidden")
    S.within(grad[1], dw, dw_off, "d_weight")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize(("n", "v", "temperature"), _CALLS)
def test_distillation(n, v, dtype, temperature):
    """The list has some k / V of the mass: a row's loss is k + 1 terms, their log probabilities off by `off` each (R is near 1)."""
    k = 5
    hidden, hd, w = S.make(n, 64, v, head="trainable", dtype=dtype, seed=n)
    hd = S.to(hd, "cuda")
    ids, lp, mask = S.teacher_list(n, v, k, seed=n)
    for kind in ("forward", "reverse", "jsd"):
        args = {"kind": kind, "beta": 0.4, "temperature": temperature, "renormalize": False, "reduction": "none"}
        z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool))
        want, _ = S.distill(z, ids, lp, mask, **args)
        h = hidden.cuda().requires_grad_(True)
        got = distillation_loss(h, hd, ids.cuda(), lp.cuda(), mask=mask.cuda(), **args)
        S.within(got, want, 32 * (S.stat(v) + 256 * S.U), f"loss, {kind}")
        ct = torch.randn(n, generator=torch.Generator().manual_seed(n + 1))
        (gz,) = torch.autograd.grad(want, z, ct.double())
        grad = torch.autograd.grad(got, (h, hd.weight), ct.cuda())
        p = torch.softmax(z.detach() / temperature, 1)
        dh, dh_off, dw, dw_off = S.gradient_bounds(gz, p, 64 * ct.abs().double() / temperature, hidden.double(), w, True, dtype, n <= 128)
        S.within(grad[0], dh, dh_off, f"d_hidden, {kind}")
        S.within(grad[1], dw, dw_off, f"d_weight, {kind}")
