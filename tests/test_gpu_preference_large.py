"""GPU: the preference and policy losses on batches that take two launches, at the borders between one launch and two, and on
views off a 16-byte boundary, against their definition in 64 bits, vectorized.

Tolerance: as test_gpu_preference.py, whose per-token errors do not grow with the number of tokens: sums are in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _preference as P

pytestmark = pytest.mark.gpu

TOL = 2e-6
# 64 sequences or fewer: one launch up to 8192 tokens (policy), 16384 (preference); more: up to 4096 tokens of 512 sequences.
# Then more pairs than join threads, and many parts of a sequence.
SIZES = [(2, 8193), (64, 80), (66, 80), (512, 8), (2600, 20), (4, 30011)]


def _keep(shape, offsets, mask):
    """(owner of each token, whether it counts), flat."""
    n = math.prod(shape)
    at = torch.arange(n)
    if offsets is None:
        owner = at // shape[1]
        keep = torch.ones(n, dtype=torch.bool)
    else:
        owner = torch.searchsorted(offsets, at, right=True) - 1
        keep = (owner >= 0) & (at < offsets[-1])
        owner = owner.clamp(0, len(offsets) - 2)
    return owner, keep if mask is None else keep & mask.reshape(-1)


def _sums(x, owner, rows):
    return torch.zeros(rows, dtype=torch.float64).index_add(0, owner, x.double())


def _preference(nll, ref, offsets, mask, rows, *, beta, kind, reduction, label_smoothing, ct):
    owner, keep = _keep(nll.shape, offsets, mask)
    gap = torch.where(keep, ref.reshape(-1).double() - nll.reshape(-1).double(), 0.0)
    count = _sums(keep, owner, rows).clamp(min=1) if kind == "ipo" else torch.ones(rows, dtype=torch.float64)
    g = _sums(gap, owner, rows) / count
    chosen, rejected = beta * g[:rows // 2], beta * g[rows // 2:]
    d = chosen - rejected
    if kind == "sigmoid":
        loss = -(1 - label_smoothing) * torch.nn.functional.logsigmoid(d) - label_smoothing * torch.nn.functional.logsigmoid(-d)
        slope = label_smoothing - torch.sigmoid(-d)
    elif kind == "hinge":
        loss, slope = (1 - d).clamp(min=0), -(d < 1).double()
    else:
        h = (d - 0.5) / beta
        loss, slope = h ** 2, 2 * h / beta
    up = ct.double() if reduction == "none" else torch.full_like(d, 1 / len(d) if reduction == "mean" else 1.0)
    total = {"none": loss, "mean": loss.mean(), "sum": loss.sum()}[reduction]
    coef = torch.cat([-slope * up, slope * up]) * beta / count   # d g / d nll = -1 / count
    return [total, chosen, rejected, torch.where(keep, coef[owner], 0.0).reshape(nll.shape)]


def _policy(nll, old, adv, ref, offsets, mask, rows, *, clip_low, clip_high, kl_coef, reduction, ct):
    owner, keep = _keep(nll.shape, offsets, mask)

    def at(t):
        return torch.where(keep, t.reshape(-1).double(), 0.0)

    x = at(nll)
    a = at(adv) if adv.shape == nll.shape else torch.where(keep, adv.double()[owner], 0.0)
    u = torch.exp(at(old) - x)
    c = u.clamp(1 - clip_low, 1 + clip_high)
    out = c * a < u * a
    loss, slope = -torch.minimum(u * a, c * a), torch.where(out, 0.0, u * a)
    kl = torch.zeros_like(x)
    if ref is not None:
        d = x - at(ref)
        kl = torch.expm1(d) - d
        loss, slope = loss + kl_coef * kl, slope + kl_coef * torch.expm1(d)
    loss, slope = torch.where(keep, loss, 0.0), torch.where(keep, slope, 0.0)
    n = keep.sum().clamp(min=1).double()
    if reduction == "none":
        total, weight = loss.reshape(nll.shape), ct.reshape(-1).double()
    elif reduction == "token":
        total, weight = loss.sum() / n, 1 / n
    else:
        per = _sums(keep, owner, rows)
        filled = (per > 0).sum().double()
        total, weight = (_sums(loss, owner, rows) / per.clamp(min=1)).sum() / filled, 1 / (per.clamp(min=1)[owner] * filled)
    return [total, kl.sum() / n, (out & keep).sum() / n, (slope * weight).reshape(nll.shape)]


def _place(t, off):
    """t on the GPU; with `off`, contiguous but one element past an aligned address."""
    if t is None:
        return None
    t = t.cuda()
    if not off:
        return t
    base = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    view = base[1:].view(t.shape)
    view.copy_(t)
    assert view.data_ptr() % 16 and view.is_contiguous()
    return view


def _compare(got, want, floor):
    for name, a, w in zip(("loss", "second", "third", "d_nll"), got, want):
        a = a.detach().double().cpu()
        assert a.shape == w.shape, name
        assert float((a - w).norm()) <= TOL * max(float(w.norm()), floor if name == "loss" else 0.0), (name, a, w)


def _check_preference(layout, seqs, t, kind, off):
    from mlx_train_perf import preference_loss

    shape, offsets, mask = P.layout(layout, seqs, t, t)
    nll, _, ref = P.tensors(shape, seqs)
    if mask is not None:
        nll[~mask], ref[~mask] = math.nan, math.inf
    g = torch.Generator().manual_seed(1)
    for reduction, smooth in (("mean", 0.0), ("none", 0.2), ("sum", 0.1)):
        args = {"beta": 0.02, "kind": kind, "reduction": reduction, "label_smoothing": smooth if kind == "sigmoid" else 0.0}
        ct = torch.randn(seqs // 2, generator=g) if reduction == "none" else None
        x = _place(nll, off).requires_grad_(True)
        r = preference_loss(x, _place(ref, off), offsets=_place(offsets, False), mask=_place(mask, off), **args)
        (d,) = torch.autograd.grad(r.loss, x, _place(ct, off))
        _compare([*r, d], _preference(nll, ref, offsets, mask, seqs, ct=ct, **args), 0.0)


def _check_policy(layout, seqs, t, reduction, off):
    from mlx_train_perf import policy_loss

    shape, offsets, mask = P.layout(layout, seqs, t, t)
    nll, old, ref = P.tensors(shape, seqs, 1.5)
    g = torch.Generator().manual_seed(2)
    if mask is not None:
        nll[~mask], old[~mask], ref[~mask] = math.nan, math.inf, math.nan
    for per_token, kl, with_ref in ((False, 0.0, False), (True, 0.3, True), (False, 0.0, True)):
        adv = torch.randn(shape if per_token else (seqs,), generator=g)
        if per_token and mask is not None:
            adv[~mask] = math.nan
        ct = torch.randn(shape, generator=g) if reduction == "none" else None
        args = {"kl_coef": kl, "reduction": reduction, "clip_low": 0.1, "clip_high": 0.25}
        x, r = _place(nll, off).requires_grad_(True), ref if with_ref else None
        got = policy_loss(x, _place(old, off), _place(adv, off), ref_nll=_place(r, off), offsets=_place(offsets, False),
                          mask=_place(mask, off), **args)
        (d,) = torch.autograd.grad(got.loss, x, _place(ct, off))
        # a mean of terms of either sign, of size |A|: held against that
        _compare([*got, d], _policy(nll, old, adv, r, offsets, mask, seqs, ct=ct, **args), 1.0 if reduction != "none" else 0.0)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize(("seqs", "t"), SIZES)
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_preference(layout, seqs, t, kind):
    _check_preference(layout, seqs, t, kind, False)


@pytest.mark.parametrize("reduction", ["token", "sequence", "none"])
@pytest.mark.parametrize(("seqs", "t"), SIZES)
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_policy(layout, seqs, t, reduction):
    _check_policy(layout, seqs, t, reduction, False)


@pytest.mark.parametrize(("seqs", "t"), [(6, 37), (40, 1500)])
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_views_off_a_boundary(layout, seqs, t):
    for kind in ("sigmoid", "ipo"):
        _check_preference(layout, seqs, t, kind, True)
    for reduction in ("token", "sequence", "none"):
        _check_policy(layout, seqs, t, reduction, True)
