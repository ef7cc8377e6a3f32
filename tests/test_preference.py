"""The preference and policy losses on the CPU: the definition against differences, impl="reference" against it, and
the refusals (all before any launch)."""
from __future__ import annotations

import math

import pytest
import torch

from mlx_train_perf import _native, policy_loss, preference_loss
from mlx_train_perf.errors import LossInputError, UnsupportedHeadError
from tests import _preference as P


def _near(a, w, tol):
    a, w = a.detach().double(), w.double()
    assert a.shape == w.shape
    assert float((a - w).norm()) <= tol * max(float(w.norm()), 1e-30) or float((a - w).norm()) <= 1e-12


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_preference_definition_and_reference(layout, kind):
    shape, offsets, mask = P.layout(layout, 6, 5, 1)
    nll, _, ref = (x.double() for x in P.tensors(shape, 2))
    smooth = 0.1 if kind == "sigmoid" else 0.0
    g = torch.Generator().manual_seed(0)
    u = torch.randn(shape, generator=g, dtype=torch.float64)
    for reduction in ("mean", "sum", "none"):
        args = {"offsets": offsets, "mask": mask, "beta": 0.3, "kind": kind, "label_smoothing": smooth, "reduction": reduction}
        ct = torch.randn(3, generator=g, dtype=torch.float64) if reduction == "none" else None
        loss, chosen, rejected, grad = P.preference(nll, ref, ct=ct, **args)

        def f(t):
            return float((P.preference(nll + t * u, ref, **args)[0] * (1.0 if ct is None else ct)).sum())

        want = (f(1e-6) - f(-1e-6)) / 2e-6   # 2^-52 |f| / h: 1e-9
        assert abs(float((grad * u).sum()) - want) <= 1e-6 * max(1.0, abs(want))
        x = nll.clone().requires_grad_(True)
        poisoned = ref.clone()
        if mask is not None:
            poisoned[~mask] = math.nan
        got = preference_loss(x, poisoned, impl="reference", **args)
        (d,) = torch.autograd.grad(got.loss, x, ct)
        for a, w in zip((*got, d), (loss, chosen, rejected, grad)):
            _near(a, w, 1e-12)
        assert not got.chosen_rewards.requires_grad


@pytest.mark.parametrize("reduction", ["token", "sequence", "none"])
@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_policy_definition_and_reference(layout, per_token, reduction):
    shape, offsets, mask = P.layout(layout, 6, 5, 3)
    nll, old, ref = (x.double() for x in P.tensors(shape, 4, 1.5))
    g = torch.Generator().manual_seed(1)
    adv = torch.randn(shape if per_token else (6,), generator=g, dtype=torch.float64)
    ct = torch.randn(shape, generator=g, dtype=torch.float64) if reduction == "none" else None
    u = torch.randn(shape, generator=g, dtype=torch.float64)
    for kl in (0.0, 0.3):
        args = {"ref_nll": ref, "offsets": offsets, "mask": mask, "kl_coef": kl, "reduction": reduction, "clip_high": 0.3}
        loss, mean_kl, share, grad = P.policy(nll, old, adv, ct=ct, **args)
        assert 0.1 < float(share) < 0.9

        def f(t):
            return float((P.policy(nll + t * u, old, adv, **args)[0] * (1.0 if ct is None else ct)).sum())

        want = (f(1e-6) - f(-1e-6)) / 2e-6
        assert abs(float((grad * u).sum()) - want) <= 1e-6 * max(1.0, abs(want))
        x = nll.clone().requires_grad_(True)
        got = policy_loss(x, old, adv, impl="reference", **args)
        (d,) = torch.autograd.grad(got.loss, x, ct)
        for a, w in zip((*got, d), (loss, mean_kl, share, grad)):
            _near(a, w, 1e-12)


def test_nothing_counts():
    x = torch.randn(4, 3, requires_grad=True)
    m = torch.zeros(4, 3, dtype=torch.bool)
    for reduction in ("token", "sequence"):
        r = policy_loss(x, x.detach(), torch.ones(4), mask=m, reduction=reduction, impl="reference")
        assert float(r.loss) == 0.0 and float(r.kl) == 0.0 and float(r.clip_fraction) == 0.0
        assert not torch.autograd.grad(r.loss, x)[0].any()
    r = preference_loss(x, x.detach(), mask=m, impl="reference")
    assert abs(float(r.loss) - math.log(2)) < 1e-6 and not torch.autograd.grad(r.loss, x)[0].any()


def test_preference_refusals():
    x = torch.zeros(4, 3)
    flat = torch.zeros(12)

    def bad(what, *a, error=LossInputError, **kw):
        with pytest.raises(error, match=what):
            preference_loss(*a, **{"impl": "reference", **kw})

    bad("reduction", x, x, reduction="token")
    bad("kind", x, x, kind="other")
    for beta in (0.0, -1.0, math.inf, math.nan):
        bad("beta", x, x, beta=beta)
    for e in (-0.1, 0.5, math.nan):
        bad("label_smoothing", x, x, label_smoothing=e)
    bad("label_smoothing belongs", x, x, label_smoothing=0.1, kind="ipo")
    bad("pairs", x[:3], x[:3])
    bad("at least one token", x[:, :0], x[:, :0])
    bad("ref_nll must have nll's shape", x, x[:2])
    bad("ref_nll must be floating", x, x.long())
    bad("nll must be floating", x.long(), x)
    bad("frozen model", x, x.clone().requires_grad_(True))
    bad("mask must be", x, x, mask=torch.ones(4, 2, dtype=torch.bool))
    bad("mask must be", x, x, mask=torch.ones(4, 3))
    bad("or \\(N,\\) with offsets", flat, flat)
    bad("with offsets nll must be", x, x, offsets=torch.tensor([0, 6, 12]))
    bad("offsets must be", flat, flat, offsets=torch.tensor([0.0, 6.0, 12.0]))
    bad("offsets must be", flat, flat, offsets=torch.tensor([0]))
    for o in ([0, 7, 5], [-1, 5, 12], [0, 5, 13]):
        bad("offsets must lie", flat, flat, offsets=torch.tensor(o))
    bad("unknown impl", x, x, impl="other")
    bad("fp32", x.double(), x.double(), impl="kernel", error=UnsupportedHeadError)
    if not torch.cuda.is_available():
        bad("gfx950", x, x, impl="auto", error=UnsupportedHeadError)


def test_policy_refusals():
    x = torch.zeros(4, 3)
    a = torch.zeros(4)

    def bad(what, *args, error=LossInputError, **kw):
        with pytest.raises(error, match=what):
            policy_loss(*args, **{"impl": "reference", **kw})

    bad("reduction", x, x, a, reduction="mean")
    for v in (-0.1, 1.1, math.nan):
        bad("clip_low", x, x, a, clip_low=v)
    for v in (-0.1, math.inf):
        bad("clip_high", x, x, a, clip_high=v)
    bad("kl_coef must", x, x, a, kl_coef=-1.0)
    bad("kl_coef needs", x, x, a, kl_coef=0.1)
    bad("advantages must be", x, x, torch.zeros(3))
    bad("advantages must be", x, x, a.long())
    bad("advantages get no gradient", x, x, a.clone().requires_grad_(True))
    bad("old_nll must have", x, x[:2], a)
    bad("old_nll belongs", x, x.clone().requires_grad_(True), a)
    bad("ref_nll must have", x, x, a, ref_nll=x[0])
    bad("fp32", x, x, a.double(), impl="kernel", error=UnsupportedHeadError)


def test_c_abi_refusals():
    lib = _native.load()
    p, bad, ws_rc = 1 << 20, _native.MTP_ERR_INPUT, _native.MTP_ERR_WORKSPACE

    def pref(pairs=2, n=8, kind=0, beta=0.1, smooth=0.0, red=1, ws=1 << 20, nll=p, workspace=p, offsets=None):
        return lib.mtp_pref_fwd(nll, p, None, offsets, pairs, n, kind, beta, smooth, red, p, p, p, workspace, ws, None)

    for kw in ({"pairs": 0}, {"n": 0}, {"n": 9}, {"kind": 3}, {"kind": -1}, {"beta": 0.0}, {"beta": math.nan}, {"smooth": 0.5},
               {"smooth": 0.1, "kind": 1}, {"red": 3}, {"red": -1}, {"nll": None}, {"pairs": 1 << 40, "offsets": p},
               {"n": 1 << 31, "offsets": p}):
        assert pref(**kw) == bad, kw
    need = lib.mtp_pref_workspace_bytes(2, 8)
    assert need > 0 and pref(ws=need - 1) == ws_rc and pref(workspace=None) == ws_rc
    assert pref(workspace=p + 4) == _native.MTP_ERR_UNSUPPORTED
    assert lib.mtp_pref_workspace_bytes(0, 8) == 0 and lib.mtp_policy_workspace_bytes(1, 0) == 0
    assert lib.mtp_pref_bwd(None, p, None, None, 2, 8, 1, p, None) == bad and lib.mtp_pref_bwd(p, p, None, None, 2, 9, 1, p, None) == bad

    def policy(rows=4, n=8, lo=0.2, hi=0.2, kl=0.0, red=1, ref=None, ws=1 << 20, old=p):
        return lib.mtp_policy_fwd(p, old, ref, p, 0, None, None, rows, n, lo, hi, kl, red, p, p, p, p, ws, None)

    for kw in ({"rows": 0}, {"rows": 3}, {"lo": -0.1}, {"lo": 1.5}, {"hi": -1.0}, {"hi": math.inf}, {"kl": 0.1}, {"kl": -1.0, "ref": p},
               {"red": 2}, {"red": 4}, {"old": None}):
        assert policy(**kw) == bad, kw
    assert policy(ws=0) == ws_rc
    assert lib.mtp_policy_bwd(p, p, p, None, p, 0, None, None, 4, 8, 0.2, 0.2, 0.1, 1, p, p, None) == bad


def test_c_abi_refuses_tokens_that_end_past_32_bits():
    """A workgroup takes 2048 tokens and counts them in 32 bits, those behind the last one too."""
    lib = _native.load()
    p, n, rows = 1 << 20, (1 << 31) - 2048, 1 << 10
    assert lib.mtp_pref_workspace_bytes(rows // 2, n) > 0 and lib.mtp_policy_workspace_bytes(rows, n) > 0
    for more in (n + rows, (1 << 31) - rows):
        assert lib.mtp_pref_workspace_bytes(rows // 2, more) == 0 and lib.mtp_policy_workspace_bytes(rows, more) == 0
        assert lib.mtp_pref_fwd(p, p, None, None, rows // 2, more, 0, 0.1, 0.0, 1, p, p, p, p, 1 << 40, None) == _native.MTP_ERR_INPUT
        assert lib.mtp_pref_bwd(p, p, None, None, rows // 2, more, 1, p, None) == _native.MTP_ERR_INPUT
        assert lib.mtp_policy_fwd(p, p, None, p, 0, None, None, rows, more, 0.2, 0.2, 0.0, 1, p, p, p, p, 1 << 40, None) == _native.MTP_ERR_INPUT
        assert lib.mtp_policy_bwd(p, p, p, None, p, 0, None, None, rows, more, 0.2, 0.2, 0.0, 1, p, p, None) == _native.MTP_ERR_INPUT


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_infinite_ratios(dtype):
    """A token that one model rules out: what the formulas leave of it is finite where a factor of 0 or a border stands."""
    P.check_infinite(lambda t: t.to(dtype), impl="reference")
