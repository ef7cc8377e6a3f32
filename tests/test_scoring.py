"""Token scoring and distillation on the CPU: the reference impl against plain formulas and differences, and the refusals."""
from __future__ import annotations

import math

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, QuantizedHead, distillation_loss, token_logprobs
from mlx_train_perf.errors import LossInputError, UnsupportedHeadError

EXACT = 1e-11   # 64-bit arithmetic: 2^-52 times what a few thousand terms and logarithms below 100 can gather


@pytest.mark.parametrize("head", ["dense", "trainable", "q4"])
@pytest.mark.parametrize(("n", "d", "v", "top", "temperature"), [(1, 64, 97, 97, 1.0), (6, 64, 130, 5, 0.7), (5, 128, 40, 0, 2.0)])
def test_reference_scoring_is_the_formula(n, d, v, top, temperature, head):
    hidden, hd, w = S.make(n, d, v, head=head, dtype="fp32" if head == "q4" else "fp64", seed=n)
    targets = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(1))
    if n > 2:
        targets[1] = -100
        hidden[1] = math.nan
    live = targets != -100
    hd = S.to(hd, "cpu")
    hidden.requires_grad_(True)
    got = token_logprobs(hidden, hd, targets, top=top, temperature=temperature, impl="reference")
    z = S.logits(hidden.detach(), w, live)
    logprobs, entropy, best, ids = S.score(z, targets, live, temperature, top)
    tol = EXACT if hidden.dtype == torch.float64 else 64 * S.U
    for a, b, what in ((got.logprobs, logprobs, "logprobs"), (got.entropy, entropy, "entropy"), (got.top_logprobs, best, "top")):
        S.within(a, b, tol, what)
    assert torch.equal(got.top_ids, ids)
    a, b = torch.randn(2, n, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    (g,) = torch.autograd.grad((logprobs * a).sum() + (entropy * b).sum(), z)
    leaves = [hidden] + ([hd.weight] if head == "trainable" else [])
    grads = torch.autograd.grad((got.logprobs * a).sum() + (got.entropy * b).sum(), leaves)
    S.within(grads[0], g @ w, 1e-9 if hidden.dtype == torch.float64 else 1e-4, "d_hidden")
    if head == "trainable":
        S.within(grads[1], g.T @ torch.where(live[:, None], hidden.detach(), 0.0), 1e-9, "d_weight")


KINDS = [("forward", False), ("forward", True), ("reverse", False), ("jsd", False), ("jsd", True)]


@pytest.mark.parametrize(("kind", "renormalize"), KINDS)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reference_distillation_is_the_formula(kind, renormalize, reduction):
    n, d, v, k = 14, 64, 50, 6
    hidden, hd, w = S.make(n, d, v, dtype="fp64", seed=5)
    ids, lp, mask = S.teacher_list(n, v, k, renormalize=renormalize)
    hidden[~mask] = math.nan
    hidden.requires_grad_(True)
    args = {"kind": kind, "beta": 0.3, "temperature": 1.5, "renormalize": renormalize, "reduction": reduction}
    got = distillation_loss(hidden, hd, ids, lp, mask=mask, impl="reference", **args)
    z = S.logits(hidden.detach(), w, mask)
    want, live = S.distill(z, ids, lp, mask, **args)
    S.within(got, want, EXACT * 100, "loss")
    ct = torch.randn(want.shape, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
    (g,) = torch.autograd.grad(want, z, ct)
    (dh,) = torch.autograd.grad(got, hidden, ct)
    S.within(dh, g @ w, 1e-9, "d_hidden")
    assert bool((dh[~live] == 0).all())


@pytest.mark.parametrize(("kind", "renormalize"), KINDS)
def test_reference_distillation_gradient_against_differences(kind, renormalize):
    hidden, hd, _ = S.make(4, 64, 20, dtype="fp64", seed=9)
    ids, lp, _ = S.teacher_list(4, 20, 5, renormalize=renormalize, holes=False)
    weight = hd.weight.clone().requires_grad_(True)
    hidden = (hidden / 8).requires_grad_(True)

    def f(h, w):
        return distillation_loss(h, DenseHead(weight=w, trainable=True), ids, lp, kind=kind, renormalize=renormalize,
                                 temperature=1.3, impl="reference", reduction="none")

    assert torch.autograd.gradcheck(f, (hidden, weight), eps=1e-6, atol=1e-6)


def test_reference_scoring_gradient_against_differences():
    hidden, hd, _ = S.make(4, 64, 20, dtype="fp64", seed=9)
    weight = hd.weight.clone().requires_grad_(True)
    hidden = (hidden / 8).requires_grad_(True)
    y = torch.tensor([1, -100, 19, 0])

    def f(h, w):
        r = token_logprobs(h, DenseHead(weight=w, trainable=True), y, temperature=0.8, impl="reference")
        return r.logprobs, r.entropy

    assert torch.autograd.gradcheck(f, (hidden, weight), eps=1e-6, atol=1e-6)


def test_a_teacher_that_is_the_student_has_no_divergence():
    hidden, hd, _ = S.make(8, 64, 60, dtype="fp64", seed=2)
    t = token_logprobs(hidden, hd, top=10, impl="reference")
    for kind in ("forward", "reverse", "jsd"):
        loss = distillation_loss(hidden, hd, t.top_ids, t.top_logprobs, kind=kind, reduction="none", impl="reference")
        assert float(loss.abs().max()) < 1e-12


def test_shapes_and_masks():
    hidden, hd, _ = S.make(6, 64, 30, dtype="fp32")
    h3 = hidden.reshape(2, 3, 64)
    r = token_logprobs(h3, hd, torch.zeros(2, 3, dtype=torch.int32), top=4, impl="reference")
    assert r.logprobs.shape == r.entropy.shape == (2, 3) and r.top_ids.shape == r.top_logprobs.shape == (2, 3, 4)
    assert token_logprobs(h3, hd, impl="reference").logprobs is None
    ids, lp, mask = S.teacher_list(6, 30, 3, holes=False)
    loss = distillation_loss(h3, hd, ids.view(2, 3, 3), lp.view(2, 3, 3), mask=mask.view(2, 3), reduction="none", impl="reference")
    assert loss.shape == (2, 3)
    none = distillation_loss(h3, hd, ids.view(2, 3, 3), lp.view(2, 3, 3), mask=torch.zeros(2, 3, dtype=torch.uint8), impl="reference")
    assert float(none) == 0.0


def _score(**kw):
    hidden, hd, _ = S.make(4, 64, 30, dtype="fp32")
    args = {"hidden": hidden, "head": hd, "targets": torch.zeros(4, dtype=torch.int64), "impl": "reference", **kw}
    return token_logprobs(args.pop("hidden"), args.pop("head"), args.pop("targets"), **args)


@pytest.mark.parametrize("kw", [{"hidden": torch.zeros(4)}, {"targets": torch.zeros(3, dtype=torch.int64)}, {"targets": torch.zeros(4)},
                                {"targets": torch.full((4,), 30)}, {"targets": torch.full((4,), -1)}, {"top": -1}, {"top": 31}, {"top": 2.5},
                                {"temperature": 0.0}, {"temperature": math.nan}, {"temperature": 1e4}, {"impl": "other"},
                                {"ignore_index": 0.5}, {"hidden": torch.zeros(4, 32)}, {"hidden": torch.zeros(4, 64, dtype=torch.bfloat16)}])
def test_scoring_refuses(kw):
    with pytest.raises(LossInputError):
        _score(**kw)


def _distill(**kw):
    hidden, hd, _ = S.make(4, 64, 30, dtype="fp32")
    ids, lp, _ = S.teacher_list(4, 30, 3, holes=False)
    args = {"hidden": hidden, "head": hd, "ids": ids, "lp": lp, "impl": "reference", **kw}
    return distillation_loss(args.pop("hidden"), args.pop("head"), args.pop("ids"), args.pop("lp"), **args)


@pytest.mark.parametrize("kw", [{"ids": torch.zeros(4, dtype=torch.int64)}, {"ids": torch.zeros(4, 3)}, {"ids": torch.zeros(4, 3, dtype=torch.bool)}, {"ids": torch.zeros(4, 3, dtype=torch.int32).view(torch.uint32)},
                                {"ids": torch.full((4, 3), 30)},
                                {"ids": torch.zeros(4, 0, dtype=torch.int64), "lp": torch.zeros(4, 0)}, {"lp": torch.zeros(4, 2)},
                                {"lp": torch.zeros(4, 3, dtype=torch.int64)}, {"lp": torch.zeros(4, 3, requires_grad=True)},
                                {"mask": torch.ones(3, dtype=torch.bool)}, {"mask": torch.ones(4)}, {"kind": "other"},
                                {"kind": "jsd", "beta": 0.0}, {"kind": "jsd", "beta": 1.0}, {"kind": "reverse", "renormalize": True},
                                {"temperature": -1.0}, {"reduction": "token"}, {"impl": "other"}, {"hidden": torch.zeros(4)}])
def test_distillation_refuses(kw):
    with pytest.raises(LossInputError):
        _distill(**kw)


def test_kernel_impl_refuses_what_it_does_not_serve():
    hidden, hd, _ = S.make(4, 64, 300, dtype="fp32")
    with pytest.raises(UnsupportedHeadError, match="reference"):
        token_logprobs(hidden.double(), DenseHead(weight=hd.weight.double()), impl="kernel")
    with pytest.raises(UnsupportedHeadError, match="at most 128"):
        token_logprobs(hidden, hd, top=129, impl="kernel")
    with pytest.raises(UnsupportedHeadError, match="at most 128"):
        distillation_loss(hidden, hd, torch.zeros(4, 129, dtype=torch.int64), torch.zeros(4, 129), impl="kernel")
    wide = DenseHead(weight=torch.zeros(1, 64).expand(2 ** 21 + 1, 64))
    with pytest.raises(UnsupportedHeadError, match="2\\^21"):
        token_logprobs(hidden, wide, impl="kernel")
    q = QuantizedHead(w_q=torch.zeros(8, 16, dtype=torch.int32), scales=torch.zeros(8, 1), biases=torch.zeros(8, 1), bits=8)
    with pytest.raises(UnsupportedHeadError, match="4-bit"):
        token_logprobs(torch.zeros(4, 64), q, impl="kernel")


def _call(name, **kw):
    from mlx_train_perf import _native as N

    lib = N.load()
    p = 1 << 20   # a pointer that nothing reads: every call here is refused before a launch
    base = {"logprobs": {"head": (p, p, None, None, None), "targets": p, "n": 4, "d": 64, "v": 100, "kind": 0, "top": 3, "t": 1.0,
                         "out": (p, p, p, p, p, p, None), "ws": p, "bytes": 1 << 40},
            "distill": {"head": (p, p, None, None, None), "lists": (p, p, None), "n": 4, "d": 64, "v": 100, "kind": 0, "k": 3,
                        "loss": 0, "beta": 0.5, "t": 1.0, "renorm": 0, "red": 1, "out": (p, p, p, p, p, p, None), "ws": p,
                        "bytes": 1 << 40}}[name]
    a = {**base, **kw}
    if name == "logprobs":
        return lib.mtp_logprobs_fwd(*a["head"], a["targets"], a["n"], a["d"], a["v"], a["kind"], -100, a["top"], a["t"], *a["out"],
                                    a["ws"], a["bytes"], None)
    return lib.mtp_distill_fwd(*a["head"], *a["lists"], a["n"], a["d"], a["v"], a["kind"], a["k"], a["loss"], a["beta"], a["t"],
                               a["renorm"], a["red"], *a["out"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize(("name", "kw", "code"), [
    ("logprobs", {"n": 0}, -1), ("logprobs", {"v": 2 ** 21 + 1}, -2), ("logprobs", {"d": 63}, -2), ("logprobs", {"top": -1}, -1),
    ("logprobs", {"top": 101}, -1), ("logprobs", {"top": 129, "v": 1000}, -2), ("logprobs", {"t": 0.0}, -1),
    ("logprobs", {"t": math.nan}, -1), ("logprobs", {"bytes": 16}, -3), ("logprobs", {"ws": None}, -3), ("logprobs", {"ws": 8}, -2), ("logprobs", {"out": (1 << 20,) * 6 + (8,)}, -2),
    ("logprobs", {"out": (None,) * 7}, -1), ("logprobs", {"head": (8, 16, None, None, None)}, -2), ("logprobs", {"kind": 1}, -1),
    ("distill", {"k": 0}, -2), ("distill", {"k": 129}, -2), ("distill", {"loss": 3}, -1), ("distill", {"loss": 2, "beta": 1.0}, -1),
    ("distill", {"loss": 1, "renorm": 1}, -1), ("distill", {"red": 3}, -1), ("distill", {"lists": (None, None, None)}, -1),
    ("distill", {"bytes": 16}, -3), ("distill", {"t": 2e3}, -1)])
def test_entry_points_refuse_before_a_launch(name, kw, code):
    assert _call(name, **kw) == code


def test_workspaces():
    from mlx_train_perf import _native as N

    lib = N.load()
    for n in (1, 128, 129, 2048, 4096, 16384, 16385, 100000):
        for top in (0, 1, 128):
            ws = lib.mtp_logprobs_fwd_workspace_bytes(n, 512, 32000, 0, top, 0)
            rows, partials = min(n, 16384), 8 << 20
            if n <= 128 or (top and n * 32000 * 4 <= 256 << 20):   # the logits, and each group's maximum (and sums)
                most = n * (32128 * 4 + 3 * 252 * 4)
            else:   # the groups that a row's alternatives are looked for in
                most = rows * top * (128 * 4 + 16) + rows * (252 + 1) * 4
            assert 0 < ws <= most + partials
    assert lib.mtp_logprobs_fwd_workspace_bytes(0, 64, 100, 0, 1, 0) == 0
    assert lib.mtp_logprobs_fwd_workspace_bytes(8, 64, 2 ** 21 + 1, 0, 1, 0) == 0
    # a staged 4-bit head adds its rows, a few tokens none
    staged, plain = (lib.mtp_logprobs_fwd_workspace_bytes(1000, 512, 32000, k, 4, 0) for k in (N.HEAD_Q4_STAGED, N.HEAD_Q4))
    assert staged == plain + 32000 * 512 * 2
    assert lib.mtp_logprobs_fwd_workspace_bytes(8, 512, 32000, N.HEAD_Q4_STAGED, 4, 0) == lib.mtp_logprobs_fwd_workspace_bytes(8, 512, 32000, N.HEAD_Q4, 4, 0)
    lce = lib.mtp_lce_bwd_workspace_bytes(300, 64, 1000, 0, 1024, 300)
    assert lib.mtp_score_bwd_workspace_bytes(300, 64, 1000, 0, 1024, 300, 5, 1) >= lce + 300 * (12 + 20) + 300 * 64 * 2
