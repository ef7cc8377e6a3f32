"""Token scoring and distillation kernels against 64-bit formulas (tests/_scoring.py: inputs whose logits are exact, and the
bounds)."""
from __future__ import annotations

import math

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, distillation_loss, linear_cross_entropy, policy_loss, token_logprobs
from mlx_train_perf.core import scoring
from mlx_train_perf.errors import LossInputError

pytestmark = pytest.mark.gpu


def _targets(n, v, seed, ignored=True):
    g = torch.Generator().manual_seed(seed)
    y = torch.randint(0, v, (n,), generator=g)
    if ignored and n > 2:
        y[torch.randperm(n, generator=g)[:max(1, n // 9)]] = -100
    return y


def _check_score(n, d, v, *, top=0, head="dense", dtype="bf16", temperature=1.0, targets=True, seed=0, grads=True, halves=None):
    hidden, hd, w = S.make(n, d, v, head=head, dtype=dtype, seed=seed)
    y = _targets(n, v, seed) if targets else None
    live = torch.ones(n, dtype=torch.bool) if y is None else y != -100
    h = hidden.clone()
    h[~live] = math.nan
    h = h.cuda().requires_grad_(grads)
    hd = S.to(hd, "cuda")
    got = token_logprobs(h, hd, None if y is None else y.cuda(), top=top, temperature=temperature)
    z = S.logits(hidden, w, live)
    logprobs, entropy, best, ids = S.score(z, y, live, temperature, top)
    off = S.stat(v) + 256 * S.U
    assert torch.equal(got.top_ids.cpu(), ids)
    S.within(got.top_logprobs, best, off, "top_logprobs")
    S.within(got.entropy, entropy, off + 128 * S.stat(v), "entropy")
    if y is not None:
        S.within(got.logprobs, logprobs, off, "logprobs")
    if not grads:
        return
    g0 = torch.Generator().manual_seed(seed + 1)
    a, b = torch.randn(2, n, generator=g0)
    outs, cts, total = [got.entropy], [torch.where(live, b, math.nan).cuda()], (entropy * b.double()).sum()
    if y is not None:
        outs, cts, total = [got.logprobs, *outs], [torch.where(live, a, math.nan).cuda(), *cts], total + (logprobs * a.double()).sum()
    else:
        a = torch.zeros(n)
    (gz,) = torch.autograd.grad(total, z)
    want_dw = head == "trainable"
    grad = torch.autograd.grad(outs, [h] + ([hd.weight] if want_dw else []), cts)
    p = torch.softmax(z.detach() / temperature, 1)
    extra = (a.abs() + 64 * b.abs()).double() / temperature
    clean = torch.where(live[:, None], hidden.double(), 0.0)
    dh, dh_off, dw, dw_off = S.gradient_bounds(gz, p, extra, clean, w, want_dw, dtype, n <= 128 if halves is None else halves)
    S.within(grad[0], dh, dh_off, "d_hidden")
    if want_dw:
        S.within(grad[1], dw, dw_off, "d_weight")


def _check_distill(n, d, v, k, *, head="dense", dtype="bf16", kind="forward", renormalize=False, reduction="mean", temperature=1.0,
                   beta=0.4, seed=0, holes=True, halves=None):
    hidden, hd, w = S.make(n, d, v, head=head, dtype=dtype, seed=seed)
    ids, lp, mask = S.teacher_list(n, v, k, seed=seed, renormalize=renormalize, holes=holes)
    args = {"kind": kind, "beta": beta, "temperature": temperature, "renormalize": renormalize, "reduction": reduction}
    z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool))
    want, live = S.distill(z, ids, lp, mask, **args)
    h = hidden.clone()
    h[~live] = math.nan
    h = h.cuda().requires_grad_(True)
    hd = S.to(hd, "cuda")
    got = distillation_loss(h, hd, ids.cuda(), lp.cuda(), mask=mask.cuda(), **args)
    # A row's loss is made of at most k + 1 terms below 32 in size, each with the log probabilities' error times its weight; the
    # rest's logarithm has the error of the list's sum over the rest, at least the floor's when that is smaller.
    q = torch.softmax(z.detach() / temperature, 1)
    left = torch.ones(n, dtype=torch.float64)
    for i in range(n):
        on = sorted({y for y in ids[i].tolist() if y >= 0})
        left[i] = max(S.TAIL, 1 - float(q[i, on].sum()))
    off = S.stat(v) + 256 * S.U
    row_off = off * (2 + 32 / left.clamp(max=1.0)) if kind != "reverse" else off * 80 + 0 * left
    bound = row_off if reduction == "none" else row_off.sum() / (max(1, int(live.sum())) if reduction == "mean" else 1)
    S.within(got, want, bound + 2 * S.U * want.detach().abs(), "loss")
    ct = torch.randn(want.shape, generator=torch.Generator().manual_seed(seed + 1), dtype=torch.float64)
    (gz,) = torch.autograd.grad(want, z, ct) if bool(live.any()) else (torch.zeros_like(z),)
    want_dw = head == "trainable"
    grad = torch.autograd.grad(got, [h] + ([hd.weight] if want_dw else []), ct.float().cuda())
    scale = ct.abs() if reduction == "none" else ct.abs() / (max(1, int(live.sum())) if reduction == "mean" else 1)
    extra = (scale * torch.ones(n, dtype=torch.float64)) * (64 + 2 / left) / temperature
    clean = torch.where(live[:, None], hidden.double(), 0.0)
    dh, dh_off, dw, dw_off = S.gradient_bounds(gz, q, extra, clean, w, want_dw, dtype, n <= 128 if halves is None else halves)
    S.within(grad[0], dh, dh_off, "d_hidden")
    assert bool((grad[0].cpu()[~live] == 0).all())
    if want_dw:
        S.within(grad[1], dw, dw_off, "d_weight")


# ---- scoring ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("head", ["dense", "trainable", "q4"])
@pytest.mark.parametrize(("n", "d", "v", "top"), [(1, 64, 97, 5), (3, 128, 1000, 20), (33, 64, 129, 1), (65, 192, 700, 128), (128, 256, 3001, 8),
                                                  (9, 1024, 300, 4), (20, 1536, 260, 6), (40, 640, 200, 3)])
def test_few_tokens(n, d, v, top, head):
    _check_score(n, d, v, top=top, head=head, seed=n)


@pytest.mark.parametrize("head", ["dense", "trainable", "q4"])
@pytest.mark.parametrize(("n", "d", "v", "top"), [(129, 64, 97, 97), (300, 128, 1000, 5), (257, 192, 3001, 64), (513, 64, 640, 0), (200, 256, 20011, 128)])
def test_many_tokens(n, d, v, top, head):
    _check_score(n, d, v, top=top, head=head, seed=n, temperature=0.7)


@pytest.mark.parametrize(("n", "d", "v", "top"), [(2, 72, 300, 4), (140, 72, 300, 4), (300, 200, 1500, 20), (129, 8, 64, 3), (5, 8, 64, 3)])
def test_hidden_dims_that_no_tile_divides(n, d, v, top):
    _check_score(n, d, v, top=top, head="trainable", seed=n, temperature=2.0)


@pytest.mark.parametrize("head", ["dense", "trainable", "q4"])
@pytest.mark.parametrize(("n", "d", "v", "top"), [(1, 64, 97, 5), (17, 192, 700, 20), (40, 64, 129, 1), (64, 128, 1000, 64), (65, 64, 300, 4),
                                                  (129, 64, 700, 20), (300, 192, 1501, 128)])
def test_fp32(n, d, v, top, head):
    _check_score(n, d, v, top=top, head=head, dtype="fp32", seed=n, temperature=0.8)


@pytest.mark.parametrize(("n", "d", "v"), [(7, 33, 301), (9, 36, 500), (131, 33, 301), (150, 70, 500)])
def test_fp32_odd_hidden_dims(n, d, v):
    _check_score(n, d, v, top=6, head="trainable", dtype="fp32", seed=n)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 90, 140])
def test_a_4bit_head_in_registers(n, dtype, monkeypatch):
    """MTP_LCE_STAGE_HEAD=0: no copy of the head's rows, forward or backward."""
    monkeypatch.setenv("MTP_LCE_STAGE_HEAD", "0")
    _check_score(n, 192, 700, top=5, head="q4", dtype=dtype, seed=n)
    _check_distill(n, 192, 700, 6, head="q4", dtype=dtype, seed=n)


@pytest.mark.parametrize("n", [4, 140])
def test_no_targets(n):
    _check_score(n, 64, 500, top=3, targets=False, seed=1)
    _check_score(n, 64, 500, top=0, targets=False, dtype="fp32", seed=2)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [2, 150])
@pytest.mark.parametrize("top", [1, 20, 128])
def test_equal_logits_go_by_index(n, top, dtype):
    """A hidden state of zeros, of either sign, makes every logit the same."""
    _, hd, _ = S.make(n, 64, 1000, dtype=dtype)
    h = torch.zeros(n, 64, dtype=hd.weight.dtype, device="cuda")
    h[::2, ::3] = -0.0
    r = token_logprobs(h, S.to(hd, "cuda"), top=top)
    assert torch.equal(r.top_ids.cpu(), torch.arange(top).expand(n, top))
    S.within(r.entropy, torch.full((n,), math.log(1000.0), dtype=torch.float64), S.stat(1000) + 256 * S.U, "entropy")


@pytest.mark.parametrize("n", [3, 140])
def test_alternatives_in_ascending_and_descending_logits(n):
    """Every logit larger (smaller) than the one before it, and all of a head's best in one group."""
    v, d = 2000, 64
    w = torch.zeros(v, d)
    w[:, 0] = torch.arange(v) // 16
    w[:, 1] = torch.arange(v) % 16
    h = torch.zeros(n, d)
    h[:, 0], h[:, 1] = 16.0, 1.0
    h[1::2] *= -1
    r = token_logprobs((h / 64).bfloat16().cuda(), DenseHead(weight=w.bfloat16().cuda(), trainable=False), top=64)
    up, down = torch.arange(v - 1, v - 65, -1), torch.arange(64)
    want = torch.stack([up if i % 2 == 0 else down for i in range(n)])
    assert torch.equal(r.top_ids.cpu(), want)


@pytest.mark.parametrize("n", [2, 130])
def test_a_vocabulary_of_many_groups(n):
    """More groups of 128 than a workgroup's small table holds."""
    v = 2048 * 128 + 77
    hidden, hd, w = S.make(n, 64, v, seed=3)
    r = token_logprobs(hidden.cuda(), S.to(hd, "cuda"), top=9)
    z = (hidden.double().cuda() @ w.T.cuda())
    value, ids = torch.sort(z, dim=1, descending=True, stable=True)
    assert torch.equal(r.top_ids, ids[:, :9])
    want = torch.log_softmax(z, 1).gather(1, ids[:, :9]).cpu()
    S.within(r.top_logprobs, want, S.stat(v) + 256 * S.U, "top_logprobs")


@pytest.mark.parametrize(("n", "d", "v", "top", "head", "dtype"), [
    (1400, 64, 50001, 20, "dense", "bf16"), (1400, 72, 50001, 3, "dense", "bf16"), (800, 64, 100003, 128, "q4", "bf16"),
    (17000, 64, 4100, 5, "dense", "bf16"), (1400, 64, 50001, 8, "dense", "fp32"), (1400, 33, 50001, 2, "dense", "fp32"),
    (800, 64, 100003, 16, "q4", "fp32"), (300, 64, 2048 * 128 + 77, 4, "dense", "bf16")])
def test_logits_that_are_not_kept(n, d, v, top, head, dtype):
    """More logits than a forward writes down: the alternatives' groups are formed again."""
    hidden, hd, w = S.make(n, d, v, head=head, dtype=dtype, seed=3)
    y = _targets(n, v, 3)
    h = hidden.clone()
    h[y == -100] = math.nan
    got = token_logprobs(h.cuda(), S.to(hd, "cuda"), y.cuda(), top=top, temperature=0.9)
    live = (y != -100).cuda()
    at = 0
    for rows in live.nonzero()[:, 0].split(400):
        z = hidden[rows.cpu()].double().cuda() @ w.T.cuda()
        value, ids = torch.sort(z, dim=1, descending=True, stable=True)
        assert torch.equal(got.top_ids[rows], ids[:, :top])
        logp = torch.log_softmax(z / 0.9, 1)
        off = S.stat(v) + 256 * S.U
        S.within(got.top_logprobs[rows], logp.gather(1, ids[:, :top]).cpu(), off, "top_logprobs")
        S.within(got.logprobs[rows], logp.gather(1, y.cuda()[rows][:, None])[:, 0].cpu(), off, "logprobs")
        S.within(got.entropy[rows], -(logp.exp() * logp).sum(1).cpu(), off + 128 * S.stat(v), "entropy")
        at += rows.numel()
    assert at == int(live.sum()) and bool((got.top_ids[~live] == -1).all()) and bool((got.top_logprobs[~live] == -math.inf).all())


def test_equal_logits_that_are_not_kept():
    _, hd, _ = S.make(1, 64, 50000)
    r = token_logprobs(torch.zeros(1400, 64, dtype=torch.bfloat16, device="cuda"), S.to(hd, "cuda"), top=70)
    assert torch.equal(r.top_ids.cpu(), torch.arange(70).expand(1400, 70))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 3, 140])
def test_the_smallest_head(n, dtype):
    """One word: certain, no entropy, nothing to learn."""
    hidden, hd, _ = S.make(n, 8, 1, head="trainable", dtype=dtype)
    hd = S.to(hd, "cuda")
    h = hidden.cuda().requires_grad_(True)
    r = token_logprobs(h, hd, torch.zeros(n, dtype=torch.int64, device="cuda"), top=1)
    assert bool((r.top_ids == 0).all()) and float(r.logprobs.detach().abs().max()) <= 64 * S.U and float(r.entropy.detach().abs().max()) <= 64 * S.U
    loss = distillation_loss(h, hd, torch.zeros(n, 1, dtype=torch.int64, device="cuda"), torch.zeros(n, 1, device="cuda"), renormalize=True)
    for g in torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + loss, (h, hd.weight)):
        assert float(g.abs().max()) <= 1e-4


@pytest.mark.parametrize("n", [2, 140])
def test_logits_that_are_no_numbers(n):
    """Rows of NaN and of infinities among others: theirs is what comes of them, the others' is as without."""
    hidden, hd, _ = S.make(n, 64, 1000, seed=5)
    hd = S.to(hd, "cuda")
    h = hidden.cuda()
    want = token_logprobs(h, hd, top=7)
    bad = h.clone()
    bad[0] = math.nan
    bad[-1, 0] = math.inf
    got = token_logprobs(bad, hd, top=7)
    assert bool(torch.isnan(got.entropy[0]))
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a[1:-1], b[1:-1])


@pytest.mark.parametrize(("n", "d", "dtype"), [(3, 72, "bf16"), (40, 72, "bf16"), (140, 72, "bf16"), (3, 36, "fp32"), (140, 36, "fp32")])
def test_a_token_that_is_ruled_out_by_its_weight(n, d, dtype):
    """-inf at a place where every hidden state is positive: a logit of -inf, and the row before it as without."""
    hidden, hd, w = S.make(n, d, 100, dtype=dtype, seed=5)
    hidden[:, 5] = 1.0
    w[8, 5] = -math.inf
    hd = DenseHead(weight=w.to(hidden.dtype).cuda(), trainable=False)
    y = torch.arange(n) % 8
    got = token_logprobs(hidden.cuda(), hd, y.cuda(), top=100)
    z = hidden.double() @ w.T
    logp = torch.log_softmax(z, 1)
    off = S.stat(100) + 256 * S.U
    S.within(got.logprobs, logp.gather(1, y[:, None])[:, 0], off, "logprobs")
    value, ids = torch.sort(logp, dim=1, descending=True, stable=True)
    assert torch.equal(got.top_ids.cpu(), ids)
    S.within(got.top_logprobs[:, :-1], value[:, :-1], off, "top_logprobs")
    assert bool((got.top_logprobs[:, -1] == -math.inf).all())


@pytest.mark.parametrize("n", [3, 140])
@pytest.mark.parametrize("temperature", [1e-3, 1e3])
def test_extreme_temperatures(n, temperature):
    """All on the likeliest, or near to evenly spread."""
    hidden, hd, w = S.make(n, 64, 500, seed=5)
    r = token_logprobs(hidden.cuda(), S.to(hd, "cuda"), top=1, temperature=temperature)
    z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool)).detach() / temperature
    p = torch.softmax(z, 1)
    want = -torch.special.xlogy(p, p).sum(1)
    size = 2 * float(z.abs().max()) + 1   # x is rounded at its own size, not below 64
    assert float((r.entropy.double().cpu() - want).abs().max()) <= (S.stat(500) + 256 * S.U) * size * 8


def test_in_inference_mode():
    hidden, hd, _ = S.make(9, 64, 300)
    h, hd = hidden.cuda(), S.to(hd, "cuda")
    want = token_logprobs(h, hd, top=3)
    ids, lp, _ = (x.cuda() for x in S.teacher_list(9, 300, 4, holes=False))
    loss = distillation_loss(h, hd, ids, lp)
    with torch.inference_mode():
        got = token_logprobs(h, hd, top=3)
        again = distillation_loss(h, hd, ids, lp)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:])) and torch.equal(again, loss)


def test_more_tokens_than_a_pass_takes():
    """Blocks of 16384 tokens: every one as if it were alone."""
    n, d, v = 16384 + 300, 64, 4100
    hidden, hd, _ = S.make(n, d, v, seed=4)
    hd = S.to(hd, "cuda")
    y = _targets(n, v, 4).cuda()
    h = hidden.cuda()
    r = token_logprobs(h, hd, y, top=3)
    for rows in (slice(0, 500), slice(16384 - 200, 16384 + 300)):
        part = token_logprobs(h[rows], hd, y[rows], top=3)
        assert torch.equal(part.top_ids, r.top_ids[rows])
        for a, b in zip(part[:3], (x[rows] for x in r[:3])):
            assert float((a - b).nan_to_num(0, 0, 0).abs().max()) <= 4 * S.stat(v)
    ids, lp = r.top_ids, r.top_logprobs
    losses = distillation_loss(h, hd, ids, lp - 0.1, reduction="none")
    part = distillation_loss(h[16384 - 200:], hd, ids[16384 - 200:], lp[16384 - 200:] - 0.1, reduction="none")
    assert float((losses[16384 - 200:] - part).abs().max()) <= 64 * S.stat(v)


def test_scoring_agrees_with_the_loss():
    hidden, hd, _ = S.make(300, 128, 900, seed=6)
    y = _targets(300, 900, 6).cuda()
    h, hd = hidden.cuda(), S.to(hd, "cuda")
    nll = linear_cross_entropy(h, hd, y, reduction="none")
    r = token_logprobs(h, hd, y, top=4)
    assert float((nll + r.logprobs).abs().max()) <= 2 * (S.stat(900) + 256 * S.U)
    # a target among the alternatives has one log probability
    at = r.top_ids == y[:, None]
    assert torch.equal(r.top_logprobs[at], r.logprobs[at.any(1)])


def test_unchecked_targets_out_of_range():
    hidden, hd, _ = S.make(140, 64, 200, seed=6)
    hd = S.to(hd, "cuda")
    for n in (5, 140):
        y = torch.zeros(n, dtype=torch.int64, device="cuda")
        y[1], y[2] = 2 ** 40, -7
        r = token_logprobs(hidden[:n].cuda().requires_grad_(True), hd, y, top=2, validate_targets=False)
        z = S.logits(hidden[:n], hd.weight.double().cpu(), torch.ones(n, dtype=torch.bool)).detach()
        S.within(r.logprobs[1:3], -torch.logsumexp(z, 1)[1:3], S.stat(200) + 256 * S.U, "no logit")
        r.logprobs.sum().backward()


# ---- distillation -------------------------------------------------------------------------------------------------

KINDS = [("forward", False), ("forward", True), ("reverse", False), ("jsd", False), ("jsd", True)]


@pytest.mark.parametrize(("kind", "renormalize"), KINDS)
@pytest.mark.parametrize(("n", "d", "v", "k", "reduction"), [(5, 64, 97, 4, "mean"), (40, 128, 1000, 64, "none"), (128, 64, 500, 128, "sum"),
                                                             (129, 64, 97, 3, "none"), (300, 192, 3001, 50, "mean"), (270, 64, 700, 1, "sum")])
def test_distillation(n, d, v, k, reduction, kind, renormalize):
    _check_distill(n, d, v, k, kind=kind, renormalize=renormalize, reduction=reduction, seed=n)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("head", ["trainable", "q4"])
@pytest.mark.parametrize(("n", "k"), [(7, 5), (200, 20)])
def test_distillation_heads(n, k, head, dtype):
    for kind in ("forward", "reverse", "jsd"):
        _check_distill(n, 128, 1100, k, head=head, dtype=dtype, kind=kind, temperature=1.7, seed=n)


@pytest.mark.parametrize(("n", "d", "dtype"), [(9, 72, "bf16"), (150, 200, "bf16"), (9, 33, "fp32"), (150, 70, "fp32")])
def test_distillation_odd_hidden_dims(n, d, dtype):
    _check_distill(n, d, 333, 11, head="trainable", dtype=dtype, seed=n)


@pytest.mark.parametrize("n", [6, 200])
def test_lists_longer_than_the_vocabulary(n):
    """Every outcome is listed, ids repeat, and nothing is left for the rest."""
    _check_distill(n, 64, 40, 128, renormalize=True, seed=n, holes=False)


@pytest.mark.parametrize("n", [6, 200])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_nothing_counts(n, reduction):
    hidden, hd, _ = S.make(n, 64, 200)
    h = torch.full_like(hidden, math.nan).cuda().requires_grad_(True)
    hd = S.to(DenseHead(weight=hd.weight, trainable=True), "cuda")
    ids = torch.full((n, 3), -1, device="cuda")
    loss = distillation_loss(h, hd, ids, torch.full((n, 3), math.nan, device="cuda"), reduction=reduction)
    assert bool((loss == 0).all())
    grads = torch.autograd.grad(loss.sum(), (h, hd.weight))
    assert all(bool((g == 0).all()) for g in grads)


@pytest.mark.parametrize("n", [6, 200])
def test_unchecked_ids_out_of_range_are_empty(n):
    hidden, hd, _ = S.make(n, 64, 200)
    h, hd = hidden.cuda(), S.to(hd, "cuda")
    ids, lp, _ = S.teacher_list(n, 200, 4, holes=False)
    far = ids.clone()
    far[:, 1] = 2 ** 33 + 5
    far[:, 2] = 200
    gone = ids.clone()
    gone[:, 1:3] = -1
    a, b = (distillation_loss(h, hd, x.cuda(), lp.cuda(), reduction="none", validate_ids=False) for x in (far, gone))
    assert torch.equal(a, b)
    with pytest.raises(LossInputError):
        distillation_loss(h, hd, far.cuda(), lp.cuda())


# ---- as they are used ---------------------------------------------------------------------------------------------

# A backward without its forward's logits forms them again; sizes as small as these keep them by themselves.
_FORMED_AGAIN = [(5, 64, 97, 4, "dense", "bf16"), (300, 128, 1000, 20, "trainable", "bf16"), (300, 200, 1500, 64, "dense", "bf16"),
                 (257, 192, 3001, 20, "q4", "bf16"), (150, 128, 1000, 20, "trainable", "fp32"), (150, 64, 700, 8, "q4", "fp32"),
                 (70, 33, 301, 5, "dense", "fp32")]


@pytest.mark.parametrize(("n", "d", "v", "k", "head", "dtype"), _FORMED_AGAIN)
def test_gradients_of_logits_formed_again(n, d, v, k, head, dtype, monkeypatch):
    monkeypatch.setattr(scoring, "_kept_bytes", lambda x: 0)
    _check_score(n, d, v, top=k, head=head, dtype=dtype, halves=False)
    _check_distill(n, d, v, k, head=head, dtype=dtype, halves=False)


@pytest.mark.parametrize(("n", "d", "head"), [(5, 512, "dense"), (5, 512, "trainable"), (32, 512, "q4"), (129, 1536, "trainable")])
def test_gradients_of_kept_logits_by_vocabulary_chunks(n, d, head, monkeypatch):
    """A budget of six times the kept logits, which the staged head's chunks and the gradient tiles overrun: several chunks."""
    v = 6000
    budget = 6 * n * 6016 * 4
    assert 2 * (n + d) * v > budget
    monkeypatch.setenv("MTP_LCE_BWD_BUDGET", str(budget))
    monkeypatch.setenv("MTP_LCE_TRANSPOSED_HEAD", "0")
    _check_score(n, d, v, top=4, head=head)
    _check_distill(n, d, v, 20, head=head)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_kept_logits_of_more_rows_than_a_grid_has(dtype):
    """A small vocabulary: 40000 tokens' logits are kept whole, and the gradient tiles take their rows in blocks."""
    n, d, v = 40000, 64, 500
    hidden, hd, w = S.make(n, d, v, head="trainable", dtype=dtype, seed=6)
    hd = S.to(hd, "cuda")
    h = hidden.cuda().requires_grad_()
    y = torch.arange(n) % v
    got = token_logprobs(h, hd, y.cuda())
    z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool))
    logp = torch.log_softmax(z, 1)
    logprobs, entropy = logp.gather(1, y[:, None])[:, 0], -(logp.exp() * logp).sum(1)
    off = S.stat(v) + 256 * S.U
    S.within(got.logprobs, logprobs, off, "logprobs")
    S.within(got.entropy, entropy, off + 128 * S.stat(v), "entropy")
    a, b = torch.randn(2, n, generator=torch.Generator().manual_seed(7))
    (gz,) = torch.autograd.grad((logprobs * a.double() + entropy * b.double()).sum(), z)
    grad = torch.autograd.grad((got.logprobs, got.entropy), (h, hd.weight), (a.cuda(), b.cuda()))
    extra = (a.abs() + 64 * b.abs()).double()
    dh, dh_off, dw, dw_off = S.gradient_bounds(gz, torch.softmax(z.detach(), 1), extra, hidden.double(), w, True, dtype, False)
    S.within(grad[0], dh, dh_off, "d_hidden")
    S.within(grad[1], dw, dw_off, "d_weight")


def test_which_logits_a_forward_keeps(monkeypatch):
    hidden, hd, _ = S.make(40, 64, 300, head="dense", dtype="bf16")
    hidden, hd = hidden.cuda().requires_grad_(), S.to(hd, "cuda")
    kept = 40 * 384 * 4
    y = torch.zeros(40, dtype=torch.long, device="cuda")
    token_logprobs(hidden, hd, y)  # the library's own first uses

    def held(grad, budget):
        monkeypatch.setenv("MTP_LCE_BWD_BUDGET", str(budget))
        before = torch.cuda.memory_allocated()
        with torch.set_grad_enabled(grad):
            out = token_logprobs(hidden, hd, y)
        now = torch.cuda.memory_allocated() - before
        del out
        return now

    assert held(True, 6 * kept) >= kept > held(True, 6 * kept - 6)
    assert held(False, 6 * kept) < kept


@pytest.mark.parametrize("n", [20, 300])
def test_a_teacher_scores_a_student_learns(n):
    """The teacher's alternatives as the student's lists: no loss against itself, a gradient against another."""
    hidden, hd, w = S.make(n, 128, 1000, seed=1)
    h, hd = hidden.cuda(), S.to(hd, "cuda")
    with torch.no_grad():
        t = token_logprobs(h, hd, top=32)
        for kind in ("forward", "reverse", "jsd"):
            rows = distillation_loss(h, hd, t.top_ids, t.top_logprobs, kind=kind, reduction="none")
            assert float(rows.abs().max()) <= 80 * (S.stat(1000) + 256 * S.U)
    student = (hidden + 1 / 32).cuda().requires_grad_(True)
    loss = distillation_loss(student, hd, t.top_ids, t.top_logprobs)
    (g,) = torch.autograd.grad(loss, student)
    assert float(loss) > 0 and bool(torch.isfinite(g).all()) and float(g.norm()) > 0


def test_a_policy_step_with_an_entropy_bonus():
    """token_logprobs into policy_loss, its gradient and the entropy's in one backward, against the loss's own path."""
    n, v = 256, 700
    hidden, hd, w = S.make(n, 128, v, seed=2)
    hd = S.to(hd, "cuda")
    y = _targets(n, v, 2, ignored=False).cuda()
    adv = torch.randn(4, generator=torch.Generator().manual_seed(3)).cuda()
    h = hidden.cuda().requires_grad_(True)
    old = linear_cross_entropy(h.detach(), hd, y, reduction="none").view(4, -1) + 0.05
    r = token_logprobs(h.view(4, -1, 128), hd, y.view(4, -1))
    loss = policy_loss(-r.logprobs, old, adv).loss - 0.01 * r.entropy.mean()
    (got,) = torch.autograd.grad(loss, h)
    z = S.logits(hidden, w, torch.ones(n, dtype=torch.bool))
    lp, ent, _, _ = S.score(z, y.cpu(), torch.ones(n, dtype=torch.bool), 1.0, 0)
    want = policy_loss(-lp.view(4, -1), old.double().cpu(), adv.double().cpu(), impl="reference").loss - 0.01 * ent.mean()
    (gz,) = torch.autograd.grad(want, z)
    p = torch.softmax(z.detach(), 1)
    dh, off, _, _ = S.gradient_bounds(gz, p, torch.full((n,), 64.0 / n, dtype=torch.float64), hidden.double(), w, False, "bf16", n <= 128)
    S.within(got, dh, off, "d_hidden")


@pytest.mark.parametrize("n", [5, 200])
def test_views_and_types_of_a_call(n):
    """A hidden state that is a transposed view, one off a 16-byte boundary, int32 targets and ids, bf16 teachers, a uint8 mask."""
    hidden, hd, _ = S.make(n, 64, 300, seed=8)
    hd = S.to(hd, "cuda")
    h = hidden.cuda()
    y = _targets(n, 300, 8).cuda()
    want = token_logprobs(h, hd, y, top=3)
    odd = torch.empty(n * 64 + 1, dtype=h.dtype, device="cuda")[1:].view(n, 64).copy_(h)
    for view in (h.t().contiguous().t(), odd):
        got = token_logprobs(view, hd, y.int(), top=3)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ids, lp, mask = S.teacher_list(n, 300, 5, seed=8)
    a = distillation_loss(h, hd, ids.cuda(), lp.bfloat16().cuda(), mask=mask.cuda(), reduction="none")
    b = distillation_loss(odd, hd, ids.int().cuda(), lp.bfloat16().float().cuda(), mask=mask.to(torch.uint8).cuda(), reduction="none")
    assert torch.equal(a, b)


def _steps(n):
    hidden, hd, _ = S.make(n, 128, 1000, head="trainable", seed=9)
    hd = S.to(hd, "cuda")
    h = hidden.cuda().requires_grad_(True)
    y = _targets(n, 1000, 9).cuda()
    ids, lp, mask = (x.cuda() for x in S.teacher_list(n, 1000, 8, seed=9))

    def step():
        r = token_logprobs(h, hd, y, top=5, validate_targets=False)
        loss = distillation_loss(h, hd, ids, lp, mask=mask, kind="jsd", validate_ids=False)
        g = torch.autograd.grad((r.logprobs.mean() + 0.1 * r.entropy.mean(), loss), (h, hd.weight))
        return [r.logprobs.detach(), r.entropy.detach(), r.top_logprobs, r.top_ids, loss.detach(), *g]

    return step, h, ids


@pytest.mark.parametrize("n", [6, 300])
def test_runs_repeat_bit_for_bit(n):
    step, _, _ = _steps(n)
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))


@pytest.mark.parametrize("n", [6, 300])
def test_the_python_functions_give_the_same_bits(n, monkeypatch):
    """Both autograd paths, with targets and without, each loss, each head."""
    from mlx_train_perf import _native

    def run():
        out = []
        for head, dtype in (("dense", "bf16"), ("trainable", "bf16"), ("q4", "bf16"), ("trainable", "fp32")):
            hidden, hd, _ = S.make(n, 64, 500, head=head, dtype=dtype, seed=11)
            hd = S.to(hd, "cuda")
            h = hidden.cuda().requires_grad_(True)
            leaves = [h] + ([hd.weight] if head == "trainable" else [])
            ids, lp, mask = (x.cuda() for x in S.teacher_list(n, 500, 6, seed=11))
            for y in (None, _targets(n, 500, 11).cuda()):
                r = token_logprobs(h, hd, y, top=3, temperature=1.2)
                out += [x.detach() for x in r if x is not None]
                out += torch.autograd.grad(r.entropy.sum() + (0 if y is None else (r.logprobs * 0.3).sum()), leaves)
            for kind in ("forward", "reverse", "jsd"):
                loss = distillation_loss(h, hd, ids, lp, mask=mask, kind=kind)
                out += [loss.detach(), *torch.autograd.grad(loss * 3, leaves)]
        return out

    assert _native.nodes() is not None
    nodes = run()
    monkeypatch.setattr(_native, "_nodes", False)
    assert _native.nodes() is None
    assert all(torch.equal(a, b) for a, b in zip(run(), nodes, strict=True))


def test_no_second_derivative(monkeypatch):
    """Asked for, it raises in both autograd paths and is not taken for 0."""
    from mlx_train_perf import _native

    hidden, hd, _ = S.make(5, 64, 100)
    hd = S.to(hd, "cuda")
    ids, lp, _ = (x.cuda() for x in S.teacher_list(5, 100, 4, holes=False))
    for nodes in (_native.nodes(), False):
        monkeypatch.setattr(_native, "_nodes", nodes)
        h = hidden.cuda().requires_grad_(True)
        for f in (lambda: token_logprobs(h, hd).entropy.sum(), lambda: distillation_loss(h, hd, ids, lp)):
            ct = torch.ones((), device="cuda", requires_grad=True)
            (g,) = torch.autograd.grad(f(), h, ct, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                g.float().sum().backward()


@pytest.mark.parametrize("n", [6, 300])
def test_on_another_stream(n):
    step, _, _ = _steps(n)
    first = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, first))


@pytest.mark.parametrize("n", [6, 300])
def test_captured_into_graphs(n):
    """Two graphs, replayed in turn with eager work between and new inputs, against eager runs."""
    step, h, ids = _steps(n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(3):
        with torch.no_grad():
            h.copy_(torch.roll(h, i, 0))
            ids.copy_(torch.roll(ids, 1, 1))
        want = [x.clone() for x in step()]
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i
