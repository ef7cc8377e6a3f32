"""GPU: the preference and policy losses against their definition in 64 bits.

Tolerances: sums are in 64 bits and each fp32 result is rounded once (2^-24 = 6e-8); a preference gradient is a product
of two rounded factors; a policy token takes expf and expm1f (some 2 ulp each) and three products: 2e-6 covers ten
roundings and the kl's series (2^-26). The policy loss is a mean of terms of either sign: its error is held against the
mean of their sizes."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _preference as P

pytestmark = pytest.mark.gpu


def _near(name, a, w, tol=2e-6, floor=0.0):
    a, w = a.detach().double().cpu(), w.double()
    assert a.shape == w.shape, name
    assert float((a - w).norm()) <= tol * max(float(w.norm()), floor), (name, a, w)


def _cuda(t):
    return None if t is None else t.cuda()


def _pref(nll, ref, offsets, mask, ct=None, **kw):
    from mlx_train_perf import preference_loss

    x = nll.cuda().requires_grad_(True)
    r = preference_loss(x, ref.cuda(), offsets=_cuda(offsets), mask=_cuda(mask), **kw)
    (d,) = torch.autograd.grad(r.loss, x, _cuda(ct))
    return [*r, d]


def _policy(nll, old, adv, ref, offsets, mask, ct=None, **kw):
    from mlx_train_perf import policy_loss

    x = nll.cuda().requires_grad_(True)
    r = policy_loss(x, old.cuda(), adv.cuda(), ref_nll=_cuda(ref), offsets=_cuda(offsets), mask=_cuda(mask), **kw)
    (d,) = torch.autograd.grad(r.loss, x, _cuda(ct))
    return [*r, d]


SIZES = [(2, 1), (2, 7), (6, 5), (10, 64), (4, 300), (34, 33), (2, 5000)]


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize(("seqs", "t"), SIZES)
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_preference(layout, seqs, t, kind):
    shape, offsets, mask = P.layout(layout, seqs, t, t)
    nll, _, ref = P.tensors(shape, seqs)
    if mask is not None:
        nll[~mask], ref[~mask] = math.nan, math.inf
    g = torch.Generator().manual_seed(1)
    for reduction, smooth in (("mean", 0.0), ("none", 0.2), ("sum", 0.1)):
        args = {"beta": 0.2, "kind": kind, "reduction": reduction, "label_smoothing": smooth if kind == "sigmoid" else 0.0}
        ct = torch.randn(seqs // 2, generator=g) if reduction == "none" else None
        got = _pref(nll, ref, offsets, mask, ct, **args)
        want = P.preference(nll, ref, offsets=offsets, mask=mask, ct=ct, **args)
        for name, a, w in zip(("loss", "chosen", "rejected", "d_nll"), got, want):
            _near(name, a, w)


@pytest.mark.parametrize("reduction", ["token", "sequence", "none"])
@pytest.mark.parametrize(("seqs", "t"), SIZES)
@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_policy(layout, seqs, t, reduction):
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
        r = ref if with_ref else None
        got = _policy(nll, old, adv, r, offsets, mask, ct, **args)
        want = P.policy(nll, old, adv, ref_nll=r, offsets=offsets, mask=mask, ct=ct, **args)
        size = 1.0   # a token's loss is about |A|, 0.8 on average
        for name, a, w in zip(("loss", "kl", "clip", "d_nll"), got, want):
            _near(name, a, w, floor=size if name == "loss" and reduction != "none" else 0.0)


def test_borders_and_extremes():
    """Ratios at, just inside and just outside a border; advantages of 0; borders of 0 and 1; ratios that overflow."""
    lo, hi = 0.2, 0.28
    steps = torch.tensor([math.log1p(hi), math.log1p(-lo)], dtype=torch.float64).float()
    near = torch.cat([steps, torch.nextafter(steps, torch.tensor(9.0)), torch.nextafter(steps, torch.tensor(-9.0)), torch.zeros(2)])
    old = near.repeat(4)[None]
    nll = torch.zeros_like(old)
    adv = torch.tensor([1.0, -1.0, 0.0, 2.0]).repeat_interleave(8)[None]
    for clip in ((lo, hi), (0.0, 0.0), (1.0, 5.0)):
        got = _policy(nll, old, adv, None, None, None, torch.ones_like(nll), clip_low=clip[0], clip_high=clip[1], reduction="none")
        u = torch.exp(old.double())
        c = u.clamp(1 - clip[0], 1 + clip[1])
        a = adv.double()
        # a float step is never exactly at a border's logarithm, except 0 at the border 1
        out = torch.where(a > 0, u > 1 + clip[1], (u < 1 - clip[0]) & (a < 0))
        _near("loss", got[0], -torch.minimum(u * a, c * a))
        _near("d_nll", got[3], torch.where(out, 0.0, u * a))
        assert float(got[2]) == pytest.approx(float(out.double().mean()))
    got = _policy(torch.zeros(1, 2), torch.full((1, 2), 200.0), torch.tensor([[1.0, -1.0]]), None, None, None, torch.ones(1, 2), reduction="none")
    assert float(got[0][0, 0]) == pytest.approx(-1.2) and float(got[0][0, 1]) == math.inf and float(got[3][0, 0]) == 0.0
    # small and large distances to the reference model: e^d - d - 1 without cancellation
    d = torch.tensor([[0.0, 1e-6, -1e-4, 3e-3, -0.05, 0.3, 0.4999, 0.5, -0.5001, 1.5, -4.0, 10.0]])
    got = _policy(d, d, torch.zeros(1), torch.zeros_like(d), None, None, torch.ones_like(d), kl_coef=1.0, reduction="none")
    dd = d.double()
    kl = torch.expm1(dd) - dd
    assert torch.allclose(got[0].double().cpu(), kl, rtol=2e-6, atol=1e-16)


def test_long_sums_of_small_differences():
    """A log ratio of 1 between sums of 10^5: fp32 sums would lose its digits."""
    n = 100_003
    ref = torch.rand(4, n, generator=torch.Generator().manual_seed(0)) + 1
    nll = ref.clone()
    nll[0, ::1000] -= 0.01
    nll[3, ::500] += 0.005
    got = _pref(nll, ref, None, None, beta=1.0)
    gap = (ref.double() - nll.double()).sum(1)
    d = gap[:2] - gap[2:]
    _near("chosen", got[1], gap[:2])
    _near("loss", got[0], torch.nn.functional.softplus(-d).mean())


def test_types_strides_streams_and_devices():
    from mlx_train_perf import policy_loss, preference_loss

    nll, old, ref = (x.cuda() for x in P.tensors((6, 50), 1))
    m = torch.rand(6, 50, device="cuda") < 0.7
    a = preference_loss(nll, ref, mask=m).loss
    assert torch.equal(a, preference_loss(nll.t().contiguous().t(), ref.t().contiguous().t(), mask=m.to(torch.uint8).t().contiguous().t()).loss)
    o = torch.tensor([0, 50, 100, 150, 200, 250, 300], device="cuda")
    flat = preference_loss(nll.reshape(-1), ref.reshape(-1), mask=m.reshape(-1), offsets=o.to(torch.int32)).loss
    assert torch.equal(a, flat)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    adv = torch.randn(6, device="cuda")
    with torch.cuda.stream(side):
        x = (nll + 0).requires_grad_(True)
        r = policy_loss(x, old, adv, ref_nll=ref, kl_coef=0.1, mask=m)
        r.loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    y = nll.clone().requires_grad_(True)
    q = policy_loss(y, old, adv, ref_nll=ref, kl_coef=0.1, mask=m)
    (q.loss * 1).backward()
    assert torch.equal(r.loss, q.loss) and torch.equal(x.grad, y.grad)
    with torch.no_grad():
        assert torch.equal(policy_loss(nll, old, adv, ref_nll=ref, kl_coef=0.1, mask=m).loss, q.loss)
    with pytest.raises(Exception, match="same GPU"):
        policy_loss(nll, old.cpu(), adv)


def test_offsets_out_of_range_stay_in_bounds():
    """Offsets that break the contract, unchecked: clamped into the tokens; no fault, tokens outside get 0."""
    from mlx_train_perf import preference_loss

    nll, _, ref = (x.cuda() for x in P.tensors((40,), 1))
    x = nll.requires_grad_(True)
    r = preference_loss(x, ref, offsets=torch.tensor([5, 20, 1000], device="cuda"), validate_offsets=False)
    (d,) = torch.autograd.grad(r.loss, x)
    assert torch.isfinite(r.loss) and not d[:5].any() and d[5:].all()


def test_large_batch_of_short_sequences():
    from mlx_train_perf import policy_loss

    nll, old, ref = (x.cuda() for x in P.tensors((3000, 3), 1))
    adv = torch.randn(3000, device="cuda")
    k = policy_loss(nll, old, adv, ref_nll=ref, kl_coef=0.2, reduction="sequence")
    w = policy_loss(nll.double(), old.double(), adv.double(), ref_nll=ref.double(), kl_coef=0.2, reduction="sequence", impl="reference")
    assert abs(float(k.loss) - float(w.loss)) <= 2e-6 and float(k.clip_fraction) == pytest.approx(float(w.clip_fraction), abs=1e-7)


@pytest.mark.parametrize("packed", [False, True])
def test_captured_steps(packed):
    """Both losses in one graph each, replayed in turn with new tensors, between eager steps."""
    from mlx_train_perf import policy_loss, preference_loss

    seqs, t = 8, 700
    def make(seed):
        shape, offsets, mask = P.layout("packed" if packed else "masked", seqs, t, seed)
        x = [v.cuda() for v in P.tensors(shape, seed)]
        return x, _cuda(offsets), _cuda(mask), torch.randn(seqs, generator=torch.Generator().manual_seed(seed)).cuda()

    def pref(s):
        x = s[0][0].detach().requires_grad_(True)
        r = preference_loss(x, s[0][2], offsets=s[1], mask=s[2], validate_offsets=False)
        return [*(v.detach() for v in r), *torch.autograd.grad(r.loss, x)]

    def pol(s):
        x = s[0][0].detach().requires_grad_(True)
        r = policy_loss(x, s[0][1], s[3], ref_nll=s[0][2], kl_coef=0.1, offsets=s[1], mask=s[2], reduction="sequence", validate_offsets=False)
        return [*(v.detach() for v in r), *torch.autograd.grad(r.loss, x)]

    graphs = []
    for n, fn in enumerate((pref, pol)):
        s = make(n)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                fn(s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn(s)
        graphs.append((fn, s, g, out))
    for turn in range(3):
        for n, (fn, s, g, out) in enumerate(graphs):
            new = make(10 + 2 * turn + n)
            for a, b in zip([*s[0], *s[1:]], [*new[0], *new[1:]]):
                if a is not None:
                    a.copy_(b)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, fn(new))), (turn, n)


@pytest.mark.parametrize("node", [True, False])
def test_infinite_ratios(node, monkeypatch):
    from mlx_train_perf import _native

    if not node:
        monkeypatch.setattr(_native, "nodes", lambda: None)
    P.check_infinite(lambda t: t.cuda())


def _both(x, ref, adv, offsets, mask, kw):
    from mlx_train_perf import policy_loss, preference_loss

    r = preference_loss(x, ref, offsets=offsets, mask=mask)
    p = policy_loss(x, ref, adv, ref_nll=ref, kl_coef=0.1, offsets=offsets, mask=mask, **kw)
    return r, p


@pytest.mark.parametrize("layout", P.LAYOUTS)
def test_node_and_function_agree(layout, monkeypatch):
    """The C++ nodes and the Python Functions are the same calls, to the bit."""
    from mlx_train_perf import _native

    shape, offsets, mask = P.layout(layout, 6, 300, 2)
    nll, ref, _ = (t.cuda() for t in P.tensors(shape, 2))
    adv = torch.randn(6, generator=torch.Generator().manual_seed(2)).cuda()

    def step():
        out = []
        for kw in ({}, {"reduction": "sequence"}, {"reduction": "none"}):
            x = nll.detach().requires_grad_(True)
            r, p = _both(x, ref, adv, _cuda(offsets), _cuda(mask), kw)
            out += [*(v.detach() for v in (*r, *p)), torch.autograd.grad(r.loss + p.loss.sum(), x)[0]]
        return out

    assert _native.nodes() is not None
    with_node = step()
    monkeypatch.setattr(_native, "nodes", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(with_node, step()))


@pytest.mark.parametrize("node", [True, False])
def test_second_derivative_is_refused(node, monkeypatch):
    from mlx_train_perf import _native

    if not node:
        monkeypatch.setattr(_native, "nodes", lambda: None)
    x = torch.rand(4, 5, device="cuda", requires_grad=True)
    for loss in _both(x, torch.rand(4, 5, device="cuda"), torch.randn(4, device="cuda"), None, None, {}):
        (d,) = torch.autograd.grad(loss.loss.square(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (d.square().sum() + x.sum()).backward()
