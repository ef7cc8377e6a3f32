"""GPU: attention with softcap, slopes and spans against the plain form in 64 bits, forward and backward.

Tolerances. bf16: P and dS are rounded to bf16 before their products, O is read back rounded for D, and each output is
rounded once: at most four roundings of at most 2^-8 of the value, of random sign, so of rms 2^-8 / sqrt(3) each and
2^-8 * 2 / sqrt(3) = 4.5e-3 together; 1e-2 is the bar of the other attention tests. dq and dk have on top what O's
rounding does through D, which no relative bound of theirs covers (_scored.attention). fp32: products and sums of up to
400 terms in some order, sqrt(400) * 2^-24 = 1.2e-6 of the largest, and the same again for the exponent of scores of up
to about 2^5 (2^5 * 2^-24 = 2e-6): 2e-5 is five times their sum."""
from __future__ import annotations

import pytest
import torch

from tests import _scored as S

pytestmark = pytest.mark.gpu

BAR = {torch.bfloat16: 1e-2, torch.float32: 2e-5}
U = {torch.bfloat16: 2 ** -8, torch.float32: 2e-6}   # of D's O: half a step of bf16; the sums' error above in fp32


def _call(q, k, v, d_o, *, mask, spans, **kw):
    from mlx_train_perf.attention import SpanMask, flash_attention

    qs = [x.detach().cuda().requires_grad_(True) for x in (q, k, v)]
    sm = None if spans is None else SpanMask(start=spans[0].cuda(), end=spans[1].cuda())
    o = flash_attention(*qs, causal=mask == "causal", spans=sm, **kw)
    return [o.detach(), *torch.autograd.grad(o, qs, d_o.cuda())]


def _check(b, hq, hkv, s, dh, *, mask, cap, biased, dtype, seed=0, std=2.0, spans=None, slopes=None, more_bar=0.0):
    print(f"[scored] b={b} hq={hq} hkv={hkv} s={s} dh={dh} {mask} cap={cap} biased={biased} {dtype}", flush=True)
    q, k, v, d_o = S.inputs(b, hq, hkv, s, dh, dtype, seed, std)
    spans = S.spans_of(mask, b, s, seed) if spans is None else spans
    slopes = None if not biased else S.slopes_of(hq).cuda() if slopes is None else slopes.cuda()
    scale = dh ** -0.5
    got = _call(q, k, v, d_o, mask=mask, spans=spans, scale=scale, softcap=cap, slopes=slopes)
    see = S.visible(mask, spans, b, s, "cuda")
    *want, tq, tk = S.attention(*(x.cuda() for x in (q, k, v, d_o)), scale=scale, see=see, softcap=cap, slopes=slopes, d_terms=True)
    more = dict(zip(("dq", "dk"), (U[dtype] * float(t.norm()) for t in (tq, tk))))
    empty = ~see.any(-1)
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(a).all(), name
        if name in ("o", "dq"):
            assert not a.transpose(1, 2)[empty].any(), f"{name}: a query that sees nothing"
        if name in ("dk", "dv"):
            assert not a.transpose(1, 2)[~see.any(1)].any(), f"{name}: a key that nothing sees"
        assert S.off(a, w) <= (BAR[dtype] + more_bar) * float(w.norm()) + more.get(name, 0.0), (name, S.rel(a, w), more)
    return got


FORMS = [(20.0, False), (None, True), (8.0, True), (None, False), (100.0, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("cap", "biased"), FORMS)
@pytest.mark.parametrize("mask", S.MASKS)
@pytest.mark.parametrize("dh", [64, 96, 128])
def test_against_64_bits(dh, mask, cap, biased, dtype):
    if cap is None and not biased and mask in ("causal", "full"):
        pytest.skip("neither cap, slopes nor spans")
    _check(2, 4, 2, 197, dh, mask=mask, cap=cap, biased=biased, dtype=dtype, seed=dh)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("s", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 400])
@pytest.mark.parametrize(("mask", "cap", "biased"), [("prefix", 30.0, False), ("ragged", 5.0, True), ("window", None, False)])
def test_lengths(s, mask, cap, biased, dtype):
    _check(2, 4, 2, s, 128 if s % 2 else 64, mask=mask, cap=cap, biased=biased, dtype=dtype, seed=s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("b", "hq", "hkv"), [(1, 1, 1), (3, 2, 2), (1, 6, 2), (2, 8, 1), (1, 5, 1), (1, 7, 7), (2, 12, 2)])
def test_head_groups(b, hq, hkv, dtype):
    _check(b, hq, hkv, 150, 64, mask="ragged", cap=10.0, biased=True, dtype=dtype, seed=hq)
    _check(b, hq, hkv, 150, 128, mask="causal", cap=None, biased=True, dtype=dtype, seed=hq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap", [0.5, 3.0, 50.0, 55.0, 56.0, 1000.0])
@pytest.mark.parametrize("std", [0.05, 30.0])
def test_caps_of_every_size(cap, std, dtype):
    """Scores far below and far above the cap. Where nearly all are above it, probabilities are nearly flat and every
    gradient through 1 - tanh^2 nearly 0: its relative error is then that of tanh near 1 (checked for o and dv)."""
    b, hq, hkv, s, dh = 1, 2, 1, 130, 64
    q, k, v, d_o = S.inputs(b, hq, hkv, s, dh, dtype, 11, std)
    got = _call(q, k, v, d_o, mask="causal", spans=None, scale=dh ** -0.5, softcap=cap)
    see = S.visible("causal", None, b, s)
    want = S.attention(q, k, v, d_o, scale=dh ** -0.5, see=see, softcap=cap)
    soft = std < 1 or cap >= 50
    # fp32: the scores reach 30 sqrt(64) / 8 * 4 = 120, of which 2^-24 is 7e-6 of a probability, beside the bar's own terms.
    bar = BAR[dtype] if dtype == torch.bfloat16 else 4e-5
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(a).all(), name
        if soft or name in ("o", "dv"):
            assert S.rel(a, w) <= bar, (name, S.rel(a, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores_and_far_keys(dtype):
    """Scores of every size under a cap near the bound of the fixed maximum, all of them at its lower end in some rows;
    and rows whose nearest visible key is hundreds of positions away under a steep bias."""
    b, hq, hkv, s, dh = 1, 2, 2, 300, 64
    q, k, v, d_o = S.inputs(b, hq, hkv, s, dh, torch.float32, 2, 1.0)
    k = k.abs()
    q[:, :, ::2] = -q[:, :, ::2].abs() * 100   # every score of these rows at -cap
    q, k, v, d_o = (x.to(dtype) for x in (q, k, v, d_o))
    got = _call(q, k, v, d_o, mask="causal", spans=None, scale=1.0, softcap=50.0)
    want = S.attention(q, k, v, d_o, scale=1.0, see=S.visible("causal", None, b, s), softcap=50.0)
    assert S.rel(got[0], want[0]) <= BAR[dtype] and S.rel(got[3], want[3]) <= BAR[dtype]
    start = torch.zeros(b, s, dtype=torch.int32)
    end = torch.full((b, s), 5, dtype=torch.int32)
    q, k, v, d_o = S.inputs(b, hq, hkv, s, dh, dtype, 3, 1.0)
    slopes = torch.tensor([4.0, 0.01])   # 1200 off at the last row: e^-1200 against a maximum of nothing nearer
    got = _call(q, k, v, d_o, mask="x", spans=(start, end), scale=dh ** -0.5, slopes=slopes.cuda())
    want = S.attention(q, k, v, d_o, scale=dh ** -0.5, see=S.visible("x", (start, end), b, s), slopes=slopes)
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        # the bias itself, up to 1200, is 2^-24 * 1200 = 7e-5 off in fp32
        assert S.rel(a, w) <= max(BAR[dtype], 2e-4), (name, S.rel(a, w))


def test_spans_equal_the_masks_they_describe():
    """A causal triangle, everything, and packed documents given as spans are the plain kernels' masks. Their O and the
    span kernels' (which divide by the sum of the rounded probabilities) have two roundings each, of rms
    2^-8 / sqrt(3) at most: 4.5e-3 together."""
    from mlx_train_perf.attention import PackedMask, SpanMask, document_spans, flash_attention
    from oracle import attention as oatt

    s = 333
    q, k, v, _ = (x.cuda() for x in S.inputs(1, 4, 2, s, 128, torch.bfloat16, 1))
    i = torch.arange(s, device="cuda", dtype=torch.int32)[None]
    zero = torch.zeros_like(i)
    for causal, spans in ((True, SpanMask(start=zero, end=i + 1)), (False, SpanMask(start=zero, end=zero + s))):
        a = flash_attention(q, k, v, scale=0.1, causal=causal)
        assert S.rel(flash_attention(q, k, v, scale=0.1, spans=spans), a.double()) <= 4.5e-3
    sid, sst = (t[None].cuda() for t in oatt.segments_from_lengths([100, 1, 77, 155]))
    seg = PackedMask(seg_id=sid, seg_start=sst)
    a = flash_attention(q, k, v, scale=0.1, segments=seg)
    assert S.rel(flash_attention(q, k, v, scale=0.1, spans=document_spans(seg)), a.double()) <= 4.5e-3
    capped = flash_attention(q, k, v, scale=0.1, segments=seg, softcap=7.0)
    assert torch.equal(capped, flash_attention(q, k, v, scale=0.1, spans=document_spans(seg), softcap=7.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_hidden_keys_may_hold_anything(dtype):
    """Padding's keys of NaN and infinity, which no query sees: the values of the others do not change. (V is kept
    finite, as a probability of 0 times NaN is NaN in any product.)"""
    b, hq, hkv, s, dh = 1, 4, 2, 150, 64
    q, k, v, d_o = S.inputs(b, hq, hkv, s, dh, dtype, 4)
    i = torch.arange(s)[None]
    spans = (torch.zeros(1, s, dtype=torch.int32), torch.where(i < 100, i + 1, 0).cummax(1).values.clamp(max=100).to(torch.int32))
    clean = _call(q, k, v, d_o, mask="x", spans=spans, scale=0.2, softcap=9.0, slopes=S.slopes_of(hq).cuda())
    k[:, :, 100:125], k[:, :, 125:] = float("nan"), float("inf")
    dirty = _call(q, k, v, d_o, mask="x", spans=spans, scale=0.2, softcap=9.0, slopes=S.slopes_of(hq).cuda())
    for name, a, c in zip(("o", "dv"), (dirty[0], dirty[3]), (clean[0], clean[3])):
        assert torch.equal(a, c), name


def test_strides_types_and_streams():
    """Views of other layouts, slopes and spans of other types and strides, and tensors made on another stream."""
    from mlx_train_perf.attention import SpanMask, flash_attention

    b, hq, hkv, s, dh = 2, 4, 2, 140, 64
    q, k, v, d_o = (x.cuda() for x in S.inputs(b, hq, hkv, s, dh, torch.bfloat16, 6))
    start, end = (t.cuda() for t in S.spans_of("prefix", b, s, 3))
    slopes = S.slopes_of(hq).cuda()
    args = {"scale": 0.125, "softcap": 12.0}
    want = flash_attention(q, k, v, slopes=slopes, spans=SpanMask(start=start, end=end), **args)
    other = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    wide = torch.zeros(hq, 3, dtype=torch.float64, device="cuda")
    wide[:, 1] = slopes
    sp = SpanMask(start=start[:, :1].expand(b, s).to(torch.int64), end=end.to(torch.int64).t().contiguous().t())
    assert torch.equal(want, flash_attention(*other, slopes=wide[:, 1], spans=sp, **args))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qs = [(x + 0).requires_grad_(True) for x in (q, k, v)]
        o = flash_attention(*qs, slopes=slopes, spans=SpanMask(start=start, end=end), validate_segments=False, **args)
        o.backward(d_o)
    torch.cuda.current_stream().wait_stream(side)
    base = [x.clone().requires_grad_(True) for x in (q, k, v)]
    flash_attention(*base, slopes=slopes, spans=SpanMask(start=start, end=end), **args).backward(d_o)
    assert torch.equal(o, want) and all(torch.equal(x.grad, y.grad) for x, y in zip(qs, base))


def test_a_step_repeats_to_the_bit():
    from mlx_train_perf.attention import SpanMask, flash_attention

    b, hq, hkv, s, dh = 2, 8, 2, 700, 128   # the dK/dV pass is split here
    q, k, v, d_o = (x.cuda() for x in S.inputs(b, hq, hkv, s, dh, torch.bfloat16, 8))
    sp = SpanMask(*(t.cuda() for t in S.spans_of("docs", b, s, 3)))
    runs = []
    for _ in range(3):
        qs = [x.clone().requires_grad_(True) for x in (q, k, v)]
        o = flash_attention(*qs, scale=0.1, softcap=20.0, spans=sp)
        o.backward(d_o)
        runs.append([o.detach(), *(x.grad for x in qs)])
    for r in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(r, runs[0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_steps(dtype):
    """Two graphs of different calls, replayed in turn with new inputs and spans, between eager steps."""
    from mlx_train_perf.attention import SpanMask, flash_attention

    b, hq, hkv, s, dh = 2, 4, 2, 260, 64
    def make(seed, mask):
        x = [t.cuda() for t in S.inputs(b, hq, hkv, s, dh, dtype, seed)]
        return x, [t.cuda() for t in S.spans_of(mask, b, s, seed)]

    def step(x, sp, cap):
        qs = [t.detach().requires_grad_(True) for t in x[:3]]
        o = flash_attention(*qs, scale=0.125, softcap=cap, spans=SpanMask(*sp), validate_segments=False)
        return [o.detach(), *torch.autograd.grad(o, qs, x[3])]

    graphs = []
    for seed, mask, cap in ((1, "docs", 10.0), (2, "ragged", None)):
        x, sp = make(seed, mask)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(x, sp, cap)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, sp, cap)
        graphs.append((g, x, sp, cap, out, mask))
    for turn in range(3):
        for n, (g, x, sp, cap, out, mask) in enumerate(graphs):
            nx, nsp = make(10 * turn + n + 5, mask)
            for old, new in zip([*x, *sp], [*nx, *nsp]):
                old.copy_(new)
            g.replay()
            torch.cuda.synchronize()
            want = step(nx, nsp, cap)
            assert all(torch.equal(a, w) for a, w in zip(out, want)), (turn, n)


def test_offsets_past_32_bits():
    """q of more than 2^31 elements: a window over a long row of many heads, checked at its far end."""
    from mlx_train_perf.attention import SpanMask, flash_attention

    hq, s, dh, w = 72, 240000, 128, 40
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(1, hq, s, dh, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    k, v = (torch.randn(1, hq, s, dh, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True) for _ in range(2))
    assert q.numel() > 2 ** 31
    i = torch.arange(s, device="cuda", dtype=torch.int32)[None]
    sp = SpanMask(start=(i - w + 1).clamp(min=0), end=i + 1)
    o = flash_attention(q, k, v, scale=dh ** -0.5, softcap=30.0, spans=sp)
    d_o = torch.zeros_like(o)
    tail = 200
    d_o[:, -1, -tail:] = torch.randn(tail, dh, generator=g, device="cuda", dtype=torch.bfloat16)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), d_o)
    cut = [x[:, -1:, -tail - w:].detach() for x in (q, k, v)]
    see = (i[0, :tail + w, None] >= i[:, :tail + w]) & (i[0, :tail + w, None] - i[:, :tail + w] < w)
    want = S.attention(*cut, d_o[:, -1:, -tail - w:], scale=dh ** -0.5, see=see[None], softcap=30.0)
    for name, a, x in zip(("o", "dq", "dk", "dv"), (o, dq, dk, dv), want):
        assert S.rel(a[:, -1:, -tail:], x[:, :, -tail:]) <= 1e-2, name
    assert not dq[:, :-1].any() and not dk[:, :-1].any() and not dq[:, -1, :-tail].any()


@pytest.mark.parametrize("dh", [64, 96, 128])
@pytest.mark.parametrize(("mask", "cap", "biased"), [("causal", 30.0, True), ("full", None, True), ("docs", 9.0, False),
                                                     ("ragged", None, False), ("window", 80.0, True)])
def test_fp32_passes_split_over_the_keys(dh, mask, cap, biased):
    """Few workgroups: the forward and dQ are split, and their parts (some without a key of a row) joined."""
    from mlx_train_perf import _native

    assert _native.load().mtp_attn_scored_fwd_f32_workspace_bytes(1, 4, 2, 777, dh) > 0
    _check(1, 4, 2, 777, dh, mask=mask, cap=cap, biased=biased, dtype=torch.float32, seed=dh)


def test_fp32_without_room_for_parts():
    """No workspace in the forward, D's alone in the backward: unsplit, the same sums in another order."""
    from mlx_train_perf import _native
    from mlx_train_perf.attention.api import scored_backward, scored_forward

    lib = _native.load()
    b, hq, hkv, s, dh = 1, 4, 2, 600, 64
    q, k, v, d_o = (x.cuda() for x in S.inputs(b, hq, hkv, s, dh, torch.float32, 3))
    slopes = S.slopes_of(hq).cuda()
    args = {"scale": 0.125, "causal": True, "softcap": 9.0}
    o, lse, low, plan = scored_forward(q, k, v, slopes, None, None, **args)
    assert low is None and plan is None   # bf16's alone
    grads = scored_backward(q, k, v, o, low, plan, lse, d_o, slopes, None, None, **args)
    o1, lse1 = torch.empty_like(o), torch.empty_like(lse)
    outs = [torch.empty_like(x) for x in (q, k, v)]
    ws = torch.empty(b * hq * s, device="cuda")
    st = _native.stream_of(q)
    common = (b, hq, hkv, s, dh, 0.125, 1, 9.0, slopes.data_ptr(), None, None)
    assert lib.mtp_attn_scored_fwd_f32(q.data_ptr(), k.data_ptr(), v.data_ptr(), *common, o1.data_ptr(), lse1.data_ptr(), None, 0, st) == 0
    assert lib.mtp_attn_scored_bwd_f32(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), d_o.data_ptr(), *common,
                                       *(x.data_ptr() for x in outs), ws.data_ptr(), ws.numel() * 4, st) == 0
    for a, c in zip((o1, lse1, *outs), (o, lse, *grads)):
        assert S.rel(a, c) <= 2 * BAR[torch.float32]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap", [20.0, 100.0, None])
@pytest.mark.parametrize("mask", ["causal", "full", "ragged", "window"])
@pytest.mark.parametrize(("s", "dh"), [(1, 64), (70, 96), (300, 64), (300, 128)])
def test_slopes_of_either_sign(s, dh, mask, cap, dtype):
    """Slopes below 0 raise far keys: biases of up to 75, past fp32's largest exponential when a cap of 20 is added. A
    score is then the last of four roundings (slope times distance, the two sums, L) of at most 75: 4 * 75 * 2^-24 on top."""
    slopes = torch.tensor([0.25, -0.25, 0.0, -0.01])
    _check(1, 4, 2, s, dh, mask=mask, cap=cap, biased=True, dtype=dtype, seed=s, slopes=slopes, more_bar=4 * 75 * 2 ** -24)


@pytest.mark.parametrize("mask", ["causal", "window"])
def test_values_of_every_size(mask):
    """Scores at a cap of 50 (probabilities against a fixed maximum span 2^144): V times a power of 2 gives O times it."""
    q, k, v, d_o = S.inputs(1, 4, 2, 200, 64, torch.bfloat16, 4, std=40.0)
    spans = S.spans_of(mask, 1, 200, 4)
    base = _call(q, k, v, d_o, mask=mask, spans=spans, scale=1.0, softcap=50.0)[0]
    assert torch.isfinite(base).all()
    for power in (24, 10, -30):
        o = _call(q, k, v * 2.0 ** power, d_o, mask=mask, spans=spans, scale=1.0, softcap=50.0)[0]
        assert S.rel(o * 2.0 ** -power, base.double()) <= 1e-6, power


def _forms():
    from mlx_train_perf.attention import SpanMask

    sp = SpanMask(*(t.cuda() for t in S.spans_of("prefix", 2, 150, 3)))
    return [{"softcap": 9.0}, {"slopes": S.slopes_of(4).cuda(), "softcap": 80.0, "spans": sp}, {"spans": sp}]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_node_and_function_agree(dtype, monkeypatch):
    """The C++ node and the Python Function are the same calls, to the bit."""
    from mlx_train_perf import _native
    from mlx_train_perf.attention import flash_attention

    x = [t.cuda() for t in S.inputs(2, 4, 2, 150, 64, dtype, 6)]

    def step(kw):
        qs = [t.detach().requires_grad_(True) for t in x[:3]]
        o = flash_attention(*qs, scale=0.125, **kw)
        return [o.detach(), *torch.autograd.grad(o, qs, x[3])]

    assert _native.nodes() is not None
    with_node = [step(kw) for kw in _forms()]
    monkeypatch.setattr(_native, "nodes", lambda: None)
    for kw, a in zip(_forms(), with_node):
        assert all(torch.equal(p, r) for p, r in zip(a, step(kw)))


@pytest.mark.parametrize("node", [True, False])
def test_second_derivative_is_refused(node, monkeypatch):
    from mlx_train_perf import _native
    from mlx_train_perf.attention import flash_attention

    if not node:
        monkeypatch.setattr(_native, "nodes", lambda: None)
    q, k, v, d_o = (t.cuda().requires_grad_(True) for t in S.inputs(1, 2, 1, 40, 64, torch.float32, 6))
    o = flash_attention(q, k, v, scale=0.125, softcap=9.0)
    dq, dk = torch.autograd.grad(o, (q, k), d_o, create_graph=True)
    want = torch.autograd.grad(flash_attention(q, k, v, scale=0.125, softcap=9.0), (q, k), d_o.detach())
    assert torch.equal(dq, want[0]) and torch.equal(dk, want[1])
    with pytest.raises(RuntimeError, match="differentiate twice"):
        (dq.square().sum() + o.sum()).backward()


@pytest.mark.parametrize(("cap", "biased"), [(None, True), (20.0, False), (20.0, True), (None, False)])
@pytest.mark.parametrize(("s", "w"), [(17, 2), (200, 3), (200, 6)])
@pytest.mark.parametrize("dh", [64, 96, 128])
def test_gradients_of_rows_with_few_keys(dh, s, w, cap, biased):
    """dS = P (dP - D) all but cancels here, so that an error of D shows: D comes from more bits of O than bf16's, and O is
    divided by the sum of the rounded probabilities. What is left in dq and dk are the roundings of those (by
    sum_j dP_j (P_j' - P_j), which is of dS's own size as both sum to 1), of dS and of the output, each of rms
    2^-8 / sqrt(3) at most: 3.9e-3 together."""
    hq, hkv = 4, 2
    q, k, v, d_o = (x.cuda() for x in S.inputs(1, hq, hkv, s, dh, torch.bfloat16, w))
    i = torch.arange(s, dtype=torch.int32)[None]
    spans = ((i - w + 1).clamp(min=0).to(torch.int32), i + 1)
    slopes = torch.tensor([0.7, 0.3, 0.1, 0.01]).cuda() if biased else None
    got = _call(q, k, v, d_o, mask="window", spans=spans, scale=dh ** -0.5, softcap=cap, slopes=slopes)
    see = S.visible("window", spans, 1, s, "cuda")
    want = S.attention(q, k, v, d_o, scale=dh ** -0.5, see=see, softcap=cap, slopes=slopes)
    for name, a, x in zip(("dq", "dk"), got[1:], want[1:]):
        assert S.rel(a, x) <= 4e-3, name


@pytest.mark.parametrize(("b", "hq", "hkv", "s", "dh"), [(1, 4, 4, 100, 64), (1, 8, 8, 700, 64), (2, 16, 4, 509, 128), (2, 8, 2, 300, 96),
                                                    (4, 32, 8, 900, 64)])
@pytest.mark.parametrize(("mask", "cap", "biased"), [("causal", 20.0, False), ("prefix", None, False), ("full", None, True)])
def test_splits_of_the_key_blocks(b, hq, hkv, s, dh, mask, cap, biased):
    """dK/dV of a key block by one workgroup, and by two, four and eight; more workgroups than run at once, in work orders
    under spans."""
    _check(b, hq, hkv, s, dh, mask=mask, cap=cap, biased=biased, dtype=torch.bfloat16, seed=s)


def test_with_and_without_a_plan():
    """Spans of many workgroups: the forward's plan (its order of work, and the backward's) changes no bit."""
    from mlx_train_perf.attention.api import scored_backward, scored_forward

    b, hq, hkv, s, dh = 4, 32, 8, 900, 64
    q, k, v, d_o = (x.cuda() for x in S.inputs(b, hq, hkv, s, dh, torch.bfloat16, 3))
    start, end = (t.cuda() for t in S.spans_of("docs", b, s, 3))
    args = {"scale": 0.125, "causal": False, "softcap": 0.0}
    o, lse, low, plan = scored_forward(q, k, v, None, start, end, **args)
    assert plan is not None
    bare = scored_forward(q, k, v, None, start, end, train=False, **args)
    assert bare[2] is None and bare[3] is None and torch.equal(o, bare[0]) and torch.equal(lse, bare[1])
    a = scored_backward(q, k, v, o, low, plan, lse, d_o, None, start, end, **args)
    c = scored_backward(q, k, v, o, low, None, lse, d_o, None, start, end, **args)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_captured_step_with_a_plan():
    """The plan belongs to the captured step: replays with new spans work out theirs, between eager steps."""
    from mlx_train_perf import _native
    from mlx_train_perf.attention import SpanMask, flash_attention

    b, hq, hkv, s, dh = 4, 32, 8, 700, 64
    assert _native.load().mtp_attn_scored_plan_bytes(b, hq, hkv, s, dh) > 0
    x = [t.cuda() for t in S.inputs(b, hq, hkv, s, dh, torch.bfloat16, 1)]
    sp = [t.cuda() for t in S.spans_of("docs", b, s, 1)]

    def step(spans):
        qs = [t.detach().requires_grad_(True) for t in x[:3]]
        o = flash_attention(*qs, scale=0.125, softcap=30.0, spans=SpanMask(*spans), validate_segments=False)
        return [o.detach(), *torch.autograd.grad(o, qs, x[3])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sp)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(sp)
    for turn, mask in enumerate(("docs", "ragged", "window", "nothing", "prefix")):
        new = [t.cuda() for t in S.spans_of(mask, b, s, turn + 7)]
        for old, t in zip(sp, new):
            old.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(out, step(new))), mask


@pytest.mark.parametrize(("b", "hq", "hkv", "s", "dh"), [(1, 2, 1, 520, 64), (1, 1, 1, 1100, 128), (1, 8, 2, 777, 96), (2, 4, 4, 300, 128),
                                                    (2, 4, 4, 600, 128)])
@pytest.mark.parametrize(("mask", "cap", "biased"), [("causal", 20.0, False), ("full", None, True), ("docs", 30.0, True),
                                                     ("ragged", None, False), ("window", 80.0, False), ("prefix", None, True),
                                                     ("causal", 20.0, True)])
def test_passes_split_over_the_keys(b, hq, hkv, s, dh, mask, cap, biased):
    """Few workgroups: the forward and dQ of bf16 are split, and their parts (some without a key of a row) joined. O, L and
    the bits below O are those of an unsplit forward but for the order of sums; without a workspace it is unsplit."""
    from mlx_train_perf import _native
    from mlx_train_perf.attention.api import scored_forward

    lib = _native.load()
    assert (lib.mtp_attn_scored_fwd_workspace_bytes(b, hq, hkv, s, dh) > 0) == (s >= 512)   # two splits of four tiles
    _check(b, hq, hkv, s, dh, mask=mask, cap=cap, biased=biased, dtype=torch.bfloat16, seed=dh)
    q, k, v, _ = (x.cuda() for x in S.inputs(b, hq, hkv, s, dh, torch.bfloat16, 3))
    slopes = S.slopes_of(hq).cuda() if biased else None
    spans = S.spans_of(mask, b, s, 3)
    start, end = (None, None) if spans is None else (t.cuda() for t in spans)
    causal = mask == "causal"
    o, lse, low, _ = scored_forward(q, k, v, slopes, start, end, scale=0.1, causal=causal, softcap=cap or 0.0)
    o1, low1, lse1 = torch.empty_like(o), torch.empty_like(low), torch.empty_like(lse)
    assert lib.mtp_attn_scored_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), b, hq, hkv, s, dh, 0.1, int(causal), cap or 0.0,
                                   _native.ptr(slopes), _native.ptr(start), _native.ptr(end), o1.data_ptr(), low1.data_ptr(), None,
                                   lse1.data_ptr(), None, 0, _native.stream_of(q)) == 0
    fine = lambda x, y: (x.float().view(torch.int32) + (y.to(torch.int32) << 8)).view(torch.float32).double()  # noqa: E731
    seen = torch.isfinite(lse1)
    assert torch.equal(seen, torch.isfinite(lse)) and torch.allclose(lse[seen], lse1[seen], rtol=2e-6, atol=2e-5)
    assert S.rel(fine(o, low), fine(o1, low1)) <= 2 ** -8   # another maximum rounds the probabilities elsewhere


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_split_step_beside_another_stream(dtype):
    """A captured step whose passes are split, replayed while an eager step of other tensors runs on a stream of its own:
    each has its workspaces."""
    from mlx_train_perf.attention import flash_attention

    b, hq, hkv, s, dh = 1, 4, 2, 900, 64
    made = [[t.cuda() for t in S.inputs(b, hq, hkv, s, dh, dtype, seed)] for seed in (1, 2)]
    slopes = S.slopes_of(hq).cuda()

    def step(x, cap):
        qs = [t.detach().requires_grad_(True) for t in x[:3]]
        o = flash_attention(*qs, scale=0.125, softcap=cap, slopes=slopes)
        return [o.detach(), *torch.autograd.grad(o, qs, x[3])]

    want = [step(made[0], 20.0), step(made[1], None)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(made[0], 20.0)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(made[0], 20.0)
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            eager = step(made[1], None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(out, want[0])) and all(torch.equal(a, w) for a, w in zip(eager, want[1]))
