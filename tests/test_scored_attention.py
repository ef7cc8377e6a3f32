"""Attention with softcap, slopes and spans on the CPU: the plain form against differences, impl="reference" against
the plain form, the span builders, and every refusal (which come before any launch)."""
from __future__ import annotations

import math
import re

import pytest
import torch

from mlx_train_perf import _native
from mlx_train_perf.attention import PackedMask, SpanMask, document_spans, flash_attention, math_attention, prefix_spans
from mlx_train_perf.attention.api import resolve_attention_impl
from mlx_train_perf.attention.segments import packed_as_spans, span_allowed, span_violation
from mlx_train_perf.errors import AttentionInputError, UnsupportedAttentionError
from oracle import attention as oatt
from tests import _scored as S

FORMS = [(None, False), (1.5, False), (None, True), (5.0, True)]


@pytest.mark.parametrize(("cap", "biased"), FORMS)
@pytest.mark.parametrize("mask", ["causal", "prefix", "ragged"])
def test_plain_gradients_against_differences(mask, cap, biased):
    b, hq, hkv, s, dh = 2, 4, 2, 9, 8
    q, k, v, d_o = (x.double() for x in S.inputs(b, hq, hkv, s, dh, torch.float64, 3))
    see = S.visible(mask, S.spans_of(mask, b, s, 1), b, s)
    args = {"scale": 0.4, "see": see, "softcap": cap, "slopes": S.slopes_of(hq) if biased else None}
    _, *grads = S.attention(q, k, v, d_o, **args)
    g = torch.Generator().manual_seed(0)
    for n, grad in enumerate(grads):
        u = torch.randn(grad.shape, generator=g, dtype=torch.float64)
        h = 1e-5

        def f(t):
            x = [q, k, v]
            x[n] = x[n] + t * u
            return float((S.attention(*x, d_o, **args)[0] * d_o).sum())

        want = (f(h) - f(-h)) / (2 * h)   # off by h^2 of the third derivative and 2^-52 |f| / h: about 1e-9
        assert abs(float((grad * u).sum()) - want) <= 1e-6 * max(1.0, abs(want))


@pytest.mark.parametrize(("cap", "biased"), FORMS)
@pytest.mark.parametrize("mask", S.MASKS)
def test_reference_impl_matches_the_plain_form(mask, cap, biased):
    if mask in ("causal", "full") and cap is None and not biased:
        pytest.skip("the plain scores and masks have their own tests")
    b, hq, hkv, s, dh = 3, 4, 2, 37, 16
    q, k, v, d_o = S.inputs(b, hq, hkv, s, dh, torch.float32, 5)
    spans = S.spans_of(mask, b, s, 2)
    slopes = S.slopes_of(hq) if biased else None
    want = S.attention(q, k, v, d_o, scale=0.25, see=S.visible(mask, spans, b, s), softcap=cap, slopes=slopes)
    qs = [x.clone().requires_grad_(True) for x in (q, k, v)]
    sm = None if spans is None else SpanMask(*spans)
    o = flash_attention(*qs, scale=0.25, causal=mask == "causal", impl="reference", softcap=cap, slopes=slopes, spans=sm)
    got = [o, *torch.autograd.grad(o, qs, d_o)]
    # fp32 sums of at most 37 terms and 16 products: some 2^-24 * sqrt(50) of the largest term each; 1e-5 is 20 times that.
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert S.rel(a, w) <= 1e-5, (name, S.rel(a, w))
    m = math_attention(q, k, v, scale=0.25, causal=mask == "causal", softcap=cap, slopes=slopes, spans=sm)
    assert S.rel(m, want[0]) <= 1e-5


def test_prefix_spans():
    sp = prefix_spans([0, 3, 5], 5)
    see = span_allowed(sp)[:, 0]
    for r, p in enumerate((0, 3, 5)):
        for i in range(5):
            for j in range(5):
                assert bool(see[r, i, j]) == (j <= i or (i < p and j < p)), (r, i, j)
    assert span_violation(sp) is None and sp.start.dtype == sp.end.dtype == torch.int32


def test_document_spans():
    sid, sst = oatt.segments_from_lengths([3, 4, 2])
    seg = PackedMask(seg_id=sid[None], seg_start=sst[None])
    assert torch.equal(span_allowed(document_spans(seg)), oatt.segment_allowed(sid[None]))
    assert torch.equal(span_allowed(packed_as_spans(seg)), oatt.segment_allowed(sid[None]))
    whole = span_allowed(document_spans(seg, causal=False))[0, 0]
    assert torch.equal(whole, sid[:, None] == sid[None, :])
    prompt = torch.tensor([[2, 2, 2, 3, 3, 3, 3, 9, 9]])   # the last is longer than its document
    sp = document_spans(seg, prefix=prompt, used=[8])
    see = span_allowed(sp)[0, 0]
    for i in range(9):
        for j in range(9):
            p = int(sst[i] + prompt[0, i])
            want = sid[i] == sid[j] and i < 8 and j < 8 and (j <= i or (i < p and j < p))
            assert bool(see[i, j]) == bool(want), (i, j)
    assert span_violation(sp) is None


@pytest.mark.parametrize(("start", "end", "what"), [
    ([[0, 1, 0]], [[1, 2, 3]], "start must not decrease"),
    ([[0, 0, 0]], [[3, 2, 3]], "end must not decrease"),
    ([[-1, 0, 0]], [[1, 2, 3]], r"start must lie in \[0, 3\]"),
    ([[0, 0, 0]], [[1, 2, 4]], r"end must lie in \[0, 3\]"),
])
def test_span_contract(start, end, what):
    q = torch.zeros(1, 2, 3, 64)
    sp = SpanMask(start=torch.tensor(start), end=torch.tensor(end))
    with pytest.raises(AttentionInputError, match=what):
        flash_attention(q, q, q, scale=1.0, impl="reference", spans=sp)


def test_refusals():
    q = torch.zeros(1, 4, 6, 64)
    z = torch.zeros(1, 6, dtype=torch.int32)
    sp = SpanMask(start=z, end=z)

    def call(**kw):
        return resolve_attention_impl(q, q, q, impl="reference", **kw)

    for cap in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(AttentionInputError, match="softcap"):
            call(softcap=cap)
    for bad in (torch.zeros(3), torch.zeros(1, 4), torch.zeros(4, dtype=torch.int64)):
        with pytest.raises(AttentionInputError, match="slopes"):
            call(slopes=bad)
    with pytest.raises(AttentionInputError, match="slopes get no gradient"):
        call(slopes=torch.zeros(4, requires_grad=True))
    with torch.no_grad():
        call(slopes=torch.zeros(4, requires_grad=True))
    with pytest.raises(AttentionInputError, match="not both"):
        call(spans=sp, segments=PackedMask(seg_id=z, seg_start=z))
    with pytest.raises(AttentionInputError, match="spans.end must have shape"):
        call(spans=SpanMask(start=z, end=z[:, :5]))
    with pytest.raises(AttentionInputError, match="spans.start must be an integer"):
        call(spans=SpanMask(start=z.float(), end=z))
    with pytest.raises(UnsupportedAttentionError):   # the kernel gate, as without a cap
        resolve_attention_impl(q.half(), q.half(), q.half(), impl="kernel", softcap=1.0)
    for cap in (1e-50, 9e-4, 1001.0):   # the first is an fp32 0
        assert call(softcap=cap) == "reference"
        with pytest.raises(UnsupportedAttentionError, match="softcap in"):
            resolve_attention_impl(q, q, q, impl="kernel", softcap=cap, slopes=torch.zeros(4))


def test_c_abi_refusals():
    lib = _native.load()
    p, none, shape = 1 << 20, None, (1, 2, 1, 8, 64)

    def fwd(scale=1.0, causal=0, cap=1.0, slopes=none, start=none, end=none, q=p, o=p, shape=shape, lib_fn=lib.mtp_attn_scored_fwd):
        f32 = lib_fn is lib.mtp_attn_scored_fwd_f32
        return lib_fn(q, p, p, *shape, scale, causal, cap, slopes, start, end, o, *(() if f32 else (none, none)), p,
                      none, 0, none)

    bad, un = _native.MTP_ERR_INPUT, _native.MTP_ERR_UNSUPPORTED
    for fn in (lib.mtp_attn_scored_fwd, lib.mtp_attn_scored_fwd_f32):
        for kw, rc, what in [({"scale": 0.0}, bad, "scale"), ({"scale": math.nan}, bad, "scale"), ({"scale": -1.0}, bad, "scale"),
                             ({"cap": -1.0}, bad, "softcap"), ({"cap": math.inf}, bad, "softcap"), ({"cap": math.nan}, bad, "softcap"),
                             ({"start": p}, bad, "span_start and span_end"), ({"start": p, "end": p, "causal": 1}, bad, "causal must be 0"),
                             ({"cap": 0.0}, bad, "no softcap"), ({"cap": 9e-4}, un, "softcap"), ({"cap": 1001.0}, un, "softcap"), ({"q": none}, bad, "non-null"), ({"o": none}, bad, "non-null"),
                             ({"q": p + 2}, un, "aligned"), ({"shape": (1, 3, 2, 8, 64)}, bad, "multiple"),
                             ({"shape": (1, 2, 1, 8, 80)}, un, "head_dim"), ({"shape": (1, 2, 1, 1 << 23, 64)}, bad, "2\\^23"),
                             ({"causal": 2}, bad, "causal")]:
            assert fwd(lib_fn=fn, **kw) == rc, kw
            assert re.search(what, _native.last_error()), (kw, _native.last_error())
    ws = lib.mtp_attn_scored_bwd_workspace_bytes(*shape)
    assert ws > 0 and lib.mtp_attn_scored_bwd_workspace_bytes(1, 3, 2, 8, 64) == 0
    assert ws % 256 == 0 and ws >= 2 * 8 * 4 + 2 * 8 * 4

    def bwd(bytes_, workspace=p, d_o=p, low=p, plan=none, fn=lib.mtp_attn_scored_bwd):
        out = (p,) if fn is lib.mtp_attn_scored_bwd_f32 else (p, low, plan)
        return fn(p, p, p, *out, p, d_o, *shape, 1.0, 0, 1.0, none, none, none, p, p, p, workspace, bytes_, none)

    assert bwd(ws - 1) == _native.MTP_ERR_WORKSPACE and bwd(ws, workspace=none) == _native.MTP_ERR_WORKSPACE
    assert bwd(ws, workspace=p + 4) == un and bwd(ws, d_o=none) == bad
    assert bwd(ws, low=none) == bad and bwd(ws, low=p + 8) == un and bwd(ws, plan=p + 8) == un
    assert lib.mtp_attn_scored_plan_bytes(*shape) == 0 and lib.mtp_attn_scored_plan_bytes(1, 16, 4, 8192, 128) >= 2 * 8192 * 4
    assert bwd(8, fn=lib.mtp_attn_scored_bwd_f32) == _native.MTP_ERR_WORKSPACE
    # fp32: parts of 4 splits of one pair of 64-query blocks of 8 heads (64 workgroups), 33 tiles of 32 keys
    assert lib.mtp_attn_scored_fwd_f32_workspace_bytes(1, 8, 2, 1000, 128) == 4 * 8 * 1000 * 130 * 4
    assert lib.mtp_attn_scored_fwd_f32_workspace_bytes(1, 32, 8, 8192, 128) == 0    # enough workgroups
    assert lib.mtp_attn_scored_fwd_f32_workspace_bytes(1, 1, 1, 100, 64) == 0       # too few tiles
    assert lib.mtp_attn_scored_bwd_f32_workspace_bytes(1, 8, 2, 1000, 128) >= 8000 * 4 + 4 * 8 * 1000 * 128 * 4


def test_spans_of_inference_mode():
    """Tensors made in inference mode have no version: their contract is checked at every call."""
    with torch.inference_mode():
        q = torch.randn(1, 2, 5, 64)
        end = torch.arange(1, 6, dtype=torch.int32)[None]
        sp = SpanMask(start=torch.zeros_like(end), end=end)
        for _ in range(2):
            o = flash_attention(q, q, q, scale=1.0, impl="reference", spans=sp)
        assert torch.allclose(o, flash_attention(q, q, q, scale=1.0, impl="reference"), atol=1e-6)
        end.fill_(6)
        with pytest.raises(AttentionInputError, match="end must lie"):
            flash_attention(q, q, q, scale=1.0, impl="reference", spans=sp)
