"""`flash_attention` public API (mirror of src/mlx_train_perf/attention/api.py on torch tensors).

Residual contract (api.py:1-18): the autograd Function returns (O, L); L is a real output, marked
non-differentiable, and only O reaches the caller. The backward reads q, k, v and the saved O, L.

`impl="auto"`/`"kernel"`: the HIP kernels of libmtp_hip.so (bf16 on bf16 MFMA, fp32 on fp32 MFMA
with fp32 outputs and gradients; head_dim in {64, 96, 128}; causal with optional packed segments,
or non-causal -- an extension: the reference kernel refuses causal=False, api.py:109-113). `impl="reference"`: the materialized oracle with the hand-written
FlashAttention backward over full tensors -- an explicit opt-in, O(N^2) memory, small N only.
No silent fallback: unsupported configs raise the reference's typed errors.

Beyond the reference: `softcap` (scores capped by a tanh), `slopes` (a bias by distance) and `spans` (a range of
keys for each query), on both impls and both dtypes, forward and backward; the kernel impl serves them by the
mtp_attn_scored_* entry points.
"""
from __future__ import annotations

import math
import weakref
from typing import Literal

import torch
from torch.autograd.function import once_differentiable

from mlx_train_perf import _compat, _native
from mlx_train_perf.attention.reference import flash_attention_reference, hide, kv_head_for, scores_of
from mlx_train_perf.attention.segments import PackedMask, SpanMask, layout_violation, packed_as_spans
from mlx_train_perf.errors import AttentionInputError, UnsupportedAttentionError

_KERNEL_DTYPES = (torch.bfloat16, torch.float32)   # the reference kernel's T (api.py:41-43)
_KERNEL_HEAD_DIMS = (64, 96, 128)
_KERNEL_CAPS = (1e-3, 1e3)   # beyond it fp32 has no tanh of the scores, or none that bends them

VJP_CALLS: dict[str, int] = {}


def _validate_shapes(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    """api.py:52-72."""
    for name, arr in (("q", q), ("k", k), ("v", v)):
        if arr.dim() != 4:
            raise AttentionInputError(f"{name} must be 4-D (B, H, N, D); got shape {tuple(arr.shape)}")
    b_q, hq, n_q, d_q = q.shape
    b_k, hkv, n_k, d_k = k.shape
    b_v, hv, n_v, d_v = v.shape
    if b_q < 1:
        raise AttentionInputError(f"batch must be >= 1; got {b_q}")
    if not (b_q == b_k == b_v):
        raise AttentionInputError(f"batch mismatch: q={b_q}, k={b_k}, v={b_v}")
    if hkv != hv:
        raise AttentionInputError(f"k/v head-count mismatch: k has {hkv} heads, v has {hv}")
    if hq % hkv != 0:
        raise AttentionInputError(f"Hq={hq} must be a multiple of Hkv={hkv} for GQA grouping")
    if not (n_q == n_k == n_v):
        raise AttentionInputError(f"sequence length mismatch: q={n_q}, k={n_k}, v={n_v}")
    if not (d_q == d_k == d_v):
        raise AttentionInputError(f"head_dim mismatch: q={d_q}, k={d_k}, v={d_v}")
    if not (q.device == k.device == v.device):
        raise AttentionInputError(f"q, k, v must be on one device; got {q.device}, {k.device}, {v.device}")


# Segment tensors whose layout passed `layout_violation`: weak references to the two tensors and their
# version counters. A model calls flash_attention once per layer with the same mask, so the check
# (one device pass and a host sync) runs once per mask rather than once per layer; an in-place edit
# bumps a version and a new tensor is a new object, so either is checked again.
_CHECKED_LAYOUTS: dict[int, tuple] = {}


def _layout_seen(segments: PackedMask) -> bool:
    ent = _CHECKED_LAYOUTS.get(id(segments.seg_id))
    return (ent is not None and ent[0]() is segments.seg_id and ent[1]() is segments.seg_start
            and ent[2] == (segments.seg_id._version, segments.seg_start._version))


def _validate_segments(q: torch.Tensor, segments: PackedMask, *, check_layout: bool = False) -> None:
    b, _, n, _ = q.shape
    for name, t in (("seg_id", segments.seg_id), ("seg_start", segments.seg_start)):
        if tuple(t.shape) != (b, n):
            raise AttentionInputError(f"segments.{name} must have shape (B, N)=({b}, {n}); got {tuple(t.shape)}")
        if t.dtype.is_floating_point or t.dtype == torch.bool or t.dtype.is_complex:
            raise AttentionInputError(f"segments.{name} must be an integer tensor; got {t.dtype}")
    if check_layout and not _layout_seen(segments):
        problem = layout_violation(segments.seg_id, segments.seg_start)
        if problem is not None:
            raise AttentionInputError(f"segments violate the packed-row layout contract: {problem}")
        if len(_CHECKED_LAYOUTS) > 64:
            _CHECKED_LAYOUTS.clear()
        sid, sst = segments.seg_id, segments.seg_start
        _CHECKED_LAYOUTS[id(sid)] = (weakref.ref(sid), weakref.ref(sst), (sid._version, sst._version))


def _validate_score(q: torch.Tensor, softcap: float | None, slopes: torch.Tensor | None, spans: SpanMask | None,
                    segments: PackedMask | None, *, check_spans: bool) -> None:
    b, hq, n, _ = q.shape
    if softcap is not None and not (math.isfinite(softcap) and softcap > 0):
        raise AttentionInputError(f"softcap must be a positive finite number, or None for none; got {softcap!r}")
    if slopes is not None:
        if tuple(slopes.shape) != (hq,) or not slopes.dtype.is_floating_point:
            raise AttentionInputError(f"slopes must be {hq} floating-point values, one per query head; got {slopes.dtype} "
                                      f"of shape {tuple(slopes.shape)}")
        if slopes.device != q.device:
            raise AttentionInputError(f"slopes are on {slopes.device}, q on {q.device}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise AttentionInputError("slopes get no gradient: detach them")
    if spans is not None:
        if segments is not None:
            raise AttentionInputError("give segments or spans, not both: spans are the whole mask")
        for name, t in (("start", spans.start), ("end", spans.end)):
            if t.shape != (b, n):
                raise AttentionInputError(f"spans.{name} must have shape (B, N)=({b}, {n}); got {tuple(t.shape)}")
            if t.dtype is not torch.int32 and (t.dtype.is_floating_point or t.dtype == torch.bool or t.dtype.is_complex):
                raise AttentionInputError(f"spans.{name} must be an integer tensor; got {t.dtype}")
        if check_spans:
            problem = spans.violation()
            if problem is not None:
                raise AttentionInputError(f"spans violate their contract: {problem}")


def resolve_attention_impl(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, impl: str, causal: bool = True,
                           segments: PackedMask | None = None, validate_segments: bool = False,
                           softcap: float | None = None, slopes: torch.Tensor | None = None,
                           spans: SpanMask | None = None) -> str:
    """api.py:75-123: "reference" is always allowed; "auto"/"kernel" run the kernel-support gate."""
    _validate_shapes(q, k, v)
    if softcap is not None or slopes is not None or spans is not None:
        _validate_score(q, softcap, slopes, spans, segments, check_spans=validate_segments)
    if segments is not None:
        _validate_segments(q, segments, check_layout=validate_segments)
        if not causal:
            raise UnsupportedAttentionError(
                "segments (packed attention) require causal=True (got causal=False); "
                "packing composes on top of the causal triangle."
            )
    if impl == "reference":
        return "reference"
    if impl not in ("auto", "kernel"):
        raise AttentionInputError(f"unknown impl {impl!r}; expected one of 'auto', 'kernel', 'reference'")
    if q.dtype not in _KERNEL_DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise UnsupportedAttentionError(
            f"kernel impl only supports fp32/bf16 (got {q.dtype}/{k.dtype}/{v.dtype}); use impl='reference'."
        )
    head_dim = q.shape[-1]
    if head_dim not in _KERNEL_HEAD_DIMS:
        raise UnsupportedAttentionError(
            f"kernel impl only supports head_dim in {_KERNEL_HEAD_DIMS} (got {head_dim}); use impl='reference'."
        )
    # (here, not in the library, which sees a cap that rounds to an fp32 0 as none)
    if softcap is not None and not _KERNEL_CAPS[0] <= softcap <= _KERNEL_CAPS[1]:
        raise UnsupportedAttentionError(
            f"kernel impl only supports a softcap in {list(_KERNEL_CAPS)} (got {softcap}); use impl='reference'."
        )
    _compat.check_device_verified(allow_unverified=False, error=UnsupportedAttentionError)
    _compat.require_gpu_tensor(q, error=UnsupportedAttentionError)
    return "kernel"


def _bwd_D(d_o: torch.Tensor, o: torch.Tensor) -> torch.Tensor:  # noqa: N802 -- the paper's name
    """D_i = sum_d dO_i,d O_i,d in fp32 (api.py:126-129)."""
    return (d_o.to(torch.float32) * o.to(torch.float32)).sum(dim=-1)


def _kv_gather(x: torch.Tensor, *, hq: int, hkv: int) -> torch.Tensor:
    group = hq // hkv
    idx = torch.tensor([kv_head_for(h, group) for h in range(hq)], device=x.device)
    return x.index_select(1, idx)


def _flash_attention_backward(q, k, v, o, lse, d_o, *, scale, causal, segments=None, softcap=None, slopes=None,
                              spans=None):
    """Hand-written FlashAttention backward over full tensors, fp32 (api.py:140-194)."""
    b, hq, n, dd = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    q32 = q.to(torch.float32)
    k_g = _kv_gather(k, hq=hq, hkv=hkv).to(torch.float32)
    v_g = _kv_gather(v, hq=hq, hkv=hkv).to(torch.float32)
    d = _bwd_D(d_o, o)
    do32 = d_o.to(torch.float32)
    s = (q32 @ k_g.transpose(-1, -2).contiguous()) * scale
    s, bend = scores_of(s, softcap=softcap, slopes=slopes)
    s = hide(s, causal=causal, segments=segments, spans=spans)
    p = torch.exp(s - lse.to(torch.float32)[..., None])
    d_p = do32 @ v_g.transpose(-1, -2).contiguous()
    d_s = p * (d_p - d[..., None])
    if bend is not None:
        d_s = d_s * bend
    d_q = scale * (d_s @ k_g)
    d_v = (p.transpose(-1, -2).contiguous() @ do32).reshape(b, hkv, group, n, dd).sum(2)
    d_k = (scale * (d_s.transpose(-1, -2).contiguous() @ q32)).reshape(b, hkv, group, n, dd).sum(2)
    return d_q.to(q.dtype), d_k.to(k.dtype), d_v.to(v.dtype)


class _ReferenceAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seg_id, seg_start, scale, causal, score=None):
        segments = None if seg_id is None else PackedMask(seg_id=seg_id, seg_start=seg_start)
        ctx.score = score or {}   # softcap, slopes, spans
        o, lse = flash_attention_reference(q, k, v, scale=scale, causal=causal, segments=segments, **ctx.score)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.segments = segments
        ctx.scale, ctx.causal = scale, causal
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    def backward(ctx, d_o, _d_l):
        VJP_CALLS["flash_attention"] = VJP_CALLS.get("flash_attention", 0) + 1
        q, k, v, o, lse = ctx.saved_tensors
        dq, dk, dv = _flash_attention_backward(q, k, v, o, lse, d_o, scale=ctx.scale, causal=ctx.causal,
                                               segments=ctx.segments, **ctx.score)
        return dq, dk, dv, None, None, None, None, None


def _seg_args(q, seg_id, seg_start):
    if seg_id is None:
        return None, None
    return seg_id.to(device=q.device, dtype=torch.int32).contiguous(), \
        seg_start.to(device=q.device, dtype=torch.int32).contiguous()


def kernel_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float,
                   seg_id: torch.Tensor | None = None, seg_start: torch.Tensor | None = None, causal: bool = True):
    """(O, L) from mtp_attn_fwd; q/k/v contiguous bf16 on the GPU. causal=False: every key visible."""
    lib = _native.load()
    b, hq, n, dh = q.shape
    hkv = k.shape[1]
    o = torch.empty_like(q)
    lse = torch.empty((b, hq, n), dtype=torch.float32, device=q.device)
    fwd = lib.mtp_attn_fwd_f32 if q.dtype == torch.float32 else lib.mtp_attn_fwd
    with _native.on_device(q):
        rc = fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), b, hq, hkv, n, dh, float(scale), int(causal),
                 _native.ptr(seg_id), _native.ptr(seg_start), o.data_ptr(), lse.data_ptr(), _native.stream_of(q))
    _native.check(rc, domain="attention")
    return o, lse


def kernel_backward(q, k, v, o, lse, d_o, *, scale: float, seg_id=None, seg_start=None, causal: bool = True):
    """(dQ, dK, dV) from mtp_attn_bwd (mtp_attn_bwd_f32 for fp32 inputs)."""
    lib = _native.load()
    b, hq, n, dh = q.shape
    hkv = k.shape[1]
    dq = torch.empty_like(q)
    dk = torch.empty_like(k)
    dv = torch.empty_like(v)
    f32 = q.dtype == torch.float32
    ws_bytes = (lib.mtp_attn_bwd_f32_workspace_bytes if f32 else lib.mtp_attn_bwd_workspace_bytes)(b, hq, hkv, n, dh)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    bwd = lib.mtp_attn_bwd_f32 if f32 else lib.mtp_attn_bwd
    with _native.on_device(q):
        rc = bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), d_o.data_ptr(), b, hq, hkv,
                 n, dh, float(scale), int(causal), _native.ptr(seg_id), _native.ptr(seg_start), dq.data_ptr(),
                 dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, _native.stream_of(q))
    _native.check(rc, domain="attention")
    return dq, dk, dv


class _KernelAttention(torch.autograd.Function):
    """The general path; flash_attention runs the C++ node of the same calls on plain tensors."""

    @staticmethod
    def forward(ctx, q, k, v, seg_id, seg_start, scale, causal):
        o, lse = kernel_forward(q, k, v, scale=scale, seg_id=seg_id, seg_start=seg_start, causal=causal)
        ctx.save_for_backward(q, k, v, o, lse, seg_id, seg_start)
        ctx.scale, ctx.causal = scale, causal
        ctx.mark_non_differentiable(lse)
        # No zeros in the place of L's gradient, which has none: autograd would fill a tensor for it in
        # every backward.
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    def backward(ctx, d_o, _d_l):
        VJP_CALLS["flash_attention"] = VJP_CALLS.get("flash_attention", 0) + 1
        VJP_CALLS["flash_attention_kernel_bwd"] = VJP_CALLS.get("flash_attention_kernel_bwd", 0) + 1
        q, k, v, o, lse, seg_id, seg_start = ctx.saved_tensors
        d_o = torch.zeros_like(o) if d_o is None else d_o.contiguous()
        dq, dk, dv = kernel_backward(q, k, v, o, lse, d_o, scale=ctx.scale, seg_id=seg_id,
                                     seg_start=seg_start, causal=ctx.causal)
        return dq, dk, dv, None, None, None, None


def scored_forward(q, k, v, slopes, start, end, *, scale: float, causal: bool, softcap: float, train: bool = True):
    """(O, L, low, plan) from mtp_attn_scored_fwd (_f32 for fp32 inputs); contiguous tensors on the GPU. low and plan are for
    the backward of bf16 inputs (None for fp32, and without `train`): the bits of O's values below its own, and what
    spans have to be known of (None where that is of no use)."""
    lib = _native.load()
    b, hq, n, dh = q.shape
    o = torch.empty_like(q)
    lse = torch.empty((b, hq, n), dtype=torch.float32, device=q.device)
    shape = (b, hq, k.shape[1], n, dh)
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), *shape, scale, int(causal), softcap, _native.ptr(slopes), _native.ptr(start),
            _native.ptr(end), o.data_ptr())
    low = plan = None
    f32 = q.dtype == torch.float32
    ws_bytes = (lib.mtp_attn_scored_fwd_f32_workspace_bytes if f32 else lib.mtp_attn_scored_fwd_workspace_bytes)(*shape)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    with _native.on_device(q):
        if f32:
            rc = lib.mtp_attn_scored_fwd_f32(*args, lse.data_ptr(), _native.ptr(ws), ws_bytes, _native.stream_of(q))
        else:
            low = torch.empty_like(q, dtype=torch.int8) if train else None
            plan_bytes = lib.mtp_attn_scored_plan_bytes(*shape) if train and start is not None else 0
            plan = torch.empty(plan_bytes // 4, dtype=torch.int32, device=q.device) if plan_bytes else None
            rc = lib.mtp_attn_scored_fwd(*args, _native.ptr(low), _native.ptr(plan), lse.data_ptr(), _native.ptr(ws),
                                         ws_bytes, _native.stream_of(q))
    _native.check(rc, domain="attention")
    return o, lse, low, plan


def scored_backward(q, k, v, o, low, plan, lse, d_o, slopes, start, end, *, scale: float, causal: bool, softcap: float):
    """(dQ, dK, dV) from mtp_attn_scored_bwd (_f32 for fp32 inputs)."""
    lib = _native.load()
    b, hq, n, dh = q.shape
    hkv = k.shape[1]
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    f32 = q.dtype == torch.float32
    ws_bytes = (lib.mtp_attn_scored_bwd_f32_workspace_bytes if f32 else lib.mtp_attn_scored_bwd_workspace_bytes)(b, hq, hkv, n, dh)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    bwd = lib.mtp_attn_scored_bwd_f32 if f32 else lib.mtp_attn_scored_bwd
    out = (o.data_ptr(),) if f32 else (o.data_ptr(), low.data_ptr(), _native.ptr(plan))
    with _native.on_device(q):
        rc = bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), *out, lse.data_ptr(), d_o.data_ptr(), b, hq, hkv, n, dh,
                 scale, int(causal), softcap, _native.ptr(slopes), _native.ptr(start), _native.ptr(end),
                 dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), ws_bytes, _native.stream_of(q))
    _native.check(rc, domain="attention")
    return dq, dk, dv


class _ScoredAttention(torch.autograd.Function):
    """Attention with softcap (0: none), slopes or spans: the general path, as _KernelAttention, whose residuals it has."""

    @staticmethod
    def forward(ctx, q, k, v, slopes, start, end, scale, causal, softcap):
        o, lse, low, plan = scored_forward(q, k, v, slopes, start, end, scale=scale, causal=causal, softcap=softcap,
                                           train=any(ctx.needs_input_grad))
        ctx.save_for_backward(q, k, v, o, low, plan, lse, slopes, start, end)
        ctx.scale, ctx.causal, ctx.softcap = scale, causal, softcap
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, _d_l):
        VJP_CALLS["flash_attention"] = VJP_CALLS.get("flash_attention", 0) + 1
        VJP_CALLS["flash_attention_kernel_bwd"] = VJP_CALLS.get("flash_attention_kernel_bwd", 0) + 1
        q, k, v, o, low, plan, lse, slopes, start, end = ctx.saved_tensors
        d_o = torch.zeros_like(o) if d_o is None else d_o.contiguous()
        dq, dk, dv = scored_backward(q, k, v, o, low, plan, lse, d_o, slopes, start, end, scale=ctx.scale, causal=ctx.causal,
                                     softcap=ctx.softcap)
        return dq, dk, dv, None, None, None, None, None, None


def _int32_on(t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.device != device:   # (asked first: a call that changes nothing costs 1 us)
        t = t.to(device=device, dtype=torch.int32)
    return t.contiguous()


def _scored_attention(q, k, v, *, scale, causal, segments, softcap, slopes, spans):
    """The kernel impl of a call with softcap, slopes or spans. Packed segments go as spans."""
    if segments is not None:
        spans = packed_as_spans(segments)
    start = end = None
    if spans is not None:
        causal = False
        start, end = _int32_on(spans.start, q.device), _int32_on(spans.end, q.device)
    if slopes is not None:
        slopes = slopes.detach().to(torch.float32).contiguous()
    args = (q.contiguous(), k.contiguous(), v.contiguous(), slopes, start, end, float(scale), bool(causal), float(softcap or 0.0))
    nodes = _native.nodes() if _native.plain(q, k, v) else None
    if nodes is not None:
        return nodes.scored_attention(*args)
    return _ScoredAttention.apply(*args)[0]


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float, causal: bool = True,
                    impl: Literal["auto", "kernel", "reference"] = "auto",
                    segments: PackedMask | None = None, validate_segments: bool = True,
                    softcap: float | None = None, slopes: torch.Tensor | None = None,
                    spans: SpanMask | None = None) -> torch.Tensor:
    """softmax(scale * Q K^T + mask) V with GQA (api.py:281-439). Only O is returned; L stays internal.

    `segments` (requires causal=True) switches on packed block-diagonal-causal attention; the
    segment tensors are passed to the kernels per call (never captured), so every step masks with
    its own layout. `validate_segments` checks the layout contract of `PackedMask` (seg_id from 0 in
    steps of 0 or 1, seg_start the first position of each segment) and raises AttentionInputError
    on a violation; the check costs one host sync per distinct mask (a model's layers share it).
    Pass False on a trusted path, like the loss's `validate_targets`.

    `softcap`: scores become softcap * tanh(score / softcap). `slopes`: (Hq,) values, slopes[h] * |i - j| is taken
    from the score of query i and key j (after the cap); they get no gradient. `spans`: a `SpanMask`, the keys that
    each query sees; it is the whole mask, so `causal` has no say beside it and `segments` may not be given (cap and
    slopes go with either). A query that sees nothing gets zeros and no gradient. `validate_segments` checks the
    contract of `spans` too, at one host sync a mask.
    The kernel impl takes a softcap in [1e-3, 1e3], with any of the three a scale above 0, and slopes of either sign. A
    row's biases count from the highest of the keys that it sees, so that rows of any length keep their digits; in bf16 a
    slope costs some 8e-6 * |slope| of a probability, 0.4% at 500 (`impl="reference"` forms biases in fp32 as they are:
    N * |slope| * 2^-24). As in a plain product, what the mask hides must be finite, padding too (V; in the backward Q,
    K and dO): 0 is what it is multiplied by. These calls differentiate once."""
    resolved = resolve_attention_impl(q, k, v, impl=impl, causal=causal, segments=segments,
                                      validate_segments=validate_segments, softcap=softcap, slopes=slopes, spans=spans)
    scored = softcap is not None or slopes is not None or spans is not None
    if scored and resolved == "kernel":
        return _scored_attention(q, k, v, scale=scale, causal=causal, segments=segments, softcap=softcap, slopes=slopes,
                                 spans=spans)
    seg_id, seg_start = (None, None) if segments is None else _seg_args(q, segments.seg_id, segments.seg_start)
    if resolved == "kernel":
        args = (q.contiguous(), k.contiguous(), v.contiguous(), seg_id, seg_start, float(scale), bool(causal))
        nodes = _native.nodes() if _native.plain(q, k, v) else None
        if nodes is not None:
            return nodes.attention(*args)
        o, _ = _KernelAttention.apply(*args)
        return o
    if spans is not None:
        spans = SpanMask(start=spans.start.to(q.device), end=spans.end.to(q.device))
    score = {"softcap": softcap, "slopes": slopes, "spans": spans} if scored else None
    o, _ = _ReferenceAttention.apply(q, k, v, seg_id, seg_start, float(scale), causal, score)
    return o
