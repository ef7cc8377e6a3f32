"""Materialized attention, `impl="reference"` (mirror of src/mlx_train_perf/attention/reference.py).

`math_attention` builds the full (N, N) scores in fp32, softmaxes and multiplies into V; autograd
differentiates through it. `flash_attention_reference` returns (O, L) with L the fp32 row
logsumexp (+inf where spans leave a query nothing to see). GQA: query head h reads kv head h // (Hq // Hkv). An explicit opt-in for small N only;
never chosen by `impl="auto"`.
"""
from __future__ import annotations

import torch

from mlx_train_perf.attention.segments import PackedMask, SpanMask, segment_allowed, span_allowed


def kv_head_for(q_head: int, group_size: int) -> int:
    """Contiguous GQA grouping (reference.py:37-39)."""
    return q_head // group_size


def distances(n: int, device: torch.device) -> torch.Tensor:
    """|i - j| as an (n, n) fp32 tensor."""
    i = torch.arange(n, device=device)
    return (i[:, None] - i[None, :]).abs().to(torch.float32)


def scores_of(x: torch.Tensor, *, softcap: float | None, slopes: torch.Tensor | None):
    """(scores, 1 - tanh^2 or None) of scaled products x (B, Hq, N, N): capped, then biased by distance."""
    bend = None
    if softcap is not None:
        t = torch.tanh(x / softcap)
        x, bend = softcap * t, 1.0 - t * t
    if slopes is not None:
        x = x - slopes.to(torch.float32)[:, None, None] * distances(x.shape[-1], x.device)
    return x, bend


def hide(scores: torch.Tensor, *, causal: bool, segments: PackedMask | None, spans: SpanMask | None) -> torch.Tensor:
    """The scores with -inf where the mask hides a key (spans are the whole mask)."""
    if spans is not None:
        return scores.masked_fill(~span_allowed(spans), float("-inf"))
    if segments is not None:
        assert causal, "segments requires causal=True"
        return scores.masked_fill(~segment_allowed(segments.seg_id), float("-inf"))
    if causal:
        n = scores.shape[-1]
        tri = torch.ones(n, n, dtype=torch.bool, device=scores.device).triu(1)
        scores = scores.masked_fill(tri, float("-inf"))
    return scores


def _masked_scaled_scores(q, k, v, *, scale, causal, segments=None, softcap=None, slopes=None, spans=None):
    hq, hkv = q.shape[1], k.shape[1]
    if hq % hkv != 0:
        raise ValueError(f"Hq={hq} must be a multiple of Hkv={hkv} for GQA grouping")
    group = hq // hkv
    idx = torch.tensor([kv_head_for(h, group) for h in range(hq)], device=q.device)
    q32 = q.to(torch.float32)
    k_g = k.index_select(1, idx).to(torch.float32)
    v_g = v.index_select(1, idx).to(torch.float32)
    scores = (q32 @ k_g.transpose(-1, -2).contiguous()) * scale
    scores, _ = scores_of(scores, softcap=softcap, slopes=slopes)
    return hide(scores, causal=causal, segments=segments, spans=spans), v_g


def _attention_core(q, k, v, *, scale, causal, segments=None, softcap=None, slopes=None, spans=None):
    scores, v_g = _masked_scaled_scores(q, k, v, scale=scale, causal=causal, segments=segments, softcap=softcap,
                                        slopes=slopes, spans=spans)
    if spans is not None:   # a query may see nothing: probabilities 0, no NaN in the gradients
        empty = (spans.end <= spans.start)[:, None, :, None]
        scores = scores.masked_fill(empty, 0.0)
        lse = torch.logsumexp(scores, dim=-1).masked_fill(empty[..., 0], float("inf"))
    else:
        lse = torch.logsumexp(scores, dim=-1)
    probs = torch.exp(scores - lse[..., None])
    o = (probs @ v_g).to(q.dtype)
    return o, lse


def math_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float, causal: bool = True,
                   segments: PackedMask | None = None, softcap: float | None = None,
                   slopes: torch.Tensor | None = None, spans: SpanMask | None = None) -> torch.Tensor:
    o, _ = _attention_core(q, k, v, scale=scale, causal=causal, segments=segments, softcap=softcap, slopes=slopes,
                           spans=spans)
    return o


def flash_attention_reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float,
                              causal: bool = True, segments: PackedMask | None = None, softcap: float | None = None,
                              slopes: torch.Tensor | None = None, spans: SpanMask | None = None):
    return _attention_core(q, k, v, scale=scale, causal=causal, segments=segments, softcap=softcap, slopes=slopes,
                           spans=spans)
