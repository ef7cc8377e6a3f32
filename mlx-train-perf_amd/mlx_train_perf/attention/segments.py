"""Segment description of a packed batch (the reference's `PackedMask`,
src/mlx_train_perf/attention/segments.py:9-29), plus the checks of its layout contract; and `SpanMask`, which
gives every query a range of keys (prompts as prefixes, whole documents, windows), with its builders."""
from __future__ import annotations

from dataclasses import dataclass, field

import torch


@dataclass(frozen=True)
class PackedMask:
    """Which documents share one packed row, as two int32 (B, L) tensors.

    seg_id: the document number of each position. Numbers start at 0 in every row and go up by
      one at each document boundary; padding at the end of a row is one more document, so every
      position has a number.
    seg_start: the index of the first position of the document each position belongs to; it never
      decreases along a row.
    """
    seg_id: torch.Tensor
    seg_start: torch.Tensor


def segment_allowed(seg_id: torch.Tensor) -> torch.Tensor:
    """Visibility as a (B, 1, N, N) bool tensor: query i may attend key j when both positions carry
    the same document number and j does not come after i."""
    same = seg_id[:, None, :, None] == seg_id[:, None, None, :]
    n = seg_id.shape[-1]
    causal = torch.tril(torch.ones(n, n, dtype=torch.bool, device=seg_id.device))[None, None]
    return same & causal


def layout_violation(seg_id: torch.Tensor, seg_start: torch.Tensor) -> str | None:
    """None when (seg_id, seg_start) follows the packed-row contract, else what is wrong.

    The contract, per row: seg_id starts at 0 and each step along the row adds 0 or 1 to it; a
    position starts a document exactly where seg_id steps up (or at 0); seg_start[i] is that start
    for every position i. The kernels mask with seg_start ranges, so a layout off the contract would
    be masked differently from seg_id equality -- hence the check. One device pass, one host sync."""
    sid = seg_id.to(torch.int64)
    sst = seg_start.to(torch.int64)
    n = sid.shape[-1]
    pos = torch.arange(n, device=sid.device).expand_as(sid)
    step = torch.diff(sid, dim=-1)
    new_doc = torch.ones_like(sid, dtype=torch.bool)
    new_doc[:, 1:] = step == 1
    # the start of each position's document: the last index <= i where a document begins
    starts = torch.cummax(torch.where(new_doc, pos, torch.zeros_like(pos)), dim=-1).values
    checks = torch.stack([
        (sid[:, 0] != 0).any(),
        ((step != 0) & (step != 1)).any(),
        (sst != starts).any(),
    ]).cpu()
    if checks[0]:
        return "seg_id must start at 0 in every row"
    if checks[1]:
        return "seg_id must be contiguous and ascending (each step along a row adds 0 or 1)"
    if checks[2]:
        return "seg_start must hold the first position of each position's segment (as implied by seg_id)"
    return None


@dataclass(frozen=True)
class SpanMask:
    """The keys that each query sees, as two integer (B, N) tensors: query i sees the keys j with
    start[b, i] <= j < end[b, i], whether they come before it or after.

    Neither tensor may decrease along a row, and both lie in [0, N]. A query whose range holds nothing (padding)
    gets an output of zeros and takes part in no gradient. A window of w keys is start = max(0, i - w + 1), end = i + 1.

    A mask remembers that its contract was checked (a host sync), for as long as neither tensor is written to, so that
    a model's layers check the mask of a step once (tensors made in inference mode do not tell of writes: checked each time).
    """
    start: torch.Tensor
    end: torch.Tensor
    _checked: list = field(default_factory=list, init=False, repr=False, compare=False)

    def violation(self) -> str | None:
        """`span_violation` of this mask, unless it was found to be none before."""
        start, end = self.start, self.end
        if start.is_inference() or end.is_inference():
            return span_violation(self)
        versions = [start._version, end._version]
        if self._checked == versions:
            return None
        problem = span_violation(self)
        if problem is None:
            self._checked[:] = versions
        return problem


def _lengths(values: torch.Tensor | list[int], device: torch.device | None) -> torch.Tensor:
    return torch.as_tensor(values, device=device).to(torch.int64)


def prefix_spans(prefix: torch.Tensor | list[int], n: int) -> SpanMask:
    """Rows of n positions whose first prefix[b] ones (a prompt) see each other whole, and whose others see
    everything up to themselves. `prefix`: (B,) integers in [0, n], on the device that the spans shall be on."""
    p = _lengths(prefix, None)
    i = torch.arange(n, device=p.device)
    end = torch.maximum(i + 1, p[:, None])
    return SpanMask(start=torch.zeros_like(end, dtype=torch.int32), end=end.to(torch.int32))


def document_spans(segments: PackedMask, *, prefix: torch.Tensor | None = None, causal: bool = True,
                   used: torch.Tensor | list[int] | None = None) -> SpanMask:
    """The documents of a packed row, each seeing itself alone.

    `prefix`: (B, N) integers, at every position the length of its document's prompt: the prompt's positions
    see each other whole, the rest of the document everything up to themselves. `causal=False`: every position
    sees its whole document. `used`: (B,) integers, the positions of each row that hold documents: those behind
    see nothing and are seen by nothing (without it padding is one more document, as in `PackedMask`)."""
    seg_start = segments.seg_start.to(torch.int64)
    n = seg_start.shape[-1]
    i = torch.arange(n, device=seg_start.device).expand_as(seg_start)
    if causal:
        end = i + 1 if prefix is None else torch.maximum(i + 1, seg_start + prefix.to(seg_start))
    else:
        end = torch.full_like(seg_start, n)
    # no further than the document: the next position that starts one
    seg_id = segments.seg_id.to(torch.int64).contiguous()
    doc_end = torch.searchsorted(seg_id, seg_id, right=True)
    start, end = seg_start, torch.minimum(end, doc_end)
    if used is not None:
        u = _lengths(used, seg_start.device)[:, None]
        start, end = torch.where(i < u, start, u), torch.where(i < u, torch.minimum(end, u), u)
    return SpanMask(start=start.to(torch.int32), end=end.to(torch.int32))


def packed_as_spans(segments: PackedMask) -> SpanMask:
    """The packed mask (same document, not after) as spans."""
    start = segments.seg_start
    end = torch.arange(1, start.shape[-1] + 1, dtype=torch.int32, device=start.device).expand(start.shape)
    return SpanMask(start=start, end=end)


def span_allowed(spans: SpanMask) -> torch.Tensor:
    """Visibility as a (B, 1, N, N) bool tensor."""
    j = torch.arange(spans.start.shape[-1], device=spans.start.device)
    return ((j >= spans.start[..., None]) & (j < spans.end[..., None]))[:, None]


def span_violation(spans: SpanMask) -> str | None:
    """None when the spans follow their contract, else what is wrong. One device pass, one host sync."""
    n = spans.start.shape[-1]
    checks = torch.stack([t for x in (spans.start, spans.end) for t in (
        ((x < 0) | (x > n)).any(), (torch.diff(x.to(torch.int64), dim=-1) < 0).any())]).cpu()
    for name, outside, down in (("start", checks[0], checks[1]), ("end", checks[2], checks[3])):
        if outside:
            return f"{name} must lie in [0, {n}]"
        if down:
            return f"{name} must not decrease along a row"
    return None
