"""Trainer adapter for torch causal LMs: `split_model`, `make_loss_fn`, `make_packed_loss_fn`
(the torch counterpart of src/mlx_train_perf/adapters/mlx_lm.py:140-297), and beyond the reference
`make_token_nll_fn`, `make_preference_loss_fn` and `make_policy_loss_fn` for steps on preferences and rewards,
`make_token_logprobs_fn` and `make_distillation_loss_fn` for scoring tokens and for learning from a teacher's scores.

Loss contract (the mlx-lm trainer's `default_loss`, quoted at adapters/mlx_lm.py:5-20):
inputs = batch[:, :-1], targets = batch[:, 1:], steps = 1..T, mask = (steps >= lengths[:, 0]) &
(steps <= lengths[:, 1]), loss = (nll * mask).sum() / ntoks, returning (loss, ntoks).
The fused loss replaces the `(B, T, V)` logits: the model's trunk produces hidden states and
`linear_cross_entropy(..., reduction="none")` the per-token NLL. This contract is only available
as documented text (mlx-lm is not installed), so its numerics are checked against a plain torch
restatement of that formula, not against mlx-lm itself.

Supported models: Hugging Face transformers causal LMs with `.model` (trunk returning
`last_hidden_state`) and `.lm_head` (`nn.Linear`), or tied word embeddings
(`config.tie_word_embeddings`). The head and its `trainable` flag are re-read from the live model
on every call (adapters/mlx_lm.py:22-33: a construction-time snapshot would go stale).
"""
from __future__ import annotations

from collections.abc import Callable
from typing import Any, Literal

import torch
from torch import nn

from mlx_train_perf.attention.segments import PackedMask, SpanMask
from mlx_train_perf.core.loss import DenseHead, HeadRef, linear_cross_entropy, resolve_impl, tied_head
from mlx_train_perf.core.preference import PolicyLoss, PreferenceLoss, policy_loss, preference_loss
from mlx_train_perf.core.scoring import TokenLogprobs, distillation_loss, token_logprobs
from mlx_train_perf.errors import AdapterError

_Impl = Literal["auto", "kernel", "chunked", "naive"]


def _head_from_linear(module: nn.Module) -> DenseHead:
    if not isinstance(module, nn.Linear):
        raise AdapterError(f"unsupported head module type {type(module).__name__!r}; expected nn.Linear")
    if module.bias is not None:
        raise AdapterError("lm_head with a bias is not supported by the fused loss")
    return DenseHead(weight=module.weight, trainable=module.weight.requires_grad)


def split_model(model: Any) -> tuple[Callable[..., torch.Tensor], HeadRef]:
    """(trunk, head): trunk(input_ids, **kw) -> hidden (B, T, D); head from lm_head or tied embeddings."""
    inner = getattr(model, "model", None)
    if inner is None or not hasattr(inner, "layers"):
        raise AdapterError(f"unsupported model architecture {type(model).__name__!r}: expected `.model.layers`")

    def trunk(x: torch.Tensor, **kw: Any) -> torch.Tensor:
        out = inner(input_ids=x, **kw)
        return out.last_hidden_state if hasattr(out, "last_hidden_state") else out

    cfg = getattr(model, "config", None)
    if cfg is not None and getattr(cfg, "tie_word_embeddings", False):
        emb = inner.embed_tokens
        return trunk, tied_head(emb.weight, trainable=emb.weight.requires_grad)
    head = getattr(model, "lm_head", None)
    if head is None:
        raise AdapterError("model has neither an lm_head nor tied word embeddings")
    return trunk, _head_from_linear(head)


def make_loss_fn(model: Any, *, impl: _Impl = "auto",
                 allow_unverified_mlx: bool = False) -> Callable[[Any, torch.Tensor, torch.Tensor], tuple[torch.Tensor, torch.Tensor]]:
    """`loss(model, batch, lengths) -> (loss, ntoks)` with the mlx-lm trainer's mask and
    normalization (adapters/mlx_lm.py:167-218). `lengths` is (B, 2) int: (offset, length)."""
    split_model(model)  # fail fast; re-derived per call
    resolved: dict[str, str] = {}

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        trunk, head = split_model(model_arg)
        inputs, targets = batch[:, :-1], batch[:, 1:]
        hidden = trunk(inputs)
        if "impl" not in resolved:
            n = hidden.shape[0] * hidden.shape[1]
            resolved["impl"] = resolve_impl(head=head, dtype=hidden.dtype, n=n, impl=impl,
                                            allow_unverified_mlx=allow_unverified_mlx).impl
        nll = linear_cross_entropy(hidden, head, targets, impl=resolved["impl"], reduction="none",
                                   validate_targets=False)
        steps = torch.arange(1, targets.shape[1] + 1, device=targets.device)
        mask = (steps >= lengths[:, 0:1]) & (steps <= lengths[:, 1:])
        ntoks = mask.sum()
        loss = (nll * mask).to(torch.float32).sum() / ntoks
        return loss, ntoks

    return loss_fn


def make_packed_loss_fn(model: Any, *, impl: _Impl = "auto", allow_unverified_mlx: bool = False):
    """`loss(model, batch, seg_id, seg_start, loss_mask) -> (loss, ntoks)` for packed rows
    (adapters/mlx_lm.py:221-297): the PackedMask is threaded to every attention call, the loss is
    normalized by `loss_mask`. Requires `enable_flash_attention(model)` first (AdapterError)."""
    from mlx_train_perf.attention.wrapper import is_enabled  # noqa: PLC0415

    split_model(model)
    if not is_enabled(model):
        raise AdapterError("make_packed_loss_fn requires enable_flash_attention(model) first")
    resolved: dict[str, str] = {}

    def loss_fn(model_arg: Any, batch: torch.Tensor, seg_id: torch.Tensor, seg_start: torch.Tensor,
                loss_mask: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        trunk, head = split_model(model_arg)
        inputs, targets = batch[:, :-1], batch[:, 1:]
        pm = PackedMask(seg_id=seg_id, seg_start=seg_start)
        hidden = trunk(inputs, mtp_segments=pm)
        if "impl" not in resolved:
            n = hidden.shape[0] * hidden.shape[1]
            resolved["impl"] = resolve_impl(head=head, dtype=hidden.dtype, n=n, impl=impl,
                                            allow_unverified_mlx=allow_unverified_mlx).impl
        nll = linear_cross_entropy(hidden, head, targets, impl=resolved["impl"], reduction="none",
                                   validate_targets=False)
        ntoks = loss_mask.sum()
        loss = (nll * loss_mask).to(torch.float32).sum() / ntoks
        return loss, ntoks

    return loss_fn


def _refuse_capped_logits(model: Any) -> None:
    cfg = getattr(model, "config", None)
    if getattr(cfg, "final_logit_softcapping", None):   # (0, like None: no cap)
        raise AdapterError("the fused loss does not cap logits (config.final_logit_softcapping is set)")


def _hidden_and_head(model: Any, batch: torch.Tensor, spans: SpanMask | None) -> tuple[torch.Tensor, HeadRef]:
    """The hidden states of the inputs batch[:, :-1] and the head."""
    from mlx_train_perf.attention.wrapper import is_enabled  # noqa: PLC0415

    trunk, head = split_model(model)
    if spans is not None and not is_enabled(model):
        raise AdapterError("spans require enable_flash_attention(model) first")
    return trunk(batch[:, :-1], **({} if spans is None else {"mtp_spans": spans})), head


def make_token_nll_fn(model: Any, *, impl: _Impl = "auto",
                      allow_unverified_mlx: bool = False) -> Callable[..., torch.Tensor]:
    """`nll(model, batch, spans=None) -> (B, T)`, the per-token losses of the targets batch[:, 1:]: what the losses
    below take from frozen models (call it under `torch.no_grad()` for those). `spans`: a `SpanMask` over the inputs
    batch[:, :-1], handed to every attention call; requires `enable_flash_attention(model)`."""
    split_model(model)
    _refuse_capped_logits(model)

    def nll_fn(model_arg: Any, batch: torch.Tensor, spans: SpanMask | None = None) -> torch.Tensor:
        hidden, head = _hidden_and_head(model_arg, batch, spans)
        return linear_cross_entropy(hidden, head, batch[:, 1:], impl=impl, reduction="none", validate_targets=False,
                                    allow_unverified_mlx=allow_unverified_mlx).to(torch.float32)

    return nll_fn


def _target_mask(lengths: torch.Tensor, t: int) -> torch.Tensor:
    """The trainer's mask of `make_loss_fn`: targets at steps offset .. length of each row."""
    steps = torch.arange(1, t + 1, device=lengths.device)
    return (steps >= lengths[:, 0:1]) & (steps <= lengths[:, 1:])


def _row_loss_impl(impl: str) -> Literal["auto", "reference"]:
    return "reference" if impl in ("naive", "chunked") else "auto"


def make_preference_loss_fn(model: Any, *, beta: float = 0.1, kind: Literal["sigmoid", "hinge", "ipo"] = "sigmoid",
                            label_smoothing: float = 0.0, impl: _Impl = "auto",
                            allow_unverified_mlx: bool = False) -> Callable[..., PreferenceLoss]:
    """`loss(model, batch, lengths, ref_nll, spans=None) -> PreferenceLoss`: `batch` (2P, T + 1) holds the P chosen
    answers, then the P rejected ones; `lengths` (2P, 2) as in `make_loss_fn` (the answer's first and last step);
    `ref_nll` (2P, T) is the reference model's `make_token_nll_fn` of the same batch."""
    nll_fn = make_token_nll_fn(model, impl=impl, allow_unverified_mlx=allow_unverified_mlx)

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor, ref_nll: torch.Tensor,
                spans: SpanMask | None = None) -> PreferenceLoss:
        nll = nll_fn(model_arg, batch, spans)
        return preference_loss(nll, ref_nll, mask=_target_mask(lengths, nll.shape[1]), beta=beta, kind=kind,
                               label_smoothing=label_smoothing, impl=_row_loss_impl(impl))

    return loss_fn


def make_policy_loss_fn(model: Any, *, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                        reduction: Literal["token", "sequence"] = "token", impl: _Impl = "auto",
                        allow_unverified_mlx: bool = False) -> Callable[..., PolicyLoss]:
    """`loss(model, batch, lengths, old_nll, advantages, ref_nll=None, spans=None) -> PolicyLoss`: `old_nll` (B, T) is
    the sampling model's `make_token_nll_fn` of the batch, `advantages` (B,) or (B, T), `lengths` as in
    `make_loss_fn`."""
    nll_fn = make_token_nll_fn(model, impl=impl, allow_unverified_mlx=allow_unverified_mlx)

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor, old_nll: torch.Tensor, advantages: torch.Tensor,
                ref_nll: torch.Tensor | None = None, spans: SpanMask | None = None) -> PolicyLoss:
        nll = nll_fn(model_arg, batch, spans)
        return policy_loss(nll, old_nll, advantages, ref_nll=ref_nll, mask=_target_mask(lengths, nll.shape[1]),
                           clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, reduction=reduction,
                           impl=_row_loss_impl(impl))

    return loss_fn


def make_token_logprobs_fn(model: Any, *, top: int = 0, temperature: float = 1.0, impl: _Impl = "auto",
                           allow_unverified_mlx: bool = False) -> Callable[..., TokenLogprobs]:
    """`score(model, batch, lengths=None, spans=None) -> TokenLogprobs` of the targets batch[:, 1:], (B, T) each, with the `top`
    alternatives of every position (a teacher's lists for `make_distillation_loss_fn`: call it under `torch.no_grad()`).
    `lengths` (B, 2) as in `make_loss_fn` leaves the positions outside out. `spans` as in `make_token_nll_fn`."""
    split_model(model)
    _refuse_capped_logits(model)

    def score_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor | None = None,
                 spans: SpanMask | None = None) -> TokenLogprobs:
        hidden, head = _hidden_and_head(model_arg, batch, spans)
        targets = batch[:, 1:]
        if lengths is not None:
            targets = targets.masked_fill(~_target_mask(lengths, targets.shape[1]), -100)
        return token_logprobs(hidden, head, targets, top=top, temperature=temperature, impl=_row_loss_impl(impl),
                              allow_unverified_mlx=allow_unverified_mlx, validate_targets=False)

    return score_fn


def make_distillation_loss_fn(model: Any, *, kind: Literal["forward", "reverse", "jsd"] = "forward", beta: float = 0.5,
                              temperature: float = 1.0, renormalize: bool = False, impl: _Impl = "auto",
                              allow_unverified_mlx: bool = False) -> Callable[..., torch.Tensor]:
    """`loss(model, batch, lengths, teacher_ids, teacher_logprobs, spans=None) -> loss`: `distillation_loss` over the positions
    of the targets batch[:, 1:] that `lengths` (as in `make_loss_fn`) takes in; the teacher's lists (B, T, K) are its
    `make_token_logprobs_fn(..., top=K)` of the same batch."""
    split_model(model)
    _refuse_capped_logits(model)

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor, teacher_ids: torch.Tensor,
                teacher_logprobs: torch.Tensor, spans: SpanMask | None = None) -> torch.Tensor:
        hidden, head = _hidden_and_head(model_arg, batch, spans)
        return distillation_loss(hidden, head, teacher_ids, teacher_logprobs, mask=_target_mask(lengths, batch.shape[1] - 1),
                                 kind=kind, beta=beta, temperature=temperature, renormalize=renormalize,
                                 impl=_row_loss_impl(impl), allow_unverified_mlx=allow_unverified_mlx, validate_ids=False)

    return loss_fn
