"""Preference and policy losses over the per-token losses of `linear_cross_entropy(..., reduction="none")`.

Both take `nll`, the model's per-token losses (-log pi), and those of frozen models, as one of:
- a batch (sequences, T), one sequence a row;
- a flat run (N,) with `offsets`, (sequences + 1,) integers: sequence r is the tokens [offsets[r], offsets[r + 1]).
  Tokens of no sequence count nowhere.
`mask` (nll's shape, bool or uint8) says which tokens count: prompts and padding do not, whatever the tensors hold
there. (An ignored token's nll is 0 under every model, so a preference loss without ratios by length needs no mask.)

The gradient goes to `nll` alone; a frozen model's losses that ask for one are refused.
- `impl="kernel"` (and "auto"): HIP kernels, fp32 tensors on a gfx950 GPU, sums in 64 bits in a fixed order.
- `impl="reference"`: torch operators in 64 bits, any device and floating type.
"""
from __future__ import annotations

import math
from typing import Literal, NamedTuple

import torch
from torch.autograd.function import once_differentiable

from mlx_train_perf import _compat, _native
from mlx_train_perf.errors import LossInputError, UnsupportedHeadError

_KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2, "token": 1, "sequence": 3}


class PreferenceLoss(NamedTuple):
    """`chosen_rewards` and `rejected_rewards` are beta times the log ratios, (pairs,), without a gradient."""
    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


class PolicyLoss(NamedTuple):
    """`kl`: the mean of e^d - d - 1, d = nll - ref_nll, over the tokens that count (0 without ref_nll);
    `clip_fraction`: the share of them whose ratio was clipped. Both without a gradient."""
    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


def _number(name: str, x: float, ok: bool, what: str) -> float:
    if not (math.isfinite(x) and ok):
        raise LossInputError(f"{name} must be {what}; got {x!r}")
    return float(x)


def _sequences(nll: torch.Tensor, frozen: dict[str, torch.Tensor | None], offsets: torch.Tensor | None,
               mask: torch.Tensor | None, validate_offsets: bool) -> int:
    """The number of sequences, after the checks that both losses share."""
    shape = nll.shape
    if not nll.dtype.is_floating_point:
        raise LossInputError(f"nll must be floating-point; got {nll.dtype}")
    if nll.numel() < 1:
        raise LossInputError(f"nll must hold at least one token; got shape {tuple(shape)}")
    for name, t in frozen.items():
        if t is None:
            continue
        if t.shape != shape:
            raise LossInputError(f"{name} must have nll's shape {tuple(shape)}; got {tuple(t.shape)}")
        if not t.dtype.is_floating_point:
            raise LossInputError(f"{name} must be floating-point; got {t.dtype}")
        if t.requires_grad and torch.is_grad_enabled():
            raise LossInputError(f"{name} belongs to a frozen model and gets no gradient: detach it")
    if mask is not None and (mask.shape != shape or mask.dtype not in (torch.bool, torch.uint8)):
        raise LossInputError(f"mask must be bool or uint8 of nll's shape {tuple(shape)}; got {mask.dtype} {tuple(mask.shape)}")
    if offsets is None:
        if len(shape) != 2:
            raise LossInputError(f"nll must be (sequences, T), or (N,) with offsets; got shape {tuple(shape)}")
        return shape[0]
    if nll.dim() != 1:
        raise LossInputError(f"with offsets nll must be (N,); got shape {tuple(nll.shape)}")
    if offsets.dim() != 1 or offsets.numel() < 2 or offsets.dtype not in (torch.int32, torch.int64):
        raise LossInputError(f"offsets must be (sequences + 1,) int32 or int64; got {offsets.dtype} {tuple(offsets.shape)}")
    if validate_offsets:   # a host sync
        if bool(((offsets < 0) | (offsets > nll.numel())).any()) or bool((torch.diff(offsets) < 0).any()):
            raise LossInputError(f"offsets must lie in [0, N={nll.numel()}] and never decrease")
    return offsets.numel() - 1


def _resolve(nll: torch.Tensor, others: dict[str, torch.Tensor | None], impl: str) -> str:
    if impl == "reference":
        return impl
    if impl not in ("auto", "kernel"):
        raise LossInputError(f"unknown impl {impl!r}; expected one of 'auto', 'kernel', 'reference'")
    others = {name: t for name, t in others.items() if t is not None}
    for name, t in {"nll": nll, **others}.items():
        dtype = t.dtype
        if dtype is not torch.float32 and dtype.is_floating_point:
            raise UnsupportedHeadError(f"kernel impl reads fp32 tensors (got {name} of {dtype}); use impl='reference'.")
    _compat.check_device_verified(allow_unverified=False, error=UnsupportedHeadError)
    _compat.require_gpu_tensor(nll, error=UnsupportedHeadError)
    device = nll.device
    for name, t in others.items():
        if t.device != device:
            raise LossInputError(f"{name} is on {t.device} but nll is on {device}; the kernel impl needs every "
                                 "input on the same GPU")
    return "kernel"


def _frozen(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else (t.detach() if t.requires_grad else t).contiguous()


def _plain_mask(mask: torch.Tensor | None) -> torch.Tensor | None:
    return None if mask is None else mask.contiguous()   # bool or uint8: bytes either way


def _plain_offsets(offsets: torch.Tensor | None) -> torch.Tensor | None:
    return None if offsets is None else offsets.to(torch.int64).contiguous()


class _Preference(torch.autograd.Function):
    """(loss, rewards) from mtp_pref_fwd; the backward spreads each sequence's factor over its tokens. The general path:
    plain tensors take the C++ node of the same calls."""

    @staticmethod
    def forward(ctx, nll, ref_nll, mask, offsets, pairs, kind, beta, smoothing, reduction):
        lib = _native.load()
        n, dev = nll.numel(), nll.device
        loss = torch.empty((pairs,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        rewards = torch.empty(2 * pairs, dtype=torch.float32, device=dev)
        coef = torch.empty_like(rewards)
        ws_bytes = lib.mtp_pref_workspace_bytes(pairs, n)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with _native.on_device(nll):
            rc = lib.mtp_pref_fwd(nll.data_ptr(), ref_nll.data_ptr(), _native.ptr(mask), _native.ptr(offsets), pairs, n, kind,
                                  beta, smoothing, reduction, loss.data_ptr(), rewards.data_ptr(), coef.data_ptr(),
                                  ws.data_ptr(), ws_bytes, _native.stream_of(nll))
        _native.check(rc, domain="loss")
        ctx.save_for_backward(coef, mask, offsets)
        ctx.shape, ctx.reduction = nll.shape, reduction
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        return loss, rewards

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss, _d_rewards):
        lib = _native.load()
        coef, mask, offsets = ctx.saved_tensors
        d_nll = torch.empty(ctx.shape, dtype=torch.float32, device=coef.device)
        if d_loss is None:
            return d_nll.zero_(), None, None, None, None, None, None, None, None
        ct = d_loss.to(torch.float32).contiguous()
        with _native.on_device(coef):
            rc = lib.mtp_pref_bwd(ct.data_ptr(), coef.data_ptr(), _native.ptr(mask), _native.ptr(offsets), coef.numel() // 2,
                                  d_nll.numel(), ctx.reduction, d_nll.data_ptr(), _native.stream_of(coef))
        _native.check(rc, domain="loss")
        return d_nll, None, None, None, None, None, None, None, None


class _Policy(torch.autograd.Function):
    """(loss, stats) from mtp_policy_fwd; the backward forms each token's gradient again from the inputs. The general
    path, as _Preference."""

    @staticmethod
    def forward(ctx, nll, old_nll, ref_nll, adv, mask, offsets, rows, clip_low, clip_high, kl_coef, reduction):
        lib = _native.load()
        n, dev = nll.numel(), nll.device
        loss = torch.empty(nll.shape if reduction == 0 else (), dtype=torch.float32, device=dev)
        stats = torch.empty(2, dtype=torch.float32, device=dev)
        weight = torch.empty(rows, dtype=torch.float32, device=dev)
        ws_bytes = lib.mtp_policy_workspace_bytes(rows, n)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        per_token = int(adv.shape == nll.shape)
        with _native.on_device(nll):
            rc = lib.mtp_policy_fwd(nll.data_ptr(), old_nll.data_ptr(), _native.ptr(ref_nll), adv.data_ptr(), per_token,
                                    _native.ptr(mask), _native.ptr(offsets), rows, n, clip_low, clip_high, kl_coef, reduction,
                                    loss.data_ptr(), stats.data_ptr(), weight.data_ptr(), ws.data_ptr(), ws_bytes,
                                    _native.stream_of(nll))
        _native.check(rc, domain="loss")
        ctx.save_for_backward(nll, old_nll, ref_nll, adv, mask, offsets, weight)
        ctx.args = (clip_low, clip_high, kl_coef, reduction)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss, _d_stats):
        lib = _native.load()
        nll, old_nll, ref_nll, adv, mask, offsets, weight = ctx.saved_tensors
        d_nll = torch.empty_like(nll)
        nothing = (None,) * 10
        if d_loss is None:
            return (d_nll.zero_(), *nothing)
        ct = d_loss.to(torch.float32).contiguous()
        with _native.on_device(nll):
            rc = lib.mtp_policy_bwd(ct.data_ptr(), nll.data_ptr(), old_nll.data_ptr(), _native.ptr(ref_nll), adv.data_ptr(),
                                    int(adv.shape == nll.shape), _native.ptr(mask), _native.ptr(offsets), weight.numel(),
                                    nll.numel(), *ctx.args, weight.data_ptr(), d_nll.data_ptr(), _native.stream_of(nll))
        _native.check(rc, domain="loss")
        return (d_nll, *nothing)


# ---- the reference impl -------------------------------------------------------------------------------------------

def _owners(nll: torch.Tensor, offsets: torch.Tensor | None, rows: int) -> torch.Tensor:
    """The sequence of every token of the flat nll; `rows` for tokens of none."""
    n = nll.numel()
    at = torch.arange(n, device=nll.device)
    if offsets is None:
        return at // (n // rows)
    o = offsets.to(device=nll.device, dtype=torch.int64)
    row = torch.searchsorted(o, at, right=True) - 1
    return torch.where((row < 0) | (row >= rows), rows, row)


def _row_sums(values: torch.Tensor, owner: torch.Tensor, rows: int) -> torch.Tensor:
    return torch.zeros(rows + 1, dtype=torch.float64, device=values.device).index_add(0, owner, values.double())[:rows]


def _counted(nll: torch.Tensor, owner: torch.Tensor, mask: torch.Tensor | None, rows: int) -> torch.Tensor:
    keep = owner < rows
    return keep if mask is None else keep & (mask.reshape(-1) != 0)


def _out(x: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return x if like.dtype == torch.float64 else x.to(torch.float32)


def _reference_preference(nll, ref_nll, offsets, mask, rows, kind, beta, smoothing, reduction):
    flat = nll.reshape(-1)
    owner = _owners(flat, offsets, rows)
    keep = _counted(flat, owner, mask, rows)
    gap = torch.where(keep, ref_nll.reshape(-1).double() - flat.double(), 0.0)
    ratio = _row_sums(gap, owner, rows)
    if kind == "ipo":
        ratio = ratio / _row_sums(keep, owner, rows).clamp(min=1)
    chosen, rejected = (beta * ratio).reshape(2, -1)
    d = chosen - rejected
    if kind == "sigmoid":
        loss = (1 - smoothing) * torch.nn.functional.softplus(-d)
        if smoothing:   # 0 of an infinite one is 0
            loss = loss + smoothing * torch.nn.functional.softplus(d)
    elif kind == "hinge":
        loss = torch.relu(1 - d)
    else:
        loss = (d / beta - 0.5 / beta) ** 2
    loss = {"none": loss, "mean": loss.mean(), "sum": loss.sum()}[reduction]
    return PreferenceLoss(_out(loss, nll), _out(chosen.detach(), nll), _out(rejected.detach(), nll))


def _reference_policy(nll, old_nll, ref_nll, adv, offsets, mask, rows, clip_low, clip_high, kl_coef, reduction):
    flat = nll.reshape(-1)
    owner = _owners(flat, offsets, rows)
    keep = _counted(flat, owner, mask, rows)

    def at(t):   # the values that count, 0 elsewhere
        return torch.where(keep, t.reshape(-1).double(), 0.0)

    x = at(flat)
    a = at(adv) if adv.shape == nll.shape else torch.where(keep, adv.double()[owner.clamp(max=rows - 1)], 0.0)
    step = at(old_nll) - x
    clipped = torch.where(a > 0, step > math.log1p(clip_high),
                          step < (math.log1p(-clip_low) if clip_low < 1 else -math.inf)) & (a != 0)
    edge = torch.where(a > 0, torch.full_like(a, 1 + clip_high), 1 - clip_low)
    flat = clipped | (a == 0)   # nothing is left of the ratio, also of an infinite one
    loss = -torch.where(flat, edge, torch.exp(torch.where(flat, 0.0, step))) * a
    kl = torch.zeros_like(loss)
    if ref_nll is not None:
        gap = x - at(ref_nll)
        kl = torch.expm1(gap) - gap
        if kl_coef:
            loss = loss + kl_coef * kl
    loss = torch.where(keep, loss, 0.0)
    count = keep.sum().clamp(min=1)
    if reduction == "token":
        total = loss.sum() / count
    elif reduction == "sequence":
        per_row = _row_sums(keep, owner, rows)
        means = _row_sums(loss, owner, rows) / per_row.clamp(min=1)
        total = means.sum() / (per_row > 0).sum().clamp(min=1)
    else:
        total = loss.reshape(nll.shape)
    return PolicyLoss(_out(total, nll), _out(kl.detach().sum() / count, nll), _out((clipped & keep).sum() / count.double(), nll))


# ---- public -------------------------------------------------------------------------------------------------------

def preference_loss(nll: torch.Tensor, ref_nll: torch.Tensor, *, offsets: torch.Tensor | None = None,
                    mask: torch.Tensor | None = None, beta: float = 0.1,
                    kind: Literal["sigmoid", "hinge", "ipo"] = "sigmoid", label_smoothing: float = 0.0,
                    reduction: Literal["none", "mean", "sum"] = "mean",
                    impl: Literal["auto", "kernel", "reference"] = "auto", validate_offsets: bool = True) -> PreferenceLoss:
    """Preference loss of pairs of sequences: of 2P sequences, p is the chosen and P + p the rejected answer of pair p.

    With the log ratio of policy to reference g = sum over a sequence of (ref_nll - nll) (for "ipo" its mean), and
    d = beta (g_chosen - g_rejected):
      "sigmoid": -(1 - label_smoothing) log sigmoid(d) - label_smoothing log sigmoid(-d);
      "hinge": max(0, 1 - d);
      "ipo": (d / beta - 1 / (2 beta))^2.
    `reduction` is over the pairs. `validate_offsets` checks the offsets at one host sync; pass False on a trusted
    path (offsets are clamped into the tokens either way)."""
    if reduction not in ("none", "mean", "sum"):
        raise LossInputError(f"unknown reduction {reduction!r}; expected 'none', 'mean' or 'sum'")
    if kind not in _KINDS:
        raise LossInputError(f"unknown kind {kind!r}; expected one of {', '.join(map(repr, _KINDS))}")
    beta = _number("beta", beta, beta > 0, "positive and finite")
    label_smoothing = _number("label_smoothing", label_smoothing, 0 <= label_smoothing < 0.5, "in [0, 0.5)")
    if label_smoothing and kind != "sigmoid":
        raise LossInputError("label_smoothing belongs to kind='sigmoid'")
    rows = _sequences(nll, {"ref_nll": ref_nll}, offsets, mask, validate_offsets)
    if rows % 2:
        raise LossInputError(f"the sequences are pairs, the chosen half first; got {rows} of them")
    if _resolve(nll, {"ref_nll": ref_nll, "offsets": offsets, "mask": mask}, impl) == "reference":
        return _reference_preference(nll, ref_nll.detach(), offsets, mask, rows, kind, beta, label_smoothing, reduction)
    pairs = rows // 2
    args = (nll.contiguous(), _frozen(ref_nll), _plain_mask(mask), _plain_offsets(offsets), pairs, _KINDS[kind], beta,
            label_smoothing, _REDUCTIONS[reduction])
    nodes = _native.nodes() if _native.plain(nll, ref_nll) else None
    if nodes is not None:
        return PreferenceLoss(*nodes.preference(*args))
    loss, rewards = _Preference.apply(*args)
    return PreferenceLoss(loss, rewards[:pairs], rewards[pairs:])


def policy_loss(nll: torch.Tensor, old_nll: torch.Tensor, advantages: torch.Tensor, *, ref_nll: torch.Tensor | None = None,
                offsets: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, reduction: Literal["token", "sequence", "none"] = "token",
                impl: Literal["auto", "kernel", "reference"] = "auto", validate_offsets: bool = True) -> PolicyLoss:
    """Clipped policy loss with a KL term. With u = exp(old_nll - nll), the advantage A of the token (`advantages` of
    nll's shape) or of its sequence ((sequences,); where that is nll's shape too, they are the tokens'), and
    d = nll - ref_nll, a token's loss is
      -min(u A, clip(u, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^d - d - 1).
    `reduction`: "token", the mean over the tokens that count; "sequence", the mean over the sequences that have such
    tokens of each one's mean; "none", per token (0 where it counts nowhere). With no token that counts the loss is 0.
    `validate_offsets` as in `preference_loss`."""
    if reduction not in ("token", "sequence", "none"):
        raise LossInputError(f"unknown reduction {reduction!r}; expected 'token', 'sequence' or 'none'")
    clip_low = _number("clip_low", clip_low, 0 <= clip_low <= 1, "in [0, 1]")
    clip_high = _number("clip_high", clip_high, clip_high >= 0, "finite and not negative")
    kl_coef = _number("kl_coef", kl_coef, kl_coef >= 0, "finite and not negative")
    if kl_coef and ref_nll is None:
        raise LossInputError("kl_coef needs ref_nll, the reference model's losses")
    rows = _sequences(nll, {"old_nll": old_nll, "ref_nll": ref_nll}, offsets, mask, validate_offsets)
    if not advantages.dtype.is_floating_point or (advantages.shape != nll.shape and tuple(advantages.shape) != (rows,)):
        raise LossInputError(f"advantages must be floating-point of nll's shape {tuple(nll.shape)} or ({rows},), one per "
                             f"sequence; got {advantages.dtype} {tuple(advantages.shape)}")
    if advantages.requires_grad and torch.is_grad_enabled():
        raise LossInputError("advantages get no gradient: detach them")
    others = {"old_nll": old_nll, "ref_nll": ref_nll, "advantages": advantages, "offsets": offsets, "mask": mask}
    if _resolve(nll, others, impl) == "reference":
        ref = None if ref_nll is None else ref_nll.detach()
        return _reference_policy(nll, old_nll.detach(), ref, advantages.detach(), offsets, mask, rows, clip_low, clip_high,
                                 kl_coef, reduction)
    args = (_frozen(old_nll), _frozen(ref_nll), _frozen(advantages), _plain_mask(mask), _plain_offsets(offsets), rows, clip_low, clip_high, kl_coef, _REDUCTIONS[reduction])
    nodes = _native.nodes() if _native.plain(nll, *(t for t in (old_nll, ref_nll, advantages) if t is not None)) else None
    if nodes is not None:
        return PolicyLoss(*nodes.policy(nll.contiguous(), *args))
    loss, stats = _Policy.apply(nll.contiguous(), *args)
    return PolicyLoss(loss, stats[0], stats[1])
