"""Token scoring and distillation over a head, without the (N, V) logits: `token_logprobs` and `distillation_loss`.

Both take `hidden` and `head` as `linear_cross_entropy` does (dense bf16 or fp32, trainable or frozen, 4-bit), and share its
product and its backward. What `token_logprobs` returns as a teacher's alternatives is what `distillation_loss` takes.

- `impl="kernel"` (and "auto"): HIP kernels on a gfx950 GPU, bf16 or fp32 hidden states.
- `impl="reference"`: torch operators in 64 bits on whole logits, any device and floating type.

Tokens that are left out (an ignored target, a mask of 0, an empty list) may hold anything, NaN too: they get no gradient
and give none.
"""
from __future__ import annotations

import math
import operator
from typing import Literal, NamedTuple

import torch
from torch.autograd.function import once_differentiable

from mlx_train_perf import _compat, _native
from mlx_train_perf.core import loss as _loss
from mlx_train_perf.core.loss import DenseHead, HeadRef
from mlx_train_perf.core.quant import dequantize
from mlx_train_perf.errors import LossInputError, UnsupportedHeadError
from mlx_train_perf.plan import launch as _plan

MAX_LIST = 128          # alternatives, and slots of a teacher's list, that the kernels serve
MAX_VOCAB = 1 << 21     # vocabulary that the kernels serve
TAIL_FLOOR = 1e-6       # least mass that the outcomes outside a list count as
_KINDS = {"forward": 0, "reverse": 1, "jsd": 2}
_ID_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class TokenLogprobs(NamedTuple):
    """`logprobs` (None without targets) and `entropy` have hidden's leading dims, in nats, with a gradient; `top_logprobs`
    and `top_ids` (int64) the alternatives last, the likeliest first, without one."""
    logprobs: torch.Tensor | None
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def _head_v(head: HeadRef) -> int:
    return _loss._head_v(head)


def _temperature(x: float) -> float:
    if not 1e-3 <= x <= 1e3:
        raise LossInputError(f"temperature must be in [1e-3, 1e3]; got {x!r}")
    return float(x)


def _resolve(hidden2: torch.Tensor, head: HeadRef, others: dict[str, torch.Tensor | None], impl: str, many: tuple[str, int],
             allow_unverified_mlx: bool) -> Literal["kernel", "reference"]:
    if impl == "reference":
        return "reference"
    if impl not in ("auto", "kernel"):
        raise LossInputError(f"unknown impl {impl!r}; expected one of 'auto', 'kernel', 'reference'")
    try:
        _loss._require_kernel_supported(head=head, dtype=hidden2.dtype)
    except UnsupportedHeadError as e:
        raise UnsupportedHeadError(str(e).replace("impl='chunked'", "impl='reference'")) from None
    name, count = many
    if count > MAX_LIST:
        raise UnsupportedHeadError(f"kernel impl serves {name} of at most {MAX_LIST} (got {count}); use impl='reference'.")
    if _head_v(head) > MAX_VOCAB:
        raise UnsupportedHeadError(f"kernel impl serves a vocabulary of at most 2^21 (got {_head_v(head)}); use impl='reference'.")
    _compat.check_device_verified(allow_unverified=allow_unverified_mlx, error=UnsupportedHeadError)
    _compat.require_gpu_tensor(hidden2, error=UnsupportedHeadError)
    parts = ({"head.weight": head.weight} if isinstance(head, DenseHead)
             else {"head.w_q": head.w_q, "head.scales": head.scales, "head.biases": head.biases})
    for name, t in {**parts, **others}.items():
        if t is not None and t.device != hidden2.device:
            raise LossInputError(f"{name} is on {t.device} but hidden is on {hidden2.device}; the kernel impl needs every "
                                 "input on the same GPU")
    return "kernel"


def _check_hidden(hidden: torch.Tensor, head: HeadRef) -> tuple[int, ...]:
    """The loss's checks of hidden and head; hidden's leading dims."""
    if hidden.dim() not in (2, 3):
        raise LossInputError(f"hidden must be 2D (N,D) or 3D (B,S,D), got shape {tuple(hidden.shape)}")
    leading = tuple(hidden.shape[:-1])
    # (targets of the right shape: theirs are checked where there are any)
    _loss._validate_inputs(hidden=hidden, head=head, targets=torch.empty(leading, dtype=torch.int64, device="meta"),
                           validate_targets=False, ignore_index=0)
    return leading


def _as_int64(ids: torch.Tensor) -> torch.Tensor:
    """Whole numbers in 64 bits, before anything is compared with them: a narrower type takes V and ignore_index into its own
    range first (300 is 44 in uint8). Others as they are, for their refusal."""
    return ids if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool else ids.to(torch.int64)


class _Inputs(NamedTuple):
    """hidden and head as the kernels read them."""
    hidden: torch.Tensor | None
    w: torch.Tensor | None
    w_q: torch.Tensor | None
    scales: torch.Tensor | None
    biases: torch.Tensor | None
    kind: int
    owner: torch.Tensor

    @property
    def v(self) -> int:
        return (self.w if self.w is not None else self.w_q).shape[0]


def _inputs(hidden2: torch.Tensor, head: HeadRef) -> _Inputs:
    h = hidden2.contiguous()
    if h.data_ptr() % 16:   # a view off a 16-byte boundary
        h = h.clone()
    if isinstance(head, DenseHead):
        w = head.weight if head.trainable else head.weight.detach()
        if not w.is_contiguous():
            raise UnsupportedHeadError("kernel impl needs a contiguous (V, D) head weight")
        return _Inputs(h, w, None, None, None, _native.HEAD_DENSE, head.weight)
    sb = torch.float32 if h.dtype == torch.float32 else torch.bfloat16
    return _Inputs(h, None, head.w_q.contiguous(), head.scales.to(sb).contiguous(), head.biases.to(sb).contiguous(),
                   _native.HEAD_Q4, head.w_q)


def _nodes(x: _Inputs, *others):
    """The C++ nodes, where every tensor of the call is plain; None: the Python Functions serve it, the same bits."""
    plain = _native.plain(*(t for t in (*x, *others) if isinstance(t, torch.Tensor)))
    return _native.nodes() if plain else None


def _forward_kind(x: _Inputs) -> int:
    """As the loss's forward: a 4-bit head dequantized into the workspace where the budget holds all of it, also in fp32."""
    n, d = x.hidden.shape
    f32 = x.hidden.dtype == torch.float32
    if f32:
        return _staged32(x)
    staged = _loss._forward_stage_bytes(_native.load(), n, d, x.v, x.kind, f32)
    return _native.HEAD_Q4_STAGED if staged else x.kind


def _staged32(x: _Inputs) -> int:
    """The kind of an fp32 call: with its weights in registers a 4-bit head's products take some four times as long."""
    fits = x.kind == _native.HEAD_Q4 and x.v * x.hidden.shape[1] * 4 <= _plan.lce_bwd_budget_bytes()
    return _native.HEAD_Q4_STAGED if fits and _loss.os.environ.get("MTP_LCE_STAGE_HEAD", "1") != "0" else x.kind


def _kept_bytes(x: _Inputs) -> int:
    """Bytes of the logits that a forward with a backward to come keeps for it, which then forms none again: a sixth of the
    backward's workspace budget holds them (256 MiB of 1.5 GiB), or 0. A product less: fp32 training at 1588 x 4096 x 10500
    5250 -> 4030 us, a 4-bit student's 488 -> 407 us."""
    nbytes = x.hidden.shape[0] * ((x.v + 127) // 128 * 128) * 4
    return nbytes if nbytes <= _plan.lce_bwd_budget_bytes() // 6 else 0


def _kept_logits(x: _Inputs) -> torch.Tensor | None:
    nbytes = _kept_bytes(x)
    return torch.empty(nbytes // 4, dtype=torch.float32, device=x.hidden.device) if nbytes else None


def _head_ptrs(x: _Inputs) -> tuple:
    return _native.ptr(x.w), _native.ptr(x.w_q), _native.ptr(x.scales), _native.ptr(x.biases)


def _workspace(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=like.device)


def _backward(x: _Inputs, k: int, want_dw: bool, call) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(dL/dhidden, dL/dw): plans vocab chunk and row block as the loss's backward does (a cached transposed head, staged
    chunks, or neither) and hands `call` the entry point's arguments before and after its own."""
    lib = _native.load()
    n, d = x.hidden.shape
    v, kind, budget = x.v, x.kind, _plan.lce_bwd_budget_bytes()
    d_hidden = torch.empty_like(x.hidden)
    d_w = torch.empty_like(x.w) if want_dw else None
    w, w_q, scales, biases = _head_ptrs(x)
    if x.hidden.dtype == torch.float32:
        kind = _staged32(x)
        chunk = lib.mtp_lce_bwd_f32_chunk(n, d, v, budget)
        ws_bytes = lib.mtp_score_bwd_f32_workspace_bytes(n, d, v, kind, chunk, k, int(want_dw))
        head, after = (w, w_q, scales, biases), (chunk,)
    else:
        mode = _loss.os.environ.get("MTP_LCE_TRANSPOSED_HEAD", "auto")
        w_t = (None if want_dw and mode != "1"
               else _loss._transposed_head(x.owner, x.w, x.w_q, x.scales, x.biases, kind, v, d))
        staged = w_t is None and d % 64 == 0 and _loss.os.environ.get("MTP_LCE_STAGE_HEAD", "1") != "0"
        if staged:
            kind = _native.HEAD_Q4_STAGED if kind == _native.HEAD_Q4 else _native.HEAD_DENSE_STAGED
            chunk, rows = lib.mtp_lce_bwd_stage_chunk(n, d, v, kind, budget), n
        else:
            rows = n if want_dw else lib.mtp_lce_bwd_row_block(n, d, v, budget)
            chunk = (v + 255) // 256 * 256 if rows < n else lib.mtp_lce_bwd_chunk(n, d, v, budget)
        ws_bytes = lib.mtp_score_bwd_workspace_bytes(n, d, v, kind, chunk, rows, k, int(want_dw))
        head, after = (w, _native.ptr(w_t), w_q, scales, biases), (chunk, rows)
    ws = _workspace(ws_bytes, x.hidden)
    with _native.on_device(x.hidden):
        rc = call(lib, (x.hidden.data_ptr(), *head), (n, d, v, kind),
                  (d_hidden.data_ptr(), _native.ptr(d_w), *after, ws.data_ptr(), ws_bytes, _native.stream_of(x.hidden)))
    _native.check(rc, domain="loss")
    return d_hidden, d_w


def _float(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.to(torch.float32).contiguous()


def _entry(lib, name: str, x: _Inputs):
    return getattr(lib, name + ("_f32" if x.hidden.dtype == torch.float32 else ""))


def _score_forward(x: _Inputs, targets, ignore_index: int, top: int, temperature: float, logits: torch.Tensor | None):
    """(logprobs, entropy, top_logprobs, top_ids, lse, tgt) of mtp_logprobs_fwd."""
    lib = _native.load()
    n, d = x.hidden.shape
    dev = x.hidden.device
    f32 = x.hidden.dtype == torch.float32
    kind = _forward_kind(x)
    # (results of their own, not views of one: a caller may change them in place)
    entropy, lse = (torch.empty(n, dtype=torch.float32, device=dev) for _ in range(2))
    logprobs, tgt = (torch.empty_like(lse) if targets is not None else None for _ in range(2))
    top_lp = torch.empty((n, top), dtype=torch.float32, device=dev)
    top_ids = torch.empty((n, top), dtype=torch.int64, device=dev)
    size = lib.mtp_logprobs_fwd_f32_workspace_bytes if f32 else lib.mtp_logprobs_fwd_workspace_bytes
    ws_bytes = size(n, d, x.v, kind, top, int(logits is not None))
    ws = _workspace(ws_bytes, x.hidden)
    with _native.on_device(x.hidden):
        rc = _entry(lib, "mtp_logprobs_fwd", x)(
            x.hidden.data_ptr(), *_head_ptrs(x), _native.ptr(targets), n, d, x.v, kind, ignore_index, top, temperature,
            _native.ptr(logprobs), entropy.data_ptr(), top_lp.data_ptr(), top_ids.data_ptr(), lse.data_ptr(), _native.ptr(tgt),
            _native.ptr(logits), ws.data_ptr(), ws_bytes, _native.stream_of(x.hidden))
    _native.check(rc, domain="loss")
    return logprobs, entropy, top_lp, top_ids, lse, tgt


class _TokenLogprobs(torch.autograd.Function):
    """Saves each token's log-sum-exp, entropy and log probability, and few enough logits; more of them the backward forms again.
    record: whether autograd is (inside a forward it is off, and what asks for a gradient asks under no_grad too)."""

    @staticmethod
    def forward(ctx, hidden, w, w_q, scales, biases, kind, owner, targets, ignore_index, top, temperature, record=True):
        x = _Inputs(hidden, w, w_q, scales, biases, kind, owner)
        logits = _kept_logits(x) if record and any(ctx.needs_input_grad[:2]) else None
        logprobs, entropy, top_lp, top_ids, lse, tgt = _score_forward(x, targets, ignore_index, top, temperature, logits)
        ctx.save_for_backward(hidden, targets, lse, entropy, tgt, logits)
        ctx.inputs, ctx.args = x._replace(hidden=None), (ignore_index, temperature)
        ctx.mark_non_differentiable(top_lp, top_ids)
        ctx.set_materialize_grads(False)
        return logprobs, entropy, top_lp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprobs, d_entropy, _d_top, _d_ids):
        hidden, targets, lse, entropy, tgt, logits = ctx.saved_tensors
        ignore_index, temperature = ctx.args
        x = ctx.inputs._replace(hidden=hidden)
        d_logprobs, d_entropy = _float(d_logprobs), _float(d_entropy)

        def call(lib, head, shape, rest):
            return _entry(lib, "mtp_logprobs_bwd", x)(
                *head, _native.ptr(targets), *shape, ignore_index, temperature, lse.data_ptr(), entropy.data_ptr(),
                _native.ptr(tgt), _native.ptr(logits), _native.ptr(d_logprobs), _native.ptr(d_entropy), *rest)

        d_hidden, d_w = _backward(x, 1, x.w is not None and ctx.needs_input_grad[1], call)
        return (d_hidden, d_w, *[None] * 10)


class _Distillation(torch.autograd.Function):
    """Saves the gradient's factors, one per token and one per slot of its list, and few enough logits."""

    @staticmethod
    def forward(ctx, hidden, w, w_q, scales, biases, kind, owner, ids, teacher, mask, loss_kind, beta, temperature,
                renormalize, reduction, record=True):
        lib = _native.load()
        x = _Inputs(hidden, w, w_q, scales, biases, kind, owner)
        n, d = hidden.shape
        k, dev = ids.shape[1], hidden.device
        f32 = hidden.dtype == torch.float32
        fwd_kind = _forward_kind(x)
        loss = torch.empty((n,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        scale = torch.empty((), dtype=torch.float32, device=dev)
        lse, rest = torch.empty((2, n), dtype=torch.float32, device=dev).unbind(0)
        coef = torch.empty((n, k), dtype=torch.float32, device=dev)
        columns = torch.empty((n, k), dtype=torch.int32, device=dev)
        size = lib.mtp_distill_fwd_f32_workspace_bytes if f32 else lib.mtp_distill_fwd_workspace_bytes
        logits = _kept_logits(x) if record and any(ctx.needs_input_grad[:2]) else None
        ws_bytes = size(n, d, x.v, fwd_kind, k, int(logits is not None))
        ws = _workspace(ws_bytes, hidden)
        with _native.on_device(hidden):
            rc = _entry(lib, "mtp_distill_fwd", x)(
                hidden.data_ptr(), *_head_ptrs(x), ids.data_ptr(), teacher.data_ptr(), _native.ptr(mask), n, d, x.v, fwd_kind, k,
                loss_kind, beta, temperature, renormalize, reduction, loss.data_ptr(), scale.data_ptr(), lse.data_ptr(),
                rest.data_ptr(), coef.data_ptr(), columns.data_ptr(), _native.ptr(logits), ws.data_ptr(), ws_bytes,
                _native.stream_of(hidden))
        _native.check(rc, domain="loss")
        ctx.save_for_backward(hidden, scale, lse, rest, coef, columns, logits)
        ctx.inputs, ctx.args = x._replace(hidden=None), (temperature, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        hidden, scale, lse, rest, coef, columns, logits = ctx.saved_tensors
        temperature, reduction = ctx.args
        x = ctx.inputs._replace(hidden=hidden)
        ct, k = _float(d_loss), coef.shape[1]

        def call(lib, head, shape, after):
            return _entry(lib, "mtp_distill_bwd", x)(
                *head, *shape, k, temperature, reduction, ct.data_ptr(), scale.data_ptr(), lse.data_ptr(), rest.data_ptr(),
                coef.data_ptr(), columns.data_ptr(), _native.ptr(logits), *after)

        d_hidden, d_w = _backward(x, k, x.w is not None and ctx.needs_input_grad[1], call)
        return (d_hidden, d_w, *[None] * 14)


# ---- the reference impl -------------------------------------------------------------------------------------------

def _reference_logits(hidden2: torch.Tensor, head: HeadRef, live: torch.Tensor, temperature: float) -> torch.Tensor:
    if isinstance(head, DenseHead):
        w = head.weight if head.trainable else head.weight.detach()
    else:   # the weights that the kernels' products take: rounded to bf16 under bf16 hidden states
        w = dequantize(head.w_q, head.scales, head.biases, group_size=head.group_size, bits=head.bits, dtype=hidden2.dtype)
    h = torch.where(live[:, None], hidden2, torch.zeros_like(hidden2))
    return (h.double() @ w.double().T) / temperature


def _out(x: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return x if like.dtype == torch.float64 else x.to(torch.float32)


def _finite(logp: torch.Tensor) -> torch.Tensor:
    """A factor of exp(logp): what is ruled out (-inf) adds 0 and no NaN, to the value and to its gradient."""
    return logp.masked_fill(logp == -math.inf, 0.0)


def _reference_score(hidden2, head, targets2, ignore_index, top, temperature):
    n = hidden2.shape[0]
    live = torch.ones(n, dtype=torch.bool, device=hidden2.device) if targets2 is None else targets2 != ignore_index
    logp = torch.log_softmax(_reference_logits(hidden2, head, live, temperature), dim=1)
    entropy = torch.where(live, -(logp.exp() * _finite(logp)).sum(1), 0.0)
    logprobs = None
    if targets2 is not None:
        y = torch.where(live, targets2, 0)
        logprobs = torch.where(live, logp.gather(1, y[:, None])[:, 0], 0.0)
        logprobs = _out(logprobs, hidden2)
    with torch.no_grad():
        value, ids = torch.sort(logp.detach(), dim=1, descending=True, stable=True)   # equal ones by index
        value = torch.where(live[:, None], value[:, :top], -math.inf)
        ids = torch.where(live[:, None], ids[:, :top], -1)
    return logprobs, _out(entropy, hidden2), _out(value, hidden2), ids


def _reference_distillation(hidden2, head, ids, teacher, mask, kind, beta, temperature, renormalize, reduction):
    v = _head_v(head)
    on = (ids >= 0) & (ids < v) & (teacher != -math.inf)
    if mask is not None:
        on = on & (mask[:, None] != 0)
    first = torch.ones_like(on)   # an id that an earlier slot has counts there
    for k in range(1, ids.shape[1]):
        first[:, k] = ~(on[:, :k] & (ids[:, :k] == ids[:, k:k + 1])).any(1)
    on = on & first
    live = on.any(1)
    logp = torch.log_softmax(_reference_logits(hidden2, head, live, temperature), dim=1)
    lq = logp.gather(1, torch.where(on, ids, 0))
    lt = torch.where(on, teacher.double(), 0.0)
    if renormalize:
        lt = torch.where(on, lt / temperature, -math.inf)
        lt = torch.where(on, lt - torch.logsumexp(torch.where(live[:, None], lt, 0.0), 1, keepdim=True), 0.0)
    q, t = torch.where(on, lq.exp(), 0.0), torch.where(on, lt.exp(), 0.0)

    def rest(p):   # the floor leaves the gradient of what it lifts
        left = 1 - p.sum(1)
        return left + (left.clamp(min=TAIL_FLOOR) - left).detach()

    rq = rest(q)
    rt = torch.zeros_like(rq) if renormalize else rest(t)
    safe = torch.where(rt > 0, rt, 1.0)
    if kind == "forward":
        loss = torch.where(on, t * (lt - lq), 0.0).sum(1) + rt * (safe / rq).log()
    elif kind == "reverse":
        loss = torch.where(on, q * (_finite(lq) - lt), 0.0).sum(1) + rq * (rq / rt).log()
    else:
        lm = torch.logaddexp(math.log(beta) + lt, math.log1p(-beta) + lq)
        rm = beta * rt + (1 - beta) * rq
        loss = torch.where(on, beta * t * (lt - lm) + (1 - beta) * q * (_finite(lq) - lm), 0.0).sum(1)
        loss = loss + beta * rt * (safe / rm).log() + (1 - beta) * rq * (rq / rm).log()
    loss = torch.where(live, loss, 0.0)
    if reduction == "mean":
        loss = loss.sum() / live.sum().clamp(min=1)
    elif reduction == "sum":
        loss = loss.sum()
    return _out(loss, hidden2)


# ---- public -------------------------------------------------------------------------------------------------------

def token_logprobs(hidden: torch.Tensor, head: HeadRef, targets: torch.Tensor | None = None, *, top: int = 0,
                   temperature: float = 1.0, impl: Literal["auto", "kernel", "reference"] = "auto",
                   allow_unverified_mlx: bool = False, validate_targets: bool = True,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of each token's target, the entropy of its distribution and its `top` likeliest alternatives under
    softmax(hidden @ head.T / temperature).

    Alternatives come in falling order, equal logits by their index; a target among them has the same log probability there
    and in `logprobs`. The gradient of `logprobs` and `entropy` goes to `hidden` and to a trainable dense head. A token whose
    target is `ignore_index` gets 0, 0, and alternatives of id -1 and log probability -inf. `validate_targets` as in
    `linear_cross_entropy`: unchecked targets outside the vocabulary count as a logit of 0."""
    leading = _check_hidden(hidden, head)
    if targets is not None:
        targets = _as_int64(targets)
        _loss._validate_inputs(hidden=hidden, head=head, targets=targets, validate_targets=validate_targets,
                               ignore_index=ignore_index)
    temperature = _temperature(temperature)
    try:
        top = operator.index(top)
    except TypeError:
        raise LossInputError(f"top must be a whole number; got {top!r}") from None
    if not 0 <= top <= _head_v(head):
        raise LossInputError(f"top must be in [0, V={_head_v(head)}]; got {top}")
    if not _loss._int64(ignore_index):
        raise LossInputError(f"ignore_index must be a whole number of 64 bits; got {ignore_index!r}")
    hidden2 = hidden.reshape(-1, hidden.shape[-1])
    targets2 = None if targets is None else targets.reshape(-1)
    if _resolve(hidden2, head, {"targets": targets}, impl, ("top", top), allow_unverified_mlx) == "reference":
        parts = _reference_score(hidden2, head, targets2, ignore_index, top, temperature)
    else:
        x = _inputs(hidden2, head)
        y = None if targets2 is None else targets2.contiguous()
        args = (y, int(ignore_index), top, temperature)
        nodes = _nodes(x, *args)
        parts = _TokenLogprobs.apply(*x, *args, torch.is_grad_enabled()) if nodes is None else nodes.logprobs(*x, _forward_kind(x), _kept_bytes(x), *args)
    *logprobs, entropy, top_lp, top_ids = parts   # (the node has none without targets)
    logprobs = logprobs[0] if logprobs else None
    return TokenLogprobs(None if logprobs is None else logprobs.view(leading), entropy.view(leading),
                         top_lp.view(*leading, top), top_ids.view(*leading, top))


def distillation_loss(hidden: torch.Tensor, head: HeadRef, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                      mask: torch.Tensor | None = None, kind: Literal["forward", "reverse", "jsd"] = "forward",
                      beta: float = 0.5, temperature: float = 1.0, renormalize: bool = False,
                      reduction: Literal["none", "mean", "sum"] = "mean",
                      impl: Literal["auto", "kernel", "reference"] = "auto", allow_unverified_mlx: bool = False,
                      validate_ids: bool = True) -> torch.Tensor:
    """Divergence between a teacher's list of likely tokens and the student softmax(hidden @ head.T / temperature).

    `teacher_ids` (integers) and `teacher_logprobs` hold K slots for each of hidden's tokens: what `token_logprobs(..., top=K)`
    of the teacher returns, at the same temperature. A slot is empty where its id is negative, its log probability -inf, or its
    id that of an earlier slot. All tokens outside the list are one further outcome, of what the list leaves of 1 (at least
    1e-6, for either model). With t the teacher, q the student:
      "forward": KL(t | q);  "reverse": KL(q | t);
      "jsd": beta KL(t | m) + (1 - beta) KL(q | m), m = beta t + (1 - beta) q, 0 < beta < 1.
    `renormalize`: the teacher's slots are logits, t = softmax(them / temperature) over the list, with nothing outside it (not
    with "reverse").
    `mask` (hidden's leading dims, bool or uint8) says which tokens count; those without any outcome in their list do
    not. "mean" is over the tokens that count (0 without any); "none" gives them 0. There is no factor of temperature squared: multiply
    by it for gradients of one size at any temperature. The gradient goes to `hidden` and to a
    trainable dense head. `validate_ids` checks at one host sync that ids lie below V; unchecked, such slots are empty."""
    if reduction not in _REDUCTIONS:
        raise LossInputError(f"unknown reduction {reduction!r}; expected 'none', 'mean' or 'sum'")
    if kind not in _KINDS:
        raise LossInputError(f"unknown kind {kind!r}; expected one of {', '.join(map(repr, _KINDS))}")
    if kind == "jsd" and not 0 < beta < 1:
        raise LossInputError(f"beta must be in (0, 1); got {beta!r}")
    if kind == "reverse" and renormalize:
        raise LossInputError("a renormalized teacher gives nothing to what its list leaves out: kind='reverse' is infinite")
    leading = _check_hidden(hidden, head)
    temperature = _temperature(temperature)
    if teacher_ids.dim() != hidden.dim() or tuple(teacher_ids.shape[:-1]) != leading or teacher_ids.shape[-1] < 1:
        raise LossInputError(f"teacher_ids must be hidden's leading dims {leading} and at least one slot; got shape "
                             f"{tuple(teacher_ids.shape)}")
    if teacher_ids.dtype not in _ID_TYPES:
        raise LossInputError(f"teacher_ids must be int8 to int64 or uint8, got {teacher_ids.dtype}")
    if teacher_logprobs.shape != teacher_ids.shape or not teacher_logprobs.dtype.is_floating_point:
        raise LossInputError(f"teacher_logprobs must be floating-point of teacher_ids' shape {tuple(teacher_ids.shape)}; got "
                             f"{teacher_logprobs.dtype} {tuple(teacher_logprobs.shape)}")
    if teacher_logprobs.requires_grad and torch.is_grad_enabled():
        raise LossInputError("teacher_logprobs belong to a frozen model and get no gradient: detach them")
    if mask is not None and (tuple(mask.shape) != leading or mask.dtype not in (torch.bool, torch.uint8)):
        raise LossInputError(f"mask must be bool or uint8 of hidden's leading dims {leading}; got {mask.dtype} {tuple(mask.shape)}")
    teacher_ids = _as_int64(teacher_ids)
    v = _head_v(head)
    if validate_ids and bool((teacher_ids >= v).any()):   # a host sync
        raise LossInputError(f"teacher_ids must be below V={v} (negative ones are empty slots)")
    hidden2 = hidden.reshape(-1, hidden.shape[-1])
    k = teacher_ids.shape[-1]
    ids2, teacher2 = teacher_ids.reshape(-1, k), teacher_logprobs.reshape(-1, k)
    mask2 = None if mask is None else mask.reshape(-1)
    others = {"teacher_ids": teacher_ids, "teacher_logprobs": teacher_logprobs, "mask": mask}
    if _resolve(hidden2, head, others, impl, ("lists", k), allow_unverified_mlx) == "reference":
        loss = _reference_distillation(hidden2, head, ids2, teacher2, mask2, kind, beta, temperature, renormalize, reduction)
    else:
        x = _inputs(hidden2, head)
        args = (ids2.contiguous(), _float(teacher2), None if mask2 is None else mask2.contiguous(), _KINDS[kind],
                float(beta), temperature, int(renormalize), _REDUCTIONS[reduction])
        nodes = _nodes(x, *args)
        loss = _Distillation.apply(*x, *args, torch.is_grad_enabled()) if nodes is None else nodes.distillation(*x, _forward_kind(x), _kept_bytes(x), *args)
    return loss.view(leading) if reduction == "none" else loss
