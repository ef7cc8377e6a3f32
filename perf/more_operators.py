"""Cases of token scoring (log probabilities, entropy and top alternatives over a head) and of distillation from a
teacher's top alternatives: the plain form in elementary torch operations, and the calls that a program makes.

Hidden states and weights are multiples of 1/64 of a power of two, no larger than bf16 holds exactly, so that every logit is a
whole multiple below 2^24 of one unit and the same number in any order of summation: which alternative comes before which,
and which two are equal, is then defined."""
import math
import sys

import torch

own = False  # run() makes the framework's calls where true, computes the plain form where false

IGNORE = -100
TAIL = 1e-6  # the least mass that the outcomes outside the teacher's list count as


def _score(name, n, d, v, *, top=0, targets=True, temperature=1.0, head="dense", dtype="bf16", mode="eval"):
    return {"name": name, "kind": "score", "n": n, "d": d, "v": v, "top": top, "targets": targets,
            "temperature": temperature, "head": head, "dtype": dtype, "mode": mode}


def _distill(name, n, d, v, k, *, loss="forward", temperature=1.0, renormalize=False, reduction="mean", head="dense",
             dtype="bf16", mode="train"):
    return {"name": name, "kind": "distill", "n": n, "d": d, "v": v, "k": k, "loss": loss, "temperature": temperature,
            "renormalize": renormalize, "reduction": reduction, "head": head, "dtype": dtype, "mode": mode}


def listed():
    return [
        # The alternatives of one next token.
        _score("score_next_token", 1, 4096, 151936, top=20, targets=False),
        # A small batch of next tokens over a 4-bit head.
        _score("score_q4_decode", 16, 4096, 151936, top=5, targets=False, head="q4"),
        # The tokens of a prompt, sampled at a temperature; an odd vocabulary.
        _score("score_prompt_odd", 333, 2048, 32003, top=8, temperature=0.7),
        # A batch of rollouts with the alternatives of each token.
        _score("score_rollout_8k", 8192, 4096, 151936, top=8),
        # A policy step's log probabilities and entropies, forward and backward.
        _score("score_policy_step", 4096, 2048, 128256, mode="train"),
        # fp32, a head that is trained too.
        _score("score_fp32_train", 500, 512, 32000, top=4, head="trainable", dtype="fp32", mode="train"),
        # The smallest call.
        _score("score_tiny", 7, 64, 1000, top=3),
        # The largest distillation step: a frozen head under an adapter.
        _distill("distill_8k", 8192, 4096, 151936, 64),
        # A small student trained whole.
        _distill("distill_full_student", 2048, 896, 151936, 32, loss="jsd", head="trainable"),
        # A 4-bit student's step, reverse divergence at a temperature.
        _distill("distill_q4_reverse", 1023, 2048, 32000, 16, loss="reverse", temperature=2.0, head="q4"),
        # fp32, the teacher's top logits alone, a loss per token.
        _distill("distill_fp32_rows", 300, 256, 8191, 8, renormalize=True, reduction="none", head="trainable", dtype="fp32"),
        # The smallest step.
        _distill("distill_tiny", 5, 64, 997, 4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    head = rng.choice(["dense", "dense", "trainable", "q4"])
    mode = rng.choice(["eval", "train"])
    d = rng.choice([64, 128, 512, 896, 1024, 2048, 4096] if head == "q4" else [64, 136, 512, 896, 1000, 1024, 2048, 4096])
    v = _log_int(rng, 500, 152000)
    n = _log_int(rng, 1, 8192)
    while n * d * v > (1 << 42 if dtype == "bf16" else 1 << 38):
        n = (n + 1) // 2
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    if rng.random() < 0.5:
        return _score("", n, d, v, top=rng.choice([0, 1, 5, 20, 64]), targets=rng.random() < 0.7 or mode == "train",
                      temperature=temperature, head=head, dtype=dtype, mode=mode)
    loss = rng.choice(["forward", "forward", "reverse", "jsd"])
    return _distill("", n, d, v, rng.choice([1, 7, 16, 50, 100]), loss=loss, temperature=temperature,
                    renormalize=loss != "reverse" and rng.random() < 0.3, reduction=rng.choice(["mean", "sum", "none"]),
                    head=head, dtype=dtype, mode=mode)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _on_grid(x, unit):
    return (x / unit).round_().clamp_(-255, 255).mul_(unit)


def _weights(case, g):
    """The head as its user holds it, and its rows in fp32 for the planting below."""
    d, v = case["d"], case["v"]
    size = 2.0 ** round(math.log2(2.0 / math.sqrt(d)))  # logits of random rows of a deviation of about 2
    if case["head"] == "q4":
        words = torch.randint(-2 ** 31, 2 ** 31, (v, d // 8), generator=g, device="cuda").to(torch.int32)
        scales = (size / 4) * 2.0 ** torch.randint(-1, 2, (v, d // 64), generator=g, device="cuda").float()
        head = {"w_q": words, "scales": scales.to(torch.bfloat16), "biases": (-8 * scales).to(torch.bfloat16)}
        return head, size
    w = torch.randn(v, d, generator=g, device="cuda").mul_(size)
    return {"w": _on_grid(w, size / 64).to(_dtype(case))}, size


def _dtype(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _head_rows(head, rows=None):
    """Rows of the head in fp32; all of them without `rows`."""
    if "w" in head:
        w = head["w"].detach()
        return (w if rows is None else w[rows]).float()
    q, s, b = (head[k] if rows is None else head[k][rows] for k in ("w_q", "scales", "biases"))
    nibbles = torch.stack([(q >> (4 * i)) & 15 for i in range(8)], dim=-1).reshape(q.shape[0], -1, 64)
    return (nibbles.float() * s.float()[..., None] + b.float()[..., None]).reshape(q.shape[0], -1)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, d, v = case["n"], case["d"], case["v"]
    head, size = _weights(case, g)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    # Each token has a list of likely words, as a language model's output has: the first of them are planted in its
    # hidden state, with logits that take from nothing to nearly all of the probability.
    k = case["k"] if case["kind"] == "distill" else 8
    first = (v * uniform(n, 1) ** 3).long()
    step = 1 + (uniform(n, 1) * max(0, v // k - 1)).long()
    ids = (first + step * torch.arange(k, device="cuda")) % v
    planted = min(k, 6)
    level = math.log(v) - 2 + 7 * uniform(n, 1) - 5 * uniform(n, planted).sort(1).values
    hidden = torch.randn(n, d, generator=g, device="cuda")
    for j in range(planted):
        rows = _head_rows(head, ids[:, j])
        hidden += rows * (level[:, j:j + 1] / rows.square().sum(1, keepdim=True).clamp(min=size))
    x = {"head": head, "hidden": _on_grid(hidden, 1 / 64).to(_dtype(case))}
    if case["kind"] == "score":
        if not case["targets"]:
            x["targets"] = None
        else:
            pick = (uniform(n) * planted).long()
            x["targets"] = torch.where(uniform(n) < 0.8, ids[torch.arange(n, device="cuda"), pick], (v * uniform(n)).long())
            x["targets"][uniform(n) < 0.1] = IGNORE
            x["hidden"][x["targets"] == IGNORE] = math.nan  # a padded position holds anything
        x["d_logprob"], x["d_entropy"] = (torch.randn(n, generator=g, device="cuda") / n for _ in range(2))
        return x
    z = torch.cat([level, level[:, -1:] - 1 - 6 * uniform(n, k - planted).sort(1).values], 1)
    z = z + torch.randn(n, k, generator=g, device="cuda")
    x["lp"] = z if case["renormalize"] else torch.log_softmax(z, 1) + torch.log(0.6 + 0.3999 * uniform(n, 1))
    x["ids"] = ids
    slot = torch.arange(k, device="cuda")
    x["ids"] = torch.where((uniform(n, 1) < 0.1) & (slot >= 2 * k // 3), -1, x["ids"])  # shorter lists
    x["lp"] = torch.where((uniform(n, 1) < 0.05) & (slot == k - 1), -math.inf, x["lp"])
    x["mask"] = uniform(n) >= 0.1
    x["hidden"][~x["mask"]] = math.nan
    x["lp"][~x["mask"]] = math.nan
    x["d_rows"] = torch.randn(n, generator=g, device="cuda") / n
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    if case["mode"] == "train":
        x["hidden"].requires_grad_(True)
        if case["head"] == "trainable":
            x["head"]["w"].requires_grad_(True)
    return {"case": case, **x}


# ---- plain forms --------------------------------------------------------------------------------------------------

def _largest(z, top):
    """The `top` largest of each row, the lowest index first among equal ones."""
    bits = (z + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2 ** 32 + torch.arange(z.shape[1] - 1, -1, -1, device=z.device)
    ids = z.shape[1] - 1 - torch.topk(key, top, dim=1).values.remainder(2 ** 32)
    return z.gather(1, ids), ids


def _plain_grads(c, dz, h, w):
    grads = {"d_hidden": (dz @ w).to(_dtype(c))}
    return {**grads, "d_weight": (dz.T @ h).to(_dtype(c))} if c["head"] == "trainable" else grads


def _plain_score(st):
    c, w, hidden, y = st["case"], _head_rows(st["head"]), st["hidden"].detach().float(), st["targets"]
    live = torch.ones(c["n"], dtype=torch.bool, device="cuda") if y is None else y != IGNORE
    h = torch.where(live[:, None], hidden, 0.0)
    z = h @ w.T
    x = z / c["temperature"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    lse = m + torch.log(s)
    logp = x - lse
    p = e / s
    entropy = -(p * logp).sum(1)
    out = {"entropy": torch.where(live, entropy, 0.0)}
    if y is not None:
        y = torch.where(live, y, 0)
        out["logprobs"] = torch.where(live, logp.gather(1, y[:, None])[:, 0], 0.0)
    if c["top"]:
        best, ids = _largest(z, c["top"])
        out["top_logprobs"] = torch.where(live[:, None], best / c["temperature"] - lse, -math.inf)
        out["top_ids"] = torch.where(live[:, None], ids, -1)
    if c["mode"] == "eval":
        return out
    ct, ce = (torch.where(live, st[k], 0.0)[:, None] for k in ("d_logprob", "d_entropy"))
    dz = -p * (ct + ce * (logp + entropy[:, None]))
    dz.scatter_add_(1, y[:, None], ct)
    return {**out, **_plain_grads(c, dz / c["temperature"], h, w)}


def _plain_distill(st):
    c, w, hidden = st["case"], _head_rows(st["head"]), st["hidden"].detach().float()
    on = (st["ids"] >= 0) & (st["lp"] != -math.inf) & st["mask"][:, None]
    live = on.any(1, keepdim=True)
    h = torch.where(live, hidden, 0.0)
    x = (h @ w.T) / c["temperature"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    ids = torch.where(on, st["ids"], 0)
    # The list's outcomes and the rest, in 64 bits: what is left of 1 is small.
    lq = x.gather(1, ids).double() - m - torch.log(s.double())
    lt = torch.where(on, st["lp"].double(), 0.0)
    if c["renormalize"]:
        lt = torch.where(on, lt / c["temperature"], -1e4)
        lt = lt - torch.logsumexp(lt, 1, keepdim=True)
    q, t = (torch.where(on, v.exp(), 0.0) for v in (lq, lt))
    left = 1 - q.sum(1, keepdim=True)
    rest_q = left.clamp(min=TAIL)
    rest_t = torch.zeros_like(rest_q) if c["renormalize"] else (1 - t.sum(1, keepdim=True)).clamp(min=TAIL)
    share = 1.0 / live.sum().clamp(min=1) if c["reduction"] == "mean" else 1.0
    # The loss; q f over the list and f of the rest, f the loss's derivative by a probability (but for a constant).
    if c["loss"] == "forward":
        loss = torch.where(on, t * (lt - lq), 0.0).sum(1, keepdim=True)
        loss = loss + (0.0 if c["renormalize"] else rest_t * torch.log(rest_t / rest_q))
        qf, f_rest = -t, -rest_t / rest_q
    elif c["loss"] == "reverse":
        qf, f_rest = torch.where(on, q * (lq - lt), 0.0), torch.log(rest_q / rest_t)
        loss = qf.sum(1, keepdim=True) + rest_q * f_rest
    else:  # halves of both against their mean
        lm = torch.logaddexp(lt, lq) - math.log(2)
        rest_m = (rest_t + rest_q) / 2
        qf, f_rest = torch.where(on, q * (lq - lm), 0.0) / 2, torch.log(rest_q / rest_m) / 2
        loss = (torch.where(on, t * (lt - lm), 0.0) / 2 + qf).sum(1, keepdim=True) + rest_q * f_rest
        if not c["renormalize"]:
            loss = loss + rest_t * torch.log(rest_t / rest_m) / 2
    loss = torch.where(live, loss, 0.0)[:, 0]
    out = {"loss": (loss if c["reduction"] == "none" else loss.sum() * share).float()}
    if c["mode"] == "eval":
        return out
    mean = qf.sum(1, keepdim=True) + left * f_rest
    dz = (e / s) * (f_rest - mean).float()
    dz.scatter_add_(1, ids, torch.where(on, qf - q * f_rest, 0.0).float())
    ct = st["d_rows"][:, None] if c["reduction"] == "none" else share
    dz = torch.where(live, dz * (ct / c["temperature"]), 0.0)
    return {**out, **_plain_grads(c, dz, h, w)}


# ---- the framework's calls ----------------------------------------------------------------------------------------

def _own_run(st):
    if "mlx-train-perf_amd" not in sys.path:
        sys.path.insert(0, "mlx-train-perf_amd")
    import mlx_train_perf as api

    c, h = st["case"], st["head"]
    head = api.QuantizedHead(**h) if "w_q" in h else api.DenseHead(weight=h["w"], trainable=c["head"] == "trainable")
    train = c["mode"] == "train"
    leaves = [st["hidden"], *([h["w"]] if c["head"] == "trainable" else [])]
    with torch.set_grad_enabled(train):
        if c["kind"] == "score":
            r = api.token_logprobs(st["hidden"], head, st["targets"], top=c["top"], temperature=c["temperature"],
                                   ignore_index=IGNORE, validate_targets=False)
            out = {} if r.logprobs is None else {"logprobs": r.logprobs.detach()}
            out["entropy"] = r.entropy.detach()
            if c["top"]:
                out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
            if train:
                grads = torch.autograd.grad((r.logprobs, r.entropy), leaves, (st["d_logprob"], st["d_entropy"]))
        else:
            loss = api.distillation_loss(st["hidden"], head, st["ids"], st["lp"], mask=st["mask"], kind=c["loss"],
                                         temperature=c["temperature"], renormalize=c["renormalize"],
                                         reduction=c["reduction"], validate_ids=False)
            out = {"loss": loss.detach()}
            if train:
                grads = torch.autograd.grad(loss, leaves, st["d_rows"] if c["reduction"] == "none" else None)
    if train:
        out["d_hidden"] = grads[0]
        if c["head"] == "trainable":
            out["d_weight"] = grads[1]
    return out


def run(state):
    if own:
        return _own_run(state)
    with torch.no_grad():
        return (_plain_score if state["case"]["kind"] == "score" else _plain_distill)(state)


# ---- work ---------------------------------------------------------------------------------------------------------

def work(case):
    n, d, v = case["n"], case["d"], case["v"]
    e = 4 if case["dtype"] == "fp32" else 2
    train, trainable = case["mode"] == "train", case["head"] == "trainable"
    weights = v * d // 2 + v * d // 64 * 4 if case["head"] == "q4" else v * d * e
    rows = n * (12 * case["top"] + 16) if case["kind"] == "score" else n * (12 * case["k"] + 9)
    moved = weights * (2 if train and trainable else 1) + n * d * e * (2 if train else 1) + rows
    products = 1 + (train and 1 + trainable)  # logits; dL/dhidden; dL/dw
    return {"bytes": float(moved), "flops": 2.0 * n * d * v * products}


# ---- values in 64 bits --------------------------------------------------------------------------------------------

def _dense64(head):
    if "w" in head:
        return head["w"].detach().double()
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    v, words = head["w_q"].shape
    nibble = torch.bitwise_and(torch.bitwise_right_shift(head["w_q"][:, :, None], shifts), 15).reshape(v, words * 8)
    return torch.addcmul(head["biases"].double().repeat_interleave(64, 1), head["scales"].double().repeat_interleave(64, 1),
                         nibble.double())


def _exact_row_block(case, x, rows, w, need):
    """(outputs, dL/dlogits) of some rows, through autograd over 64-bit log probabilities; the rows all count."""
    h = x["hidden"][rows].double()
    z = (h @ w.T).requires_grad_(need)
    logp = torch.log_softmax(z / case["temperature"], dim=1)
    if case["kind"] == "score":
        out = {}
        entropy = torch.special.entr(logp.exp()).sum(1)
        scalar = (entropy * x["d_entropy"][rows].double()).sum()
        if x["targets"] is not None:
            out["logprobs"] = -torch.nn.functional.nll_loss(logp, x["targets"][rows], reduction="none")
            scalar = scalar + (out["logprobs"] * x["d_logprob"][rows].double()).sum()
        out["entropy"] = entropy
        if case["top"]:
            left = z.detach().clone()
            ids = []
            for _ in range(case["top"]):  # one after the other: the first index that holds the maximum
                columns = torch.arange(left.shape[1], device="cuda").expand_as(left)
                best = columns.masked_fill(left != left.amax(1, keepdim=True), left.shape[1]).amin(1, keepdim=True)
                ids.append(best)
                left.scatter_(1, best, -math.inf)
            out["top_ids"] = torch.cat(ids, 1)
            out["top_logprobs"] = logp.detach().gather(1, out["top_ids"])
    else:
        on = (x["ids"][rows] >= 0) & (x["lp"][rows] > -math.inf)
        never = -1e4  # the logarithm of 0
        s = torch.where(on, logp.gather(1, x["ids"][rows].clamp(min=0)), never)
        t = x["lp"][rows].double().masked_fill(~on, never)

        def with_rest(a):  # the floor leaves the gradient of what it lifts
            rest = 1 - a.exp().sum(1, keepdim=True)
            return torch.cat([a, (rest + (rest.clamp(min=TAIL) - rest).detach()).log()], 1)

        def divergence(a, b):
            return (a.exp() * (a - b)).sum(1)

        if case["renormalize"]:
            t = torch.log_softmax((t / case["temperature"]).masked_fill(~on, never), 1)
            t = torch.nn.functional.pad(t, (0, 1), value=never)
        else:
            t = with_rest(t)
        s = with_rest(s)
        if case["loss"] == "forward":
            loss = divergence(t, s)
        elif case["loss"] == "reverse":
            loss = divergence(s, t)
        else:
            middle = torch.logaddexp(s, t) - math.log(2)
            loss = (divergence(t, middle) + divergence(s, middle)) / 2
        out = {"loss": loss}
        scalar = (loss * (x["d_rows"][rows].double() if case["reduction"] == "none" else x["share"])).sum()
    dz = torch.autograd.grad(scalar, z)[0] if need else None
    return {k: v.detach() for k, v in out.items()}, h, dz


def exact(case, seed):
    n, d, v = case["n"], case["d"], case["v"]
    if n * d * v > 1 << 43:
        return None
    x = _inputs(case, seed)
    w = _dense64(x["head"])
    if case["kind"] == "score":
        live = torch.ones(n, dtype=torch.bool, device="cuda") if x["targets"] is None else x["targets"] != IGNORE
        out = {"logprobs": torch.zeros(n, dtype=torch.float64, device="cuda")} if x["targets"] is not None else {}
        out["entropy"] = torch.zeros(n, dtype=torch.float64, device="cuda")
        if case["top"]:
            out["top_logprobs"] = torch.full((n, case["top"]), -math.inf, dtype=torch.float64, device="cuda")
            out["top_ids"] = torch.full((n, case["top"]), -1, dtype=torch.int64, device="cuda")
    else:
        live = x["mask"] & ((x["ids"] >= 0) & (x["lp"] > -math.inf)).any(1)
        x["share"] = 1.0 / max(1, int(live.sum())) if case["reduction"] == "mean" else 1.0
        out = {"loss": torch.zeros(n, dtype=torch.float64, device="cuda")}
    train = case["mode"] == "train"
    d_hidden = torch.zeros(n, d, dtype=torch.float64, device="cuda") if train else None
    d_weight = torch.zeros(v, d, dtype=torch.float64, device="cuda") if train and case["head"] == "trainable" else None
    for rows in live.nonzero()[:, 0].split(max(1, (1 << 27) // v)):
        part, h, dz = _exact_row_block(case, x, rows, w, train)
        for k, value in part.items():
            out[k][rows] = value
        if train:
            d_hidden[rows] = dz @ w
            if d_weight is not None:
                d_weight.addmm_(dz.T, h)
    if case["kind"] == "distill" and case["reduction"] != "none":
        out["loss"] = out["loss"].sum() * x["share"]
    if train:
        out["d_hidden"] = d_hidden
        if d_weight is not None:
            out["d_weight"] = d_weight
    return out
