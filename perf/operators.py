"""Cases of the attention variants (capped scores, a bias by distance, key spans) and of the preference and policy
losses: the plain form in elementary torch operations, and the calls that a training program makes."""
import math
import sys

import torch

own = False  # run() makes the framework's calls where true, computes the plain form where false


def _attn(name, b, hq, hkv, s, dh, *, mask="causal", cap=0.0, slopes=False, dtype="bf16", mode="train"):
    return {"name": name, "kind": "attn", "b": b, "hq": hq, "hkv": hkv, "s": s, "dh": dh, "mask": mask, "cap": cap,
            "slopes": slopes, "dtype": dtype, "mode": mode}


def _pref(name, pairs, tokens, *, layout="padded", loss="sigmoid"):
    return {"name": name, "kind": "pref", "pairs": pairs, "tokens": tokens, "layout": layout, "loss": loss}


def _policy(name, rows, tokens, *, layout="padded", adv="sequence", reduction="token", kl=0.05):
    return {"name": name, "kind": "policy", "rows": rows, "tokens": tokens, "layout": layout, "adv": adv,
            "reduction": reduction, "kl": kl}


def listed():
    return [
        # A long-context training layer of a model with capped scores.
        _attn("attn_cap_8k", 1, 32, 8, 8192, 128, cap=50.0),
        # A layer of a model with a distance bias in place of rotary positions.
        _attn("attn_slopes_2k", 4, 16, 16, 2048, 64, slopes=True),
        # Packed prompt and response documents: each prompt sees itself whole, the tail is padding.
        _attn("attn_docs_prefix_8k", 1, 16, 4, 8192, 128, mask="docs"),
        # A short fine-tuning batch with prompts as prefixes and capped scores.
        _attn("attn_cap_prefix_short", 4, 16, 8, 509, 64, mask="prefix", cap=30.0),
        # An encoder's validation pass: bidirectional, capped and biased, head dim 96.
        _attn("attn_cap_slopes_full_eval", 2, 16, 4, 2050, 96, mask="full", cap=30.0, slopes=True, mode="eval"),
        # An fp32 layer, capped and biased.
        _attn("attn_fp32_cap_slopes", 1, 8, 2, 1000, 128, cap=30.0, slopes=True, dtype="fp32"),
        # The smallest call: a prompt of a few tokens, forward only.
        _attn("attn_cap_tiny_eval", 1, 4, 2, 40, 64, mask="prefix", cap=50.0, mode="eval"),
        # A preference step of eight padded pairs.
        _pref("pref_padded", 8, 1024),
        # A large preference step of packed responses, averaged log ratios.
        _pref("pref_packed_ipo", 128, 2048, layout="packed", loss="ipo"),
        # A policy step on a small padded group of responses.
        _policy("policy_padded", 8, 512),
        # A large policy step of packed responses, one advantage per token, averaged per response.
        _policy("policy_packed_1m", 512, 2048, layout="packed", adv="token", reduction="sequence"),
        # Per-token losses of a rollout batch without a KL term.
        _policy("policy_tokens_no_kl", 64, 1024, adv="token", reduction="none", kl=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "pref", "policy"])
    if kind == "pref":
        tokens = _log_int(rng, 16, 8192)
        pairs = _log_int(rng, 1, min(256, (1 << 18) // tokens))
        return _pref("", pairs, tokens, layout=rng.choice(["padded", "packed"]), loss=rng.choice(["sigmoid", "ipo", "hinge"]))
    if kind == "policy":
        tokens = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(512, (1 << 20) // tokens))
        return _policy("", rows, tokens, layout=rng.choice(["padded", "packed"]), adv=rng.choice(["sequence", "token"]),
                       reduction=rng.choice(["token", "sequence", "none"]), kl=rng.choice([0.0, 0.02, 0.2]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    mode = rng.choice(["train", "train", "eval"])
    mask = rng.choice(["causal", "prefix", "docs", "full", "window"])
    cap, slopes = rng.choice([(50.0, False), (20.0, False), (0.0, True), (30.0, True), (100.0, False)])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4])
    dh = rng.choice([64, 96, 128])
    s = _log_int(rng, 16, 1500 if dtype == "fp32" else 4096)
    b = rng.choice([1, 2, 3])
    while b * hq * s * s > 24 * 4096 * 4096:
        s = s * 3 // 4
    return _attn("", b, hq, hkv, s, dh, mask=mask, cap=cap, slopes=slopes, dtype=dtype, mode=mode)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _spans(case, seed):
    """(start, end) int32 (b, s): the keys [start, end) that each query sees."""
    b, s, mask = case["b"], case["s"], case["mask"]
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(s).expand(b, s)
    start, end = torch.zeros(b, s, dtype=torch.int64), i + 1
    if mask == "prefix":  # a prompt of a tenth to a half of each row
        prompt = torch.randint(s // 10, s // 2 + 1, (b, 1), generator=g)
        end = torch.maximum(end, prompt)
    elif mask == "window":
        start = (i - max(1, s // 8)).clamp(min=0)
    elif mask == "docs":
        start, end = start.clone(), end.clone()
        used = s - s // 32  # the tail is padding that sees nothing
        lo, hi = max(1, min(64, s // 8)), max(1, min(2048, s // 2))
        for row in range(b):
            at = 0
            while at < used:
                stop = min(used, at + int(torch.randint(lo, hi + 1, (1,), generator=g)))
                prompt = at + (stop - at) // 3
                start[row, at:stop] = at
                end[row, at:stop] = end[row, at:stop].clamp(min=prompt)
                at = stop
            start[row, used:] = end[row, used:] = used
    return start.to(torch.int32).cuda(), end.to(torch.int32).cuda()


def _offsets(rows, tokens, seed):
    """Where ragged responses begin in rows * tokens packed tokens, a few short or empty ones among them."""
    g = torch.Generator().manual_seed(seed + 1)
    cuts = torch.randint(0, rows * tokens + 1, (rows - 1,), generator=g).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([rows * tokens])]).cuda()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dt=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    if case["kind"] == "attn":
        b, hq, hkv, s, dh = (case[k] for k in ("b", "hq", "hkv", "s", "dh"))
        dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        # Queries of twice the usual size: scores large enough that a cap bends them.
        x = {"q": normal(b, hq, s, dh, std=2.0, dt=dt), "k": normal(b, hkv, s, dh, dt=dt), "v": normal(b, hkv, s, dh, dt=dt)}
        x["d_o"] = normal(b, hq, s, dh, dt=dt) if case["mode"] == "train" else None
        x["slopes"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)).float() if case["slopes"] else None
        x["spans"] = _spans(case, seed) if case["mask"] not in ("causal", "full") else None
        return x
    rows, tokens = 2 * case["pairs"] if case["kind"] == "pref" else case["rows"], case["tokens"]
    x = {"offsets": None, "mask": None}
    if case["layout"] == "packed":
        x["offsets"], shape = _offsets(rows, tokens, seed), (rows * tokens,)
    else:  # left-over positions of a padded batch hold anything, NaN too
        shape = (rows, tokens)
        lens = torch.randint(1, tokens + 1, (rows, 1), generator=torch.Generator().manual_seed(seed)).cuda()
        x["mask"] = torch.arange(tokens, device="cuda")[None, :] < lens
    x["nll"] = normal(*shape).abs() * 1.5
    for name, std in (("ref", 0.3), ("old", 0.15)):
        x[name] = x["nll"] + normal(*shape, std=std)
    if x["mask"] is not None:
        x["ref"].masked_fill_(~x["mask"], math.nan)
    if case["kind"] == "policy":
        x["adv"] = normal(*(shape if case["adv"] == "token" else (rows,)))
        x["ct"] = normal(*shape) if case["reduction"] == "none" else None
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "attn" and case["mode"] == "train":
        for name in ("q", "k", "v"):
            x[name].requires_grad_(True)
    if case["kind"] != "attn":
        x["nll"].requires_grad_(True)
    return {"case": case, **x}


# ---- plain forms --------------------------------------------------------------------------------------------------

def _visible(case, spans, dev):
    j = torch.arange(case["s"], device=dev)
    if spans is not None:
        return ((j >= spans[0][..., None]) & (j < spans[1][..., None]))[:, None]
    return j[None, :] <= j[:, None] if case["mask"] == "causal" else None


def _plain_attention(st):
    c = st["case"]
    b, hq, hkv, s, dh = (c[k] for k in ("b", "hq", "hkv", "s", "dh"))
    scale, g, dt = dh ** -0.5, hq // hkv, st["q"].dtype
    q, k, v = (st[n].detach().float() for n in ("q", "k", "v"))
    qg = q.reshape(b, hkv, g * s, dh)  # the heads of a group one after the other: products and their sums over heads
    z = (qg @ k.transpose(2, 3).contiguous()).reshape(b, hq, s, s) * scale
    t = None
    if c["cap"]:
        t = torch.tanh(z / c["cap"])
        z = c["cap"] * t
    if st["slopes"] is not None:
        i = torch.arange(s, device=z.device, dtype=torch.float32)
        z = z - st["slopes"][:, None, None] * (i[None, :] - i[:, None]).abs()
    see = _visible(c, st["spans"], z.device)
    if see is not None:
        z = torch.where(see, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    pg = p.reshape(b, hkv, g * s, s)
    o = (pg @ v).reshape(b, hq, s, dh)
    if c["mode"] == "eval":
        return {"o": o.to(dt)}
    do = st["d_o"].float().reshape(b, hkv, g * s, dh)
    dp = (do @ v.transpose(2, 3).contiguous()).reshape(b, hq, s, s)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    if t is not None:
        ds = ds * (1 - t * t)
    ds = ds.reshape(b, hkv, g * s, s)
    dq = (ds @ k).reshape(b, hq, s, dh) * scale
    dk = (ds.transpose(2, 3) @ qg) * scale
    dv = pg.transpose(2, 3) @ do
    return {"o": o.to(dt), "d_q": dq.to(dt), "d_k": dk.to(dt), "d_v": dv.to(dt)}


BETA, SMOOTH = 0.1, 0.05


def _row_of(x):
    """The sequence of each packed token, and how many sequences there are."""
    n = x["offsets"].numel() - 1
    at = torch.arange(x["nll"].numel(), device="cuda")
    return torch.searchsorted(x["offsets"], at, right=True) - 1, n


def _row_sums(values, x):
    """Sums over each sequence, in 64 bits (long sums of nearly equal terms)."""
    if x["offsets"] is None:
        return values.double().sum(1)
    row, n = _row_of(x)
    return torch.zeros(n, dtype=torch.float64, device="cuda").index_add_(0, row, values.double())


def _spread(per_row, x):
    """A value of each sequence at each of its tokens."""
    return per_row[:, None].expand_as(x["nll"]) if x["offsets"] is None else per_row[_row_of(x)[0]]


def _plain_pref(st):
    c, nll = st["case"], st["nll"].detach()
    one = torch.ones_like(nll) if st["mask"] is None else st["mask"].float()
    ratio = _row_sums(torch.where(one > 0, st["ref"] - nll, 0.0), st)
    weight = torch.ones_like(ratio)
    if c["loss"] == "ipo":
        weight = 1.0 / _row_sums(one, st).clamp(min=1)
    reward = BETA * ratio * weight
    chosen, rejected = reward.reshape(2, -1)
    d = chosen - rejected
    if c["loss"] == "sigmoid":
        loss = (1 - SMOOTH) * torch.logaddexp(-d, torch.zeros_like(d)) + SMOOTH * torch.logaddexp(d, torch.zeros_like(d))
        slope = SMOOTH - torch.sigmoid(-d)
    elif c["loss"] == "hinge":
        loss, slope = (1 - d).clamp(min=0), -(d < 1).double()
    else:
        h = d / BETA - 1 / (2 * BETA)
        loss, slope = h * h, 2 * h / BETA
    by_row = torch.cat([-slope, slope]) * BETA * weight / d.numel()
    grad = torch.where(one > 0, _spread(by_row.float(), st), 0.0)
    return {"loss": loss.mean().float(), "chosen": chosen.float(), "rejected": rejected.float(), "d_nll": grad}


CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _plain_policy(st):
    c, nll = st["case"], st["nll"].detach()
    keep = torch.ones_like(nll, dtype=torch.bool) if st["mask"] is None else st["mask"]
    adv = st["adv"] if c["adv"] == "token" else _spread(st["adv"], st)
    step = st["old"].double() - nll.double()  # whether a ratio is past its border is told in 64 bits
    ratio = torch.exp(step).float()
    clipped = torch.where(adv > 0, step > math.log1p(CLIP_HIGH), step < math.log1p(-CLIP_LOW)) & (adv != 0)
    edge = torch.where(adv > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)
    loss = -torch.where(clipped, edge, ratio) * adv
    slope = torch.where(clipped, 0.0, ratio * adv)
    kl = torch.zeros_like(loss)
    if c["kl"]:
        gap = nll.double() - st["ref"].double()  # e^x - x - 1 of small x loses its digits in 32 bits
        kl = (torch.expm1(gap) - gap).float()
        loss, slope = loss + c["kl"] * kl, slope + c["kl"] * torch.expm1(gap).float()
    loss, slope, kl = (torch.where(keep, v, 0.0) for v in (loss, slope, kl))
    count = keep.sum().clamp(min=1)
    out = {"kl": (kl.double().sum() / count).float(), "clipped": ((clipped & keep).sum().double() / count).float()}
    if c["reduction"] == "none":
        return {"loss": loss, "d_nll": slope * st["ct"], **out}
    if c["reduction"] == "token":
        return {"loss": (loss.double().sum() / count).float(), "d_nll": slope / count, **out}
    per_row = _row_sums(keep.float(), st)
    weight = 1.0 / (per_row.clamp(min=1) * (per_row > 0).sum().clamp(min=1))
    return {"loss": (_row_sums(loss, st) * weight).sum().float(), "d_nll": slope * _spread(weight.float(), st), **out}


# ---- the framework's calls ----------------------------------------------------------------------------------------

def _own_calls():
    if "mlx-train-perf_amd" not in sys.path:
        sys.path.insert(0, "mlx-train-perf_amd")
    import mlx_train_perf
    import mlx_train_perf.attention

    return mlx_train_perf, mlx_train_perf.attention


def _own_run(st):
    api, attention = _own_calls()
    c = st["case"]
    if c["kind"] == "attn":
        spans = None if st["spans"] is None else attention.SpanMask(start=st["spans"][0], end=st["spans"][1])
        args = {"scale": c["dh"] ** -0.5, "causal": c["mask"] == "causal", "softcap": c["cap"] or None,
                "slopes": st["slopes"], "spans": spans, "validate_segments": False}
        if c["mode"] == "eval":
            with torch.no_grad():
                return {"o": attention.flash_attention(st["q"], st["k"], st["v"], **args)}
        o = attention.flash_attention(st["q"], st["k"], st["v"], **args)
        dq, dk, dv = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["d_o"])
        return {"o": o.detach(), "d_q": dq, "d_k": dk, "d_v": dv}
    rows = {"offsets": st["offsets"], "mask": st["mask"]}
    if c["kind"] == "pref":
        r = api.preference_loss(st["nll"], st["ref"], beta=BETA, kind=c["loss"],
                                label_smoothing=SMOOTH if c["loss"] == "sigmoid" else 0.0, validate_offsets=False, **rows)
        (grad,) = torch.autograd.grad(r.loss, st["nll"])
        return {"loss": r.loss.detach(), "chosen": r.chosen_rewards, "rejected": r.rejected_rewards, "d_nll": grad}
    r = api.policy_loss(st["nll"], st["old"], st["adv"], ref_nll=st["ref"] if c["kl"] else None, kl_coef=c["kl"],
                        clip_low=CLIP_LOW, clip_high=CLIP_HIGH, reduction=c["reduction"], validate_offsets=False, **rows)
    (grad,) = torch.autograd.grad(r.loss, st["nll"], st["ct"])
    return {"loss": r.loss.detach(), "kl": r.kl, "clipped": r.clip_fraction, "d_nll": grad}


def run(state):
    if own:
        return _own_run(state)
    plain = {"attn": _plain_attention, "pref": _plain_pref, "policy": _plain_policy}[state["case"]["kind"]]
    with torch.no_grad():
        return plain(state)


# ---- work ---------------------------------------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of one head over the batch; spans at the mean of their layouts."""
    b, s, mask = case["b"], case["s"], case["mask"]
    if mask == "full":
        return b * s * s
    if mask == "window":
        w = max(1, s // 8) + 1
        return b * (s * w - w * (w - 1) / 2)
    if mask == "prefix":  # the triangle, and the half of the prompt's square above it
        return b * (s * (s + 1) / 2 + (0.3 * s) ** 2 / 2)
    if mask == "docs":  # about 2/3 of a longest document's length, a triangle and the prompt's square
        lo, hi = max(1, min(64, s // 8)), max(1, min(2048, s // 2))
        mean2 = (lo * lo + lo * hi + hi * hi) / 3
        return b * (s - s // 32) / ((lo + hi) / 2) * mean2 * (0.5 + 1 / 18)
    return b * s * (s + 1) / 2


def work(case):
    if case["kind"] == "attn":
        e = 4 if case["dtype"] == "fp32" else 2
        train = case["mode"] == "train"
        q = case["b"] * case["hq"] * case["s"] * case["dh"] * e
        kv = case["b"] * case["hkv"] * case["s"] * case["dh"] * e
        return {"bytes": (4 * q + 4 * kv) if train else (2 * q + 2 * kv),
                "flops": 2.0 * case["dh"] * case["hq"] * _pairs(case) * (7 if train else 2)}
    rows = 2 * case["pairs"] if case["kind"] == "pref" else case["rows"]
    n = rows * case["tokens"]
    each = 12  # nll and another loss read, the gradient written
    if case["kind"] == "policy":
        each += (4 if case["kl"] else 0) + (4 if case["adv"] == "token" else 0) + (8 if case["reduction"] == "none" else 0)
    if case["layout"] == "padded":
        each += 1
    return {"bytes": float(n * each), "flops": 10.0 * n}


# ---- values in 64 bits --------------------------------------------------------------------------------------------

def _exact_attention(case, x):
    b, hq, hkv, s, dh = (case[k] for k in ("b", "hq", "hkv", "s", "dh"))
    scale, cap, train = 1.0 / math.sqrt(dh), case["cap"], case["mode"] == "train"
    q, k, v = (x[n].double() for n in ("q", "k", "v"))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    i = torch.arange(s, device="cuda")
    away = (i[:, None] - i[None, :]).abs().double()
    for row in range(b):
        hidden = torch.zeros(s, s, dtype=torch.bool, device="cuda")
        if x["spans"] is not None:
            hidden = (i[None, :] < x["spans"][0][row][:, None]) | (i[None, :] >= x["spans"][1][row][:, None])
        elif case["mask"] == "causal":
            hidden = i[None, :] > i[:, None]
        for head in range(hq):
            kv = head * hkv // hq
            w = (q[row, head] @ k[row, kv].T).mul_(scale)
            bend = None
            if cap:
                w.div_(cap).tanh_()
                bend = 1 - w ** 2
                w.mul_(cap)
            if x["slopes"] is not None:
                w.sub_(away, alpha=float(x["slopes"][head]))
            w.masked_fill_(hidden, -math.inf)
            p = torch.softmax(w, dim=1).nan_to_num_(nan=0.0)
            o[row, head] = p @ v[row, kv]
            if not train:
                continue
            do = x["d_o"][row, head].double()
            dv[row, kv] += p.T @ do
            ds = p * ((do @ v[row, kv].T) - (do * o[row, head]).sum(1, keepdim=True))
            if bend is not None:
                ds.mul_(bend)
            dq[row, head] = (ds @ k[row, kv]).mul_(scale)
            dk[row, kv] += (ds.T @ q[row, head]).mul_(scale)
    return {"o": o, "d_q": dq, "d_k": dk, "d_v": dv} if train else {"o": o}


def _exact_rows(x):
    """The tokens that count, of each sequence, as indices into the flat tensors."""
    total = x["nll"].numel()
    if x["offsets"] is not None:
        edges = x["offsets"].tolist()
        return [torch.arange(a, z, device="cuda") for a, z in zip(edges, edges[1:])]
    width = x["nll"].shape[1]
    keep = x["mask"].reshape(-1)
    return [r[keep[r]] for r in torch.arange(total, device="cuda").split(width)]


def _exact_pref(case, x):
    nll, ref = x["nll"].double().reshape(-1), x["ref"].double().reshape(-1)
    rows = _exact_rows(x)
    pairs = case["pairs"]
    gap = torch.stack([(nll[r] - ref[r]).sum() for r in rows])
    if case["loss"] == "ipo":
        share = torch.tensor([1.0 / max(1, r.numel()) for r in rows], dtype=torch.float64, device="cuda")
    else:
        share = torch.ones_like(gap)
    gap.requires_grad_(True)
    reward = -BETA * gap * share
    margin = reward[:pairs] - reward[pairs:]
    if case["loss"] == "sigmoid":
        loss = -(1 - SMOOTH) * torch.nn.functional.logsigmoid(margin) - SMOOTH * torch.nn.functional.logsigmoid(-margin)
    elif case["loss"] == "hinge":
        loss = torch.relu(1 - margin)
    else:
        loss = (margin / BETA - 0.5 / BETA) ** 2
    (by_row,) = torch.autograd.grad(loss.mean(), gap)
    grad = torch.zeros_like(nll)
    for r, value in zip(rows, by_row):
        grad[r] = value
    return {"loss": loss.mean().detach(), "chosen": reward[:pairs].detach(), "rejected": reward[pairs:].detach(),
            "d_nll": grad.reshape(x["nll"].shape)}


def _exact_policy(case, x):
    shape = x["nll"].shape
    rows = _exact_rows(x)
    nll = x["nll"].double().reshape(-1).requires_grad_(True)
    old, ref = x["old"].double().reshape(-1), x["ref"].double().reshape(-1)
    counted = torch.cat(rows)
    owner = torch.cat([torch.full_like(r, n) for n, r in enumerate(rows)])
    adv = x["adv"].double().reshape(-1)
    adv = adv[counted] if case["adv"] == "token" else adv[owner]
    ratio = torch.exp(old[counted] - nll[counted])
    inside = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    loss = -torch.minimum(ratio * adv, inside * adv)
    kl = torch.zeros_like(loss)
    if case["kl"]:
        gap = nll[counted] - ref[counted]
        kl = torch.expm1(gap) - gap
    loss = loss + case["kl"] * kl
    n = max(1, counted.numel())
    cut = (inside * adv < ratio * adv).double().sum() / n
    if case["reduction"] == "none":
        total = torch.zeros_like(nll).index_put((counted,), loss)
        (grad,) = torch.autograd.grad(total, nll, x["ct"].double().reshape(-1))
        total = total.reshape(shape)
    else:
        if case["reduction"] == "token":
            total = loss.sum() / n
        else:
            sizes = torch.tensor([max(1, r.numel()) for r in rows], dtype=torch.float64, device="cuda")
            total = (loss / sizes[owner]).sum() / max(1, sum(r.numel() > 0 for r in rows))
        (grad,) = torch.autograd.grad(total, nll)
    return {"loss": total.detach(), "d_nll": grad.reshape(shape), "kl": (kl.sum() / n).detach(), "clipped": cut}


def exact(case, seed):
    x = _inputs(case, seed)
    return {"attn": _exact_attention, "pref": _exact_pref, "policy": _exact_policy}[case["kind"]](case, x)
