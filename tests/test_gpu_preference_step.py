"""GPU: the new operators in one step, as a trainer uses them: attention with capped scores over packed prompts and
answers, the fused loss of the answers, and a preference or policy loss; kernels against the reference impls."""
from __future__ import annotations

import pytest
import torch

from tests._scored import rel

pytestmark = pytest.mark.gpu


def _layout(n, docs, seed):
    """One packed row: documents of a prompt and an answer, then padding. PackedMask, prompt lengths, offsets of the
    answers' targets, positions used."""
    from mlx_train_perf.attention import PackedMask

    g = torch.Generator().manual_seed(seed)
    cuts = [0, *sorted(int(x) for x in torch.randperm(n - 40, generator=g)[: docs - 1] + 10), n - 17]
    sid, sst, prompt = (torch.zeros(1, n, dtype=torch.int32) for _ in range(3))
    mask = torch.zeros(n, dtype=torch.bool)
    for d, (a, z) in enumerate(zip(cuts, cuts[1:])):
        sid[0, a:z], sst[0, a:z] = d, a
        p = max(1, (z - a) // 3)
        prompt[0, a:z] = p
        mask[a + p - 1: z - 1] = True   # the inputs whose targets are the answer's tokens
    sid[0, cuts[-1]:], sst[0, cuts[-1]:] = docs, cuts[-1]
    return PackedMask(seg_id=sid.cuda(), seg_start=sst.cuda()), prompt.cuda(), torch.tensor(cuts).cuda(), mask.cuda(), [cuts[-1]]


def _step(impl, x, wq, head, targets, spans, loss_of):
    from mlx_train_perf import DenseHead, linear_cross_entropy
    from mlx_train_perf.attention import flash_attention

    n, h, dh = x.shape[0], 4, 64
    qkv = (x @ wq).view(n, 3, h, dh).permute(1, 2, 0, 3)[:, None]   # strided views
    o = flash_attention(qkv[0], qkv[1], qkv[2], scale=0.3, softcap=6.0, spans=spans, impl="auto" if impl == "auto" else "reference")
    hidden = o.transpose(1, 2).reshape(n, h * dh)
    nll = linear_cross_entropy(hidden, DenseHead(weight=head, trainable=False), targets, reduction="none", validate_targets=False,
                               impl="auto" if impl == "auto" else "chunked")
    return loss_of(nll, impl)


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_one_step(which):
    from mlx_train_perf import policy_loss, preference_loss
    from mlx_train_perf.attention import document_spans

    n, docs, d, v = 700, 6, 256, 1000
    seg, prompt, offsets, mask, used = _layout(n, docs, 1)
    spans = document_spans(seg, prefix=prompt, used=used)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(n, d, generator=g).cuda()
    wq = (torch.randn(d, 3 * d, generator=g) * d ** -0.5).cuda()
    head = (torch.randn(v, d, generator=g) * 0.1).cuda()
    targets = torch.randint(0, v, (n,), generator=g).cuda()
    adv = torch.randn(docs, generator=g).cuda()

    def loss_of(nll, impl):
        frozen = nll.detach() + 0.1 * torch.sin(torch.arange(n, device="cuda"))
        kw = {"offsets": offsets, "mask": mask, "impl": "auto" if impl == "auto" else "reference"}
        if which == "preference":
            return preference_loss(nll, frozen, beta=0.3, **kw)
        return policy_loss(nll, frozen, adv, ref_nll=frozen, kl_coef=0.2, clip_low=0.05, clip_high=0.05, reduction="sequence", **kw)

    out = {}
    for impl in ("auto", "reference"):
        xs, ws = x.clone().requires_grad_(True), wq.clone().requires_grad_(True)
        r = _step(impl, xs, ws, head, targets, spans, loss_of)
        out[impl] = [*(t.detach() for t in r), *torch.autograd.grad(r.loss, (xs, ws))]
        assert not out[impl][-2][used[0]:].any()   # the padding has no part in it
    # fp32 chains of three products and two softmaxes, each within 2e-5 of 64 bits (the operators' own bars), on both sides
    for a, w in zip(out["auto"], out["reference"]):
        assert rel(a, w) <= 2e-4
