"""Hidden dims whose rows leave the kernels' 31-bit offsets: bf16 is refused, fp32 takes a core without them."""
from __future__ import annotations

import pytest
import torch

from mlx_train_perf import DenseHead, _native, distillation_loss, token_logprobs

_WIDE = 2 ** 22


def test_few_fp32_tokens_leave_the_kernel_of_31_bit_offsets():
    """Workspaces tell: hidden dims that no chunk of 4 divides never take it."""
    lib = _native.load()
    for size in (lib.mtp_logprobs_fwd_f32_workspace_bytes, lib.mtp_distill_fwd_f32_workspace_bytes):
        few, wide, odd = (size(8, d, 500, _native.HEAD_DENSE, 3, 0) for d in (_WIDE - 4, _WIDE, _WIDE - 3))
        assert wide == odd != few


def test_bf16_is_refused():
    lib = _native.load()
    p = 1 << 20   # a pointer that nothing reads
    for d, code in ((_WIDE, -2), (_WIDE + 64, -2), (_WIDE - 64, -3)):   # (-3: only the workspace is missing)
        head = (p, p, None, None, None)
        assert lib.mtp_logprobs_fwd(*head, p, 4, d, 100, 0, -100, 3, 1.0, p, p, p, p, p, p, None, None, 0, None) == code
        assert lib.mtp_distill_fwd(*head, p, p, None, 4, d, 100, 0, 3, 0, 0.5, 1.0, 0, 1, p, p, p, p, p, p, None, None, 0, None) == code
        back = lib.mtp_logprobs_bwd(p, p, None, None, None, None, p, 4, d, 100, 0, -100, 1.0, p, p, p, None, p, None, p, None, 256, 4, None, 0, None)
        assert back == code
        back = lib.mtp_distill_bwd(p, p, None, None, None, None, 4, d, 100, 0, 3, 1.0, 1, p, p, p, p, p, p, None, p, None, 256, 4, None, 0, None)
        assert back == code


@pytest.mark.gpu
def test_fp32_rows_of_2_22_dims():
    """Every row's first and last dims count, so rows past the 31-bit range do."""
    n, d, v = 3, _WIDE + 4, 130
    w = torch.zeros(v, d, device="cuda")
    g = torch.Generator().manual_seed(1)
    part = (torch.randint(-8, 9, (v, 8), generator=g) / 4).cuda()
    w[:, :4], w[:, -4:] = part[:, :4], part[:, 4:]
    x = (torch.randint(-8, 9, (n, 8), generator=g) / 8).cuda()
    h = torch.zeros(n, d, device="cuda")
    h[:, :4], h[:, -4:] = x[:, :4], x[:, 4:]
    h.requires_grad_(True)
    z = (x.double() @ part.double().T).requires_grad_(True)
    logp = torch.log_softmax(z, 1)
    y = torch.tensor([129, 64, 0], device="cuda")
    head = DenseHead(weight=w, trainable=False)
    got = token_logprobs(h, head, y, top=5)
    want = logp.gather(1, y[:, None])[:, 0]
    assert float((got.logprobs.double() - want).abs().max()) < 1e-5   # 130 terms of 2^-24 and a log-sum-exp below 32
    ids = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :5]
    assert torch.equal(got.top_ids, ids)
    loss = distillation_loss(h, head, ids, got.top_logprobs - 0.1, kind="reverse")
    lt, lq = (got.top_logprobs - 0.1).double(), logp.gather(1, ids)
    rt, rq = 1 - lt.exp().sum(1), 1 - lq.exp().sum(1)
    expect = ((lq.exp() * (lq - lt)).sum(1) + rq * (rq / rt).log()).mean()
    assert float((loss.double() - expect).abs()) < 1e-5
    for a, b in ((got.logprobs.sum(), want.sum()), (loss, expect)):
        (dh,) = torch.autograd.grad(a, h)
        (dz,) = torch.autograd.grad(b, z, retain_graph=True)
        ref = dz @ part.double()
        assert float((torch.cat([dh[:, :4], dh[:, -4:]], 1).double() - ref).abs().max()) < 2e-5
        assert not bool(dh[:, 4:-4].any())
