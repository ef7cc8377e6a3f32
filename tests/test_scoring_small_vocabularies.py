"""Many tokens over a small vocabulary: the logits that a forward with alternatives keeps stay within 256 MiB, in passes."""
from __future__ import annotations

import _scoring as S
import pytest
import torch

from mlx_train_perf import DenseHead, _native, token_logprobs


@pytest.mark.parametrize(("n", "v"), [(500000, 130), (4000000, 16), (300000, 129), (67108864, 1), (16000, 4100)])
def test_workspaces(n, v):
    """256 MiB of logits, a maximum of each group and three partials of each token of a pass (up to 524288 of them)."""
    lib = _native.load()
    for size in (lib.mtp_logprobs_fwd_workspace_bytes, lib.mtp_logprobs_fwd_f32_workspace_bytes):
        for top in (1, min(v, 20)):
            assert 0 < size(n, 64, v, _native.HEAD_DENSE, top, 0) <= 280 << 20


@pytest.mark.parametrize(("n", "v"), [(1, 2 ** 21), (10, 2 ** 21), (32, 2 ** 21 - 1), (60, 2 ** 20), (511, 131000), (200, 300)])
def test_no_more_than_the_tokens_that_there_are(n, v):
    """fp32 hidden dims that no chunk of 4 divides: few tokens, tiles, their logits."""
    lib = _native.load()
    ldz = int(lib.mtp_score_logits_ld(v))
    size = lib.mtp_logprobs_fwd_f32_workspace_bytes(n, 33, v, _native.HEAD_DENSE, 5, 0)
    assert n * ldz * 4 <= size <= n * ldz * 4 + n * (ldz // 128 + 1) * 4 + (8 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize(("n", "v"), [(300001, 130), (600000, 5)])
def test_passes(n, v, dtype):
    """Tokens of every pass against 64 bits."""
    g = torch.Generator().manual_seed(1)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    hidden, w = S.grid(g, n, 16).to(dt).cuda(), (S.grid(g, v, 16) / 2).to(dt).cuda()
    y = torch.randint(0, v, (n,), generator=g).cuda()
    y[::9] = -100
    with torch.no_grad():
        got = token_logprobs(hidden, DenseHead(weight=w), y, top=3, temperature=0.9)
    z = hidden.double() @ w.double().T
    logp = torch.log_softmax(z / 0.9, 1)
    live = y != -100
    off = S.stat(v) + 256 * S.U
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(got.top_ids, torch.where(live[:, None], ids, -1))
    S.within(got.logprobs, torch.where(live, logp.gather(1, y.clamp(min=0)[:, None])[:, 0], 0).cpu(), off, "logprobs")
    S.within(got.entropy, torch.where(live, torch.special.entr(logp.exp()).sum(1), 0).cpu(), off + 128 * S.stat(v), "entropy")
    S.within(got.top_logprobs[live], logp.gather(1, ids)[live].cpu(), off, "top_logprobs")
