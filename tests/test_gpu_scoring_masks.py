"""Which slots of a teacher's list count, by mask and by slot: a call with a mask is the call whose left-out rows are empty."""
from __future__ import annotations

import _scoring as S
import pytest
import torch

from mlx_train_perf import distillation_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k", [1, 7, 64, 65, 128])
@pytest.mark.parametrize("n", [1, 5, 64, 130, 300])
def test_masks(n, k, dtype):
    hidden, hd, _ = S.make(n, 64, 500, dtype=dtype, seed=n)
    hd = S.to(hd, "cuda")
    ids, lp, _ = S.teacher_list(n, 500, k, seed=n)
    lp = lp.nan_to_num(nan=-3.0)
    g = torch.Generator().manual_seed(k)
    for counts in (torch.rand(n, generator=g) < 0.6, torch.ones(n, dtype=torch.bool), torch.zeros(n, dtype=torch.bool)):
        gone = torch.where(counts[:, None], ids, -1)
        for kind in ("forward", "reverse", "jsd"):
            outs = []
            for of, mask in ((gone, None), (ids, counts), (ids, counts.to(torch.uint8)), (ids, counts.to(torch.uint8) * 255), (gone, counts)):
                h = hidden.cuda().requires_grad_(True)
                loss = distillation_loss(h, hd, of.cuda(), lp.cuda(), mask=None if mask is None else mask.cuda(), kind=kind, reduction="none")
                outs.append((loss.detach(), *torch.autograd.grad(loss.sum(), h)))
            live = counts & ((ids >= 0) & (lp != -torch.inf)).any(1)
            assert bool((outs[0][0].cpu()[~live] == 0).all()) and bool((outs[0][1].cpu()[~live] == 0).all())
            assert bool((outs[0][1].cpu()[live] != 0).any(1).all())
            for out in outs[1:]:
                assert all(torch.equal(a, b) for a, b in zip(out, outs[0], strict=True))
