"""GPU: scored attention of scores past what fp32 tells apart."""
from __future__ import annotations

import pytest
import torch

from tests import _scored as S

pytestmark = pytest.mark.gpu


def _step(q, k, v, d_o, **kw):
    from mlx_train_perf.attention import flash_attention

    qs = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = flash_attention(*qs, **kw)
    return [o.detach(), *torch.autograd.grad(o, qs, d_o)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["spans", "slopes", "full"])
def test_scores_past_the_digits_of_fp32(form, dtype):
    """Scores of 10^6 to 10^9, of which fp32's steps are 2^-4 to 2^6: a probability formed again from L may come out far above
    1, and must leave neither fp16 (in which the dK/dV pass hands it over) nor fp32."""
    from mlx_train_perf.attention import SpanMask

    hq, hkv, s, dh = 4, 2, 700, 64
    q, k, v, d_o = (x.cuda() for x in S.inputs(1, hq, hkv, s, dh, dtype, 9))
    i = torch.arange(s, device="cuda", dtype=torch.int32)[None]
    kw = {"spans": {"spans": SpanMask(start=(i - 40).clamp(min=0), end=i + 1)}, "slopes": {"slopes": torch.full((hq,), 0.5).cuda()},
          "full": {"slopes": torch.tensor([0.5, -0.5, 300.0, -300.0]).cuda(), "causal": False}}[form]
    for power in (8, 10, 12):
        got = _step(q * 2.0 ** power, k * 2.0 ** power, v, d_o, scale=1.0, **kw)
        for name, x in zip(("o", "dq", "dk", "dv"), got):
            assert torch.isfinite(x).all(), (name, power)
