"""Targets, teachers' ids and ignore_index of every integer type, over vocabularies past the type's range: the same call as with int64."""
from __future__ import annotations

import _scoring as S
import pytest
import torch

from mlx_train_perf import distillation_loss, token_logprobs
from mlx_train_perf.errors import LossInputError

_TYPES = [torch.int8, torch.uint8, torch.int16, torch.int32]
_IMPLS = ["reference", pytest.param("kernel", marks=pytest.mark.gpu)]


def _call(impl, v):
    hidden, hd, _ = S.make(6, 64, v, dtype="fp32", seed=3)
    device = "cuda" if impl == "kernel" else "cpu"
    return hidden.to(device), S.to(hd, device), device


@pytest.mark.parametrize("impl", _IMPLS)
@pytest.mark.parametrize("v", [101, 300, 500, 32768, 70000])
@pytest.mark.parametrize("dtype", _TYPES)
def test_teacher_ids(dtype, v, impl):
    hidden, hd, device = _call(impl, v)
    ids = torch.tensor([[100, 7, 0], [1, 2, 3], [99, 98, 97], [0, 100, 50], [5, 4, 3], [100, 99, 98]])
    lp = torch.log_softmax(torch.randn(6, 4, generator=torch.Generator().manual_seed(1)), 1)[:, :3].to(device)
    want = distillation_loss(hidden, hd, ids.to(device), lp, reduction="none", impl=impl)
    for validate in (True, False):
        got = distillation_loss(hidden, hd, ids.to(dtype).to(device), lp, reduction="none", impl=impl, validate_ids=validate)
        assert torch.equal(got, want)


@pytest.mark.parametrize("impl", _IMPLS)
@pytest.mark.parametrize("v", [101, 300, 500, 32768, 70000])
@pytest.mark.parametrize("dtype", _TYPES)
def test_targets(dtype, v, impl):
    """156 and -100 are one byte; -100 among the targets is left out where the type holds it."""
    hidden, hd, device = _call(impl, v)
    y = torch.tensor([100, 0, 7, 50, 99, 100])
    if dtype is torch.uint8 and v > 156:
        y[2] = 156
    if dtype is not torch.uint8:
        y[4] = -100
    want = token_logprobs(hidden, hd, y.to(device), top=2, impl=impl)
    for validate in (True, False):
        got = token_logprobs(hidden, hd, y.to(dtype).to(device), top=2, impl=impl, validate_targets=validate)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ids_past_the_vocabulary_are_refused():
    hidden, hd, _ = _call("reference", 90)
    for dtype in _TYPES:
        with pytest.raises(LossInputError, match="below V"):
            distillation_loss(hidden, hd, torch.full((6, 2), 90, dtype=dtype), torch.zeros(6, 2), impl="reference")
        with pytest.raises(LossInputError, match="0 <= t < V"):
            token_logprobs(hidden, hd, torch.full((6,), 90, dtype=dtype), impl="reference")
