"""CPU: a layer or configuration that writes "no cap" as 0 runs without one through the model hooks and adapters, as one
that writes None; `flash_attention` itself takes None alone."""
from __future__ import annotations

import pytest
import torch

from mlx_train_perf.adapters.transformers_lm import make_token_nll_fn
from mlx_train_perf.attention import enable_flash_attention, flash_attention, math_attention, wrapper
from mlx_train_perf.attention.wrapper import FlashAttentionWrapper, _hf_flash_attention
from mlx_train_perf.errors import AttentionInputError
from tests.test_adapters import _tiny_llama
from tests.test_preference_step import _MlxStyleAttention

NONE = [None, 0, 0.0]


@pytest.mark.parametrize("cap", NONE)
def test_a_layer_that_passes_no_cap(cap):
    layer = torch.nn.Module()
    layer.config = type("Config", (), {"_mtp_flash_impl": "reference"})()
    q, k, v = (torch.randn(1, 2, 8, 64, generator=torch.Generator().manual_seed(n)) for n in range(3))
    got, _ = _hf_flash_attention(layer, q, k, v, None, 0.5, softcap=cap)
    assert torch.allclose(got, math_attention(q, k, v, scale=0.5).transpose(1, 2), atol=1e-5)


@pytest.mark.parametrize("cap", NONE)
def test_a_module_that_holds_no_cap(cap):
    stock = _MlxStyleAttention()
    x = torch.randn(2, 6, 64, generator=torch.Generator().manual_seed(0))
    want = FlashAttentionWrapper(stock, impl="reference")(x)
    stock.attn_logit_softcapping = cap
    assert torch.equal(FlashAttentionWrapper(stock, impl="reference")(x), want)


@pytest.mark.parametrize("cap", NONE)
def test_a_configuration_that_writes_no_cap(cap, monkeypatch):
    seen = []
    monkeypatch.setattr(wrapper, "_prewarm", lambda model, **kw: seen.append(kw["softcap"]))
    m = _tiny_llama(head_dim=64)
    m.config.attn_logit_softcapping = cap
    enable_flash_attention(m, seq_len=16)
    assert seen == [None]


@pytest.mark.parametrize("cap", NONE)
def test_a_model_that_does_not_cap_its_logits(cap):
    m = _tiny_llama()
    batch = torch.randint(0, 50, (2, 7), generator=torch.Generator().manual_seed(0))
    want = make_token_nll_fn(m, impl="naive")(m, batch)
    m.config.final_logit_softcapping = cap
    assert torch.equal(make_token_nll_fn(m, impl="naive")(m, batch), want)


def test_a_cap_below_0_is_refused():
    q = torch.zeros(1, 2, 4, 64)
    layer = torch.nn.Module()
    layer.config = type("Config", (), {"_mtp_flash_impl": "reference"})()
    with pytest.raises(AttentionInputError, match="softcap"):
        _hf_flash_attention(layer, q, q, q, None, 0.5, softcap=-1.0)
    with pytest.raises(AttentionInputError, match="softcap"):
        flash_attention(q, q, q, scale=0.5, impl="reference", softcap=0.0)
