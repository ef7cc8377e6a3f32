"""Preference and policy steps through the trainer adapters on a tiny random-init model (CPU): prompts as prefixes,
capped scores, the losses' contract, and the adapters' refusals."""
from __future__ import annotations

import pytest
import torch

from mlx_train_perf.adapters.transformers_lm import make_policy_loss_fn, make_preference_loss_fn, make_token_nll_fn
from mlx_train_perf.attention import FlashAttentionWrapper, enable_flash_attention, math_attention, prefix_spans
from mlx_train_perf.attention.wrapper import _hf_flash_attention, _resolve_mask
from mlx_train_perf.errors import AdapterError, AttentionInputError
from tests import _preference as P
from tests.test_adapters import _MlxStyleAttention, _tiny_llama


def _batch(rows, t, seed=1):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.stack([torch.full((rows,), 3), torch.randint(4, t, (rows,), generator=g)], dim=1)
    return torch.randint(0, 97, (rows, t + 1), generator=g), lengths


def _plain_nll(model, batch, allowed=None):
    logits = model(input_ids=batch[:, :-1], **({} if allowed is None else {"attention_mask": allowed})).logits.float()
    return torch.nn.functional.cross_entropy(logits.transpose(1, 2), batch[:, 1:], reduction="none")


def _mask(lengths, t):
    steps = torch.arange(1, t + 1)
    return (steps >= lengths[:, :1]) & (steps <= lengths[:, 1:])


@pytest.mark.parametrize("kind", ["sigmoid", "ipo"])
def test_preference_step(kind):
    m, ref = _tiny_llama(seed=0), _tiny_llama(seed=1)
    batch, lengths = _batch(4, 11)
    with torch.no_grad():
        ref_nll = make_token_nll_fn(ref, impl="naive")(ref, batch)
        assert torch.allclose(ref_nll, _plain_nll(ref, batch), atol=1e-5)
    got = make_preference_loss_fn(m, beta=0.5, kind=kind, impl="naive")(m, batch, lengths, ref_nll)
    nll = _plain_nll(m, batch)
    want = P.preference(nll, ref_nll, mask=_mask(lengths, 11), beta=0.5, kind=kind)
    assert abs(float(got.loss.detach()) - float(want[0])) < 1e-4 * max(1.0, abs(float(want[0])))
    assert torch.allclose(got.chosen_rewards.double(), want[1], atol=1e-4)
    got.loss.backward()
    grad = m.model.layers[0].self_attn.q_proj.weight.grad.clone()
    m.zero_grad()
    nll.backward(want[3].float())
    assert torch.allclose(grad, m.model.layers[0].self_attn.q_proj.weight.grad, atol=1e-5)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_step(reduction):
    m, old = _tiny_llama(seed=0), _tiny_llama(seed=2)
    batch, lengths = _batch(3, 10)
    adv = torch.tensor([0.7, -1.2, 0.1])
    with torch.no_grad():
        old_nll = make_token_nll_fn(old, impl="chunked")(old, batch)
    fn = make_policy_loss_fn(m, kl_coef=0.1, clip_low=0.1, clip_high=0.3, reduction=reduction, impl="chunked")
    got = fn(m, batch, lengths, old_nll, adv, old_nll)
    want = P.policy(_plain_nll(m, batch), old_nll, adv, ref_nll=old_nll, mask=_mask(lengths, 10), kl_coef=0.1, clip_low=0.1,
                    clip_high=0.3, reduction=reduction)
    for a, w in zip(got, want):
        assert abs(float(a.detach()) - float(w)) < 1e-5
    got.loss.backward()
    assert m.model.layers[0].self_attn.q_proj.weight.grad.abs().sum() > 0


def test_prompts_as_prefixes_reach_every_layer():
    m = _tiny_llama(head_dim=64)
    batch, _ = _batch(2, 9)
    spans = prefix_spans([4, 0], 9)
    see = torch.zeros(2, 1, 9, 9).masked_fill(~((torch.arange(9) < spans.end[..., None])[:, None]), float("-inf"))
    want = _plain_nll(m, batch, see)    # an additive mask of the same pairs
    with pytest.raises(AdapterError, match="enable_flash_attention"):
        make_token_nll_fn(m, impl="naive")(m, batch, spans)
    enable_flash_attention(m, impl="reference")
    got = make_token_nll_fn(m, impl="naive")(m, batch, spans)
    assert torch.allclose(got, want, atol=1e-4)
    assert not torch.allclose(got[0], make_token_nll_fn(m, impl="naive")(m, batch)[0], atol=1e-3)


def test_a_layers_cap_reaches_the_attention():
    class Layer(torch.nn.Module):
        pass

    layer = Layer()
    layer.config = type("Config", (), {"_mtp_flash_impl": "reference"})()
    g = torch.Generator().manual_seed(0)
    q, k, v = (3 * torch.randn(1, 2, 8, 64, generator=g) for _ in range(3))
    got, _ = _hf_flash_attention(layer, q, k, v, None, 0.5, softcap=2.0)
    want = math_attention(q, k, v, scale=0.5, softcap=2.0).transpose(1, 2)
    assert torch.allclose(got, want, atol=1e-5) and not torch.allclose(got, math_attention(q, k, v, scale=0.5).transpose(1, 2), atol=1e-2)
    stock = _MlxStyleAttention()
    stock.attn_logit_softcapping = 0.3
    w = FlashAttentionWrapper(stock, impl="reference")
    x = 4 * torch.randn(2, 6, 64, generator=g)
    capped = w(x)
    w.softcap = None
    assert not torch.allclose(capped, w(x), atol=1e-3)
    spans = prefix_spans([6, 6], 6)
    assert _resolve_mask(spans) is spans
    assert not torch.allclose(w(x), w(x, mask=spans), atol=1e-3)


def test_refusals_of_the_adapters():
    m = _tiny_llama()
    m.config.final_logit_softcapping = 30.0
    with pytest.raises(AdapterError, match="cap logits"):
        make_preference_loss_fn(m)
    with pytest.raises(AdapterError):
        make_policy_loss_fn(torch.nn.Linear(2, 2))


def test_a_masks_contract_is_checked_once_until_it_is_written():
    sp = prefix_spans([2], 4)
    assert sp.violation() is None
    calls = []
    real = torch.diff
    torch.diff = lambda *a, **k: calls.append(1) or real(*a, **k)
    try:
        assert sp.violation() is None and not calls
        sp.end[0, 3] = 1
        assert "end must not decrease" in sp.violation() and calls
    finally:
        torch.diff = real
    q = torch.zeros(1, 1, 4, 64)
    from mlx_train_perf.attention import flash_attention
    with pytest.raises(AttentionInputError):
        flash_attention(q, q, q, scale=1.0, impl="reference", spans=sp)
    flash_attention(q, q, q, scale=1.0, impl="reference", spans=sp, validate_segments=False)
