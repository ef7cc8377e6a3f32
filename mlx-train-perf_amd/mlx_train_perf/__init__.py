"""mlx-train-perf hot path for AMD MI355X (gfx950): fused linear cross-entropy, flash attention, the preference
and policy losses over per-token losses, token scoring and distillation.

Same public names as the reference package (src/mlx_train_perf/__init__.py:1-12); tensors are torch
tensors and the kernel impls run hand-written HIP through the C-ABI library libmtp_hip.so.
"""
from mlx_train_perf.core.loss import (
    DenseHead,
    HeadRef,
    QuantizedHead,
    Resolution,
    linear_cross_entropy,
    resolve_impl,
    tied_head,
)
from mlx_train_perf.core.preference import PolicyLoss, PreferenceLoss, policy_loss, preference_loss
from mlx_train_perf.core.scoring import TokenLogprobs, distillation_loss, token_logprobs

__all__ = ["DenseHead", "HeadRef", "PolicyLoss", "PreferenceLoss", "QuantizedHead", "Resolution", "TokenLogprobs",
           "distillation_loss", "linear_cross_entropy", "policy_loss", "preference_loss", "resolve_impl", "tied_head",
           "token_logprobs"]
