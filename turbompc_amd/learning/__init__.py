"""A learned model upstream of the differentiable solve: its operators (ops) as
HIP kernels behind the C ABI of include/tmpc.h, with their gradients."""
from .ops import decay_attention, decay_attention_step, gated_feed_forward, rms_norm_residual

__all__ = ["decay_attention", "decay_attention_step", "gated_feed_forward", "rms_norm_residual"]
