"""A learned model upstream of the differentiable solve: its operators (ops, delta_ops, norm_ops) as
HIP kernels behind the C ABI of include/tmpc.h, with their gradients, and a model
of tracking weights from histories that uses them (weights_model)."""
from .delta_ops import delta_attention, delta_attention_step
from .norm_ops import dropout, layer_norm_residual
from .ops import decay_attention, decay_attention_step, gated_feed_forward, rms_norm_residual
from .weights_model import HistoryState, HistoryWeights

__all__ = ["HistoryState", "HistoryWeights", "decay_attention", "decay_attention_step", "delta_attention",
           "delta_attention_step", "dropout", "gated_feed_forward", "layer_norm_residual", "rms_norm_residual"]
