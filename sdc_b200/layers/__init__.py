"""Operators of a model's layers beside its protected GEMMs.

``head_norm_rotary`` (between the query/key projections and attention),
``low_rank_adapters`` (beside a shared, possibly quantised and protected,
projection) and ``distillation_loss`` (after the last one), each with its
backward pass, on hand-written sm_100a kernels (first derivatives, reverse
mode; others raise). Extensions: the reference has no counterpart. Like the rest
of the package they run on the current CUDA stream, do not synchronise with the
host and have no CPU fallback. Only ``AdapterBatch``, the layout that all
adapters of a batch share, waits for its copy to the device when it is built.

Waits inside the kernels are bounded. Where one runs out (2 s), everything that
its block was to write is NaN, and ``sdc_read_device_error`` of the C ABI tells.
"""
from .adapters import AdapterBatch, low_rank_adapters, low_rank_adapters_
from .distillation import distillation_loss, distillation_loss_and_grad
from .rotary import head_norm_rotary, rotary_table

__all__ = ["AdapterBatch", "distillation_loss", "distillation_loss_and_grad", "head_norm_rotary",
           "low_rank_adapters", "low_rank_adapters_", "rotary_table"]
