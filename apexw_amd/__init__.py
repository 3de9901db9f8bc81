"""apexw_amd: MI355X-native (gfx950) fused optimizer step for ApexW.

Drop-in host API (``ApexW``, ``HybridApexW``, ``ApexMuon``) over hand-written
HIP kernels in ``libapexw_hip.so`` (built in-tree by ``apexw_amd._build``), and
operators that a training program runs around the step (``apexw_amd.ops``): layer
norm, expert products, the clip by the global norm.
"""

from .optimizer import ApexW
from .muon import ApexMuon
from .hybrid import HybridApexW, partition_parameters_for_hybrid
from .ops import (clip_grad_norm_, clip_grads, expert_matmul, expert_matmul_forward, expert_matmul_rows_grad,
                  expert_matmul_weight_grad, grad_norm, layer_norm, layer_norm_backward, layer_norm_forward,
                  scale_grads)

__version__ = "0.1.0"
__all__ = ["ApexW", "ApexMuon", "HybridApexW", "partition_parameters_for_hybrid",
           "layer_norm", "layer_norm_forward", "layer_norm_backward",
           "expert_matmul", "expert_matmul_forward", "expert_matmul_rows_grad", "expert_matmul_weight_grad",
           "clip_grads", "clip_grad_norm_", "grad_norm", "scale_grads"]
