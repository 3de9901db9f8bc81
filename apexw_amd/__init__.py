"""apexw_amd: MI355X-native (gfx950) fused optimizer step for ApexW.

Drop-in host API (``ApexW``, ``HybridApexW``, ``ApexMuon``) over hand-written
HIP kernels in ``libapexw_hip.so`` (built in-tree by ``apexw_amd._build``), and
operators that a training program runs around the step: layer norm, expert products,
the clip by the global norm (``apexw_amd.ops``), tokens by expert and the embedding
(``apexw_amd.tokens``), the cross entropy of a linear head (``apexw_amd.head``).
"""

from .optimizer import ApexW
from .muon import ApexMuon
from .hybrid import HybridApexW, partition_parameters_for_hybrid
from .ops import (clip_grad_norm_, clip_grads, expert_matmul, expert_matmul_forward, expert_matmul_rows_grad,
                  expert_matmul_weight_grad, grad_norm, layer_norm, layer_norm_backward, layer_norm_forward,
                  scale_grads)
from .tokens import (ExpertOrder, embedding, embedding_forward, embedding_weight_grad, expert_combine,
                     expert_combine_backward, expert_combine_forward, expert_dispatch, expert_dispatch_backward,
                     expert_dispatch_forward, expert_order)
from .head import linear_cross_entropy, linear_cross_entropy_backward, linear_cross_entropy_forward

__version__ = "0.1.0"
__all__ = ["ApexW", "ApexMuon", "HybridApexW", "partition_parameters_for_hybrid",
           "layer_norm", "layer_norm_forward", "layer_norm_backward",
           "expert_matmul", "expert_matmul_forward", "expert_matmul_rows_grad", "expert_matmul_weight_grad",
           "ExpertOrder", "expert_order", "expert_dispatch", "expert_dispatch_forward", "expert_dispatch_backward",
           "expert_combine", "expert_combine_forward", "expert_combine_backward",
           "embedding", "embedding_forward", "embedding_weight_grad",
           "linear_cross_entropy", "linear_cross_entropy_forward", "linear_cross_entropy_backward",
           "clip_grads", "clip_grad_norm_", "grad_norm", "scale_grads"]
