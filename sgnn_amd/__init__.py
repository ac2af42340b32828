"""sgnn_amd — MI355X-native sparse propagation for SGNN / SGC / GCN.

Public surface (mirrors the reference's entry points for this path):
  utils.csr_to_sparse_Tensor, utils.coo_to_sparse_Tensor,
  utils.process_data_with_adjacency, utils.process_data_with_adjacency_high_order,
  nn.SGConv, nn.GCNConv, and the NormAdj handle they share.
Beside them: nn.class_cross_entropy (a label head of any width, without its logits) and nn.save_int8,
  nn.linear_saved_int8, nn.SavedInt8 (layer inputs kept in 8 bits for the backward pass).
"""
from .norm_adj import NormAdj  # noqa: F401
from . import utils, nn  # noqa: F401

__all__ = ["NormAdj", "utils", "nn"]
