"""Kernel registry, block-sparse matmul, the coordinate joins and the expert operators."""

from .block_sparse import block_sparse_matmul, block_sparse_matmul_generic
from .experts import (
    ExpertRouting,
    fp8_matmul,
    group_by_expert,
    int8_matmul,
    quantize_blocks,
    quantize_rows,
)
from .join import coordinate_join_hash, coordinate_join_sorted
from .registry import KernelInfo, KernelRegistry

__all__ = [
    "KernelRegistry", "KernelInfo", "block_sparse_matmul", "block_sparse_matmul_generic",
    "coordinate_join_sorted", "coordinate_join_hash", "ExpertRouting", "group_by_expert",
    "int8_matmul", "quantize_rows", "fp8_matmul", "quantize_blocks",
]
