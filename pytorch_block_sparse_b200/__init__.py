"""B200-native block-sparse Linear engine with the pytorch_block_sparse API."""
from .block_sparse import BlockSparseMatrix, BlockSparseMatrixBase, BlockSparseMatrixEmulator
from .block_sparse_linear import BlockSparseLinear, BlockSparseLinearFunction, PseudoBlockSparseLinear
from .gated_linear import BlockSparseGatedLinear
from .dropout import dropout_residual, new_rng_state, next_rng
from .adapters import AdapterRequests, LowRankAdapters
from .sparse_optimizer import SparseOptimizer
from .util import BlockSparseModelPatcher
from .native import set_default_precision

__all__ = [
    "BlockSparseMatrix",
    "BlockSparseMatrixBase",
    "BlockSparseMatrixEmulator",
    "BlockSparseLinear",
    "BlockSparseLinearFunction",
    "PseudoBlockSparseLinear",
    "BlockSparseGatedLinear",
    "dropout_residual",
    "new_rng_state",
    "next_rng",
    "AdapterRequests",
    "LowRankAdapters",
    "BlockSparseModelPatcher",
    "SparseOptimizer",
    "set_default_precision",
]
