"""xspmm_b200 -- B200-native (sm_100a) xSpMM hot path.

Tier-1 BCSR 16x16 block SpMM on tensor cores and the Tier-2 pipeline around it (exact greedy
Jaccard row clustering, CSR row permutation, CSR->BCSR conversion, unpermute), all on the device,
behind the C ABI in include/xspmm_b200.h (libxspmm_b200.so). This package is the Python view of
that ABI, mirroring the reference's API names. Next to the product stand the operators of the layer around
it: layer norm, group norm, dropout and the gated feed-forward block, forward and backward, 8-bit rows and
their product, and the orthogonalised update of a weight (layers.py).
"""
from .api import (  # noqa: F401
    BCSRMatrix,
    CSRMatrix,
    CudaExecutor,
    SpMMPlan,
    SpMMTimings,
    apply_permutation,
    compute_1d_jaccard_clustering,
    csr_to_bcsr,
    spmm,
    unpermute_dense_matrix,
)
from .layers import (  # noqa: F401
    dropout,
    dropout_backward,
    gated_ffn,
    gated_ffn_backward,
    group_norm,
    group_norm_backward,
    layer_norm,
    layer_norm_backward,
    linear_int8,
    orthogonalize,
    quantize_rows,
)
from ._lib import XSpMMError, lib  # noqa: F401
