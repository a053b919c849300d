"""periodicdent42_b200 -- B200-native (sm_100a) BlackwellSparseK operator family.

Drop-in for the reference package ``blackwellsparsek`` (BlackwellSparseK/python/__init__.py): same
functions and signatures, backed by hand-written tcgen05/TMA kernels behind a C ABI
(include/bsk_capi.h, libbsk_sm100.so) and the torch extension ``periodicdent42_b200._C``.

    >>> import periodicdent42_b200 as bsk
    >>> C = bsk.sparse_mm(A_bsr, B)          # BSR x dense, fp16 -> fp32
    >>> C = bsk.gemm(A, B)                   # dense fp16 -> fp32
    >>> D = bsk.gemm_fp8(Aq, Bq, sa, sb)     # e4m3 -> bf16, per-tensor scales
    >>> O = bsk.attention_forward(Q, K, V, block_mask=mask, causal=True)
    >>> O = bsk.attention_varlen(Q, K, V, cu_seqlens)             # packed sequences, grouped heads, autograd
    >>> Q, K = bsk.rotary_embedding(Q, K, positions, inv_freq)    # serving: rotary, cache, attention over the cache
    >>> bsk.kv_cache_append(K, V, k_cache, v_cache, slots, k_scale, v_scale)
    >>> O = bsk.attention_paged(Q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, k_scale=k_scale, v_scale=v_scale)
"""

__version__ = "0.9.0+sm100a"

from .ops import (attention_forward, attention_paged, attention_varlen, gemm, gemm_fp8, gemm_from_host, has_cuda_ext,
                  kv_cache_append, kv_cache_gather, quantize_e4m3, rotary_embedding, rotary_frequencies, sparse_mm,
                  sparse_mm_benchmark, synchronize_and_check)
from .utils import convert_to_bsr, get_optimal_block_size, validate_sparse_matrix

__all__ = [
    "sparse_mm",
    "sparse_mm_benchmark",
    "convert_to_bsr",
    "validate_sparse_matrix",
    "get_optimal_block_size",
    "gemm",
    "gemm_fp8",
    "gemm_from_host",
    "quantize_e4m3",
    "attention_forward",
    "attention_paged",
    "attention_varlen",
    "kv_cache_append",
    "kv_cache_gather",
    "rotary_embedding",
    "rotary_frequencies",
    "has_cuda_ext",
    "synchronize_and_check",
    "__version__",
]
