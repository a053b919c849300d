"""Operator API: the reference's ``blackwellsparsek`` functions (BlackwellSparseK/python/ops.py) re-pointed
at the sm_100a kernels, plus the operators the reference never exposed (dense GEMM, FP8 GEMM,
block-sparse attention).

Every operator runs through the torch extension ``periodicdent42_b200._C``, which calls the C ABI of
libbsk_sm100.so. There is no CPU fallback: CPU tensors raise ``ValueError`` (as the reference's
``sparse_mm`` does, ops.py:64-65) and a missing extension raises ``ImportError`` on first use.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _capi

from . import workloads as _wl

_C_MOD = None


def _C():
    global _C_MOD
    if _C_MOD is None:
        try:
            from . import _C as mod  # noqa: N814
        except ImportError as e:  # pragma: no cover - exercised on broken installs only
            raise ImportError(
                "periodicdent42_b200._C is not built: run `python -m periodicdent42_b200.build` "
                "(no CPU fallback exists for these operators)") from e
        _C_MOD = mod
    return _C_MOD


def has_cuda_ext() -> bool:
    """Whether the extension imports (the reference's HAS_CUDA_EXT, ops.py:13-22)."""
    try:
        _C()
        return True
    except ImportError:
        return False


KERNEL_BLOCK = 128  # block edge of the sm_100 BSR kernel (tcgen05 M = 128)


# ----------------------------------------------------------------------------------------- BSR SpMM
def sparse_mm(A: torch.Tensor, B: torch.Tensor, block_size: int = 16, autotune: bool = False) -> torch.Tensor:
    """C = A @ B for sparse A (BSR or CSR, fp16, CUDA) and B dense or BSR / CSR (fp16, CUDA); returns fp32 [M, N].

    Same signature and argument checks as the reference (BlackwellSparseK/python/ops.py:25-69).
    ``block_size`` and ``autotune`` keep their meaning for the tile-config dicts
    (``_default_config`` / ``_autotune_config``) but the sm_100 kernel always computes on 128x128 blocks:
    inputs in another layout (CSR, or BSR with another block size) are re-blocked on the device first.
    A B in BSR or CSR layout takes the BSR x BSR kernel (B's blocks looked up per A block, as the reference's
    sparse-B kernel path does, src/sparse_h100_async.cu:105-119); a COO B is rejected as in the reference.
    """
    if not A.is_sparse and A.layout not in (torch.sparse_csr, torch.sparse_bsr):
        raise ValueError("A must be a sparse tensor")
    if B.is_sparse:
        raise ValueError("B must be a dense tensor")
    if A.device != B.device:
        raise ValueError("A and B must be on the same device")
    if not A.is_cuda:
        raise ValueError("CUDA tensors required (CPU not supported)")
    M, K1 = A.shape
    K2, N = B.shape
    if K1 != K2:
        raise ValueError(f"Dimension mismatch: A is {M}×{K1}, B is {K2}×{N}")
    config = _autotune_config(M, N, K1) if autotune else _default_config(M, N, K1)
    A_bsr = _to_kernel_bsr(A)
    if B.dtype != torch.float16:
        raise ValueError("B must be float16")
    if autotune and B.layout == torch.strided:
        _ensure_tuned("spmm_bsr", M, N, K1, lambda: _tune_spmm(A_bsr, B.contiguous(), M))
    if B.layout in (torch.sparse_bsr, torch.sparse_csr):
        if N % KERNEL_BLOCK:
            raise ValueError(f"a sparse B needs N divisible by {KERNEL_BLOCK}, got {N}")
        B_bsr = _to_kernel_bsr(B)
        crow, col = B_bsr.crow_indices(), B_bsr.col_indices()
        if col.numel() == (K2 // KERNEL_BLOCK) * (N // KERNEL_BLOCK):  # every block stored: plain dense product
            Bc = B_bsr.to_dense()
        else:
            return _C().sparse_mm_bsr(A_bsr.crow_indices(), A_bsr.col_indices(), A_bsr.values(), crow, col,
                                      B_bsr.values(), M, N, K1, config["BM"], config["BN"], config["BK"])
    else:
        Bc = B.contiguous()
    dummy = torch.zeros(1, dtype=torch.int32, device=A.device)
    return _C().sparse_mm_bsr(A_bsr.crow_indices(), A_bsr.col_indices(), A_bsr.values(), dummy, dummy, Bc, M, N, K1,
                              config["BM"], config["BN"], config["BK"])


def _ensure_tuned(op: str, M: int, N: int, K: int, tune_fn) -> None:
    """Registers the cached launch configuration of (op, M, N, K) for this device, tuning (and caching) it on
    first use -- the reference's ``autotune=True`` switch, backed by measurements instead of size buckets."""
    from . import autotune as at

    if at.registered(op, M, N, K) is not None:
        return
    cache = at.AutotuneCache()
    e = cache.get(at.device_key(), at.shape_key(op, M, N, K))
    if e is not None:
        at.register(op, M, N, K, int(e["tile"]), int(e["group_m"]))
    else:
        tune_fn()


def _tune_spmm(A_bsr: torch.Tensor, B: torch.Tensor, M: int) -> None:
    from . import autotune as at

    rp = A_bsr.crow_indices().to(torch.int32)
    ci = A_bsr.col_indices().to(torch.int32)
    at.tune_spmm_bsr(rp, ci, A_bsr.values().contiguous(), B, M)


def _to_kernel_bsr(A: torch.Tensor) -> torch.Tensor:
    """BSR with 128x128 blocks, on A's device: CSR / COO input through the device converter; BSR with another
    block size re-blocked through its dense form (the reference left CSR -> BSR unimplemented,
    ops.py:193-197)."""
    if A.layout == torch.sparse_bsr and tuple(A.values().shape[1:]) == (KERNEL_BLOCK, KERNEL_BLOCK):
        return A
    if A.layout not in (torch.sparse_csr, torch.sparse_bsr, torch.sparse_coo):
        raise ValueError(f"Unsupported sparse layout: {A.layout}")
    M, K = A.shape
    if M % KERNEL_BLOCK or K % KERNEL_BLOCK:
        raise ValueError(f"A's shape must be a multiple of {KERNEL_BLOCK} in both dimensions, got {M}x{K}")
    return _convert_csr_to_bsr(A, KERNEL_BLOCK)


def _convert_csr_to_bsr(A_csr: torch.Tensor, block_size: int) -> torch.Tensor:
    """Sparse (CSR / COO / BSR) -> BSR with square blocks, keeping only blocks that hold a nonzero (the
    reference's stub, ops.py:193-197). On CUDA: CSR / COO by the device CSR converter, BSR of another block size
    by the device dense converter on its dense form; on the CPU through torch's dense form."""
    if A_csr.is_cuda and A_csr.dtype in (torch.float16, torch.bfloat16, torch.float32):
        from .utils import convert_to_bsr

        src = A_csr.to_dense() if A_csr.layout == torch.sparse_bsr else A_csr
        return convert_to_bsr(src, block_size, sparsity_threshold=0.0)
    return A_csr.to_dense().to_sparse_bsr((block_size, block_size))


def _default_config(M: int, N: int, K: int) -> dict:
    """Tile configuration dict of the reference (ops.py:200-206); the sm_100 kernel's own tile is
    128 x 256 with 128-wide K slabs, independent of these values."""
    return {"BM": 256, "BN": 128, "BK": 32}


def _autotune_config(M: int, N: int, K: int) -> dict:
    """Size-bucketed tile dict of the reference (ops.py:209-217); informational for the sm_100 kernel."""
    if M < 4096:
        return {"BM": 128, "BN": 64, "BK": 32}
    elif M < 16384:
        return {"BM": 256, "BN": 128, "BK": 32}
    return {"BM": 512, "BN": 256, "BK": 64}


def sparse_mm_benchmark(A: torch.Tensor, B: torch.Tensor,
                        implementations: Tuple[str, ...] = ("blackwellsparsek", "pytorch", "cutlass"),
                        num_iterations: int = 100, warmup_iterations: int = 5) -> dict:
    """Timing dict with the reference's keys (ops.py:123-190): ``blackwellsparsek_ms``,
    ``blackwellsparsek_tflops``, ``pytorch_ms``, ``pytorch_tflops``, ``speedup_vs_pytorch``.
    Times are CUDA-event times on the current stream. FLOPs = 2 * (stored nonzero values) * N: the
    reference's ``2 * A._nnz() * N`` counts blocks, not values, for BSR input. "cutlass" has no
    implementation on this path and is ignored."""
    M, K = A.shape
    _, N = B.shape
    nnz = A.values().numel()
    flops = 2 * nnz * N
    results = {}

    def _time(fn) -> float:
        for _ in range(warmup_iterations):
            fn()
        s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        s.record()
        for _ in range(num_iterations):
            fn()
        e.record()
        torch.cuda.synchronize()
        return s.elapsed_time(e) / num_iterations

    if "blackwellsparsek" in implementations:
        ms = _time(lambda: sparse_mm(A, B))
        results["blackwellsparsek_ms"] = ms
        results["blackwellsparsek_tflops"] = flops / (ms * 1e-3) / 1e12
    if "pytorch" in implementations:
        ms = _time(lambda: torch.sparse.mm(A, B))
        results["pytorch_ms"] = ms
        results["pytorch_tflops"] = flops / (ms * 1e-3) / 1e12
    if "blackwellsparsek_tflops" in results and "pytorch_tflops" in results:
        results["speedup_vs_pytorch"] = results["blackwellsparsek_tflops"] / results["pytorch_tflops"]
    return results


# ----------------------------------------------------------------------------------------- dense GEMM
def gemm(A: torch.Tensor, B: torch.Tensor, out_dtype: torch.dtype = torch.float32, k_range=None,
         split_k: Optional[int] = None, autotune: bool = False) -> torch.Tensor:
    """C = A @ B, fp16 inputs, fp32 output. A [M, K] row-major; B [K, N], column-major preferred
    (``B = Bt.t()`` with Bt contiguous costs nothing; a row-major B is transposed once). ``k_range``
    = (k_begin, k_end) restricts the contraction (split-K shards across ranks). ``split_k``: None = one pass;
    0 = split K across CTA pairs automatically when the output has too few tiles to fill the GPU; n > 0 =
    n splits (partials in a torch-allocated workspace, summed deterministically). ``autotune``: use the tuned
    tile / rasterisation for this shape (measured and cached on first use, see ``autotune``)."""
    _check_cuda_f16(A, B)
    if out_dtype != torch.float32:
        raise ValueError("gemm computes fp16 x fp16 -> fp32; out_dtype must be torch.float32")
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[0]:
        raise ValueError(f"gemm: shape mismatch {tuple(A.shape)} @ {tuple(B.shape)}")
    A = A if A.stride(1) == 1 else A.contiguous()
    Bt = B.t()
    Bt = Bt if Bt.stride(1) == 1 else Bt.contiguous()
    if split_k is not None:
        if k_range is not None:
            raise ValueError("gemm: k_range and split_k are exclusive")
        return _C().gemm_f16f32_splitk(A, Bt, int(split_k))
    kb, ke = (0, -1) if k_range is None else k_range
    if autotune:
        from . import autotune as at

        M, K = A.shape
        kr = (K if ke < 0 else ke) - kb
        _ensure_tuned("gemm_f16f32", M, Bt.shape[0], kr, lambda: at.tune_gemm(M, Bt.shape[0], kr))
    return _C().gemm_f16f32(A, Bt, kb, ke)


def gemm_from_host(A: torch.Tensor, B: torch.Tensor, out: Optional[torch.Tensor] = None, k_chunk: int = 0,
                   device=None, sync: bool = True) -> torch.Tensor:
    """C = A @ B for fp16 operands in HOST memory, fp32 result in host memory, computed on the GPU with the
    K dimension streamed in chunks: the PCIe copy of chunk i+1 overlaps the tensor-core work on chunk i and C
    accumulates on the device (the last chunk by row panels, each panel's C rows copied back while the next
    panel uploads). A [M, K] row-major; B [K, N], column-major preferred
    (``B = Bt.t()``). Use page-locked tensors (``pin_memory=True``) for A, B and ``out``: pageable memory works
    but its copies do not overlap. ``k_chunk``: K per chunk (multiple of 64), 0 = automatic. ``sync``: wait for
    the result (False leaves it pending on the current stream of ``device``)."""
    for t in (A, B):
        if t.is_cuda:
            raise ValueError("gemm_from_host takes host tensors (use gemm for device tensors)")
        if t.dtype != torch.float16:
            raise ValueError("float16 tensors required")
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[0]:
        raise ValueError(f"gemm_from_host: shape mismatch {tuple(A.shape)} @ {tuple(B.shape)}")
    A = A if A.stride(1) == 1 else A.contiguous()
    Bt = B.t()
    Bt = Bt if Bt.stride(1) == 1 else Bt.contiguous()
    M, K = A.shape
    N = Bt.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32, pin_memory=True)
    elif out.is_cuda or out.dtype != torch.float32 or tuple(out.shape) != (M, N) or out.stride(1) != 1:
        raise ValueError(f"out must be a host float32 [{M}, {N}] tensor with unit column stride")
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        ws = torch.empty(_capi.gemm_host_workspace_bytes(M, N, K, k_chunk), dtype=torch.uint8, device=dev)
        stream = torch.cuda.current_stream(dev)
        _capi.gemm_f16f32_host(A, Bt, out, ws, k_chunk, stream)
        if sync:
            stream.synchronize()
    return out


def quantize_e4m3(x: torch.Tensor):
    """Per-tensor amax quantisation to e4m3: (x_q, scale) with scale = amax / 448, x_q = e4m3(x / scale)."""
    return _wl.quantize_e4m3(x)


def gemm_fp8(A_q: torch.Tensor, B_q: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
             out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """D = (A_q @ B_q) * scale_a * scale_b in bf16; A_q e4m3 [M, K] row-major, B_q e4m3 [K, N]
    (column-major preferred), per-tensor fp32 scales. Same semantics as
    ``torch._scaled_mm(A_q, B_q, scale_a, scale_b, out_dtype=torch.bfloat16)``."""
    if not (A_q.is_cuda and B_q.is_cuda):
        raise ValueError("CUDA tensors required (CPU not supported)")
    if out_dtype != torch.bfloat16:
        raise ValueError("gemm_fp8 produces bfloat16")
    Bt = B_q.t()
    Bt = Bt if Bt.stride(1) == 1 else Bt.contiguous()
    A = A_q if A_q.stride(1) == 1 else A_q.contiguous()
    sa = scale_a.to(device=A.device, dtype=torch.float32).reshape(1)
    sb = scale_b.to(device=A.device, dtype=torch.float32).reshape(1)
    return _C().gemm_e4m3(A, Bt, sa, sb)


def _check_cuda_f16(*ts):
    for t in ts:
        if not t.is_cuda:
            raise ValueError("CUDA tensors required (CPU not supported)")
        if t.dtype != torch.float16:
            raise ValueError("float16 tensors required")


# ----------------------------------------------------------------------------------------- attention
def attention_forward(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, scale: Optional[float] = None,
                      block_mask=None, block_size: int = 128, causal: bool = False) -> torch.Tensor:
    """O = softmax(scale * Q K^T) V, optionally restricted to a 128x128 block mask.

    Keeps the reference's signature ``attention_forward(Q, K, V, scale=None)``
    (.archive/src_experiments/blackwell_sparsek/__init__.py:52-109) and its checks (CUDA, 4-D, equal
    shapes, fp16, D in {64, 128}), and also accepts bf16; S must be a multiple of 128.
      block_mask: None (all blocks), a bool tensor [S/128, S/128] shared by every (b, h) or
                  [B, H, S/128, S/128], or a BSR tuple (row_ptr, col_idx) over the B*H*(S/128) block
                  rows (pairs in (b, h) order, within-sequence block indices).
      causal:     mask the diagonal block elementwise-causally; with block_mask=None it also restricts
                  to the lower-triangular blocks (standard causal attention).
    """
    if not (Q.is_cuda and K.is_cuda and V.is_cuda):
        raise ValueError("All tensors must be on CUDA device")
    if Q.dim() != 4 or K.dim() != 4 or V.dim() != 4:
        raise ValueError("All tensors must be 4D [B, H, S, D]")
    Bsz, H, S, D = Q.shape
    if K.shape != (Bsz, H, S, D) or V.shape != (Bsz, H, S, D):
        raise ValueError("Q, K, V must have the same shape")
    if Q.dtype not in (torch.float16, torch.bfloat16) or K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise ValueError("All tensors must be FP16 (torch.float16) or all BF16 (torch.bfloat16)")
    if D not in (64, 128):
        raise ValueError(f"Head dimension must be 64 or 128, got {D}")
    if block_size != 128:
        raise ValueError("block_size must be 128")
    if S % 128:
        raise ValueError(f"Sequence length must be a multiple of 128, got {S}")
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    row_ptr, col_idx = block_mask_to_bsr(block_mask, Bsz, H, S // 128, causal, Q.device)
    if torch.is_grad_enabled() and (Q.requires_grad or K.requires_grad or V.requires_grad):
        return _BlockSparseAttention.apply(Q, K, V, row_ptr, col_idx, float(scale), bool(causal))
    return _C().bsattn_fwd(Q, K, V, row_ptr, col_idx, float(scale), bool(causal))


class _BlockSparseAttention(torch.autograd.Function):
    """Autograd for block-sparse attention on the sm_100 kernels: the forward also keeps the row log-sum-exp,
    the backward recomputes the scores block by block (dK/dV per key block, dQ per query block). Replaces the
    reference's SparseKAttentionFunction (.archive/.../kernels/sparsek.py:100-142), whose CUDA backward was a
    stub."""

    @staticmethod
    def forward(ctx, Q, K, V, row_ptr, col_idx, scale, causal):
        Qc, Kc, Vc = Q.contiguous(), K.contiguous(), V.contiguous()
        B, H, S, _ = Qc.shape
        O = torch.empty_like(Qc)
        lse = torch.empty(B * H * S, dtype=torch.float32, device=Qc.device)
        _capi.bsattn_fwd_ex(Qc, Kc, Vc, O, lse, row_ptr, col_idx, scale, causal)
        ctx.save_for_backward(Qc, Kc, Vc, O, lse, row_ptr, col_idx)
        ctx.scale, ctx.causal = scale, causal
        return O

    @staticmethod
    def backward(ctx, dO):
        Q, K, V, O, lse, row_ptr, col_idx = ctx.saved_tensors
        B, H, S, _ = Q.shape
        col_ptr, row_idx = _capi.bsattn_mask_transpose(row_ptr, col_idx, B * H, S // 128)
        dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
        _capi.bsattn_bwd(dO.to(Q.dtype).contiguous(), Q, K, V, O, lse, dQ, dK, dV, row_ptr, col_idx, col_ptr,
                         row_idx, ctx.scale, ctx.causal)
        return dQ, dK, dV, None, None, None, None


def block_mask_to_bsr(block_mask, B: int, H: int, nqb: int, causal: bool, device):
    """Normalise the accepted block-mask forms to (row_ptr, col_idx) int32 on `device`."""
    if isinstance(block_mask, tuple):
        rp, ci = block_mask
        return rp.to(device=device, dtype=torch.int32), ci.to(device=device, dtype=torch.int32)
    if block_mask is None:
        m = torch.ones(nqb, nqb, dtype=torch.bool)
        if causal:
            m = torch.tril(m)
        block_mask = m
    m = block_mask.to("cpu", torch.bool)
    if m.dim() == 2:
        if m.shape != (nqb, nqb):
            raise ValueError(f"block_mask must be [{nqb}, {nqb}]")
        crow, col = _wl.mask_to_bsr(m)
        P = B * H
        nnz = crow[-1]
        row_ptr = torch.cat([crow[:-1] + p * nnz for p in range(P)] + [torch.tensor([P * nnz])])
        col_idx = col.repeat(P)
    elif m.dim() == 4:
        if m.shape != (B, H, nqb, nqb):
            raise ValueError(f"block_mask must be [{B}, {H}, {nqb}, {nqb}]")
        crow, col = _wl.mask_to_bsr(m.reshape(B * H * nqb, nqb))
        row_ptr, col_idx = crow, col
    else:
        raise ValueError("block_mask must be 2-D or 4-D")
    return row_ptr.to(device=device, dtype=torch.int32), col_idx.to(device=device, dtype=torch.int32)


# ----------------------------------------------------------------------------------------- rotary positions
def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0, device=None):
    """(inv_freq, scale) for :func:`rotary_embedding`: inv_freq[i] = base^(-2i / rotary_dim) as float32
    [rotary_dim / 2] on ``device``, computed in 64 bits, and the factor on the rotated elements.

    ``scaling`` stretches a model trained on ``original_length`` positions by ``factor``:
      None      as trained, scale 1
      "linear"  every frequency divided by factor, scale 1
      "ntk"     base multiplied by factor^(rotary_dim / (rotary_dim - 2)) (the slowest frequency is divided by factor,
                the fastest kept), scale 1
      "yarn"    frequencies that turn more than beta_fast times in original_length kept, those that turn less than
                beta_slow times divided by factor, a linear ramp over i between; scale 0.1 ln(factor) + 1"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not (base > 0 and math.isfinite(base)):
        raise ValueError("base must be positive and finite")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'ntk' or 'yarn'")
    if scaling is not None and not (factor >= 1 and math.isfinite(factor)):
        raise ValueError("factor must be at least 1 and finite")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    scale = 1.0
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("'ntk' scaling needs rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv_freq = base ** -i
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "yarn":
        if original_length < 1 or not beta_fast > beta_slow > 0:
            raise ValueError("'yarn' scaling needs original_length >= 1 and beta_fast > beta_slow > 0")
        if base <= 1:
            raise ValueError("'yarn' scaling needs a base above 1")

        def index_of(turns):  # the (fractional) pair that turns this often in original_length positions
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo = max(math.floor(index_of(beta_fast)), 0)
        hi = min(math.ceil(index_of(beta_slow)), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv_freq = inv_freq * (1 - ramp) + inv_freq / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    return inv_freq.to(torch.float32).to(device if device is not None else "cpu"), scale


def rotary_embedding(Q: torch.Tensor, K: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
                     interleaved: bool = False, scale: float = 1.0):
    """Rotary positions of Q [tokens, heads, dim] and K [tokens, kv_heads, dim] (K may be None) in one launch; returns
    new contiguous (Q', K'). fp16, bf16 or fp32; any strides with a unit inner stride are read in place.

    Pair i of a head -- elements (i, i + r/2), or (2i, 2i+1) with ``interleaved`` -- turns by positions[t] * inv_freq[i]
    and is multiplied by ``scale``; r = 2 * len(inv_freq), elements from r on are copied unchanged (and unscaled).
    positions: int32 or int64 [tokens], any value (angles are exact to fp32 at every one of them); inv_freq: float32 (see
    :func:`rotary_frequencies`). Differentiable (once, in reverse mode) in Q and K."""
    return _C().rotary_embedding(Q, K, positions, inv_freq, interleaved, scale)


# ----------------------------------------------------------------------------------------- paged key/value cache
def kv_cache_append(K: torch.Tensor, V: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
    """Write rows K, V [tokens, kv_heads, dim] (fp16 / bf16, dim 64 or 128) to the slots of a paged cache, in place.

    k_cache, v_cache: contiguous [pages, page size, kv_heads, dim] of K's dtype, or float8_e4m3fn with k_scale, v_scale
    float32 [pages, page size, kv_heads]: then each row is quantised as it is written (scale = max|x| / 448, code =
    e4m3(x / scale); :func:`quantize_e4m3` per row). slots: int32 or int64 [tokens], page * page_size + offset, no slot
    twice in a call; a negative slot marks padding and is skipped. A slot behind the cache is skipped and reported by
    :func:`synchronize_and_check`. Has no gradient: tensors that require one are refused outside torch.no_grad()."""
    _C().kv_cache_append(K, V, k_cache, v_cache, slots, k_scale, v_scale)


def kv_cache_gather(k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                    dtype: torch.dtype = torch.bfloat16, k_scale: Optional[torch.Tensor] = None,
                    v_scale: Optional[torch.Tensor] = None):
    """Read rows back from a paged cache (layout and slots as in :func:`kv_cache_append`; a slot may occur more than
    once): (K, V) contiguous [tokens, kv_heads, dim] in ``dtype`` (float16 or bfloat16; the caches' own unless they hold
    e4m3 codes, which are multiplied by their scales and rounded once). Negative slots read as zeros. Has no gradient, as
    above."""
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("kv_cache_gather: dtype must be torch.float16 or torch.bfloat16")
    return _C().kv_cache_gather(k_cache, v_cache, slots, dtype == torch.float16, k_scale, v_scale)


# ----------------------------------------------------------------------------------------- packed and paged attention
def attention_paged(Q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_seqlens: torch.Tensor, scale: Optional[float] = None,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each sequence's new tokens (one or many) over its cached tokens; returns O like Q.

    Q: [tokens, heads, dim] (fp16 / bf16, dim 64 or 128), the new tokens of all sequences packed: sequence i owns rows
    cu_seqlens[i] .. cu_seqlens[i+1]. Its keys are its first kv_lens[i] cached tokens, the new tokens' own among them
    (:func:`kv_cache_append` first); new token t sees positions <= kv_lens[i] - n_i + t. heads is a multiple of the
    caches' kv_heads: query head h reads kv head h // (heads / kv_heads).
    block_table [batch, width]: page numbers, position p in page block_table[i, p // page_size]; caches and scales as in
    :func:`kv_cache_append`, page size a power of two from 8 to 1024. Index tensors are int32 or int64 (narrowed first;
    a value beyond 32 bits is out of range like any other).
    A row that sees no key is zero, and so are rows behind the last sequence. Stale contents of a page behind its
    sequence's end reach no row, NaN among them; a non-finite value inside a sequence may make rows of it NaN that see it
    with weight zero or are masked for it, fewer than 256 tokens before it. The softmax's weights are rounded to Q's type for
    their product with V; over e4m3 caches they are weight times the value's scale, rounded to fp16. For serving: has no
    gradient, and tensors that require one are refused outside torch.no_grad()."""
    if scale is None:
        scale = Q.shape[-1] ** -0.5 if Q.dim() and Q.shape[-1] else 1.0
    return _C().attention_paged(Q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, scale, k_scale, v_scale)


def attention_varlen(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, cu_seqlens: torch.Tensor,
                     scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
    """Attention over packed sequences of different lengths (each within itself, causal by default); returns O like Q.

    Q [tokens, heads, dim], K and V [tokens, kv_heads, dim] (fp16 / bf16, dim 64 or 128, heads a multiple of kv_heads:
    query head h reads kv head h // (heads / kv_heads)); sequence i owns rows cu_seqlens[i] .. cu_seqlens[i+1]
    (int32 or int64 [batch + 1], starting at 0; any lengths, zero included). Rows behind the last sequence are zero.
    Sequences do not reach one another, non-finite values included; inside one, a non-finite row of V may make rows NaN
    that are masked for it, fewer than 256 tokens before it. Differentiable (once, in reverse mode) in Q, K and V
    (deterministic, no atomics). The softmax's weights and, for the gradients, dS are rounded to Q's type for their products."""
    if scale is None:
        scale = Q.shape[-1] ** -0.5 if Q.dim() and Q.shape[-1] else 1.0
    return _C().attention_varlen(Q, K, V, cu_seqlens, scale, causal)


def synchronize_and_check() -> None:
    """Synchronise and raise if any kernel recorded a device-side error (bounded-wait timeout or an
    out-of-range BSR index)."""
    word = _C().device_error()
    if word:
        kind = {1: "device wait timed out", 2: "out-of-range index"}.get(word & 0xFF, "device error")
        raise RuntimeError(f"{kind} (error word 0x{word:08x})")
