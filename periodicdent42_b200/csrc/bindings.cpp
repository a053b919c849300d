// torch C++ extension periodicdent42_b200._C: the reference's blackwellsparsek._C surface
// (BlackwellSparseK/python/bsk_bindings.cpp:61-158) plus the operators the reference never exposed.
// Each function validates its tensors (TORCH_CHECK -> RuntimeError), allocates the output with torch,
// and calls the C ABI (include/bsk_capi.h) on the current CUDA stream under a device guard.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <limits>

#include "bsk_capi.h"

namespace {

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == BSK_OK, what, " failed (code ", rc, "): ", bsk_last_error());
}

void* stream_of(const torch::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

torch::Tensor as_int32(const torch::Tensor& t) {
  TORCH_CHECK(t.dim() == 1, "index tensors must be 1-D");
  return t.to(torch::kInt32).contiguous();
}

// Reference signature (bsk_bindings.cpp:141-158). B is the dense operand: the reference Python layer
// passes B_dense.reshape(-1, bs, bs) as "B_vals" (ops.py:104-107), whose memory is row-major [K, N];
// B_row_ptr / B_col_idx describe the all-blocks pattern and are not needed. BM/BN/BK are accepted and
// ignored: the sm_100 kernel uses 128 x 256 output tiles.
torch::Tensor sparse_mm_bsr(torch::Tensor A_row_ptr, torch::Tensor A_col_idx, torch::Tensor A_vals,
                            torch::Tensor B_row_ptr, torch::Tensor B_col_idx, torch::Tensor B_vals, int64_t M,
                            int64_t N, int64_t K, int64_t BM, int64_t BN, int64_t BK) {
  (void)BM;
  (void)BN;
  (void)BK;
  TORCH_CHECK(A_row_ptr.is_cuda() && A_col_idx.is_cuda() && A_vals.is_cuda() && B_vals.is_cuda(),
              "sparse_mm_bsr: all tensors must be CUDA tensors");
  TORCH_CHECK(A_vals.scalar_type() == torch::kFloat16, "A_vals must be float16");
  TORCH_CHECK(B_vals.scalar_type() == torch::kFloat16, "B_vals must be float16");
  TORCH_CHECK(A_vals.dim() == 3, "A_vals must be [nnzb, block_rows, block_cols]");
  const at::cuda::CUDAGuard guard(A_vals.device());
  // A sparse B (fewer stored blocks than the full (K/128) x (N/128) grid): B_vals are its 128 x 128 blocks, located
  // through B_row_ptr / B_col_idx (the reference kernel's binary search, src/sparse_h100_async.cu:105-119). With
  // every block present, B_vals is read as the dense row-major K x N operand, as the reference's Python layer
  // passes it (python/ops.py:104-107).
  const int64_t full_b = (K / 128) * (N / 128);
  if (B_vals.dim() == 3 && B_vals.size(1) == 128 && B_vals.size(2) == 128 && B_col_idx.numel() < full_b) {
    TORCH_CHECK(B_row_ptr.is_cuda() && B_col_idx.is_cuda(), "sparse_mm_bsr: B indices must be CUDA tensors");
    TORCH_CHECK(B_row_ptr.numel() == K / 128 + 1, "sparse_mm_bsr: B_row_ptr must have K/128 + 1 entries");
    auto rp = as_int32(A_row_ptr);
    auto ci = as_int32(A_col_idx);
    auto brp = as_int32(B_row_ptr);
    auto bci = as_int32(B_col_idx);
    auto av = A_vals.contiguous();
    auto bv = B_vals.contiguous();
    const int Mb = static_cast<int>(rp.numel() - 1);
    TORCH_CHECK(av.size(1) == 128 && av.size(2) == 128 && Mb * 128 == M, "sparse_mm_bsr: A needs 128x128 blocks");
    auto C = torch::empty({M, N}, A_vals.options().dtype(torch::kFloat32));
    check_rc(bsk_spmm_bsr_bsr_f16f32(rp.data_ptr<int32_t>(), ci.data_ptr<int32_t>(), av.data_ptr(), Mb,
                                     static_cast<int>(ci.numel()), brp.data_ptr<int32_t>(), bci.data_ptr<int32_t>(),
                                     bv.data_ptr(), static_cast<int>(bci.numel()), C.data_ptr<float>(), N,
                                     static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), 0, Mb,
                                     stream_of(C)),
             "bsk_spmm_bsr_bsr_f16f32");
    return C;
  }
  TORCH_CHECK(B_vals.numel() == K * N, "B_vals must hold the dense K x N operand");
  auto rp = as_int32(A_row_ptr);
  auto ci = as_int32(A_col_idx);
  auto vals = A_vals.contiguous();
  auto Bd = B_vals.contiguous();
  const int br = static_cast<int>(vals.size(1)), bc = static_cast<int>(vals.size(2));
  const int Mb = static_cast<int>(rp.numel() - 1);
  TORCH_CHECK(Mb * br == M, "sparse_mm_bsr: row_ptr length does not match M / block rows");
  auto C = torch::empty({M, N}, A_vals.options().dtype(torch::kFloat32));
  check_rc(bsk_spmm_bsr_f16f32(rp.data_ptr<int32_t>(), ci.data_ptr<int32_t>(), vals.data_ptr(), br, bc, Mb,
                               static_cast<int>(ci.numel()), Bd.data_ptr(), N, C.data_ptr<float>(), N,
                               static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), 0, Mb, stream_of(C)),
           "bsk_spmm_bsr_f16f32");
  return C;
}

// C = A @ B with A fp16 [M, K] row-major and B given as Bt = B^T, fp16 [N, K] row-major.
torch::Tensor gemm_f16f32(torch::Tensor A, torch::Tensor Bt, int64_t k_begin, int64_t k_end) {
  TORCH_CHECK(A.is_cuda() && Bt.is_cuda(), "gemm_f16f32: CUDA tensors required");
  TORCH_CHECK(A.scalar_type() == torch::kFloat16 && Bt.scalar_type() == torch::kFloat16, "gemm_f16f32: float16 inputs");
  TORCH_CHECK(A.dim() == 2 && Bt.dim() == 2 && A.size(1) == Bt.size(1), "gemm_f16f32: A [M,K] and Bt [N,K] expected");
  TORCH_CHECK(A.stride(1) == 1 && Bt.stride(1) == 1, "gemm_f16f32: inner dimension must be contiguous");
  const at::cuda::CUDAGuard guard(A.device());
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(0);
  if (k_end < 0) k_end = K;
  auto C = torch::empty({M, N}, A.options().dtype(torch::kFloat32));
  check_rc(bsk_gemm_f16f32(A.data_ptr(), A.stride(0), Bt.data_ptr(), Bt.stride(0), C.data_ptr<float>(), N,
                           static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(k_begin),
                           static_cast<int>(k_end), stream_of(C)),
           "bsk_gemm_f16f32");
  return C;
}

// C = A @ B with K split across CTA pairs (workspace from torch's caching allocator); splits <= 0: automatic.
torch::Tensor gemm_f16f32_splitk(torch::Tensor A, torch::Tensor Bt, int64_t splits) {
  TORCH_CHECK(A.is_cuda() && Bt.is_cuda(), "gemm_f16f32_splitk: CUDA tensors required");
  TORCH_CHECK(A.scalar_type() == torch::kFloat16 && Bt.scalar_type() == torch::kFloat16, "gemm_f16f32_splitk: float16 inputs");
  TORCH_CHECK(A.dim() == 2 && Bt.dim() == 2 && A.size(1) == Bt.size(1), "gemm_f16f32_splitk: A [M,K] and Bt [N,K] expected");
  TORCH_CHECK(A.stride(1) == 1 && Bt.stride(1) == 1, "gemm_f16f32_splitk: inner dimension must be contiguous");
  const at::cuda::CUDAGuard guard(A.device());
  const int64_t M = A.size(0), K = A.size(1), N = Bt.size(0);
  const int64_t need = bsk_gemm_splitk_workspace_bytes(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K),
                                                       static_cast<int>(splits));
  TORCH_CHECK(need >= 0, "bsk_gemm_splitk_workspace_bytes failed: ", bsk_last_error());
  auto ws = torch::empty({need > 0 ? need : 1}, A.options().dtype(torch::kUInt8));
  auto C = torch::empty({M, N}, A.options().dtype(torch::kFloat32));
  check_rc(bsk_gemm_f16f32_splitk(A.data_ptr(), A.stride(0), Bt.data_ptr(), Bt.stride(0), C.data_ptr<float>(), N,
                                  static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), static_cast<int>(splits),
                                  ws.data_ptr(), need, stream_of(C)),
           "bsk_gemm_f16f32_splitk");
  return C;
}

// D (bf16) = (Aq @ Bq) * scale_a * scale_b, Aq e4m3 [M, K], Bq given as Bqt e4m3 [N, K].
torch::Tensor gemm_e4m3(torch::Tensor Aq, torch::Tensor Bqt, torch::Tensor scale_a, torch::Tensor scale_b) {
  TORCH_CHECK(Aq.is_cuda() && Bqt.is_cuda() && scale_a.is_cuda() && scale_b.is_cuda(), "gemm_e4m3: CUDA tensors required");
  TORCH_CHECK(Aq.scalar_type() == at::kFloat8_e4m3fn && Bqt.scalar_type() == at::kFloat8_e4m3fn,
              "gemm_e4m3: float8_e4m3fn inputs");
  TORCH_CHECK(scale_a.scalar_type() == torch::kFloat32 && scale_b.scalar_type() == torch::kFloat32 &&
                  scale_a.numel() == 1 && scale_b.numel() == 1,
              "gemm_e4m3: per-tensor fp32 scales");
  TORCH_CHECK(Aq.dim() == 2 && Bqt.dim() == 2 && Aq.size(1) == Bqt.size(1), "gemm_e4m3: Aq [M,K] and Bqt [N,K] expected");
  TORCH_CHECK(Aq.stride(1) == 1 && Bqt.stride(1) == 1, "gemm_e4m3: inner dimension must be contiguous");
  const at::cuda::CUDAGuard guard(Aq.device());
  const int64_t M = Aq.size(0), K = Aq.size(1), N = Bqt.size(0);
  auto sa = scale_a.contiguous(), sb = scale_b.contiguous();
  auto D = torch::empty({M, N}, Aq.options().dtype(torch::kBFloat16));
  check_rc(bsk_gemm_e4m3_bf16(Aq.data_ptr(), Aq.stride(0), Bqt.data_ptr(), Bqt.stride(0), sa.data_ptr<float>(),
                              sb.data_ptr<float>(), D.data_ptr(), N, static_cast<int>(M), static_cast<int>(N),
                              static_cast<int>(K), stream_of(D)),
           "bsk_gemm_e4m3_bf16");
  return D;
}

// Block-sparse attention forward over a per-(b,h) BSR block mask.
torch::Tensor bsattn_fwd(torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor row_ptr,
                         torch::Tensor col_idx, double scale, bool causal_diag) {
  TORCH_CHECK(Q.is_cuda() && K.is_cuda() && V.is_cuda() && row_ptr.is_cuda() && col_idx.is_cuda(),
              "bsattn_fwd: CUDA tensors required");
  const auto dt = Q.scalar_type();
  TORCH_CHECK((dt == torch::kBFloat16 || dt == torch::kFloat16) && K.scalar_type() == dt && V.scalar_type() == dt,
              "bsattn_fwd: Q, K, V all bfloat16 or all float16");
  TORCH_CHECK(Q.dim() == 4 && K.sizes() == Q.sizes() && V.sizes() == Q.sizes(), "bsattn_fwd: Q, K, V [B,H,S,D] of one shape");
  const at::cuda::CUDAGuard guard(Q.device());
  auto q = Q.contiguous(), k = K.contiguous(), v = V.contiguous();
  auto rp = as_int32(row_ptr), ci = as_int32(col_idx);
  const int B = static_cast<int>(Q.size(0)), H = static_cast<int>(Q.size(1)), S = static_cast<int>(Q.size(2)),
            D = static_cast<int>(Q.size(3));
  TORCH_CHECK(S % 128 == 0, "bsattn_fwd: S must be a multiple of 128");
  TORCH_CHECK(rp.numel() == static_cast<int64_t>(B) * H * (S / 128) + 1, "bsattn_fwd: row_ptr must be [B*H*(S/128)+1]");
  auto O = torch::empty_like(q);
  auto fn = dt == torch::kFloat16 ? bsk_bsattn_fwd_f16 : bsk_bsattn_fwd_bf16;
  check_rc(fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), O.data_ptr(), rp.data_ptr<int32_t>(), ci.data_ptr<int32_t>(), B,
              H, S, D, 128, static_cast<float>(scale), causal_diag ? 1 : 0, 0, B * H, stream_of(O)),
           dt == torch::kFloat16 ? "bsk_bsattn_fwd_f16" : "bsk_bsattn_fwd_bf16");
  return O;
}

// ------------------------------------------------------------------ rotary, paged cache, packed and paged attention
// Argument errors of these operators are ValueErrors (TORCH_CHECK_VALUE), as in the Python layer.
using OptTensor = std::optional<torch::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_cuda(const torch::Tensor& t, const torch::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), op, ": CUDA tensors required (CPU not supported), ", name, " is not one");
  TORCH_CHECK_VALUE(t.device() == like.device(), op, ": ", name, " is on another device");
}

// Derivatives that an operator does not have are errors, never left out silently: forward-mode tangents everywhere ...
void no_tangent(const char* op, std::initializer_list<const torch::Tensor*> ts) {
  for (const auto* t : ts)
    if (t) TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
}
// ... and gradients of the operators for serving.
void no_gradient(const char* op, std::initializer_list<const torch::Tensor*> ts) {
  no_tangent(op, ts);
  if (!at::GradMode::is_enabled()) return;
  for (const auto* t : ts)
    if (t) TORCH_CHECK_VALUE(!t->requires_grad(), op, " has no gradient: call it under torch.no_grad() or with detached tensors");
}
const torch::Tensor* some(const OptTensor& t) { return t ? &*t : nullptr; }

int dtype_code(const torch::Tensor& t, const char* op, bool f32_ok = false) {
  const auto dt = t.scalar_type();
  if (dt == torch::kBFloat16) return 0;
  if (dt == torch::kFloat16) return 1;
  TORCH_CHECK_VALUE(f32_ok && dt == torch::kFloat32, op, ": tensors must be float16 or bfloat16", f32_ok ? " or float32" : "");
  return 2;
}

// [tokens, heads, D] rows that the kernels can read in 16-byte pieces at a token and a head stride; a tensor with
// another inner stride, other alignment or broadcast (stride 0) rows is copied once.
struct Rows {
  torch::Tensor t;
  int64_t ts, hs;
  const void* p() const { return t.data_ptr(); }
};

Rows as_rows(const torch::Tensor& x, bool any_alignment = false) {
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2), e = x.element_size();
  const auto fits = [&](const torch::Tensor& t) {
    if (D > 1 && t.stride(2) != 1) return false;
    const int64_t ts = T > 1 ? t.stride(0) : H * D, hs = H > 1 ? t.stride(1) : D;
    if (any_alignment) return true;
    return ts > 0 && hs > 0 && ts * e % 16 == 0 && hs * e % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  torch::Tensor t = fits(x) ? x : x.clone(at::MemoryFormat::Contiguous);
  return {t, T > 1 ? t.stride(0) : H * D, H > 1 ? t.stride(1) : D};
}

// 1-D (or 2-D) int32 index tensor on `like`'s device. int64 is narrowed to the nearest value: what does not fit stays out of
// every range, so the kernels report it.
torch::Tensor as_index(const torch::Tensor& t, const torch::Tensor& like, const char* op, const char* name, int64_t dim) {
  check_cuda(t, like, op, name);
  TORCH_CHECK_VALUE(t.dim() == dim, op, ": ", name, " must have ", dim, " dimension(s)");
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64, op, ": ", name, " must be int32 or int64");
  if (t.scalar_type() == torch::kInt32) return t.contiguous();
  return t.clamp(-1, std::numeric_limits<int32_t>::max()).to(torch::kInt32).contiguous();
}

int narrow(int64_t v, const char* op, const char* name) {
  TORCH_CHECK_VALUE(v >= 0 && v < (int64_t{1} << 31), op, ": ", name, " (", v, ") out of range");
  return static_cast<int>(v);
}

// Checked positions ([tokens], or with axes [num_axes, tokens]), axes and frequencies of rows Q (and K) [tokens, heads, dim].
struct Angles {
  torch::Tensor pos, axes, freq;
  int num_axes = 1;
  const int32_t* axes_ptr() const { return axes.defined() ? axes.data_ptr<int32_t>() : nullptr; }
};

Angles check_rotary(const char* op, const torch::Tensor& Q, const OptTensor& K, const torch::Tensor& positions,
                    const torch::Tensor& inv_freq, const OptTensor& axes, double scale) {
  check_cuda(Q, Q, op, "Q");
  TORCH_CHECK_VALUE(Q.dim() == 3, op, ": Q must be [tokens, heads, dim]");
  const int64_t T = Q.size(0), D = Q.size(2);
  if (K) {
    check_cuda(*K, Q, op, "K");
    TORCH_CHECK_VALUE(K->dim() == 3 && K->size(0) == T && K->size(2) == D, op, ": K must be [tokens, kv_heads, dim] like Q");
    TORCH_CHECK_VALUE(K->scalar_type() == Q.scalar_type(), op, ": K and Q must have one dtype");
  }
  check_cuda(positions, Q, op, "positions");
  if (axes) {
    TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(0) >= 1 && positions.size(1) == T, op,
                      ": positions must be [number of axes, tokens]");
  } else {
    TORCH_CHECK_VALUE(positions.dim() == 1 && positions.size(0) == T, op, ": positions must be [tokens]");
  }
  TORCH_CHECK_VALUE(positions.scalar_type() == torch::kInt32 || positions.scalar_type() == torch::kInt64, op,
                    ": positions must be int32 or int64");
  check_cuda(inv_freq, Q, op, "inv_freq");
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && inv_freq.scalar_type() == torch::kFloat32, op, ": inv_freq must be 1-D float32");
  TORCH_CHECK_VALUE(inv_freq.size(0) >= 1 && 2 * inv_freq.size(0) <= D, op, ": inv_freq must hold 1 to dim / 2 frequencies");
  TORCH_CHECK_VALUE(scale > -1e30 && scale < 1e30, op, ": scale must be finite and below 1e30 in size");
  TORCH_CHECK_VALUE(D % 2 == 0 && D <= 512, op, ": the head dimension must be even and at most 512, got ", D);
  const at::cuda::CUDAGuard guard(Q.device());
  Angles a;
  a.pos = positions.contiguous();
  a.freq = inv_freq.contiguous();
  if (axes) {
    a.axes = as_index(*axes, Q, op, "axes", 1);
    TORCH_CHECK_VALUE(a.axes.size(0) == inv_freq.size(0), op, ": axes must hold one axis for each frequency");
    a.num_axes = narrow(positions.size(0), op, "number of axes");
  }
  return a;
}

std::tuple<torch::Tensor, OptTensor> rotary(torch::Tensor Q, OptTensor K, torch::Tensor positions, torch::Tensor inv_freq,
                                            OptTensor axes, bool interleaved, double scale, bool backward) {
  const char* op = "rotary_embedding";
  const Angles g = check_rotary(op, Q, K, positions, inv_freq, axes, scale);
  const int code = dtype_code(Q, op, true);
  const int64_t T = Q.size(0), D = Q.size(2);
  const at::cuda::CUDAGuard guard(Q.device());
  const Rows q = as_rows(Q, true);
  auto qo = torch::empty({T, Q.size(1), D}, Q.options());
  Rows k{};
  OptTensor ko;
  if (K) {
    k = as_rows(*K, true);
    ko = torch::empty({T, K->size(1), D}, K->options());
  }
  const int heads = narrow(Q.size(1), op, "heads"), kv_heads = K ? narrow(K->size(1), op, "kv_heads") : 0,
            tokens = narrow(T, op, "tokens"), dim = static_cast<int>(D), turned = static_cast<int>(2 * g.freq.size(0)),
            bytes = static_cast<int>(g.pos.element_size());
  const void* kp = K ? k.p() : nullptr;
  void* kop = K ? ko->data_ptr() : nullptr;
  if (axes)
    check_rc(bsk_rotary_axes(code, q.p(), q.ts, q.hs, qo.data_ptr(), heads, kp, k.ts, k.hs, kop, kv_heads, g.pos.data_ptr(), bytes,
                             g.axes_ptr(), g.num_axes, g.freq.data_ptr<float>(), tokens, dim, turned, interleaved,
                             static_cast<float>(scale), backward, stream_of(Q)),
             "bsk_rotary_axes");
  else
    check_rc(bsk_rotary(code, q.p(), q.ts, q.hs, qo.data_ptr(), heads, kp, k.ts, k.hs, kop, kv_heads, g.pos.data_ptr(), bytes,
                        g.freq.data_ptr<float>(), tokens, dim, turned, interleaved, static_cast<float>(scale), backward,
                        stream_of(Q)),
             "bsk_rotary");
  return {qo, ko};
}

// A head's norm weight: [dim] of the rows' type or float32.
void check_weight(const char* op, const char* name, const torch::Tensor& w, const torch::Tensor& x) {
  check_cuda(w, x, op, name);
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(2), op, ": ", name, " must be [dim]");
  TORCH_CHECK_VALUE(w.scalar_type() == x.scalar_type() || w.scalar_type() == torch::kFloat32, op, ": ", name,
                    " must be of the rows' dtype or float32");
}

void check_norm(const char* op, const torch::Tensor& Q, const OptTensor& K, const torch::Tensor& q_weight, const OptTensor& k_weight,
                double eps) {
  check_weight(op, "q_weight", q_weight, Q);
  TORCH_CHECK_VALUE(K.has_value() == k_weight.has_value(), op, ": K and k_weight go together");
  if (K) {
    check_weight(op, "k_weight", *k_weight, *K);
    TORCH_CHECK_VALUE(k_weight->scalar_type() == q_weight.scalar_type(), op, ": the weights must have one dtype");
  }
  TORCH_CHECK_VALUE(eps >= 1e-30 && eps < 1e30, op, ": eps must be at least 1e-30 and finite");
}

std::tuple<torch::Tensor, OptTensor> norm_rotary_fwd(torch::Tensor Q, OptTensor K, torch::Tensor q_weight, OptTensor k_weight,
                                                     torch::Tensor positions, torch::Tensor inv_freq, OptTensor axes,
                                                     bool interleaved, double scale, double eps) {
  const char* op = "qk_norm_rotary";
  const Angles g = check_rotary(op, Q, K, positions, inv_freq, axes, scale);
  const int code = dtype_code(Q, op, true);
  check_norm(op, Q, K, q_weight, k_weight, eps);
  const at::cuda::CUDAGuard guard(Q.device());
  const int64_t T = Q.size(0), D = Q.size(2);
  const auto qw = q_weight.contiguous(), kw = K ? k_weight->contiguous() : torch::Tensor();
  const Rows q = as_rows(Q, true), k = K ? as_rows(*K, true) : Rows{};
  auto qo = torch::empty({T, Q.size(1), D}, Q.options());
  OptTensor ko;
  if (K) ko = torch::empty({T, K->size(1), D}, K->options());
  check_rc(bsk_qk_norm_rotary(code, q.p(), q.ts, q.hs, qo.data_ptr(), narrow(Q.size(1), op, "heads"), K ? k.p() : nullptr, k.ts, k.hs,
                              K ? ko->data_ptr() : nullptr, K ? narrow(K->size(1), op, "kv_heads") : 0, qw.data_ptr(),
                              K ? kw.data_ptr() : nullptr, qw.scalar_type() == torch::kFloat32, g.pos.data_ptr(),
                              static_cast<int>(g.pos.element_size()), g.axes_ptr(), g.num_axes, g.freq.data_ptr<float>(),
                              narrow(T, op, "tokens"), static_cast<int>(D), static_cast<int>(2 * g.freq.size(0)), interleaved,
                              static_cast<float>(scale), static_cast<float>(eps), stream_of(Q)),
           "bsk_qk_norm_rotary");
  return {qo, ko};
}

// (dQ, dK, dq_weight, dk_weight); a result's gradient that is absent gives none for its input and weight.
variable_list norm_rotary_bwd(OptTensor dQo, OptTensor dKo, torch::Tensor Q, OptTensor K, torch::Tensor q_weight, OptTensor k_weight,
                              torch::Tensor positions, torch::Tensor inv_freq, OptTensor axes, bool interleaved, double scale,
                              double eps) {
  const char* op = "qk_norm_rotary backward";
  const Angles g = check_rotary(op, Q, K, positions, inv_freq, axes, scale);
  const int code = dtype_code(Q, op, true);
  check_norm(op, Q, K, q_weight, k_weight, eps);
  const at::cuda::CUDAGuard guard(Q.device());
  const int64_t T = Q.size(0), D = Q.size(2);
  const bool has_q = dQo.has_value(), has_k = K && dKo.has_value();
  const auto rows_of = [&](const OptTensor& t, const torch::Tensor& like) {
    check_cuda(*t, like, op, "a gradient");
    TORCH_CHECK_VALUE(t->sizes() == like.sizes(), op, ": a gradient differs from its result in shape");
    return as_rows(t->to(like.scalar_type()), true);
  };
  Rows dq{}, dk{}, q{}, k{};
  torch::Tensor dQ, dK, dqw, dkw, qw, kw;
  if (has_q) {
    dq = rows_of(dQo, Q);
    q = as_rows(Q, true);
    dQ = torch::empty({T, Q.size(1), D}, Q.options());
    qw = q_weight.contiguous();
    dqw = torch::empty({D}, q_weight.options());
  }
  if (has_k) {
    dk = rows_of(dKo, *K);
    k = as_rows(*K, true);
    dK = torch::empty({T, K->size(1), D}, K->options());
    kw = k_weight->contiguous();
    dkw = torch::empty({D}, k_weight->options());
  }
  const int tokens = narrow(T, op, "tokens"), heads = has_q ? narrow(Q.size(1), op, "heads") : 0,
            kv_heads = has_k ? narrow(K->size(1), op, "kv_heads") : 0;
  const int64_t need = bsk_qk_norm_rotary_workspace_bytes(tokens, heads, kv_heads, static_cast<int>(D));
  TORCH_CHECK(need >= 0, "bsk_qk_norm_rotary_workspace_bytes failed: ", bsk_last_error());
  auto ws = torch::empty({need}, Q.options().dtype(torch::kUInt8));
  if (has_q && heads == 0) dqw.zero_();
  if (has_k && kv_heads == 0) dkw.zero_();
  const auto at = [](const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  check_rc(bsk_qk_norm_rotary_bwd(code, at(dq.t), dq.ts, dq.hs, at(q.t), q.ts, q.hs, at(dQ), heads, at(dk.t), dk.ts, dk.hs, at(k.t),
                                  k.ts, k.hs, at(dK), kv_heads, at(qw), at(kw), q_weight.scalar_type() == torch::kFloat32, at(dqw),
                                  at(dkw), g.pos.data_ptr(), static_cast<int>(g.pos.element_size()), g.axes_ptr(), g.num_axes,
                                  g.freq.data_ptr<float>(), tokens, static_cast<int>(D), static_cast<int>(2 * g.freq.size(0)),
                                  interleaved, static_cast<float>(scale), static_cast<float>(eps), ws.data_ptr(), need,
                                  stream_of(Q)),
           "bsk_qk_norm_rotary_bwd");
  return {dQ, dK, dqw, dkw};
}

// The caches' checks shared by append, gather and attention: returns whether they hold e4m3 codes.
bool check_caches(const char* op, const torch::Tensor& like, const torch::Tensor& kc, const torch::Tensor& vc,
                  const OptTensor& ks, const OptTensor& vs, at::ScalarType dtype) {
  check_cuda(kc, like, op, "k_cache");
  check_cuda(vc, like, op, "v_cache");
  TORCH_CHECK_VALUE(kc.dim() == 4 && vc.sizes() == kc.sizes(), op, ": caches must be [pages, page size, kv_heads, dim] of one shape");
  TORCH_CHECK_VALUE(kc.is_contiguous() && vc.is_contiguous(), op, ": caches must be contiguous");
  TORCH_CHECK_VALUE(kc.scalar_type() == vc.scalar_type(), op, ": caches must have one dtype");
  TORCH_CHECK_VALUE(kc.size(3) == 64 || kc.size(3) == 128, op, ": head dimension must be 64 or 128, got ", kc.size(3));
  if (kc.scalar_type() != at::kFloat8_e4m3fn) {
    TORCH_CHECK_VALUE(kc.scalar_type() == dtype, op, ": the caches must be float8_e4m3fn or of the rows' dtype");
    TORCH_CHECK_VALUE(!ks && !vs, op, ": k_scale and v_scale go with float8_e4m3fn caches only");
    return false;
  }
  TORCH_CHECK_VALUE(ks && vs, op, ": float8_e4m3fn caches need k_scale and v_scale");
  for (const auto* s : {&*ks, &*vs}) {
    check_cuda(*s, like, op, "k_scale / v_scale");
    TORCH_CHECK_VALUE(s->scalar_type() == torch::kFloat32 && s->is_contiguous() && s->dim() == 3 && s->size(0) == kc.size(0) &&
                          s->size(1) == kc.size(1) && s->size(2) == kc.size(2),
                      op, ": scales must be contiguous float32 [pages, page size, kv_heads]");
  }
  return true;
}

float* scale_ptr(const OptTensor& s) { return s ? s->data_ptr<float>() : nullptr; }

torch::Tensor check_slots(const char* op, const torch::Tensor& slots, const torch::Tensor& like) {
  check_cuda(slots, like, op, "slots");
  TORCH_CHECK_VALUE(slots.dim() == 1 && (slots.scalar_type() == torch::kInt32 || slots.scalar_type() == torch::kInt64), op,
                    ": slots must be 1-D int32 or int64");
  return slots.contiguous();
}

void kv_cache_append(torch::Tensor K, torch::Tensor V, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor slots,
                     OptTensor k_scale, OptTensor v_scale) {
  const char* op = "kv_cache_append";
  check_cuda(K, K, op, "K");
  check_cuda(V, K, op, "V");
  no_gradient(op, {&K, &V, &k_cache, &v_cache, some(k_scale), some(v_scale)});
  TORCH_CHECK_VALUE(K.dim() == 3 && V.sizes() == K.sizes(), op, ": K and V must be [tokens, kv_heads, dim] of one shape");
  const int code = dtype_code(K, op);
  TORCH_CHECK_VALUE(V.scalar_type() == K.scalar_type(), op, ": K and V must have one dtype");
  const bool e4m3 = check_caches(op, K, k_cache, v_cache, k_scale, v_scale, K.scalar_type());
  TORCH_CHECK_VALUE(K.size(1) == k_cache.size(2) && K.size(2) == k_cache.size(3), op, ": K and the caches differ in kv_heads or dim");
  const at::cuda::CUDAGuard guard(K.device());
  const auto at = check_slots(op, slots, K);
  TORCH_CHECK_VALUE(at.size(0) == K.size(0), op, ": slots must be [tokens]");
  const Rows k = as_rows(K), v = as_rows(V);
  check_rc(bsk_kv_cache_append(code, k.p(), k.ts, k.hs, v.p(), v.ts, v.hs, k_cache.data_ptr(), v_cache.data_ptr(), e4m3,
                               scale_ptr(k_scale), scale_ptr(v_scale), at.data_ptr(), static_cast<int>(at.element_size()),
                               narrow(K.size(0), op, "tokens"), narrow(K.size(1), op, "kv_heads"),
                               static_cast<int>(K.size(2)), k_cache.size(0) * k_cache.size(1), stream_of(K)),
           "bsk_kv_cache_append");
  for (const auto& t : {k_cache, v_cache})  // written in place: autograd's version counters notice
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  for (const auto& t : {k_scale, v_scale})
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

std::tuple<torch::Tensor, torch::Tensor> kv_cache_gather(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor slots,
                                                         bool f16, OptTensor k_scale, OptTensor v_scale) {
  const char* op = "kv_cache_gather";
  const auto dtype = f16 ? torch::kFloat16 : torch::kBFloat16;
  const bool e4m3 = check_caches(op, k_cache, k_cache, v_cache, k_scale, v_scale, dtype);
  no_gradient(op, {&k_cache, &v_cache, some(k_scale), some(v_scale)});
  const at::cuda::CUDAGuard guard(k_cache.device());
  const auto at = check_slots(op, slots, k_cache);
  auto K = torch::empty({at.size(0), k_cache.size(2), k_cache.size(3)}, k_cache.options().dtype(dtype));
  auto V = torch::empty_like(K);
  check_rc(bsk_kv_cache_gather(f16, k_cache.data_ptr(), v_cache.data_ptr(), e4m3, scale_ptr(k_scale), scale_ptr(v_scale),
                               at.data_ptr(), static_cast<int>(at.element_size()), K.data_ptr(), V.data_ptr(),
                               narrow(K.size(0), op, "tokens"), narrow(K.size(1), op, "kv_heads"),
                               static_cast<int>(K.size(2)), k_cache.size(0) * k_cache.size(1), stream_of(K)),
           "bsk_kv_cache_gather");
  return {K, V};
}

// (slots, positions, cu_seqlens, kv_lens, free_count) after a step; entries of opened pages are written to block_table.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> kv_cache_plan(
    torch::Tensor kv_lens, torch::Tensor new_lens, torch::Tensor block_table, torch::Tensor free_pages, torch::Tensor free_count,
    int64_t page_size, int64_t tokens) {
  const char* op = "kv_cache_plan";
  check_cuda(block_table, block_table, op, "block_table");
  TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.scalar_type() == torch::kInt32, op, ": block_table must be int32 [batch, width]");
  const int64_t batch = block_table.size(0), width = block_table.size(1);
  TORCH_CHECK_VALUE((width <= 1 || block_table.stride(1) == 1) && (batch <= 1 || block_table.stride(0) >= std::max<int64_t>(width, 1)),
                    op, ": rows of block_table must be contiguous and apart");
  const at::cuda::CUDAGuard guard(block_table.device());
  const auto kv = as_index(kv_lens, block_table, op, "kv_lens", 1), n = as_index(new_lens, block_table, op, "new_lens", 1);
  TORCH_CHECK_VALUE(kv.size(0) == batch && n.size(0) == batch, op, ": kv_lens, new_lens and block_table differ in the batch");
  for (const auto& [t, name] : {std::pair<const torch::Tensor&, const char*>{free_pages, "free_pages"}, {free_count, "free_count"}}) {
    check_cuda(t, block_table, op, name);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.scalar_type() == torch::kInt32, op, ": ", name, " must be 1-D int32");
  }
  TORCH_CHECK_VALUE(free_count.size(0) == 1, op, ": free_count must hold one number");
  TORCH_CHECK_VALUE(page_size >= 1, op, ": page_size must be positive, got ", page_size);
  const int rows = narrow(tokens, op, "tokens");
  const auto pages = free_pages.contiguous();
  const auto i32 = block_table.options();
  // one allocation, whose parts the results are (each allocation costs the host 0.8 us, all else of the call 5)
  const auto buffer = torch::empty({2 * tokens + tokens + 2 * batch + 2}, i32);
  int64_t used = 0;  // 4-byte words
  const auto part = [&](int64_t n, at::ScalarType type) {
    const int64_t bytes = at::elementSize(type);
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), at::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    t.unsafeGetTensorImpl()->set_storage_offset(used * 4 / bytes);
    used += n * bytes / 4;
    return t;
  };
  const auto slots = part(tokens, torch::kInt64);
  const auto positions = part(tokens, torch::kInt32), cu = part(batch + 1, torch::kInt32), lens = part(batch, torch::kInt32),
             left = part(1, torch::kInt32);
  check_rc(bsk_kv_cache_plan(kv.data_ptr<int32_t>(), n.data_ptr<int32_t>(), narrow(batch, op, "batch"), block_table.data_ptr<int32_t>(),
                             batch > 1 ? block_table.stride(0) : width, narrow(width, op, "table width"), pages.data_ptr<int32_t>(),
                             narrow(pages.size(0), op, "free pages"), free_count.data_ptr<int32_t>(), narrow(page_size, op, "page_size"),
                             slots.data_ptr<int64_t>(), positions.data_ptr<int32_t>(), rows, cu.data_ptr<int32_t>(),
                             lens.data_ptr<int32_t>(), left.data_ptr<int32_t>(), stream_of(block_table)),
           "bsk_kv_cache_plan");
  if (!block_table.is_inference()) block_table.unsafeGetTensorImpl()->bump_version();
  return {slots, positions, cu, lens, left};
}

void check_heads(const char* op, const torch::Tensor& Q, int64_t kv_heads, double scale) {
  TORCH_CHECK_VALUE(Q.size(2) == 64 || Q.size(2) == 128, op, ": head dimension must be 64 or 128, got ", Q.size(2));
  TORCH_CHECK_VALUE(kv_heads > 0 && Q.size(1) > 0 && Q.size(1) % kv_heads == 0, op, ": heads (", Q.size(1),
                    ") must be a positive multiple of kv_heads (", kv_heads, ")");
  TORCH_CHECK_VALUE(Q.size(1) / kv_heads <= 128, op, ": at most 128 heads per kv head");
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0.0f && scale < 1e30, op, ": scale must be positive and below 1e30 in float32");
}

// window 0: none (the Python layer's None). Larger ones than any sequence are as good as that.
void check_window(const char* op, int64_t& window, int64_t& sinks, bool causal) {
  TORCH_CHECK_VALUE(window >= 0, op, ": window must be at least 1, got ", window);
  TORCH_CHECK_VALUE(sinks >= 0, op, ": sinks must not be negative, got ", sinks);
  TORCH_CHECK_VALUE(window > 0 || sinks == 0, op, ": sinks go with a window");
  TORCH_CHECK_VALUE(window == 0 || causal, op, ": a window needs causal attention");
  constexpr int64_t kMost = std::numeric_limits<int32_t>::max();
  window = std::min(window, kMost);
  sinks = std::min(sinks, kMost);
}

torch::Tensor attention_paged(torch::Tensor Q, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor block_table,
                              torch::Tensor kv_lens, torch::Tensor cu_seqlens, double scale, OptTensor k_scale,
                              OptTensor v_scale, int64_t window, int64_t sinks) {
  const char* op = "attention_paged";
  check_cuda(Q, Q, op, "Q");
  check_window(op, window, sinks, true);
  no_gradient(op, {&Q, &k_cache, &v_cache, some(k_scale), some(v_scale)});
  TORCH_CHECK_VALUE(Q.dim() == 3, op, ": Q must be [tokens, heads, dim]");
  const int code = dtype_code(Q, op);
  const bool e4m3 = check_caches(op, Q, k_cache, v_cache, k_scale, v_scale, Q.scalar_type());
  TORCH_CHECK_VALUE(Q.size(2) == k_cache.size(3), op, ": Q and the caches differ in the head dimension");
  check_heads(op, Q, k_cache.size(2), scale);
  const int64_t page = k_cache.size(1);
  TORCH_CHECK_VALUE(page >= 8 && page <= 1024 && (page & (page - 1)) == 0, op, ": the page size must be a power of two from 8 to 1024");
  const at::cuda::CUDAGuard guard(Q.device());
  const auto table = as_index(block_table, Q, op, "block_table", 2), lens = as_index(kv_lens, Q, op, "kv_lens", 1),
             cu = as_index(cu_seqlens, Q, op, "cu_seqlens", 1);
  TORCH_CHECK_VALUE(cu.size(0) == lens.size(0) + 1 && table.size(0) == lens.size(0), op,
                    ": block_table [batch, width], kv_lens [batch] and cu_seqlens [batch + 1] differ in the batch");
  const Rows q = as_rows(Q);
  auto O = torch::empty({Q.size(0), Q.size(1), Q.size(2)}, Q.options());
  const int64_t need = bsk_attention_paged_workspace_bytes(
      narrow(Q.size(0), op, "tokens"), narrow(lens.size(0), op, "batch"), static_cast<int>(Q.size(1)),
      static_cast<int>(k_cache.size(2)), static_cast<int>(Q.size(2)), narrow(k_cache.size(0), op, "pages"));
  TORCH_CHECK(need >= 0, "bsk_attention_paged_workspace_bytes failed: ", bsk_last_error());
  torch::Tensor ws;
  if (need > 0) ws = torch::empty({need}, Q.options().dtype(torch::kUInt8));
  const int tokens = narrow(Q.size(0), op, "tokens"), batch = narrow(lens.size(0), op, "batch"), heads = static_cast<int>(Q.size(1)),
            kv_heads = static_cast<int>(k_cache.size(2)), dim = static_cast<int>(Q.size(2)),
            pages = narrow(k_cache.size(0), op, "pages"), width = narrow(table.size(1), op, "table width");
  void* const ws_ptr = need > 0 ? ws.data_ptr() : nullptr;
  if (window > 0)
    check_rc(bsk_attention_paged_window(code, q.p(), q.ts, q.hs, k_cache.data_ptr(), v_cache.data_ptr(), e4m3, scale_ptr(k_scale),
                                        scale_ptr(v_scale), table.data_ptr<int32_t>(), table.size(1), width,
                                        lens.data_ptr<int32_t>(), cu.data_ptr<int32_t>(), O.data_ptr(), tokens, batch, heads,
                                        kv_heads, dim, pages, static_cast<int>(page), static_cast<float>(scale),
                                        static_cast<int>(window), static_cast<int>(sinks), ws_ptr, need, stream_of(Q)),
             "bsk_attention_paged_window");
  else
    check_rc(bsk_attention_paged(code, q.p(), q.ts, q.hs, k_cache.data_ptr(), v_cache.data_ptr(), e4m3, scale_ptr(k_scale),
                                 scale_ptr(v_scale), table.data_ptr<int32_t>(), table.size(1), width, lens.data_ptr<int32_t>(),
                                 cu.data_ptr<int32_t>(), O.data_ptr(), tokens, batch, heads, kv_heads, dim, pages,
                                 static_cast<int>(page), static_cast<float>(scale), ws_ptr, need, stream_of(Q)),
             "bsk_attention_paged");
  return O;
}

torch::Tensor varlen_workspace(const torch::Tensor& Q, int64_t batch, int64_t kv_heads, int64_t window, int64_t sinks, bool backward) {
  const int tokens = static_cast<int>(Q.size(0)), heads = static_cast<int>(Q.size(1)), dim = static_cast<int>(Q.size(2));
  const int64_t n = window > 0 ? bsk_attention_varlen_window_workspace_bytes(tokens, static_cast<int>(batch), heads,
                                                                             static_cast<int>(kv_heads), dim, static_cast<int>(window),
                                                                             static_cast<int>(sinks), backward)
                               : bsk_attention_varlen_workspace_bytes(tokens, static_cast<int>(batch), heads,
                                                                      static_cast<int>(kv_heads), dim, backward);
  TORCH_CHECK(n >= 0, "attention_varlen: workspace size failed: ", bsk_last_error());
  return torch::empty({n}, Q.options().dtype(torch::kUInt8));
}

void check_varlen(const char* op, const torch::Tensor& Q, const torch::Tensor& K, const torch::Tensor& V, double scale) {
  check_cuda(Q, Q, op, "Q");
  check_cuda(K, Q, op, "K");
  check_cuda(V, Q, op, "V");
  TORCH_CHECK_VALUE(Q.dim() == 3 && K.dim() == 3 && V.sizes() == K.sizes() && K.size(0) == Q.size(0) && K.size(2) == Q.size(2), op,
                    ": Q must be [tokens, heads, dim], K and V [tokens, kv_heads, dim]");
  TORCH_CHECK_VALUE(K.scalar_type() == Q.scalar_type() && V.scalar_type() == Q.scalar_type(), op, ": Q, K and V must have one dtype");
  check_heads(op, Q, K.size(1), scale);
  narrow(Q.size(0), op, "tokens");
}

// (O, LSE): the log-sum-exp [tokens, heads] only when asked for (else an empty tensor).
std::tuple<torch::Tensor, torch::Tensor> attention_varlen_fwd(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                                              torch::Tensor cu_seqlens, double scale, bool causal,
                                                              int64_t window, int64_t sinks, bool want_lse) {
  const char* op = "attention_varlen";
  check_varlen(op, Q, K, V, scale);
  const int code = dtype_code(Q, op);
  const at::cuda::CUDAGuard guard(Q.device());
  const auto cu = as_index(cu_seqlens, Q, op, "cu_seqlens", 1);
  TORCH_CHECK_VALUE(cu.size(0) >= 1, op, ": cu_seqlens must be [batch + 1]");
  const int64_t batch = cu.size(0) - 1;
  const Rows q = as_rows(Q), k = as_rows(K), v = as_rows(V);
  auto O = torch::empty({Q.size(0), Q.size(1), Q.size(2)}, Q.options());
  auto lse = torch::empty({want_lse ? Q.size(0) : 0, Q.size(1)}, Q.options().dtype(torch::kFloat32));
  auto ws = varlen_workspace(Q, batch, K.size(1), window, sinks, false);
  float* const lse_ptr = want_lse ? lse.data_ptr<float>() : nullptr;
  const int tokens = static_cast<int>(Q.size(0)), n = narrow(batch, op, "batch"), heads = static_cast<int>(Q.size(1)),
            kv_heads = static_cast<int>(K.size(1)), dim = static_cast<int>(Q.size(2));
  if (window > 0)
    check_rc(bsk_attention_varlen_window_fwd(code, q.p(), q.ts, q.hs, k.p(), k.ts, k.hs, v.p(), v.ts, v.hs, cu.data_ptr<int32_t>(),
                                             O.data_ptr(), lse_ptr, tokens, n, heads, kv_heads, dim, static_cast<float>(scale),
                                             static_cast<int>(window), static_cast<int>(sinks), ws.data_ptr(), ws.numel(),
                                             stream_of(Q)),
             "bsk_attention_varlen_window_fwd");
  else
    check_rc(bsk_attention_varlen_fwd(code, q.p(), q.ts, q.hs, k.p(), k.ts, k.hs, v.p(), v.ts, v.hs, cu.data_ptr<int32_t>(),
                                      O.data_ptr(), lse_ptr, tokens, n, heads, kv_heads, dim, static_cast<float>(scale), causal,
                                      ws.data_ptr(), ws.numel(), stream_of(Q)),
             "bsk_attention_varlen_fwd");
  return {O, lse};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attention_varlen_bwd(torch::Tensor dO, torch::Tensor Q, torch::Tensor K,
                                                                             torch::Tensor V, torch::Tensor O, torch::Tensor lse,
                                                                             torch::Tensor cu_seqlens, double scale, bool causal,
                                                                             int64_t window, int64_t sinks) {
  const char* op = "attention_varlen backward";
  check_varlen(op, Q, K, V, scale);
  const int code = dtype_code(Q, op);
  check_cuda(dO, Q, op, "dO");
  check_cuda(O, Q, op, "O");
  check_cuda(lse, Q, op, "lse");
  TORCH_CHECK_VALUE(dO.sizes() == Q.sizes() && O.sizes() == Q.sizes() && dO.scalar_type() == Q.scalar_type() &&
                        O.scalar_type() == Q.scalar_type() && O.is_contiguous(),
                    op, ": dO and O must be like Q, O contiguous");
  TORCH_CHECK_VALUE(lse.scalar_type() == torch::kFloat32 && lse.is_contiguous() && lse.numel() == Q.size(0) * Q.size(1), op,
                    ": lse must be float32 [tokens, heads]");
  const at::cuda::CUDAGuard guard(Q.device());
  const auto cu = as_index(cu_seqlens, Q, op, "cu_seqlens", 1);
  TORCH_CHECK_VALUE(cu.size(0) >= 1, op, ": cu_seqlens must be [batch + 1]");
  const int64_t batch = cu.size(0) - 1;
  const Rows g = as_rows(dO), q = as_rows(Q), k = as_rows(K), v = as_rows(V);
  auto dQ = torch::empty({Q.size(0), Q.size(1), Q.size(2)}, Q.options());
  auto dK = torch::empty({K.size(0), K.size(1), K.size(2)}, K.options());
  auto dV = torch::empty_like(dK);
  auto ws = varlen_workspace(Q, batch, K.size(1), window, sinks, true);
  const int tokens = static_cast<int>(Q.size(0)), n = narrow(batch, op, "batch"), heads = static_cast<int>(Q.size(1)),
            kv_heads = static_cast<int>(K.size(1)), dim = static_cast<int>(Q.size(2));
  if (window > 0)
    check_rc(bsk_attention_varlen_window_bwd(code, g.p(), g.ts, g.hs, q.p(), q.ts, q.hs, k.p(), k.ts, k.hs, v.p(), v.ts, v.hs,
                                             O.data_ptr(), lse.data_ptr<float>(), cu.data_ptr<int32_t>(), dQ.data_ptr(),
                                             dK.data_ptr(), dV.data_ptr(), tokens, n, heads, kv_heads, dim,
                                             static_cast<float>(scale), static_cast<int>(window), static_cast<int>(sinks),
                                             ws.data_ptr(), ws.numel(), stream_of(Q)),
             "bsk_attention_varlen_window_bwd");
  else
    check_rc(bsk_attention_varlen_bwd(code, g.p(), g.ts, g.hs, q.p(), q.ts, q.hs, k.p(), k.ts, k.hs, v.p(), v.ts, v.hs,
                                      O.data_ptr(), lse.data_ptr<float>(), cu.data_ptr<int32_t>(), dQ.data_ptr(), dK.data_ptr(),
                                      dV.data_ptr(), tokens, n, heads, kv_heads, dim, static_cast<float>(scale), causal,
                                      ws.data_ptr(), ws.numel(), stream_of(Q)),
             "bsk_attention_varlen_bwd");
  return {dQ, dK, dV};
}

// ------------------------------------------------------------------ autograd (no Python between the engine and the kernels)
// Gradients that cannot be differentiated again: an error in the place of a silently wrong second derivative.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)  // (the error hangs on inputs that require a gradient only)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return (*std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is not twice differentiable", grads.size()))(
      std::move(grads));
}

// Packed attention: the forward keeps the rows' log-sum-exp, the backward recomputes the scores.
struct VarlenAttention : public torch::autograd::Function<VarlenAttention> {
  static torch::Tensor forward(AutogradContext* ctx, torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                               torch::Tensor cu_seqlens, double scale, bool causal, int64_t window, int64_t sinks) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [O, lse] = attention_varlen_fwd(Q, K, V, cu_seqlens, scale, causal, window, sinks, true);
    ctx->save_for_backward({Q, K, V, O, lse, cu_seqlens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return O;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(8);
    {
      at::AutoGradMode no_grad(false);
      auto [dQ, dK, dV] = attention_varlen_bwd(grads[0].to(s[0].scalar_type()), s[0], s[1], s[2], s[3], s[4], s[5],
                                               ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(),
                                               ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt());
      if (ctx->needs_input_grad(0)) out[0] = dQ;
      if (ctx->needs_input_grad(1)) out[1] = dK;
      if (ctx->needs_input_grad(2)) out[2] = dV;
    }
    return once(std::move(out), "attention_varlen");
  }
};

torch::Tensor attention_varlen(torch::Tensor Q, torch::Tensor K, torch::Tensor V, torch::Tensor cu_seqlens, double scale,
                               bool causal, int64_t window, int64_t sinks) {
  no_tangent("attention_varlen", {&Q, &K, &V});
  check_window("attention_varlen", window, sinks, causal);
  if (at::GradMode::is_enabled() && (Q.requires_grad() || K.requires_grad() || V.requires_grad()))
    return VarlenAttention::apply(Q, K, V, cu_seqlens, scale, causal, window, sinks);
  return std::get<0>(attention_varlen_fwd(Q, K, V, cu_seqlens, scale, causal, window, sinks, false));
}

// Rotary positions: the gradient of a turn is the turn back.
struct Rotary : public torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, torch::Tensor Q, OptTensor K, torch::Tensor positions,
                               torch::Tensor inv_freq, OptTensor axes, bool interleaved, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [q, k] = rotary(Q, K, positions, inv_freq, axes, interleaved, scale, false);
    ctx->save_for_backward({positions, inv_freq, axes ? *axes : torch::Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    variable_list out{q};
    if (k) out.push_back(*k);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const bool need_q = ctx->needs_input_grad(0) && grads[0].defined();
    const bool need_k = grads.size() > 1 && ctx->needs_input_grad(1) && grads[1].defined();
    variable_list out(7);
    if (need_q || need_k) {
      at::AutoGradMode no_grad(false);
      auto [a, b] = rotary(need_q ? grads[0] : grads[1], need_q && need_k ? OptTensor(grads[1]) : std::nullopt, s[0], s[1],
                           s[2].defined() ? OptTensor(s[2]) : std::nullopt, ctx->saved_data["interleaved"].toBool(),
                           ctx->saved_data["scale"].toDouble(), true);
      if (need_q) out[0] = a;
      if (need_k) out[1] = need_q ? *b : a;
    }
    return once(std::move(out), "rotary_embedding");
  }
};

std::tuple<torch::Tensor, OptTensor> rotary_embedding(torch::Tensor Q, OptTensor K, torch::Tensor positions,
                                                      torch::Tensor inv_freq, bool interleaved, double scale, OptTensor axes) {
  no_tangent("rotary_embedding", {&Q, some(K), &inv_freq});
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK_VALUE(!inv_freq.requires_grad(), "rotary_embedding has no gradient for inv_freq");
    if (Q.requires_grad() || (K && K->requires_grad())) {
      auto out = Rotary::apply(Q, K, positions, inv_freq, axes, interleaved, scale);
      return {out[0], K ? OptTensor(out[1]) : std::nullopt};
    }
  }
  return rotary(Q, K, positions, inv_freq, axes, interleaved, scale, false);
}

// Norm and rotation: the backward takes the inputs again and recomputes the rows' norms.
struct NormRotary : public torch::autograd::Function<NormRotary> {
  static variable_list forward(AutogradContext* ctx, torch::Tensor Q, OptTensor K, torch::Tensor q_weight, OptTensor k_weight,
                               torch::Tensor positions, torch::Tensor inv_freq, OptTensor axes, bool interleaved, double scale,
                               double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [q, k] = norm_rotary_fwd(Q, K, q_weight, k_weight, positions, inv_freq, axes, interleaved, scale, eps);
    ctx->save_for_backward({Q, K ? *K : torch::Tensor(), q_weight, K ? *k_weight : torch::Tensor(), positions, inv_freq,
                            axes ? *axes : torch::Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    variable_list out{q};
    if (k) out.push_back(*k);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto opt = [](const torch::Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    // Which of Q, K, q_weight, k_weight ask for a gradient. needs_input_grad counts the tensors that were given: without K and
    // k_weight, q_weight is the second one.
    const bool with_k = s[1].defined();
    const bool need[4] = {ctx->needs_input_grad(0), with_k && ctx->needs_input_grad(1), ctx->needs_input_grad(with_k ? 2 : 1),
                          with_k && ctx->needs_input_grad(3)};
    // only the halves that something asks for
    const bool need_q = (need[0] || need[2]) && grads[0].defined();
    const bool need_k = grads.size() > 1 && (need[1] || need[3]) && grads[1].defined();
    variable_list out(10);
    if (need_q || need_k) {
      at::AutoGradMode no_grad(false);
      auto d = norm_rotary_bwd(need_q ? OptTensor(grads[0]) : std::nullopt, need_k ? OptTensor(grads[1]) : std::nullopt, s[0],
                               opt(s[1]), s[2], opt(s[3]), s[4], s[5], opt(s[6]), ctx->saved_data["interleaved"].toBool(),
                               ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble());
      for (int i = 0; i < 4; ++i)
        if (need[i]) out[i] = d[i];
    }
    return once(std::move(out), "qk_norm_rotary");
  }
};

std::tuple<torch::Tensor, OptTensor> qk_norm_rotary(torch::Tensor Q, OptTensor K, torch::Tensor q_weight, OptTensor k_weight,
                                                    torch::Tensor positions, torch::Tensor inv_freq, bool interleaved, double scale,
                                                    double eps, OptTensor axes) {
  const char* op = "qk_norm_rotary";
  no_tangent(op, {&Q, some(K), &q_weight, some(k_weight), &inv_freq});
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK_VALUE(!inv_freq.requires_grad(), op, " has no gradient for inv_freq");
    if (Q.requires_grad() || q_weight.requires_grad() || (K && K->requires_grad()) || (k_weight && k_weight->requires_grad())) {
      auto out = NormRotary::apply(Q, K, q_weight, k_weight, positions, inv_freq, axes, interleaved, scale, eps);
      return {out[0], K ? OptTensor(out[1]) : std::nullopt};
    }
  }
  return norm_rotary_fwd(Q, K, q_weight, k_weight, positions, inv_freq, axes, interleaved, scale, eps);
}

int64_t device_error() {
  uint32_t w = 0;
  check_rc(bsk_device_error(&w), "bsk_device_error");
  return static_cast<int64_t>(w);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("sparse_mm_bsr", &sparse_mm_bsr, "BSR x dense SpMM (sm_100a)", py::arg("A_row_ptr"), py::arg("A_col_idx"),
        py::arg("A_vals"), py::arg("B_row_ptr"), py::arg("B_col_idx"), py::arg("B_vals"), py::arg("M"), py::arg("N"),
        py::arg("K"), py::arg("BM") = 256, py::arg("BN") = 128, py::arg("BK") = 32);
  m.def("gemm_f16f32", &gemm_f16f32, "fp16 x fp16 -> fp32 GEMM (sm_100a)", py::arg("A"), py::arg("Bt"),
        py::arg("k_begin") = 0, py::arg("k_end") = -1);
  m.def("gemm_f16f32_splitk", &gemm_f16f32_splitk, "fp16 x fp16 -> fp32 GEMM with split K (sm_100a)", py::arg("A"),
        py::arg("Bt"), py::arg("splits") = 0);
  m.def("gemm_e4m3", &gemm_e4m3, "e4m3 x e4m3 -> bf16 GEMM with per-tensor scales (sm_100a)", py::arg("Aq"),
        py::arg("Bqt"), py::arg("scale_a"), py::arg("scale_b"));
  m.def("bsattn_fwd", &bsattn_fwd, "block-sparse attention forward (sm_100a)", py::arg("Q"), py::arg("K"),
        py::arg("V"), py::arg("row_ptr"), py::arg("col_idx"), py::arg("scale"), py::arg("causal_diag") = true);
  m.def("rotary_embedding", &rotary_embedding, "rotary positions of Q and K, with gradients (sm_100a)", py::arg("Q"),
        py::arg("K"), py::arg("positions"), py::arg("inv_freq"), py::arg("interleaved") = false, py::arg("scale") = 1.0,
        py::arg("axes") = py::none());
  m.def("qk_norm_rotary", &qk_norm_rotary, "norm of each head of Q and K, then rotary positions, with gradients (sm_100a)",
        py::arg("Q"), py::arg("K"), py::arg("q_weight"), py::arg("k_weight"), py::arg("positions"), py::arg("inv_freq"),
        py::arg("interleaved") = false, py::arg("scale") = 1.0, py::arg("eps") = 1e-6, py::arg("axes") = py::none());
  m.def("kv_cache_plan", &kv_cache_plan, "block tables, slots and positions of a serving step (sm_100a)", py::arg("kv_lens"),
        py::arg("new_lens"), py::arg("block_table"), py::arg("free_pages"), py::arg("free_count"), py::arg("page_size"),
        py::arg("tokens"));
  m.def("kv_cache_append", &kv_cache_append, "write rows to a paged key/value cache (sm_100a)", py::arg("K"), py::arg("V"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none());
  m.def("kv_cache_gather", &kv_cache_gather, "read rows of a paged key/value cache (sm_100a)", py::arg("k_cache"),
        py::arg("v_cache"), py::arg("slots"), py::arg("f16"), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none());
  m.def("attention_paged", &attention_paged, "attention of new tokens over a paged cache (sm_100a)", py::arg("Q"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"), py::arg("kv_lens"), py::arg("cu_seqlens"),
        py::arg("scale"), py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(), py::arg("window") = 0,
        py::arg("sinks") = 0);
  m.def("attention_varlen", &attention_varlen, "attention over packed sequences, with gradients (sm_100a)", py::arg("Q"),
        py::arg("K"), py::arg("V"), py::arg("cu_seqlens"), py::arg("scale"), py::arg("causal") = true, py::arg("window") = 0,
        py::arg("sinks") = 0);
  m.def("device_error", &device_error, "read and clear the device error word");
}
