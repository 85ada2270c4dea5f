// `_C_gguf` PyTorch extension: the same op schemas the reference registers
// (vllm_gguf_plugin/csrc/torch_bindings.cpp:22-61), implemented by calling the libkq C ABI
// (include/kq_gguf.h).  torch supplies device memory, the current stream and the dispatcher; all
// arithmetic happens behind the C ABI.
//
// Differences from the reference bindings, on purpose:
//   - outputs come from at::empty (the kernels write every element; the reference memsets with new_zeros);
//   - an unsupported GGML type raises instead of silently returning zeros
//     (reference: switch without default, csrc/gguf/gguf_kernel.cu:119-215);
//   - ops of this library's own beside the reference's six: ggml_dequant_mul_mat, ggml_dequantize_rows,
//     ggml_mul_mat_merged, fused_moe_swiglu (no derivative: kaillm_b200/linear.py calls them for plain tensors only);
//   - the operators between the projections of a decode step (qk_norm_rope, qk_norm_rope_store, paged_attention, plan_pages,
//     moe_route), which refuse inputs that require a gradient.
#include <Python.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <utility>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <ATen/core/stack.h>
#include <torch/library.h>

#include "../../include/kq_gguf.h"
#include "kq_direct.h"

namespace {

int kq_dtype_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return KQ_F32;
    case at::kHalf: return KQ_F16;
    case at::kBFloat16: return KQ_BF16;
    default: TORCH_CHECK(false, what, ": dtype must be float32, float16 or bfloat16, got ", t);
  }
}

void check_weight(const at::Tensor& W, const char* fn) {
  TORCH_CHECK(W.is_cuda(), fn, ": W must be a CUDA tensor");
  TORCH_CHECK(W.scalar_type() == at::kByte, fn, ": W must be uint8 GGUF wire bytes");
  TORCH_CHECK(W.is_contiguous(), fn, ": W must be contiguous");
}

at::Tensor mul_mat_impl(bool mmq, const at::Tensor& W, const at::Tensor& X, int64_t type, int64_t row) {
  const char* fn = mmq ? "ggml_mul_mat_a8" : "ggml_mul_mat_vec_a8";
  check_weight(W, fn);
  TORCH_CHECK(X.is_cuda() && X.dim() == 2, fn, ": X must be a 2-D CUDA tensor");
  TORCH_CHECK(X.get_device() == W.get_device(), fn, ": W and X are on different devices");
  TORCH_CHECK(X.stride(1) == 1, fn, ": X must be contiguous along its last dimension");
  const int64_t m = X.size(0), k = X.size(1);
  const int xdt = kq_dtype_of(X.scalar_type(), fn);
  int blk = 0, bytes = 0;
  TORCH_CHECK(kq_block_geometry((int)type, &blk, &bytes) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(k % blk == 0, fn, ": X.size(1)=", k, " is not a multiple of the block size ", blk);
  TORCH_CHECK(row >= 0 && W.numel() >= row * (k / blk) * bytes, fn, ": W holds fewer than `row` rows of K=", k);
  const c10::cuda::CUDAGuard guard(X.device());
  at::Tensor Y = at::empty({m, row}, X.options());
  if (m == 0 || row == 0) return Y;
  const size_t ws = kq_workspace_bytes((int)type, m, row, k);
  at::Tensor scratch = at::empty({(int64_t)ws}, W.options());
  auto stream = at::cuda::getCurrentCUDAStream(X.get_device()).stream();
  auto fnp = mmq ? kq_mul_mat_a8 : kq_mul_mat_vec_a8;
  const int rc = fnp(W.data_ptr(), (int)type, row, k, X.data_ptr(), xdt, m, X.stride(0), Y.data_ptr(), xdt,
                     Y.stride(0), scratch.data_ptr(), ws, (void*)stream);
  TORCH_CHECK(rc == KQ_OK, fn, ": ", kq_last_error());
  return Y;
}

at::Tensor ggml_mul_mat_vec_a8(const at::Tensor& W, const at::Tensor& X, int64_t type, c10::SymInt row) {
  return mul_mat_impl(false, W, X, type, row.expect_int());
}

at::Tensor ggml_mul_mat_a8(const at::Tensor& W, const at::Tensor& X, int64_t type, c10::SymInt row) {
  return mul_mat_impl(true, W, X, type, row.expect_int());
}

// Projections of different types over the same activations (q/k/v of a mixed-type file): one quantization, every shard's
// kernel writes its own columns of the merged output.  mmq[i]: which of the two ops shard i is.
at::Tensor ggml_mul_mat_merged(at::TensorList Ws, const at::Tensor& X, at::IntArrayRef types, at::IntArrayRef mmq) {
  const char* fn = "ggml_mul_mat_merged";
  TORCH_CHECK(!Ws.empty() && Ws.size() == types.size() && Ws.size() == mmq.size(), fn, ": one type and flavour per shard");
  TORCH_CHECK(X.is_cuda() && X.dim() == 2 && X.stride(1) == 1, fn, ": X must be a 2-D CUDA tensor, contiguous along its last dimension");
  const int64_t m = X.size(0), k = X.size(1);
  const int xdt = kq_dtype_of(X.scalar_type(), fn);
  int64_t total = 0, widest = 0;
  size_t ws = 0;
  for (size_t i = 0; i < Ws.size(); ++i) {
    const at::Tensor& W = Ws[i];
    check_weight(W, fn);
    int blk = 0, bytes = 0;
    TORCH_CHECK(kq_block_geometry((int)types[i], &blk, &bytes) == KQ_OK, fn, ": ", kq_last_error());
    TORCH_CHECK(W.dim() == 2 && W.get_device() == X.get_device(), fn, ": W must be 2-D and on X's device");
    TORCH_CHECK(k % blk == 0 && W.size(1) == k / blk * bytes, fn, ": a shard does not hold rows of K=", k);
    total += W.size(0);
    widest = std::max(widest, W.size(0));
  }
  for (size_t i = 0; i < Ws.size(); ++i) ws = std::max(ws, kq_workspace_bytes((int)types[i], m, widest, k));
  const c10::cuda::CUDAGuard guard(X.device());
  at::Tensor Y = at::empty({m, total}, X.options());
  if (m == 0 || total == 0) return Y;
  at::Tensor scratch = at::empty({(int64_t)ws}, X.options().dtype(at::kByte));
  void* stream = (void*)at::cuda::getCurrentCUDAStream(X.get_device()).stream();
  TORCH_CHECK(kq_prepare_q8((int)types[0], widest, k, X.data_ptr(), xdt, m, X.stride(0), scratch.data_ptr(), ws, 0, stream) == KQ_OK, fn, ": ", kq_last_error());
  int64_t col = 0;
  for (size_t i = 0; i < Ws.size(); ++i) {
    const int64_t n = Ws[i].size(0);
    if (n == 0) continue;
    void* y = static_cast<char*>(Y.data_ptr()) + col * (int64_t)Y.element_size();
    TORCH_CHECK(kq_mul_mat_prepared(Ws[i].data_ptr(), (int)types[i], n, k, m, y, xdt, total, (int)mmq[i], scratch.data_ptr(), ws, stream) == KQ_OK,
                fn, ": ", kq_last_error());
    col += n;
  }
  return Y;
}

at::Tensor ggml_dequantize(const at::Tensor& W, int64_t type, c10::SymInt m_, c10::SymInt n_,
                           std::optional<at::ScalarType> dtype) {
  const char* fn = "ggml_dequantize";
  check_weight(W, fn);
  const int64_t m = m_.expect_int(), n = n_.expect_int();
  const at::ScalarType dt = dtype.value_or(at::kHalf);
  const int odt = kq_dtype_of(dt, fn);
  int blk = 0, bytes = 0;
  TORCH_CHECK(kq_block_geometry((int)type, &blk, &bytes) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(m >= 0 && n >= 0 && (m * n) % blk == 0, fn, ": m*n must be a multiple of the block size ", blk);
  TORCH_CHECK(W.numel() >= (m * n) / blk * bytes, fn, ": W holds fewer than m*n weights");
  const c10::cuda::CUDAGuard guard(W.device());
  at::Tensor DW = at::empty({m, n}, W.options().dtype(dt));
  if (m * n == 0) return DW;
  auto stream = at::cuda::getCurrentCUDAStream(W.get_device()).stream();
  const int rc = kq_dequantize(W.data_ptr(), (int)type, m * n, DW.data_ptr(), odt, (void*)stream);
  TORCH_CHECK(rc == KQ_OK, fn, ": ", kq_last_error());
  return DW;
}

// X @ dequantize(W)^T: one kernel where it covers the call, otherwise the two steps
at::Tensor ggml_dequant_mul_mat(const at::Tensor& W, const at::Tensor& X, int64_t type, c10::SymInt row_) {
  const char* fn = "ggml_dequant_mul_mat";
  const int64_t row = row_.expect_int();
  int blk = 0, bytes = 0;
  TORCH_CHECK(kq_block_geometry((int)type, &blk, &bytes) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(W.dim() == 2, fn, ": W must be 2-D");
  const bool half = X.scalar_type() == at::kHalf || X.scalar_type() == at::kBFloat16;
  if (half && W.is_cuda() && X.is_cuda() && W.get_device() == X.get_device() && W.scalar_type() == at::kByte && W.is_contiguous() &&
      X.dim() == 2 && X.stride(1) == 1 && W.size(0) == row && X.size(1) % blk == 0 && W.size(1) == X.size(1) / blk * bytes) {
    const int64_t m = X.size(0), k = X.size(1);
    const int xdt = kq_dtype_of(X.scalar_type(), fn);
    // short rows leave a second wave of tiles little to share its start-up with: 24576x1024 at 9 / 65 / 129 tokens, two steps / one kernel,
    // us: IQ4_NL 27 / 29 / 31 against 31 / 33 / 35, IQ4_XS 29 / 30 / 32 against 32 / 33 / 35; 32000x1024 33 / 33 / 35 against 31 / 31 / 35
    const bool short_rows = type != 21 && k < 2048 && row > 148 * 128 && row < 30000;   // IQ3_S: 31 against 29
    if (!short_rows && kq_dequant_mul_mat_preferred(row, m) && kq_dequant_mul_mat_supported(W.data_ptr(), (int)type, row, k, X.data_ptr(), xdt, m, X.stride(0))) {
      const c10::cuda::CUDAGuard guard(X.device());
      at::Tensor Y = at::empty({m, row}, X.options());
      auto stream = at::cuda::getCurrentCUDAStream(X.get_device()).stream();
      TORCH_CHECK(kq_dequant_mul_mat(W.data_ptr(), (int)type, row, k, X.data_ptr(), xdt, m, X.stride(0), Y.data_ptr(), Y.stride(0),
                                     (void*)stream) == KQ_OK, fn, ": ", kq_last_error());
      return Y;
    }
  }
  return at::matmul(X, ggml_dequantize(W, type, c10::SymInt(row), c10::SymInt(W.size(1) / bytes * blk), X.scalar_type()).t());
}

// rows `ids` (any shape) of the [n, row bytes] table W, dequantized: [*ids.shape, k]
at::Tensor ggml_dequantize_rows(const at::Tensor& W, const at::Tensor& ids, int64_t type, int64_t k, at::ScalarType dtype, bool f32_math) {
  const char* fn = "ggml_dequantize_rows";
  check_weight(W, fn);
  TORCH_CHECK(W.dim() == 2 && ids.is_cuda() && ids.get_device() == W.get_device(), fn, ": W must be 2-D and the ids on its device");
  const int odt = kq_dtype_of(dtype, fn);
  int blk = 0, bytes = 0;
  TORCH_CHECK(kq_block_geometry((int)type, &blk, &bytes) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(k > 0 && k % blk == 0 && W.size(1) == k / blk * bytes, fn, ": rows of W do not hold k=", k, " weights");
  const c10::cuda::CUDAGuard guard(W.device());
  const at::Tensor flat = ids.to(at::kLong).contiguous();
  auto shape = ids.sizes().vec();
  shape.push_back(k);
  at::Tensor out = at::empty(shape, W.options().dtype(dtype));
  const int rc = kq_dequantize_rows(W.data_ptr(), (int)type, W.size(0), k, flat.data_ptr<int64_t>(), flat.numel(), out.data_ptr(), odt,
                                    f32_math, (void*)at::cuda::getCurrentCUDAStream(W.get_device()).stream());
  TORCH_CHECK(rc == KQ_OK, fn, ": ", kq_last_error());
  return out;
}

// W: [E, row, row bytes] (or any contiguous uint8 tensor holding E matrices back to back)
at::Tensor moe_impl(bool block, const at::Tensor& X, const at::Tensor& W, const at::Tensor& ids, const at::Tensor* expert_ids,
                    const at::Tensor* num_post_padded, int64_t type, int64_t row, int64_t top_k, int64_t tokens) {
  const char* fn = block ? "ggml_moe_a8" : "ggml_moe_a8_vec";
  check_weight(W, fn);
  TORCH_CHECK(X.is_cuda() && X.dim() == 2, fn, ": X must be a 2-D CUDA tensor");
  TORCH_CHECK(X.get_device() == W.get_device(), fn, ": W and X are on different devices");
  TORCH_CHECK(X.stride(1) == 1, fn, ": X must be contiguous along its last dimension");
  TORCH_CHECK(tokens >= 0 && tokens <= X.size(0), fn, ": `tokens` exceeds X.size(0)");
  TORCH_CHECK(top_k > 0 && row >= 0, fn, ": top_k must be positive");
  const int64_t k = X.size(1);
  const int xdt = kq_dtype_of(X.scalar_type(), fn);
  int blk = 0, bytes = 0;
  TORCH_CHECK(kq_block_geometry((int)type, &blk, &bytes) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(k % blk == 0, fn, ": X.size(1)=", k, " is not a multiple of the block size ", blk);
  const int64_t per_expert = row * (k / blk) * bytes;
  TORCH_CHECK(per_expert > 0 && W.numel() % per_expert == 0, fn, ": W is not a whole number of [row, K] matrices");
  const int64_t experts = W.numel() / per_expert;
  auto as_i32 = [&](const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == X.get_device(), fn, ": ", name, " must be on X's device");
    return t.scalar_type() == at::kInt && t.is_contiguous() ? t : t.to(at::kInt).contiguous();
  };
  const c10::cuda::CUDAGuard guard(X.device());
  at::Tensor Y = at::zeros({tokens * top_k, row}, X.options());   // rows nobody writes read as zero, as in the reference
  if (tokens == 0 || row == 0) return Y;
  const at::Tensor ids32 = as_i32(ids, block ? "sorted_token_ids" : "topk_ids");
  const size_t ws = kq_workspace_bytes((int)type, tokens, row, k);
  at::Tensor scratch = at::empty({(int64_t)ws}, W.options());
  auto stream = at::cuda::getCurrentCUDAStream(X.get_device()).stream();
  int rc;
  if (block) {
    const at::Tensor e32 = as_i32(*expert_ids, "expert_ids"), n32 = as_i32(*num_post_padded, "num_tokens_post_padded");
    TORCH_CHECK(n32.numel() >= 1, fn, ": num_tokens_post_padded is empty");
    TORCH_CHECK(e32.numel() * kq_moe_block_size((int)type) >= ids32.numel(), fn, ": expert_ids has fewer entries than blocks of sorted tokens");
    rc = kq_moe_a8(W.data_ptr(), (int)type, experts, row, k, X.data_ptr(), xdt, tokens, X.stride(0), ids32.data_ptr<int32_t>(),
                   ids32.numel(), e32.data_ptr<int32_t>(), n32.data_ptr<int32_t>(), (int)top_k, Y.data_ptr(), xdt, Y.stride(0),
                   scratch.data_ptr(), ws, (void*)stream);
  } else {
    TORCH_CHECK(ids32.numel() >= tokens * top_k, fn, ": topk_ids has fewer than tokens * top_k entries");
    rc = kq_moe_a8_vec(W.data_ptr(), (int)type, experts, row, k, X.data_ptr(), xdt, tokens, X.stride(0), ids32.data_ptr<int32_t>(),
                       (int)top_k, Y.data_ptr(), xdt, Y.stride(0), scratch.data_ptr(), ws, (void*)stream);
  }
  TORCH_CHECK(rc == KQ_OK, fn, ": ", kq_last_error());
  return Y;
}

at::Tensor ggml_moe_a8(const at::Tensor& X, const at::Tensor& W, const at::Tensor& sorted_token_ids, const at::Tensor& expert_ids,
                       const at::Tensor& num_tokens_post_padded, int64_t type, c10::SymInt row, c10::SymInt top_k,
                       c10::SymInt tokens) {
  return moe_impl(true, X, W, sorted_token_ids, &expert_ids, &num_tokens_post_padded, type, row.expect_int(), top_k.expect_int(),
                  tokens.expect_int());
}

at::Tensor ggml_moe_a8_vec(const at::Tensor& X, const at::Tensor& W, const at::Tensor& topk_ids, int64_t top_k, int64_t type,
                           c10::SymInt row, c10::SymInt tokens) {
  return moe_impl(false, X, W, topk_ids, nullptr, nullptr, type, row.expect_int(), top_k, tokens.expect_int());
}

// The whole SiLU feed-forward of linear.fused_moe_gguf: 5 launches (per-pair branch) or 6 (expert-sorted branch).
// W1 [E, 2 * inter, row bytes], W2 [E, hidden_out, row bytes], topk_ids [tokens, top_k], topk_weights of as many entries.
at::Tensor fused_moe_swiglu(const at::Tensor& X, const at::Tensor& W1, const at::Tensor& W2, const at::Tensor& topk_weights,
                            const at::Tensor& topk_ids, int64_t type1, int64_t type2, bool block) {
  const char* fn = "fused_moe_swiglu";
  check_weight(W1, fn);
  check_weight(W2, fn);
  TORCH_CHECK(W1.dim() == 3 && W2.dim() == 3 && X.dim() == 2 && topk_ids.dim() == 2, fn, ": bad dimensions");
  TORCH_CHECK(X.is_cuda() && X.stride(1) == 1, fn, ": X must be a CUDA tensor, contiguous along its last dimension");
  for (const at::Tensor* t : {&W1, &W2, &topk_weights, &topk_ids}) TORCH_CHECK(t->is_cuda() && t->get_device() == X.get_device(), fn, ": all tensors must be on X's device");
  const int64_t tokens = X.size(0), k1 = X.size(1), e = W1.size(0), n1 = W1.size(1), n2 = W2.size(1), top_k = topk_ids.size(1), pairs = tokens * top_k;
  const int64_t k2 = n1 / 2;
  int b1 = 0, s1 = 0, b2 = 0, s2 = 0;
  TORCH_CHECK(kq_block_geometry((int)type1, &b1, &s1) == KQ_OK && kq_block_geometry((int)type2, &b2, &s2) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(tokens > 0 && top_k > 0 && n1 % 2 == 0 && n1 > 0 && n2 > 0 && topk_ids.size(0) == tokens && topk_weights.numel() == pairs, fn, ": sizes do not match");
  TORCH_CHECK(k1 % b1 == 0 && W1.size(2) == k1 / b1 * s1 && k2 % b2 == 0 && W2.size(2) == k2 / b2 * s2 && W2.size(0) == e, fn, ": weight sizes do not match");
  const int xdt = kq_dtype_of(X.scalar_type(), fn), wdt = kq_dtype_of(topk_weights.scalar_type(), fn);
  const c10::cuda::CUDAGuard guard(X.device());
  auto stream = (void*)at::cuda::getCurrentCUDAStream(X.get_device()).stream();
  const at::Tensor ids = topk_ids.to(at::kInt).contiguous();
  const at::Tensor tw = topk_weights.contiguous();
  const auto iopt = X.options().dtype(at::kInt);
  at::Tensor sorted, eids, post, flag;
  at::cuda::CUDAEvent copied;
  if (block) {
    const int64_t bs = kq_moe_block_size((int)type1), nb = (pairs + e * (bs - 1) + bs - 1) / bs;
    sorted = at::empty({nb * bs}, iopt); eids = at::empty({nb}, iopt); post = at::empty({2}, iopt);
    TORCH_CHECK(kq_moe_align(ids.data_ptr<int32_t>(), pairs, e, sorted.data_ptr<int32_t>(), nb * bs, eids.data_ptr<int32_t>(), nb,
                             post.data_ptr<int32_t>(), stream) == KQ_OK, fn, ": ", kq_last_error());
    // an expert id outside [0, E) is an error in this branch: the flag travels to the host while the kernels below run, and the host
    // waits for it (so for all earlier work of the stream) at the end of the call; not capturable, as the chain of ops is not either
    flag = at::empty({2}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
    flag.copy_(post, /*non_blocking=*/true);
    copied.record(at::cuda::getCurrentCUDAStream(X.get_device()));
  }
  const size_t ws1 = kq_workspace_bytes((int)type1, tokens, n1, k1), ws2 = kq_workspace_bytes((int)type2, pairs, n2, k2);
  at::Tensor scratch = at::empty({(int64_t)(ws1 > ws2 ? ws1 : ws2)}, W1.options());
  at::Tensor h = at::empty({pairs, n1}, X.options()), y = at::empty({pairs, n2}, X.options()), out = at::empty({tokens, n2}, X.options());
  const int32_t* idp = block ? sorted.data_ptr<int32_t>() : ids.data_ptr<int32_t>();
  const int32_t* ep = block ? eids.data_ptr<int32_t>() : nullptr;
  const int32_t* pp = block ? post.data_ptr<int32_t>() : nullptr;
  const int64_t nid = block ? sorted.numel() : pairs;
  TORCH_CHECK(kq_moe_project(0, W1.data_ptr(), (int)type1, e, n1, k1, X.data_ptr(), xdt, tokens, X.stride(0), idp, nid, ep, pp, (int)top_k,
                             h.data_ptr(), xdt, n1, scratch.data_ptr(), scratch.numel(), stream) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(kq_moe_project(1, W2.data_ptr(), (int)type2, e, n2, k2, h.data_ptr(), xdt, pairs, n1, idp, nid, ep, pp, 1, y.data_ptr(), xdt,
                             n2, scratch.data_ptr(), scratch.numel(), stream) == KQ_OK, fn, ": ", kq_last_error());
  TORCH_CHECK(kq_moe_combine(y.data_ptr(), xdt, tw.data_ptr(), wdt, tokens, n2, (int)top_k, out.data_ptr(), stream) == KQ_OK, fn, ": ", kq_last_error());
  if (block) {
    copied.synchronize();
    TORCH_CHECK(flag.data_ptr<int32_t>()[1] == 0, fn, ": topk_ids holds an expert id outside [0, ", e, ")");
  }
  return out;
}

// an output or scratch tensor without the dispatcher's part of at::empty: a decode step makes these calls in every layer, and the
// host's time is most of a call's there
at::Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// no input that backward or forward differentiation would follow (a tangent also counts under no_grad, which is backward's alone)
void no_gradient(const char* fn, std::initializer_list<const at::Tensor*> ts) {
  const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !((backward && t->requires_grad()) || (forward && t->_fw_grad(0).defined())), fn, ": has no derivative, and an input requires one");
}

// defined, on `like`'s device and of one of the given types
void check_on(const char* fn, const char* name, const at::Tensor& t, const at::Tensor& like, std::initializer_list<at::ScalarType> types) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == like.get_device(), fn, ": ", name, " must be on the device of the first argument");
  bool ok = false;
  for (at::ScalarType s : types) ok |= t.scalar_type() == s;
  TORCH_CHECK(ok, fn, ": ", name, " has the wrong dtype ", t.scalar_type());
}

struct RopeCall { int64_t tokens, kv, d; int wdt; const void *qw, *kw; };

RopeCall rope_checks(const char* fn, const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq, int64_t heads, int64_t kv,
                     const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight) {
  TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 2 && (qkv.size(1) == 1 || qkv.stride(1) == 1), fn, ": qkv must be a 2-D CUDA tensor, contiguous along its last dimension");
  TORCH_CHECK(heads > 0 && kv > 0 && heads <= 65536 && kv <= 65536 && qkv.size(1) > 0 && qkv.size(1) % (heads + 2 * kv) == 0, fn,
              ": qkv.size(1)=", qkv.size(1), " is not a whole number of values for ", heads, " query and ", kv, " key and value heads");
  RopeCall c{qkv.size(0), kv, qkv.size(1) / (heads + 2 * kv), KQ_F32, nullptr, nullptr};
  check_on(fn, "positions", positions, qkv, {at::kInt, at::kLong});
  TORCH_CHECK(positions.dim() == 1 && positions.size(0) == c.tokens && positions.is_contiguous(), fn, ": positions must be contiguous, one per token");
  check_on(fn, "inv_freq", inv_freq, qkv, {at::kFloat});
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.is_contiguous() && 2 * inv_freq.size(0) <= c.d, fn, ": inv_freq must be contiguous, one value per rotated pair, at most ", c.d / 2);
  const at::Tensor none;
  const at::Tensor &qw = q_weight.has_value() ? *q_weight : none, &kw = k_weight.has_value() ? *k_weight : none;
  for (const at::Tensor* w : {&qw, &kw})
    if (w->defined()) {
      check_on(fn, "norm weight", *w, qkv, {at::kFloat, qkv.scalar_type()});
      TORCH_CHECK(w->dim() == 1 && w->size(0) == c.d && w->is_contiguous(), fn, ": norm weights must be contiguous, ", c.d, " values");
      c.wdt = kq_dtype_of(w->scalar_type(), fn);
    }
  TORCH_CHECK(!qw.defined() || !kw.defined() || qw.scalar_type() == kw.scalar_type(), fn, ": the norm weights must have one dtype");
  c.qw = qw.defined() ? qw.data_ptr() : nullptr;
  c.kw = kw.defined() ? kw.data_ptr() : nullptr;
  no_gradient(fn, {&qkv, &inv_freq, &qw, &kw});
  return c;
}

// caches [pages, page size, kv heads, head dim]; any order of the first three dimensions
void cache_checks(const char* fn, const at::Tensor& k, const at::Tensor& v, const at::Tensor& like) {
  for (const at::Tensor* t : {&k, &v}) {
    check_on(fn, "cache", *t, like, {like.scalar_type()});
    TORCH_CHECK(t->dim() == 4 && (t->size(3) == 1 || t->stride(3) == 1), fn, ": caches are [pages, page size, kv heads, head dim], dense along the last");
  }
  TORCH_CHECK(k.sizes() == v.sizes(), fn, ": the caches of keys and values differ in size");
  no_gradient(fn, {&k, &v});
}

// addresses [first, second) that a view spans
std::pair<uintptr_t, uintptr_t> span_of(const at::Tensor& t) {
  const uintptr_t begin = (uintptr_t)t.const_data_ptr();
  if (t.numel() == 0) return {begin, begin};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {begin, begin + (uintptr_t)(last + 1) * t.element_size()};
}
bool spans_meet(const at::Tensor& a, const at::Tensor& b) {
  const auto x = span_of(a), y = span_of(b);
  return x.first < y.second && y.first < x.second;
}
// whether some sum of stride[i] * d[i], |d[i]| < size[i], is `off`; strides descending.  A stride that is no less than what the later ones
// reach leaves two values of d to try; where there are more (views of no usual layout) the answer is no.
bool reachable(int64_t off, const std::pair<int64_t, int64_t>* dims, int n) {
  if (n == 0) return off == 0;
  int64_t rest = 0;
  for (int i = 1; i < n; ++i) rest += dims[i].first * (dims[i].second - 1);
  if (std::abs(off) > rest + dims[0].first * (dims[0].second - 1)) return false;
  int tried = 0;
  for (int64_t d = std::max((off - rest) / dims[0].first - 1, 1 - dims[0].second); d < dims[0].second && off - d * dims[0].first >= -rest; ++d)
    if (off - d * dims[0].first <= rest && tried++ < 4 && reachable(off - d * dims[0].first, dims + 1, n - 1)) return true;
  return false;
}
// Whether two caches of one size and type share an element: exact for equal strides (also where keys and values lie page by page or
// head by head in one tensor) and for dense tensors
bool caches_meet(const at::Tensor& a, const at::Tensor& b) {
  if (!spans_meet(a, b)) return false;
  c10::SmallVector<std::pair<int64_t, int64_t>, 4> dims;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1) {
      if (a.stride(i) != b.stride(i)) return at::get_overlap_status(a, b) != at::MemOverlapStatus::No && at::get_overlap_status(a, b) != at::MemOverlapStatus::TooHard;
      dims.push_back({a.stride(i), a.size(i)});
    }
  std::sort(dims.begin(), dims.end(), [](const auto& x, const auto& y) { return x.first > y.first; });
  const int64_t bytes = (int64_t)((intptr_t)b.const_data_ptr() - (intptr_t)a.const_data_ptr()), size = a.element_size();
  return bytes % size != 0 || reachable(bytes / size, dims.data(), (int)dims.size());
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq, int64_t heads,
                                                int64_t kv, const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight,
                                                double eps, bool interleaved, double factor) {
  const char* fn = "qk_norm_rope";
  const RopeCall c = rope_checks(fn, qkv, positions, inv_freq, heads, kv, q_weight, k_weight);
  const int dt = kq_dtype_of(qkv.scalar_type(), fn);
  const c10::cuda::CUDAGuard guard(qkv.device());
  at::Tensor q = new_cuda({c.tokens, heads, c.d}, qkv.scalar_type(), qkv), k = new_cuda({c.tokens, kv, c.d}, qkv.scalar_type(), qkv);
  TORCH_CHECK(kq_qk_norm_rope(qkv.data_ptr(), dt, c.tokens, qkv.stride(0), heads, kv, c.d, positions.data_ptr(), positions.scalar_type() == at::kLong,
                              inv_freq.data_ptr<float>(), 2 * inv_freq.size(0), interleaved, (float)factor, c.qw, c.kw, c.wdt, (float)eps,
                              q.data_ptr(), k.data_ptr(), nullptr, nullptr, nullptr, nullptr, 0, 0, 0,
                              (void*)at::cuda::getCurrentCUDAStream(qkv.get_device()).stream()) == KQ_OK, fn, ": ", kq_last_error());
  return {q, k};
}

at::Tensor qk_norm_rope_store(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& inv_freq, int64_t heads,
                              const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& slots,
                              const std::optional<at::Tensor>& q_weight, const std::optional<at::Tensor>& k_weight, double eps,
                              bool interleaved, double factor) {
  const char* fn = "qk_norm_rope_store";
  at::assert_no_internal_overlap(k_cache);
  at::assert_no_internal_overlap(v_cache);
  cache_checks(fn, k_cache, v_cache, qkv);
  TORCH_CHECK(k_cache.size(0) > 0 && k_cache.size(1) > 0, fn, ": the caches have no pages");
  TORCH_CHECK(!caches_meet(k_cache, v_cache), fn, ": the caches of keys and values overlap");
  TORCH_CHECK(!spans_meet(qkv, k_cache) && !spans_meet(qkv, v_cache), fn, ": qkv lies in a cache");
  const RopeCall c = rope_checks(fn, qkv, positions, inv_freq, heads, k_cache.size(2), q_weight, k_weight);
  TORCH_CHECK(k_cache.size(3) == c.d, fn, ": the caches hold heads of ", k_cache.size(3), " values, qkv of ", c.d);
  check_on(fn, "slots", slots, qkv, {at::kInt, at::kLong});
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == c.tokens && slots.is_contiguous(), fn, ": slots must be contiguous, one per token");
  const int dt = kq_dtype_of(qkv.scalar_type(), fn);
  const c10::cuda::CUDAGuard guard(qkv.device());
  at::Tensor q = new_cuda({c.tokens, heads, c.d}, qkv.scalar_type(), qkv);
  TORCH_CHECK(kq_qk_norm_rope(qkv.data_ptr(), dt, c.tokens, qkv.stride(0), heads, c.kv, c.d, positions.data_ptr(), positions.scalar_type() == at::kLong,
                              inv_freq.data_ptr<float>(), 2 * inv_freq.size(0), interleaved, (float)factor, c.qw, c.kw, c.wdt, (float)eps,
                              q.data_ptr(), k_cache.data_ptr(), k_cache.strides().data(), v_cache.data_ptr(), v_cache.strides().data(),
                              slots.data_ptr(), slots.scalar_type() == at::kLong, k_cache.size(0), k_cache.size(1),
                              (void*)at::cuda::getCurrentCUDAStream(qkv.get_device()).stream()) == KQ_OK, fn, ": ", kq_last_error());
  return q;
}

std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                   const at::Tensor& block_table, const at::Tensor& seq_lens, double scale, int64_t window,
                                                   double softcap, bool lse) {
  const char* fn = "paged_attention";
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && (q.size(2) == 1 || q.stride(2) == 1), fn, ": q must be [batch, heads, head dim] on a GPU, dense along the last");
  cache_checks(fn, k_cache, v_cache, q);
  TORCH_CHECK(k_cache.size(3) == q.size(2), fn, ": the caches hold heads of ", k_cache.size(3), " values, q of ", q.size(2));
  check_on(fn, "block_table", block_table, q, {at::kInt});
  check_on(fn, "seq_lens", seq_lens, q, {at::kInt});
  const int64_t b = q.size(0), h = q.size(1), d = q.size(2);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == b && (block_table.size(1) <= 1 || block_table.stride(1) == 1), fn, ": block_table must be [batch, pages], dense along the last");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == b && seq_lens.is_contiguous(), fn, ": seq_lens must be contiguous, one per sequence");
  no_gradient(fn, {&q});
  const int dt = kq_dtype_of(q.scalar_type(), fn);
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = new_cuda({b, h, d}, q.scalar_type(), q), norm;
  if (lse) norm = new_cuda({b, h}, at::kFloat, q);
  const size_t ws = kq_paged_attention_workspace_bytes(b, h, k_cache.size(2), d);
  at::Tensor scratch = new_cuda({(int64_t)ws}, at::kByte, q);
  TORCH_CHECK(kq_paged_attention(q.data_ptr(), dt, b, h, k_cache.size(2), d, q.stride(0), q.stride(1), k_cache.data_ptr(), k_cache.strides().data(),
                                 v_cache.data_ptr(), v_cache.strides().data(), k_cache.size(0), k_cache.size(1), block_table.data_ptr<int32_t>(),
                                 block_table.stride(0), block_table.size(1), seq_lens.data_ptr<int32_t>(), (float)scale, window, (float)softcap,
                                 out.data_ptr(), lse ? norm.data_ptr<float>() : nullptr, scratch.data_ptr(), ws,
                                 (void*)at::cuda::getCurrentCUDAStream(q.get_device()).stream()) == KQ_OK, fn, ": ", kq_last_error());
  return {out, norm};
}

// (total_lens, starts, positions, slots, taken); fresh pages are entered into block_table in place
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> plan_pages(const at::Tensor& block_table, const at::Tensor& seq_lens,
                                                                                  const at::Tensor& new_lens, const at::Tensor& free_pages,
                                                                                  const at::Tensor& taken, int64_t page_size, int64_t num_tokens) {
  const char* fn = "plan_pages";
  TORCH_CHECK(block_table.is_cuda() && block_table.dim() == 2 && block_table.scalar_type() == at::kInt && (block_table.size(1) <= 1 || block_table.stride(1) == 1), fn,
              ": block_table must be an int32 CUDA tensor [requests, pages], dense along the last");
  at::assert_no_internal_overlap(block_table);
  const int64_t r = block_table.size(0);
  for (const at::Tensor* t : {&seq_lens, &new_lens, &free_pages, &taken}) {
    check_on(fn, "index tensor", *t, block_table, {at::kInt});
    TORCH_CHECK(t->dim() == 1 && t->is_contiguous(), fn, ": seq_lens, new_lens, free_pages and taken must be contiguous and 1-D");
  }
  TORCH_CHECK(seq_lens.size(0) == r && new_lens.size(0) == r && taken.size(0) == 1, fn, ": one length per row of block_table, and one value in taken");
  TORCH_CHECK(num_tokens >= 0 && page_size > 0, fn, ": page_size must be positive and num_tokens not negative");
  const c10::cuda::CUDAGuard guard(block_table.device());
  at::Tensor total = new_cuda({r}, at::kInt, block_table), starts = new_cuda({r + 1}, at::kInt, block_table), after = new_cuda({1}, at::kInt, block_table);
  at::Tensor positions = new_cuda({num_tokens}, at::kInt, block_table), slots = new_cuda({num_tokens}, at::kLong, block_table);
  TORCH_CHECK(kq_plan_pages(block_table.data_ptr<int32_t>(), block_table.stride(0), block_table.size(1), seq_lens.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(), r,
                            free_pages.data_ptr<int32_t>(), free_pages.size(0), taken.data_ptr<int32_t>(), page_size, num_tokens,
                            total.data_ptr<int32_t>(), starts.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
                            after.data_ptr<int32_t>(), (void*)at::cuda::getCurrentCUDAStream(block_table.get_device()).stream()) == KQ_OK, fn, ": ", kq_last_error());
  return {total, starts, positions, slots, after};
}

std::tuple<at::Tensor, at::Tensor> moe_route(const at::Tensor& logits, int64_t top_k, bool sigmoid, const std::optional<at::Tensor>& bias_, int64_t groups,
                                             int64_t top_groups, bool renormalize, double scale) {
  const char* fn = "moe_route";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1), fn, ": logits must be a 2-D CUDA tensor, contiguous along its last dimension");
  const int dt = kq_dtype_of(logits.scalar_type(), fn);
  const at::Tensor none;
  const at::Tensor& bias = bias_.has_value() ? *bias_ : none;
  const int64_t t = logits.size(0), e = logits.size(1);
  if (bias.defined()) {
    check_on(fn, "bias", bias, logits, {at::kFloat});
    TORCH_CHECK(bias.dim() == 1 && bias.size(0) == e && bias.is_contiguous(), fn, ": bias must be contiguous, one value per expert");
  }
  no_gradient(fn, {&logits, &bias});
  TORCH_CHECK(top_k > 0 && top_k <= e, fn, ": top_k=", top_k, " is not between 1 and ", e);
  const c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor w = new_cuda({t, top_k}, at::kFloat, logits), ids = new_cuda({t, top_k}, at::kInt, logits);
  TORCH_CHECK(kq_moe_route(logits.data_ptr(), dt, t, e, logits.stride(0), top_k, sigmoid, bias.defined() ? bias.data_ptr<float>() : nullptr, groups, top_groups,
                           renormalize, (float)scale, w.data_ptr<float>(), ids.data_ptr<int32_t>(),
                           (void*)at::cuda::getCurrentCUDAStream(logits.get_device()).stream()) == KQ_OK, fn, ": ", kq_last_error());
  return {w, ids};
}

// The same refusal where autograd looks at a call: inside torch.func's transforms the kernel sees tensors without the level that is
// being differentiated.
void refuse_derivatives(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size()))
    if (v.isTensor()) no_gradient(op.schema().name().c_str(), {&v.toTensor()});
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

int64_t ggml_moe_get_block_size(int64_t type) { return kq_moe_block_size((int)type); }

}  // namespace

TORCH_LIBRARY(_C_gguf, ops) {
  ops.def("ggml_dequantize(Tensor W, int type, SymInt m, SymInt n, ScalarType? dtype) -> Tensor");
  ops.def("ggml_mul_mat_vec_a8(Tensor W, Tensor X, int type, SymInt row) -> Tensor");
  ops.def("ggml_mul_mat_a8(Tensor W, Tensor X, int type, SymInt row) -> Tensor");
  ops.def("ggml_dequant_mul_mat(Tensor W, Tensor X, int type, SymInt row) -> Tensor");
  ops.def("ggml_dequantize_rows(Tensor W, Tensor ids, int type, int k, ScalarType dtype, bool f32_math) -> Tensor");
  ops.def("ggml_mul_mat_merged(Tensor[] W, Tensor X, int[] types, int[] mmq) -> Tensor");
  ops.def(
      "ggml_moe_a8(Tensor X, Tensor W, Tensor sorted_token_ids, Tensor expert_ids, Tensor "
      "num_tokens_post_padded, int type, SymInt row, SymInt top_k, SymInt tokens) -> Tensor");
  ops.def("ggml_moe_a8_vec(Tensor X, Tensor W, Tensor topk_ids, int top_k, int type, SymInt row, SymInt tokens) -> Tensor");
  ops.def(
      "fused_moe_swiglu(Tensor X, Tensor W1, Tensor W2, Tensor topk_weights, Tensor topk_ids, int type1, int type2, bool block) "
      "-> Tensor");
  ops.def("ggml_moe_get_block_size(int type) -> int");
  ops.def(
      "qk_norm_rope(Tensor qkv, Tensor positions, Tensor inv_freq, int num_heads, int num_kv_heads, Tensor? q_weight, Tensor? k_weight, "
      "float eps, bool interleaved, float factor) -> (Tensor, Tensor)");
  ops.def(
      "qk_norm_rope_store(Tensor qkv, Tensor positions, Tensor inv_freq, int num_heads, Tensor(a!) k_cache, Tensor(b!) v_cache, "
      "Tensor slots, Tensor? q_weight, Tensor? k_weight, float eps, bool interleaved, float factor) -> Tensor");
  ops.def(
      "paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, float scale, int window, "
      "float softcap, bool lse) -> (Tensor, Tensor)");
  ops.def(
      "plan_pages(Tensor(a!) block_table, Tensor seq_lens, Tensor new_lens, Tensor free_pages, Tensor taken, int page_size, "
      "int num_tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  ops.def(
      "moe_route(Tensor logits, int top_k, bool sigmoid, Tensor? bias, int groups, int top_groups, bool renormalize, float scale) "
      "-> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(_C_gguf, CUDA, ops) {
  ops.impl("ggml_dequantize", &ggml_dequantize);
  ops.impl("ggml_mul_mat_vec_a8", &ggml_mul_mat_vec_a8);
  ops.impl("ggml_mul_mat_a8", &ggml_mul_mat_a8);
  ops.impl("ggml_dequant_mul_mat", &ggml_dequant_mul_mat);
  ops.impl("ggml_dequantize_rows", &ggml_dequantize_rows);
  ops.impl("ggml_mul_mat_merged", &ggml_mul_mat_merged);
  ops.impl("ggml_moe_a8", &ggml_moe_a8);
  ops.impl("ggml_moe_a8_vec", &ggml_moe_a8_vec);
  ops.impl("fused_moe_swiglu", &fused_moe_swiglu);
  ops.impl("qk_norm_rope", &qk_norm_rope);
  ops.impl("qk_norm_rope_store", &qk_norm_rope_store);
  ops.impl("paged_attention", &paged_attention);
  ops.impl("plan_pages", &plan_pages);
  ops.impl("moe_route", &moe_route);
}

TORCH_LIBRARY_IMPL(_C_gguf, Autograd, ops) {
  for (const char* name : {"qk_norm_rope", "qk_norm_rope_store", "paged_attention", "plan_pages", "moe_route"})
    ops.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_derivatives>());
}

TORCH_LIBRARY_IMPL(_C_gguf, CompositeExplicitAutograd, ops) {
  ops.impl("ggml_moe_get_block_size", &ggml_moe_get_block_size);
}

// direct(name, overload): the operator's function without the dispatcher, for calls from Python (kq_direct.h)
static PyMethodDef kq_direct_defs[] = {
    {"qk_norm_rope", (PyCFunction)(void*)kq_direct::Direct<&qk_norm_rope>::call, METH_FASTCALL, nullptr},
    {"qk_norm_rope_store", (PyCFunction)(void*)kq_direct::Direct<&qk_norm_rope_store>::call, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void*)kq_direct::Direct<&paged_attention>::call, METH_FASTCALL, nullptr},
    {"plan_pages", (PyCFunction)(void*)kq_direct::Direct<&plan_pages>::call, METH_FASTCALL, nullptr},
    {"moe_route", (PyCFunction)(void*)kq_direct::Direct<&moe_route>::call, METH_FASTCALL, nullptr},
};
static PyObject* kq_direct_of(PyObject*, PyObject* args) {
  const char* name = nullptr;
  PyObject* overload = nullptr;
  if (!PyArg_ParseTuple(args, "sO", &name, &overload)) return nullptr;
  for (PyMethodDef& d : kq_direct_defs)
    if (!std::strcmp(d.ml_name, name)) return PyCFunction_New(&d, overload);
  PyErr_Format(PyExc_KeyError, "%s has no direct call", name);
  return nullptr;
}
static PyMethodDef kq_module_methods[] = {{"direct", kq_direct_of, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
static struct PyModuleDef kq_module_def = {PyModuleDef_HEAD_INIT, "_C_gguf", nullptr, -1, kq_module_methods};

extern "C" PyObject* PyInit__C_gguf(void) { return PyModule_Create(&kq_module_def); }
