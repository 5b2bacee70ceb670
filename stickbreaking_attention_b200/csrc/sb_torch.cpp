// Host path of the public operators: from torch tensors to the C ABI and back, with the autograd node, in one native call.
//
// What bounds a small call is not the GPU: building the argument block in Python, the ctypes transition and a Python
// autograd.Function cost 49 us per forward and about 210 us per forward + backward (measured on 200-token and 1243-token
// calls), several times the kernels' own time.  Everything between the public Python function and the launches is
// therefore here.  The kernels stay behind the C ABI (include/sb_b200.h); nothing in this file computes.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <atomic>
#include <mutex>

#include "../../include/sb_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::variable_list;

std::atomic<long long> g_launches{0};   // process-wide: the backward runs on autograd's threads

// What one call is, apart from its tensors.
struct Call {
  bool fixed, fused, leading_zero;
  int32_t max_seqlen, attend_current, flags;
  float scale;
};

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SB_DTYPE_F32;
    case at::kBFloat16: return SB_DTYPE_BF16;
    case at::kHalf: return SB_DTYPE_F16;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t);
  }
  return -1;
}

// One int32[4] status word per device, written by kernels that find a problem; lives as long as the process.
Tensor status_word(int device) {
  static std::mutex mu;
  static std::array<Tensor, 64> words;
  std::lock_guard<std::mutex> guard(mu);
  TORCH_CHECK(device >= 0 && device < (int)words.size(), "device ordinal ", device, " not supported");
  Tensor &w = words[device];
  if (!w.defined()) w = at::zeros({4}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
  return w;
}
int32_t *status_ptr(int device) {
  static std::array<std::atomic<int32_t *>, 64> ptrs{};
  if (device < 0 || device >= (int)ptrs.size()) return static_cast<int32_t *>(status_word(device).data_ptr());
  int32_t *p = ptrs[device].load(std::memory_order_acquire);
  if (p == nullptr) {
    p = static_cast<int32_t *>(status_word(device).data_ptr());
    ptrs[device].store(p, std::memory_order_release);
  }
  return p;
}

// Unit innermost stride, 16-byte aligned base and outer strides (what TMA and the vector accesses need) and, for the types
// the tensor maps are for, no axis that repeats its elements (an expanded tensor: a key head shared by several heads, the
// gradient of a sum); copies only where that does not hold, so that forward and backward take the same kernels whatever
// the strides.  Rows that are no multiple of 16 bytes take the CUDA-core kernels: any stride will do.
Tensor tma_ready(const Tensor &t) {
  const int64_t mult = 16 / t.element_size(), nd = t.dim();
  bool ok = t.stride(-1) == 1;
  if (ok && t.size(-1) % mult == 0) {
    ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; ok && i + 1 < nd; ++i) ok = t.size(i) == 1 || (t.stride(i) % mult == 0 && (t.stride(i) > 0 || mult < 8));
  }
  return ok ? t : t.contiguous();
}

Tensor empty_cuda(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor &like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}
// Same sizes and, for a dense tensor (permuted views included), the same strides: torch.empty_like without the dispatcher.
Tensor empty_as(const Tensor &t) {
  if (t.is_non_overlapping_and_dense()) return at::detail::empty_strided_cuda(t.sizes(), t.strides(), t.scalar_type(), t.device());
  return at::empty_like(t);
}

SbTensor arg(const Tensor &t, bool fixed) {
  return fixed ? SbTensor{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)} : SbTensor{t.data_ptr(), 0, t.stride(0), t.stride(1)};
}

void check_inputs(const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &cu, const Call &c) {
  TORCH_CHECK_VALUE(q.is_cuda(), "stick-breaking attention runs on a CUDA device only (no CPU path)");
  dtype_code(q.scalar_type());
  TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k, v must share a dtype");
  TORCH_CHECK_VALUE(q.sizes() == k.sizes() && q.sizes() == v.sizes(), "q, k, v must share a shape");
  TORCH_CHECK_VALUE(q.device() == k.device() && q.device() == v.device(), "q, k, v must share a device");
  TORCH_CHECK_VALUE(q.dim() == (c.fixed ? 4 : 3), "expected (B,H,T,d) for sb_attn and (H,T,d) for sb_attn_varlen");
  if (!c.fixed) {
    TORCH_CHECK_VALUE(cu->is_cuda() && cu->dim() == 1, "cu_seqlens must be a 1-D CUDA tensor");
    TORCH_CHECK_VALUE(cu->device() == q.device(), "cu_seqlens must be on the device of q, k, v");
    TORCH_CHECK_VALUE(cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong, "cu_seqlens must be int32 or int64");
    TORCH_CHECK_VALUE(cu->numel() <= 1 || cu->stride(0) == 1, "cu_seqlens must be contiguous");
  }
}

// The backward's own inputs: the kernels go by the shapes of q.
void check_gradients(const Tensor &dout, const Tensor &drem, const Tensor &q) {
  if (dout.defined())
    TORCH_CHECK_VALUE(dout.device() == q.device() && dout.sizes() == q.sizes(), "the gradient of o must have the shape and device of q");
  if (drem.defined())
    TORCH_CHECK_VALUE(drem.device() == q.device() && drem.numel() * q.size(-1) == q.numel(),
                      "the gradient of rem must have one value per row of q, on its device");
}
void check_log_rem(const Tensor &log_rem, const Tensor &q) {
  TORCH_CHECK_VALUE(log_rem.scalar_type() == at::kDouble && log_rem.is_contiguous() && log_rem.device() == q.device() &&
                        log_rem.numel() * q.size(-1) == q.numel(),
                    "log_rem must be what the forward returned: fp64, contiguous, one value per row of q");
}

void fill(SbParams &p, const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &cu, const Call &c) {
  memset(&p, 0, sizeof(p));
  p.struct_bytes = (int32_t)sizeof(SbParams);
  p.dtype = dtype_code(q.scalar_type());
  const int64_t nd = q.dim();
  p.batch = c.fixed ? (int32_t)q.size(0) : 1;
  p.heads = (int32_t)q.size(nd - 3);
  p.tokens = q.size(nd - 2);
  p.head_dim = (int32_t)q.size(nd - 1);
  if (!c.fixed) {   // the C ABI takes the sequence ends only
    const int64_t skip = c.leading_zero ? 1 : 0;
    p.num_seq = (int32_t)(cu->numel() - skip);
    p.cu_seqlens = static_cast<const char *>(cu->data_ptr()) + skip * cu->element_size();
    p.cu_seqlens_int64 = cu->scalar_type() == at::kLong;
  }
  p.max_seqlen = c.max_seqlen;
  p.attend_current = c.attend_current;
  p.logit_scale = c.scale;
  p.flags = c.flags | (c.leading_zero && !c.fixed ? SB_FLAG_CHECK_LEADING_ZERO : 0) | (c.fused ? SB_FLAG_FUSE_REM_V : 0);
  p.q = arg(q, c.fixed);
  p.k = arg(k, c.fixed);
  p.v = arg(v, c.fixed);
}

// An error the library reported; reaches Python as _cabi.SbError (see set_python_error).
struct LibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void raise_library_error(const char *what, int rc) {
  if (rc < 0) throw LibraryError(std::string("invalid parameters: ") + sb_last_error());
  throw LibraryError(std::string(what) + " failed with status " + std::to_string(rc) + ": " + sb_last_error());
}
void set_python_error(const LibraryError &e) {   // with the GIL held
  const py::object type = py::module_::import("stickbreaking_attention_b200._cabi").attr("SbError");
  PyErr_SetString(type.ptr(), e.what());
}

size_t workspace_bytes(const SbParams &p, bool backward) {
  const size_t need = sb_workspace_bytes(&p, backward);
  if (need == (size_t)-1) raise_library_error("sb_workspace_bytes", -1);
  return need < 256 ? 256 : need;
}

void launch(SbParams &p, bool backward, char *workspace, size_t bytes, const Tensor &q) {
  p.workspace = workspace;
  p.workspace_bytes = bytes;
  p.status = status_ptr(q.get_device());
  void *stream = at::cuda::getCurrentCUDAStream(q.get_device()).stream();
  const int rc = backward ? sb_bwd(&p, stream) : sb_fwd(&p, stream);
  if (rc != SB_OK) raise_library_error(backward ? "sb_bwd" : "sb_fwd", rc);
  g_launches.fetch_add(sb_last_launch_count(), std::memory_order_relaxed);
}

// `state`: what the backward needs, one fp64 buffer -- log_rem (batch, heads, tokens) and, where the call keeps them, the
// int32 tile starts (batch * heads, ceil(tokens / 32)) behind it.
struct Forward { Tensor out, rem, state; };

void attach_state(SbParams &p, double *state, bool tile_starts) {
  const int64_t rows = (int64_t)p.batch * p.heads;
  p.log_rem = state;
  if (tile_starts) {
    p.tile_start = reinterpret_cast<int32_t *>(state + rows * p.tokens);
    p.tile_start_stride = (p.tokens + 31) / 32;
  }
}
int64_t state_doubles(const SbParams &p) {
  const int64_t rows = (int64_t)p.batch * p.heads;
  return rows * p.tokens + (rows * ((p.tokens + 31) / 32) + 1) / 2;
}

// kLogRem: log_rem over all keys, as a tensor of the rows' shape; kState: the operator's own saved state; kNothing: no
// backward will come, and the state is scratch like the rest and shares its allocation.
enum class Keep { kNothing, kState, kLogRem };

Forward run_forward(const Tensor &q_in, const Tensor &k_in, const Tensor &v_in, const std::optional<Tensor> &cu, const Call &c,
                    Keep keep) {
  check_inputs(q_in, k_in, v_in, cu, c);
  c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = tma_ready(q_in), k = tma_ready(k_in), v = tma_ready(v_in);
  Forward f;
  f.out = empty_as(q);
  const auto row_sizes = q.sizes().slice(0, q.dim() - 1);
  f.rem = empty_cuda(row_sizes, q.scalar_type(), q);
  SbParams p;
  fill(p, q, k, v, cu, c);
  p.o = arg(f.out, c.fixed);
  p.rem = f.rem.data_ptr();
  const size_t ws = (workspace_bytes(p, false) + 255) / 256 * 256;
  size_t bytes = ws;
  if (keep == Keep::kLogRem) f.state = empty_cuda(row_sizes, at::kDouble, q);
  else if (keep == Keep::kState) f.state = empty_cuda({state_doubles(p)}, at::kDouble, q);
  else bytes += sizeof(double) * (size_t)state_doubles(p);
  // freed on return: the caching allocator hands the block out again only behind this stream's work
  const Tensor scratch = empty_cuda({(int64_t)bytes}, at::kByte, q);
  char *base = static_cast<char *>(scratch.data_ptr());
  attach_state(p, f.state.defined() ? static_cast<double *>(f.state.data_ptr()) : reinterpret_cast<double *>(base + ws),
               keep != Keep::kLogRem);
  launch(p, false, base, ws, q);
  return f;
}

std::array<Tensor, 3> run_backward(const Tensor &dout_in, const Tensor &drem_in, const Tensor &q_in, const Tensor &k_in, const Tensor &v_in,
                                   const std::optional<Tensor> &cu, const Tensor &state, bool tile_starts, const Call &c) {
  check_inputs(q_in, k_in, v_in, cu, c);
  check_gradients(dout_in, drem_in, q_in);
  c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = tma_ready(q_in), k = tma_ready(k_in), v = tma_ready(v_in);
  const Tensor dout = dout_in.defined() ? tma_ready(dout_in.scalar_type() == q.scalar_type() ? dout_in : dout_in.to(q.scalar_type()))
                                        : at::zeros_like(q);
  Tensor drem;
  if (drem_in.defined()) drem = drem_in.to(q.scalar_type()).contiguous();
  else if (!c.fused) drem = at::zeros(q.sizes().slice(0, q.dim() - 1), q.options());
  const Tensor dq = empty_as(q), dk = empty_as(k), dv = empty_as(v);
  SbParams p;
  fill(p, q, k, v, cu, c);
  attach_state(p, static_cast<double *>(state.data_ptr()), tile_starts);
  p.d_o = arg(dout, c.fixed);
  p.d_rem = drem.defined() ? drem.data_ptr() : nullptr;
  p.dq = arg(dq, c.fixed);
  p.dk = arg(dk, c.fixed);
  p.dv = arg(dv, c.fixed);
  size_t bytes = workspace_bytes(p, true);
  Tensor scratch;
  try {
    scratch = empty_cuda({(int64_t)bytes}, at::kByte, q);
  } catch (const c10::OutOfMemoryError &) {
    // the stored-tiles backward asks for up to the scratch budget; where that does not fit, the recomputing kernels and
    // their few MB do the same work instead of failing
    if (p.flags & SB_FLAG_BWD_RECOMPUTE) throw;
    p.flags |= SB_FLAG_BWD_RECOMPUTE;
    bytes = workspace_bytes(p, true);
    scratch = empty_cuda({(int64_t)bytes}, at::kByte, q);
  }
  launch(p, true, static_cast<char *>(scratch.data_ptr()), bytes, q);
  return {dq, dk, dv};
}

// The operator's node in the autograd graph (reference: StickBreakingAttention.backward, sb_varlen/__init__.py:48-68).
struct StickBreakingAttentionBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable q, k, v, state, cu;
  Call call{};
  bool released = false;

  std::string name() const override { return "StickBreakingAttentionBackward"; }
  void release_variables() override {
    q.reset_data(); k.reset_data(); v.reset_data(); state.reset_data(); cu.reset_data();
    released = true;
  }
  variable_list apply(variable_list &&grads) override {
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    // Saved-tensor hooks run here and may record operations of their own (activation checkpointing runs the forward again).
    const Tensor sq = q.unpack(), sk = k.unpack(), sv = v.unpack(), saved = state.unpack();
    std::optional<Tensor> ends;
    if (!call.fixed) ends = cu.unpack();
    at::AutoDispatchBelowADInplaceOrView below;   // plain tensors from here on: conversions and copies record nothing
    std::array<Tensor, 3> g;
    try {
      g = run_backward(grads[0], grads.size() > 1 ? grads[1] : Tensor(), sq, sk, sv, ends, saved, true, call);
    } catch (const LibraryError &e) {   // on an autograd thread: the exception keeps its Python type on its way to the caller
      py::gil_scoped_acquire gil;
      set_python_error(e);
      python_error err;
      err.persist();
      throw std::move(err);
    }
    variable_list out(3);
    for (size_t i = 0; i < 3; ++i)
      if (task_should_compute_output(i)) out[i] = std::move(g[i]);
    return out;
  }
};

Call make_call(bool fixed, std::optional<int64_t> max_seqlens, double scale, bool attend_current, bool leading_zero, bool fused,
               int64_t flags) {
  Call c;
  c.fixed = fixed;
  c.fused = fused;
  c.leading_zero = leading_zero;
  c.max_seqlen = (int32_t)max_seqlens.value_or(0);
  c.attend_current = attend_current;
  c.flags = (int32_t)flags;
  c.scale = (float)scale;
  return c;
}

// The differentiable operator: (out, rem), or (out,) with out = o + rem * v.
variable_list attention(const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &cu,
                        std::optional<int64_t> max_seqlens, double scale, bool attend_current, bool leading_zero, bool fused,
                        int64_t flags) {
  const Call c = make_call(!cu.has_value(), max_seqlens, scale, attend_current, leading_zero, fused, flags);
  for (const Tensor *t : {&q, &k, &v})
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "stick-breaking attention has no forward-mode derivative");
  const bool grad = torch::autograd::compute_requires_grad(q, k, v);
  Forward f;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    f = run_forward(q, k, v, cu, c, grad ? Keep::kState : Keep::kNothing);
  }
  if (grad) {
    auto node = std::shared_ptr<StickBreakingAttentionBackward>(new StickBreakingAttentionBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
    node->call = c;
    node->q = torch::autograd::SavedVariable(q, false);
    node->k = torch::autograd::SavedVariable(k, false);
    node->v = torch::autograd::SavedVariable(v, false);
    node->state = torch::autograd::SavedVariable(f.state, false);
    if (cu.has_value()) node->cu = torch::autograd::SavedVariable(*cu, false);
    torch::autograd::set_history(f.out, node);
    if (!fused) torch::autograd::set_history(f.rem, node);
  }
  if (fused) return {f.out};
  return {f.out, f.rem};
}

// The launchers: no autograd, the saved state handed out and back in.
std::tuple<Tensor, Tensor, Tensor> forward(const Tensor &q, const Tensor &k, const Tensor &v, const std::optional<Tensor> &cu,
                                           std::optional<int64_t> max_seqlens, double scale, bool attend_current, bool leading_zero,
                                           bool fused, int64_t flags) {
  at::AutoDispatchBelowADInplaceOrView below;
  Forward f = run_forward(q, k, v, cu, make_call(!cu.has_value(), max_seqlens, scale, attend_current, leading_zero, fused, flags),
                          Keep::kLogRem);
  return {f.out, f.rem, f.state};
}
std::tuple<Tensor, Tensor, Tensor> backward(const Tensor &dout, const std::optional<Tensor> &drem, const Tensor &q, const Tensor &k,
                                            const Tensor &v, const std::optional<Tensor> &cu, std::optional<int64_t> max_seqlens,
                                            const Tensor &log_rem, double scale, bool attend_current, bool leading_zero, bool fused,
                                            int64_t flags) {
  at::AutoDispatchBelowADInplaceOrView below;
  check_log_rem(log_rem, q);
  std::array<Tensor, 3> g = run_backward(dout, drem.value_or(Tensor()), q, k, v, cu, log_rem, false,
                                         make_call(!cu.has_value(), max_seqlens, scale, attend_current, leading_zero, fused, flags));
  return {g[0], g[1], g[2]};
}

// ---- serving: a paged key-value cache and attention over it ------------------------------------------------------------

void refuse_grad(const char *what, std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && t->requires_grad()) && !t->_fw_grad(0).defined(), what,
                                " has no derivative: call it under torch.no_grad(), or detach its inputs");
}
// What the call wrote to: a backward that saved it earlier has to notice.
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void check_int32(const Tensor &t, int64_t dim, const char *name, const Tensor &like) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == dim, name,
                    " must be a ", dim == 1 ? "1-D" : "2-D", " int32 tensor on the device of the cache");
  TORCH_CHECK_VALUE(t.size(dim - 1) <= 1 || t.stride(dim - 1) == 1, name, " must be contiguous in its last axis");
}
void check_table(const Tensor &table, const Tensor &lens, const Tensor &like) {
  check_int32(table, 2, "page_table", like);
  check_int32(lens, 1, "seq_lens", like);
  TORCH_CHECK_VALUE(table.size(0) == lens.size(0), "page_table must have a row for each entry of seq_lens");
}
// Pools of keys and values: (pages, kv_heads, page_size, head_dim), with the layers before that where `layers`.
void check_pools(const Tensor &k, const Tensor &v, bool layers) {
  TORCH_CHECK_VALUE(k.is_cuda(), "the cache must be on a CUDA device (no CPU path)");
  dtype_code(k.scalar_type());
  TORCH_CHECK_VALUE(k.scalar_type() == v.scalar_type() && k.device() == v.device() && k.sizes() == v.sizes(),
                    "the caches of keys and values must share dtype, device and shape");
  TORCH_CHECK_VALUE(k.dim() == 4 || (layers && k.dim() == 5), "expected a cache of shape (", layers ? "[layers,] " : "",
                    "pages, kv_heads, page_size, head_dim)");
  TORCH_CHECK_VALUE(k.size(-1) <= 1 || (k.stride(-1) == 1 && v.stride(-1) == 1), "the cache must be contiguous in head_dim");
}
int64_t stride_of(const Tensor &t, int64_t axis) { return t.size(axis) == 1 ? 0 : t.stride(axis); }
SbCache cache_arg(const Tensor &t) {
  const int64_t a = t.dim() - 4;
  return SbCache{t.data_ptr(), a ? stride_of(t, 0) : 0, stride_of(t, a), stride_of(t, a + 1), stride_of(t, a + 2)};
}
SbTensor rows_arg(const Tensor &t) {   // (batch, heads, tokens, d), or packed (heads, tokens, d)
  const int64_t a = t.dim() - 3;
  return SbTensor{t.data_ptr(), a ? stride_of(t, 0) : 0, stride_of(t, a), stride_of(t, a + 1)};
}
int32_t to_int32(int64_t x, const char *name) {
  TORCH_CHECK_VALUE(x >= 0 && x <= 0x7fffffff, name, " ", std::to_string(x), " is out of range");
  return (int32_t)x;
}
void count_launches(const char *what, int rc) {
  if (rc != SB_OK) raise_library_error(what, rc);
  g_launches.fetch_add(sb_last_launch_count(), std::memory_order_relaxed);
}
void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// The output for queries q, by a rule that an operator without data can follow too (ops.py): what torch.empty_like(q) gives, where
// that has unit stride in head_dim, else contiguous; whether or not q itself has to be copied for the kernel.
Tensor rows_like(const Tensor &q) {
  const Tensor o = empty_as(q);
  return o.size(3) <= 1 || o.stride(3) == 1 ? o : empty_cuda(q.sizes(), q.scalar_type(), q);
}

std::tuple<Tensor, Tensor> decode(const Tensor &q_in, const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lens,
                                  double scale, bool attend_current, int64_t flags) {
  refuse_grad("sb_attn_decode", {&q_in, &k, &v});
  at::AutoDispatchBelowADInplaceOrView below;
  check_pools(k, v, false);
  TORCH_CHECK_VALUE(q_in.device() == k.device() && q_in.scalar_type() == k.scalar_type(), "q must share the cache's device and dtype");
  TORCH_CHECK_VALUE(q_in.dim() == 4, "expected q of shape (batch, heads, new_tokens, head_dim)");
  TORCH_CHECK_VALUE(q_in.size(3) == k.size(3), "q and the cache must share head_dim");
  check_table(table, lens, k);
  TORCH_CHECK_VALUE(lens.size(0) == q_in.size(0), "seq_lens must have an entry for each sequence of q");
  c10::cuda::CUDAGuard guard(k.device());
  // rows of pairs of elements (only an odd slice has others), so that the kernel does not depend on where q comes from
  bool pairs = q_in.size(3) <= 1 || q_in.stride(3) == 1;
  if (pairs && q_in.element_size() == 2 && q_in.size(3) % 8 == 0)
    pairs = reinterpret_cast<uintptr_t>(q_in.data_ptr()) % 4 == 0 && stride_of(q_in, 0) % 2 == 0 && stride_of(q_in, 1) % 2 == 0 && stride_of(q_in, 2) % 2 == 0;
  const Tensor q = pairs ? q_in : q_in.contiguous();
  const Tensor o = rows_like(q_in), rem = empty_cuda(q.sizes().slice(0, 3), q.scalar_type(), q);
  SbDecodeParams p;
  memset(&p, 0, sizeof(p));
  p.struct_bytes = (int32_t)sizeof(p);
  p.dtype = dtype_code(q.scalar_type());
  p.batch = to_int32(q.size(0), "batch");
  p.heads = to_int32(q.size(1), "heads");
  p.new_tokens = to_int32(q.size(2), "new_tokens");
  p.head_dim = to_int32(q.size(3), "head_dim");
  p.num_pages = to_int32(k.size(0), "pages");
  p.kv_heads = to_int32(k.size(1), "kv_heads");
  p.page_size = to_int32(k.size(2), "page_size");
  p.max_pages = to_int32(table.size(1), "pages per sequence");
  p.attend_current = attend_current;
  p.logit_scale = (float)scale;
  p.flags = (int32_t)(flags & (SB_FLAG_FORCE_SIMT | SB_FLAG_DENSE_ROW_PASS));
  p.q = rows_arg(q);
  p.o = rows_arg(o);
  p.rem = rem.data_ptr();
  p.k = cache_arg(k);
  p.v = cache_arg(v);
  p.page_table = static_cast<const int32_t *>(table.data_ptr());
  p.page_table_stride = table.stride(0);
  p.seq_lens = static_cast<const int32_t *>(lens.data_ptr());
  p.status = status_ptr(k.get_device());
  const size_t need = sb_attn_decode_workspace_bytes(&p);
  if (need == (size_t)-1) raise_library_error("sb_attn_decode", -1);
  const Tensor scratch = empty_cuda({(int64_t)need}, at::kByte, k);
  p.workspace = scratch.data_ptr();
  p.workspace_bytes = need;
  count_launches("sb_attn_decode", sb_attn_decode(&p, stream_of(k)));
  return {o, rem};
}

void append(const Tensor &k_in, const Tensor &v_in, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table,
            const Tensor &lens, const std::optional<Tensor> &cu, bool leading_zero) {
  refuse_grad("kv_append", {&k_in, &v_in, &k_pages, &v_pages});
  at::AutoDispatchBelowADInplaceOrView below;
  check_pools(k_pages, v_pages, false);
  TORCH_CHECK_VALUE(k_in.scalar_type() == k_pages.scalar_type() && v_in.scalar_type() == k_pages.scalar_type() &&
                        k_in.device() == k_pages.device() && v_in.device() == k_pages.device(),
                    "k and v must share the cache's dtype and device");
  TORCH_CHECK_VALUE(k_in.sizes() == v_in.sizes() && k_in.dim() == (cu.has_value() ? 3 : 4),
                    "expected k and v of shape (batch, kv_heads, tokens, head_dim), or (kv_heads, tokens, head_dim) with cu_seqlens");
  TORCH_CHECK_VALUE(k_in.size(-1) == k_pages.size(3) && k_in.size(-3) == k_pages.size(1), "k, v and the cache must share kv_heads and head_dim");
  check_table(table, lens, k_pages);
  c10::cuda::CUDAGuard guard(k_pages.device());
  const bool unit = k_in.size(-1) <= 1;
  const Tensor k = unit || k_in.stride(-1) == 1 ? k_in : k_in.contiguous(), v = unit || v_in.stride(-1) == 1 ? v_in : v_in.contiguous();
  SbAppendParams p;
  memset(&p, 0, sizeof(p));
  p.struct_bytes = (int32_t)sizeof(p);
  p.dtype = dtype_code(k.scalar_type());
  p.num_seq = to_int32(lens.size(0), "sequences");
  p.tokens = k.size(-2);
  if (cu.has_value()) {
    TORCH_CHECK_VALUE(cu->is_cuda() && cu->dim() == 1 && cu->device() == k.device() &&
                          (cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong) && (cu->numel() <= 1 || cu->stride(0) == 1),
                      "cu_seqlens must be a contiguous 1-D int32 or int64 tensor on the device of the cache");
    TORCH_CHECK_VALUE(cu->numel() == lens.size(0) + leading_zero, "cu_seqlens must have an end for each entry of seq_lens",
                      leading_zero ? " behind its leading zero" : "");
    p.cu_seqlens = static_cast<const char *>(cu->data_ptr()) + (leading_zero ? cu->element_size() : 0);
    p.cu_seqlens_int64 = cu->scalar_type() == at::kLong;
    p.flags = leading_zero ? SB_FLAG_CHECK_LEADING_ZERO : 0;
  } else {
    TORCH_CHECK_VALUE(k.size(0) == lens.size(0), "seq_lens must have an entry for each sequence of k and v");
  }
  p.num_pages = to_int32(k_pages.size(0), "pages");
  p.kv_heads = to_int32(k_pages.size(1), "kv_heads");
  p.page_size = to_int32(k_pages.size(2), "page_size");
  p.head_dim = to_int32(k_pages.size(3), "head_dim");
  p.max_pages = to_int32(table.size(1), "pages per sequence");
  p.k = rows_arg(k);
  p.v = rows_arg(v);
  p.k_cache = cache_arg(k_pages);
  p.v_cache = cache_arg(v_pages);
  p.page_table = static_cast<const int32_t *>(table.data_ptr());
  p.page_table_stride = table.stride(0);
  p.seq_lens = static_cast<const int32_t *>(lens.data_ptr());
  p.status = status_ptr(k_pages.get_device());
  count_launches("sb_kv_append", sb_kv_append(&p, stream_of(k_pages)));
  written(k_pages);
  written(v_pages);
}

SbPagesParams pages_params(const Tensor &table, const Tensor &lens, const Tensor &refs, int64_t page_size) {
  TORCH_CHECK_VALUE(table.is_cuda(), "the page tables must be on a CUDA device (no CPU path)");
  check_table(table, lens, table);
  check_int32(refs, 1, "page_refs", table);
  SbPagesParams p;
  memset(&p, 0, sizeof(p));
  p.struct_bytes = (int32_t)sizeof(p);
  p.max_seqs = to_int32(table.size(0), "sequences");
  p.max_pages = to_int32(table.size(1), "pages per sequence");
  p.num_pages = to_int32(refs.size(0), "pages");
  p.page_size = to_int32(page_size, "page_size");
  p.page_table = static_cast<int32_t *>(table.data_ptr());
  p.page_table_stride = table.stride(0);
  p.seq_lens = static_cast<int32_t *>(lens.data_ptr());
  p.page_refs = static_cast<int32_t *>(refs.data_ptr());
  p.status = status_ptr(table.get_device());
  return p;
}
void set_pools(SbPagesParams &p, const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &refs) {
  refuse_grad("the keeping of a cache's pages", {&k, &v});
  check_pools(k, v, true);
  TORCH_CHECK_VALUE(k.device() == table.device(), "page_table must be on the device of the cache");
  TORCH_CHECK_VALUE(k.size(-4) == refs.size(0), "page_refs must have an entry for each page of the cache");
  p.dtype = dtype_code(k.scalar_type());
  p.layers = k.dim() == 5 ? to_int32(k.size(0), "layers") : 1;
  p.kv_heads = to_int32(k.size(-3), "kv_heads");
  p.head_dim = to_int32(k.size(-1), "head_dim");
  p.k_cache = cache_arg(k);
  p.v_cache = cache_arg(v);
}
void listed(const Tensor &t, const char *name, const Tensor &table) {
  check_int32(t, 1, name, table);
}
void run_pages(SbPagesParams &p, int (*call)(const SbPagesParams *, void *), const char *what, const Tensor &table, bool scratch_needed) {
  c10::cuda::CUDAGuard guard(table.device());
  Tensor scratch;
  if (scratch_needed) {
    const size_t need = sb_kv_pages_workspace_bytes(&p);
    if (need == (size_t)-1) raise_library_error(what, -1);
    scratch = empty_cuda({(int64_t)need}, at::kByte, table);
    p.workspace = scratch.data_ptr();
    p.workspace_bytes = need;
  }
  count_launches(what, call(&p, stream_of(table)));
}

void kv_extend(const Tensor &table, const Tensor &lens, const Tensor &refs, const std::optional<Tensor> &counts, int64_t count,
               int64_t page_size) {
  SbPagesParams p = pages_params(table, lens, refs, page_size);
  if (counts.has_value()) {
    listed(*counts, "counts", table);
    TORCH_CHECK_VALUE(counts->size(0) == lens.size(0), "counts must have an entry for each entry of seq_lens");
    p.first = static_cast<const int32_t *>(counts->data_ptr());
  } else {
    p.count = to_int32(count, "counts");
  }
  run_pages(p, sb_kv_extend, "sb_kv_extend", table, true);
  for (const Tensor *t : {&table, &lens, &refs}) written(*t);
}
void kv_fork(const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lens, const Tensor &refs, const Tensor &src,
             const Tensor &dst) {
  check_pools(k, v, true);
  SbPagesParams p = pages_params(table, lens, refs, k.size(-2));
  set_pools(p, k, v, table, refs);
  listed(src, "src", table);
  listed(dst, "dst", table);
  TORCH_CHECK_VALUE(src.size(0) == dst.size(0), "src and dst must have the same number of entries");
  p.n = to_int32(src.size(0), "listed sequences");
  p.first = static_cast<const int32_t *>(src.data_ptr());
  p.second = static_cast<const int32_t *>(dst.data_ptr());
  run_pages(p, sb_kv_fork, "sb_kv_fork", table, true);
  for (const Tensor *t : {&k, &v, &table, &lens, &refs}) written(*t);
}
void kv_free(const Tensor &table, const Tensor &lens, const Tensor &refs, const Tensor &seqs, int64_t page_size) {
  SbPagesParams p = pages_params(table, lens, refs, page_size);
  listed(seqs, "seqs", table);
  p.n = to_int32(seqs.size(0), "listed sequences");
  p.first = static_cast<const int32_t *>(seqs.data_ptr());
  run_pages(p, sb_kv_free, "sb_kv_free", table, false);
  for (const Tensor *t : {&table, &lens, &refs}) written(*t);
}
void kv_compact(const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lens, const Tensor &refs) {
  check_pools(k, v, true);
  SbPagesParams p = pages_params(table, lens, refs, k.size(-2));
  set_pools(p, k, v, table, refs);
  run_pages(p, sb_kv_compact, "sb_kv_compact", table, true);
  for (const Tensor *t : {&k, &v, &table, &lens, &refs}) written(*t);
}

}  // namespace

PYBIND11_MODULE(_sb_torch, m) {
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const LibraryError &err) {
      set_python_error(err);
    }
  });
  m.def("attention", &attention, py::call_guard<py::gil_scoped_release>());
  m.def("forward", &forward, py::call_guard<py::gil_scoped_release>());
  m.def("backward", &backward, py::call_guard<py::gil_scoped_release>());
  m.def("decode", &decode, py::call_guard<py::gil_scoped_release>());
  m.def("append", &append, py::call_guard<py::gil_scoped_release>());
  m.def("kv_extend", &kv_extend, py::call_guard<py::gil_scoped_release>());
  m.def("kv_fork", &kv_fork, py::call_guard<py::gil_scoped_release>());
  m.def("kv_free", &kv_free, py::call_guard<py::gil_scoped_release>());
  m.def("kv_compact", &kv_compact, py::call_guard<py::gil_scoped_release>());
  m.def("tma_ready", &tma_ready);
  m.def("status_word", &status_word, py::call_guard<py::gil_scoped_release>());
  m.def("launches", [] { return g_launches.load(); });
}
