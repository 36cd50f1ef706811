// PyTorch operators over the C ABI of libfa_sm100.so (include/fa_sm100.h).
//
//   torch.ops.fav.fwd(q, k, v, causal, sm_scale) -> (out, lse)
//   torch.ops.fav.bwd(dout, q, k, v, out, lse, causal, sm_scale, deterministic=False)
//       -> (dq, dk, dv)
//   torch.ops.fav.status(device) -> the device's int32 status word
//   torch.ops.fav.merge_(acc_o, acc_lse, o, lse, first)  (ring: in-place LSE merge)
//   torch.ops.fav.rotary, rotary_qk                      (rotary positions, with gradients)
//   torch.ops.fav.kv_append, kv_read, decode, decode_lse (paged key/value cache)
//
// These are the only callers of the C core on the Python side
// (flash_attn_volta_b200/forward.py, backward.py, autograd.py): the
// reference's flash_attn_forward / flash_attn_backward
// (flash_attn_volta/triton_fa.py:291-397, triton_fa_bwd.py:587-700) become a
// few Python assertions plus one dispatcher call each.  Registered for the
// CUDA key only; shape functions for FakeTensor / meta tensors (torch.compile)
// and the autograd formula are registered from Python (ops.py).
//
// The operators take (B, S, H, D) fp16 / bf16 CUDA tensors (any strides: other
// layouts and misaligned views are copied), k / v with H_kv heads
// (H % H_kv == 0) and S_k rows, lse (B, H, S_q) fp32, and return contiguous
// tensors.  The Python wrappers check the reference's preconditions first;
// errors of the C ABI raise RuntimeError with the library's message.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <atomic>
#include <mutex>
#include <tuple>

#include "../../include/fa_sm100.h"

namespace {

int dtype_code(const at::Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16,
              "flash_attn_volta_b200: fp16 or bf16 tensors only, got ", t.scalar_type());
  return t.scalar_type() == at::kHalf ? FA_DTYPE_F16 : FA_DTYPE_BF16;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == FA_OK, what, " failed: ", fa_sm100_error_string(rc), " (code ", rc, ")");
}

// Contiguous (B, S, H, D) with a 16-byte aligned base (what the TMA tensor
// maps need): a view of another layout is copied, and so is a contiguous view
// whose storage offset breaks the alignment.
at::Tensor kernel_input(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 4, name, " must be (batch, seqlen, heads, head_dim)");
  at::Tensor c = t.contiguous();
  if (reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 != 0) c = c.clone();
  return c;
}

// The C ABI takes every extent from q and k, so each other tensor must have
// exactly the shape it implies, and every tensor must sit on q's device (a
// mismatch would otherwise become an out-of-bounds or peer read on the GPU).
void check_like(const at::Tensor& t, at::IntArrayRef sizes, const at::Tensor& q, const char* name) {
  TORCH_CHECK(t.sizes() == sizes, name, " has shape ", t.sizes(), ", expected ", sizes);
  TORCH_CHECK(t.device() == q.device(), name, " is on ", t.device(), ", q on ", q.device());
}

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k, v must have the same dtype");
  check_like(k, {q.size(0), k.size(1), k.size(2), q.size(3)}, q, "k");
  check_like(v, k.sizes(), q, "v");
  TORCH_CHECK(k.size(2) > 0 && q.size(2) % k.size(2) == 0,
              "the query heads must be a multiple of the key/value heads");
}

// One int32 status word per device, created on first use (make that first
// call before any CUDA graph capture).
constexpr int kMaxDev = 64;
std::mutex g_status_mu;
at::Tensor g_status[kMaxDev];

at::Tensor status_word(int64_t device) {
  TORCH_CHECK(device >= 0 && device < kMaxDev, "device index out of range");
  std::lock_guard<std::mutex> lock(g_status_mu);
  if (!g_status[device].defined()) {
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    g_status[device] =
        at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
  }
  return g_status[device];
}

std::tuple<at::Tensor, at::Tensor> fwd_cuda(const at::Tensor& q_in, const at::Tensor& k_in,
                                            const at::Tensor& v_in, bool causal, double sm_scale) {
  const at::Tensor q = kernel_input(q_in, "q");
  const at::Tensor k = kernel_input(k_in, "k");
  const at::Tensor v = kernel_input(v_in, "v");
  const int dt = dtype_code(q);
  check_qkv(q, k, v);
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), D = q.size(3);
  const int64_t Sk = k.size(1), Hkv = k.size(2);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = at::empty(q.sizes(), q.options());
  at::Tensor lse = at::empty({B, H, Sq}, q.options().dtype(at::kFloat));
  if (q.numel() == 0) return {out, lse};
  if (Sk == 0) {
    // no keys: every query row is fully masked (O = 0, LSE = +inf)
    out.zero_();
    lse.fill_(std::numeric_limits<float>::infinity());
    return {out, lse};
  }
  at::Tensor st = status_word(q.get_device());
  const int rc = fa_sm100_fwd_ex(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 lse.data_ptr<float>(), (int)B, (int)Sq, (int)Sk, (int)H,
                                 (int)Hkv, (int)D, dt, (float)sm_scale, causal ? 1 : 0,
                                 st.data_ptr<int>(), at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_fwd_ex");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bwd_cuda(
    const at::Tensor& dout_in, const at::Tensor& q_in, const at::Tensor& k_in,
    const at::Tensor& v_in, const at::Tensor& out_in, const at::Tensor& lse_in, bool causal,
    double sm_scale, bool deterministic) {
  const at::Tensor dout = kernel_input(dout_in, "dout");
  const at::Tensor q = kernel_input(q_in, "q");
  const at::Tensor k = kernel_input(k_in, "k");
  const at::Tensor v = kernel_input(v_in, "v");
  const at::Tensor out = kernel_input(out_in, "out");
  const int dt = dtype_code(q);
  check_qkv(q, k, v);
  TORCH_CHECK(dout.scalar_type() == q.scalar_type() && out.scalar_type() == q.scalar_type(),
              "dout and out must have q's dtype");
  TORCH_CHECK(lse_in.scalar_type() == at::kFloat, "lse must be fp32");
  const at::Tensor lse = lse_in.contiguous();
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), D = q.size(3);
  const int64_t Sk = k.size(1), Hkv = k.size(2);
  check_like(dout, q.sizes(), q, "dout");
  check_like(out, q.sizes(), q, "out");
  check_like(lse, {B, H, Sq}, q, "lse");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor dq = at::empty(q.sizes(), q.options());
  at::Tensor dk = at::empty(k.sizes(), k.options());
  at::Tensor dv = at::empty(v.sizes(), v.options());
  if (q.numel() == 0 || Sk == 0) {
    dq.zero_();
    dk.zero_();
    dv.zero_();
    return {dq, dk, dv};
  }
  const int flags = deterministic ? FA_BWD_DETERMINISTIC : 0;
  const size_t nbytes = fa_sm100_bwd_workspace_bytes_flags((int)B, (int)Sq, (int)H, (int)D, flags);
  TORCH_CHECK(nbytes > 0, "fa_sm100_bwd_workspace_bytes: unsupported shape");
  at::Tensor ws = at::empty({(int64_t)nbytes}, q.options().dtype(at::kByte));
  at::Tensor st = status_word(q.get_device());
  const int rc = fa_sm100_bwd_flags(
      dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
      lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), nbytes,
      (int)B, (int)Sq, (int)Sk, (int)H, (int)Hkv, (int)D, dt, (float)sm_scale, causal ? 1 : 0,
      flags, st.data_ptr<int>(), at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_bwd_flags");
  return {dq, dk, dv};
}

void merge_cuda(at::Tensor& acc_o, at::Tensor& acc_lse, const at::Tensor& o_in,
                const at::Tensor& lse_in, bool first) {
  TORCH_CHECK(acc_o.scalar_type() == at::kFloat && acc_o.is_contiguous(),
              "acc_o must be contiguous fp32");
  TORCH_CHECK(acc_lse.scalar_type() == at::kFloat && acc_lse.is_contiguous(),
              "acc_lse must be contiguous fp32");
  const at::Tensor o = kernel_input(o_in, "o");
  const at::Tensor lse = lse_in.contiguous();
  check_like(acc_o, o.sizes(), o, "acc_o");
  TORCH_CHECK(lse.scalar_type() == at::kFloat, "lse must be fp32");
  check_like(lse, {o.size(0), o.size(2), o.size(1)}, o, "lse");
  check_like(acc_lse, lse.sizes(), o, "acc_lse");
  c10::cuda::CUDAGuard guard(o.device());
  const int rc = fa_sm100_merge(acc_o.data_ptr<float>(), acc_lse.data_ptr<float>(), o.data_ptr(),
                                lse.data_ptr<float>(), (int)o.size(0), (int)o.size(1),
                                (int)o.size(2), (int)o.size(3), dtype_code(o), first ? 1 : 0,
                                at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_merge");
}

// The serving operators run on a few tokens at a time, where the host's steps
// are what counts: outputs are allocated without a dispatch, and the status
// word's address is kept.
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}

int* status_ptr(at::Device device) {
  static std::atomic<int*> kept[kMaxDev];
  const int i = device.index();
  if (i < 0 || i >= kMaxDev) return status_word(i).data_ptr<int>();  // refuses the index
  int* ptr = kept[i].load(std::memory_order_acquire);
  if (!ptr) {
    ptr = status_word(i).data_ptr<int>();
    kept[i].store(ptr, std::memory_order_release);
  }
  return ptr;
}

// ------------------------------------------------------------ rotary positions
using OptTensor = std::optional<at::Tensor>;

// (B, S, heads, D) as the C ABI takes it: any strides but a dense last
// dimension, pairs of elements 4-byte aligned where `pairs`; anything else is
// copied.
at::Tensor heads_input(const at::Tensor& t, const char* name, bool pairs) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == 4, name, " must be (batch, seqlen, heads, head_dim)");
  bool fine = t.size(3) <= 1 || t.stride(3) == 1;
  if (pairs) {
    fine = fine && reinterpret_cast<uintptr_t>(t.data_ptr()) % 4 == 0;
    for (int i = 0; i < 3; ++i) fine = fine && (t.size(i) <= 1 || t.stride(i) % 2 == 0);
  }
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

fa_sm100_heads heads_of(const at::Tensor& t, const at::Tensor* out) {
  fa_sm100_heads h;
  h.in = t.data_ptr();
  h.out = out ? out->data_ptr() : nullptr;
  // a dimension of one element has no stride worth keeping
  h.stride_batch = t.size(0) > 1 ? t.stride(0) : 0;
  h.stride_seq = t.size(1) > 1 ? t.stride(1) : 0;
  h.stride_head = t.size(2) > 1 ? t.stride(2) : 0;
  h.heads = (int)t.size(2);
  return h;
}

void check_freq(const at::Tensor& inv_freq, const at::Tensor& q) {
  TORCH_CHECK(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.size(0) > 0,
              "inv_freq must be a 1-D fp64 tensor");
  TORCH_CHECK(inv_freq.device() == q.device(), "inv_freq is on ", inv_freq.device(), ", q on ",
              q.device());
  TORCH_CHECK(2 * inv_freq.size(0) <= q.size(3) && q.size(3) % 2 == 0, "rotary dim ",
              2 * inv_freq.size(0), " does not fit head_dim ", q.size(3));
}

void rotary_launch(const at::Tensor& q_in, const at::Tensor* k_in, at::Tensor& q_out,
                   at::Tensor* k_out, const at::Tensor& inv_freq_in, const OptTensor& positions_in,
                   int64_t first, bool interleaved, double magnitude, bool inverse) {
  const at::Tensor q = heads_input(q_in, "q", interleaved);
  const int dt = dtype_code(q);
  check_freq(inv_freq_in, q);
  const at::Tensor inv_freq = inv_freq_in.contiguous();
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  at::Tensor k;
  if (k_in) {
    k = heads_input(*k_in, "k", interleaved);
    TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have the same dtype");
    check_like(k, {B, S, k.size(2), D}, q, "k");
  }
  at::Tensor positions;
  int64_t pos_stride = 0;
  if (positions_in) {
    positions = *positions_in;
    TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
                "positions must be int32 or int64");
    if (positions.dim() == 1) {
      check_like(positions, {S}, q, "positions");
    } else {
      check_like(positions, {B, S}, q, "positions");
    }
    if (S > 1 && positions.stride(-1) != 1) positions = positions.contiguous();
    pos_stride = positions.dim() == 2 && B > 1 ? positions.stride(0) : 0;
  }
  if (B * S == 0) return;
  const bool no_q = q.size(2) == 0, no_k = !k_in || k.size(2) == 0;
  if (no_q && no_k) return;
  fa_sm100_heads hq, hk;
  if (!no_q) hq = heads_of(q, &q_out);
  if (!no_k) hk = heads_of(k, k_out);
  const int rc = fa_sm100_rotary(
      no_q ? &hk : &hq, no_q || no_k ? nullptr : &hk, inv_freq.data_ptr<double>(),
      2 * (int)inv_freq.size(0), interleaved, (float)magnitude, inverse,
      positions.defined() ? positions.data_ptr() : nullptr,
      positions.defined() && positions.scalar_type() == at::kLong, pos_stride, first, (int)B, (int)S,
      (int)D, dt, at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_rotary");
}

at::Tensor rotary_cuda(const at::Tensor& x, const at::Tensor& inv_freq, const OptTensor& positions,
                       int64_t first, bool interleaved, double magnitude, bool inverse) {
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  at::Tensor out = new_tensor(x.sizes(), x.scalar_type(), x.device());
  rotary_launch(x, nullptr, out, nullptr, inv_freq, positions, first, interleaved, magnitude, inverse);
  return out;
}

std::tuple<at::Tensor, at::Tensor> rotary_qk_cuda(const at::Tensor& q, const at::Tensor& k,
                                                  const at::Tensor& inv_freq,
                                                  const OptTensor& positions, int64_t first,
                                                  bool interleaved, double magnitude, bool inverse) {
  c10::cuda::CUDAGuard guard(q.device());
  TORCH_CHECK(q.is_cuda() && k.device() == q.device(), "q and k must be on one CUDA device");
  at::Tensor qo = new_tensor(q.sizes(), q.scalar_type(), q.device());
  at::Tensor ko = new_tensor(k.sizes(), k.scalar_type(), k.device());
  rotary_launch(q, &k, qo, &ko, inv_freq, positions, first, interleaved, magnitude, inverse);
  return {qo, ko};
}

at::Tensor rotary_op(const at::Tensor& x, const at::Tensor& inv_freq, const OptTensor& positions,
                     int64_t first, bool interleaved, double magnitude, bool inverse) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("fav::rotary", "")
                       .typed<decltype(rotary_cuda)>();
  return op.call(x, inv_freq, positions, first, interleaved, magnitude, inverse);
}
std::tuple<at::Tensor, at::Tensor> rotary_qk_op(const at::Tensor& q, const at::Tensor& k,
                                                const at::Tensor& inv_freq,
                                                const OptTensor& positions, int64_t first,
                                                bool interleaved, double magnitude, bool inverse) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("fav::rotary_qk", "")
                       .typed<decltype(rotary_qk_cuda)>();
  return op.call(q, k, inv_freq, positions, first, interleaved, magnitude, inverse);
}

// The gradient of a rotation by a is the rotation by -a, through the same
// operators (so it has a gradient itself).
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

void save_turn(AutogradContext* ctx, const at::Tensor& inv_freq, const OptTensor& positions,
               int64_t first, bool interleaved, double magnitude, bool inverse) {
  ctx->save_for_backward({inv_freq, positions.value_or(at::Tensor())});
  ctx->saved_data["first"] = first;
  ctx->saved_data["interleaved"] = interleaved;
  ctx->saved_data["magnitude"] = magnitude;
  ctx->saved_data["inverse"] = inverse;
}

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& inv_freq,
                          const OptTensor& positions, int64_t first, bool interleaved,
                          double magnitude, bool inverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    save_turn(ctx, inv_freq, positions, first, interleaved, magnitude, inverse);
    return rotary_op(x, inv_freq, positions, first, interleaved, magnitude, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const OptTensor positions = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    at::Tensor dx;
    if (grads[0].defined())
      dx = rotary_op(grads[0], saved[0], positions, ctx->saved_data["first"].toInt(),
                     ctx->saved_data["interleaved"].toBool(), ctx->saved_data["magnitude"].toDouble(),
                     !ctx->saved_data["inverse"].toBool());
    return {dx, Variable(), Variable(), Variable(), Variable(), Variable(), Variable()};
  }
};

struct RotaryQkFn : public torch::autograd::Function<RotaryQkFn> {
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k,
                               const Variable& inv_freq, const OptTensor& positions, int64_t first,
                               bool interleaved, double magnitude, bool inverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    save_turn(ctx, inv_freq, positions, first, interleaved, magnitude, inverse);
    ctx->set_materialize_grads(false);
    auto [qo, ko] = rotary_qk_op(q, k, inv_freq, positions, first, interleaved, magnitude, inverse);
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const OptTensor positions = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    const int64_t first = ctx->saved_data["first"].toInt();
    const bool inter = ctx->saved_data["interleaved"].toBool();
    const double mag = ctx->saved_data["magnitude"].toDouble();
    const bool inv = !ctx->saved_data["inverse"].toBool();
    const bool want_q = grads[0].defined() && ctx->needs_input_grad(0);
    const bool want_k = grads[1].defined() && ctx->needs_input_grad(1);
    at::Tensor dq, dk;
    if (want_q && want_k) {
      std::tie(dq, dk) = rotary_qk_op(grads[0], grads[1], saved[0], positions, first, inter, mag, inv);
    } else if (want_q) {
      dq = rotary_op(grads[0], saved[0], positions, first, inter, mag, inv);
    } else if (want_k) {
      dk = rotary_op(grads[1], saved[0], positions, first, inter, mag, inv);
    }
    return {dq, dk, Variable(), Variable(), Variable(), Variable(), Variable(), Variable()};
  }
};

// What an operator has no derivative for is refused, not dropped: a forward-mode
// tangent (as the C++ autograd functions do themselves), or a gradient of
// `reverse` tensors.
bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
void check_derivatives(const char* op, std::initializer_list<const at::Tensor*> forward,
                       std::initializer_list<const at::Tensor*> reverse) {
  for (const at::Tensor* t : forward)
    TORCH_CHECK(!t || !has_tangent(*t), op, ": forward-mode derivatives are not implemented");
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : reverse)
    TORCH_CHECK(!t || !t->defined() || !t->requires_grad(), op, ": ",
                "no gradient is computed for a tensor that requires one (detach it, or call under no_grad)");
}
const at::Tensor* ptr(const OptTensor& t) { return t ? &*t : nullptr; }

at::Tensor rotary_autograd(const at::Tensor& x, const at::Tensor& inv_freq,
                           const OptTensor& positions, int64_t first, bool interleaved,
                           double magnitude, bool inverse) {
  check_derivatives("rotary", {&x, &inv_freq}, {&inv_freq});
  if (at::GradMode::is_enabled() && x.requires_grad())
    return RotaryFn::apply(x, inv_freq, positions, first, interleaved, magnitude, inverse);
  at::AutoDispatchBelowADInplaceOrView below;
  return rotary_op(x, inv_freq, positions, first, interleaved, magnitude, inverse);
}

std::tuple<at::Tensor, at::Tensor> rotary_qk_autograd(const at::Tensor& q, const at::Tensor& k,
                                                      const at::Tensor& inv_freq,
                                                      const OptTensor& positions, int64_t first,
                                                      bool interleaved, double magnitude,
                                                      bool inverse) {
  check_derivatives("rotary_qk", {&q, &k, &inv_freq}, {&inv_freq});
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())) {
    auto r = RotaryQkFn::apply(q, k, inv_freq, positions, first, interleaved, magnitude, inverse);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return rotary_qk_op(q, k, inv_freq, positions, first, interleaved, magnitude, inverse);
}

// ------------------------------------------------------------ key/value cache
// 16-bit: two page tensors; 4-bit (v_pages absent): blocks of 20 * head_dim bytes.
fa_sm100_kv_cache cache_of(const at::Tensor& k_pages, const OptTensor& v_pages, int dtype) {
  TORCH_CHECK(k_pages.is_cuda(), "the cache must be a CUDA tensor");
  TORCH_CHECK(k_pages.dim() == 4 && k_pages.is_contiguous(), "cache pages must be contiguous and 4-D");
  fa_sm100_kv_cache c;
  c.k_pages = k_pages.data_ptr();
  c.num_pages = (int)k_pages.size(0);
  c.nheads_kv = (int)k_pages.size(1);
  c.dtype = dtype;
  TORCH_CHECK(k_pages.size(0) <= 2147483647 && k_pages.size(1) <= 2147483647, "too many pages");
  if (v_pages) {
    TORCH_CHECK(dtype_code(k_pages) == dtype, "the tensors must have the cache's dtype");
    TORCH_CHECK(v_pages->scalar_type() == k_pages.scalar_type() && v_pages->is_contiguous(),
                "v_pages must be contiguous, of k_pages' dtype");
    check_like(*v_pages, k_pages.sizes(), k_pages, "v_pages");
    c.v_pages = v_pages->data_ptr();
    c.page_size = (int)k_pages.size(2);
    c.head_dim = (int)k_pages.size(3);
    c.bits = 16;
  } else {
    TORCH_CHECK(k_pages.scalar_type() == at::kByte && k_pages.size(3) % 20 == 0,
                "4-bit pages must be uint8 (pages, kv heads, page_size / 16, 20 * head_dim)");
    c.v_pages = nullptr;
    c.page_size = (int)k_pages.size(2) * 16;
    c.head_dim = (int)k_pages.size(3) / 20;
    c.bits = 4;
  }
  return c;
}

// (batch, ...) int32, on the cache's device, contiguous.
at::Tensor int_input(const at::Tensor& t, int64_t dim, int64_t batch, const at::Tensor& pages,
                     const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim && t.size(0) == batch, name,
              " must be int32 with ", dim, " dimension(s), the first of ", batch);
  TORCH_CHECK(t.device() == pages.device(), name, " is on ", t.device(), ", the cache on ",
              pages.device());
  return t.contiguous();
}

at::Tensor kv_append_cuda(const at::Tensor& k_pages, const OptTensor& v_pages, const at::Tensor& k_in,
                          const at::Tensor& v_in, const OptTensor& q_in,
                          const at::Tensor& table_in, const at::Tensor& starts_in,
                          const OptTensor& counts_in, const OptTensor& freq_in, bool interleaved,
                          double magnitude) {
  const at::Tensor k = heads_input(k_in, "k", false), v = heads_input(v_in, "v", false);
  const int dt = dtype_code(k);
  const fa_sm100_kv_cache cache = cache_of(k_pages, v_pages, dt);
  const int64_t B = k.size(0), S = k.size(1), D = k.size(3);
  check_like(k, {B, S, cache.nheads_kv, cache.head_dim}, k_pages, "k");
  check_like(v, k.sizes(), k, "v");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), "k and v must have the same dtype");
  at::Tensor q, q_out;
  c10::cuda::CUDAGuard guard(k_pages.device());
  if (q_in) {
    q = heads_input(*q_in, "q", false);
    check_like(q, {B, S, q.size(2), D}, k, "q");
    TORCH_CHECK(q.scalar_type() == k.scalar_type(), "q must have k's dtype");
    q_out = new_tensor(q.sizes(), q.scalar_type(), q.device());
  } else {
    q_out = new_tensor({0}, k.scalar_type(), k.device());
  }
  const at::Tensor table = int_input(table_in, 2, B, k_pages, "page_table");
  const at::Tensor starts = int_input(starts_in, 1, B, k_pages, "starts");
  at::Tensor counts, freq;
  if (counts_in) counts = int_input(*counts_in, 1, B, k_pages, "counts");
  if (freq_in) {
    check_freq(*freq_in, k);
    freq = freq_in->contiguous();
  }
  if (B * S == 0) return q_out;
  const fa_sm100_heads hk = heads_of(k, nullptr), hv = heads_of(v, nullptr);
  fa_sm100_heads hq;
  const bool with_q = q.defined() && q.size(2) > 0;
  if (with_q) hq = heads_of(q, &q_out);
  const int rc = fa_sm100_kv_append(
      &cache, &hk, &hv, with_q ? &hq : nullptr, table.data_ptr<int>(), (int)table.size(1),
      starts.data_ptr<int>(), counts.defined() ? counts.data_ptr<int>() : nullptr,
      freq.defined() ? freq.data_ptr<double>() : nullptr,
      freq.defined() ? 2 * (int)freq.size(0) : 0, interleaved, (float)magnitude, (int)B, (int)S,
      status_ptr(k_pages.device()), at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_kv_append");
  return q_out;
}

std::tuple<at::Tensor, at::Tensor> kv_read_cuda(const at::Tensor& k_pages, const OptTensor& v_pages,
                                                at::ScalarType dtype, const at::Tensor& table_in,
                                                const at::Tensor& lengths_in, int64_t max_len) {
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, "fp16 or bf16 only");
  const fa_sm100_kv_cache cache =
      cache_of(k_pages, v_pages, dtype == at::kHalf ? FA_DTYPE_F16 : FA_DTYPE_BF16);
  const int64_t B = lengths_in.numel();
  const at::Tensor table = int_input(table_in, 2, B, k_pages, "page_table");
  const at::Tensor lengths = int_input(lengths_in, 1, B, k_pages, "lengths");
  TORCH_CHECK(max_len >= 0 && max_len <= 2147483647, "max_len out of range");
  c10::cuda::CUDAGuard guard(k_pages.device());
  at::Tensor k = new_tensor({B, max_len, cache.nheads_kv, cache.head_dim}, dtype, k_pages.device());
  at::Tensor v = new_tensor({B, max_len, cache.nheads_kv, cache.head_dim}, dtype, k_pages.device());
  if (B == 0 || max_len == 0) return {k, v};
  const int rc = fa_sm100_kv_read(&cache, table.data_ptr<int>(), (int)table.size(1),
                                  lengths.data_ptr<int>(), k.data_ptr(), v.data_ptr(), (int)B,
                                  (int)max_len, status_ptr(k_pages.device()),
                                  at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_kv_read");
  return {k, v};
}

// out, and lse if it is not null.
at::Tensor decode_launch(const at::Tensor& q_in, const at::Tensor& k_pages,
                         const OptTensor& v_pages, const at::Tensor& table_in,
                         const at::Tensor& lengths_in, const OptTensor& starts_in, bool causal,
                         double sm_scale, at::Tensor* lse) {
  const at::Tensor q = kernel_input(q_in, "q");
  const fa_sm100_kv_cache cache = cache_of(k_pages, v_pages, dtype_code(q));
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2);
  check_like(q, {B, S, H, cache.head_dim}, k_pages, "q");
  TORCH_CHECK(H > 0 && cache.nheads_kv > 0 && H % cache.nheads_kv == 0,
              "the query heads must be a multiple of the cache's heads");
  const at::Tensor table = int_input(table_in, 2, B, k_pages, "page_table");
  const at::Tensor lengths = int_input(lengths_in, 1, B, k_pages, "lengths");
  at::Tensor starts;
  if (starts_in) starts = int_input(*starts_in, 1, B, k_pages, "starts");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = new_tensor(q.sizes(), q.scalar_type(), q.device());
  if (lse) *lse = new_tensor({B, H, S}, at::kFloat, q.device());
  if (B * S == 0) return out;
  const size_t nbytes = fa_sm100_decode_workspace_bytes(&cache, (int)table.size(1), (int)B, (int)S, (int)H);
  TORCH_CHECK(nbytes > 0, "fa_sm100_decode: unsupported shape");
  // 256 bytes mean that the shape needs none
  at::Tensor ws;
  if (nbytes > 256) ws = new_tensor({(int64_t)nbytes}, at::kByte, q.device());
  const int rc = fa_sm100_decode(
      &cache, q.data_ptr(), out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr,
      table.data_ptr<int>(), (int)table.size(1), lengths.data_ptr<int>(),
      starts.defined() ? starts.data_ptr<int>() : nullptr,
      ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? nbytes : 0, (int)B, (int)S,
      (int)H, (float)sm_scale, causal ? 1 : 0, status_ptr(q.device()),
      at::cuda::getCurrentCUDAStream().stream());
  check_rc(rc, "fa_sm100_decode");
  return out;
}

at::Tensor decode_cuda(const at::Tensor& q, const at::Tensor& k_pages, const OptTensor& v_pages,
                       const at::Tensor& table, const at::Tensor& lengths, const OptTensor& starts,
                       bool causal, double sm_scale) {
  return decode_launch(q, k_pages, v_pages, table, lengths, starts, causal, sm_scale, nullptr);
}
std::tuple<at::Tensor, at::Tensor> decode_lse_cuda(const at::Tensor& q, const at::Tensor& k_pages,
                                                   const OptTensor& v_pages, const at::Tensor& table,
                                                   const at::Tensor& lengths, const OptTensor& starts,
                                                   bool causal, double sm_scale) {
  at::Tensor lse;
  at::Tensor out = decode_launch(q, k_pages, v_pages, table, lengths, starts, causal, sm_scale, &lse);
  return {out, lse};
}

// The cache operators are for inference: under autograd they check that nothing
// asks for a derivative, and go on below it.
template <typename F>
auto below_autograd(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
at::Tensor kv_append_autograd(const at::Tensor& k_pages, const OptTensor& v_pages, const at::Tensor& k,
                              const at::Tensor& v, const OptTensor& q, const at::Tensor& table,
                              const at::Tensor& starts, const OptTensor& counts, const OptTensor& freq,
                              bool interleaved, double magnitude) {
  const auto all = {&k_pages, ptr(v_pages), &k, &v, ptr(q), ptr(freq)};
  check_derivatives("kv_append", all, all);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = below_autograd("fav::kv_append", kv_append_cuda);
  return op.call(k_pages, v_pages, k, v, q, table, starts, counts, freq, interleaved, magnitude);
}
std::tuple<at::Tensor, at::Tensor> kv_read_autograd(const at::Tensor& k_pages, const OptTensor& v_pages,
                                                    at::ScalarType dtype, const at::Tensor& table,
                                                    const at::Tensor& lengths, int64_t max_len) {
  const auto all = {&k_pages, ptr(v_pages)};
  check_derivatives("kv_read", all, all);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = below_autograd("fav::kv_read", kv_read_cuda);
  return op.call(k_pages, v_pages, dtype, table, lengths, max_len);
}
at::Tensor decode_autograd(const at::Tensor& q, const at::Tensor& k_pages, const OptTensor& v_pages,
                           const at::Tensor& table, const at::Tensor& lengths, const OptTensor& starts,
                           bool causal, double sm_scale) {
  const auto all = {&q, &k_pages, ptr(v_pages)};
  check_derivatives("decode", all, all);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = below_autograd("fav::decode", decode_cuda);
  return op.call(q, k_pages, v_pages, table, lengths, starts, causal, sm_scale);
}
std::tuple<at::Tensor, at::Tensor> decode_lse_autograd(const at::Tensor& q, const at::Tensor& k_pages,
                                                       const OptTensor& v_pages, const at::Tensor& table,
                                                       const at::Tensor& lengths, const OptTensor& starts,
                                                       bool causal, double sm_scale) {
  const auto all = {&q, &k_pages, ptr(v_pages)};
  check_derivatives("decode_lse", all, all);
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = below_autograd("fav::decode_lse", decode_lse_cuda);
  return op.call(q, k_pages, v_pages, table, lengths, starts, causal, sm_scale);
}

}  // namespace

TORCH_LIBRARY(fav, m) {
  m.def("fwd(Tensor q, Tensor k, Tensor v, bool causal, float sm_scale) -> (Tensor, Tensor)");
  m.def(
      "bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, bool causal, "
      "float sm_scale, bool deterministic=False) -> (Tensor, Tensor, Tensor)");
  m.def("status(int device) -> Tensor", &status_word);
  m.def("merge_(Tensor(a!) acc_o, Tensor(b!) acc_lse, Tensor o, Tensor lse, bool first) -> ()");
  m.def(
      "rotary(Tensor x, Tensor inv_freq, Tensor? positions, int first, bool interleaved, "
      "float magnitude, bool inverse) -> Tensor");
  m.def(
      "rotary_qk(Tensor q, Tensor k, Tensor inv_freq, Tensor? positions, int first, "
      "bool interleaved, float magnitude, bool inverse) -> (Tensor, Tensor)");
  m.def(
      "kv_append(Tensor(a!) k_pages, Tensor(b!)? v_pages, Tensor k, Tensor v, Tensor? q, "
      "Tensor page_table, Tensor starts, Tensor? counts, Tensor? inv_freq, bool interleaved, "
      "float magnitude) -> Tensor");
  m.def(
      "kv_read(Tensor k_pages, Tensor? v_pages, ScalarType dtype, Tensor page_table, "
      "Tensor lengths, int max_len) -> (Tensor, Tensor)");
  m.def(
      "decode(Tensor q, Tensor k_pages, Tensor? v_pages, Tensor page_table, Tensor lengths, "
      "Tensor? starts, bool causal, float sm_scale) -> Tensor");
  m.def(
      "decode_lse(Tensor q, Tensor k_pages, Tensor? v_pages, Tensor page_table, Tensor lengths, "
      "Tensor? starts, bool causal, float sm_scale) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(fav, CUDA, m) {
  m.impl("fwd", &fwd_cuda);
  m.impl("bwd", &bwd_cuda);
  m.impl("merge_", &merge_cuda);
  m.impl("rotary", &rotary_cuda);
  m.impl("rotary_qk", &rotary_qk_cuda);
  m.impl("kv_append", &kv_append_cuda);
  m.impl("kv_read", &kv_read_cuda);
  m.impl("decode", &decode_cuda);
  m.impl("decode_lse", &decode_lse_cuda);
}

TORCH_LIBRARY_IMPL(fav, Autograd, m) {
  m.impl("rotary", &rotary_autograd);
  m.impl("rotary_qk", &rotary_qk_autograd);
  m.impl("kv_append", &kv_append_autograd);
  m.impl("kv_read", &kv_read_autograd);
  m.impl("decode", &decode_autograd);
  m.impl("decode_lse", &decode_lse_autograd);
}
