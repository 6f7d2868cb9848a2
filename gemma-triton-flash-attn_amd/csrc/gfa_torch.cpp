// Native host path of the PyTorch entry points: the same calls into the C ABI that attention.py makes
// through ctypes (allocation of the outputs, the argument block, the launch), as C++ on ATen
// tensors, with the autograd node in C++ too.
//
// Why: on a short sequence the kernels take 30-100 us and the host path took longer. A Python autograd
// function's backward runs on the engine's device thread, which must first take the interpreter
// lock from the thread that waits for it; a plain backward here never touches the interpreter. Host
// time per call at N=128, ctypes path against this one: forward and backward 165 -> 77 us (an elementwise
// product's takes 59 on the same host: the rest is the engine's thread), a transformers layer
// without gradients 55 -> 19 us, inference 16 -> 8 us.
//
// Arguments arrive checked (attention.py: _check_inputs, _norm_window, ...). Only what depends on
// this call's tensors is decided here, by attention.py's rules: copies of inputs whose layout the
// ABI cannot address, outputs in the input's layout where it can. Nothing is kept between calls.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <optional>

#include "gfa.h"

namespace py = pybind11;
using at::Tensor;

namespace {

// The C ABI of the library that the Python binding has loaded, and its exception type.
struct Api {
  decltype(&gfa_fwd) fwd = nullptr;
  decltype(&gfa_bwd) bwd = nullptr;
  decltype(&gfa_bwd_workspace_bytes) workspace_bytes = nullptr;
  decltype(&gfa_segments_from_positions) positions = nullptr;
  decltype(&gfa_kv4_write) kv4_write = nullptr;
  decltype(&gfa_kv4_read) kv4_read = nullptr;
  decltype(&gfa_kv4_plan) kv4_plan = nullptr;
  decltype(&gfa_kv4_attn) kv4_attn = nullptr;
  decltype(&gfa_kv4_attn_workspace_bytes) kv4_attn_workspace_bytes = nullptr;
  decltype(&gfa_kv4_fork) kv4_fork = nullptr;
  decltype(&gfa_kv4_compact) kv4_compact = nullptr;
  decltype(&gfa_kv4_pages_workspace_bytes) kv4_pages_workspace_bytes = nullptr;
  decltype(&gfa_kv4_copy) kv4_copy = nullptr;
  decltype(&gfa_kv4_share) kv4_share = nullptr;
  decltype(&gfa_kv4_verify) kv4_verify = nullptr;
  decltype(&gfa_kv4_verify_workspace_bytes) kv4_verify_workspace_bytes = nullptr;
  decltype(&gfa_last_error) last_error = nullptr;
  PyObject* error_type = nullptr;  // GfaError(status, message); held for the process
} api;

// A non-zero status as the Python binding raises it. Called with or without the interpreter lock;
// python_error carries the exception through the autograd engine's threads.
void check(int status) {
  if (status == 0) return;
  const std::string message = api.last_error();  // this thread's
  py::gil_scoped_acquire gil;
  PyObject* e = PyObject_CallFunction(api.error_type, "is", status, message.c_str());
  if (e != nullptr) {
    PyErr_SetObject(api.error_type, e);
    Py_DECREF(e);
  }
  python_error err;
  err.persist();
  throw err;
}

constexpr int64_t kSliceLimit = 0xFFFFFFFFll;  // attention.py, _layout_ok
constexpr int64_t kTileOverrun = 128;

bool needs_copy(const Tensor& t) {
  const auto s = t.strides();
  if (s[3] != 1) return true;
  for (int i = 0; i < 3; ++i)
    if (s[i] % 8 != 0 || s[i] < 0) return true;
  if (((t.size(2) - 1 + kTileOverrun) * s[2] + t.size(3)) * t.element_size() > kSliceLimit) return true;
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0;
}
Tensor prep(const Tensor& t) {
  if (t.is_neg()) return prep(t.resolve_neg());  // a view that negates on reading
  return needs_copy(t) ? t.contiguous() : t;
}
// An output with t's layout, or contiguous where the ABI cannot address that layout.
Tensor out_like(const Tensor& t) {
  Tensor o = at::empty_like(t);
  return needs_copy(o) ? at::empty(t.sizes(), t.options()) : o;
}

gfa_strides strides_of(const Tensor& t) { return gfa_strides{t.stride(0), t.stride(1), t.stride(2)}; }
int64_t lse_ld(int64_t n) { return (n + 63) / 64 * 64; }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? GFA_DTYPE_BF16 : GFA_DTYPE_FP16; }
void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

struct Options {
  bool causal;
  int64_t window;
  double scale, softcap, dropout_p;
  int64_t seed, block_kv;
  Tensor lo, hi;       // segment tables, or undefined
  bool as_op = false;  // autograd as the registered op's (Attention)
};

// O, and the LSE where asked for, of prepared inputs. Profilers list it, and the backward below, under
// the registered ops' names.
std::pair<Tensor, Tensor> forward_call(const Tensor& q, const Tensor& k, const Tensor& v, const Options& x,
                                       bool store_lse) {
  RECORD_FUNCTION("gfa::attn_fwd", c10::ArrayRef<const c10::IValue>{});
  const c10::DeviceGuard on_device(q.device());
  Tensor o = out_like(q);
  const int64_t ld = lse_ld(q.size(2));
  Tensor lse;
  if (store_lse) lse = at::empty({q.size(0), q.size(1), ld}, q.options().dtype(at::kFloat));
  gfa_fwd_args a{};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = o.data_ptr();
  a.lse = store_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  a.q_strides = strides_of(q);
  a.k_strides = strides_of(k);
  a.v_strides = strides_of(v);
  a.o_strides = strides_of(o);
  a.batch = (int32_t)q.size(0);
  a.heads_q = (int32_t)q.size(1);
  a.heads_kv = (int32_t)k.size(1);
  a.seq_len = (int32_t)q.size(2);
  a.head_dim = (int32_t)q.size(3);
  a.causal = x.causal;
  a.window = (int32_t)x.window;
  a.scale = (float)x.scale;
  a.dtype = dtype_of(q);
  a.block_kv = (int32_t)x.block_kv;
  a.lse_ld = (int32_t)ld;
  a.softcap = (float)x.softcap;
  a.dropout_p = (float)x.dropout_p;
  a.dropout_seed = (uint64_t)x.seed;
  a.stream = stream_of(q);
  if (x.lo.defined()) {
    a.seg_lo = static_cast<const int32_t*>(x.lo.data_ptr());
    a.seg_hi = static_cast<const int32_t*>(x.hi.data_ptr());
  }
  check(api.fwd(&a));
  return {o, lse};
}

// Whether something stands between the engine and the tensors of a backward that a launch on their
// pointers would pass by: compiled autograd's or a subclass's stand-ins for them, batched
// gradients, zeros without memory, a dispatch mode, a trace.
bool watched(const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet keys({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched,
                                      DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched, DispatchKey::ZeroTensor});
  return t.key_set().has_any(keys);
}
bool watched(const torch::autograd::variable_list& tensors) {
  using c10::DispatchKey;
  for (const auto key : {DispatchKey::Python, DispatchKey::FuncTorchDynamicLayerFrontMode, DispatchKey::Tracer})
    if (c10::impl::tls_is_dispatch_key_included(key)) return true;
  for (const Tensor& t : tensors)
    if (t.defined() && watched(t)) return true;
  return false;
}

// dQ, dK, dV through the registered op gfa::attn_bwd (ops.py).
std::tuple<Tensor, Tensor, Tensor> backward_op(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                                               const Tensor& lse, const Tensor& dout, const Options& x,
                                               const Tensor& seed) {
  using Maybe = std::optional<Tensor>;
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("gfa::attn_bwd", "")
          .typed<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                    const Tensor&, const Tensor&, bool, c10::SymInt, double,
                                                    const Maybe&, const Maybe&, double, double, const Maybe&)>();
  const auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
  return op.call(q, k, v, o, lse, dout, x.causal, x.window, x.scale, maybe(x.lo), maybe(x.hi), x.softcap, x.dropout_p,
                 maybe(seed));
}

// The autograd node of a call. With as_op (the transformers adapter, which is the registered op
// gfa::attn_fwd everywhere else) a backward that itself records a graph (create_graph) calls the
// op gfa::attn_bwd too: its gradients then refuse to be differentiated again, where the launch
// below would give gradients without a graph and drop the second-order terms. Any watched
// backward calls that op as well, so compiled autograd traces it into its one graph.
struct Attention : public torch::autograd::Function<Attention> {
  static constexpr bool is_traceable = true;

  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const Options& x) {
    auto [o, lse] = forward_call(prep(q), prep(k), prep(v), x, true);
    torch::autograd::variable_list saved{q, k, v, o, lse};
    if (x.lo.defined()) saved.insert(saved.end(), {x.lo, x.hi});
    // As the op does, a one-element CPU tensor: a compiled backward takes another seed each time.
    if (x.as_op && x.dropout_p > 0.0) saved.push_back(at::full({1}, x.seed, at::kLong));
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["whole"] = std::vector<int64_t>{x.causal, x.window, x.seed, x.as_op, x.lo.defined()};
    ctx->saved_data["real"] = std::vector<double>{x.scale, x.softcap, x.dropout_p};
    return o;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &o = saved[3], &lse = saved[4];
    const auto whole = ctx->saved_data["whole"].toIntVector();
    const auto real = ctx->saved_data["real"].toDoubleVector();
    Options x{whole[0] != 0, whole[1], real[0], real[1], real[2], whole[2]};
    x.as_op = whole[3] != 0;
    if (whole[4] != 0) {
      x.lo = saved[5];
      x.hi = saved[6];
    }
    Tensor seed;
    if (x.dropout_p > 0.0 && x.as_op) seed = saved.back();
    if ((x.as_op && at::GradMode::is_enabled()) || watched(grads) || watched(saved)) {
      if (x.dropout_p > 0.0 && !x.as_op) seed = at::full({1}, x.seed, at::kLong);
      auto [dq, dk, dv] = backward_op(saved[0], saved[1], saved[2], o, lse, grads[0], x, seed);
      return {dq, dk, dv, Tensor()};
    }
    RECORD_FUNCTION("gfa::attn_bwd", c10::ArrayRef<const c10::IValue>{});
    if (seed.defined()) x.seed = seed.item<int64_t>();
    const Tensor q = prep(saved[0]), k = prep(saved[1]), v = prep(saved[2]);
    const c10::DeviceGuard on_device(q.device());
    Tensor dout = prep(grads[0]);
    if (dout.scalar_type() != q.scalar_type()) dout = dout.to(q.scalar_type());
    Tensor dq = out_like(q), dk = out_like(k), dv = out_like(v);
    Tensor delta = at::empty(lse.sizes(), lse.options());
    gfa_bwd_args a{};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.o = o.data_ptr();
    a.dout = dout.data_ptr();
    a.lse = static_cast<const float*>(lse.data_ptr());
    a.delta = static_cast<float*>(delta.data_ptr());
    a.dq = dq.data_ptr();
    a.dk = dk.data_ptr();
    a.dv = dv.data_ptr();
    a.q_strides = strides_of(q);
    a.k_strides = strides_of(k);
    a.v_strides = strides_of(v);
    a.o_strides = strides_of(o);
    a.do_strides = strides_of(dout);
    a.dq_strides = strides_of(dq);
    a.dk_strides = strides_of(dk);
    a.dv_strides = strides_of(dv);
    a.batch = (int32_t)q.size(0);
    a.heads_q = (int32_t)q.size(1);
    a.heads_kv = (int32_t)k.size(1);
    a.seq_len = (int32_t)q.size(2);
    a.head_dim = (int32_t)q.size(3);
    a.causal = x.causal;
    a.window = (int32_t)x.window;
    a.scale = (float)x.scale;
    a.dtype = dtype_of(q);
    a.lse_ld = (int32_t)lse.size(2);
    a.softcap = (float)x.softcap;
    a.dropout_p = (float)x.dropout_p;
    a.dropout_seed = (uint64_t)x.seed;
    a.stream = stream_of(q);
    if (x.lo.defined()) {
      a.seg_lo = static_cast<const int32_t*>(x.lo.data_ptr());
      a.seg_hi = static_cast<const int32_t*>(x.hi.data_ptr());
    }
    Tensor ws;
    const size_t need = api.workspace_bytes(&a);
    if (need > 0) {
      ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      a.workspace = ws.data_ptr();
      a.workspace_bytes = need;
    }
    check(api.bwd(&a));
    return {dq, dk, dv, Tensor()};
  }
};

// ---- The key/value cache in 4 bits (kv4.py): argument checks, outputs, launches ----

bool on_gpu(const Tensor& t, const c10::Device& device) { return t.is_cuda() && t.device() == device; }
// A caller's array of one type on the call's GPU.
void check_array(const char* name, const Tensor& t, at::ScalarType type, int64_t dim, const c10::Device& device) {
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == dim, name, " must be ", dim, "-D, got shape ", t.sizes());
  TORCH_CHECK_VALUE(on_gpu(t, device), name, " must be on the call's GPU (", device, "; the engine has no CPU path), is on ",
                    t.device());
}
Tensor dense(const Tensor& t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }

bool block_size_ok(int64_t n) { return n >= 32 && n <= 1024 && (n & (n - 1)) == 0; }

gfa_kv4_cache cache_of(const Tensor& codes, const Tensor& scales, bool bf16) {
  gfa_kv4_cache c{};
  c.codes = codes.data_ptr();
  c.scales = scales.data_ptr();
  c.num_blocks = (int32_t)codes.size(0);
  c.heads_kv = (int32_t)codes.size(1);
  c.block_size = (int32_t)codes.size(3);
  c.head_dim = (int32_t)(2 * codes.size(4));
  c.dtype = bf16 ? GFA_DTYPE_BF16 : GFA_DTYPE_FP16;
  return c;
}

void check_cache(const Tensor& codes, const Tensor& scales) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, "codes and scales must be uint8");
  TORCH_CHECK_VALUE(codes.dim() == 5 && scales.dim() == 5,
                    "codes and scales must be 5-D (num_blocks, heads_kv, 2, block_size, bytes)");
  const auto c = codes.sizes(), s = scales.sizes();
  const int64_t d = 2 * c[4];
  TORCH_CHECK_VALUE(d == 64 || d == 128 || d == 256 || d == 512, "HEAD_DIM=", d, " not built (64, 128, 256, 512)");
  TORCH_CHECK_VALUE(c[2] == 2 && s[0] == c[0] && s[1] == c[1] && s[2] == 2 && s[3] == c[3] && s[4] * 16 == c[4], "codes ", c,
                    " and scales ", s, " do not belong together");
  TORCH_CHECK_VALUE(block_size_ok(c[3]), "block_size=", c[3], " must be a power of two, 32 to 1024");
  TORCH_CHECK_VALUE(c[0] > 0 && c[0] <= INT32_MAX && c[1] > 0 && c[1] <= 65535, "a cache of ", c[0], " blocks and ", c[1], " heads");
  TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous() && !codes.is_neg() && !scales.is_neg(),
                    "codes and scales must be contiguous");
  TORCH_CHECK_VALUE(codes.is_cuda() && on_gpu(scales, codes.device()),
                    "codes and scales must be on one GPU (the engine has no CPU path)");
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(codes.const_data_ptr()) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(scales.const_data_ptr()) % 16 == 0,
                    "codes and scales must be 16-byte aligned");
}

void check_token_rows(const char* name, const Tensor& t, const Tensor& codes, bool bf16, bool kv) {
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be 4-D (B, H, N, D), got shape ", t.sizes());
  const auto type = bf16 ? at::kBFloat16 : at::kHalf;
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " is ", t.scalar_type(), ", the cache is for ", type);
  TORCH_CHECK_VALUE(t.size(3) == 2 * codes.size(4) && (!kv || t.size(1) == codes.size(1)), name, " ", t.sizes(),
                    " does not fit a cache of ", codes.size(1), " heads of dim ", 2 * codes.size(4));
  TORCH_CHECK_VALUE(on_gpu(t, codes.device()), name, " must be on the cache's GPU (", codes.device(), "), is on ", t.device());
  TORCH_CHECK_VALUE(t.size(0) * t.size(2) <= INT32_MAX, name, " has more than 2^31 - 1 tokens");
}

// Rows apart of an int32 (requests, width) block table.
int64_t check_table(const Tensor& table, int64_t requests, const c10::Device& device) {
  check_array("table", table, at::kInt, 2, device);
  TORCH_CHECK_VALUE(table.size(0) == requests, "table has ", table.size(0), " rows for ", requests, " requests");
  TORCH_CHECK_VALUE(requests > 0 && table.size(1) > 0 && requests < INT32_MAX && table.size(1) <= INT32_MAX,
                    "a block table of shape ", table.sizes());
  TORCH_CHECK_VALUE((table.stride(1) == 1 || table.size(1) == 1) && (requests == 1 || table.stride(0) >= table.size(1)) && !table.is_neg(),
                    "table rows must be contiguous and apart from each other");
  return requests == 1 ? table.size(1) : table.stride(0);
}

// A tensor over part of a buffer's memory: outputs of one call from one allocation (an allocation through the
// dispatcher takes about 0.8 us of host time, as a view through it would).
Tensor part_of(const Tensor& buffer, int64_t offset, at::IntArrayRef sizes, at::IntArrayRef strides) {
  auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
  t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides, buffer.storage_offset() + offset);
  return t;
}

gfa_kv4_rows_args rows_args(const Tensor& codes, const Tensor& scales, bool bf16, const Tensor& k, const Tensor& v,
                            const Tensor& slots) {
  gfa_kv4_rows_args a{};
  a.cache = cache_of(codes, scales, bf16);
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_strides = strides_of(k);
  a.v_strides = strides_of(v);
  a.batch = (int32_t)k.size(0);
  a.seq_len = (int32_t)k.size(2);
  a.slots = static_cast<const int64_t*>(slots.data_ptr());
  a.stream = stream_of(codes);
  return a;
}

void kv4_write(const Tensor& codes, const Tensor& scales, bool bf16, const Tensor& k, const Tensor& v, const Tensor& slots) {
  check_cache(codes, scales);
  check_token_rows("k", k, codes, bf16, true);
  check_token_rows("v", v, codes, bf16, true);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "shape mismatch: k ", k.sizes(), ", v ", v.sizes());
  check_array("slots", slots, at::kLong, 1, codes.device());
  TORCH_CHECK_VALUE(slots.size(0) == k.size(0) * k.size(2), "slots holds ", slots.size(0), " entries for ",
                    k.size(0) * k.size(2), " tokens");
  if (slots.size(0) == 0) return;
  const c10::DeviceGuard guard(codes.device());
  const Tensor kp = prep(k), vp = prep(v), sp = dense(slots);
  const auto a = rows_args(codes, scales, bf16, kp, vp, sp);
  check(api.kv4_write(&a));
}

// `apart`: outputs with memory of their own, as a registered op's have to be.
std::tuple<Tensor, Tensor> kv4_read(const Tensor& codes, const Tensor& scales, bool bf16, const Tensor& slots, bool apart) {
  check_cache(codes, scales);
  check_array("slots", slots, at::kLong, 1, codes.device());
  TORCH_CHECK_VALUE(slots.size(0) <= INT32_MAX, "slots holds more than 2^31 - 1 entries");
  const c10::DeviceGuard guard(codes.device());
  const auto options = codes.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
  const int64_t T = slots.size(0), H = codes.size(1), D = 2 * codes.size(4);
  // (1, H, T, D) views of token-major rows
  const Tensor kv = at::empty({(apart ? 1 : 2) * T * H * D}, options), kv2 = apart ? at::empty({T * H * D}, options) : kv;
  const Tensor k = part_of(kv, 0, {1, H, T, D}, {T * H * D, D, H * D, 1});
  const Tensor v = part_of(kv2, apart ? 0 : T * H * D, {1, H, T, D}, {T * H * D, D, H * D, 1});
  if (T > 0) {
    const Tensor sp = dense(slots);
    const auto a = rows_args(codes, scales, bf16, k, v, sp);
    check(api.kv4_read(&a));
  }
  return {k, v};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> kv4_plan(const Tensor& lens, const Tensor& fresh, const Tensor& table,
                                                            const Tensor& free_ids, const Tensor& used, int64_t block_size,
                                                            int64_t tokens, bool apart) {
  const auto device = lens.device();
  check_array("lens", lens, at::kInt, 1, device);
  const int64_t B = lens.size(0);
  check_array("new", fresh, at::kInt, 1, device);
  TORCH_CHECK_VALUE(fresh.size(0) == B, "new holds ", fresh.size(0), " entries for ", B, " requests");
  const int64_t stride = check_table(table, B, device);
  check_array("free", free_ids, at::kInt, 1, device);
  check_array("used", used, at::kInt, 1, device);
  TORCH_CHECK_VALUE(used.size(0) == 1 && free_ids.size(0) <= INT32_MAX, "used must hold one entry");
  TORCH_CHECK_VALUE(block_size_ok(block_size), "block_size=", block_size, " must be a power of two, 32 to 1024");
  TORCH_CHECK_VALUE(tokens >= 0 && tokens <= INT32_MAX, "tokens=", tokens, " must be in [0, 2^31)");
  const c10::DeviceGuard guard(device);
  const Tensor l = dense(lens), n = dense(fresh), f = dense(free_ids), u = dense(used);
  const Tensor slots = at::empty({tokens}, lens.options().dtype(at::kLong));
  const Tensor rest = apart ? Tensor() : at::empty({tokens + 2 * B + 2}, lens.options());
  const auto out = [&](int64_t offset, int64_t n) { return apart ? at::empty({n}, lens.options()) : part_of(rest, offset, {n}, {1}); };
  const Tensor positions = out(0, tokens), cu = out(tokens, B + 1), lens_out = out(tokens + B + 1, B);
  const Tensor used_out = out(tokens + 2 * B + 1, 1);
  const auto ints = [](const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
  gfa_kv4_plan_args a{};
  a.lens = ints(l);
  a.fresh = ints(n);
  a.table = ints(table);
  a.table_stride = stride;
  a.free_ids = ints(f);
  a.used = ints(u);
  a.requests = (int32_t)B;
  a.table_width = (int32_t)table.size(1);
  a.free_count = (int32_t)f.size(0);
  a.block_size = (int32_t)block_size;
  a.tokens = (int32_t)tokens;
  a.slots = static_cast<int64_t*>(slots.data_ptr());
  a.positions = ints(positions);
  a.cu = ints(cu);
  a.lens_out = ints(lens_out);
  a.used_out = ints(used_out);
  a.stream = stream_of(lens);
  check(api.kv4_plan(&a));
  return {slots, positions, cu, lens_out, used_out};
}

Tensor kv4_attention(const Tensor& q, const Tensor& codes, const Tensor& scales, bool bf16, const Tensor& table,
                     const Tensor& lens, const std::optional<Tensor>& cu, int64_t max_new, bool causal, int64_t window,
                     double scale, double softcap, const std::optional<Tensor>& shared_skip, const std::optional<Tensor>& shared_cu,
                     const std::optional<Tensor>& shared_lens, bool apart) {
  check_cache(codes, scales);
  check_token_rows("q", q, codes, bf16, false);
  const int64_t B = q.size(0), Hq = q.size(1), N = q.size(2), Hkv = codes.size(1);
  TORCH_CHECK_VALUE(Hq > 0 && Hq % Hkv == 0, "N_Q_HEADS=", Hq, " must be a multiple of N_KV_HEADS=", Hkv);
  TORCH_CHECK_VALUE(B > 0 && N > 0, "empty sequence or batch");
  const auto device = codes.device();
  check_array("lens", lens, at::kInt, 1, device);
  const int64_t R = lens.size(0);
  const int64_t stride = check_table(table, R, device);
  if (cu) {
    check_array("cu", *cu, at::kInt, 1, device);
    TORCH_CHECK_VALUE(cu->size(0) == R + 1, "cu holds ", cu->size(0), " entries for ", R, " requests");
  } else {
    TORCH_CHECK_VALUE(B * N % R == 0, B * N, " tokens do not divide among ", R, " requests (pass cu)");
  }
  TORCH_CHECK_VALUE(window >= 0, "slide_size must be >= 0");
  TORCH_CHECK_VALUE(max_new >= 0, "max_new must be at least 1");
  const bool shared = shared_skip && shared_cu && shared_lens;
  TORCH_CHECK_VALUE(shared || (!shared_skip && !shared_cu && !shared_lens), "shared must hold all of skip, cu and lens");
  if (shared) {
    check_array("shared.skip", *shared_skip, at::kInt, 1, device);
    check_array("shared.cu", *shared_cu, at::kInt, 1, device);
    check_array("shared.lens", *shared_lens, at::kInt, 1, device);
    TORCH_CHECK_VALUE(cu && shared_skip->size(0) == R && shared_cu->size(0) == R + 1 && shared_lens->size(0) == R,
                      "shared is for ", shared_skip->size(0), " requests with cu, the call has ", R, cu ? "" : " without");
  }
  const c10::DeviceGuard guard(device);
  const Tensor ss = shared ? dense(*shared_skip) : Tensor(), sc = shared ? dense(*shared_cu) : Tensor(), sl = shared ? dense(*shared_lens) : Tensor();
  const Tensor qp = prep(q), lp = dense(lens), cp = cu ? dense(*cu) : Tensor();
  const Tensor o = out_like(qp);
  gfa_kv4_attn_args a{};
  a.cache = cache_of(codes, scales, bf16);
  a.q = qp.data_ptr();
  a.o = o.data_ptr();
  a.q_strides = strides_of(qp);
  a.o_strides = strides_of(o);
  a.batch = (int32_t)B;
  a.heads_q = (int32_t)Hq;
  a.seq_len = (int32_t)N;
  a.requests = (int32_t)R;
  a.table = static_cast<const int32_t*>(table.data_ptr());
  a.table_stride = stride;
  a.lens = static_cast<const int32_t*>(lp.data_ptr());
  a.cu = cu ? static_cast<const int32_t*>(cp.data_ptr()) : nullptr;
  a.table_width = (int32_t)table.size(1);
  a.causal = causal;
  a.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
  a.max_new = (int32_t)std::min<int64_t>(max_new, INT32_MAX);
  a.scale = (float)scale;
  a.softcap = (float)softcap;
  a.stream = stream_of(q);
  if (shared) {
    a.shared_skip = static_cast<const int32_t*>(ss.data_ptr());
    a.shared_cu = static_cast<const int32_t*>(sc.data_ptr());
    a.shared_lens = static_cast<const int32_t*>(sl.data_ptr());
    a.shared_apart = apart;
  }
  Tensor ws;
  const size_t need = api.kv4_attn_workspace_bytes(&a);
  if (need > 0) {
    ws = at::empty({(int64_t)need}, codes.options());
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
  }
  check(api.kv4_attn(&a));
  return o;
}

// ---- Requests with something in common (kv4.py) ----

int32_t* ints_of(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

std::vector<gfa_kv4_cache> caches_of(const std::vector<Tensor>& codes, const std::vector<Tensor>& scales) {
  TORCH_CHECK_VALUE(!codes.empty() && codes.size() == scales.size(), "at least one cache is needed");
  std::vector<gfa_kv4_cache> out(codes.size());
  for (size_t i = 0; i < codes.size(); ++i) {
    check_cache(codes[i], scales[i]);
    TORCH_CHECK_VALUE(codes[i].device() == codes[0].device() && codes[i].size(0) == codes[0].size(0) && codes[i].size(3) == codes[0].size(3),
                      "caches of ", codes[0].sizes(), " on ", codes[0].device(), " and ", codes[i].sizes(), " on ", codes[i].device(),
                      " do not belong to one table");
    out[i] = cache_of(codes[i], scales[i], true);  // bytes, whatever the type
  }
  return out;
}

// The free list, which is changed in place.
void check_free(const Tensor& free_ids, const c10::Device& device) {
  check_array("free", free_ids, at::kInt, 1, device);
  TORCH_CHECK_VALUE(free_ids.is_contiguous() && !free_ids.is_neg() && free_ids.size(0) <= INT32_MAX, "free must be contiguous");
}

void check_rows_of_pages(const Tensor& table, int64_t rows) {
  TORCH_CHECK_VALUE(rows > 0 && rows <= 4096 && table.size(0) <= 4096, table.size(0), " requests and ", rows, " rows (1 to 4096)");
}

std::tuple<Tensor, Tensor, Tensor> kv4_fork(const std::vector<Tensor>& codes, const std::vector<Tensor>& scales, const Tensor& table,
                                            const Tensor& lens, const Tensor& free_ids, const Tensor& used,
                                            const std::optional<Tensor>& parents, const std::optional<Tensor>& keep, bool apart) {
  const auto caches = caches_of(codes, scales);
  const auto device = codes[0].device();
  check_array("lens", lens, at::kInt, 1, device);
  const int64_t B = lens.size(0), stride = check_table(table, B, device), M = table.size(1);
  check_free(free_ids, device);
  check_array("used", used, at::kInt, 1, device);
  TORCH_CHECK_VALUE(used.size(0) == 1, "used must hold one entry");
  if (parents) check_array("parents", *parents, at::kInt, 1, device);
  const int64_t R = parents ? parents->size(0) : B;
  if (keep) {
    check_array("keep", *keep, at::kInt, 1, device);
    TORCH_CHECK_VALUE(keep->size(0) == R, "keep holds ", keep->size(0), " entries for ", R, " rows");
  }
  check_rows_of_pages(table, R);
  const c10::DeviceGuard guard(device);
  const Tensor l = dense(lens), u = dense(used), pp = parents ? dense(*parents) : Tensor(), kp = keep ? dense(*keep) : Tensor();
  const size_t need = api.kv4_pages_workspace_bytes((int32_t)R);
  const int64_t ws_ints = (int64_t)(need / 4);
  const Tensor rest = at::empty({apart ? ws_ints : R * M + R + 1 + ws_ints}, lens.options());
  const Tensor table_out = apart ? at::empty({R, M}, lens.options()) : part_of(rest, 0, {R, M}, {M, 1});
  const Tensor lens_out = apart ? at::empty({R}, lens.options()) : part_of(rest, R * M, {R}, {1});
  const Tensor used_out = apart ? at::empty({1}, lens.options()) : part_of(rest, R * M + R, {1}, {1});
  gfa_kv4_pages_args a{};
  a.caches = caches.data();
  a.layers = (int32_t)caches.size();
  a.table = ints_of(table);
  a.table_stride = stride;
  a.lens = ints_of(l);
  a.requests = (int32_t)B;
  a.table_width = (int32_t)M;
  a.parents = parents ? ints_of(pp) : nullptr;
  a.keep = keep ? ints_of(kp) : nullptr;
  a.rows = (int32_t)R;
  a.free_count = (int32_t)free_ids.size(0);
  a.free_ids = ints_of(free_ids);
  a.used = ints_of(u);
  a.table_out = ints_of(table_out);
  a.lens_out = ints_of(lens_out);
  a.used_out = ints_of(used_out);
  a.workspace = ints_of(rest) + (apart ? 0 : R * M + R + 1);
  a.workspace_bytes = need;
  a.stream = stream_of(codes[0]);
  check(api.kv4_fork(&a));
  return {table_out, lens_out, used_out};
}

std::tuple<Tensor, Tensor> kv4_compact(const std::vector<Tensor>& codes, const std::vector<Tensor>& scales, const Tensor& table,
                                       const Tensor& lens, const Tensor& free_ids, bool apart) {
  const auto caches = caches_of(codes, scales);
  const auto device = codes[0].device();
  check_array("lens", lens, at::kInt, 1, device);
  const int64_t B = lens.size(0), stride = check_table(table, B, device), M = table.size(1), blocks = codes[0].size(0);
  check_free(free_ids, device);
  TORCH_CHECK_VALUE(free_ids.size(0) == blocks, "free holds ", free_ids.size(0), " entries, a compacted pool's all of its ", blocks, " blocks");
  check_rows_of_pages(table, B);
  const c10::DeviceGuard guard(device);
  const Tensor l = dense(lens);
  const size_t need = api.kv4_pages_workspace_bytes((int32_t)blocks);
  const int64_t ws_ints = (int64_t)(need / 4);
  // the workspace is the larger part, and nobody keeps it
  const Tensor ws = at::empty({ws_ints}, lens.options()), out = at::empty({apart ? B * M : B * M + 1}, lens.options());
  const Tensor table_out = part_of(out, 0, {B, M}, {M, 1});
  const Tensor used_out = apart ? at::empty({1}, lens.options()) : part_of(out, B * M, {1}, {1});
  gfa_kv4_pages_args a{};
  a.caches = caches.data();
  a.layers = (int32_t)caches.size();
  a.table = ints_of(table);
  a.table_stride = stride;
  a.lens = ints_of(l);
  a.requests = (int32_t)B;
  a.table_width = (int32_t)M;
  a.free_count = (int32_t)blocks;
  a.free_ids = ints_of(free_ids);
  a.table_out = ints_of(table_out);
  a.used_out = ints_of(used_out);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = need;
  a.stream = stream_of(codes[0]);
  check(api.kv4_compact(&a));
  return {table_out, used_out};
}

void kv4_copy(const std::vector<Tensor>& codes, const std::vector<Tensor>& scales, const Tensor& src, const Tensor& dst) {
  const auto caches = caches_of(codes, scales);
  const auto device = codes[0].device();
  check_array("src", src, at::kInt, 1, device);
  check_array("dst", dst, at::kInt, 1, device);
  TORCH_CHECK_VALUE(src.size(0) == dst.size(0) && src.size(0) <= INT32_MAX, "src holds ", src.size(0), " entries, dst ", dst.size(0));
  const c10::DeviceGuard guard(device);
  const Tensor s = dense(src), d = dense(dst);
  check(api.kv4_copy(caches.data(), (int32_t)caches.size(), ints_of(s), ints_of(d), (int32_t)s.size(0), stream_of(codes[0])));
}

std::tuple<Tensor, Tensor, Tensor> kv4_share(const Tensor& table, const Tensor& lens, const Tensor& cu, int64_t block_size, int64_t least,
                                             bool apart) {
  const auto device = lens.device();
  check_array("lens", lens, at::kInt, 1, device);
  const int64_t R = lens.size(0), stride = check_table(table, R, device);
  check_array("cu", cu, at::kInt, 1, device);
  TORCH_CHECK_VALUE(cu.size(0) == R + 1, "cu holds ", cu.size(0), " entries for ", R, " requests");
  TORCH_CHECK_VALUE(block_size_ok(block_size), "block_size=", block_size, " must be a power of two, 32 to 1024");
  TORCH_CHECK_VALUE(least >= 1, "least=", least, " must be at least 1");
  TORCH_CHECK_VALUE(R <= 4096, R, " requests (most 4096)");
  const c10::DeviceGuard guard(device);
  const Tensor l = dense(lens), c = dense(cu);
  const Tensor all = apart ? Tensor() : at::empty({3 * R + 1}, lens.options());
  const auto out = [&](int64_t offset, int64_t n) { return apart ? at::empty({n}, lens.options()) : part_of(all, offset, {n}, {1}); };
  const Tensor skip = out(0, R), cu_out = out(R, R + 1), lens_out = out(2 * R + 1, R);
  gfa_kv4_share_args a{};
  a.table = ints_of(table);
  a.table_stride = stride;
  a.lens = ints_of(l);
  a.cu = ints_of(c);
  a.requests = (int32_t)R;
  a.table_width = (int32_t)table.size(1);
  a.block_size = (int32_t)block_size;
  a.least = (int32_t)std::min<int64_t>(least, INT32_MAX);
  a.skip = ints_of(skip);
  a.cu_out = ints_of(cu_out);
  a.lens_out = ints_of(lens_out);
  a.stream = stream_of(lens);
  check(api.kv4_share(&a));
  return {skip, cu_out, lens_out};
}

// Rows of probabilities, read in place where their entries are side by side.
Tensor probability_rows(const Tensor& t) {
  if (t.is_neg()) return t.resolve_neg().contiguous();
  return (t.size(1) == 1 || t.stride(1) == 1) && t.stride(0) >= 0 ? t : t.contiguous();
}

std::tuple<Tensor, Tensor, Tensor> kv4_verify(const Tensor& target, const std::optional<Tensor>& draft, const Tensor& tokens,
                                              const Tensor& accept, const Tensor& sample, const Tensor& lens, const std::optional<Tensor>& cu,
                                              bool apart) {
  const auto type = target.scalar_type();
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kHalf || type == at::kBFloat16, "target is ", type, " (fp32, fp16 or bf16)");
  TORCH_CHECK_VALUE(target.dim() == 2, "target must be 2-D (tokens, vocabulary), got shape ", target.sizes());
  TORCH_CHECK_VALUE(target.is_cuda(), "target must be on a GPU (the engine has no CPU path), is on ", target.device());
  const auto device = target.device();
  const int64_t T = target.size(0), V = target.size(1);
  TORCH_CHECK_VALUE(T > 0 && V > 0 && T <= INT32_MAX && V <= 1 << 30, "target of shape ", target.sizes());
  if (draft) {
    TORCH_CHECK_TYPE(draft->scalar_type() == type, "draft is ", draft->scalar_type(), ", target ", type);
    TORCH_CHECK_VALUE(draft->sizes() == target.sizes(), "shape mismatch: target ", target.sizes(), ", draft ", draft->sizes());
    TORCH_CHECK_VALUE(on_gpu(*draft, device), "draft must be on the call's GPU (", device, "), is on ", draft->device());
  }
  check_array("tokens", tokens, at::kLong, 1, device);
  check_array("accept", accept, at::kFloat, 1, device);
  TORCH_CHECK_VALUE(tokens.size(0) == T && accept.size(0) == T, "tokens holds ", tokens.size(0), " entries and accept ", accept.size(0),
                    " for ", T, " rows of target");
  check_array("lens", lens, at::kInt, 1, device);
  check_array("sample", sample, at::kFloat, 1, device);
  const int64_t R = lens.size(0);
  TORCH_CHECK_VALUE(R > 0 && R <= 65535 && sample.size(0) == R, "sample holds ", sample.size(0), " entries for ", R, " requests (1 to 65535)");
  if (cu) {
    check_array("cu", *cu, at::kInt, 1, device);
    TORCH_CHECK_VALUE(cu->size(0) == R + 1, "cu holds ", cu->size(0), " entries for ", R, " requests");
  } else {
    TORCH_CHECK_VALUE(T % R == 0, T, " tokens do not divide among ", R, " requests (pass cu)");
  }
  const c10::DeviceGuard guard(device);
  const Tensor p = probability_rows(target), q = draft ? probability_rows(*draft) : Tensor();
  const Tensor x = dense(tokens), u = dense(accept), r = dense(sample), l = dense(lens), c = cu ? dense(*cu) : Tensor();
  // the workspace in front: its numbers are of 64 bits
  const size_t need = api.kv4_verify_workspace_bytes((int32_t)R, (int32_t)V);
  const int64_t ws_ints = (int64_t)(need / 4);
  const Tensor rest = at::empty({ws_ints + (apart ? 0 : 2 * R)}, lens.options());
  const auto out = [&](int64_t offset) { return apart ? at::empty({R}, lens.options()) : part_of(rest, offset, {R}, {1}); };
  const Tensor follows = at::empty({T}, tokens.options()), accepted = out(ws_ints), lens_out = out(ws_ints + R);
  gfa_kv4_verify_args a{};
  a.target = p.data_ptr();
  a.draft = draft ? q.data_ptr() : nullptr;
  a.target_stride = p.stride(0);
  a.draft_stride = draft ? q.stride(0) : 0;
  a.type = type == at::kFloat ? 2 : type == at::kBFloat16 ? 1 : 0;
  a.token_count = (int32_t)T;
  a.vocab = (int32_t)V;
  a.requests = (int32_t)R;
  a.tokens = static_cast<const int64_t*>(x.data_ptr());
  a.accept = static_cast<const float*>(u.data_ptr());
  a.sample = static_cast<const float*>(r.data_ptr());
  a.lens = ints_of(l);
  a.cu = cu ? ints_of(c) : nullptr;
  a.follows = static_cast<int64_t*>(follows.data_ptr());
  a.accepted = ints_of(accepted);
  a.lens_out = ints_of(lens_out);
  a.workspace = rest.data_ptr();
  a.workspace_bytes = need;
  a.stream = stream_of(target);
  check(api.kv4_verify(&a));
  return {follows, accepted, lens_out};
}

template <typename F>
F pointer(uintptr_t p) {
  return reinterpret_cast<F>(p);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("version") = GFA_VERSION;
  m.def("bind", [](uintptr_t fwd, uintptr_t bwd, uintptr_t workspace_bytes, uintptr_t positions, uintptr_t last_error,
                   py::object error_type) {
    api.fwd = pointer<decltype(api.fwd)>(fwd);
    api.bwd = pointer<decltype(api.bwd)>(bwd);
    api.workspace_bytes = pointer<decltype(api.workspace_bytes)>(workspace_bytes);
    api.positions = pointer<decltype(api.positions)>(positions);
    api.last_error = pointer<decltype(api.last_error)>(last_error);
    api.error_type = error_type.release().ptr();
  });
  m.def("bind_kv4", [](uintptr_t write, uintptr_t read, uintptr_t plan, uintptr_t attn, uintptr_t workspace_bytes) {
    api.kv4_write = pointer<decltype(api.kv4_write)>(write);
    api.kv4_read = pointer<decltype(api.kv4_read)>(read);
    api.kv4_plan = pointer<decltype(api.kv4_plan)>(plan);
    api.kv4_attn = pointer<decltype(api.kv4_attn)>(attn);
    api.kv4_attn_workspace_bytes = pointer<decltype(api.kv4_attn_workspace_bytes)>(workspace_bytes);
  });
  m.def("bind_kv4_pages", [](uintptr_t fork, uintptr_t compact, uintptr_t workspace_bytes, uintptr_t copy, uintptr_t share, uintptr_t verify,
                             uintptr_t verify_workspace_bytes) {
    api.kv4_fork = pointer<decltype(api.kv4_fork)>(fork);
    api.kv4_compact = pointer<decltype(api.kv4_compact)>(compact);
    api.kv4_pages_workspace_bytes = pointer<decltype(api.kv4_pages_workspace_bytes)>(workspace_bytes);
    api.kv4_copy = pointer<decltype(api.kv4_copy)>(copy);
    api.kv4_share = pointer<decltype(api.kv4_share)>(share);
    api.kv4_verify = pointer<decltype(api.kv4_verify)>(verify);
    api.kv4_verify_workspace_bytes = pointer<decltype(api.kv4_verify_workspace_bytes)>(verify_workspace_bytes);
  });
  m.def("kv4_fork", torch::wrap_pybind_function_no_gil(kv4_fork));
  m.def("kv4_compact", torch::wrap_pybind_function_no_gil(kv4_compact));
  m.def("kv4_copy", torch::wrap_pybind_function_no_gil(kv4_copy));
  m.def("kv4_share", torch::wrap_pybind_function_no_gil(kv4_share));
  m.def("kv4_verify", torch::wrap_pybind_function_no_gil(kv4_verify));
  m.def("kv4_cache", torch::wrap_pybind_function_no_gil(check_cache));
  m.def("kv4_write", torch::wrap_pybind_function_no_gil(kv4_write));
  m.def("kv4_read", torch::wrap_pybind_function_no_gil(kv4_read));
  m.def("kv4_plan", torch::wrap_pybind_function_no_gil(kv4_plan));
  m.def("kv4_attention", torch::wrap_pybind_function_no_gil(kv4_attention));
  // Bodies run without the interpreter lock: an allocation or a launch that waits for the driver does
  // not hold up other Python threads (a data loader's, another stream's).
  const auto or_undefined = [](const std::optional<Tensor>& t) { return t ? *t : Tensor(); };
  // O alone, without autograd.
  m.def("infer", torch::wrap_pybind_function_no_gil(
                     [or_undefined](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, int64_t window,
                                    double scale, double softcap, double dropout_p, int64_t seed, int64_t block_kv,
                                    const std::optional<Tensor>& lo, const std::optional<Tensor>& hi) {
                       const Options x{causal, window, scale, softcap, dropout_p, seed, block_kv,
                                       or_undefined(lo), or_undefined(hi)};
                       return forward_call(prep(q), prep(k), prep(v), x, false).first;
                     }));
  // O with autograd.
  m.def("train", torch::wrap_pybind_function_no_gil(
                     [or_undefined](const Tensor& q, const Tensor& k, const Tensor& v, bool causal, int64_t window,
                                    double scale, double softcap, double dropout_p, int64_t seed,
                                    const std::optional<Tensor>& lo, const std::optional<Tensor>& hi, bool as_op) {
                       const Options x{causal, window, scale, softcap, dropout_p, seed, 0,
                                       or_undefined(lo), or_undefined(hi), as_op};
                       return Attention::apply(q, k, v, x);
                     }));
  // (lo, hi) tables, int32 (batch, seq_len), of unit-stride position ids (rows of stride 0 included).
  m.def("positions", torch::wrap_pybind_function_no_gil([](const Tensor& pos) {
          const c10::DeviceGuard guard(pos.device());
          const Tensor t = at::empty({2, pos.size(0), pos.size(1)}, pos.options().dtype(at::kInt));
          const Tensor lo = t.select(0, 0), hi = t.select(0, 1);
          check(api.positions(pos.data_ptr(), 8 * (int32_t)pos.element_size(), pos.stride(0), (int32_t)pos.size(0),
                              (int32_t)pos.size(1), static_cast<int32_t*>(lo.data_ptr()),
                              static_cast<int32_t*>(hi.data_ptr()), stream_of(pos)));
          return std::make_tuple(lo, hi);
        }));
}
