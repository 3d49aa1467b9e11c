// torch binding of the differential-attention stack's operators: argument checks, buffers and the autograd nodes, in C++.
//
// A training step of these operators over one batch of sessions is 30 - 200 us of GPU time; the same nodes written in Python cost 130 - 240 us
// of host time per step (argument checks 25, ctypes conversions 10, a Python node's backward and the interpreter lock's hand-over to the
// engine's thread 40 - 60 us per node), so the host set the pace.  The kernels stay behind the C entries of librectools_hip.so
// (include/rectools_hip.h); this file holds no device code.  Errors are the Python layer's: ValueError (arguments), NotImplementedError
// (sizes the kernels do not hold), HipLibraryError (not a float32 HIP tensor; a failed launch).
#include <dlfcn.h>

#include <cmath>

#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "../../include/rectools_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> OptTensor;

namespace {

// ---- the library ------------------------------------------------------------------------------------------------------------------------
struct Lib {
  decltype(&rt_rotary) rotary = nullptr;
  decltype(&rt_diff_lambda_fwd) lambda_fwd = nullptr;
  decltype(&rt_diff_lambda_bwd) lambda_bwd = nullptr;
  decltype(&rt_diffattn_saved_bytes) attn_saved = nullptr;
  decltype(&rt_diffattn_fwd_workspace_bytes) attn_fwd_ws = nullptr;
  decltype(&rt_diffattn_fwd) attn_fwd = nullptr;
  decltype(&rt_diffattn_bwd_workspace_bytes) attn_bwd_ws = nullptr;
  decltype(&rt_diffattn_bwd) attn_bwd = nullptr;
  decltype(&rt_norm_gate_fwd) norm_fwd = nullptr;
  decltype(&rt_norm_gate_bwd_workspace_bytes) norm_bwd_ws = nullptr;
  decltype(&rt_norm_gate_bwd) norm_bwd = nullptr;
  decltype(&rt_last_error) last_error = nullptr;
} L;
PyObject* g_library_error = nullptr;      // rectools_amd._lib.HipLibraryError

// the library that the Python layer has loaded (its dlopen handle), and its exception class
void bind(uintptr_t handle, py::object library_error) {
  void* h = reinterpret_cast<void*>(handle);
#define RT_BIND(field, name)                                                        \
  L.field = reinterpret_cast<decltype(L.field)>(dlsym(h, #name));                   \
  if (L.field == nullptr) throw std::runtime_error("librectools_hip.so misses " #name)
  RT_BIND(rotary, rt_rotary);
  RT_BIND(lambda_fwd, rt_diff_lambda_fwd);
  RT_BIND(lambda_bwd, rt_diff_lambda_bwd);
  RT_BIND(attn_saved, rt_diffattn_saved_bytes);
  RT_BIND(attn_fwd_ws, rt_diffattn_fwd_workspace_bytes);
  RT_BIND(attn_fwd, rt_diffattn_fwd);
  RT_BIND(attn_bwd_ws, rt_diffattn_bwd_workspace_bytes);
  RT_BIND(attn_bwd, rt_diffattn_bwd);
  RT_BIND(norm_fwd, rt_norm_gate_fwd);
  RT_BIND(norm_bwd_ws, rt_norm_gate_bwd_workspace_bytes);
  RT_BIND(norm_bwd, rt_norm_gate_bwd);
  RT_BIND(last_error, rt_last_error);
#undef RT_BIND
  g_library_error = library_error.release().ptr();
}

// ---- errors: raised from the calling thread (forward); an autograd thread raises RuntimeError ----------------------------------------------------
[[noreturn]] void raise(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw py::error_already_set();
}
[[noreturn]] void bad(const char* what, const std::string& text) { raise(PyExc_ValueError, std::string(what) + ": " + text); }

void status(int rc, const char* what, bool forward) {
  if (rc == RT_OK) return;
  const std::string text = std::string(what) + (rc == RT_ERR_INVALID_ARG ? ": invalid argument" : rc == RT_ERR_UNSUPPORTED ? ": unsupported configuration"
                           : rc == RT_ERR_WORKSPACE ? ": workspace missing or too small" : std::string(": HIP launch failed ") + L.last_error());
  if (!forward) TORCH_CHECK(false, text);
  raise(rc == RT_ERR_INVALID_ARG ? PyExc_ValueError : rc == RT_ERR_UNSUPPORTED ? PyExc_NotImplementedError : g_library_error, text);
}

std::string shape(const Tensor& t) {
  std::ostringstream s;
  s << t.sizes();
  return s.str();
}
void check_f32(const Tensor& t, const char* what) {
  if (!t.is_cuda() || t.scalar_type() != at::kFloat) {
    std::ostringstream s;
    s << what << ": expected a float32 HIP tensor (no CPU fallback), got " << t.scalar_type() << " on " << t.device();
    raise(g_library_error, s.str());
  }
}
void check_device(const Tensor& t, const Tensor& first, const char* what) {
  if (t.device() != first.device()) {
    std::ostringstream s;
    s << "tensors on " << first.device() << " and " << t.device();
    bad(what, s.str());
  }
}
// A float32 matrix whose rows the kernels read in place: unit column stride, rows that do not overlap; else a copy (one that autograd sees)
Tensor rows(const Tensor& t, int64_t cols, const char* what) {
  check_f32(t, what);
  if (t.dim() != 2 || (cols >= 0 && t.size(1) != cols)) bad(what, "expected [rows, " + (cols < 0 ? std::string("columns") : std::to_string(cols)) + "], got " + shape(t));
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) return t.contiguous();
  return t;
}
Tensor dense_rows(const Tensor& t) {      // the same for a gradient
  return ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) ? t.contiguous() : t;
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
Tensor ints(const OptTensor& t, int64_t n, const Tensor& first, const char* what) {
  if (!t.has_value()) return Tensor();
  if (t->scalar_type() != at::kLong || !t->is_cuda() || t->dim() != 1 || t->size(0) != n) {
    std::ostringstream s;
    s << "expected " << n << " int64 values on the HIP device, got " << t->scalar_type() << " " << t->sizes() << " on " << t->device();
    bad(what, s.str());
  }
  check_device(*t, first, what);
  return t->contiguous();
}
Tensor vec(const OptTensor& t, at::IntArrayRef want, const Tensor& first, const char* what) {
  if (!t.has_value()) return Tensor();
  check_f32(*t, what);
  if (t->sizes() != want) {
    std::ostringstream s;
    s << "expected " << want << ", got " << t->sizes();
    bad(what, s.str());
  }
  check_device(*t, first, what);
  return t->contiguous();
}
constexpr int64_t MOST = 0x7FFFFFFF;      // the C entries count heads and columns in 32 bits
void check_eps(double eps, const char* what) {      // (as the kernels see it: without it a row of zeros has no norm)
  if (!((float)eps > 0.f)) bad(what, "eps is positive, got " + std::to_string(eps));
}
float* f(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
int64_t* i64(const Tensor& t) { return t.defined() ? static_cast<int64_t*>(t.data_ptr()) : nullptr; }
rt_stream_t stream_of(const Tensor& t) { return reinterpret_cast<rt_stream_t>(c10::hip::getCurrentHIPStream(t.get_device()).stream()); }
Tensor scratch(size_t n, const Tensor& like) { return n > 0 ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor(); }
// an absent tensor goes through an autograd node's arguments as an empty optional
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor got(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool on_tape(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Forward-mode derivatives are refused, as second ones are: a tensor with a tangent need not require a gradient, and without a node its tangent would be
// dropped in silence (a zero derivative).
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) raise(PyExc_NotImplementedError, std::string(what) + " has no forward-mode derivative");
}
void once(const char* what) {      // grad mode is on in a backward pass only under create_graph
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative (create_graph=True)");
}

// Leaves whose gradient node was made on the default stream (by a graph that lives outside a capture, or by this call on that stream): the engine
// hands their gradients over on that stream, which no capture can follow; the process would end there.  Noted in the forward pass, refused when
// the backward pass runs under a capture.  `held`: the same of the caller's own tensors, where the node is given a dense copy of one (rows(), contiguous()).
bool default_stream_leaves(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) {
    if (!t->defined() || !t->is_leaf() || !t->requires_grad()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto s = node->stream();
    if (s.has_value() && s->id() == 0) return true;
  }
  return false;
}
void capturable(AutogradContext* ctx, const char* what) {
  if (ctx->saved_data["leaves"].toBool() && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
    TORCH_CHECK(false, what, ": a backward pass cannot be captured while a graph made on the default stream holds the same leaf tensors; drop that graph first");
}

// ---- rotary -----------------------------------------------------------------------------------------------------------------------------
struct RotaryMeta { int64_t n_heads, n_kv_heads, hd; bool interleaved; double gain; };
void rotary_call(const Tensor& q, const Tensor& k, const Tensor& q2, const Tensor& k2, const Tensor& pos, const Tensor& freq, const RotaryMeta& m, bool backward) {
  c10::DeviceGuard guard(pos.device());
  const bool hq = q.defined(), hk = k.defined();
  status(L.rotary(f(q), hq ? ld(q) : 0, f(q2), hq ? q2.size(1) : 0, hq ? m.n_heads : 0, f(k), hk ? ld(k) : 0, f(k2), hk ? k2.size(1) : 0, hk ? m.n_kv_heads : 0, i64(pos),
                  static_cast<const double*>(freq.data_ptr()), pos.size(0), m.hd, 2 * freq.size(0), m.interleaved, (float)m.gain, backward, stream_of(pos)),
         "rt_rotary", !backward);
}
Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }

struct RotaryNode : torch::autograd::Function<RotaryNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_opt, const Tensor& pos, const Tensor& freq, int64_t n_heads, int64_t n_kv_heads,
                               int64_t hd, bool interleaved, double gain, bool held) {
    const Tensor k = got(k_opt);
    ctx->saved_data["leaves"] = held || default_stream_leaves({&q, &k});
    ctx->save_for_backward({pos, freq});
    ctx->saved_data["m"] = std::vector<int64_t>{n_heads, n_kv_heads, hd, interleaved};
    ctx->saved_data["g"] = gain;
    ctx->set_materialize_grads(false);
    variable_list out{like(q)};
    if (k.defined()) out.push_back(like(k));
    rotary_call(q, k, out[0], k.defined() ? out[1] : Tensor(), pos, freq, {n_heads, n_kv_heads, hd, interleaved, gain}, false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("rotary");
    capturable(ctx, "rotary");
    variable_list out(10);
    Tensor gq = g[0].defined() ? dense_rows(g[0]) : Tensor(), gk = g.size() > 1 && g[1].defined() ? dense_rows(g[1]) : Tensor();
    if (!gq.defined() && !gk.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    out[0] = like(gq);
    out[1] = like(gk);
    rotary_call(gq, gk, out[0], out[1], saved[0], saved[1], {m[0], m[1], m[2], m[3] != 0, ctx->saved_data["g"].toDouble()}, true);
    return out;
  }
};

std::vector<Tensor> rotary(const Tensor& q_in, const OptTensor& k_in, const Tensor& pos_in, const Tensor& freq_in, int64_t n_heads, int64_t n_kv_heads, bool interleaved,
                           double gain) {
  const Tensor k_any = got(k_in);
  no_tangent("rotary", {&q_in, &k_any, &freq_in});
  if (at::GradMode::is_enabled() && freq_in.requires_grad()) raise(PyExc_NotImplementedError, "rotary has no gradient of the frequencies: detach them");
  if (n_heads <= 0 || (k_in.has_value() && (n_kv_heads <= 0 || n_kv_heads > MOST))) bad("rotary", "head counts must be positive, got " + std::to_string(n_heads) + " and " + std::to_string(n_kv_heads));
  const Tensor q = rows(q_in, -1, "rotary");
  const int64_t M = q.size(0), cols = q.size(1);
  if (cols > MOST) raise(PyExc_NotImplementedError, "rotary: at most 2^31 - 1 columns, got " + std::to_string(cols));
  if (cols == 0 || cols % n_heads != 0) bad("rotary", std::to_string(cols) + " columns do not split into " + std::to_string(n_heads) + " heads");
  const int64_t hd = cols / n_heads;
  Tensor k;
  if (k_in.has_value()) {
    k = rows(*k_in, n_kv_heads * hd, "rotary");
    if (k.size(1) > MOST) raise(PyExc_NotImplementedError, "rotary: at most 2^31 - 1 columns, got " + std::to_string(k.size(1)));
    if (k.size(0) != M) bad("rotary", std::to_string(M) + " query rows and " + std::to_string(k.size(0)) + " key rows");
    check_device(k, q, "rotary");
  }
  const Tensor pos = ints(pos_in, M, q, "rotary positions");
  if (freq_in.scalar_type() != at::kDouble || freq_in.dim() != 1 || !freq_in.is_cuda() || freq_in.size(0) <= 0 || 2 * freq_in.size(0) > hd) {
    std::ostringstream s;
    s << "expected at most " << hd / 2 << " float64 frequencies on the HIP device (rotary_frequencies), got " << freq_in.scalar_type() << " " << freq_in.sizes() << " on "
      << freq_in.device();
    bad("rotary", s.str());
  }
  check_device(freq_in, q, "rotary");
  const Tensor freq = freq_in.contiguous();
  if (on_tape({&q, &k})) return RotaryNode::apply(q, opt(k), pos, freq, n_heads, n_kv_heads, hd, interleaved, gain, default_stream_leaves({&q_in, &k_any}));
  variable_list out{like(q)};
  if (k.defined()) out.push_back(like(k));
  rotary_call(q, k, out[0], k.defined() ? out[1] : Tensor(), pos, freq, {n_heads, n_kv_heads, hd, interleaved, gain}, false);
  return out;
}

// ---- lambda -----------------------------------------------------------------------------------------------------------------------------
Tensor lambda_call(const Tensor& q1, const Tensor& k1, const Tensor& q2, const Tensor& k2, double init) {
  c10::DeviceGuard guard(q1.device());
  const Tensor lam = at::empty({q1.size(0)}, q1.options());
  status(L.lambda_fwd(f(q1), f(k1), f(q2), f(k2), (float)init, q1.size(0), q1.size(1), f(lam), stream_of(q1)), "rt_diff_lambda_fwd", true);
  return lam;
}
struct LambdaNode : torch::autograd::Function<LambdaNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q1, const Tensor& k1, const Tensor& q2, const Tensor& k2, double init, bool held) {
    ctx->saved_data["leaves"] = held || default_stream_leaves({&q1, &k1, &q2, &k2});
    ctx->save_for_backward({q1, k1, q2, k2});
    return lambda_call(q1, k1, q2, k2, init);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("diff_lambda");
    capturable(ctx, "diff_lambda");
    const auto s = ctx->get_saved_variables();
    c10::DeviceGuard guard(s[0].device());
    variable_list out{like(s[0]), like(s[0]), like(s[0]), like(s[0]), Tensor(), Tensor()};
    const Tensor up = g[0].contiguous();
    status(L.lambda_bwd(f(up), f(s[0]), f(s[1]), f(s[2]), f(s[3]), s[0].size(0), s[0].size(1), f(out[0]), f(out[1]), f(out[2]), f(out[3]), stream_of(s[0])),
           "rt_diff_lambda_bwd", false);
    return out;
  }
};
Tensor diff_lambda(const Tensor& q1_in, const Tensor& k1_in, const Tensor& q2_in, const Tensor& k2_in, double init) {
  no_tangent("diff_lambda", {&q1_in, &k1_in, &q2_in, &k2_in});
  check_f32(q1_in, "diff_lambda");
  if (q1_in.dim() != 2 || q1_in.size(1) == 0) bad("diff_lambda", "expected [heads, columns], got " + shape(q1_in));
  if (q1_in.size(0) > MOST || q1_in.size(1) > MOST) raise(PyExc_NotImplementedError, "diff_lambda: at most 2^31 - 1 heads and columns, got " + shape(q1_in));
  const Tensor q1 = q1_in.contiguous(), k1 = vec(k1_in, q1_in.sizes(), q1_in, "diff_lambda"), q2 = vec(q2_in, q1_in.sizes(), q1_in, "diff_lambda"),
               k2 = vec(k2_in, q1_in.sizes(), q1_in, "diff_lambda");
  if (on_tape({&q1, &k1, &q2, &k2})) return LambdaNode::apply(q1, k1, q2, k2, init, default_stream_leaves({&q1_in, &k1_in, &q2_in, &k2_in}));
  return lambda_call(q1, k1, q2, k2, init);
}

// ---- differential attention -----------------------------------------------------------------------------------------------------------------
struct AttnMeta { int64_t B, H, Hkv, hd, Lq, Lk, causal; double scale, out_scale, eps; };
Tensor attention_call(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& cu_q, const Tensor& cu_k, const Tensor& ids, const Tensor& w,
                      const AttnMeta& m, Tensor* saved) {
  c10::DeviceGuard guard(q.device());
  const int64_t Nq = q.size(0), Nk = k.size(0);
  const Tensor y = at::empty({Nq, 2 * m.H * m.hd}, q.options());
  size_t kept = 0;
  if (saved != nullptr) {
    kept = L.attn_saved(m.H, m.Hkv, m.hd, Nq, Nk);
    *saved = scratch(kept, q);
  }
  const size_t n = L.attn_fwd_ws(m.B, m.H, m.Hkv, m.hd, m.Lq, m.Lk, Nq, Nk, saved != nullptr);
  const Tensor ws = scratch(n, q);
  status(L.attn_fwd(f(q), ld(q), f(k), ld(k), f(v), ld(v), f(lam), i64(cu_q), i64(cu_k), i64(ids), m.B, m.H, m.Hkv, m.hd, m.Lq, m.Lk, Nq, Nk, (float)m.scale, m.causal, f(w),
                    (float)m.out_scale, (float)m.eps, f(y), y.size(1), saved != nullptr ? saved->data_ptr() : nullptr, kept, ws.defined() ? ws.data_ptr() : nullptr, n,
                    stream_of(q)),
         "rt_diffattn_fwd", true);
  return y;
}
struct AttentionNode : torch::autograd::Function<AttentionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const OptTensor& w_opt, const OptTensor& cu_q_opt,
                        const OptTensor& cu_k_opt, const OptTensor& ids_opt, std::vector<int64_t> sizes, double scale, double out_scale, double eps, bool held) {
    const AttnMeta m{sizes[0], sizes[1], sizes[2], sizes[3], sizes[4], sizes[5], sizes[6], scale, out_scale, eps};
    const Tensor w = got(w_opt), cu_q = got(cu_q_opt), cu_k = got(cu_k_opt), ids = got(ids_opt);
    Tensor saved;
    const Tensor y = attention_call(q, k, v, lam, cu_q, cu_k, ids, w, m, &saved);
    ctx->saved_data["leaves"] = held || default_stream_leaves({&q, &k, &v, &lam, &w});
    ctx->save_for_backward({lam, w, cu_q, cu_k, ids, saved});      // (not q, k, v: their planes are in `saved`)
    sizes.push_back(q.size(0));
    sizes.push_back(k.size(0));
    ctx->saved_data["s"] = std::move(sizes);
    ctx->saved_data["f"] = std::vector<double>{scale, out_scale, eps};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("diff_attention");
    capturable(ctx, "diff_attention");
    const auto s = ctx->get_saved_variables();
    const Tensor &lam = s[0], &w = s[1], &saved = s[5];
    const auto z = ctx->saved_data["s"].toIntVector();
    const auto x = ctx->saved_data["f"].toDoubleVector();
    c10::DeviceGuard guard(lam.device());
    const Tensor dy = dense_rows(g[0]);
    const int64_t H = z[1], Hkv = z[2], hd = z[3], Nq = z[7], Nk = z[8];
    variable_list out(13);
    out[0] = at::empty({Nq, 2 * H * hd}, lam.options());
    out[1] = at::empty({Nk, 2 * Hkv * hd}, lam.options());
    out[2] = at::empty({Nk, 2 * Hkv * hd}, lam.options());
    out[3] = like(lam);
    out[4] = like(w);
    const size_t n = L.attn_bwd_ws(H, hd, Nq);
    const Tensor ws = scratch(n, lam);
    status(L.attn_bwd(saved.data_ptr(), saved.numel(), f(lam), i64(s[2]), i64(s[3]), i64(s[4]), z[0], H, Hkv, hd, z[4], z[5], Nq, Nk, (float)x[0], z[6], f(w), (float)x[1],
                      (float)x[2], f(dy), ld(dy), f(out[0]), out[0].size(1), f(out[1]), out[1].size(1), f(out[2]), out[2].size(1), f(out[3]), f(out[4]), ws.data_ptr(), n,
                      stream_of(lam)),
           "rt_diffattn_bwd", false);
    return out;
  }
};

Tensor diff_attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& lam_in, const OptTensor& cu_q_in, const OptTensor& cu_k_in, int64_t B, int64_t H,
                      int64_t Hkv, int64_t Lq, int64_t Lk, bool causal, const OptTensor& ids_in, const OptTensor& w_in, double out_scale, double eps, c10::optional<double> scale) {
  const char* what = "diff_attention";
  const Tensor w_any = got(w_in);
  no_tangent(what, {&q_in, &k_in, &v_in, &lam_in, &w_any});
  if (B < 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || Lq < 0 || Lk < 0 || B > MOST || H > MOST || Lq > MOST || Lk > MOST)
    bad(what, "B=" + std::to_string(B) + ", H=" + std::to_string(H) + ", H_kv=" + std::to_string(Hkv) + ", Lq=" + std::to_string(Lq) + ", Lk=" + std::to_string(Lk));
  const Tensor q = rows(q_in, -1, "diff_attention q");
  if (q.size(1) == 0 || q.size(1) % (2 * H) != 0) bad(what, std::to_string(q.size(1)) + " query columns do not split into " + std::to_string(H) + " heads of two maps");
  const int64_t hd = q.size(1) / (2 * H);
  if (hd > 64) raise(PyExc_NotImplementedError, "diff_attention: at most 64 columns per map (128 value columns per head), got " + std::to_string(hd));
  const Tensor k = rows(k_in, 2 * Hkv * hd, "diff_attention k"), v = rows(v_in, 2 * Hkv * hd, "diff_attention v");
  if (k.size(0) != v.size(0)) bad(what, std::to_string(k.size(0)) + " key rows and " + std::to_string(v.size(0)) + " value rows");
  check_device(k, q, what);
  check_device(v, q, what);
  if (!cu_q_in.has_value() && q.size(0) != B * Lq) bad(what, std::to_string(q.size(0)) + " query rows for " + std::to_string(B) + " sessions of " + std::to_string(Lq));
  if (!cu_k_in.has_value() && k.size(0) != B * Lk) bad(what, std::to_string(k.size(0)) + " key rows for " + std::to_string(B) + " sessions of " + std::to_string(Lk));
  const Tensor cu_q = ints(cu_q_in, B + 1, q, "diff_attention cu_q"), cu_k = ints(cu_k_in, B + 1, q, "diff_attention cu_k"),
               ids = ints(ids_in, k.size(0), q, "diff_attention key_ids"), lam = vec(lam_in, {H}, q, "diff_attention lam"), w = vec(w_in, {2 * hd}, q, "diff_attention norm_w");
  if (scale.has_value() && !((float)*scale > 0.f && std::isfinite((float)*scale))) bad(what, "the logit scale is positive, got " + std::to_string(*scale));
  if (w.defined()) check_eps(eps, what);
  const AttnMeta m{B, H, Hkv, hd, Lq, Lk, causal, scale.value_or(0.0), out_scale, eps};
  if (on_tape({&q, &k, &v, &lam, &w}))
    return AttentionNode::apply(q, k, v, lam, opt(w), opt(cu_q), opt(cu_k), opt(ids), std::vector<int64_t>{B, H, Hkv, hd, Lq, Lk, causal}, m.scale, out_scale, eps,
                                default_stream_leaves({&q_in, &k_in, &v_in, &lam_in, &w_any}));
  return attention_call(q, k, v, lam, cu_q, cu_k, ids, w, m, nullptr);
}

// ---- norms, gate, residual scale ---------------------------------------------------------------------------------------------------------
struct NormMeta { bool layer; double alpha, eps, p; uint64_t seed, sid; };
variable_list norm_call(const Tensor& x, const Tensor& b, const Tensor& z, const Tensor& sc, const Tensor& pw, const Tensor& pb, const Tensor& nw, const Tensor& nb,
                        const NormMeta& m, Tensor* stat) {
  c10::DeviceGuard guard(x.device());
  variable_list out{like(x)};
  if (nw.defined()) out.push_back(like(x));
  if (stat != nullptr) *stat = at::empty({x.size(0), 4}, x.options());
  status(L.norm_fwd(f(x), f(b), f(z), f(sc), f(pw), f(pb), f(nw), f(nb), m.layer, (float)m.alpha, (float)m.eps, (float)m.p, m.seed, m.sid, x.size(0), x.size(1), f(out[0]),
                    nw.defined() ? f(out[1]) : nullptr, stat != nullptr ? f(*stat) : nullptr, stream_of(x)),
         "rt_norm_gate_fwd", true);
  return out;
}
struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& b, const OptTensor& z_opt, const OptTensor& sc_opt, const OptTensor& pw_opt,
                               const OptTensor& pb_opt, const OptTensor& nw_opt, const OptTensor& nb_opt, bool layer, double alpha, double eps, double p, int64_t seed, int64_t sid,
                               bool held) {
    const Tensor z = got(z_opt), sc = got(sc_opt), pw = got(pw_opt), pb = got(pb_opt), nw = got(nw_opt), nb = got(nb_opt);
    Tensor stat;
    variable_list out = norm_call(x, b, z, sc, pw, pb, nw, nb, {layer, alpha, eps, p, (uint64_t)seed, (uint64_t)sid}, &stat);
    ctx->saved_data["leaves"] = held || default_stream_leaves({&x, &b, &z, &sc, &pw, &pb, &nw, &nb});
    ctx->save_for_backward({nw.defined() ? out[0] : Tensor(), b, z, sc, pw, pb, nw, stat});
    ctx->saved_data["i"] = std::vector<int64_t>{layer, seed, sid, nb.defined()};
    ctx->saved_data["f"] = std::vector<double>{alpha, p};
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("norm_gate_residual");
    capturable(ctx, "norm_gate_residual");
    variable_list out(15);
    Tensor gy = g[0].defined() ? g[0].contiguous() : Tensor(), gh = g.size() > 1 && g[1].defined() ? g[1].contiguous() : Tensor();
    if (!gy.defined() && !gh.defined()) return out;
    const auto s = ctx->get_saved_variables();
    const Tensor &y = s[0], &b = s[1], &z = s[2], &sc = s[3], &pw = s[4], &pb = s[5], &nw = s[6], &stat = s[7];
    const auto i = ctx->saved_data["i"].toIntVector();
    const auto x = ctx->saved_data["f"].toDoubleVector();
    c10::DeviceGuard guard(b.device());
    const int64_t M = b.size(0), d = b.size(1);
    out[0] = like(b);
    out[1] = like(b);
    out[2] = like(z);
    out[3] = like(sc);
    out[4] = like(pw);
    out[5] = like(pb);
    out[6] = like(nw);
    if (i[3]) out[7] = like(nw);
    const size_t n = L.norm_bwd_ws(M, d);
    const Tensor ws = scratch(n, b);
    status(L.norm_bwd(f(gy), f(gh), gh.defined() ? f(y) : nullptr, f(b), f(z), f(sc), f(pw), f(pb), f(nw), i[0], (float)x[0], (float)x[1], (uint64_t)i[1], (uint64_t)i[2], M, d, f(stat),
                      f(out[0]), f(out[1]), f(out[2]), f(out[3]), f(out[4]), f(out[5]), f(out[6]), f(out[7]), ws.defined() ? ws.data_ptr() : nullptr, n, stream_of(b)),
           "rt_norm_gate_bwd", false);
    return out;
  }
};
std::vector<Tensor> norm_gate(const Tensor& x_in, const Tensor& f_in, const OptTensor& z_in, const OptTensor& sc_in, const OptTensor& pw_in, const OptTensor& pb_in,
                              const OptTensor& nw_in, const OptTensor& nb_in, bool layer, double alpha, double eps, double p, uint64_t seed, uint64_t sid) {
  const char* what = "norm_gate_residual";
  const Tensor z_any = got(z_in), sc_any = got(sc_in), pw_any = got(pw_in), pb_any = got(pb_in), nw_any = got(nw_in), nb_any = got(nb_in);
  const std::initializer_list<const Tensor*> given{&x_in, &f_in, &z_any, &sc_any, &pw_any, &pb_any, &nw_any, &nb_any};
  no_tangent(what, given);
  check_f32(x_in, what);
  if (x_in.dim() != 2 || x_in.size(1) == 0) bad(what, "expected [rows, columns], got " + shape(x_in));
  const int64_t d = x_in.size(1);
  if (d > 8192) raise(PyExc_NotImplementedError, "norm_gate_residual: rows of at most 8,192 columns, got " + std::to_string(d));
  const Tensor x = x_in.contiguous(), b = vec(f_in, x_in.sizes(), x_in, what), z = vec(z_in, x_in.sizes(), x_in, what), sc = vec(sc_in, {d}, x_in, what),
               pw = vec(pw_in, {d}, x_in, what), pb = vec(pb_in, {d}, x_in, what), nw = vec(nw_in, {d}, x_in, what), nb = vec(nb_in, {d}, x_in, what);
  check_eps(eps, what);
  if (on_tape({&x, &b, &z, &sc, &pw, &pb, &nw, &nb})) return NormNode::apply(x, b, opt(z), opt(sc), opt(pw), opt(pb), opt(nw), opt(nb), layer, alpha, eps, p, (int64_t)seed, (int64_t)sid,
                                                                            default_stream_leaves(given));
  return norm_call(x, b, z, sc, pw, pb, nw, nb, {layer, alpha, eps, p, seed, sid}, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("rotary", &rotary);
  m.def("diff_lambda", &diff_lambda);
  m.def("diff_attention", &diff_attention);
  m.def("norm_gate", &norm_gate);
}
