// The linear-attention and layer-norm operators as torch functions: argument
// checks, allocation, autograd.  The work goes through the C ABI of gdn2.h,
// whose functions `init` receives as addresses from the loaded library.
// In C++ because a small call's cost is this layer: a decode step 24 -> 8 us, a
// layer norm's forward and backward on few rows 125 -> 68 us against the same in Python
// (autograd runs a C++ backward without the interpreter; torch's own product of two
// tensors with its gradient takes 50 us on the same machine).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/utils/pybind.h>

#include "gdn2.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct {
  decltype(&gdn2_linear_attn_workspace_size) la_ws;
  decltype(&gdn2_linear_attn_fwd) la_fwd;
  decltype(&gdn2_linear_attn_bwd_workspace_size) la_bwd_ws;
  decltype(&gdn2_linear_attn_bwd) la_bwd;
  decltype(&gdn2_linear_attn_recurrent_fwd) la_rec;
  decltype(&gdn2_layer_norm_fwd) ln_fwd;
  decltype(&gdn2_layer_norm_bwd_workspace_size) ln_bwd_ws;
  decltype(&gdn2_layer_norm_bwd) ln_bwd;
  decltype(&gdn2_status_string) status;
  decltype(&gdn2_device_supported) supported;
} api;

void check(int st, const char* what) {
  TORCH_CHECK(st == 0, what, " failed with status ", st, ": ", api.status(st));
}

bool is_dtype(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? GDN2_BF16 : GDN2_F32; }

void require_device(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "gdn2 B200 operators run only on CUDA tensors (no CPU fallback); got a tensor on ", t.device());
  static std::atomic<uint64_t> seen{0};
  const uint64_t bit = uint64_t(1) << (t.get_device() & 63);
  if (seen.load(std::memory_order_relaxed) & bit) return;
  TORCH_CHECK(api.supported(t.get_device()), "libgdn2_b200 is built for sm_100a; device ", t.get_device(), " is not");
  seen.fetch_or(bit, std::memory_order_relaxed);
}

// Tangents would vanish without a trace: the kernels run on the values.
void refuse_tangents(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                "linear attention and layer norm have no forward-mode derivative");
}

// The gradients are not differentiable: under create_graph they lead to a node that
// raises when it is reached on the way to an input or a cotangent, instead of counting as constants.
variable_list once(const variable_list& cotangents, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::edge_list edges = torch::autograd::get_current_node()->next_edges();
  for (torch::autograd::Edge& e : torch::autograd::collect_next_edges(cotangents)) edges.push_back(std::move(e));
  const auto error = std::make_shared<torch::autograd::Error>(
      "the gradients of linear attention and layer norm cannot be differentiated", std::move(edges));
  for (Tensor& t : grads) {
    if (t.defined()) t = t.detach();
    torch::autograd::set_history(t, error);
  }
  return grads;
}

gdn2_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<gdn2_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor bytes(const Tensor& like, size_t n) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }
Tensor like(const Tensor& t, at::ScalarType dt) { return at::empty(t.sizes(), t.options().dtype(dt).requires_grad(false)); }
bool off_grid(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) != 0; }
// contiguous and on the 16-byte grid: `t` itself, or a copy (contiguous() alone returns a tensor off the grid as it is)
Tensor on_grid(const Tensor& t) {
  return !t.defined() || (t.is_contiguous() && !off_grid(t)) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ---------------------------------------------------------------------------
// linear attention
// ---------------------------------------------------------------------------
// `t` itself where the kernels can read it as it lies (contiguous innermost
// dimension, 16-byte aligned base and steps), else a copy, with its steps of
// batch, token and head.  A dimension of one element gets the step of a dense tensor.
Tensor as_view(const Tensor& t, int64_t (&step)[3]) {
  const int64_t B = t.size(0), T = t.size(1), H = t.size(2), D = t.size(3);
  int64_t sb = t.stride(0), st = t.stride(1), sh = t.stride(2);
  if (H == 1) sh = D;
  if (T == 1) st = H * sh;
  if (B == 1) sb = T * st;
  const int64_t per = 16 / t.element_size();
  const bool fits = (t.stride(3) == 1 || D == 1) && sh > 0 && st > 0 && sb > 0 && sh % per == 0 && st % per == 0 &&
                    sb % per == 0 && !off_grid(t);
  if (fits || t.numel() == 0) {
    step[0] = sb, step[1] = st, step[2] = sh;
    if (t.numel() == 0) step[0] = T * H * D, step[1] = H * D, step[2] = D;
    return t;
  }
  step[0] = T * H * D, step[1] = H * D, step[2] = D;
  return t.clone(at::MemoryFormat::Contiguous);
}

// Shapes, types and devices; the number of sequences.  `states`: first dimension
// that initial_state must have, or -1 for one state per sequence.
int64_t check_attn(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& h0, const Tensor& cu,
                   int64_t states) {
  TORCH_CHECK_VALUE(q.dim() == 4 && q.sizes() == k.sizes(), "q and k must have one shape [B, T, H, K]; got ", q.sizes(),
                    " and ", k.sizes(), ".");
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), K = q.size(3);
  TORCH_CHECK_VALUE(v.dim() == 4 && v.size(0) == B && v.size(1) == T && H > 0 && v.size(2) > 0 && v.size(2) % H == 0,
                    "v must have shape [B, T, HV, V] with HV a multiple of H=", H, "; got ", v.sizes(), " vs q ", q.sizes(),
                    ".");
  const int64_t HV = v.size(2), V = v.size(3);
  TORCH_CHECK_VALUE((K == 64 || K == 128) && (V == 64 || V == 128), "head dims K and V must be 64 or 128, got ", K, " and ",
                    V, ".");
  TORCH_CHECK_TYPE(is_dtype(q) && q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                   "q, k, v must all be bf16 or all fp32; got ", q.scalar_type(), ", ", k.scalar_type(), ", ",
                   v.scalar_type(), ".");
  if (g.defined()) {
    TORCH_CHECK_TYPE(is_dtype(g), "g must be bf16 or fp32, got ", g.scalar_type(), ".");
    const bool ok = (g.dim() == 1 && g.size(0) == HV) ||
                    (g.dim() == 3 && g.size(0) == B && g.size(1) == T && g.size(2) == HV);
    TORCH_CHECK_VALUE(ok, "g must have shape [HV] or [B, T, HV]; got ", g.sizes(), " for B=", B, ", T=", T, ", HV=", HV, ".");
  }
  int64_t N = B;
  if (cu.defined()) {
    TORCH_CHECK_VALUE(B == 1, "The batch size is expected to be 1 rather than ", B,
                      " when using `cu_seqlens`. Please flatten variable-length inputs before processing.");
    TORCH_CHECK_VALUE(cu.dim() == 1 && cu.size(0) >= 1, "cu_seqlens must be a vector of N + 1 offsets, got shape ",
                      cu.sizes(), ".");
    N = cu.size(0) - 1;
  }
  if (h0.defined()) {
    TORCH_CHECK_TYPE(h0.scalar_type() == at::kFloat, "initial_state must be in float32, got ", h0.scalar_type(), ".");
    const int64_t n = states < 0 ? N : states;
    TORCH_CHECK_VALUE(h0.dim() == 4 && h0.size(0) == n && h0.size(1) == HV && h0.size(2) == K && h0.size(3) == V,
                      "initial_state must have shape [", n, ", ", HV, ", ", K, ", ", V, "], got ", h0.sizes(), ".");
  }
  const std::pair<const char*, const Tensor*> all[] = {
      {"k", &k}, {"v", &v}, {"g", &g}, {"initial_state", &h0}, {"cu_seqlens", &cu}};
  for (const auto& [name, t] : all)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == q.device(), name, " is on ", t->device(), ", q on ", q.device(), ".");
  refuse_tangents({&q, &k, &v, &g, &h0});
  require_device(q);
  return N;
}

Tensor as_offsets(const Tensor& cu) { return cu.defined() ? cu.to(at::kLong).contiguous() : cu; }

// q, k, v: what as_view returned, with its steps already in `a`
void fill(gdn2_linear_attn_args& a, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& h0,
          const Tensor& ht, const Tensor& o, const Tensor& cu, double scale, int64_t N, int flags) {
  a.B = q.size(0), a.T = q.size(1), a.H = q.size(2), a.HV = v.size(2), a.K = q.size(3), a.V = v.size(3);
  a.N = N;
  if (g.defined()) {
    a.decay = g.dim() == 1 ? GDN2_DECAY_HEAD : GDN2_DECAY_TOKEN;
    a.dtype_g = dtype_of(g);
    if (g.dim() == 1) a.g_stride[2] = g.stride(0);
    else
      for (int i = 0; i < 3; ++i) a.g_stride[i] = g.stride(i);
    a.g = g.const_data_ptr();
  }
  a.cu_seqlens = static_cast<const int64_t*>(ptr(cu));
  a.scale = (float)scale;
  a.flags = flags | (h0.defined() ? GDN2_HAS_H0 : 0) | (ht.defined() ? GDN2_STORE_FINAL : 0);
  a.dtype = dtype_of(q);
  a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr();
  a.h0 = static_cast<const float*>(ptr(h0));
  a.ht = static_cast<float*>(mptr(ht));
  a.o = mptr(o);
}

struct Forward {
  Tensor q, k, v, h0, o, ht, ws;
};
Forward attn_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& g, const Tensor& h00,
                     const Tensor& cu, double scale, bool final_state, int64_t N, bool save) {
  const c10::cuda::CUDAGuard guard(q0.device());
  gdn2_linear_attn_args a{};
  Forward f;
  f.q = as_view(q0, a.q_stride), f.k = as_view(k0, a.k_stride), f.v = as_view(v0, a.v_stride);
  f.h0 = on_grid(h00);
  f.o = like(v0);
  if (final_state)
    f.ht = at::empty({N, v0.size(2), q0.size(3), v0.size(3)}, v0.options().dtype(at::kFloat).requires_grad(false));
  fill(a, f.q, f.k, f.v, g, f.h0, f.ht, f.o, cu, scale, N, save ? GDN2_SAVE_FOR_BWD : 0);
  const size_t need = api.la_ws(&a);
  f.ws = bytes(f.o, need);
  check(api.la_fwd(&a, mptr(f.ws), need, stream_of(f.o)), "gdn2_linear_attn_fwd");
  return f;
}

struct ChunkLinearAttn : torch::autograd::Function<ChunkLinearAttn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& g,
                               const OptTensor& h0, const OptTensor& cu, double scale, bool final_state, int64_t N) {
    Forward f = attn_forward(q, k, v, get(g), get(h0), get(cu), scale, final_state, N, true);
    ctx->save_for_backward({f.q, f.k, f.v, get(g), get(cu), f.ws});  // (not h0: its values are not needed)
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["n"] = N;
    ctx->saved_data["need"] = (int64_t)(wants(get(g)) | wants(get(h0)) << 1 | h0.has_value() << 2);
    ctx->set_materialize_grads(false);
    return final_state ? variable_list{f.o, f.ht} : variable_list{f.o};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &g = s[3], &cu = s[4], &ws = s[5];
    const int64_t N = ctx->saved_data["n"].toInt(), need_grad = ctx->saved_data["need"].toInt();
    const c10::cuda::CUDAGuard guard(q.device());
    gdn2_linear_attn_args a{};
    const Tensor qv = as_view(q, a.q_stride), kv = as_view(k, a.k_stride), vv = as_view(v, a.v_stride);
    fill(a, qv, kv, vv, g, Tensor(), Tensor(), Tensor(), cu, ctx->saved_data["scale"].toDouble(), N,
         GDN2_SAVE_FOR_BWD | (need_grad & 4 ? GDN2_HAS_H0 : 0));
    const Tensor dout = grads[0].defined() ? on_grid(grads[0]) : at::zeros(v.sizes(), v.options());
    const Tensor dht = grads.size() > 1 ? on_grid(grads[1]) : Tensor();
    const Tensor dq = like(q), dk = like(k), dv = like(v);
    const Tensor dg = need_grad & 1 ? like(g) : Tensor();
    Tensor dh0;
    if (need_grad & 2)
      dh0 = at::empty({N, v.size(2), q.size(3), v.size(3)}, v.options().dtype(at::kFloat).requires_grad(false));
    gdn2_linear_attn_grads r{dout.const_data_ptr(), static_cast<const float*>(ptr(dht)), mptr(dq), mptr(dk), mptr(dv),
                             mptr(dg), static_cast<float*>(mptr(dh0))};
    const size_t need = api.la_bwd_ws(&a);
    const Tensor bws = bytes(q, need);
    check(api.la_bwd(&a, &r, ptr(ws), ws.defined() ? (size_t)ws.numel() : 0, mptr(bws), need, stream_of(q)),
          "gdn2_linear_attn_bwd");
    return once(grads, {dq, dk, dv, dg, dh0, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, OptTensor> chunk_linear_attn(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& g,
                                                std::optional<double> scale, const OptTensor& h0, bool final_state,
                                                const OptTensor& cu0) {
  const int64_t N = check_attn(q, k, v, get(g), get(h0), get(cu0), -1);
  const double sc = scale.value_or(1.0 / std::sqrt((double)q.size(3)));
  const Tensor cu = as_offsets(get(cu0));
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(get(g)) || wants(get(h0)))) {
    const variable_list out = ChunkLinearAttn::apply(q, k, v, g, h0, cu.defined() ? OptTensor(cu) : OptTensor(), sc,
                                                     final_state, N);
    return {out[0], final_state ? OptTensor(out[1]) : OptTensor()};
  }
  const at::NoGradGuard no_grad;
  Forward f = attn_forward(q, k, v, get(g), get(h0), cu, sc, final_state, N, false);
  return {f.o, final_state ? OptTensor(f.ht) : OptTensor()};
}

std::tuple<Tensor, OptTensor> recurrent_linear_attn(const Tensor& q0, const Tensor& k0, const Tensor& v0, const OptTensor& g,
                                                    std::optional<double> scale, const OptTensor& h00, bool final_state,
                                                    bool inplace, const OptTensor& cu0, const OptTensor& slots0) {
  const at::NoGradGuard no_grad;
  Tensor h0 = get(h00), slots = get(slots0), ht;
  if (slots.defined())
    TORCH_CHECK_VALUE(inplace && h0.defined() && h0.dim() == 4,
                      "ssm_state_indices needs a pool of states as initial_state and inplace_final_state=True");
  const int64_t N = check_attn(q0, k0, v0, get(g), h0, get(cu0), slots.defined() ? h0.size(0) : -1);
  TORCH_CHECK_VALUE(!inplace || h0.defined(), "inplace_final_state=True requires an initial_state");
  const c10::cuda::CUDAGuard guard(q0.device());
  gdn2_linear_attn_args a{};
  if (slots.defined()) {
    TORCH_CHECK_VALUE(slots.dim() == 1 && slots.size(0) == N && slots.device() == q0.device() &&
                          at::isIntegralType(slots.scalar_type(), false),
                      "ssm_state_indices must be a vector of ", N, " slots on ", q0.device());
    if (slots.scalar_type() != at::kInt || !slots.is_contiguous())
      slots = slots.to(at::kLong).clamp(-1, INT32_MAX).to(at::kInt).contiguous();
    a.num_slots = h0.size(0);
    a.state_indices = slots.const_data_ptr<int>();
  }
  const int64_t K = q0.size(3), V = v0.size(3);
  const int64_t one = v0.size(2) * K * V;  // elements of a state
  if (h0.defined() && h0.numel() > 0 &&
      (h0.stride(3) != 1 || h0.stride(2) != V || (h0.size(1) > 1 && h0.stride(1) != K * V) ||
       (h0.size(0) > 1 && h0.stride(0) % 4) || off_grid(h0))) {
    TORCH_CHECK_VALUE(!inplace, "an initial_state that is updated in place must be contiguous within a state and 16-byte "
                                "aligned");
    h0 = h0.clone(at::MemoryFormat::Contiguous);
  }
  TORCH_CHECK_VALUE(!inplace || h0.size(0) < 2 || h0.stride(0) >= one, "states that are updated in place must not share "
                                                                       "memory");
  const Tensor q = as_view(q0, a.q_stride), k = as_view(k0, a.k_stride), v = as_view(v0, a.v_stride), o = like(v0);
  if (inplace) ht = h0;
  else if (final_state) ht = at::empty({N, v0.size(2), K, V}, o.options().dtype(at::kFloat));
  const Tensor cu = as_offsets(get(cu0));
  fill(a, q, k, v, get(g), h0, ht, o, cu, scale.value_or(1.0 / std::sqrt((double)K)), N, 0);
  a.state_stride_in = h0.defined() && h0.size(0) > 1 ? h0.stride(0) : one;  // (the step of a single state is never taken)
  a.state_stride_out = ht.defined() && ht.size(0) > 1 ? ht.stride(0) : one;
  check(api.la_rec(&a, stream_of(o)), "gdn2_linear_attn_recurrent_fwd");
  if (inplace && !h0.is_inference()) h0.unsafeGetTensorImpl()->bump_version();  // as every update in place
  return {o, inplace ? h00 : ht.defined() ? OptTensor(ht) : OptTensor()};
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

struct Norm {
  Tensor x, w, b, r, y, s, stats;
  gdn2_layer_norm_args a{};
};
Norm norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Tensor& r, bool save) {
  const c10::cuda::CUDAGuard guard(x.device());
  Norm n{dense(x), dense(w), dense(b), dense(r)};
  n.a.D = x.size(-1);
  n.a.rows = x.numel() / n.a.D;
  n.a.eps = (float)eps;
  n.y = like(x);
  if (r.defined()) n.s = like(r);
  if (save) n.stats = at::empty({2, n.a.rows}, x.options().dtype(at::kFloat).requires_grad(false));
  n.a.dtype = dtype_of(x);
  n.a.dtype_residual = dtype_of(r.defined() ? r : x);
  n.a.dtype_weight = w.defined() ? dtype_of(w) : b.defined() ? dtype_of(b) : GDN2_F32;
  n.a.x = n.x.const_data_ptr(), n.a.residual = ptr(n.r), n.a.weight = ptr(n.w), n.a.bias = ptr(n.b);
  n.a.y = mptr(n.y), n.a.s = mptr(n.s);
  if (save) {
    n.a.mean = static_cast<float*>(n.stats.mutable_data_ptr());
    n.a.rstd = n.a.mean + n.a.rows;
  }
  check(api.ln_fwd(&n.a, stream_of(x)), "gdn2_layer_norm_fwd");
  return n;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
                               const OptTensor& r) {
    Norm n = norm_forward(x, get(w), get(b), eps, get(r), true);
    const bool res = n.s.defined();
    ctx->save_for_backward({res ? n.s : n.x, n.w, n.stats});
    // types, and which gradients are wanted
    const int64_t d = (x.scalar_type() == at::kBFloat16 ? 0 : 1) | n.a.dtype_weight << 1 | res << 2 | wants(x) << 3 |
                      wants(get(w)) << 4 | wants(get(b)) << 5 | wants(get(r)) << 6;
    ctx->saved_data["d"] = d;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return res ? variable_list{n.y, n.s} : variable_list{n.y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &w = saved[1], &stats = saved[2];
    const c10::cuda::CUDAGuard guard(s.device());
    const int64_t d = ctx->saved_data["d"].toInt();
    const auto dt = d & 1 ? at::kFloat : at::kBFloat16, wdt = d & 2 ? at::kFloat : at::kBFloat16;
    const bool res = d & 4;
    gdn2_layer_norm_args a{};
    a.D = s.size(-1), a.rows = s.numel() / a.D, a.eps = (float)ctx->saved_data["eps"].toDouble();
    a.dtype = (int)(d & 1), a.dtype_residual = dtype_of(s), a.dtype_weight = (int)(d >> 1 & 1);
    a.residual = res ? s.const_data_ptr() : nullptr, a.weight = ptr(w);
    a.mean = static_cast<float*>(stats.mutable_data_ptr()), a.rstd = a.mean + a.rows;
    const Tensor dy = grads[0].defined() ? grads[0].contiguous() : at::zeros(s.sizes(), s.options().dtype(dt));
    const Tensor ds = res && grads[1].defined() ? grads[1].contiguous() : Tensor();
    const bool need_x = d & 8;
    Tensor dx, dr, dw, db;
    if (d & 64) dr = like(s);
    const bool shared = dr.defined() && s.scalar_type() == dt;  // one gradient serves x and the residual
    if (!shared && (need_x || !dr.defined())) dx = like(s, dt);
    const auto wopt = s.options().dtype(wdt);
    if (d & 16) dw = at::empty({a.D}, wopt);
    if (d & 32) db = at::empty({a.D}, wopt);
    const size_t need = dw.defined() || db.defined() ? api.ln_bwd_ws(&a) : 0;
    const Tensor ws = bytes(s, need);
    gdn2_layer_norm_grads g{dy.const_data_ptr(), ptr(ds), s.const_data_ptr(), mptr(dx), mptr(dr), mptr(dw), mptr(db)};
    check(api.ln_bwd(&a, &g, mptr(ws), need, stream_of(s)), "gdn2_layer_norm_bwd");
    return once(grads, {!need_x ? Tensor() : shared ? dr : dx, dw, db, Tensor(), dr});
  }
};

std::tuple<Tensor, OptTensor> layer_norm(const Tensor& x, const OptTensor& w0, const OptTensor& b0, double eps,
                                         const OptTensor& r0) {
  const Tensor w = get(w0), b = get(b0), r = get(r0);
  TORCH_CHECK_TYPE(x.dim() >= 1 && is_dtype(x), "layer_norm takes bf16 or fp32, got ", x.scalar_type(), ".");
  const int64_t D = x.size(-1);
  TORCH_CHECK_VALUE(D >= 1 && D <= 32768, "layer_norm takes rows of 1 to 32768 elements, got ", D, ".");
  const std::pair<const char*, const Tensor*> params[] = {{"weight", &w}, {"bias", &b}};
  for (const auto& [name, t] : params) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == D, name, " must have shape [", D, "], got ", t->sizes(), ".");
    TORCH_CHECK_TYPE(is_dtype(*t), name, " must be bf16 or fp32, got ", t->scalar_type(), ".");
    TORCH_CHECK_VALUE(t->device() == x.device(), name, " is on ", t->device(), ", x on ", x.device(), ".");
  }
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                   "weight and bias must have one type, got ", w0.has_value() ? w.scalar_type() : at::kFloat, " and ",
                   b0.has_value() ? b.scalar_type() : at::kFloat, ".");
  if (r.defined()) {
    TORCH_CHECK_VALUE(r.sizes() == x.sizes(), "residual must have x's shape ", x.sizes(), ", got ", r.sizes(), ".");
    TORCH_CHECK_TYPE(r.scalar_type() == x.scalar_type() || r.scalar_type() == at::kFloat, "residual must be in x's type ",
                     x.scalar_type(), " or fp32, got ", r.scalar_type(), ".");
    TORCH_CHECK_VALUE(r.device() == x.device(), "residual is on ", r.device(), ", x on ", x.device(), ".");
  }
  refuse_tangents({&x, &w, &b, &r});
  require_device(x);
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) {
    const variable_list out = LayerNorm::apply(x, w0, b0, eps, r0);
    return {out[0], r.defined() ? OptTensor(out[1]) : OptTensor()};
  }
  const at::NoGradGuard no_grad;
  Norm n = norm_forward(x, w, b, eps, r, false);
  return {n.y, r.defined() ? OptTensor(n.s) : OptTensor()};
}

void init(const std::vector<uintptr_t>& f) {
  TORCH_CHECK(f.size() == 10);
  size_t i = 0;
  auto set = [&](auto& p) { p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(f[i++]); };
  set(api.la_ws), set(api.la_fwd), set(api.la_bwd_ws), set(api.la_bwd), set(api.la_rec);
  set(api.ln_fwd), set(api.ln_bwd_ws), set(api.ln_bwd), set(api.status), set(api.supported);
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  namespace py = pybind11;
  using nogil = py::call_guard<py::gil_scoped_release>;
  m.def("init", &init);
  m.def("chunk_linear_attn", &chunk_linear_attn, nogil());
  m.def("recurrent_linear_attn", &recurrent_linear_attn, nogil());
  m.def("layer_norm", &layer_norm, nogil());
}
