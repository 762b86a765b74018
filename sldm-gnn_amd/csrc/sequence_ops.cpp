// PyTorch operators of the sequence encoder (sldm_sage/sequence.py), over the
// C ABI of libsldm_sage.so:
//
//   sldm::layer_norm             layer norm over the last dimension
//   sldm::rotary_axes            rotary positions over several axes
//   sldm::decay_attention        linear attention with a decay for each head
//   sldm::decay_attention_step   one token of it, the state moved on in place
//
// Autograd is in C++ here (torch::autograd::Function): short sequences are
// bound by the host, and a Python autograd function costs several times the
// kernels it launches.  Arguments are checked before the device, so a wrong
// call is refused the same way on any tensor; every kernel runs on the current
// stream of its tensors' device and allocates through the caching allocator.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "sldm_sage.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

int dtype_code(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return SLDM_F32;
  if (t.scalar_type() == at::kBFloat16) return SLDM_BF16;
  TORCH_CHECK_TYPE(false, what, ": unsupported dtype ", t.scalar_type(), " (float32 or bfloat16)");
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == SLDM_OK, what, " failed (status ", rc, "): ", sldm_last_error());
}

void require_gpu(const char* what, const Tensor& ref, std::initializer_list<const Tensor*> ts) {
  TORCH_CHECK(ref.is_cuda(), what, ": sldm_sage runs only on the GPU (HIP/gfx950); got a tensor on '",
              ref.device(), "'. There is no CPU fallback: move the inputs to a ROCm device.");
  for (const Tensor* t : ts)
    if (t && t->defined())
      TORCH_CHECK(t->device() == ref.device(), what, ": tensors on different devices (", ref.device(), ", ",
                  t->device(), ")");
}

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

bool given(const optional<Tensor>& t) { return t.has_value() && t->defined(); }
Tensor or_none(const optional<Tensor>& t) { return given(t) ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// fp32 contiguous view of a small parameter
Tensor f32c(const Tensor& t) {
  if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
  return t.to(at::kFloat).contiguous();
}
// columns contiguous (any other strides are read as they are)
Tensor cols(const Tensor& t) { return t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// The gradients of these operators' gradients do not exist.
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated (create_graph=True)");
}

// Neither do forward-mode ones.  The kernels fill their outputs through pointers, so
// that a tangent would be dropped, and read as zero, where no input requires grad.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what,
                " has no forward-mode derivative; detach the tangents (torch.autograd.forward_ad.unpack_dual)");
}

// --------------------------------------------------------------- layer norm --
struct Rows {
  Tensor t;
  int64_t rows, ld;
};
Rows as_rows(const Tensor& x) {
  const int64_t w = x.size(-1), n = x.numel() / w;
  if (x.is_contiguous()) return {x, n, w};
  Tensor y = x.dim() == 2 ? x : x.reshape({n, w});     // a view where the leading dims allow one
  if (w > 1 && y.stride(1) != 1) y = y.contiguous();
  return {y, n, n > 1 ? y.stride(0) : w};
}

// stats: [2, rows], the rows' means and 1 / sqrt(var + eps)
Tensor norm_fwd(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
  DeviceGuard guard(x.device());
  const Rows r = as_rows(x);
  Tensor y = at::empty(x.sizes(), x.options());
  if (stats) *stats = at::empty({2, r.rows}, x.options().dtype(at::kFloat));
  float* mean = stats ? fptr(*stats) : nullptr;
  const Tensor w = f32c(weight), b = f32c(bias);
  check(sldm_layer_norm_fwd(dtype_code(x, "layer_norm"), r.t.data_ptr(), r.ld, r.rows, x.size(-1), fptr(w), fptr(b),
                            (float)eps, y.data_ptr(), mean, mean ? mean + r.rows : nullptr, stream_of(x)),
        "sldm_layer_norm_fwd");
  return y;
}

struct NormFn : torch::autograd::Function<NormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                        const optional<Tensor>& bias, double eps) {
    Tensor stats;
    const Tensor w = or_none(weight), b = or_none(bias);
    Tensor y = norm_fwd(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["bias"] = b.defined() ? (int64_t)b.scalar_type() : (int64_t)-1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("layer_norm");
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    DeviceGuard guard(x.device());
    const int64_t bias = ctx->saved_data["bias"].toInt(), width = x.size(-1);
    const bool need_x = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(1),
               need_b = bias >= 0 && ctx->needs_input_grad(w.defined() ? 2 : 1);
    const Rows r = as_rows(x), g = as_rows(grads[0].scalar_type() == x.scalar_type() ? grads[0]
                                                                                       : grads[0].to(x.scalar_type()));
    const int code = dtype_code(x, "layer_norm");
    Tensor dx, ws, dw, db;
    if (need_x) dx = at::empty(x.sizes(), x.options());
    const auto f32 = x.options().dtype(at::kFloat);
    const size_t bytes = sldm_layer_norm_bwd_workspace_bytes(code, r.rows, width);
    if (need_w || need_b) {
      ws = at::empty({(int64_t)(bytes / 4)}, f32);
      if (need_w) dw = at::empty({width}, f32);
      if (need_b) db = at::empty({width}, f32);
    }
    const Tensor wf = f32c(w);
    const float* mean = fptr(saved[2]);
    check(sldm_layer_norm_bwd(code, r.t.data_ptr(), r.ld, g.t.data_ptr(), g.ld, r.rows, width, fptr(wf),
                              mean, mean + r.rows, ptr(dx), fptr(dw), fptr(db), ptr(ws),
                              ws.defined() ? bytes : 0, stream_of(x)),
          "sldm_layer_norm_bwd");
    out[0] = dx;
    if (need_w) out[1] = dw.to(w.scalar_type());
    if (need_b) out[2] = db.to((at::ScalarType)bias);
    return out;
  }
};

Tensor layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps) {
  dtype_code(x, "layer_norm");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: the last dimension is normalised; got a tensor of shape ",
                    x.sizes());
  const Tensor w = or_none(weight), b = or_none(bias);
  for (const Tensor* t : {&w, &b})
    if (t->defined()) {
      TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1), "layer_norm: weight and bias are [", x.size(-1),
                        "], got ", t->sizes());
      TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type(),
                       "layer_norm: weight and bias are float32 or of the input's dtype, got ", t->scalar_type());
    }
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must not be negative");
  no_tangents("layer_norm", {&x, &w, &b});
  require_gpu("layer_norm", x, {&w, &b});
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))) return NormFn::apply(x, weight, bias, eps);
  return norm_fwd(x, w, b, eps, nullptr);
}

// ------------------------------------------------------------------- rotary --
// [.., H, D] as [B, T, H, D] (leading dimensions flattened unless there are two)
Tensor as4(const Tensor& t) {
  const Tensor c = cols(t);
  if (c.dim() == 4) return c;
  if (c.dim() == 3) return c.unsqueeze(0);
  return cols(c.reshape({1, c.numel() / (c.size(-1) * c.size(-2)), c.size(-2), c.size(-1)}));
}

int pos_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kInt: return SLDM_POS_I32;
    case at::kLong: return SLDM_POS_I64;
    case at::kFloat: return SLDM_POS_F32;
    case at::kDouble: return SLDM_POS_F64;
    default: TORCH_CHECK_TYPE(false, "rotary_axes: positions are int32, int64, float32 or float64, got ", t.scalar_type());
  }
}

// q (and k) turned; either may be undefined
std::pair<Tensor, Tensor> turn(Tensor q, Tensor k, const Tensor& positions, const Tensor& inv_freq,
                               const std::vector<int64_t>& sections, bool interleaved, bool inverse) {
  const bool swapped = !q.defined();
  if (swapped) std::swap(q, k);
  DeviceGuard guard(q.device());
  const Tensor q4 = as4(q), k4 = k.defined() ? as4(k) : Tensor();
  const int64_t B = q4.size(0), T = q4.size(1), A = (int64_t)sections.size();
  Tensor pos = positions;
  if (q.dim() == 3) pos = pos.unsqueeze(0);
  else if (q.dim() > 4) pos = pos.reshape({1, T, A});
  Tensor oq = at::empty(q.sizes(), q.options()), ok = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
  const int64_t lq[3] = {q4.stride(0), q4.stride(1), q4.stride(2)};
  const int64_t lp[3] = {pos.stride(0), pos.stride(1), pos.stride(2)};
  int64_t lk[3] = {0, 0, 0};
  if (k.defined())
    for (int i = 0; i < 3; ++i) lk[i] = k4.stride(i);
  const Tensor f = inv_freq.contiguous();
  check(sldm_rotary_axes(dtype_code(q, "rotary_axes"), q4.data_ptr(), lq, q4.size(2), ptr(k4), lk,
                         k.defined() ? k4.size(2) : 0, B, T, q4.size(3), pos.data_ptr(), pos_code(pos), lp,
                         f.data_ptr<double>(), sections.data(), A, interleaved, inverse, oq.data_ptr(), ptr(ok),
                         stream_of(q)),
        "sldm_rotary_axes");
  if (swapped) return {Tensor(), oq};
  return {oq, ok};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const optional<Tensor>& k,
                               const Tensor& positions, const Tensor& inv_freq, std::vector<int64_t> sections,
                               bool interleaved) {
    ctx->set_materialize_grads(false);
    const auto out = turn(q, or_none(k), positions, inv_freq, sections, interleaved, false);
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["dtype"] = (int64_t)q.scalar_type();
    variable_list r{out.first};
    if (out.second.defined()) r.push_back(out.second);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("rotary_axes");
    variable_list out(6);
    const bool has_k = grads.size() > 1;
    const auto dt = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    Tensor gq = ctx->needs_input_grad(0) ? grads[0] : Tensor();
    Tensor gk = has_k && ctx->needs_input_grad(1) ? grads[1] : Tensor();
    if (gq.defined()) gq = gq.to(dt);
    if (gk.defined()) gk = gk.to(dt);
    if (!gq.defined() && !gk.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto d = turn(gq, gk, saved[0], saved[1], ctx->saved_data["sections"].toIntVector(),
                        ctx->saved_data["interleaved"].toBool(), true);
    out[0] = d.first;
    if (has_k) out[1] = d.second;
    return out;
  }
};

std::tuple<Tensor, Tensor> rotary_axes(const Tensor& q, const optional<Tensor>& k_in, const Tensor& positions,
                                       const Tensor& inv_freq, at::IntArrayRef sections, bool interleaved) {
  dtype_code(q, "rotary_axes");
  const Tensor k = or_none(k_in);
  TORCH_CHECK_VALUE(q.dim() >= 3, "rotary_axes: q is [.., tokens, heads, head size], got ", q.sizes());
  const auto lead = q.sizes().slice(0, q.dim() - 2);
  int64_t pairs = 0;
  TORCH_CHECK_VALUE(sections.size() >= 1 && sections.size() <= 8, "rotary_axes: 1 to 8 axes, got ", sections.size());
  for (int64_t s : sections) {
    TORCH_CHECK_VALUE(s >= 0 && s <= q.size(-1), "rotary_axes: sections ", sections, " for a head of ", q.size(-1));
    pairs += s;
  }
  TORCH_CHECK_VALUE(pairs >= 1 && 2 * pairs <= q.size(-1), "rotary_axes: sections ", sections, " turn ", pairs,
                    " pairs of a head of ", q.size(-1));
  TORCH_CHECK_VALUE(q.size(-1) <= 1024 && q.size(-2) >= 1, "rotary_axes: 1 or more heads of at most 1024, got ", q.sizes());
  if (k.defined()) {
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "rotary_axes: q is ", q.scalar_type(), ", k ", k.scalar_type());
    TORCH_CHECK_VALUE(k.dim() == q.dim() && k.sizes().slice(0, k.dim() - 2) == lead && k.size(-1) == q.size(-1) &&
                          k.size(-2) >= 1,
                      "rotary_axes: q is ", q.sizes(), ", k ", k.sizes());
  }
  pos_code(positions);
  std::vector<int64_t> want(lead.begin(), lead.end());
  want.push_back((int64_t)sections.size());
  TORCH_CHECK_VALUE(positions.sizes() == at::IntArrayRef(want), "rotary_axes: positions are ", at::IntArrayRef(want), ", got ",
                    positions.sizes());
  TORCH_CHECK_TYPE(inv_freq.scalar_type() == at::kDouble, "rotary_axes: inv_freq is float64, got ", inv_freq.scalar_type());
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && inv_freq.size(0) == pairs, "rotary_axes: inv_freq is [", pairs, "], got ",
                    inv_freq.sizes());
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK(!(grad && (wants(positions) || wants(inv_freq))),
              "rotary_axes: positions and inv_freq have no gradient; detach them");
  no_tangents("rotary_axes", {&q, &k, &positions, &inv_freq});
  require_gpu("rotary_axes", q, {&k, &positions, &inv_freq});
  if (grad && (wants(q) || wants(k))) {
    auto r = RotaryFn::apply(q, k_in, positions, inv_freq, sections.vec(), interleaved);
    return {r[0], r.size() > 1 ? r[1] : at::empty({0}, q.options())};
  }
  auto r = turn(q, k, positions, inv_freq, sections.vec(), interleaved, false);
  return {r.first, r.second.defined() ? r.second : at::empty({0}, q.options())};
}

// ---------------------------------------------------------- decay attention --
struct Dims {
  int64_t B, T, H, Hk, dk, dv;
};
void check_log_decay(const Tensor& t, int64_t H, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what, ": log_decay is float32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == H, what, ": log_decay is [", H, "], got ", t.sizes());
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what,
              ": the decays are fixed numbers and have no gradient; detach log_decay");
}
void check_state(const Tensor& t, const Dims& d, const char* what) {
  if (!t.defined()) return;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what, ": the state is float32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == at::IntArrayRef({d.B, d.H, d.dk, d.dv}), what, ": the state is [", d.B, ", ", d.H, ", ",
                    d.dk, ", ", d.dv, "], got ", t.sizes());
}
// q, k, v with `lead` dimensions before heads and columns
Dims check_qkv(const Tensor& q, const Tensor& k, const Tensor& v, int64_t lead, const char* what) {
  dtype_code(q, what);
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), what, ": q, k and v are ",
                   q.scalar_type(), ", ", k.scalar_type(), " and ", v.scalar_type());
  const char* form = lead == 2 ? "[batch, tokens, heads, head size]" : "[batch, heads, head size]";
  TORCH_CHECK_VALUE(q.dim() == lead + 2 && k.dim() == lead + 2 && v.dim() == lead + 2, what, ": q, k and v are ", form,
                    ", got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  const Dims d{q.size(0), lead == 2 ? q.size(1) : 1, q.size(-2), k.size(-2), q.size(-1), v.size(-1)};
  TORCH_CHECK_VALUE(k.sizes().slice(0, lead) == q.sizes().slice(0, lead) &&
                        v.sizes().slice(0, lead) == q.sizes().slice(0, lead) && k.size(-1) == d.dk && v.size(-2) == d.Hk,
                    what, ": q, k and v do not fit: ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(d.Hk >= 1 && d.H >= 1 && d.H % d.Hk == 0, what, ": ", d.H, " heads over ", d.Hk, " key heads");
  TORCH_CHECK_VALUE(d.dk >= 1 && d.dk <= 128 && d.dv >= 1 && d.dv <= 128, what, ": head sizes are 1 to 128, got ", d.dk,
                    " and ", d.dv);
  return d;
}
struct Ld {
  int64_t s[3];
  // the stride of a dimension of one says nothing, and may be any number
  explicit Ld(const Tensor& t) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) == 1 ? 0 : t.stride(i);
  }
};
Dims dims_of(const Tensor& q, const Tensor& k, const Tensor& v) {
  return {q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), v.size(3)};
}

struct Attended {
  Tensor out, end, states;     // states: before each segment of a long axis (for the backward)
};
Attended attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                const Tensor& lengths, double scale) {
  DeviceGuard guard(q.device());
  const Dims d = dims_of(q, k, v);
  const int code = dtype_code(q, "decay_attention");
  const auto f32 = q.options().dtype(at::kFloat);
  Attended r;
  r.out = at::empty({d.B, d.T, d.H, d.dv}, q.options());
  r.end = at::empty({d.B, d.H, d.dk, d.dv}, f32);
  const size_t bytes = sldm_decay_attention_states_bytes(code, d.B, d.T, d.H, d.Hk, d.dk, d.dv);
  if (bytes) r.states = at::empty({(int64_t)(bytes / 4)}, f32);
  const Ld lq(q), lk(k), lv(v);
  check(sldm_decay_attention_fwd(code, q.data_ptr(), lq.s, k.data_ptr(), lk.s, v.data_ptr(), lv.s, d.B, d.T, d.H, d.Hk,
                                 d.dk, d.dv, fptr(log_decay), (float)scale, fptr(state), ptr(lengths),
                                 lengths.defined() && lengths.scalar_type() == at::kLong, r.out.data_ptr(), fptr(r.end),
                                 fptr(r.states), bytes, stream_of(q)),
        "sldm_decay_attention_fwd");
  return r;
}

struct DecayFn : torch::autograd::Function<DecayFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                               const Tensor& log_decay, const optional<Tensor>& state_in,
                               const optional<Tensor>& lengths_in, double scale) {
    ctx->set_materialize_grads(false);
    const Tensor q = cols(q_in), k = cols(k_in), v = cols(v_in), g = log_decay.contiguous(), lengths = or_none(lengths_in);
    const Tensor state = given(state_in) ? state_in->contiguous() : Tensor();
    const auto r = attend(q, k, v, g, state, lengths, scale);
    ctx->save_for_backward({q, k, v, g, state, lengths, r.states});
    ctx->saved_data["scale"] = scale;
    return {r.out, r.end};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("decay_attention");
    variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &g = saved[3], &state = saved[4], &lengths = saved[5];
    DeviceGuard guard(q.device());
    const Dims d = dims_of(q, k, v);
    const Tensor dout = grads[0].defined() ? cols(grads[0].to(q.scalar_type()))
                                           : at::zeros({d.B, d.T, d.H, d.dv}, q.options());
    const Tensor dend = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor dq, dk, dv, ds;
    if (ctx->needs_input_grad(0)) dq = at::empty(q.sizes(), q.options());
    if (ctx->needs_input_grad(1)) dk = at::empty(k.sizes(), k.options());
    if (ctx->needs_input_grad(2)) dv = at::empty(v.sizes(), v.options());
    if (state.defined() && ctx->needs_input_grad(4)) ds = at::empty(state.sizes(), state.options());
    const int code = dtype_code(q, "decay_attention");
    const size_t bytes = sldm_decay_attention_bwd_workspace_bytes(code, d.B, d.T, d.H, d.Hk, d.dk, d.dv);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)(bytes / 4)}, q.options().dtype(at::kFloat));
    const Ld lq(q), lk(k), lv(v), ld(dout);
    check(sldm_decay_attention_bwd(code, q.data_ptr(), lq.s, k.data_ptr(), lk.s,
                                   v.data_ptr(), lv.s, dout.data_ptr(), ld.s, d.B, d.T, d.H, d.Hk, d.dk, d.dv, fptr(g),
                                   (float)ctx->saved_data["scale"].toDouble(), fptr(state), fptr(saved[6]),
                                   fptr(dend), ptr(lengths),
                                   lengths.defined() && lengths.scalar_type() == at::kLong, ptr(dq), ptr(dk), ptr(dv),
                                   fptr(ds), ptr(ws), bytes, stream_of(q)),
          "sldm_decay_attention_bwd");
    out[0] = dq;
    out[1] = dk;
    out[2] = dv;
    out[4] = ds;
    return out;
  }
};

std::tuple<Tensor, Tensor> decay_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                           const optional<Tensor>& state_in, const optional<Tensor>& lengths_in,
                                           optional<double> scale_in) {
  const char* what = "decay_attention";
  const Dims d = check_qkv(q, k, v, 2, what);
  const Tensor state = or_none(state_in), lengths = or_none(lengths_in);
  check_log_decay(log_decay, d.H, what);
  check_state(state, d, what);
  if (lengths.defined()) {
    TORCH_CHECK_TYPE(lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong,
                     "decay_attention: lengths are int32 or int64, got ", lengths.scalar_type());
    TORCH_CHECK_VALUE(lengths.dim() == 1 && lengths.size(0) == d.B, "decay_attention: lengths are [", d.B, "], got ",
                      lengths.sizes());
  }
  no_tangents(what, {&q, &k, &v, &log_decay, &state});
  require_gpu(what, q, {&k, &v, &log_decay, &state, &lengths});
  const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt((double)d.dk);
  optional<Tensor> lens = lengths_in;
  if (lengths.defined() && !lengths.is_contiguous()) lens = lengths.contiguous();
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(state))) {
    auto r = DecayFn::apply(q, k, v, log_decay, state_in, lens, scale);
    return {r[0], r[1]};
  }
  auto r = attend(cols(q), cols(k), cols(v), log_decay.contiguous(), state.defined() ? state.contiguous() : state,
                  or_none(lens), scale);
  return {r.out, r.end};
}

Tensor decay_attention_step(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& log_decay,
                            Tensor state, optional<double> scale_in) {
  const char* what = "decay_attention_step";
  const Dims d = check_qkv(q_in, k_in, v_in, 1, what);
  check_log_decay(log_decay, d.H, what);
  TORCH_CHECK_VALUE(state.defined(), what, ": the state is needed");
  check_state(state, d, what);
  TORCH_CHECK_VALUE(state.is_contiguous(), what, ": the state is moved on in place and has to be contiguous");
  TORCH_CHECK(!(at::GradMode::is_enabled() && (wants(q_in) || wants(k_in) || wants(v_in) || wants(state))), what,
              " moves the state on in place and has no gradient; use decay_attention, or torch.no_grad()");
  no_tangents(what, {&q_in, &k_in, &v_in, &log_decay, &state});
  require_gpu(what, q_in, {&k_in, &v_in, &log_decay, &state});
  DeviceGuard guard(q_in.device());
  const Tensor q = cols(q_in), k = cols(k_in), v = cols(v_in), g = log_decay.contiguous();
  const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt((double)d.dk);
  Tensor out = at::empty({d.B, d.H, d.dv}, q.options());
  const int64_t lq[2] = {q.stride(0), q.stride(1)}, lk[2] = {k.stride(0), k.stride(1)}, lv[2] = {v.stride(0), v.stride(1)};
  check(sldm_decay_attention_step(dtype_code(q, what), q.data_ptr(), lq, k.data_ptr(), lk, v.data_ptr(), lv, d.B, d.H,
                                  d.Hk, d.dk, d.dv, fptr(g), (float)scale, fptr(state), out.data_ptr(), stream_of(q)),
        "sldm_decay_attention_step");
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();   // autograd sees the write
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sldm, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("rotary_axes(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, int[] sections, bool interleaved) -> "
        "(Tensor, Tensor)");
  m.def("decay_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? state, Tensor? lengths, "
        "float? scale) -> (Tensor, Tensor)");
  m.def("decay_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, float? scale) -> "
        "Tensor");
}

// Differentiable as a whole, so above autograd: the operators are their own
// autograd kernels, for every device (other devices are refused inside).
TORCH_LIBRARY_IMPL(sldm, CompositeImplicitAutograd, m) {
  m.impl("layer_norm", layer_norm);
  m.impl("rotary_axes", rotary_axes);
  m.impl("decay_attention", decay_attention);
  m.impl("decay_attention_step", decay_attention_step);
}
