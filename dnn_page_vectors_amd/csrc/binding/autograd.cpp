// Autograd nodes in C++ (Python module pagevec_torch) of the operators called by themselves; the transformer tower's own
// layers are Python nodes over the same kernels (ops/*.py).
//
// A Python autograd.Function around two small kernels costs about 100 us of host time per forward and
// backward on this host (the backward runs on the engine's device thread, which has to take the
// interpreter for every line of it); the same calls from C++ cost 49 us (1440 tokens x 300, the same kernels), a lookup
// alone 8 instead of 12.4 us.  The kernels themselves are those of the HIP library: their
// launchers' addresses are handed in by init(), so that the release and the debug library both work.
// Arguments are checked in Python (ops/*.py) before they come here.
#include <ATen/ATen.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>
#include <vector>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Launchers {
  int (*wattn_fwd)(const void*, const void*, const void*, void*, const long*, const void*, long, int, float*, void*,
                   int, int, int, int, int, int, int, int, float, void*) = nullptr;
  long (*wattn_bwd_ws)(int, int, int, int, int, int, int) = nullptr;
  int (*wattn_bwd)(const void*, const void*, const void*, const void*, const void*, void*, void*, void*, const long*,
                   const void*, long, int, float*, const void*, float*, float*, long, int, int, int, int, int, int, int, int, float,
                   void*) = nullptr;
  int (*temb_fwd)(const void*, int, const void*, int, void*, int, long, long, int, float, const float*, const float*,
                  const int*, const int*, int, void*) = nullptr;
  long (*temb_grad_ws)(long, long, int) = nullptr;
  int (*temb_grad)(const void*, int, const void*, int, float*, long, long, int, long, float, int, void*, long,
                   void*) = nullptr;
  int (*pack)(const void*, int, void*, void*, long, int, void*) = nullptr;
  int (*unpack)(const void*, const void*, void*, int, long, int, void*) = nullptr;
  int (*gelu_fwd)(const void*, const float*, void*, void*, void*, long, int, void*) = nullptr;
  long (*gelu_bwd_ws)(long, int) = nullptr;
  int (*gelu_bwd)(const void*, const void*, const void*, void*, void*, float*, int, float*, long, int, void*) = nullptr;
} hip;

template <typename F>
void take(const pybind11::dict& d, const char* name, F& f) {
  f = reinterpret_cast<F>(d[name].cast<size_t>());
}

void init(const pybind11::dict& d) {
  take(d, "pv_wattn_fwd", hip.wattn_fwd);
  take(d, "pv_wattn_bwd_ws", hip.wattn_bwd_ws);
  take(d, "pv_wattn_bwd", hip.wattn_bwd);
  take(d, "pv_temb_fwd", hip.temb_fwd);
  take(d, "pv_temb_grad_ws", hip.temb_grad_ws);
  take(d, "pv_temb_grad", hip.temb_grad);
  take(d, "pv_ckpt8_pack", hip.pack);
  take(d, "pv_ckpt8_unpack", hip.unpack);
  take(d, "pv_ckpt8_gelu_fwd", hip.gelu_fwd);
  take(d, "pv_ckpt8_gelu_bwd_ws", hip.gelu_bwd_ws);
  take(d, "pv_ckpt8_gelu_bwd", hip.gelu_bwd);
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check(int rc, const char* name) { TORCH_CHECK(rc == 0, name, " failed with status ", rc); }

float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

// Gradients that a backward with create_graph returns have no graph of their own: using them again is an error,
// not a silent zero.
variable_list once(variable_list&& out, const char* what) {
  if (!at::GradMode::is_enabled()) return std::move(out);
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once",
                                                             static_cast<int64_t>(out.size()));
  return (*err)(std::move(out));
}

// The kernels run below autograd, where a forward-mode tangent would be lost: an error, not a silent result without one.
void refuse_tangents(std::initializer_list<const Tensor*> ts, const char* what) {
  for (const Tensor* t : ts) TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

// Autograd keeps one accumulation node per leaf, on the stream of the graph that first used it, for as long as a graph
// holds it.  A captured backward would have to wait for that stream, which the capture does not survive (nor does
// the process, when the broken graph is destroyed): such a capture is refused while it is still whole.
void check_capture(std::initializer_list<const Tensor*> ts, const char* what) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor* t : ts) {
    if (!t->is_cuda() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto s = node->stream();
    TORCH_CHECK(s && *s == c10::hip::getCurrentHIPStream(t->get_device()).unwrap(), what,
                ": a graph made on another stream still holds an argument of this capture (delete its outputs first)");
  }
}

// Memset nodes of a captured graph (a hipGraph_t).  Replays after the first have run such nodes wrongly.
int64_t graph_memsets(size_t graph) {
  size_t n = 0;
  TORCH_CHECK(hipGraphGetNodes(reinterpret_cast<hipGraph_t>(graph), nullptr, &n) == hipSuccess, "hipGraphGetNodes failed");
  std::vector<hipGraphNode_t> nodes(n);
  if (n) TORCH_CHECK(hipGraphGetNodes(reinterpret_cast<hipGraph_t>(graph), nodes.data(), &n) == hipSuccess, "hipGraphGetNodes failed");
  int64_t sets = 0;
  for (const hipGraphNode_t node : nodes) {
    hipGraphNodeType type;
    TORCH_CHECK(hipGraphNodeGetType(node, &type) == hipSuccess, "hipGraphNodeGetType failed");
    sets += type == hipGraphNodeTypeMemset;
  }
  return sets;
}

// ---- windowed attention ------------------------------------------------------------------------------------------

// t, or a copy of it where the kernels' 16-byte row reads or 32-bit offsets within a tile of 64 rows could not take it
Tensor rows16(const Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<size_t>(t.data_ptr()) % 16 == 0 && t.stride(1) < (1 << 24);
  for (int i = 0; i < 3 && ok; ++i) ok = t.size(i) <= 1 || t.stride(i) % 8 == 0;
  return ok ? t : t.is_contiguous() ? t.clone() : t.contiguous();
}

struct Window {
  int left, right, sinks;
  float scale;
};

void strides(long* st, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    for (int i = 0; i < 3; ++i) *st++ = t->stride(i);
}

void attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask, const Window& w,
                       const Tensor& out, const Tensor& lse, const Tensor& rest) {
  long st[12];
  strides(st, {&q, &k, &v, &out});
  const int H = q.size(2), G = H / k.size(2);
  check(hip.wattn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), st, mask.defined() ? mask.data_ptr() : nullptr,
                      mask.defined() ? mask.stride(0) : 0, mask.defined() ? mask.element_size() : 1, floats(lse),
                      rest.defined() ? rest.data_ptr() : nullptr, q.size(0), q.size(1), H, G, q.size(3), w.left, w.right, w.sinks, w.scale, stream_of(q)),
        "pv_wattn_fwd");
}

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0,
                        const std::optional<Tensor>& mask, int64_t left, int64_t right, int64_t sinks, double scale) {
    const c10::DeviceGuard guard(q0.device());
    const Tensor q = rows16(q0), k = rows16(k0), v = rows16(v0), m = mask ? *mask : Tensor();
    Tensor out = at::empty(q.sizes(), q.options());
    Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    Tensor rest = at::empty({q.size(0), q.size(2), (q.size(1) + 31) / 32 * 32, q.size(3)}, q.options().dtype(at::kByte));
    attention_forward(q, k, v, m, {(int)left, (int)right, (int)sinks, (float)scale}, out, lse, rest);
    ctx->save_for_backward({q, k, v, out, lse, rest, m});
    ctx->saved_data["left"] = left;
    ctx->saved_data["right"] = right;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[3], &lse = s[4], &rest = s[5], &m = s[6];
    const c10::DeviceGuard guard(q.device());
    const int left = ctx->saved_data["left"].toInt(), right = ctx->saved_data["right"].toInt(),
              sinks = ctx->saved_data["sinks"].toInt();
    const float scale = (float)ctx->saved_data["scale"].toDouble();
    const int N = q.size(0), L = q.size(1), H = q.size(2), d = q.size(3), G = H / k.size(2);
    at::AutoDispatchBelowADInplaceOrView below;  // plain tensors from here on
    const Tensor go = rows16(grad[0].to(q.scalar_type()));
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
    const Tensor dd = at::empty(lse.sizes(), lse.options());
    const long n = sinks ? hip.wattn_bwd_ws(N, L, H, G, d, left, sinks) : 0;
    const Tensor ws = n ? at::empty({n}, lse.options()) : Tensor();
    long st[24];
    strides(st, {&q, &k, &v, &out, &go, &dq, &dk, &dv});
    check(hip.wattn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), go.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                        dv.data_ptr(), st, m.defined() ? m.data_ptr() : nullptr, m.defined() ? m.stride(0) : 0,
                        m.defined() ? m.element_size() : 1, floats(lse), rest.data_ptr(), floats(dd), floats(ws), n, N, L, H, G, d, left, right,
                        sinks, scale, stream_of(q)),
          "pv_wattn_bwd");
    variable_list g = once({dq, dk, dv}, "window_attention");
    return {g[0], g[1], g[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& mask, int64_t left,
                        int64_t right, int64_t sinks, double scale) {
  refuse_tangents({&q, &k, &v}, "window_attention");
  if (wants_grad({&q, &k, &v})) {
    check_capture({&q, &k, &v}, "window_attention");
    return WindowAttention::apply(q, k, v, mask, left, right, sinks, scale);
  }
  const c10::DeviceGuard guard(q.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor qq = rows16(q), kk = rows16(k), vv = rows16(v);
  const Tensor out = at::empty(qq.sizes(), qq.options());
  attention_forward(qq, kk, vv, mask ? *mask : Tensor(), {(int)left, (int)right, (int)sinks, (float)scale}, out,
                    Tensor(), Tensor());
  return out;
}

// ---- scaled embedding --------------------------------------------------------------------------------------------

Tensor lookup(const Tensor& W, const Tensor& ids, double scale, bool bf16) {
  auto shape = ids.sizes().vec();
  shape.push_back(W.size(1));
  Tensor out = at::empty(shape, W.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  check(hip.temb_fwd(ids.data_ptr(), ids.scalar_type() == at::kLong, W.data_ptr(), W.scalar_type() == at::kBFloat16,
                     out.data_ptr(), bf16, ids.numel(), W.size(0), W.size(1), (float)scale, nullptr, nullptr, nullptr,
                     nullptr, 0, stream_of(W)),
        "pv_temb_fwd");
  return out;
}

struct ScaledEmbedding : torch::autograd::Function<ScaledEmbedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& W, const Tensor& ids, double scale, int64_t pad, bool bf16) {
    const c10::DeviceGuard guard(W.device());
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["V"] = W.size(0);
    ctx->saved_data["bf16_table"] = W.scalar_type() == at::kBFloat16;
    return lookup(W.contiguous(), ids, scale, bf16);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const c10::DeviceGuard guard(ids.device());
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t V = ctx->saved_data["V"].toInt(), T = ids.numel(), E = grad[0].size(-1);
    Tensor g = grad[0].contiguous();
    if (g.scalar_type() != at::kBFloat16 && g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
    Tensor dW = at::empty({V, E}, g.options().dtype(at::kFloat));
    const long n = hip.temb_grad_ws(T, V, E);
    const Tensor ws = n ? at::empty({n}, g.options().dtype(at::kByte)) : Tensor();
    check(hip.temb_grad(ids.data_ptr(), ids.scalar_type() == at::kLong, g.data_ptr(), g.scalar_type() == at::kBFloat16,
                        floats(dW), T, V, E, ctx->saved_data["pad"].toInt(), (float)ctx->saved_data["scale"].toDouble(), 0,
                        n ? ws.data_ptr() : nullptr, n, stream_of(g)),
          "pv_temb_grad");
    if (ctx->saved_data["bf16_table"].toBool()) dW = dW.to(at::kBFloat16);
    return {once({dW}, "scaled_embedding")[0], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor scaled_embedding(const Tensor& W, const Tensor& ids, double scale, int64_t pad, bool bf16) {
  refuse_tangents({&W}, "scaled_embedding");
  if (wants_grad({&W})) {
    check_capture({&W}, "scaled_embedding");
    return ScaledEmbedding::apply(W, ids, scale, pad, bf16);
  }
  const c10::DeviceGuard guard(W.device());
  at::AutoDispatchBelowADInplaceOrView below;
  return lookup(W.contiguous(), ids, scale, bf16);
}

// ---- 8-bit checkpoints -------------------------------------------------------------------------------------------

std::pair<Tensor, Tensor> kept(const Tensor& x) {
  auto shape = x.sizes().vec();
  shape.back() = (shape.back() + 31) / 32;
  return {at::empty(x.sizes(), x.options().dtype(at::kByte)), at::empty(shape, x.options().dtype(at::kByte))};
}

std::pair<Tensor, Tensor> pack(const Tensor& x0) {
  const c10::DeviceGuard guard(x0.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor x = x0.contiguous();
  auto [q, s] = kept(x);
  check(hip.pack(x.data_ptr(), x.scalar_type() == at::kBFloat16, q.data_ptr(), s.data_ptr(), x.numel() / x.size(-1),
                 x.size(-1), stream_of(x)),
        "pv_ckpt8_pack");
  return {q, s};
}

Tensor unpack(const Tensor& q0, const Tensor& s0, bool bf16) {
  const c10::DeviceGuard guard(q0.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor q = q0.contiguous(), s = s0.contiguous();
  Tensor x = at::empty(q.sizes(), q.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  check(hip.unpack(q.data_ptr(), s.data_ptr(), x.data_ptr(), bf16, q.numel() / q.size(-1), q.size(-1), stream_of(q)),
        "pv_ckpt8_unpack");
  return x;
}

struct BiasGelu8 : torch::autograd::Function<BiasGelu8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const Tensor& b0) {
    const c10::DeviceGuard guard(x0.device());
    const Tensor x = x0.contiguous(), b = b0.to(at::kFloat).contiguous();
    Tensor y = at::empty(x.sizes(), x.options());
    auto [q, s] = kept(x);
    check(hip.gelu_fwd(x.data_ptr(), floats(b), y.data_ptr(), q.data_ptr(), s.data_ptr(), x.numel() / x.size(-1), x.size(-1),
                       stream_of(x)),
          "pv_ckpt8_gelu_fwd");
    ctx->save_for_backward({q, s});
    ctx->saved_data["bias_type"] = (int64_t)b0.scalar_type();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto kp = ctx->get_saved_variables();
    const c10::DeviceGuard guard(kp[0].device());
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor dy = grad[0].to(at::kBFloat16).contiguous();
    const int64_t D = dy.size(-1), T = dy.numel() / D;
    Tensor dx = at::empty(dy.sizes(), dy.options()), db = at::empty({D}, dy.options().dtype(at::kFloat));
    const Tensor ws = at::empty({hip.gelu_bwd_ws(T, D)}, db.options());
    check(hip.gelu_bwd(kp[0].data_ptr(), kp[1].data_ptr(), dy.data_ptr(), dx.data_ptr(), nullptr, floats(db), 0, floats(ws), T,
                       D, stream_of(dy)),
          "pv_ckpt8_gelu_bwd");
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["bias_type"].toInt());
    if (type != at::kFloat) db = db.to(type);
    return once({dx, db}, "ckpt8.bias_gelu");
  }
};

}  // namespace

PYBIND11_MODULE(pagevec_torch, m) {
  using pybind11::call_guard;
  using pybind11::gil_scoped_release;
  m.def("init", &init);
  m.def("window_attention", &window_attention, call_guard<gil_scoped_release>());
  m.def("scaled_embedding", &scaled_embedding, call_guard<gil_scoped_release>());
  m.def("pack", &pack, call_guard<gil_scoped_release>());
  m.def("unpack", &unpack, call_guard<gil_scoped_release>());
  m.def("bias_gelu8", [](const Tensor& x, const Tensor& b) {
    refuse_tangents({&x, &b}, "ckpt8.bias_gelu");
    check_capture({&x, &b}, "ckpt8.bias_gelu");
    return Tensor(BiasGelu8::apply(x, b));
  }, call_guard<gil_scoped_release>());
  m.def("graph_memsets", &graph_memsets);
  m.def("check_capture", [](const Tensor& t, const char* what) { check_capture({&t}, what); });
}
