// Torch operators over the sequence kernels (K22-K24): allocation, streams and autograd for ops/sequence.py.
//
// The other kernels cross from Python as raw pointers (hip_py.cc) and their autograd nodes are written in Python. These
// are called many times in a training step on small tensors, where that costs more than the kernels: a Python node's
// backward runs on the engine's device thread, and with its allocations and launch takes about 35 us of host time
// there, against about 6 us here. Arguments are checked in ops/sequence.py before they arrive.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include <optional>

#include "kernels.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int code(at::ScalarType t) {  // ElemType of vec_types.h
  switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK_VALUE(false, "fp32, bf16 or fp16 tensors on the GPU");
  }
}

at::ScalarType type_of(int64_t c) { return c == 0 ? at::kFloat : c == 1 ? at::kBFloat16 : at::kHalf; }

Tensor rows(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

Tensor made(at::IntArrayRef size, const Tensor& like, at::ScalarType t) { return at::empty(size, like.options().dtype(t)); }

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor plain(const OptTensor& t) { return t ? *t : Tensor(); }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The kernels carry no tangents: a dual tensor is refused, with or without requires_grad.
void refuse_tangents(const char* who, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), who, ": no forward-mode derivatives on the GPU");
}

// Inside a graph's capture, a leaf whose gradient accumulator an eager graph on the default stream keeps alive would have
// the captured backward pass wait on that stream, which ends the process. Said here instead.
void check_capture(std::initializer_list<const Tensor*> leaves) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor* t : leaves) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (accumulator == nullptr) continue;
    const auto stream = accumulator->stream();
    TORCH_CHECK(!stream || stream->id() != 0, "a graph made outside the capture still holds a leaf of this call: "
                "release its outputs, or capture with leaves of its own");
  }
}

// Gradients that say so when they are differentiated again. Only a pass with create_graph runs with gradients enabled.
template <typename F>
variable_list first_order(const char* who, const variable_list& grads, F&& compute) {
  for (const Tensor& g : grads) refuse_tangents(who, {&g});
  if (!at::GradMode::is_enabled()) return compute();
  variable_list out;
  {
    at::AutoGradMode off(false);
    out = compute();
  }
  for (Tensor& t : out) {
    if (!t.defined()) continue;
    auto error = std::make_shared<torch::autograd::DelayedError>("the sequence operators are differentiable once", 1);
    t = (*error)({t.detach().set_requires_grad(true)})[0];
  }
  return out;
}

// ------------------------------------------------------------------------------------------ embedding
Tensor embedding_run(const Tensor& ids, const Tensor& weight, double scale, at::ScalarType type) {
  const c10::DeviceGuard guard(weight.device());
  const Tensor w = rows(weight);
  std::vector<int64_t> size = ids.sizes().vec();
  size.push_back(w.size(1));
  Tensor out = made(size, w, type);
  rmm::hip::embedding_fwd(ptr(ids), ids.scalar_type() == at::kLong, ptr(w), code(w.scalar_type()), w.stride(0), ptr(out),
                          code(type), ids.numel(), w.size(0), w.size(1), float(scale), stream_of(w));
  return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t pad,
                        int64_t type) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["cols"] = weight.size(1);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["type"] = int64_t(code(weight.scalar_type()));
    return embedding_run(ids, weight, scale, type_of(type));
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Tensor ids = ctx->get_saved_variables()[0];
    return first_order("embedding backward", grads, [&]() -> variable_list {
      const c10::DeviceGuard guard(ids.device());
      const int64_t n = ids.numel(), V = ctx->saved_data["rows"].toInt(), D = ctx->saved_data["cols"].toInt();
      const Tensor dy = rows(grads[0].reshape({n, D}));
      Tensor dw = made({V, D}, dy, type_of(ctx->saved_data["type"].toInt()));
      const Tensor ws = made({rmm::hip::embedding_grad_workspace(n, V, D)}, dy, at::kByte);
      rmm::hip::embedding_grad(ptr(ids), ids.scalar_type() == at::kLong, ptr(dy), code(dy.scalar_type()), dy.stride(0),
                               ptr(dw), code(dw.scalar_type()), n, V, D, ctx->saved_data["pad"].toInt(),
                               float(ctx->saved_data["scale"].toDouble()), ptr(ws), stream_of(dy));
      return {Tensor(), dw, Tensor(), Tensor(), Tensor()};
    });
  }
};

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, int64_t pad, int64_t type) {
  refuse_tangents("embedding", {&weight});
  const Tensor i = ids.contiguous();
  if (!wants_grad({&weight})) return embedding_run(i, weight, scale, type_of(type));
  check_capture({&weight});
  return Embedding::apply(i, weight, scale, pad, type);
}

// ------------------------------------------------------------------------------------------ dropout
// `ctr` (may be undefined) holds the counter in the place of `offset`; `used` (may be undefined) receives it.
Tensor dropout_run(const Tensor& x, const Tensor& res, double p, int64_t seed, int64_t offset, const Tensor& ctr,
                   const Tensor& used) {
  const c10::DeviceGuard guard(x.device());
  const Tensor in = x.contiguous(), add = res.defined() ? res.contiguous() : res;
  Tensor out = made(in.sizes(), in, in.scalar_type());
  rmm::hip::dropout(ptr(in), ptr(add), ptr(out), code(in.scalar_type()), in.numel(), p, uint64_t(seed), uint64_t(offset),
                    ptr<const int64_t>(ctr), ptr<int64_t>(used), stream_of(in));
  return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, double p, int64_t seed,
                        int64_t offset, const OptTensor& counter) {
    const Tensor res = plain(residual), ctr = plain(counter);
    const Tensor used = ctr.defined() ? made({1}, x, at::kLong) : Tensor();
    ctx->save_for_backward({used});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["res"] = res.defined();
    return dropout_run(x, res, p, seed, offset, ctr, used);
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const Tensor used = ctx->get_saved_variables()[0];
    return first_order("dropout backward", grads, [&]() -> variable_list {
      Tensor dx;
      if (ctx->needs_input_grad(0))
        dx = dropout_run(grads[0], Tensor(), ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(),
                         ctx->saved_data["offset"].toInt(), used, Tensor());
      return {dx, ctx->saved_data["res"].toBool() ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

Tensor dropout(const Tensor& x, const OptTensor& res, double p, uint64_t seed, uint64_t offset, const OptTensor& ctr) {
  const Tensor r = plain(res);
  refuse_tangents("dropout", {&x, &r});
  if (!wants_grad({&x, &r})) return dropout_run(x, r, p, int64_t(seed), int64_t(offset), plain(ctr), Tensor());
  check_capture({&x, &r});
  return Dropout::apply(x, res, p, int64_t(seed), int64_t(offset), ctr);
}

// ------------------------------------------------------------------------------------------ gated scan
struct ScanCall {
  rmm::hip::ScanArgs p;
  const void *x = nullptr, *g = nullptr;
  int type = 0;
  Tensor ws;

  // x and gate (undefined: the second half of x) with consecutive channels
  ScanCall(const Tensor& xt, const Tensor& gate, const Tensor& resets, const Tensor& lengths) {
    type = code(xt.scalar_type());
    p.B = xt.size(0), p.L = xt.size(1), p.D = gate.defined() ? xt.size(2) : xt.size(2) / 2;
    p.xsb = xt.stride(0), p.xst = xt.stride(1);
    x = ptr(xt);
    if (gate.defined()) {
      g = ptr(gate);
      p.gsb = gate.stride(0), p.gst = gate.stride(1);
    } else {
      g = static_cast<const char*>(x) + p.D * xt.element_size();
      p.gsb = p.xsb, p.gst = p.xst;
    }
    p.resets = ptr<const uint8_t>(resets);
    p.lengths = ptr<const int64_t>(lengths);
    if (const int64_t n = rmm::hip::gated_scan_workspace(p.B, p.L, p.D, type)) {
      ws = made({n}, xt, at::kByte);
      p.workspace = ptr(ws);
    }
  }
};

// (y, h_last, saved states or undefined)
std::tuple<Tensor, Tensor, Tensor> scan_run(const Tensor& x, const Tensor& gate, const Tensor& h0, const Tensor& resets,
                                            const Tensor& lengths, bool keep) {
  const c10::DeviceGuard guard(x.device());
  ScanCall c(x, gate, resets, lengths);
  Tensor y = made({c.p.B, c.p.L, c.p.D}, x, x.scalar_type()), last = made({c.p.B, c.p.D}, x, at::kFloat), ckpt;
  if (keep) ckpt = made({c.p.B, rmm::hip::gated_scan_checkpoints(c.p.L, c.type), c.p.D}, x, at::kFloat);
  c.p.h0 = ptr<const float>(h0);
  c.p.ckpt = ptr<float>(ckpt);
  c.p.h_last = ptr<float>(last);
  rmm::hip::gated_scan_fwd(c.p, c.x, c.g, ptr(y), c.type, stream_of(x));
  return {y, last, ckpt};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gate, const OptTensor& h0,
                               const OptTensor& resets, const OptTensor& lengths) {
    ctx->set_materialize_grads(false);
    const Tensor xr = rows(x), gr = gate ? rows(*gate) : Tensor(), r = plain(resets), n = plain(lengths);
    auto [y, last, ckpt] = scan_run(xr, gr, plain(h0), r, n, true);
    ctx->save_for_backward({xr, gr, r, n, ckpt});
    ctx->saved_data["h0"] = h0.has_value();
    return {y, last};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    return first_order("gated_scan backward", grads, [&]() -> variable_list {
      const Tensor &x = saved[0], &gate = saved[1], &ckpt = saved[4];
      const c10::DeviceGuard guard(x.device());
      ScanCall c(x, gate, saved[2], saved[3]);
      Tensor dx = made(x.sizes(), x, x.scalar_type()), dg, dh0, dy = grads[0], dh = grads[1];
      c.p.dsb = dx.stride(0), c.p.dst = dx.stride(1);
      void* dgp = static_cast<char*>(ptr(dx)) + c.p.D * x.element_size();
      if (gate.defined()) {
        dg = made(x.sizes(), x, x.scalar_type());
        dgp = ptr(dg);
      }
      if (ctx->saved_data["h0"].toBool()) dh0 = made({c.p.B, c.p.D}, x, at::kFloat);
      if (dy.defined()) {
        dy = rows(dy);
        c.p.ysb = dy.stride(0), c.p.yst = dy.stride(1);
      }
      if (dh.defined()) dh = dh.contiguous();
      c.p.ckpt = ptr<float>(ckpt);
      c.p.dh_last = ptr<const float>(dh);
      c.p.dh0 = ptr<float>(dh0);
      rmm::hip::gated_scan_bwd(c.p, c.x, c.g, ptr(dy), ptr(dx), dgp, c.type, stream_of(x));
      return {dx, dg, dh0, Tensor(), Tensor()};
    });
  }
};

OptTensor flags(const OptTensor& resets) {
  if (!resets) return std::nullopt;
  return (resets->scalar_type() == at::kBool ? *resets : resets->ne(0)).contiguous();
}

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const OptTensor& gate, const OptTensor& h0, const OptTensor& resets,
                                      const OptTensor& lengths) {
  const Tensor g = plain(gate), first = plain(h0);
  refuse_tangents("gated_scan", {&x, &g, &first});
  OptTensor h, n;
  if (h0) h = h0->to(at::kFloat).contiguous();
  if (lengths) n = lengths->to(at::kLong).contiguous();
  const OptTensor r = flags(resets);
  const Tensor state = plain(h);
  if (!wants_grad({&x, &g, &state})) {
    auto [y, last, ckpt] = scan_run(rows(x), gate ? rows(g) : g, state, plain(r), plain(n), false);
    return {y, last};
  }
  check_capture({&x, &g, &first});  // h0 itself: its fp32 copy is no leaf
  const variable_list out = GatedScan::apply(x, gate, h, r, n);
  return {out[0], out[1]};
}

// Whether the memory that a and b span meets (a with any strides that are not negative, b contiguous).
bool meets(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  int64_t last = 0;
  for (int64_t d = 0; d < a.dim(); d++) last += (a.size(d) - 1) * a.stride(d);
  const char *a0 = static_cast<const char*>(a.data_ptr()), *b0 = static_cast<const char*>(b.data_ptr());
  return a0 < b0 + b.nbytes() && b0 < a0 + (last + 1) * a.element_size();
}

std::tuple<Tensor, Tensor> gated_scan_step(const Tensor& x, const OptTensor& gate, const Tensor& state,
                                           const OptTensor& resets, const OptTensor& out) {
  const Tensor gt = plain(gate), ot = plain(out);
  refuse_tangents("gated_scan_step", {&x, &gt, &state, &ot});
  const c10::DeviceGuard guard(x.device());
  // a lane reads its own inputs before it writes its state, but not those of others: inputs under `out` are copied
  const auto apart = [&](const Tensor& t) { return ot.defined() && t.defined() && meets(t, ot) ? t.clone() : t; };
  const Tensor xr = apart(rows(x)), g = apart(gate ? rows(*gate) : Tensor()), r = apart(plain(flags(resets)));
  const int64_t B = state.size(0), D = state.size(1);
  Tensor to = out ? *out : made(state.sizes(), state, at::kFloat), y = made({B, D}, x, x.scalar_type());
  const void* gp = g.defined() ? ptr(g) : static_cast<char*>(ptr(xr)) + D * xr.element_size();
  rmm::hip::gated_scan_step(ptr(xr), xr.stride(0), gp, g.defined() ? g.stride(0) : xr.stride(0), ptr<const uint8_t>(r),
                            ptr<const float>(state), ptr<float>(to), ptr(y), code(x.scalar_type()), B, D, stream_of(x));
  if (out) torch::autograd::impl::bump_version(to);  // written in place
  return {y, to};
}

}  // namespace

PYBIND11_MODULE(_seq, m) {
  m.doc() = "Torch operators over the sequence kernels";
  m.def("embedding", &embedding);
  m.def("dropout", &dropout);
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_step", &gated_scan_step);
}
