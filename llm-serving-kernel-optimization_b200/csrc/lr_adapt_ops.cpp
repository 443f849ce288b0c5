// lr_adapt_ops.cpp -- torch custom ops of the router's training path (with
// their autograd formulas) and of the low-rank adapters.
//
// balanced_gating, gate_projection, dispatch_tokens and combine_tokens are
// differentiable once: a backward pass that is itself recorded
// (create_graph=True) is refused.
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <vector>

#include "lr_ops_common.h"

namespace {

using namespace lr_ops;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Contiguous, 16-byte aligned, of type `type` (a copy only where it is not already).
at::Tensor rows16(const at::Tensor& t, at::ScalarType type) {
  if (t.scalar_type() == type && t.is_contiguous() &&
      (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0)
    return t;
  at::Tensor r = t.detach().to(type).contiguous();
  if (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15u) r = r.clone(at::MemoryFormat::Contiguous);
  return r;
}

// An fp32 weight rounded to fp16 by our own kernel (4 us of host time instead of a cast's 10);
// anything else as rows16.
at::Tensor half_weight(const at::Tensor& w) {
  if (w.scalar_type() != at::kFloat || !w.is_contiguous() || w.numel() % 8 != 0 ||
      (reinterpret_cast<uintptr_t>(w.data_ptr()) & 15u) != 0)
    return rows16(w, at::kHalf);
  auto out = at::empty(w.sizes(), w.options().dtype(at::kHalf));
  check_status(lr_round_half(w.data_ptr<float>(), out.data_ptr(), w.numel(), cur_stream()),
               "gate_projection");
  return out;
}

void check_same_device(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", expected ",
              like.device());
}

void check_int32(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
  check_cuda(t, name);
  check_same_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.numel() == n, name, ": ", n, " int32 expected");
}

void check_once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "lightning_router.", what,
              " is differentiable once: backward with create_graph=True is not supported");
}

// ---------------------------------------------------------------------------
// balanced gating
// ---------------------------------------------------------------------------
// The functions' outputs are the differentiable ones; the others leave through `rest`.
struct BalancedGating : public torch::autograd::Function<BalancedGating> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits_in,
                               const OptTensor& mask_in, int64_t k, double lbw,
                               std::vector<at::Tensor>* rest) {
    TORCH_CHECK(logits_in.is_cuda(), "logits must be a CUDA tensor");
    TORCH_CHECK(logits_in.dim() == 2 && logits_in.scalar_type() == at::kFloat,
                "logits: (T,E) fp32");
    c10::cuda::CUDAGuard g(logits_in.device());
    const at::Tensor logits =
        logits_in.is_contiguous() ? logits_in : logits_in.detach().contiguous();
    const int64_t T = logits.size(0), E = logits.size(1);
    TORCH_CHECK(E >= 1 && E <= 64 && k >= 1 && k <= 8 && k <= E,
                "balanced_gating: 1 <= E <= 64 and 1 <= k <= min(E, 8) expected, got E=", E,
                ", k=", k);
    at::Tensor mask;
    if (given(mask_in)) {
      check_same_device(*mask_in, logits, "token_mask");
      TORCH_CHECK(mask_in->scalar_type() == at::kBool && mask_in->numel() == T,
                  "token_mask: (T,) bool");
      mask = mask_in->reshape({-1}).contiguous();
    }
    auto ids = at::empty({T * k}, logits.options().dtype(at::kInt));
    auto gw = at::empty({T * k}, logits.options());
    auto stats = at::empty({E + 1}, logits.options().dtype(at::kInt));
    auto aux = at::empty({}, logits.options());
    const size_t wsb = lr_balanced_gating_workspace_bytes(as_int(T), as_int(E));
    at::Tensor ws;
    if (wsb) ws = workspace(wsb, logits);
    check_status(lr_balanced_gating(logits.data_ptr<float>(),
                                    mask.defined() ? static_cast<const uint8_t*>(mask.data_ptr())
                                                   : nullptr,
                                    as_int(T), as_int(E), as_int(k), float(lbw),
                                    ids.data_ptr<int32_t>(), gw.data_ptr<float>(),
                                    stats.data_ptr<int32_t>(), aux.data_ptr<float>(),
                                    wsb ? ws.data_ptr() : nullptr, wsb, cur_stream()),
                 "balanced_gating");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits_in, mask, ids, stats});
    ctx->saved_data["k"] = k;
    ctx->saved_data["lbw"] = lbw;
    *rest = {ids, stats.narrow(0, 0, E)};  // without the live count
    return {gw, aux};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("balanced_gating");
    const auto saved = ctx->get_saved_variables();
    const int64_t k = ctx->saved_data["k"].toInt();
    const double lbw = ctx->saved_data["lbw"].toDouble();
    if (!grads[0].defined() && !grads[1].defined()) return {{}, {}, {}, {}, {}};
    c10::cuda::CUDAGuard g(saved[0].device());
    const at::Tensor logits = saved[0].is_contiguous() ? saved[0] : saved[0].detach().contiguous();
    const at::Tensor dw = grads[0].defined() ? grads[0].contiguous() : grads[0];
    const at::Tensor da = grads[1].defined() ? grads[1].contiguous() : grads[1];
    auto dl = at::empty(logits.sizes(), logits.options());
    check_status(
        lr_balanced_gating_backward(
            logits.data_ptr<float>(),
            saved[1].defined() ? static_cast<const uint8_t*>(saved[1].data_ptr()) : nullptr,
            saved[2].data_ptr<int32_t>(), saved[3].data_ptr<int32_t>(), 0,
            dw.defined() ? dw.data_ptr<float>() : nullptr,
            da.defined() ? da.data_ptr<float>() : nullptr, as_int(logits.size(0)),
            as_int(logits.size(1)), as_int(k), float(lbw), dl.data_ptr<float>(), cur_stream()),
        "balanced_gating (backward)");
    return {dl, {}, {}, {}, {}};
  }
};

std::vector<at::Tensor> balanced_gating(const at::Tensor& logits, const OptTensor& token_mask,
                                        int64_t k, double lbw) {
  std::vector<at::Tensor> rest;
  const auto out = BalancedGating::apply(logits, token_mask, k, lbw, &rest);
  return {rest[0], out[0], rest[1], out[1]};
}

// ---------------------------------------------------------------------------
// gate projection
// ---------------------------------------------------------------------------
struct GateProjection : public torch::autograd::Function<GateProjection> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& h, const at::Tensor& w,
                            const OptTensor& bias) {
    TORCH_CHECK(h.is_cuda() && w.is_cuda(), "hidden and gate_weight must be CUDA tensors");
    TORCH_CHECK(h.dim() == 2 && w.dim() == 2 && h.size(1) == w.size(1),
                "gate_projection: hidden (T,d) and gate_weight (E,d) expected");
    TORCH_CHECK(at::isFloatingType(h.scalar_type()) && at::isFloatingType(w.scalar_type()),
                "gate_projection: floating-point inputs expected");
    check_same_device(w, h, "gate_weight");
    c10::cuda::CUDAGuard g(h.device());
    const int64_t T = h.size(0), d = h.size(1), E = w.size(0);
    const at::Tensor hh = rows16(h, at::kHalf), wh = half_weight(w);
    at::Tensor b;
    if (given(bias)) {
      check_same_device(*bias, h, "bias");
      TORCH_CHECK(bias->numel() == E, "bias: (E,)");
      b = *bias;
      if (b.scalar_type() != at::kFloat || !b.is_contiguous())
        b = b.detach().to(at::kFloat).contiguous();
    }
    auto out = at::empty({T, E}, h.options().dtype(at::kFloat));
    check_status(lr_gate_logits(hh.data_ptr(), wh.data_ptr(),
                                b.defined() ? b.data_ptr<float>() : nullptr, as_int(T), as_int(d),
                                as_int(E), out.data_ptr<float>(), cur_stream()),
                 "gate_projection");
    ctx->set_materialize_grads(false);
    // an input that is used as it is goes in as the input, so that writing to it
    // before the backward pass is noticed
    ctx->save_for_backward({hh.data_ptr() == h.data_ptr() ? h : hh,
                            wh.data_ptr() == w.data_ptr() ? w : wh});
    // what needs a gradient, and the types that differ from the kernels'
    int64_t need = h.requires_grad() | w.requires_grad() << 1;
    if (given(bias) && bias->requires_grad()) need |= 4;
    ctx->saved_data["need"] = need;
    if (h.scalar_type() != at::kHalf) ctx->saved_data["h_type"] = int64_t(h.scalar_type());
    if (w.scalar_type() != at::kFloat) ctx->saved_data["w_type"] = int64_t(w.scalar_type());
    if (need & 4 && (bias->scalar_type() != at::kFloat || bias->dim() != 1)) {
      ctx->saved_data["b_type"] = int64_t(bias->scalar_type());
      ctx->saved_data["b_shape"] = bias->sizes().vec();
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("gate_projection");
    if (!grads[0].defined()) return {{}, {}, {}};
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &h = saved[0], &w = saved[1];
    c10::cuda::CUDAGuard g(h.device());
    const at::Tensor dl = grads[0].contiguous();
    const int64_t T = h.size(0), d = h.size(1), E = w.size(0);
    const int64_t need = ctx->saved_data["need"].toInt();
    const bool need_h = need & 1, need_b = need & 4, need_w = need & 6;
    const auto fopt = dl.options();
    at::Tensor dh, dw, db;
    // hidden rows of other types than fp16 get the sums as they are, rounded once at the end
    const bool rows32 = ctx->saved_data.find("h_type") != ctx->saved_data.end();
    if (need_h) dh = at::empty({T, d}, fopt.dtype(rows32 ? at::kFloat : at::kHalf));
    if (need_w) dw = at::empty({E, d}, fopt);
    if (need_b) db = at::empty({E}, fopt);
    const size_t wsb = lr_gate_backward_workspace_bytes(as_int(T), as_int(d), as_int(E));
    at::Tensor ws;
    if (wsb) ws = workspace(wsb, dl);
    const auto run = [&](auto entry, auto* dh_ptr) {
      check_status(entry(h.data_ptr(), w.data_ptr(), dl.data_ptr<float>(), as_int(T), as_int(d),
                         as_int(E), dh_ptr, need_w ? dw.data_ptr<float>() : nullptr,
                         need_b ? db.data_ptr<float>() : nullptr, wsb ? ws.data_ptr() : nullptr,
                         wsb, cur_stream()),
                   "gate_projection (backward)");
    };
    if (rows32)
      run(lr_gate_backward_rows32, need_h ? dh.data_ptr<float>() : nullptr);
    else
      run(lr_gate_backward, need_h ? dh.data_ptr() : nullptr);
    const auto cast = [&](at::Tensor& t, const char* key) {
      const auto it = ctx->saved_data.find(key);
      if (t.defined() && it != ctx->saved_data.end())
        t = t.to(at::ScalarType(it->second.toInt()));
    };
    cast(dh, "h_type");
    cast(dw, "w_type");
    cast(db, "b_type");
    if (const auto it = ctx->saved_data.find("b_shape"); it != ctx->saved_data.end())
      db = db.view(it->second.toIntVector());
    return {dh, dw, db};
  }
};

at::Tensor gate_projection(const at::Tensor& h, const at::Tensor& w, const OptTensor& bias) {
  return GateProjection::apply(h, w, bias);
}

// ---------------------------------------------------------------------------
// dispatch
// ---------------------------------------------------------------------------
using DispatchSig = std::vector<at::Tensor>(const OptTensor&, const at::Tensor&, int64_t, int64_t,
                                            double, bool, bool, const OptTensor&);

// Outputs as topk_gating_dispatch: ids 0, weights 1, tokens 2, offsets 3, kept 4,
// aux 5, permuted 6, routing weights 7, sources 8, slot rows 9.
struct DispatchTokens : public torch::autograd::Function<DispatchTokens> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& logits,
                               int64_t k, int64_t capacity, double lbw, const OptTensor& err,
                               std::vector<at::Tensor>* all) {
    TORCH_CHECK(x.is_cuda() && logits.is_cuda(), "x and logits must be CUDA tensors");
    TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kHalf, "x: (T,d) fp16");
    TORCH_CHECK(logits.dim() == 2 && logits.scalar_type() == at::kFloat &&
                    logits.size(0) == x.size(0),
                "logits: (T,E) fp32");
    check_same_device(logits, x, "logits");
    c10::cuda::CUDAGuard g(x.device());
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("lightning_router::topk_gating_dispatch", "")
                               .typed<DispatchSig>();
    *all = op.call(rows16(x, at::kHalf), logits.detach().contiguous(), k, capacity, lbw, true,
                   true, err);
    const auto& out = *all;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, out[0], out[3], out[9]});
    ctx->saved_data["k"] = k;
    ctx->saved_data["lbw"] = lbw;
    ctx->saved_data["d"] = x.size(1);
    return {out[1], out[5], out[6]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("dispatch_tokens");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor logits = saved[0].detach().contiguous();
    c10::cuda::CUDAGuard g(logits.device());
    const int64_t T = logits.size(0), E = logits.size(1);
    const int64_t k = ctx->saved_data["k"].toInt(), d = ctx->saved_data["d"].toInt();
    const double lbw = ctx->saved_data["lbw"].toDouble();
    at::Tensor dx, dl;
    if (grads[2].defined() && ctx->needs_input_grad(0)) {
      const at::Tensor dp = rows16(grads[2], at::kHalf);
      dx = at::empty({T, d}, dp.options());
      check_status(lr_dispatch_backward(dp.data_ptr(), saved[3].data_ptr<int32_t>(), as_int(T),
                                        as_int(k), as_int(d), dx.data_ptr(), cur_stream()),
                   "dispatch_tokens (backward)");
    }
    if ((grads[0].defined() || grads[1].defined()) && ctx->needs_input_grad(1)) {
      const at::Tensor dw = grads[0].defined() ? grads[0].contiguous() : grads[0];
      const at::Tensor da = grads[1].defined() ? grads[1].contiguous() : grads[1];
      dl = at::empty_like(logits);
      check_status(lr_balanced_gating_backward(
                       logits.data_ptr<float>(), nullptr, saved[1].data_ptr<int32_t>(),
                       saved[2].data_ptr<int32_t>(), 1,
                       dw.defined() ? dw.data_ptr<float>() : nullptr,
                       da.defined() ? da.data_ptr<float>() : nullptr, as_int(T), as_int(E),
                       as_int(k), float(lbw), dl.data_ptr<float>(), cur_stream()),
                   "dispatch_tokens (backward)");
    }
    return {dx, dl, {}, {}, {}, {}, {}};
  }
};

std::vector<at::Tensor> dispatch_tokens(const at::Tensor& x, const at::Tensor& logits, int64_t k,
                                        int64_t capacity, double lbw, const OptTensor& err) {
  std::vector<at::Tensor> all;
  const auto out = DispatchTokens::apply(x, logits, k, capacity, lbw, err, &all);
  all[1] = out[0];
  all[5] = out[1];
  all[6] = out[2];
  return all;
}

// ---------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------
struct CombineTokens : public torch::autograd::Function<CombineTokens> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& w,
                            const at::Tensor& slot_pos, const at::Tensor& offsets,
                            const at::Tensor& kept, int64_t k) {
    TORCH_CHECK(y.is_cuda() && w.is_cuda(), "y and gate_weights must be CUDA tensors");
    const int64_t S = slot_pos.numel();
    TORCH_CHECK(k >= 1 && S % k == 0, "slot count must be T*k");
    TORCH_CHECK(y.dim() == 2 && y.scalar_type() == at::kHalf && y.size(0) == S,
                "y: one fp16 row per slot, (T*k, d)");
    TORCH_CHECK(w.scalar_type() == at::kFloat && w.numel() == S, "gate_weights: (T*k,) fp32");
    check_same_device(w, y, "gate_weights");
    check_int32(slot_pos, y, S, "slot_pos");
    const int64_t E = kept.numel();
    check_int32(kept, y, E, "kept_counts");
    check_int32(offsets, y, E + 1, "offsets");
    c10::cuda::CUDAGuard g(y.device());
    const at::Tensor yc = rows16(y, at::kHalf), wc = w.detach().contiguous();
    const int64_t T = S / k, d = y.size(1);
    auto out = at::empty({T, d}, yc.options());
    check_status(lr_combine(yc.data_ptr(), wc.data_ptr<float>(), slot_pos.data_ptr<int32_t>(),
                            as_int(T), as_int(k), as_int(d), out.data_ptr(), cur_stream()),
                 "combine_tokens");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({yc.data_ptr() == y.data_ptr() ? y : yc, w, slot_pos, offsets, kept});
    ctx->saved_data["k"] = k;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_once("combine_tokens");
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}, {}};
    const auto saved = ctx->get_saved_variables();
    const at::Tensor y = saved[0].detach(), w = saved[1].detach().contiguous();
    c10::cuda::CUDAGuard g(y.device());
    const int64_t k = ctx->saved_data["k"].toInt();
    const int64_t S = y.size(0), d = y.size(1), E = saved[4].numel();
    const at::Tensor dout = rows16(grads[0], at::kHalf);
    const bool need_y = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    at::Tensor dy, dw;
    if (need_y) dy = at::empty({S, d}, y.options());
    if (need_w) dw = at::empty({S}, w.options());
    check_status(lr_combine_backward(dout.data_ptr(), y.data_ptr(), w.data_ptr<float>(),
                                     saved[2].data_ptr<int32_t>(), saved[3].data_ptr<int32_t>(),
                                     saved[4].data_ptr<int32_t>(), as_int(S / k), as_int(k),
                                     as_int(d), as_int(E), need_y ? dy.data_ptr() : nullptr,
                                     need_w ? dw.data_ptr<float>() : nullptr, cur_stream()),
                 "combine_tokens (backward)");
    if (need_w) dw = dw.view(w.sizes());
    return {dy, dw, {}, {}, {}, {}};
  }
};

at::Tensor combine_tokens(const at::Tensor& y, const at::Tensor& w, const at::Tensor& slot_pos,
                          const at::Tensor& offsets, const at::Tensor& kept, int64_t k) {
  return CombineTokens::apply(y, w, slot_pos, offsets, kept, k);
}

// ---------------------------------------------------------------------------
// low-rank adapters
// ---------------------------------------------------------------------------
struct Bank {
  const void* a;
  const void* b;
  const float* scale;
  int64_t n, r, K, N;
};

Bank check_bank(const at::Tensor& a, const at::Tensor& b, const OptTensor& scale,
                const at::Tensor& x) {
  check_cuda(a, "adapter a");
  check_cuda(b, "adapter b");
  check_same_device(a, x, "adapter a");
  check_same_device(b, x, "adapter b");
  TORCH_CHECK(a.dim() == 3 && b.dim() == 3 && a.size(0) == b.size(0) && a.size(1) == b.size(2) &&
                  a.scalar_type() == at::kHalf && b.scalar_type() == at::kHalf,
              "adapters: a (n, rank, K) and b (n, N, rank) fp16 expected");
  const int64_t n = a.size(0), r = a.size(1);
  TORCH_CHECK(n >= 1, "adapters: an empty bank");
  TORCH_CHECK(r >= 8 && r <= 128 && r % 8 == 0 && a.size(2) % 8 == 0 && b.size(1) % 8 == 0,
              "adapters: rank (at most 128), K and N must be multiples of 8, got rank=", r,
              ", K=", a.size(2), ", N=", b.size(1));
  const float* s = nullptr;
  if (given(scale)) {
    check_cuda(*scale, "adapter scale");
    check_same_device(*scale, x, "adapter scale");
    TORCH_CHECK(scale->scalar_type() == at::kFloat && scale->numel() == n,
                "adapter scale: (n,) fp32");
    s = scale->data_ptr<float>();
  }
  TORCH_CHECK(x.size(1) == a.size(2), "adapters: x has ", x.size(1), " columns, a ", a.size(2));
  return {a.data_ptr(), b.data_ptr(), s, n, r, a.size(2), b.size(1)};
}

void check_rows(const at::Tensor& t, const at::Tensor& x, int64_t N, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  check_same_device(t, x, name);
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kHalf && t.size(0) == x.size(0) &&
                  t.size(1) == N,
              name, ": (", x.size(0), ", ", N, ") fp16 expected");
}

// A given result may share memory with the rows it is computed from only as the
// very same tensor.
void check_out(const at::Tensor& out, const at::Tensor& x, int64_t N,
               std::initializer_list<at::Tensor> reads) {
  check_rows(out, x, N, "out");
  TORCH_CHECK(out.is_contiguous() && (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15u) == 0,
              "out must be contiguous and 16-byte aligned");
  const char* o0 = static_cast<const char*>(out.data_ptr());
  const char* o1 = o0 + out.nbytes();
  for (const at::Tensor& t : reads) {
    const char* t0 = static_cast<const char*>(t.data_ptr());
    const char* t1 = t0 + t.nbytes();
    TORCH_CHECK(t0 == o0 || t1 <= o0 || o1 <= t0, "out overlaps an input at another offset");
  }
}

void check_index(const at::Tensor& index, const at::Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.scalar_type() == at::kHalf,
              "x: a CUDA tensor (R,K) fp16 expected");
  check_int32(index, x, x.size(0), "index");
}

at::Tensor adapter_add_rows(const at::Tensor& x_in, const at::Tensor& index, const at::Tensor& a,
                            const at::Tensor& b, const OptTensor& scale,
                            const at::Tensor& base_in, const OptTensor& out_in,
                            const OptTensor& err) {
  check_index(index, x_in);
  const Bank k = check_bank(a, b, scale, x_in);
  check_rows(base_in, x_in, k.N, "base");
  c10::cuda::CUDAGuard g(x_in.device());
  const at::Tensor x = rows16(x_in, at::kHalf), base = rows16(base_in, at::kHalf);
  if (given(out_in)) check_out(*out_in, x, k.N, {base});
  at::Tensor out = given(out_in) ? *out_in : at::empty({x.size(0), k.N}, x.options());
  const int64_t R = x.size(0);
  auto ws = workspace(lr_adapter_workspace_bytes(as_int(R), as_int(k.r), 1), x);
  check_status(lr_adapter_add(x.data_ptr(), as_int(R), as_int(k.K), index.data_ptr<int32_t>(),
                              as_int(k.n), k.a, k.b, k.scale, as_int(k.r), as_int(k.N),
                              base.data_ptr(), out.data_ptr(), ws.data_ptr(), size_t(ws.numel()),
                              err_ptr(err), cur_stream()),
               "adapter_add");
  return out;
}

at::Tensor adapter_swiglu_rows(const at::Tensor& x_in, const at::Tensor& index,
                               const at::Tensor& a_gate, const at::Tensor& b_gate,
                               const OptTensor& scale_gate, const at::Tensor& a_up,
                               const at::Tensor& b_up, const OptTensor& scale_up,
                               const at::Tensor& gate_in, const at::Tensor& up_in,
                               const OptTensor& out_in, const OptTensor& err) {
  check_index(index, x_in);
  const Bank kg = check_bank(a_gate, b_gate, scale_gate, x_in);
  const Bank ku = check_bank(a_up, b_up, scale_up, x_in);
  TORCH_CHECK(kg.n == ku.n && kg.r == ku.r && kg.N == ku.N,
              "adapter_swiglu: the gate and up banks differ in size");
  check_rows(gate_in, x_in, kg.N, "gate");
  check_rows(up_in, x_in, kg.N, "up");
  c10::cuda::CUDAGuard g(x_in.device());
  const at::Tensor x = rows16(x_in, at::kHalf), gate = rows16(gate_in, at::kHalf),
                   up = rows16(up_in, at::kHalf);
  if (given(out_in)) check_out(*out_in, x, kg.N, {gate, up});
  at::Tensor out = given(out_in) ? *out_in : at::empty({x.size(0), kg.N}, x.options());
  const int64_t R = x.size(0);
  auto ws = workspace(lr_adapter_workspace_bytes(as_int(R), as_int(kg.r), 2), x);
  check_status(lr_adapter_swiglu(x.data_ptr(), as_int(R), as_int(kg.K), index.data_ptr<int32_t>(),
                                 as_int(kg.n), kg.a, kg.b, kg.scale, ku.a, ku.b, ku.scale,
                                 as_int(kg.r), as_int(kg.N), gate.data_ptr(), up.data_ptr(),
                                 out.data_ptr(), ws.data_ptr(), size_t(ws.numel()), err_ptr(err),
                                 cur_stream()),
               "adapter_swiglu");
  return out;
}

at::Tensor adapter_add(const at::Tensor& x, const at::Tensor& index, const at::Tensor& a,
                       const at::Tensor& b, const OptTensor& scale, const at::Tensor& base,
                       const OptTensor& err) {
  return adapter_add_rows(x, index, a, b, scale, base, {}, err);
}

void adapter_add_out(const at::Tensor& x, const at::Tensor& index, const at::Tensor& a,
                     const at::Tensor& b, const OptTensor& scale, const at::Tensor& base,
                     const at::Tensor& out, const OptTensor& err) {
  adapter_add_rows(x, index, a, b, scale, base, out, err);
  written(out);
}

at::Tensor adapter_swiglu(const at::Tensor& x, const at::Tensor& index, const at::Tensor& a_gate,
                          const at::Tensor& b_gate, const OptTensor& scale_gate,
                          const at::Tensor& a_up, const at::Tensor& b_up,
                          const OptTensor& scale_up, const at::Tensor& gate,
                          const at::Tensor& up, const OptTensor& err) {
  return adapter_swiglu_rows(x, index, a_gate, b_gate, scale_gate, a_up, b_up, scale_up, gate, up,
                             {}, err);
}

void adapter_swiglu_out(const at::Tensor& x, const at::Tensor& index, const at::Tensor& a_gate,
                        const at::Tensor& b_gate, const OptTensor& scale_gate,
                        const at::Tensor& a_up, const at::Tensor& b_up, const OptTensor& scale_up,
                        const at::Tensor& gate, const at::Tensor& up, const at::Tensor& out,
                        const OptTensor& err) {
  adapter_swiglu_rows(x, index, a_gate, b_gate, scale_gate, a_up, b_up, scale_up, gate, up, out,
                      err);
  written(out);
}

at::Tensor adapter_rows(const at::Tensor& adapter_ids, const at::Tensor& source_idx,
                        const at::Tensor& offsets, const at::Tensor& kept, int64_t num_adapters,
                        const OptTensor& err) {
  check_cuda(adapter_ids, "adapter_ids");
  check_int32(adapter_ids, adapter_ids, adapter_ids.numel(), "adapter_ids");
  const int64_t S = source_idx.numel(), E = kept.numel();
  check_int32(source_idx, adapter_ids, S, "source_indices");
  check_int32(kept, adapter_ids, E, "kept_counts");
  check_int32(offsets, adapter_ids, E + 1, "offsets");
  c10::cuda::CUDAGuard g(adapter_ids.device());
  auto index = at::empty({S}, adapter_ids.options());
  check_status(lr_adapter_rows(adapter_ids.data_ptr<int32_t>(), as_int(adapter_ids.numel()),
                               as_int(num_adapters), source_idx.data_ptr<int32_t>(),
                               offsets.data_ptr<int32_t>(), kept.data_ptr<int32_t>(), as_int(S),
                               as_int(E), index.data_ptr<int32_t>(), err_ptr(err), cur_stream()),
               "adapter_rows");
  return index;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(lightning_router, m) {
  m.def("balanced_gating(Tensor logits, Tensor? token_mask, int k, float lbw) -> Tensor[]");
  m.def("gate_projection(Tensor hidden, Tensor gate_weight, Tensor? bias) -> Tensor");
  m.def(
      "dispatch_tokens(Tensor x, Tensor logits, int k, int capacity, float lbw, Tensor? err) -> "
      "Tensor[]");
  m.def(
      "combine_tokens(Tensor y, Tensor gate_weights, Tensor slot_pos, Tensor offsets, Tensor "
      "kept_counts, int k) -> Tensor");
  m.def(
      "adapter_add(Tensor x, Tensor index, Tensor a, Tensor b, Tensor? scale, Tensor base, "
      "Tensor? err) -> Tensor");
  m.def(
      "adapter_add_out(Tensor x, Tensor index, Tensor a, Tensor b, Tensor? scale, Tensor base, "
      "Tensor(a!) out, Tensor? err) -> ()");
  m.def(
      "adapter_swiglu(Tensor x, Tensor index, Tensor a_gate, Tensor b_gate, Tensor? scale_gate, "
      "Tensor a_up, Tensor b_up, Tensor? scale_up, Tensor gate, Tensor up, Tensor? err) -> "
      "Tensor");
  m.def(
      "adapter_swiglu_out(Tensor x, Tensor index, Tensor a_gate, Tensor b_gate, Tensor? "
      "scale_gate, Tensor a_up, Tensor b_up, Tensor? scale_up, Tensor gate, Tensor up, "
      "Tensor(a!) out, Tensor? err) -> ()");
  m.def(
      "adapter_rows(Tensor adapter_ids, Tensor source_idx, Tensor offsets, Tensor kept_counts, "
      "int num_adapters, Tensor? err) -> Tensor");
}

// The same functions below autograd (inference mode): apply() then records nothing.
TORCH_LIBRARY_IMPL(lightning_router, CUDA, m) {
  m.impl("balanced_gating", &balanced_gating);
  m.impl("gate_projection", &gate_projection);
  m.impl("dispatch_tokens", &dispatch_tokens);
  m.impl("combine_tokens", &combine_tokens);
  m.impl("adapter_add", &adapter_add);
  m.impl("adapter_add_out", &adapter_add_out);
  m.impl("adapter_swiglu", &adapter_swiglu);
  m.impl("adapter_swiglu_out", &adapter_swiglu_out);
  m.impl("adapter_rows", &adapter_rows);
}

TORCH_LIBRARY_IMPL(lightning_router, AutogradCUDA, m) {
  m.impl("balanced_gating", &balanced_gating);
  m.impl("gate_projection", &gate_projection);
  m.impl("dispatch_tokens", &dispatch_tokens);
  m.impl("combine_tokens", &combine_tokens);
}
