// The routing and low-rank operators as torch functions (module _torch_ops): checks
// of tensors, outputs, and autograd around the C ABI of libxpager.so.
//
// These calls are a few microseconds on the GPU for a decode step, and through ctypes
// and a Python autograd function most of an eager call was the host's time: on a
// B200 host a route of one token took 18 us and a balance loss with its gradient 99 us,
// here 9 and 59 (torch's own sum and its gradient: 47).  The Python modules routing.py and
// adapters.py document the functions; this file keeps their argument checks.
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <sstream>

#include "xpager.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

template <typename... Parts>
std::string words(const Parts &...parts) {
  std::ostringstream s;
  (s << ... << parts);
  return s.str();
}

template <typename... Parts>
void require(bool ok, const Parts &...parts) {
  if (!ok) throw py::value_error(words(parts...));
}

std::string shape_of(const Tensor &t) {
  std::ostringstream s;
  s << "[";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << "]";
  return s.str();
}

std::string type_of(const Tensor &t) { return c10::toString(t.scalar_type()); }

void require_cuda(const Tensor &t) {
  require(t.is_cuda(), "vllm-expert-pager: expected a CUDA tensor, got one on ", t.device().str());
}

// A dual tensor's tangent would be lost, and the result pass for a constant.
void require_no_tangent(const Tensor &t, const char *what) {
  require(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(),
          what, " has no forward-mode derivative");
}

// A status of libxpager.so as native.check words it.
void check_status(int rc, const char *what) {
  if (rc == XP_OK) return;
  const std::string text = words("vllm-expert-pager: ", what, " failed (", rc, ": ",
                                 xp_status_string(rc), ")");
  if (rc < 0) throw py::value_error(text);
  throw std::runtime_error(text);
}

void *stream_of(const Tensor &t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

template <typename P = void>
P *ptr(const Tensor &t) {
  return t.defined() ? static_cast<P *>(t.data_ptr()) : nullptr;
}

// XP_F32, XP_BF16 or XP_F16; -1 for other types.
int type_code(at::ScalarType t) {
  return t == at::kFloat ? XP_F32 : (t == at::kBFloat16 ? XP_BF16 : (t == at::kHalf ? XP_F16 : -1));
}

// ---- routing ----

void check_logits(const Tensor &logits, const MaybeTensor &valid) {
  require(logits.dim() == 2 && type_code(logits.scalar_type()) >= 0,
          "logits must be a float32, bfloat16 or float16 [tokens, experts] tensor, got ",
          type_of(logits), " ", shape_of(logits));
  const int64_t T = logits.size(0), E = logits.size(1);
  require(E >= 1 && E <= XP_MAX_EXPERTS, "between 1 and ", XP_MAX_EXPERTS,
          " experts are supported, got ", E);
  require_no_tangent(logits, "routing");
  require(T <= XP_MAX_TOKENS, "at most ", XP_MAX_TOKENS, " tokens are supported, got ", T);
  if (valid) {
    require((valid->scalar_type() == at::kBool || valid->scalar_type() == at::kByte) &&
                valid->dim() == 1 && valid->size(0) == T,
            "valid must be a bool or uint8 tensor of ", T, " tokens, got ", type_of(*valid), " ",
            shape_of(*valid));
  }
}

void check_devices(const Tensor &logits, const MaybeTensor &valid) {
  require_cuda(logits);
  if (valid) {
    require_cuda(*valid);
    require(valid->device() == logits.device(), "valid is on ", valid->device().str(),
            ", logits on ", logits.device().str());
  }
}

// Logits whose rows are contiguous (any distance between rows).
Tensor rows_of(const Tensor &logits) {
  return logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
}

struct Routed {
  Tensor weights, ids, counts, loss, tokens;
};

// One forward pass on checked arguments; `given`: ids chosen elsewhere, or undefined.
Routed forward_pass(const Tensor &logits, int64_t topk, bool renormalize, const Tensor &valid,
                    bool balance, const Tensor &given, bool count_tokens) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t T = logits.size(0), E = logits.size(1);
  const auto on = logits.options().requires_grad(false);
  Routed r;
  r.counts = at::empty({E}, on.dtype(at::kLong));
  // Without padding the backward pass knows the number of tokens: all rows.
  if (count_tokens && valid.defined()) r.tokens = at::empty({1}, on.dtype(at::kLong));
  if (balance) r.loss = at::empty({}, on.dtype(at::kFloat));
  const int64_t need = xp_route_scratch_bytes(T, E);
  Tensor scratch;
  if (need > 0) scratch = at::empty({need}, on.dtype(at::kByte));
  const int type = type_code(logits.scalar_type());
  if (given.defined()) {
    check_status(xp_balance(ptr(logits), type, T, E, logits.stride(0), ptr<uint8_t>(valid),
                            ptr(given), static_cast<int>(given.element_size()), topk,
                            ptr<int64_t>(r.counts), ptr<int64_t>(r.tokens), ptr<float>(r.loss),
                            ptr(scratch), need, stream_of(logits)),
                 "balance_loss");
  } else {
    r.weights = at::empty({T, topk}, on.dtype(at::kFloat));
    r.ids = at::empty({T, topk}, on.dtype(at::kInt));
    check_status(xp_route(ptr(logits), type, T, E, logits.stride(0), ptr<uint8_t>(valid), topk,
                          renormalize, ptr<float>(r.weights), ptr<int32_t>(r.ids),
                          ptr<int64_t>(r.counts), ptr<int64_t>(r.tokens), ptr<float>(r.loss),
                          ptr(scratch), need, stream_of(logits)),
                 "route");
  }
  return r;
}

Tensor backward_pass(const Tensor &logits, int64_t topk, bool renormalize, const Tensor &valid,
                     const Tensor &ids, const Tensor &weights, const Tensor &grad_weights,
                     const Tensor &counts, const Tensor &tokens, const Tensor &grad_loss) {
  // Under create_graph the result would pass for a constant of the logits.
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "vllm-expert-pager: routing is differentiable once; its gradient cannot be taken "
              "with create_graph=True");
  const c10::cuda::CUDAGuard guard(logits.device());
  const Tensor gw = grad_weights.defined() ? grad_weights.contiguous() : grad_weights;
  Tensor grad = at::empty({logits.size(0), logits.size(1)},
                          logits.options().requires_grad(false));
  const int rc = xp_route_backward(
      ptr(logits), type_code(logits.scalar_type()), logits.size(0), logits.size(1),
      logits.stride(0), ptr<uint8_t>(valid), ptr<int32_t>(ids), ptr<float>(weights), topk,
      renormalize, ptr<float>(gw), ptr<int64_t>(counts), ptr<int64_t>(tokens),
      ptr<float>(grad_loss), ptr(grad), stream_of(logits));
  TORCH_CHECK(rc == XP_OK, "vllm-expert-pager: route_backward failed (", rc, ": ",
              xp_status_string(rc), ")");
  return grad;
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, int64_t topk,
                               bool renormalize, const MaybeTensor &flags, bool balance) {
    const Tensor valid = flags.value_or(Tensor());
    Routed r = forward_pass(logits, topk, renormalize, valid, balance, Tensor(), balance);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.ids, r.counts});
    ctx->save_for_backward({logits, valid, r.ids, r.weights, balance ? r.counts : Tensor(),
                            r.tokens});
    ctx->saved_data["topk"] = topk;
    ctx->saved_data["renormalize"] = renormalize;
    if (balance) return {r.weights, r.ids, r.counts, r.loss};
    return {r.weights, r.ids, r.counts};
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const Tensor loss = grads.size() > 3 ? grads[3] : Tensor();
    Tensor grad;
    if (grads[0].defined() || loss.defined()) {
      const variable_list s = ctx->get_saved_variables();
      grad = backward_pass(s[0], ctx->saved_data["topk"].toInt(),
                           ctx->saved_data["renormalize"].toBool(), s[1], s[2], s[3], grads[0],
                           s[4], s[5], loss);
    }
    return {grad, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct BalanceFunction : torch::autograd::Function<BalanceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &ids,
                               const MaybeTensor &flags) {
    const Tensor valid = flags.value_or(Tensor());
    Routed r = forward_pass(logits, ids.size(1), false, valid, true, ids, true);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.counts});
    ctx->save_for_backward({logits, valid, r.counts, r.tokens});
    ctx->saved_data["topk"] = ids.size(1);
    return {r.loss, r.counts};
  }

  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    Tensor grad;
    if (grads[0].defined()) {
      const variable_list s = ctx->get_saved_variables();
      grad = backward_pass(s[0], ctx->saved_data["topk"].toInt(), false, s[1], Tensor(), Tensor(),
                           Tensor(), s[2], s[3], grads[0]);
    }
    return {grad, Tensor(), Tensor()};
  }
};

py::object maybe(const Tensor &t) { return t.defined() ? py::cast(t) : py::none(); }

py::tuple route(const Tensor &logits_in, int64_t topk, bool renormalize, const MaybeTensor &valid,
                bool balance) {
  check_logits(logits_in, valid);
  const int64_t most = std::min<int64_t>(logits_in.size(1), XP_MAX_TOPK);
  require(topk >= 1 && topk <= most, "topk must be between 1 and ", most, " for ",
          logits_in.size(1), " experts, got ", topk);
  check_devices(logits_in, valid);
  const Tensor logits = rows_of(logits_in);
  const MaybeTensor flags = valid ? MaybeTensor(valid->contiguous()) : MaybeTensor();
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    const variable_list out = RouteFunction::apply(logits, topk, renormalize, flags, balance);
    return py::make_tuple(out[0], out[1], out[2], maybe(balance ? out[3] : Tensor()));
  }
  const Routed r = forward_pass(logits, topk, renormalize, flags.value_or(Tensor()), balance,
                                Tensor(), false);
  return py::make_tuple(r.weights, r.ids, r.counts, maybe(r.loss));
}

py::tuple balance_loss(const Tensor &logits_in, const Tensor &ids_in, const MaybeTensor &valid) {
  check_logits(logits_in, valid);
  require(ids_in.dim() == 2 && ids_in.size(0) == logits_in.size(0) && ids_in.size(1) >= 1,
          "topk_ids must be [", logits_in.size(0), ", topk], got ", shape_of(ids_in));
  require(at::isIntegralType(ids_in.scalar_type(), /*includeBool=*/false),
          "topk_ids must be integers, got ", type_of(ids_in));
  check_devices(logits_in, valid);
  require_cuda(ids_in);
  require(ids_in.device() == logits_in.device(), "topk_ids are on ", ids_in.device().str(),
          ", logits on ", logits_in.device().str());
  Tensor ids = ids_in;
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
  ids = ids.contiguous();
  const Tensor logits = rows_of(logits_in);
  const MaybeTensor flags = valid ? MaybeTensor(valid->contiguous()) : MaybeTensor();
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    const variable_list out = BalanceFunction::apply(logits, ids, flags);
    return py::make_tuple(out[0], out[1]);
  }
  const Routed r = forward_pass(logits, ids.size(1), false, flags.value_or(Tensor()), true, ids,
                                false);
  return py::make_tuple(r.loss, r.counts);
}

// ---- low-rank adapters ----

// Whether two operands of `rows` rows of 16-bit values have bytes in common: first
// address, row stride and width of each.  Columns of one buffer that lie apart have none.
bool overlap(int64_t p, int64_t ps, int64_t pw, int64_t q, int64_t qs, int64_t qw, int64_t rows) {
  if (q + 2 * ((rows - 1) * qs + qw) <= p || p + 2 * ((rows - 1) * ps + pw) <= q) return false;
  if (ps == qs && ps > 0) {
    const int64_t pitch = 2 * ps, off = ((q - p) % pitch + pitch) % pitch;
    if (off >= 2 * pw && off + 2 * qw <= pitch) return false;
  }
  return true;
}

bool is_id_type(const Tensor &t) {
  return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong;
}

Tensor add_low_rank(const Tensor &y_in, const Tensor &x_in, const Tensor &a, const Tensor &b,
                    const Tensor &ids_in, const MaybeTensor &scale_in, const MaybeTensor &map_in,
                    const MaybeTensor &out_in) {
  const Tensor &out = out_in ? *out_in : y_in;
  Tensor x = x_in, y = y_in;
  require(x.dim() == 2 && y.dim() == 2 && a.dim() == 3 && b.dim() == 3 && ids_in.dim() == 1,
          "expected x [M, in], y [M, out], a [slots, rank, in], b [slots, out, rank] and ids [M], "
          "got ",
          shape_of(x), ", ", shape_of(y), ", ", shape_of(a), ", ", shape_of(b), " and ",
          shape_of(ids_in));
  const int64_t M = x.size(0), H = x.size(1), N = y.size(1), S = a.size(0), r = a.size(1);
  require(y.size(0) == M && ids_in.size(0) == M && out.sizes() == y.sizes() && a.size(2) == H &&
              b.size(0) == S && b.size(1) == N && b.size(2) == r,
          "shapes do not fit: x ", shape_of(x), ", y ", shape_of(y), ", out ", shape_of(out),
          ", a ", shape_of(a), ", b ", shape_of(b), ", ids ", shape_of(ids_in));
  const at::ScalarType t = x.scalar_type();
  require((t == at::kBFloat16 || t == at::kHalf) && y.scalar_type() == t && a.scalar_type() == t &&
              b.scalar_type() == t && out.scalar_type() == t,
          "x, y, a, b and out must all be bfloat16 or all float16, got ", type_of(x), ", ",
          type_of(y), ", ", type_of(a), ", ", type_of(b), " and ", type_of(out));
  require(H >= 1 && N >= 1 && S >= 1 && S <= XP_MAX_ADAPTER_SLOTS && r >= 1 && r <= XP_MAX_RANK,
          "sizes must be at least 1, the rank at most ", XP_MAX_RANK, " and the slots at most ",
          XP_MAX_ADAPTER_SLOTS, ", got in ", H, ", out ", N, ", rank ", r, ", slots ", S);
  require(M <= XP_MAX_TOKENS, "at most ", XP_MAX_TOKENS, " rows are supported, got ", M);
  require(is_id_type(ids_in), "ids must be int32 or int64, got ", type_of(ids_in));
  if (scale_in)
    require(scale_in->scalar_type() == at::kFloat && scale_in->dim() == 1 &&
                scale_in->size(0) == S,
            "scale must be float32 [", S, "], got ", type_of(*scale_in), " ",
            shape_of(*scale_in));
  if (map_in)
    require(is_id_type(*map_in) && map_in->dim() == 1,
            "slot_map must be an int32 or int64 vector, got ", type_of(*map_in), " ",
            shape_of(*map_in));
  if (at::GradMode::is_enabled())
    require(!(x.requires_grad() || y.requires_grad() || a.requires_grad() || b.requires_grad() ||
              out.requires_grad() || (scale_in && scale_in->requires_grad())),
            "add_low_rank has no gradient: call it under torch.no_grad() or on detached tensors");
  for (const Tensor *v : {&x_in, &y_in, &a, &b, &out}) require_no_tangent(*v, "add_low_rank");
  if (scale_in) require_no_tangent(*scale_in, "add_low_rank");
  require(a.is_contiguous() && b.is_contiguous(), "adapter slabs must be contiguous");
  require((out.stride(1) == 1 || N == 1) && (out.stride(0) >= N || M <= 1),
          "the rows of out must be contiguous and apart");
  if (M > 0) {
    const auto at = [](const Tensor &v) { return reinterpret_cast<int64_t>(v.data_ptr()); };
    const bool same = at(out) == at(y) && (out.stride(0) == y.stride(0) || M == 1) &&
                      (out.stride(1) == y.stride(1) || N == 1);
    require(!overlap(at(out), out.stride(0), N, at(x), x.stride(0), H, M) &&
                (same || !overlap(at(out), out.stride(0), N, at(y), y.stride(0), N, M)),
            "out may be y itself, and may not overlap x or other rows of y");
    for (const Tensor *v : {&a, &b})
      require(at(*v) + 2 * v->numel() <= at(out) || at(out) + 2 * ((M - 1) * out.stride(0) + N) <= at(*v),
              "out may not overlap the adapter slabs");
  }
  for (const Tensor *v : {&x_in, &y_in, &a, &b, &ids_in, &out}) require_cuda(*v);
  if (scale_in) require_cuda(*scale_in);
  if (map_in) require_cuda(*map_in);
  const auto dev = x.device();
  require(y.device() == dev && a.device() == dev && b.device() == dev && ids_in.device() == dev &&
              out.device() == dev && (!scale_in || scale_in->device() == dev) &&
              (!map_in || map_in->device() == dev),
          "all operands must be on one device");
  if (M == 0) return out;
  const c10::cuda::CUDAGuard guard(dev);
  if (x.stride(1) != 1) x = x.contiguous();
  if (y.stride(1) != 1 && N > 1) y = y.contiguous();
  const Tensor ids = ids_in.contiguous();
  const Tensor scale = scale_in ? scale_in->contiguous() : Tensor();
  const Tensor map = map_in ? map_in->contiguous() : Tensor();
  // A map of no adapters has no storage, and is still a map: no row has an adapter.  Nothing
  // is read from where it points.
  const void *slot_of = map.defined() && map.numel() == 0 ? ptr(ids) : ptr(map);
  // out changes under autograd's eyes, as by torch's own updates in place: a backward pass
  // that saved its old values then raises.
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
  const int64_t need = xp_low_rank_scratch_bytes(M, S);
  Tensor scratch;
  if (need > 0) scratch = at::empty({need}, x.options().dtype(at::kByte).requires_grad(false));
  check_status(
      xp_add_low_rank(ptr(x), x.stride(0), ptr(y), y.stride(0), ptr(out), out.stride(0),
                      type_code(t), M, H, N, r, ptr(a), ptr(b), S, ptr<float>(scale), ptr(ids),
                      static_cast<int>(ids.element_size()), slot_of,
                      map.defined() ? static_cast<int>(map.element_size()) : 0,
                      map.defined() ? map.size(0) : 0, ptr(scratch), need, stream_of(x)),
      "add_low_rank");
  return out;
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("route", &route);
  m.def("balance_loss", &balance_loss);
  m.def("add_low_rank", &add_low_rank);
  m.def("overlap", &overlap);
}
