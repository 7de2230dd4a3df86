// Torch binding of the routed-experts operators: argument checks, allocation and autograd in C++, the work itself through the
// C ABI of libflashsinkhorn_b200.so, whose entry points the Python side hands over when it loads this module. These
// operators run in a few microseconds for a decoding batch; a backward pass through Python costs 60 us of thread and
// interpreter hand-over by itself, three times what all of this takes.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/cuda/EmptyTensor.h>

#include "../../include/flash_sinkhorn_b200.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxExperts = 1024, kMaxK = 32, kBlock = 32, kMaxRows = (int64_t(1) << 31) - 512;  // rows: of products

// Entry points of the library that is loaded.
#define FS_ENTRIES(F)                                                                                                     \
  F(fs_last_error) F(fs_route_bytes) F(fs_route) F(fs_route_grad) F(fs_grouped_mm) F(fs_grouped_mm_in_order) F(fs_grouped_mm_wgrad) F(fs_gated_act) \
  F(fs_gated_act_grad) F(fs_combine) F(fs_combine_grad) F(fs_layer_norm) F(fs_layer_norm_grad_bytes) F(fs_layer_norm_grad) F(fs_weights8)             \
  F(fs_grouped_mm8_bytes) F(fs_grouped_mm8) F(fs_orthogonalize_bytes) F(fs_orthogonalize)
struct Library {
#define FS_MEMBER(name) decltype(&::name) name = nullptr;
  FS_ENTRIES(FS_MEMBER)
#undef FS_MEMBER
} lib;

struct CallFailed : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check_status(const char* name, int status) {
  if (status == FS_OK) return;
  static const char* const names[] = {"FS_OK", "FS_ERR_BAD_ARG", "FS_ERR_UNSUPPORTED", "FS_ERR_CUDA", "FS_ERR_TIMEOUT", "FS_ERR_WORKSPACE"};
  throw CallFailed(std::string(name) + " failed with " + (status > 0 && status < 6 ? names[status] : std::to_string(status)) + ": " +
                   lib.fs_last_error());
}
// A refused argument (ValueError).
struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(const c10::Device& d) { return d.str(); }
template <typename... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  throw Refused((text(parts) + ...));
}
#define REQUIRE(holds, ...) /* the message is put together only where it is needed */ \
  do {                                                                                \
    if (!(holds)) refuse(__VA_ARGS__);                                                \
  } while (0)
#define FS_CALL(name, ...) check_status(#name, lib.name(__VA_ARGS__))

// The device of a call's tensors, current while it lives, and the stream of the caller there.
struct Place {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Place(const Tensor& t) : guard(t.device()), stream(at::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// Without a way through the dispatcher, which takes longer than the allocation.
Tensor fresh(at::IntArrayRef size, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(size, type, like.device(), c10::nullopt); }
Tensor fresh(at::IntArrayRef size, const Tensor& like) { return fresh(size, like.scalar_type(), like); }

int type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? FS_TYPE_F32 : t.scalar_type() == at::kHalf ? FS_TYPE_F16 : FS_TYPE_BF16;
}
std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
const char* type_name(const Tensor& t) { return c10::toString(t.scalar_type()); }
void check_type(const char* name, const Tensor& t, bool fp32) {
  const auto k = t.scalar_type();
  REQUIRE(k == at::kHalf || k == at::kBFloat16 || (fp32 && k == at::kFloat), name, " must be of type ",
                    fp32 ? "float32, float16 or bfloat16" : "float16 or bfloat16", ", got ", type_name(t));
}
void check_cuda(const char* name, const Tensor& t) { REQUIRE(t.is_cuda(), name, " must be a CUDA tensor."); }
void check_place(const char* name, const Tensor& t, const char* first, const Tensor& f) {
  REQUIRE(t.device() == f.device(), name, " must be on the same CUDA device as ", first, " (", f.device(), "), got ", t.device());
}
// A field of a routing of `position`'s tokens and slots.
void check_field(const char* name, const Tensor& t, const Tensor& position, bool per_row, at::ScalarType type, const Tensor& on) {
  const bool fits = per_row ? t.dim() == 1 && t.size(0) == position.size(0) * position.size(1) : t.sizes() == position.sizes();
  REQUIRE(fits && t.scalar_type() == type && t.device() == on.device() && t.is_contiguous(), "routing.", name,
                    " must be a contiguous ", c10::toString(type), " tensor on ", on.device(), " that fits ", shape_of(position),
                    " (tokens, slots), got ", type_name(t), " ", shape_of(t), " on ", t.device());
}
void check_position(const Tensor& position, const Tensor& on) {
  REQUIRE(position.dim() == 2 && position.size(1) >= 1, "routing.position must be of shape (T, k), got ", shape_of(position));
  check_field("position", position, position, false, at::kInt, on);
}
void check_offsets(const Tensor& offsets, const Tensor& on) {
  REQUIRE(offsets.dim() == 1 && offsets.scalar_type() == at::kInt && offsets.is_contiguous() && offsets.device() == on.device() &&
                        offsets.size(0) > 1,
                    "offsets must be a contiguous int32 tensor of shape (E + 1,) on ", on.device());
}

const int* ints(const Tensor& t) { return t.defined() ? t.const_data_ptr<int>() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// Distance of two rows; the stride of a single row says nothing.
int64_t ld(const Tensor& t) { return t.defined() ? std::max(t.stride(0), t.size(1)) : 0; }
Tensor none(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

// `t` itself where its rows are contiguous and do not overlap, else a copy.
Tensor rows_of(const Tensor& t) { return t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous(); }
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// Rows [R, C] of `t`, `from` values apart, copied 8 ceil(C / 8) values apart.
Tensor padded(const Tensor& t, int64_t r, int64_t c, int64_t from) {
  const Place at(t);
  const int64_t to = (c + 7) / 8 * 8;
  Tensor out = fresh({r, to}, t);
  FS_CALL(fs_combine, t.data_ptr(), type_of(t), from, (int)r, (int)r, 1, (int)c, nullptr, nullptr, out.data_ptr(), type_of(t), to, at.stream);
  return out;
}
// `t [R, C]` as tensor loads take it: rows a multiple of 16 bytes apart, the first one aligned to 16 bytes; `t` itself, or a
// copy with padded rows.
Tensor loadable_rows(const Tensor& t0) {
  const int64_t r = t0.size(0), c = t0.size(1);
  if (t0.stride(1) == 1 && t0.stride(0) >= c && t0.stride(0) % 8 == 0 && aligned16(t0)) return t0;
  const Tensor t = rows_of(t0);
  return padded(t, r, c, ld(t)).narrow(1, 0, c);
}
// `w [E, N, K]` where one of its two matrix dimensions is contiguous and the other strides are multiples of 16 bytes.
Tensor loadable_weights(const Tensor& w0) {
  const int64_t e = w0.size(0), n = w0.size(1), k = w0.size(2), se = w0.stride(0), sn = w0.stride(1), sk = w0.stride(2);
  if (aligned16(w0) && se % 8 == 0 && (se > 0 || e == 1) && ((sk == 1 && sn >= k && sn % 8 == 0) || (sn == 1 && sk >= n && sk % 8 == 0))) return w0;
  Tensor w = w0.contiguous();
  if (w.stride(0) != n * k || w.stride(1) != k || w.stride(2) != 1) w = w.as_strided({e, n, k}, {n * k, k, 1});  // of dimensions of size 1
  if (k % 8 == 0 && aligned16(w)) return w;
  REQUIRE(e * n < (int64_t(1) << 31), "weight of ", k, " columns has too many rows to be padded");
  return padded(w, e * n, k, k).view({e, n, (k + 7) / 8 * 8}).narrow(2, 0, k);
}

// Whether a call goes by way of autograd: for a gradient, and for tensors with a forward-mode tangent (whatever the gradient
// mode), which these operators have no rule for: autograd's refusal is better than a result whose tangent counts as zero.
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// For calls whose results carry no gradient: a forward-mode tangent would be dropped without a word.
void check_tangent(const char* name, const Tensor& t) {
  REQUIRE(!t._fw_grad(0).defined(), name, " must not have a forward-mode tangent");
}
// Gradients of a backward pass that cannot be differentiated itself: an error where that is tried.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  return torch::autograd::DelayedError("the gradients of routed experts cannot be differentiated again", grads.size())(std::move(grads));
}

// ------------------------------------------------------------------ raw calls
std::vector<Tensor> route_raw(const Tensor& logits, int64_t k, const Tensor& bias, const Tensor& mask, bool over_all) {
  const Place at(logits);
  const int64_t t = logits.size(0), e = logits.size(1), n = t * k;
  const size_t bytes = lib.fs_route_bytes((int)t, (int)e, (int)k);
  Tensor gates = fresh({t, k}, at::kFloat, logits), experts = fresh({t, k}, at::kInt, logits), offsets = fresh({e + 1}, at::kInt, logits);
  Tensor pairs = fresh({n}, at::kInt, logits), rows = fresh({n}, at::kInt, logits), position = fresh({t, k}, at::kInt, logits), ws;
  if (bytes) ws = fresh({(int64_t)bytes}, at::kByte, logits);
  FS_CALL(fs_route, logits.data_ptr(), type_of(logits), ld(logits), (int)t, (int)e, (int)k, floats(bias), static_cast<const uint8_t*>(data(mask)),
          over_all, floats(gates), experts.data_ptr<int>(), offsets.data_ptr<int>(), pairs.data_ptr<int>(), rows.data_ptr<int>(),
          position.data_ptr<int>(), data(ws), bytes, at.stream);
  return {gates, experts, offsets, pairs, rows, position};
}

// pad: rows of the result a multiple of 8 values apart.
Tensor combine_raw(const Tensor& o, const Tensor& gates, const Tensor& position, at::ScalarType type, bool pad = false) {
  const Place at(o);
  const int64_t t = position.size(0), d = o.size(1), ldy = pad ? (d + 7) / 8 * 8 : d;
  Tensor y = fresh({t, ldy}, type, o);
  FS_CALL(fs_combine, o.data_ptr(), type_of(o), ld(o), (int)o.size(0), (int)t, (int)position.size(1), (int)d, floats(gates), ints(position),
          y.data_ptr(), type_of(y), ldy, at.stream);
  return pad ? y.narrow(1, 0, d) : y;
}
// x[rows] as the products take it, zeros for the rows of no pair.
Tensor gather_raw(const Tensor& x, const Tensor& rows) { return combine_raw(rows_of(x), Tensor(), rows.view({-1, 1}), x.scalar_type(), true); }

Tensor mm_raw(const Tensor& x0, const Tensor& rows0, int64_t count, const Tensor& w0, const Tensor& offsets, bool transposed, bool fp32) {
  const Place at(x0);
  const bool order = rows0.defined() && lib.fs_grouped_mm_in_order((int)count, (int)w0.size(0), (int)w0.size(transposed ? 2 : 1));
  const Tensor x = order ? gather_raw(x0, rows0) : loadable_rows(x0), rows = order ? Tensor() : rows0, w = loadable_weights(w0);
  int64_t n = w.size(1), k = w.size(2), sn = w.stride(1), sk = w.stride(2);
  if (transposed) {
    std::swap(n, k);
    std::swap(sn, sk);
  }
  Tensor out = fresh({count, n}, fp32 ? at::kFloat : x.scalar_type(), x);
  FS_CALL(fs_grouped_mm, x.data_ptr(), ld(x), (int)x.size(0), ints(rows), (int)count, w.data_ptr(), w.stride(0), sn, sk, (int)w.size(0), (int)n,
          (int)k, ints(offsets), out.data_ptr(), type_of(out), n, type_of(x), at.stream);
  return out;
}
Tensor wgrad_raw(const Tensor& dy0, const Tensor& x0, const Tensor& offsets) {
  const Place at(x0);
  const Tensor dy = loadable_rows(dy0), x = loadable_rows(x0);
  const int64_t e = offsets.size(0) - 1, n = dy.size(1), k = x.size(1);
  Tensor out = fresh({e, n, k}, x);
  FS_CALL(fs_grouped_mm_wgrad, dy.data_ptr(), ld(dy), x.data_ptr(), ld(x), (int)x.size(0), (int)e, (int)n, (int)k, ints(offsets), out.data_ptr(),
          type_of(x), at.stream);
  return out;
}

// The result and, with `checkpoint`, one buffer with the codes [R, 2 F] and behind them their scales.
std::pair<Tensor, Tensor> act_raw(const Tensor& u, const Tensor& gates, const Tensor& pairs, bool checkpoint) {
  const Place at(u);
  const int64_t r = u.size(0), f = u.size(1) / 2;
  Tensor h = fresh({r, f}, u), held;
  int8_t* codes = nullptr;
  if (checkpoint) {
    held = fresh({r * (2 * f + 2 * ((f + kBlock - 1) / kBlock))}, at::kByte, u);
    codes = static_cast<int8_t*>(held.data_ptr());
  }
  FS_CALL(fs_gated_act, u.data_ptr(), type_of(u), ld(u), (int)r, (int)f, floats(gates), ints(pairs), h.data_ptr(), codes,
          codes ? reinterpret_cast<uint8_t*>(codes) + r * 2 * f : nullptr, at.stream);
  return {h, held};
}
std::tuple<Tensor, Tensor, Tensor> act_grad_raw(const Tensor& u, const Tensor& held, const Tensor& gates, const Tensor& pairs, const Tensor& position,
                                                const Tensor& dh, bool want_gates, bool want_h) {
  const Place at(dh);
  const int64_t r = dh.size(0), f = dh.size(1);
  Tensor du = fresh({r, 2 * f}, dh), dgates, h;
  if (want_gates) dgates = fresh(gates.sizes(), gates);
  if (want_h) h = fresh({r, f}, dh);
  const auto codes = static_cast<const int8_t*>(data(held));
  FS_CALL(fs_gated_act_grad, data(u), ld(u), codes, codes ? reinterpret_cast<const uint8_t*>(codes) + r * 2 * f : nullptr, type_of(dh), (int)r, (int)f,
          floats(gates), ints(pairs), ints(position), dh.data_ptr(), ld(dh), du.data_ptr(), floats(dgates), data(h), at.stream);
  return {du, dgates, h};
}

// Rows [R, F] of a tensor of any number of dimensions, and the call on them.
Tensor as_rows(const Tensor& t) {
  const int64_t f = t.size(-1);
  return rows_of(t.dim() == 2 ? t : t.reshape({t.numel() / f, f}));
}
struct Norm {
  Tensor y, mean, rstd;
};
Norm norm_raw(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool keep) {
  const Place at(x);
  Norm n;
  n.y = fresh(x.sizes(), x);
  if (keep) {  // one buffer
    const Tensor both = fresh({2, x.size(0)}, at::kFloat, x);
    n.mean = both.select(0, 0);
    n.rstd = both.select(0, 1);
  }
  FS_CALL(fs_layer_norm, data(x), type_of(x), ld(x), (int)x.size(0), (int)x.size(1), data(w), data(b), type_of(w.defined() ? w : b.defined() ? b : x),
          (float)eps, data(n.y), floats(n.mean), floats(n.rstd), at.stream);
  return n;
}

// Codes [E, N, K], rows and experts a multiple of 16 apart, and scales.
std::pair<Tensor, Tensor> weights8_raw(const Tensor& w0) {
  const Place at(w0);
  const Tensor w = w0.stride(2) == 1 && w0.stride(1) >= w0.size(2) && w0.stride(0) >= 0 ? w0 : w0.contiguous();
  const int64_t e = w.size(0), n = w.size(1), k = w.size(2), to = (k + 15) / 16 * 16;
  const Tensor codes = fresh({e, n, to}, at::kFloat8_e4m3fn, w), scales = fresh({e, (n + 127) / 128, (k + 127) / 128}, at::kFloat, w);
  // strides of dimensions of size 1 say nothing
  FS_CALL(fs_weights8, w.data_ptr(), type_of(w), w.stride(0), std::max(w.stride(1), k), (int)e, (int)n, (int)k, static_cast<uint8_t*>(codes.data_ptr()), n * to,
          to, floats(scales), at.stream);
  return {codes.narrow(2, 0, k), scales};
}
// `codes [E, N, K]` as tensor loads take them; themselves, or a copy with padded rows.
Tensor loadable_codes(const Tensor& c) {
  const int64_t e = c.size(0), n = c.size(1), k = c.size(2), to = (k + 15) / 16 * 16;
  if (aligned16(c) && c.stride(2) == 1 && c.stride(1) % 16 == 0 && c.stride(1) >= k && c.stride(0) % 16 == 0 && (c.stride(0) > 0 || e == 1)) return c;
  const Place at(c);
  const Tensor out = fresh({e, n, to}, c).narrow(2, 0, k);
  out.copy_(c);
  return out;
}
// x in order (rows undefined) or x[rows], times the weights or their transposes.
Tensor mm8_raw(const Tensor& x, const Tensor& rows, int64_t count, const Tensor& codes0, const Tensor& scales, const Tensor& offsets, bool transposed,
               bool fp32) {
  const Place at(x);
  const Tensor codes = loadable_codes(codes0);
  const int64_t n = codes.size(transposed ? 2 : 1), k = codes.size(transposed ? 1 : 2);
  const size_t bytes = lib.fs_grouped_mm8_bytes((int)count, (int)k, transposed);
  Tensor out = fresh({count, n}, fp32 ? at::kFloat : x.scalar_type(), x), ws;
  if (bytes) ws = fresh({(int64_t)bytes}, at::kByte, x);
  FS_CALL(fs_grouped_mm8, data(x), type_of(x), ld(x), (int)x.size(0), ints(rows), (int)count,
          static_cast<const uint8_t*>(codes.data_ptr()), codes.stride(0), codes.stride(1), floats(scales), (int)codes.size(0), (int)n, (int)k, transposed,
          ints(offsets), data(out), type_of(out), n, data(ws), bytes, at.stream);
  return out;
}

// ------------------------------------------------------------------ autograd
struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits0, int64_t k, const optional<Tensor>& bias0, const optional<Tensor>& mask0,
                               bool over_all) {
    const Tensor bias = none(bias0), mask = none(mask0), logits = rows_of(logits0);
    auto out = route_raw(logits, k, bias, mask, over_all);
    ctx->save_for_backward({logits, bias, mask, out[0], out[1]});
    ctx->saved_data["all"] = over_all;
    ctx->mark_non_differentiable({out[1], out[2], out[3], out[4], out[5]});
    ctx->set_materialize_grads(false);  // five zero gradients of whole numbers
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &logits = s[0], &gates = s[3];
    const bool over_all = ctx->saved_data["all"].toBool();
    const Place at(logits);
    Tensor out;
    if (grads[0].defined()) {
      const Tensor grad = grads[0].contiguous();
      out = fresh(logits.sizes(), logits);
      FS_CALL(fs_route_grad, logits.data_ptr(), type_of(logits), ld(logits), (int)logits.size(0), (int)logits.size(1), (int)gates.size(1),
              floats(s[1]), static_cast<const uint8_t*>(data(s[2])), over_all, floats(gates), ints(s[4]), floats(grad), out.data_ptr(), at.stream);
    }
    return once({out, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct GroupedMm : torch::autograd::Function<GroupedMm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const Tensor& w0, const Tensor& offsets, const optional<Tensor>& rows0,
                        const optional<Tensor>& position, int64_t count) {
    const Tensor rows = none(rows0), w = loadable_weights(w0);
    const Tensor x = rows.defined() ? rows_of(x0) : loadable_rows(x0);  // whatever reads gathered rows again copies them into order
    ctx->save_for_backward({x, w, offsets, rows, none(position)});
    return mm_raw(x, rows, count, w, offsets, false, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &offsets = s[2], &rows = s[3], &position = s[4];
    Tensor dx, dw;
    if (grads[0].defined()) {
      const Place at(x);
      const Tensor dy = loadable_rows(grads[0]);
      if (ctx->needs_input_grad(0)) {
        // of gathered rows in fp32, so that the sum over a token's rows is rounded once
        dx = mm_raw(dy, Tensor(), dy.size(0), w, offsets, true, rows.defined());
        if (rows.defined()) dx = combine_raw(dx, Tensor(), position, x.scalar_type());
      }
      // a copy of the rows in order costs less than fetching them one by one for every tile of the product
      if (ctx->needs_input_grad(1)) dw = wgrad_raw(dy, rows.defined() ? gather_raw(x, rows) : x, offsets);
    }
    return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct GatedAct : torch::autograd::Function<GatedAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& u0, const optional<Tensor>& gates0, const optional<Tensor>& pairs0,
                        const optional<Tensor>& position, bool checkpoint) {
    const Tensor u = rows_of(u0), gates = none(gates0), pairs = none(pairs0);
    auto [h, held] = act_raw(u, gates, pairs, checkpoint);
    ctx->save_for_backward({checkpoint ? Tensor() : u, held, gates, pairs, none(position)});
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    Tensor du, dgates;
    if (grads[0].defined())
      std::tie(du, dgates, std::ignore) = act_grad_raw(s[0], s[1], s[2], s[3], s[4], rows_of(grads[0]), s[2].defined() && ctx->needs_input_grad(1), false);
    return once({ctx->needs_input_grad(0) ? du : Tensor(), dgates, Tensor(), Tensor(), Tensor()});
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& o0, const optional<Tensor>& gates0, const Tensor& position, const Tensor& pairs) {
    const Tensor o = rows_of(o0), gates = none(gates0);
    const bool keep = gates.defined() && gates.requires_grad();
    ctx->save_for_backward({keep ? o : Tensor(), gates, position, pairs});
    return combine_raw(o, gates, position, o.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &o = s[0], &gates = s[1], &position = s[2];
    Tensor d_o, dgates;
    if (grads[0].defined()) {
      const Place at(position);
      const Tensor dy = rows_of(grads[0]);
      const int64_t t = position.size(0), k = position.size(1), d = dy.size(1);
      d_o = fresh({t * k, d}, dy);
      if (o.defined()) dgates = fresh(gates.sizes(), gates);
      FS_CALL(fs_combine_grad, data(o), type_of(dy), ld(o), (int)t, (int)k, (int)d, floats(gates), ints(position), ints(s[3]), dy.data_ptr(), ld(dy),
              d_o.data_ptr(), floats(dgates), at.stream);
    }
    return once({ctx->needs_input_grad(0) ? d_o : Tensor(), dgates, Tensor(), Tensor()});
  }
};

// Keeps x, the routing and u (in 8 bits) from the forward pass. The gates are in the activation, so the backward pass needs
// neither the experts' outputs nor their gradients: both of its products with the outer weights read dy.
struct Mlp : torch::autograd::Function<Mlp> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const Tensor& w_in0, const Tensor& w_out0, const Tensor& gates, const Tensor& offsets,
                        const Tensor& pairs, const Tensor& rows, const Tensor& position, bool checkpoint) {
    const Tensor x = rows_of(x0), w_in = loadable_weights(w_in0), w_out = loadable_weights(w_out0);
    const int64_t count = pairs.size(0);
    const Tensor u = mm_raw(x, rows, count, w_in, offsets, false, false);
    auto [h, held] = act_raw(u, gates, pairs, checkpoint);
    ctx->save_for_backward({x, w_in, w_out, gates, offsets, pairs, rows, position, checkpoint ? Tensor() : u, held});
    return combine_raw(mm_raw(h, Tensor(), count, w_out, offsets, false, false), Tensor(), position, x.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w_in = s[1], &w_out = s[2], &gates = s[3], &offsets = s[4], &pairs = s[5], &rows = s[6], &position = s[7];
    Tensor dx, dw_in, dw_out, dgates;
    if (grads[0].defined()) {
      const int64_t count = pairs.size(0);
      const Tensor dy = gather_raw(grads[0], rows);  // for two products
      const Tensor dh = mm_raw(dy, Tensor(), count, w_out, offsets, true, false);
      Tensor du, h;
      std::tie(du, dgates, h) = act_grad_raw(s[8], s[9], gates, pairs, position, dh, ctx->needs_input_grad(3), ctx->needs_input_grad(2));
      if (ctx->needs_input_grad(0))  // rows in fp32, so that the sum over a token's rows is rounded once
        dx = combine_raw(mm_raw(du, Tensor(), count, w_in, offsets, true, true), Tensor(), position, x.scalar_type());
      if (ctx->needs_input_grad(1)) dw_in = wgrad_raw(du, gather_raw(x, rows), offsets);
      if (ctx->needs_input_grad(2)) dw_out = wgrad_raw(dy, h, offsets);
    }
    return once({dx, dw_in, dw_out, dgates, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const optional<Tensor>& w0, const optional<Tensor>& b0, double eps) {
    const Tensor x = as_rows(x0), w = none(w0), b = none(b0);
    const Norm n = norm_raw(x, w, b, eps, true);
    ctx->save_for_backward({x, w, n.mean, n.rstd});
    ctx->saved_data["type"] = type_of(w.defined() ? w : b.defined() ? b : x);
    ctx->saved_data["bias"] = b.defined();
    return n.y.view(x0.sizes());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1];
    Tensor dx, dw, db;
    if (grads[0].defined()) {
      const Place at(x);
      const Tensor dy = as_rows(grads[0]);
      const int64_t r = x.size(0), f = x.size(1), w_type = ctx->saved_data["type"].toInt();
      const auto like = w_type == FS_TYPE_F32 ? at::kFloat : w_type == FS_TYPE_F16 ? at::kHalf : at::kBFloat16;
      if (ctx->needs_input_grad(0)) dx = fresh(x.sizes(), x);
      size_t input = 1;  // of those that are there
      if (w.defined() && ctx->needs_input_grad(input++)) dw = fresh({f}, like, x);
      if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(input)) db = fresh({f}, like, x);
      Tensor ws;
      const size_t bytes = dw.defined() || db.defined() ? lib.fs_layer_norm_grad_bytes((int)r, (int)f) : 0;
      if (bytes) ws = fresh({(int64_t)bytes}, at::kByte, x);
      FS_CALL(fs_layer_norm_grad, data(x), type_of(x), ld(x), (int)r, (int)f, data(w), (int)w_type, floats(s[2]), floats(s[3]), data(dy), ld(dy), data(dx),
              data(dw), data(db), data(ws), bytes, at.stream);
      if (dx.defined()) dx = dx.view(grads[0].sizes());
    }
    return once({dx, dw, db, Tensor()});
  }
};

// The gradient to x goes through the same codes of the weights, that to 16-bit weights is of the rows as they were.
struct GroupedMm8 : torch::autograd::Function<GroupedMm8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x0, const optional<Tensor>& w, const optional<Tensor>& codes0, const optional<Tensor>& scales0,
                        const Tensor& offsets, const optional<Tensor>& rows0, const optional<Tensor>& position0, int64_t count) {
    const Tensor x = rows_of(x0), rows = none(rows0), position = none(position0);
    Tensor codes = none(codes0), scales = none(scales0);
    if (w.has_value()) std::tie(codes, scales) = weights8_raw(*w);
    const bool grad_x = x0.requires_grad(), grad_w = w.has_value() && w->requires_grad();
    ctx->save_for_backward({grad_w ? x : Tensor(), grad_x ? codes : Tensor(), grad_x ? scales : Tensor(), offsets, rows, position});
    return mm8_raw(x, rows, count, codes, scales, offsets, false, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &codes = s[1], &offsets = s[3], &rows = s[4], &position = s[5];
    Tensor dx, dw;
    if (grads[0].defined()) {
      const Tensor dy = rows_of(grads[0]);
      if (ctx->needs_input_grad(0)) {
        // of gathered rows in fp32, so that the sum over a token's rows is rounded once
        dx = mm8_raw(dy, Tensor(), dy.size(0), codes, s[2], offsets, true, rows.defined());
        if (rows.defined()) dx = combine_raw(dx, Tensor(), position, dy.scalar_type());
      }
      if (ctx->needs_input_grad(1)) dw = wgrad_raw(dy, rows.defined() ? gather_raw(x, rows) : x, offsets);
    }
    return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// ------------------------------------------------------------------ public calls
std::vector<Tensor> route_tokens(const Tensor& logits0, int64_t k, const optional<Tensor>& bias0, const optional<Tensor>& mask0, bool over_all) {
  REQUIRE(logits0.dim() == 2, "logits must be 2D [T, E], got shape ", shape_of(logits0));
  check_type("logits", logits0, true);
  check_cuda("logits", logits0);
  const int64_t t = logits0.size(0), e = logits0.size(1);
  REQUIRE(e >= 1 && e <= kMaxExperts, "the number of experts must be between 1 and ", kMaxExperts, ", got ", e);
  REQUIRE(k >= 1 && k <= std::min(e, kMaxK), "k must be between 1 and ", std::min(e, kMaxK), ", got ", k);
  REQUIRE(t * k < (int64_t(1) << 31), "T * k must be below 2^31");
  Tensor bias = none(bias0), mask = none(mask0);
  if (bias.defined()) {
    check_place("bias", bias, "logits", logits0);
    REQUIRE(bias.dim() == 1 && bias.size(0) == e, "bias must have shape (", e, ",), got ", shape_of(bias));
    REQUIRE(!bias.requires_grad(), "bias must not require grad (it only takes part in the choice)");
    bias = bias.to(at::kFloat).contiguous();
  }
  if (mask.defined()) {
    check_place("mask", mask, "logits", logits0);
    REQUIRE(mask.dim() == 1 && mask.size(0) == t && mask.scalar_type() == at::kBool, "mask must be a bool tensor of shape (", t, ",), got ",
                      type_name(mask), " ", shape_of(mask));
    mask = mask.contiguous();
  }
  if (wants_grad({&logits0})) return Route::apply(logits0, k, maybe(bias), maybe(mask), over_all);
  return route_raw(rows_of(logits0), k, bias, mask, over_all);
}

Tensor grouped_mm(const Tensor& x0, const Tensor& w0, const Tensor& offsets, const optional<Tensor>& rows0, const optional<Tensor>& position0,
                  bool gather) {
  REQUIRE(x0.dim() == 2 && w0.dim() == 3, "x must be 2D and weight 3D [E, N, K], got shapes ", shape_of(x0), " and ", shape_of(w0));
  check_type("x", x0, false);
  REQUIRE(w0.scalar_type() == x0.scalar_type(), "weight must be of the type of x (", type_name(x0), "), got ", type_name(w0));
  check_cuda("x", x0);
  check_place("weight", w0, "x", x0);
  const int64_t e = w0.size(0), n = w0.size(1), k = w0.size(2);
  REQUIRE(x0.size(1) == k && k > 0 && n > 0, "x must have as many columns as weight (", k, " > 0), got ", x0.size(1),
                    "; N must be > 0, got ", n);
  check_offsets(offsets, x0);
  int64_t count = x0.size(0);
  Tensor rows, position = none(position0);
  if (position.defined()) {  // of a routing
    check_position(position, x0);
    count = position.numel();
    if (gather) {
      rows = none(rows0);
      check_field("rows", rows, position, true, at::kInt, x0);
    } else {
      position = Tensor();
    }
    const int64_t want = gather ? position.size(0) : count;
    REQUIRE(x0.size(0) == want, "x must have ", want, " rows, got ", x0.size(0));
  }
  REQUIRE(!gather || position.size(1) <= kMaxK, "k must be at most ", kMaxK);
  REQUIRE(offsets.size(0) == e + 1 && e <= kMaxExperts, "groups must have as many experts as weight (", e, ", at most ", kMaxExperts,
                    "), got ", offsets.size(0) - 1);
  REQUIRE(count <= kMaxRows && x0.size(0) <= kMaxRows, "rows must be at most 2^31 - 512");
  if (!wants_grad({&x0, &w0})) return mm_raw(x0, rows, count, w0, offsets, false, false);
  return GroupedMm::apply(x0, w0, offsets, maybe(rows), maybe(position), count);
}

Tensor gated_act(const Tensor& u0, const optional<Tensor>& gates0, const optional<Tensor>& pairs0, const optional<Tensor>& position0, bool checkpoint) {
  REQUIRE(u0.dim() == 2 && u0.size(1) > 0 && u0.size(1) % 2 == 0, "u must be 2D [R, 2 F] with F > 0, got shape ", shape_of(u0));
  check_type("u", u0, true);
  check_cuda("u", u0);
  const Tensor gates = none(gates0), pairs = none(pairs0), position = none(position0);
  if (position.defined()) {
    check_position(position, u0);
    check_field("gates", gates, position, false, at::kFloat, u0);
    check_field("pairs", pairs, position, true, at::kInt, u0);
    REQUIRE(u0.size(0) == pairs.size(0), "u must have ", pairs.size(0), " rows, got ", u0.size(0));
  }
  REQUIRE(u0.size(0) < (int64_t(1) << 31), "rows must be fewer than 2^31");
  if (!wants_grad({&u0, &gates})) return act_raw(rows_of(u0), gates, pairs, false).first;
  return GatedAct::apply(u0, maybe(gates), maybe(pairs), maybe(position), checkpoint);
}

Tensor combine_rows(const Tensor& o0, const Tensor& gates0, const Tensor& pairs, const Tensor& position, bool weighted) {
  REQUIRE(o0.dim() == 2 && o0.size(1) > 0, "o must be 2D [T * k, D] with D > 0, got shape ", shape_of(o0));
  check_type("o", o0, true);
  check_cuda("o", o0);
  check_position(position, o0);
  check_field("gates", gates0, position, false, at::kFloat, o0);
  check_field("pairs", pairs, position, true, at::kInt, o0);
  REQUIRE(o0.size(0) == pairs.size(0), "o must have ", pairs.size(0), " rows, got ", o0.size(0));
  REQUIRE(position.size(1) <= kMaxK, "k must be at most ", kMaxK, ", got ", position.size(1));
  REQUIRE(o0.size(0) < (int64_t(1) << 31), "rows must be fewer than 2^31");
  const Tensor gates = weighted ? gates0 : Tensor();
  if (wants_grad({&o0, &gates})) return Combine::apply(o0, maybe(gates), position, pairs);
  return combine_raw(rows_of(o0), gates, position, o0.scalar_type());
}

Tensor expert_mlp(const Tensor& x0, const Tensor& w_in0, const Tensor& w_out0, const Tensor& gates, const Tensor& offsets, const Tensor& pairs,
                  const Tensor& rows, const Tensor& position, bool checkpoint) {
  REQUIRE(x0.dim() == 2 && w_in0.dim() == 3 && w_out0.dim() == 3, "x must be 2D, w_in and w_out 3D");
  check_type("x", x0, false);
  REQUIRE(w_in0.scalar_type() == x0.scalar_type() && w_out0.scalar_type() == x0.scalar_type(), "w_in and w_out must be of the type of x (",
                    type_name(x0), "), got ", type_name(w_in0), " and ", type_name(w_out0));
  check_cuda("x", x0);
  check_place("w_in", w_in0, "x", x0);
  check_place("w_out", w_out0, "x", x0);
  check_position(position, x0);
  check_field("gates", gates, position, false, at::kFloat, x0);
  check_field("pairs", pairs, position, true, at::kInt, x0);
  check_field("rows", rows, position, true, at::kInt, x0);
  check_offsets(offsets, x0);
  const int64_t t = x0.size(0), d = x0.size(1), e = w_in0.size(0), f = w_out0.size(2);
  REQUIRE(w_in0.size(1) == 2 * f && w_in0.size(2) == d && w_out0.size(0) == e && w_out0.size(1) == d && d > 0 && f > 0,
                    "w_in must be [E, 2 F, ", d, "] and w_out [E, ", d, ", F], got ", shape_of(w_in0), " and ", shape_of(w_out0));
  REQUIRE(position.size(0) == t && offsets.size(0) == e + 1 && position.size(1) <= kMaxK && e <= kMaxExperts && position.numel() <= kMaxRows,
                    "routing must be of ", t, " tokens and ", e, " experts (at most ", kMaxExperts, "), at most ", kMaxK, " for a token and 2^31 - 512 in all");
  if (wants_grad({&x0, &w_in0, &w_out0, &gates})) return Mlp::apply(x0, w_in0, w_out0, gates, offsets, pairs, rows, position, checkpoint);
  const int64_t count = pairs.size(0);
  const Tensor h = act_raw(mm_raw(x0, rows, count, w_in0, offsets, false, false), gates, pairs, false).first;
  return combine_raw(mm_raw(h, Tensor(), count, w_out0, offsets, false, false), Tensor(), position, x0.scalar_type());
}

Tensor layer_norm(const Tensor& x, const optional<Tensor>& w0, const optional<Tensor>& b0, double eps) {
  REQUIRE(x.dim() >= 1 && x.size(-1) > 0, "x must be [..., F] with F > 0, got shape ", shape_of(x));
  check_type("x", x, true);
  check_cuda("x", x);
  const Tensor w = none(w0), b = none(b0);
  const int64_t f = x.size(-1);
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"weight", w}, {"bias", b}}) {
    if (!t.defined()) continue;
    check_place(name, t, "x", x);
    REQUIRE(t.dim() == 1 && t.size(0) == f, name, " must have shape (", f, ",), got ", shape_of(t));
    REQUIRE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, name, " must be float32 or of the type of x (", type_name(x), "), got ",
            type_name(t));
  }
  REQUIRE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight and bias must be of one type");
  REQUIRE(eps >= 0 && eps < 3e38, "eps must not be negative");
  REQUIRE(f <= (1 << 24) && x.numel() / f < (int64_t(1) << 31), "F must be at most 2^24, rows fewer than 2^31");
  const Tensor wc = w.defined() ? w.contiguous() : w, bc = b.defined() ? b.contiguous() : b;
  if (wants_grad({&x, &w, &b})) return LayerNorm::apply(x, maybe(wc), maybe(bc), eps);
  return norm_raw(as_rows(x), wc, bc, eps, false).y.view(x.sizes());
}

std::pair<Tensor, Tensor> to_blocks8(const Tensor& w) {
  REQUIRE(w.dim() == 3 && w.size(0) > 0 && w.size(1) > 0 && w.size(2) > 0, "weight must be 3D [E, N, K] and not empty, got shape ", shape_of(w));
  check_type("weight", w, false);
  check_cuda("weight", w);
  check_tangent("weight", w);
  REQUIRE(w.size(0) <= kMaxExperts && w.size(1) <= (1 << 22) && w.size(2) <= (1 << 22), "weight must have at most ", kMaxExperts,
          " experts, N and K be at most 2^22");
  return weights8_raw(w);
}

Tensor grouped_mm8(const Tensor& x0, const optional<Tensor>& w0, const optional<Tensor>& codes0, const optional<Tensor>& scales0, const Tensor& offsets,
                   const optional<Tensor>& rows0, const optional<Tensor>& position0, bool gather) {
  const Tensor w16 = none(w0), codes = none(codes0), scales = none(scales0);
  const Tensor& w = w16.defined() ? w16 : codes;
  REQUIRE(x0.dim() == 2 && w.dim() == 3, "x must be 2D and weight 3D [E, N, K], got shapes ", shape_of(x0), " and ", shape_of(w));
  check_type("x", x0, false);
  const int64_t e = w.size(0), n = w.size(1), k = w.size(2);
  if (w16.defined()) {
    REQUIRE(w.scalar_type() == x0.scalar_type(), "weight must be of the type of x (", type_name(x0), ") or a Blocks8, got ", type_name(w));
  } else {
    REQUIRE(w.scalar_type() == at::kFloat8_e4m3fn, "codes must be of type float8_e4m3fn, got ", type_name(w));
    REQUIRE(scales.scalar_type() == at::kFloat && scales.is_contiguous() && scales.dim() == 3 && scales.size(0) == e && scales.size(1) == (n + 127) / 128 &&
                scales.size(2) == (k + 127) / 128,
            "scales must be a contiguous float32 tensor of shape (E, ceil(N / 128), ceil(K / 128)) for codes ", shape_of(w), ", got ", type_name(scales), " ",
            shape_of(scales));
    REQUIRE(!scales.requires_grad() && !w.requires_grad(), "codes and scales must not require grad");
    check_tangent("scales", scales);
  }
  check_cuda("x", x0);
  check_place("weight", w, "x", x0);
  if (scales.defined()) check_place("scales", scales, "x", x0);
  REQUIRE(x0.size(1) == k && k > 0 && n > 0, "x must have as many columns as weight (", k, " > 0), got ", x0.size(1), "; N must be > 0, got ", n);
  REQUIRE(n <= (1 << 22) && k <= (1 << 22), "N and K must be at most 2^22");
  check_offsets(offsets, x0);
  int64_t count = x0.size(0);
  Tensor rows, position = none(position0);
  if (position.defined()) {  // of a routing
    check_position(position, x0);
    count = position.numel();
    if (gather) {
      rows = none(rows0);
      check_field("rows", rows, position, true, at::kInt, x0);
    } else {
      position = Tensor();
    }
    const int64_t want = gather ? position.size(0) : count;
    REQUIRE(x0.size(0) == want, "x must have ", want, " rows, got ", x0.size(0));
  }
  REQUIRE(!gather || position.size(1) <= kMaxK, "k must be at most ", kMaxK);
  REQUIRE(offsets.size(0) == e + 1 && e <= kMaxExperts, "groups must have as many experts as weight (", e, ", at most ", kMaxExperts, "), got ",
          offsets.size(0) - 1);
  REQUIRE(count <= kMaxRows && x0.size(0) <= kMaxRows, "rows must be at most 2^31 - 512");
  if (wants_grad({&x0, &w16})) return GroupedMm8::apply(x0, maybe(w16), maybe(codes), maybe(scales), offsets, maybe(rows), maybe(position), count);
  if (!w16.defined()) return mm8_raw(rows_of(x0), rows, count, codes, scales, offsets, false, false);
  const auto [c, s] = weights8_raw(w16);
  return mm8_raw(rows_of(x0), rows, count, c, s, offsets, false, false);
}

Tensor orthogonalize(const Tensor& g0, int64_t steps, double a, double b, double c, double eps, bool bf16) {
  REQUIRE(g0.dim() >= 2 && g0.size(-1) > 0 && g0.size(-2) > 0, "g must be [..., N, K] with N, K > 0, got shape ", shape_of(g0));
  check_type("g", g0, true);
  check_cuda("g", g0);
  const int64_t n = g0.size(-2), k = g0.size(-1), batch = g0.numel() / (n * k);
  check_tangent("g", g0);
  REQUIRE(n <= 65536 && k <= 65536, "N and K must be at most 65536, got ", n, " and ", k);
  REQUIRE(batch < (1 << 20), "a stack must have fewer than 2^20 matrices");
  REQUIRE(steps >= 1 && steps <= 64, "steps must be between 1 and 64, got ", steps);
  REQUIRE(std::abs(a) <= 16 && std::abs(b) + std::abs(c) <= 32, "coefficients must be at most 16, and the last two together at most 32, in magnitude");
  REQUIRE(eps >= 1e-30 && eps < 3e38, "eps must be positive (1e-30 at least)");
  Tensor g = g0.dim() == 3 ? g0 : g0.reshape({batch, n, k});
  if (g.stride(2) != 1 || g.stride(1) < k || g.stride(0) < 0) g = g.contiguous();
  const Place at(g);
  const Tensor out = fresh(g0.sizes(), bf16 ? at::kBFloat16 : at::kHalf, g);
  const size_t bytes = lib.fs_orthogonalize_bytes((int)batch, (int)n, (int)k);
  const Tensor ws = fresh({(int64_t)bytes}, at::kByte, g);
  FS_CALL(fs_orthogonalize, data(g), type_of(g), g.stride(0), std::max(g.stride(1), k), (int)batch, (int)n, (int)k, (int)steps, (float)a, (float)b, (float)c,
          (float)eps, data(out), type_of(out), data(ws), bytes, at.stream);
  return out;
}

}  // namespace

namespace py = pybind11;

PYBIND11_MODULE(fs_torch, m) {
  // addresses: entry point name -> address in the loaded library; error: the exception of a failed call
  m.def("attach", [](const py::dict& addresses, py::object error) {
#define FS_TAKE(name) lib.name = reinterpret_cast<decltype(lib.name)>(addresses[#name].cast<uintptr_t>());
    FS_ENTRIES(FS_TAKE)
#undef FS_TAKE
    static PyObject* raised = nullptr;
    raised = error.release().ptr();
    py::register_exception_translator([](std::exception_ptr p) {
      try {
        if (p) std::rethrow_exception(p);
      } catch (const CallFailed& e) {
        PyErr_SetString(raised, e.what());
      } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
      } catch (const c10::Error&) {  // as torch's own calls raise it: ValueError, OutOfMemoryError, ...
        torch::translate_exception_to_python(std::current_exception());
      }
    });
  });
  m.def("entries", []() {
    std::vector<std::string> names;
#define FS_NAME(name) names.push_back(#name);
    FS_ENTRIES(FS_NAME)
#undef FS_NAME
    return names;
  });
  const auto no_gil = py::call_guard<py::gil_scoped_release>();
  m.def("route_tokens", &route_tokens, no_gil);
  m.def("grouped_mm", &grouped_mm, no_gil);
  m.def("gated_act", &gated_act, no_gil);
  m.def("combine_rows", &combine_rows, no_gil);
  m.def("expert_mlp", &expert_mlp, no_gil);
  m.def("layer_norm", &layer_norm, no_gil);
  m.def("to_blocks8", &to_blocks8, no_gil);
  m.def("grouped_mm8", &grouped_mm8, no_gil);
  m.def("orthogonalize", &orthogonalize, no_gil);
  // the kernels by themselves, without autograd
  m.def("mm", [](const Tensor& x, const optional<Tensor>& rows, int64_t count, const Tensor& w, const Tensor& offsets, bool transposed, bool fp32) {
    return mm_raw(x, none(rows), count, w, offsets, transposed, fp32);
  }, no_gil);
  m.def("wgrad", &wgrad_raw, no_gil);
  m.def("gather", &gather_raw, no_gil);
  m.def("act", [](const Tensor& u, const optional<Tensor>& gates, const optional<Tensor>& pairs, bool checkpoint) {
    auto [h, held] = act_raw(u, none(gates), none(pairs), checkpoint);
    return std::make_pair(h, checkpoint ? optional<Tensor>(held) : optional<Tensor>());
  }, no_gil);
  m.def("act_grad", [](const optional<Tensor>& u, const optional<Tensor>& held, const optional<Tensor>& gates, const optional<Tensor>& pairs,
                       const optional<Tensor>& position, const Tensor& dh, bool want_gates, bool want_h) {
    auto [du, dgates, h] = act_grad_raw(none(u), none(held), none(gates), none(pairs), none(position), dh, want_gates, want_h);
    return std::make_tuple(du, dgates.defined() ? optional<Tensor>(dgates) : optional<Tensor>(), h.defined() ? optional<Tensor>(h) : optional<Tensor>());
  }, no_gil);
}
