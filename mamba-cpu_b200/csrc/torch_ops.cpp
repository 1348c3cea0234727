// torch_ops.cpp -- torch binding of the gated linear recurrence and the norms (libmamba_b200_torch.so).
//
// The operators' dispatcher entries (namespace mamba_b200), written against the C ABI of
// libmamba_b200.so. They are bound in C++ rather than from Python because their calls are short: one
// decoded token, or the backward of a small norm, costs a few microseconds on the GPU, and a Python
// node in the autograd engine costs tens of them on the host.
//
//   *_fwd, *_bwd, *_update_   CUDA implementations: allocate the results, fill the parameter block, enqueue
//   gated_scan, gated_step,   what the public functions of mamba_cpu_b200.ops call: argument checks, casts,
//   norm, gated_norm          and the autograd nodes
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <tuple>

#include "mamba_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr auto kF32 = at::kFloat;

void check_status(int status, const char* what) {
  if (status == MB200_OK) return;
  const auto text = c10::str(what, ": ", mb200_status_string(status), " (status ", status, ")");
  switch (status) {
    case MB200_ERR_BAD_DTYPE: TORCH_CHECK_TYPE(false, text);
    case MB200_ERR_UNSUPPORTED: TORCH_CHECK_NOT_IMPLEMENTED(false, text);
    case MB200_ERR_WORKSPACE:
    case MB200_ERR_CUDA: TORCH_CHECK(false, text);
    default: TORCH_CHECK_VALUE(false, text);
  }
}

bool is_io(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

int code(at::ScalarType t) {
  TORCH_CHECK_TYPE(is_io(t), "mamba_b200: float32, bfloat16 or float16 expected, got ", t);
  return t == at::kFloat ? MB200_F32 : t == at::kBFloat16 ? MB200_BF16 : MB200_F16;
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

template <typename T = void>
T* ptr(const Tensor& t) { return static_cast<T*>(t.defined() ? t.data_ptr() : nullptr); }
template <typename T = void>
T* ptr(const OptTensor& t) { return t.has_value() ? ptr<T>(*t) : nullptr; }

// Straight from the caching allocator: half the time of at::empty, which counts where a call takes 8 us.
Tensor make(at::IntArrayRef sizes, const Tensor& like, at::ScalarType t) {
  return Tensor(at::detail::empty_cuda(sizes, t, like.device(), std::nullopt));
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// What the kernels read as float32 is cast on the way there: an imaginary part would be lost.
void want_real(const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.is_complex(), "complex ", name, " is not supported yet");
}

// The tensor whose type a result takes: results would be cut to integers.
void want_floating(const char* name, const Tensor& t) {
  want_real(name, t);
  TORCH_CHECK_TYPE(t.is_floating_point(), name, " must be of floating point, got ", t.scalar_type());
}

void want_shape(const char* name, const OptTensor& t, at::IntArrayRef shape, const Tensor& on, const char* on_name) {
  if (!given(t)) return;
  want_real(name, *t);
  TORCH_CHECK_VALUE(t->sizes() == shape, name, " must be ", shape, ", got ", t->sizes());
  TORCH_CHECK_VALUE(t->device() == on.device(), name, " must be on ", on_name, "'s device ", on.device(), ", got ",
                    t->device());
}

void want_cuda(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "mamba_cpu_b200 runs on CUDA tensors, got device ", t.device());
}

// The kernels get addresses: all of one device.
void want_device(std::initializer_list<const Tensor*> ts, std::initializer_list<const OptTensor*> more, const char* name) {
  const auto device = (*ts.begin())->device();
  for (const Tensor* t : ts) TORCH_CHECK_VALUE(t->device() == device, name, ": tensors must be on one device");
  for (const OptTensor* t : more)
    TORCH_CHECK_VALUE(!given(*t) || (*t)->device() == device, name, ": tensors must be on one device");
}

Tensor cast(const Tensor& t, at::ScalarType to) { return t.scalar_type() == to ? t : t.to(to); }
OptTensor dense(const OptTensor& t, at::ScalarType to) {
  return given(t) ? OptTensor(cast(*t, to).contiguous()) : std::nullopt;
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Nothing here has a forward-mode derivative. A tangent that the kernels passed over would come back as zero.
void no_tangents(std::initializer_list<const Tensor*> ts, std::initializer_list<const OptTensor*> more) {
  const auto check = [](const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "forward-mode derivatives are not supported by mamba_cpu_b200");
  };
  for (const Tensor* t : ts) check(*t);
  for (const OptTensor* t : more)
    if (t->has_value()) check(**t);
}
Tensor or_undefined(const OptTensor& t) { return given(t) ? *t : Tensor(); }

// ---- gated linear recurrence ----------------------------------------------------------------------

// (batch, dim, seqlen) rows the kernels read in place: contiguous along seqlen, no stride of 0
// (which the C ABI takes for the dense one).
bool rows_in_place(const Tensor& t) {
  return (t.size(2) <= 1 || t.stride(2) == 1) && (t.size(0) <= 1 || t.stride(0) > 0) &&
         (t.size(1) <= 1 || t.stride(1) > 0);
}

int64_t state_floats(const mb200_gated_scan_params& p) { return MB200_GATED_SCAN_STATES(p.batch, p.dim, p.seqlen); }

mb200_gated_scan_params scan_params(const Tensor& u, const Tensor& r, const Tensor& i, const Tensor& A,
                                    const OptTensor& h0, const OptTensor& ids) {
  want_device({&u, &r, &i, &A}, {&h0, &ids}, "mamba_b200::gated_scan");
  TORCH_CHECK_VALUE(u.dim() == 3, "mamba_b200::gated_scan: u must be (batch, dim, seqlen)");
  for (const Tensor* t : {&u, &r, &i})
    TORCH_CHECK_VALUE(t->scalar_type() == u.scalar_type() && t->sizes() == u.sizes() && rows_in_place(*t),
                      "mamba_b200::gated_scan: u and the gates must be alike, with contiguous rows");
  const int64_t b = u.size(0), d = u.size(1), l = u.size(2);
  const auto plain = [](const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
    return t.scalar_type() == type && t.sizes() == shape && t.is_contiguous();
  };
  TORCH_CHECK_VALUE(plain(A, kF32, {d}), "mamba_b200::gated_scan: A must be contiguous float32 (dim,)");
  TORCH_CHECK_VALUE(!given(h0) || plain(*h0, kF32, {b, d}),
                    "mamba_b200::gated_scan: initial_state must be contiguous float32 (batch, dim)");
  TORCH_CHECK_VALUE(!given(ids) || plain(*ids, at::kInt, {b, l}),
                    "mamba_b200::gated_scan: seq_idx must be contiguous int32 (batch, seqlen)");
  mb200_gated_scan_params p = {};
  p.u = ptr(u);
  p.decay_gate = ptr(r);
  p.input_gate = ptr(i);
  p.A = ptr<float>(A);
  p.initial_state = ptr<float>(h0);
  p.seq_idx = ptr<int32_t>(ids);
  p.batch = b;
  p.dim = d;
  p.seqlen = l;
  p.u_batch_stride = u.stride(0);
  p.u_dim_stride = u.stride(1);
  p.decay_gate_batch_stride = r.stride(0);
  p.decay_gate_dim_stride = r.stride(1);
  p.input_gate_batch_stride = i.stride(0);
  p.input_gate_dim_stride = i.stride(1);
  p.io_dtype = code(u.scalar_type());
  return p;
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_fwd(const Tensor& u, const Tensor& r, const Tensor& i, const Tensor& A,
                                                  const OptTensor& h0, const OptTensor& ids, bool save_states) {
  auto p = scan_params(u, r, i, A, h0, ids);
  const c10::cuda::CUDAGuard guard(u.device());
  Tensor out = make(u.sizes(), u, u.scalar_type());
  Tensor last = make({p.batch, p.dim}, u, kF32);
  Tensor states = make({save_states ? state_floats(p) : 0}, u, kF32);
  p.out = ptr(out);
  p.last_state = ptr<float>(last);
  p.chunk_states = save_states ? ptr<float>(states) : nullptr;
  check_status(mb200_gated_scan_fwd(&p, stream_of(u)), "mamba_b200::gated_scan_fwd");
  return {out, last, states};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_scan_bwd(const Tensor& u, const Tensor& r, const Tensor& i,
                                                                  const Tensor& A, const OptTensor& h0,
                                                                  const OptTensor& ids, const Tensor& states,
                                                                  const Tensor& dout, const OptTensor& dlast) {
  mb200_gated_scan_bwd_params p = {};
  p.fwd = scan_params(u, r, i, A, h0, ids);
  const int64_t b = p.fwd.batch, d = p.fwd.dim;
  want_device({&u, &states, &dout}, {&dlast}, "mamba_b200::gated_scan_bwd");
  TORCH_CHECK_VALUE(dout.sizes() == u.sizes() && dout.scalar_type() == u.scalar_type() && dout.is_contiguous(),
                    "mamba_b200::gated_scan_bwd: dout must be contiguous with u's shape and dtype");
  TORCH_CHECK_VALUE(!given(dlast) || (dlast->scalar_type() == kF32 && dlast->sizes() == at::IntArrayRef({b, d}) &&
                                      dlast->is_contiguous()),
                    "mamba_b200::gated_scan_bwd: dlast_state must be contiguous float32 (batch, dim)");
  TORCH_CHECK_VALUE(states.scalar_type() == kF32 && states.is_contiguous() &&
                        states.sizes() == at::IntArrayRef({state_floats(p.fwd)}),
                    "mamba_b200::gated_scan_bwd: chunk_states must come from gated_scan_fwd(save_states=True)");
  const c10::cuda::CUDAGuard guard(u.device());
  const auto io = u.scalar_type();
  Tensor du = make(u.sizes(), u, io), dr = make(u.sizes(), u, io), di = make(u.sizes(), u, io);
  Tensor dA = make({d}, u, kF32), dh0;
  dh0 = given(h0) ? make({b, d}, u, kF32) : make({0}, u, kF32);
  p.fwd.chunk_states = ptr<float>(states);
  p.dout = ptr(dout);
  p.dlast_state = ptr<float>(dlast);
  p.du = ptr(du);
  p.ddecay_gate = ptr(dr);
  p.dinput_gate = ptr(di);
  p.dA = ptr<float>(dA);
  p.dinitial_state = given(h0) ? ptr<float>(dh0) : nullptr;
  const auto bytes = static_cast<int64_t>(mb200_gated_scan_bwd_workspace_size(&p));
  Tensor ws = bytes > 0 ? make({bytes}, u, at::kByte) : Tensor();
  check_status(mb200_gated_scan_bwd(&p, ptr(ws), bytes, stream_of(u)), "mamba_b200::gated_scan_bwd");
  return {du, dr, di, dA, dh0};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& r, const Tensor& i, const Tensor& A,
                               const OptTensor& h0, const OptTensor& ids) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_b200::gated_scan_fwd", "")
                         .typed<decltype(gated_scan_fwd)>();
    auto [out, last, states] = op.call(u, r, i, A, h0, ids, true);
    ctx->save_for_backward({u, r, i, A, or_undefined(h0), or_undefined(ids), states});
    ctx->set_materialize_grads(false);
    return {out, last};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(6);
    if (!grads[0].defined() && !grads[1].defined()) return none;
    const auto s = ctx->get_saved_variables();
    const auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_b200::gated_scan_bwd", "")
                         .typed<decltype(gated_scan_bwd)>();
    const Tensor dout = grads[0].defined() ? grads[0].contiguous() : at::zeros(s[0].sizes(), s[0].options());
    const OptTensor dlast = grads[1].defined() ? OptTensor(grads[1].contiguous()) : std::nullopt;
    auto [du, dr, di, dA, dh0] = op.call(s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]), s[6], dout, dlast);
    return {du, dr, di, dA, s[4].defined() ? dh0 : Tensor(), Tensor()};
  }
};

Tensor as_rows(const Tensor& t, at::ScalarType io) {
  const Tensor c = cast(t, io);
  return rows_in_place(c) ? c : c.contiguous();
}

at::ScalarType common_io(const Tensor& u, const Tensor& r, const Tensor& i) {
  const auto t = u.scalar_type();
  return is_io(t) && r.scalar_type() == t && i.scalar_type() == t ? t : kF32;
}

std::tuple<Tensor, Tensor> gated_scan(const Tensor& u, const Tensor& decay_gate, const Tensor& input_gate,
                                      const Tensor& A, const OptTensor& initial_state, const OptTensor& seq_idx) {
  want_cuda(u);
  want_floating("u", u);
  TORCH_CHECK_VALUE(u.dim() == 3, "u must be (batch, dim, seqlen), got ", u.sizes());
  const int64_t b = u.size(0), d = u.size(1), l = u.size(2);
  want_shape("decay_gate", decay_gate, u.sizes(), u, "u");
  want_shape("input_gate", input_gate, u.sizes(), u, "u");
  want_shape("A", A, {d}, u, "u");
  want_shape("initial_state", initial_state, {b, d}, u, "u");
  want_shape("seq_idx", seq_idx, {b, l}, u, "u");
  no_tangents({&u, &decay_gate, &input_gate, &A}, {&initial_state});
  TORCH_CHECK_TYPE(!given(seq_idx) || at::isIntegralType(seq_idx->scalar_type(), /*includeBool=*/false),
                   "seq_idx must hold integers, got ", seq_idx->scalar_type());
  const auto io = common_io(u, decay_gate, input_gate);
  const Tensor uk = as_rows(u, io), rk = as_rows(decay_gate, io), ik = as_rows(input_gate, io);
  const Tensor Ak = cast(A, kF32).contiguous();
  const OptTensor h0 = dense(initial_state, kF32), ids = dense(seq_idx, at::kInt);
  Tensor out, last;
  if (wants_grad({&uk, &rk, &ik, &Ak}) || (given(h0) && wants_grad({&*h0}))) {
    auto r = GatedScan::apply(uk, rk, ik, Ak, h0, ids);
    out = r[0], last = r[1];
  } else {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_b200::gated_scan_fwd", "")
                         .typed<decltype(gated_scan_fwd)>();
    std::tie(out, last, std::ignore) = op.call(uk, rk, ik, Ak, h0, ids, false);
  }
  return {cast(out, u.scalar_type()), last};
}

// Whether two tensors of rows (contiguous along the last dimension, a row stride along the first of two)
// share memory in another way than element by element.
bool overlap_in_part(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  struct Rows {
    int64_t at, width, pitch, end;
    explicit Rows(const Tensor& t) {
      const int64_t rows = t.dim() == 2 ? t.size(0) : 1, es = t.element_size();
      at = reinterpret_cast<int64_t>(t.data_ptr());
      width = t.size(-1) * es;
      pitch = rows > 1 ? t.stride(0) * es : 0;
      end = at + pitch * (rows - 1) + width;
    }
  };
  const Rows p(a), q(b);
  if (p.end <= q.at || q.end <= p.at) return false;
  if (p.pitch != q.pitch || p.pitch == 0) return p.at != q.at || p.pitch != q.pitch || p.width != q.width;
  const int64_t apart = ((q.at - p.at) % p.pitch + p.pitch) % p.pitch;  // q's rows within p's pitch
  if (apart >= p.width && apart + q.width <= p.pitch) return false;
  return p.at != q.at || p.width != q.width;
}

bool step_rows(const Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) > 0);
}

Tensor step(const Tensor& state, const Tensor& u, const Tensor& r, const Tensor& i, const Tensor& A,
            const Tensor& new_state) {
  want_device({&state, &u, &r, &i, &A, &new_state}, {}, "mamba_b200::gated_scan_update");
  for (const Tensor* t : {&state, &u, &r, &i, &new_state})
    TORCH_CHECK_VALUE(t->dim() == 2 && t->sizes() == u.sizes() && step_rows(*t),
                      "mamba_b200::gated_scan_update: (batch, dim) tensors with contiguous rows expected");
  TORCH_CHECK_VALUE(r.scalar_type() == u.scalar_type() && i.scalar_type() == u.scalar_type() &&
                        new_state.scalar_type() == state.scalar_type(),
                    "mamba_b200::gated_scan_update: u and the gates, and the states, must share a dtype");
  TORCH_CHECK_VALUE(A.scalar_type() == kF32 && A.dim() == 1 && A.size(0) == u.size(1) && A.is_contiguous(),
                    "mamba_b200::gated_scan_update: A must be contiguous float32 (dim,)");
  TORCH_CHECK_VALUE(!overlap_in_part(state, new_state), "out_state must not overlap state in part");
  for (const Tensor* t : {&u, &r, &i, &A})
    TORCH_CHECK_VALUE(!overlap_in_part(*t, new_state), "the state that is written must not overlap the inputs in part");
  const c10::cuda::CUDAGuard guard(u.device());
  new_state.unsafeGetTensorImpl()->bump_version();
  Tensor out = make(u.sizes(), u, u.scalar_type());
  const auto row = [](const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; };
  mb200_gated_step_params p = {};
  p.state = ptr(state);
  p.new_state = ptr(new_state);
  p.u = ptr(u);
  p.decay_gate = ptr(r);
  p.input_gate = ptr(i);
  p.A = ptr<float>(A);
  p.out = ptr(out);
  p.batch = u.size(0);
  p.dim = u.size(1);
  p.state_stride = row(state);
  p.new_state_stride = row(new_state);
  p.u_stride = row(u);
  p.decay_gate_stride = row(r);
  p.input_gate_stride = row(i);
  p.io_dtype = code(u.scalar_type());
  p.state_dtype = code(state.scalar_type());
  check_status(mb200_gated_scan_update(&p, stream_of(u)), "mamba_b200::gated_scan_update");
  return out;
}

Tensor gated_scan_update(Tensor& state, const Tensor& u, const Tensor& r, const Tensor& i, const Tensor& A) {
  return step(state, u, r, i, A, state);
}

Tensor gated_scan_update_out(const Tensor& state, const Tensor& u, const Tensor& r, const Tensor& i, const Tensor& A,
                             Tensor& new_state) {
  return step(state, u, r, i, A, new_state);
}

Tensor gated_step(Tensor state, const Tensor& u, const Tensor& decay_gate, const Tensor& input_gate, const Tensor& A,
                  OptTensor out_state) {
  want_cuda(u);
  want_floating("u", u);
  TORCH_CHECK_VALUE(u.dim() == 2, "u must be (batch, dim), got ", u.sizes());
  const int64_t b = u.size(0), d = u.size(1);
  want_shape("state", state, u.sizes(), u, "u");
  want_floating("state", state);
  want_shape("decay_gate", decay_gate, u.sizes(), u, "u");
  want_shape("input_gate", input_gate, u.sizes(), u, "u");
  want_shape("A", A, {d}, u, "u");
  want_shape("out_state", out_state, u.sizes(), u, "u");
  no_tangents({&state, &u, &decay_gate, &input_gate, &A}, {&out_state});
  const bool apart = given(out_state) && !out_state->is_same(state);
  Tensor target = apart ? *out_state : state;
  TORCH_CHECK_TYPE(target.scalar_type() == state.scalar_type(), "out_state must have state's dtype ",
                   state.scalar_type(), ", got ", target.scalar_type());
  TORCH_CHECK_VALUE(!(b > 1 && target.stride(0) == 0) && !(d > 1 && target.stride(1) == 0) &&
                        !(b > 1 && d > 1 && target.stride(1) == 1 && target.stride(0) < d),
                    "the rows of the state that is written must not share memory");
  const auto io = common_io(u, decay_gate, input_gate);
  const auto rows = [&](const Tensor& t) {
    const Tensor c = cast(t, io);
    return step_rows(c) ? c : c.contiguous();
  };
  const auto in_place = [&](const Tensor& t) {
    return (t.scalar_type() == kF32 || t.scalar_type() == io) && (d <= 1 || t.stride(1) == 1) &&
           (b <= 1 || t.stride(0) >= d);
  };
  const Tensor uk = rows(u), rk = rows(decay_gate), ik = rows(input_gate), Ak = cast(A, kF32).contiguous();
  Tensor out;
  if (!apart && in_place(state)) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_b200::gated_scan_update", "")
                         .typed<decltype(gated_scan_update)>();
    out = op.call(state, uk, rk, ik, Ak);
  } else {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("mamba_b200::gated_scan_update_out", "")
                         .typed<decltype(gated_scan_update_out)>();
    const Tensor src = in_place(state) ? state : state.to(kF32).contiguous();
    const bool direct = in_place(target) && target.scalar_type() == src.scalar_type();
    Tensor work = direct ? target : at::empty_like(src);
    out = op.call(src, uk, rk, ik, Ak, work);
    if (!direct) target.copy_(work);
  }
  return cast(out, u.scalar_type());
}

// ---- norms ------------------------------------------------------------------------------------------

// t as (rows, dim) with rows that the kernels read in place (contiguous, no row stride of 0), copied
// where that takes a copy.
Tensor as_matrix(const Tensor& t, int64_t dim) {
  Tensor m = t;
  if (t.dim() != 2) {
    int64_t rows = 1;
    for (int64_t k = 0; k + 1 < t.dim(); ++k) rows *= t.size(k);
    m = t.reshape({rows, dim});
  }
  return (dim <= 1 || m.stride(1) == 1) && (m.size(0) <= 1 || m.stride(0) > 0) ? m : m.contiguous();
}

int64_t row_stride(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : 0; }

mb200_norm_params norm_params(const Tensor& x, const OptTensor& z, const OptTensor& weight, const OptTensor& bias,
                              at::ScalarType io, at::ScalarType w_type, double eps, int64_t group, bool rms,
                              int64_t gate) {
  mb200_norm_params p = {};
  p.x = ptr(x);
  p.z = ptr(z);
  p.weight = ptr(weight);
  p.bias = ptr(bias);
  p.rows = x.size(0);
  p.dim = x.size(1);
  p.group_size = group;
  p.x_stride = row_stride(x);
  p.z_stride = given(z) ? row_stride(*z) : 0;
  p.eps = static_cast<float>(eps);
  p.io_dtype = code(io);
  p.residual_dtype = p.io_dtype;
  p.weight_dtype = code(w_type);
  p.rms = rms;
  p.gate = static_cast<int32_t>(gate);
  return p;
}

void want_columns(const OptTensor& t, const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(!given(t) || (t->dim() == 1 && t->size(0) == x.size(-1) && t->is_contiguous()), what,
                    ": weight and bias must be contiguous (dim,)");
}

std::tuple<Tensor, Tensor> norm_fwd(const Tensor& x, const OptTensor& residual, const OptTensor& z,
                                    const OptTensor& weight, const OptTensor& bias, double eps, int64_t group,
                                    bool rms, int64_t gate, bool want_sum) {
  constexpr const char* name = "mamba_b200::norm_fwd";
  want_device({&x}, {&residual, &z, &weight, &bias}, name);
  TORCH_CHECK_VALUE(x.dim() >= 1, name, ": x must have at least one dimension");
  const int64_t dim = x.size(-1);
  want_columns(weight, x, name);
  want_columns(bias, x, name);
  TORCH_CHECK_VALUE(!given(residual) || residual->sizes() == x.sizes(), name, ": residual must have x's shape");
  TORCH_CHECK_VALUE(!given(z) || (z->sizes() == x.sizes() && z->scalar_type() == x.scalar_type()), name,
                    ": z must have x's shape and dtype");
  TORCH_CHECK_VALUE(!given(weight) || !given(bias) || weight->scalar_type() == bias->scalar_type(), name,
                    ": weight and bias must share a dtype");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto io = x.scalar_type();
  const Tensor xm = as_matrix(x, dim);
  const OptTensor zm = given(z) ? OptTensor(as_matrix(*z, dim)) : std::nullopt;
  const auto w_type = given(weight) ? weight->scalar_type() : given(bias) ? bias->scalar_type() : kF32;
  auto p = norm_params(xm, zm, weight, bias, io, w_type, eps, group, rms, gate);
  Tensor out = make(x.sizes(), x, io), total, rm;
  if (given(residual)) {
    rm = as_matrix(*residual, dim);
    total = want_sum ? make(x.sizes(), x, rm.scalar_type()) : make({0}, x, rm.scalar_type());
    p.residual = ptr(rm);
    p.residual_dtype = code(rm.scalar_type());
    p.residual_stride = row_stride(rm);
    p.sum_out = want_sum ? ptr(total) : nullptr;
    // an empty residual has no address, and it is its address that says it is there: nothing to add anyway
  } else {
    total = make({0}, x, io);
  }
  p.out = ptr(out);
  check_status(mb200_norm_fwd(&p, stream_of(x)), name);
  return {out, total};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> norm_bwd(const Tensor& dout, const OptTensor& dsum,
                                                            const Tensor& rows, const OptTensor& z,
                                                            const OptTensor& weight,
                                                            std::optional<at::ScalarType> residual_type,
                                                            std::optional<at::ScalarType> bias_type, double eps,
                                                            int64_t group, bool rms, int64_t gate,
                                                            bool want_dresidual, bool want_dweight) {
  constexpr const char* name = "mamba_b200::norm_bwd";
  const auto io = dout.scalar_type();
  want_device({&dout, &rows}, {&dsum, &z, &weight}, name);
  TORCH_CHECK_VALUE(dout.dim() >= 1 && rows.sizes() == dout.sizes() && dout.is_contiguous() &&
                        rows.scalar_type() == residual_type.value_or(io),
                    name, ": dout must be contiguous with the rows' shape");
  TORCH_CHECK_VALUE(!given(dsum) || (residual_type && dsum->sizes() == dout.sizes() && dsum->is_contiguous() &&
                                     dsum->scalar_type() == *residual_type),
                    name, ": dsum must be contiguous with the sum's shape and dtype");
  TORCH_CHECK_VALUE(!given(z) || (z->sizes() == dout.sizes() && z->scalar_type() == io), name,
                    ": z must have dout's shape and dtype");
  want_columns(weight, dout, name);
  TORCH_CHECK_VALUE(!given(weight) || !bias_type || weight->scalar_type() == *bias_type, name,
                    ": weight and bias must share a dtype");
  const int64_t dim = dout.size(-1);
  const c10::cuda::CUDAGuard guard(dout.device());
  const Tensor vm = as_matrix(rows, dim);
  const OptTensor zm = given(z) ? OptTensor(as_matrix(*z, dim)) : std::nullopt;
  const auto w_type = given(weight) ? weight->scalar_type() : bias_type.value_or(kF32);
  mb200_norm_bwd_params p = {};
  p.fwd = norm_params(vm, zm, weight, std::nullopt, io, w_type, eps, group, rms, gate);
  if (residual_type) {  // the backward asks only whether there was one
    p.fwd.residual = p.fwd.x;
    p.fwd.residual_dtype = code(*residual_type);
  }
  const bool own_dres = want_dresidual && residual_type && *residual_type != io;
  const auto maybe = [&](bool want, at::IntArrayRef shape, at::ScalarType t) {
    return want ? make(shape, dout, t) : make({0}, dout, t);
  };
  Tensor dx = make(dout.sizes(), dout, io);
  Tensor dres = maybe(own_dres, dout.sizes(), own_dres ? *residual_type : io);
  Tensor dz = maybe(given(z), dout.sizes(), io);
  const bool want_dw = given(weight) && want_dweight;
  Tensor dw = maybe(want_dw, {dim}, want_dw ? w_type : io);
  Tensor db = maybe(bias_type.has_value(), {dim}, bias_type.value_or(io));
  p.dout = ptr(dout);
  p.dsum = ptr(dsum);
  p.dx = ptr(dx);
  p.dresidual = own_dres ? ptr(dres) : nullptr;
  p.dz = given(z) ? ptr(dz) : nullptr;
  p.dweight = want_dw ? ptr(dw) : nullptr;
  p.dbias = bias_type ? ptr(db) : nullptr;
  const auto bytes = static_cast<int64_t>(mb200_norm_bwd_workspace_size(&p));
  Tensor ws = bytes > 0 ? make({bytes}, dout, at::kByte) : Tensor();
  check_status(mb200_norm_bwd(&p, ptr(ws), bytes, stream_of(dout)), name);
  return {dx, dres, dz, dw, db};
}

auto& norm_fwd_op() {
  static auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("mamba_b200::norm_fwd", "").typed<decltype(norm_fwd)>();
  return op;
}
auto& norm_bwd_op() {
  static auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("mamba_b200::norm_bwd", "").typed<decltype(norm_bwd)>();
  return op;
}

struct Norm : torch::autograd::Function<Norm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual,
                               const OptTensor& weight, const OptTensor& bias, double eps, bool rms) {
    const bool res = given(residual);
    ctx->saved_data["f"] = std::vector<int64_t>{
        res ? static_cast<int64_t>(residual->scalar_type()) : -1,
        given(bias) && bias->requires_grad() ? static_cast<int64_t>(bias->scalar_type()) : -1,
        static_cast<int64_t>(x.scalar_type()), rms, res && residual->requires_grad(),
        given(weight) && weight->requires_grad()};
    ctx->saved_data["eps"] = eps;
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, total] = norm_fwd_op().call(x, residual, std::nullopt, weight, bias, eps, x.size(-1), rms,
                                           MB200_GATE_NONE, res);
    // The sum is an output whether or not the caller takes it: as one it is saved with its way back to x and the
    // residual, on which a second backward raises.
    ctx->save_for_backward({res ? total : x, or_undefined(weight)});
    ctx->set_materialize_grads(false);
    if (res) return {out, total};
    return {out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(6);
    const Tensor dsum = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !dsum.defined()) return none;
    const auto s = ctx->get_saved_variables();
    const auto f = ctx->saved_data["f"].toIntVector();
    const auto type = [](int64_t t) {
      return t < 0 ? std::nullopt : std::optional<at::ScalarType>(static_cast<at::ScalarType>(t));
    };
    const auto io = *type(f[2]);
    const Tensor dout = grads[0].defined() ? grads[0].contiguous() : at::zeros(s[0].sizes(), s[0].options().dtype(io));
    const OptTensor ds = dsum.defined() ? OptTensor(dsum.contiguous()) : std::nullopt;
    auto [dx, dres, dz, dw, db] =
        norm_bwd_op().call(dout, ds, s[0], std::nullopt, s[1].defined() ? OptTensor(s[1]) : std::nullopt, type(f[0]),
                           type(f[1]), ctx->saved_data["eps"].toDouble(), s[0].size(-1), f[3] != 0, MB200_GATE_NONE,
                           f[4] != 0, f[5] != 0);
    none[0] = dx;
    if (f[4]) none[1] = *type(f[0]) == io ? dx : dres;
    if (f[5]) none[2] = dw;
    if (f[1] >= 0) none[3] = db;
    return none;
  }
};

struct GatedNorm : torch::autograd::Function<GatedNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& z, const OptTensor& weight,
                               double eps, int64_t group, int64_t gate) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, total] = norm_fwd_op().call(x, std::nullopt, z, weight, std::nullopt, eps, group, true, gate, false);
    ctx->save_for_backward({x, z, or_undefined(weight)});
    ctx->saved_data["f"] = std::vector<int64_t>{group, gate, given(weight) && weight->requires_grad()};
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return {out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list none(6);
    if (!grads[0].defined()) return none;
    const auto s = ctx->get_saved_variables();
    const auto f = ctx->saved_data["f"].toIntVector();
    auto [dx, dres, dz, dw, db] =
        norm_bwd_op().call(grads[0].contiguous(), std::nullopt, s[0], s[1],
                           s[2].defined() ? OptTensor(s[2]) : std::nullopt, std::nullopt, std::nullopt,
                           ctx->saved_data["eps"].toDouble(), f[0], true, f[1], false, f[2] != 0);
    none[0] = dx, none[1] = dz;
    if (f[2]) none[2] = dw;
    return none;
  }
};

// weight and bias as the kernels take them: contiguous, of one dtype, float32 or x's.
at::ScalarType weight_type(const OptTensor& w, const OptTensor& b, at::ScalarType io) {
  const auto one = given(w) ? w->scalar_type() : given(b) ? b->scalar_type() : kF32;
  const bool alike = !given(w) || !given(b) || w->scalar_type() == b->scalar_type();
  return alike && one == io ? io : kF32;
}

std::tuple<Tensor, Tensor> norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                const OptTensor& residual, double eps, bool prenorm, bool residual_in_fp32, bool rms) {
  want_cuda(x);
  want_floating("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  const int64_t dim = x.size(-1);
  want_shape("weight", weight, {dim}, x, "x");
  want_shape("bias", bias, {dim}, x, "x");
  want_shape("residual", residual, x.sizes(), x, "x");
  no_tangents({&x}, {&weight, &bias, &residual});
  TORCH_CHECK_NOT_IMPLEMENTED(dim <= MB200_NORM_MAX_DIM, "a last dimension > ", MB200_NORM_MAX_DIM,
                              " is not supported by the B200 kernels");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  const auto io = is_io(x.scalar_type()) ? x.scalar_type() : kF32;
  const Tensor xk = cast(x, io);
  const auto wt = weight_type(weight, bias, io);
  const OptTensor w = dense(weight, wt), b = dense(bias, wt);
  OptTensor res;
  if (given(residual))
    res = cast(*residual, residual->scalar_type() == io && !residual_in_fp32 ? io : kF32);
  const bool carried = prenorm && res.has_value();
  Tensor out, total;
  if (wants_grad({&xk}) || (res && wants_grad({&*res})) || (w && wants_grad({&*w})) || (b && wants_grad({&*b}))) {
    auto r = Norm::apply(xk, res, w, b, eps, rms);
    out = r[0];
    if (carried) total = r[1];
  } else {
    std::tie(out, total) =
        norm_fwd_op().call(xk, res, std::nullopt, w, b, eps, dim, rms, MB200_GATE_NONE, carried);
  }
  if (prenorm && !res.has_value()) total = residual_in_fp32 ? cast(x, kF32) : x;
  return {cast(out, x.scalar_type()), prenorm ? total : Tensor()};
}

Tensor gated_norm(const Tensor& x, const Tensor& z, const OptTensor& weight, double eps,
                  std::optional<int64_t> group_size, bool norm_before_gate) {
  want_cuda(x);
  want_floating("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  const int64_t dim = x.size(-1);
  want_shape("z", z, x.sizes(), x, "x");
  want_shape("weight", weight, {dim}, x, "x");
  no_tangents({&x, &z}, {&weight});
  const int64_t group = group_size.value_or(dim);
  TORCH_CHECK_VALUE(dim == 0 || (group >= 1 && dim % group == 0), "group_size must divide the last dimension ", dim,
                    ", got ", group);
  TORCH_CHECK_NOT_IMPLEMENTED(dim == 0 || (group <= MB200_NORM_MAX_DIM && dim / group <= 65535), "group_size up to ",
                              MB200_NORM_MAX_DIM, " and at most 65535 groups are supported by the B200 kernels");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  const auto io = is_io(x.scalar_type()) && z.scalar_type() == x.scalar_type() ? x.scalar_type() : kF32;
  const Tensor xk = cast(x, io), zk = cast(z, io);
  const OptTensor w = dense(weight, weight_type(weight, std::nullopt, io));
  const int64_t gate = norm_before_gate ? MB200_GATE_AFTER_NORM : MB200_GATE_BEFORE_NORM;
  Tensor out;
  if (wants_grad({&xk, &zk}) || (w && wants_grad({&*w})))
    out = GatedNorm::apply(xk, zk, w, eps, group, gate)[0];
  else
    out = std::get<0>(norm_fwd_op().call(xk, std::nullopt, zk, w, std::nullopt, eps, group, true, gate, false));
  return cast(out, x.scalar_type());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mamba_b200, m) {
  m.def(
      "gated_scan_fwd(Tensor u, Tensor decay_gate, Tensor input_gate, Tensor A, Tensor? initial_state, "
      "Tensor? seq_idx, bool save_states) -> (Tensor, Tensor, Tensor)");
  m.def(
      "gated_scan_bwd(Tensor u, Tensor decay_gate, Tensor input_gate, Tensor A, Tensor? initial_state, "
      "Tensor? seq_idx, Tensor chunk_states, Tensor dout, Tensor? dlast_state) "
      "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("gated_scan_update(Tensor(a!) state, Tensor u, Tensor decay_gate, Tensor input_gate, Tensor A) -> Tensor");
  m.def(
      "gated_scan_update_out(Tensor state, Tensor u, Tensor decay_gate, Tensor input_gate, Tensor A, "
      "Tensor(a!) new_state) -> Tensor");
  m.def(
      "norm_fwd(Tensor x, Tensor? residual, Tensor? z, Tensor? weight, Tensor? bias, float eps, int group_size, "
      "bool rms, int gate, bool want_sum) -> (Tensor, Tensor)");
  m.def(
      "norm_bwd(Tensor dout, Tensor? dsum, Tensor rows, Tensor? z, Tensor? weight, ScalarType? residual_dtype, "
      "ScalarType? bias_dtype, float eps, int group_size, bool rms, int gate, bool want_dresidual, "
      "bool want_dweight=True) "
      "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "gated_scan(Tensor u, Tensor decay_gate, Tensor input_gate, Tensor A, Tensor? initial_state, Tensor? seq_idx) "
      "-> (Tensor, Tensor)",
      gated_scan);
  m.def(
      "gated_step(Tensor(a!) state, Tensor u, Tensor decay_gate, Tensor input_gate, Tensor A, Tensor(b!)? out_state) "
      "-> Tensor",
      gated_step);
  m.def(
      "norm(Tensor x, Tensor? weight, Tensor? bias, Tensor? residual, float eps, bool prenorm, bool residual_in_fp32, "
      "bool rms) -> (Tensor, Tensor)",
      norm);
  m.def(
      "gated_norm(Tensor x, Tensor z, Tensor? weight, float eps, int? group_size, bool norm_before_gate) -> Tensor",
      gated_norm);
}

TORCH_LIBRARY_IMPL(mamba_b200, CUDA, m) {
  m.impl("gated_scan_fwd", gated_scan_fwd);
  m.impl("gated_scan_bwd", gated_scan_bwd);
  m.impl("gated_scan_update", gated_scan_update);
  m.impl("gated_scan_update_out", gated_scan_update_out);
  m.impl("norm_fwd", norm_fwd);
  m.impl("norm_bwd", norm_bwd);
}

// Gradients are differentiable once: a second backward raises.
TORCH_LIBRARY_IMPL(mamba_b200, Autograd, m) {
  m.impl("gated_scan_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("norm_bwd", torch::autograd::autogradNotImplementedFallback());
}
