// torch custom ops of the sequence operators over the C ABI
// (include/pla_b200.h): torch.ops.pla_b200.{causal_depthwise, qk_norm_rotate,
// gated_delta_rule} with their gradients, and the single-token forms.
//
// As in torch_ops.cpp: TORCH_CHECK argument errors, a CUDAGuard on the input's
// device, outputs and workspaces allocated by the op on the current stream's
// allocator, the launch on the current stream, a Meta kernel per op.  The
// three training ops carry a C++ autograd function whose backward is an op of
// its own, so autograd, fake tensors and graph capture see the same calls; a
// second derivative and a forward-mode one raise.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/pla_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kHalf: return PLA_F16;
    case at::kFloat: return PLA_F32;
    case at::kBFloat16: return PLA_BF16;
    default: TORCH_CHECK(false, op, ": unsupported dtype ", t.scalar_type());
  }
}
void check(int st, const char* what) {
  if (st == PLA_OK) return;
  const std::string detail = st == PLA_ERR_CUDA ? pla_last_cuda_error() : "";
  TORCH_CHECK(false, what, ": ", pla_status_string(st), detail.empty() ? "" : " (" + detail + ")");
}
pla_stream_t stream_of(const Tensor& x) {
  return reinterpret_cast<pla_stream_t>(c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
}
const void* data(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
Tensor or_none(const optional<Tensor>& t) { return t && t->defined() ? *t : Tensor(); }
optional<Tensor> as_optional(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }
// The innermost dimension dense; other strides are the kernels' to follow.
Tensor dense_rows(const Tensor& t) { return t.defined() && t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }
int as_int(int64_t v, const char* op) {
  TORCH_CHECK(v <= INT32_MAX, op, ": size exceeds int32");
  return static_cast<int>(v);
}

void on_device(const Tensor& x, const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), op, ": ", name, " must be a CUDA tensor on the input's device");
}
void like_input(const Tensor& x, const Tensor& t, const char* op, const char* name) {
  on_device(x, t, op, name);
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), op, ": ", name, " dtype ", t.scalar_type(), " does not match the input's ",
              x.scalar_type());
}
// Sequences of a batch: rows, or what cu_seqlens cuts one row into.
int64_t sequences_of(const Tensor& x, const Tensor& cu, const char* op) {
  if (!cu.defined()) return x.size(0);
  on_device(x, cu, op, "cu_seqlens");
  TORCH_CHECK(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.numel() >= 2 && cu.is_contiguous(), op,
              ": cu_seqlens must be a contiguous int32 vector of at least 2 entries");
  TORCH_CHECK(x.size(0) == 1, op, ": a ragged batch (cu_seqlens) has one batch row");
  return cu.numel() - 1;
}

// ---- causal depthwise convolution ------------------------------------------
constexpr const char* kCausal = "causal_depthwise";

struct CausalArgs {
  Tensor x, w, b, cu, state;
  pla_causal a = {};
};
Tensor filter_rows(const Tensor& weight, int64_t channels, const char* op) {
  TORCH_CHECK((weight.dim() == 2 || (weight.dim() == 3 && weight.size(1) == 1)) && weight.size(0) == channels, op,
              ": weight must have shape [C, taps] or [C, 1, taps], got ", weight.sizes());
  TORCH_CHECK(weight.size(-1) >= 2 && weight.size(-1) <= 4, op, ": 2 to 4 taps are supported, got ", weight.size(-1));
  return weight.contiguous();
}
CausalArgs causal_args(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, bool silu,
                       const optional<Tensor>& cu, const optional<Tensor>& state) {
  TORCH_CHECK(x.is_cuda(), kCausal, ": x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 3, kCausal, ": x must have shape [batch, tokens, channels], got ", x.sizes());
  CausalArgs r;
  r.a.dtype = code_of(x, kCausal);
  r.x = dense_rows(x);
  const int64_t C = x.size(2);
  like_input(x, weight, kCausal, "weight");
  r.w = filter_rows(weight, C, kCausal);
  r.b = or_none(bias);
  if (r.b.defined()) {
    like_input(x, r.b, kCausal, "bias");
    TORCH_CHECK(r.b.dim() == 1 && r.b.numel() == C, kCausal, ": bias must have ", C, " elements");
    r.b = r.b.contiguous();
  }
  r.cu = or_none(cu);
  const int64_t n = sequences_of(x, r.cu, kCausal);
  const int64_t taps = r.w.size(-1);
  r.state = or_none(state);
  if (r.state.defined()) {
    like_input(x, r.state, kCausal, "state");
    TORCH_CHECK(r.state.dim() == 3 && r.state.size(0) == n && r.state.size(1) == taps - 1 && r.state.size(2) == C, kCausal,
                ": state must have shape [", n, ", ", taps - 1, ", ", C, "], got ", r.state.sizes());
    r.state = r.state.contiguous();
  }
  r.a.x = data(r.x);
  r.a.x_batch = r.x.stride(0);
  r.a.x_token = r.x.stride(1);
  r.a.w = data(r.w);
  r.a.b = data(r.b);
  r.a.cu_seqlens = r.cu.defined() ? r.cu.data_ptr<int>() : nullptr;
  r.a.state_in = data(r.state);
  r.a.batch = as_int(x.size(0), kCausal);
  r.a.tokens = as_int(x.size(1), kCausal);
  r.a.channels = as_int(C, kCausal);
  r.a.taps = static_cast<int>(taps);
  r.a.sequences = as_int(n, kCausal);
  r.a.silu = silu;
  return r;
}

std::tuple<Tensor, Tensor> causal_cuda(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias, bool silu,
                                       const optional<Tensor>& cu, const optional<Tensor>& state, bool return_state) {
  CausalArgs r = causal_args(x, weight, bias, silu, cu, state);
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor last = return_state ? at::empty({r.a.sequences, r.a.taps - 1, r.a.channels}, x.options()) : at::empty({0}, x.options());
  r.a.y = out(y);
  r.a.state_out = return_state ? out(last) : nullptr;
  check(pla_causal_depthwise_forward(&r.a, stream_of(x)), "pla_causal_depthwise_forward");
  return {y, last};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> causal_backward_cuda(const Tensor& dy, const optional<Tensor>& dstate,
                                                                const Tensor& x, const Tensor& weight,
                                                                const optional<Tensor>& bias, bool silu,
                                                                const optional<Tensor>& cu, const optional<Tensor>& state) {
  CausalArgs r = causal_args(x, weight, bias, silu, cu, state);
  c10::cuda::CUDAGuard guard(x.device());
  like_input(x, dy, kCausal, "dy");
  TORCH_CHECK(dy.sizes() == x.sizes(), kCausal, ": dy must have x's shape");
  const Tensor g = dense_rows(dy);
  Tensor dlast = or_none(dstate);
  if (dlast.defined()) {
    like_input(x, dlast, kCausal, "dstate");
    TORCH_CHECK(dlast.numel() == static_cast<int64_t>(r.a.sequences) * (r.a.taps - 1) * r.a.channels, kCausal,
                ": dstate must have the state's shape");
    dlast = dlast.contiguous();
  }
  Tensor dx = at::empty(x.sizes(), x.options()), dw = at::empty(weight.sizes(), x.options());
  Tensor db = r.b.defined() ? at::empty({r.a.channels}, x.options()) : at::empty({0}, x.options());
  Tensor dfirst = r.state.defined() ? at::empty(r.state.sizes(), x.options()) : at::empty({0}, x.options());
  const size_t bytes = pla_causal_depthwise_workspace(&r.a);
  Tensor work = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  pla_causal_gradient grad = {};
  grad.dy = data(g);
  grad.dy_batch = g.stride(0);
  grad.dy_token = g.stride(1);
  grad.dstate_out = data(dlast);
  grad.dx = out(dx);
  grad.dw = out(dw);
  grad.db = out(db);
  grad.dstate_in = out(dfirst);
  grad.workspace = out(work);
  grad.workspace_bytes = bytes;
  check(pla_causal_depthwise_backward(&r.a, &grad, stream_of(x)), "pla_causal_depthwise_backward");
  return {dx, dw, db, dfirst};
}

Tensor causal_step_cuda(const Tensor& x, const Tensor& state, const Tensor& weight, const optional<Tensor>& bias, bool silu) {
  const char* op = "causal_depthwise_step";
  TORCH_CHECK(x.is_cuda(), op, ": x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 2, op, ": x must have shape [sequences, channels], got ", x.sizes());
  const int code = code_of(x, op);
  const int64_t n = x.size(0), C = x.size(1);
  like_input(x, weight, op, "weight");
  const Tensor w = filter_rows(weight, C, op);
  const int64_t taps = w.size(-1);
  Tensor b = or_none(bias);
  if (b.defined()) {
    like_input(x, b, op, "bias");
    TORCH_CHECK(b.dim() == 1 && b.numel() == C, op, ": bias must have ", C, " elements");
    b = b.contiguous();
  }
  like_input(x, state, op, "state");
  TORCH_CHECK(state.dim() == 3 && state.size(0) == n && state.size(1) == taps - 1 && state.size(2) == C, op,
              ": state must have shape [", n, ", ", taps - 1, ", ", C, "], got ", state.sizes());
  TORCH_CHECK(n == 0 || C == 0 || state[0].is_contiguous(), op, ": a sequence's state must be dense (it is updated in place)");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor xs = dense_rows(x);
  Tensor y = at::empty(x.sizes(), x.options());
  check(pla_causal_depthwise_step(data(xs), xs.stride(0), out(state), state.stride(0), data(w), data(b), out(y),
                                  as_int(n, op), as_int(C, op), static_cast<int>(taps), silu, code, stream_of(x)),
        "pla_causal_depthwise_step");
  return y;
}

// ---- norms of queries and keys with the position rotation -------------------
constexpr const char* kNorm = "qk_norm_rotate";

struct NormArgs {
  Tensor q, k, wq, wk, cos, sin, pos;
  pla_qk_norm a = {};
};
NormArgs norm_args(const Tensor& q, const Tensor& k, const optional<Tensor>& wq, const optional<Tensor>& wk,
                   const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& positions, bool l2,
                   double eps, bool interleaved) {
  TORCH_CHECK(q.is_cuda(), kNorm, ": q must be a CUDA tensor");
  NormArgs r;
  r.a.dtype = code_of(q, kNorm);
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, kNorm, ": q and k must have shape [batch, tokens, heads, dim]");
  like_input(q, k, kNorm, "k");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3), kNorm,
              ": q and k must agree in batch, tokens and dim, got ", q.sizes(), " and ", k.sizes());
  const int64_t D = q.size(3);
  TORCH_CHECK(D <= 256, kNorm, ": heads of at most 256 features are supported, got ", D);
  TORCH_CHECK(eps >= 0, kNorm, ": eps must not be negative");
  r.q = dense_rows(q);
  r.k = dense_rows(k);
  r.wq = or_none(wq);
  r.wk = or_none(wk);
  for (Tensor* w : {&r.wq, &r.wk})
    if (w->defined()) {
      like_input(q, *w, kNorm, "weight");
      TORCH_CHECK(w->dim() == 1 && w->numel() == D, kNorm, ": a weight must have ", D, " elements");
      *w = w->contiguous();
    }
  r.cos = or_none(cos);
  r.sin = or_none(sin);
  r.pos = or_none(positions);
  TORCH_CHECK(r.cos.defined() == r.sin.defined(), kNorm, ": cos and sin come together");
  TORCH_CHECK(!r.pos.defined() || r.cos.defined(), kNorm, ": positions need the tables cos and sin");
  if (r.cos.defined()) {
    for (const Tensor* t : {&r.cos, &r.sin}) {
      on_device(q, *t, kNorm, "cos / sin");
      TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->sizes() == r.cos.sizes() && 2 * t->size(1) <= D, kNorm,
                  ": cos and sin must be float32 [positions, rotated / 2] with at most ", D, " rotated features");
    }
    r.cos = r.cos.contiguous();
    r.sin = r.sin.contiguous();
    r.a.rot = static_cast<int>(2 * r.cos.size(1));
    r.a.table_rows = as_int(r.cos.size(0), kNorm);
    r.a.cos_table = r.a.rot ? r.cos.data_ptr<float>() : nullptr;
    r.a.sin_table = r.a.rot ? r.sin.data_ptr<float>() : nullptr;
  }
  if (r.pos.defined()) {
    on_device(q, r.pos, kNorm, "positions");
    TORCH_CHECK(r.pos.scalar_type() == at::kInt || r.pos.scalar_type() == at::kLong, kNorm, ": positions must be int32 or int64");
    TORCH_CHECK((r.pos.dim() == 1 && r.pos.size(0) == q.size(1)) ||
                    (r.pos.dim() == 2 && (r.pos.size(0) == q.size(0) || r.pos.size(0) == 1) && r.pos.size(1) == q.size(1)),
                kNorm, ": positions must have shape [tokens], [1, tokens] or [batch, tokens], got ", r.pos.sizes());
    r.pos = r.pos.contiguous();
    r.a.positions = data(r.pos);
    r.a.position_batch = r.pos.dim() == 2 && r.pos.size(0) > 1 ? r.pos.stride(0) : 0;
    r.a.position_bytes = static_cast<int>(r.pos.element_size());
  }
  r.a.batch = as_int(q.size(0), kNorm);
  r.a.tokens = as_int(q.size(1), kNorm);
  r.a.dim = static_cast<int>(D);
  r.a.interleaved = interleaved;
  r.a.l2 = l2;
  r.a.eps = static_cast<float>(eps);
  const Tensor* x[2] = {&r.q, &r.k};
  const Tensor* w[2] = {&r.wq, &r.wk};
  pla_norm_side* side[2] = {&r.a.q, &r.a.k};
  for (int i = 0; i < 2; ++i) {
    side[i]->x = data(*x[i]);
    side[i]->x_batch = x[i]->stride(0);
    side[i]->x_token = x[i]->stride(1);
    side[i]->x_head = x[i]->stride(2);
    side[i]->w = data(*w[i]);
    side[i]->heads = as_int(x[i]->size(2), kNorm);
  }
  return r;
}

std::tuple<Tensor, Tensor> norm_cuda(const Tensor& q, const Tensor& k, const optional<Tensor>& wq, const optional<Tensor>& wk,
                                     const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& pos,
                                     bool l2, double eps, bool interleaved) {
  NormArgs r = norm_args(q, k, wq, wk, cos, sin, pos, l2, eps, interleaved);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  r.a.q.y = out(yq);
  r.a.k.y = out(yk);
  check(pla_qk_norm_rotate_forward(&r.a, stream_of(q)), "pla_qk_norm_rotate_forward");
  return {yq, yk};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> norm_backward_cuda(const Tensor& gq, const Tensor& gk, const Tensor& q,
                                                              const Tensor& k, const optional<Tensor>& wq,
                                                              const optional<Tensor>& wk, const optional<Tensor>& cos,
                                                              const optional<Tensor>& sin, const optional<Tensor>& pos, bool l2,
                                                              double eps, bool interleaved) {
  NormArgs r = norm_args(q, k, wq, wk, cos, sin, pos, l2, eps, interleaved);
  c10::cuda::CUDAGuard guard(q.device());
  like_input(q, gq, kNorm, "dq");
  like_input(q, gk, kNorm, "dk");
  TORCH_CHECK(gq.sizes() == q.sizes() && gk.sizes() == k.sizes(), kNorm, ": gradients must have their outputs' shapes");
  const Tensor dy[2] = {dense_rows(gq), dense_rows(gk)};
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  Tensor dwq = at::empty({r.wq.defined() ? r.a.dim : 0}, q.options()), dwk = at::empty({r.wk.defined() ? r.a.dim : 0}, q.options());
  pla_norm_side* side[2] = {&r.a.q, &r.a.k};
  for (int i = 0; i < 2; ++i) {
    side[i]->dy = data(dy[i]);
    side[i]->dy_batch = dy[i].stride(0);
    side[i]->dy_token = dy[i].stride(1);
    side[i]->dy_head = dy[i].stride(2);
    side[i]->y = out(i ? dk : dq);
    side[i]->dw = out(i ? dwk : dwq);
  }
  const size_t bytes = pla_qk_norm_rotate_workspace(&r.a);
  Tensor work = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  check(pla_qk_norm_rotate_backward(&r.a, out(work), bytes, stream_of(q)), "pla_qk_norm_rotate_backward");
  return {dq, dk, dwq, dwk};
}

// ---- gated delta rule ------------------------------------------------------
constexpr const char* kDelta = "gated_delta_rule";

struct DeltaArgs {
  Tensor q, k, v, g, beta, cu, state;
  pla_delta a = {};
};
void check_gates(const Tensor& x, const Tensor& g, const Tensor& beta, const char* op) {
  on_device(x, g, op, "g");
  on_device(x, beta, op, "beta");
  TORCH_CHECK(g.scalar_type() == beta.scalar_type() && (g.scalar_type() == x.scalar_type() || g.scalar_type() == at::kFloat), op,
              ": g and beta must both have the input's dtype or both be float32");
}
DeltaArgs delta_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, double scale,
                     const optional<Tensor>& cu, const optional<Tensor>& state) {
  TORCH_CHECK(q.is_cuda(), kDelta, ": q must be a CUDA tensor");
  DeltaArgs r;
  r.a.dtype = code_of(q, kDelta);
  like_input(q, k, kDelta, "k");
  like_input(q, v, kDelta, "v");
  check_gates(q, g, beta, kDelta);
  TORCH_CHECK(q.dim() == 4 && v.dim() == 4 && k.sizes() == q.sizes(), kDelta,
              ": q and k must have one shape [batch, tokens, key heads, Dk], v [batch, tokens, value heads, Dv]");
  const int64_t B = q.size(0), T = q.size(1), Hk = q.size(2), Dk = q.size(3), Hv = v.size(2), Dv = v.size(3);
  TORCH_CHECK(v.size(0) == B && v.size(1) == T, kDelta, ": v must have q's batch and tokens");
  TORCH_CHECK(Hk >= 1 && Hv >= 1 && Hv % Hk == 0, kDelta, ": value heads must be a multiple of key heads, got ", Hv, " and ", Hk);
  TORCH_CHECK(Dk >= 1 && Dk <= 128 && Dv >= 1 && Dv <= 128, kDelta, ": Dk and Dv from 1 to 128 are supported, got ", Dk, " and ", Dv);
  for (const Tensor* t : {&g, &beta})
    TORCH_CHECK(t->dim() == 3 && t->size(0) == B && t->size(1) == T && t->size(2) == Hv, kDelta,
                ": g and beta must have shape [batch, tokens, value heads]");
  r.q = dense_rows(q);
  r.k = dense_rows(k);
  r.v = dense_rows(v);
  r.g = g;
  r.beta = beta;
  r.cu = or_none(cu);
  const int64_t n = sequences_of(q, r.cu, kDelta);
  r.state = or_none(state);
  if (r.state.defined()) {
    on_device(q, r.state, kDelta, "state");
    TORCH_CHECK(r.state.scalar_type() == at::kFloat && r.state.dim() == 4 && r.state.size(0) == n && r.state.size(1) == Hv &&
                    r.state.size(2) == Dk && r.state.size(3) == Dv,
                kDelta, ": state must be float32 [", n, ", ", Hv, ", ", Dk, ", ", Dv, "], got ", r.state.sizes());
    r.state = r.state.contiguous();
  }
  pla_delta& a = r.a;
  a.q = data(r.q), a.k = data(r.k), a.v = data(r.v), a.g = data(r.g), a.beta = data(r.beta);
  a.q_batch = r.q.stride(0), a.q_token = r.q.stride(1), a.q_head = r.q.stride(2);
  a.k_batch = r.k.stride(0), a.k_token = r.k.stride(1), a.k_head = r.k.stride(2);
  a.v_batch = r.v.stride(0), a.v_token = r.v.stride(1), a.v_head = r.v.stride(2);
  a.g_batch = g.stride(0), a.g_token = g.stride(1), a.g_head = g.stride(2);
  a.beta_batch = beta.stride(0), a.beta_token = beta.stride(1), a.beta_head = beta.stride(2);
  a.cu_seqlens = r.cu.defined() ? r.cu.data_ptr<int>() : nullptr;
  a.state_in = static_cast<const float*>(data(r.state));
  a.batch = as_int(B, kDelta), a.tokens = as_int(T, kDelta), a.sequences = as_int(n, kDelta);
  a.hk = as_int(Hk, kDelta), a.hv = as_int(Hv, kDelta), a.dk = static_cast<int>(Dk), a.dv = static_cast<int>(Dv);
  a.gates32 = g.scalar_type() == at::kFloat;
  a.scale = static_cast<float>(scale);
  return r;
}
Tensor delta_workspace(pla_delta* a, const Tensor& x, bool backward) {
  a->workspace_bytes = pla_gated_delta_rule_workspace(a, backward);
  Tensor work = at::empty({static_cast<int64_t>(a->workspace_bytes)}, x.options().dtype(at::kByte));
  a->workspace = out(work);
  return work;
}

std::tuple<Tensor, Tensor> delta_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                      double scale, const optional<Tensor>& cu, const optional<Tensor>& state,
                                      bool return_state) {
  DeltaArgs r = delta_args(q, k, v, g, beta, scale, cu, state);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor o = at::empty(v.sizes(), v.options());
  const auto f32 = q.options().dtype(at::kFloat);
  Tensor last = return_state ? at::empty({r.a.sequences, r.a.hv, r.a.dk, r.a.dv}, f32) : at::empty({0}, f32);
  r.a.o = out(o);
  r.a.state_out = return_state ? static_cast<float*>(out(last)) : nullptr;
  const Tensor work = delta_workspace(&r.a, q, false);
  check(pla_gated_delta_rule_forward(&r.a, stream_of(q)), "pla_gated_delta_rule_forward");
  return {o, last};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> delta_backward_cuda(
    const Tensor& d_o, const optional<Tensor>& dstate, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
    const Tensor& beta, double scale, const optional<Tensor>& cu, const optional<Tensor>& state) {
  DeltaArgs r = delta_args(q, k, v, g, beta, scale, cu, state);
  c10::cuda::CUDAGuard guard(q.device());
  like_input(q, d_o, kDelta, "do");
  TORCH_CHECK(d_o.sizes() == v.sizes(), kDelta, ": do must have v's shape");
  const Tensor go = dense_rows(d_o);
  Tensor dlast = or_none(dstate);
  const auto f32 = q.options().dtype(at::kFloat);
  if (dlast.defined()) {
    on_device(q, dlast, kDelta, "dstate");
    TORCH_CHECK(dlast.scalar_type() == at::kFloat &&
                    dlast.numel() == static_cast<int64_t>(r.a.sequences) * r.a.hv * r.a.dk * r.a.dv,
                kDelta, ": dstate must have the state's shape and dtype");
    dlast = dlast.contiguous();
  }
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
  Tensor dg = at::empty(g.sizes(), g.options()), dbeta = at::empty(beta.sizes(), beta.options());
  Tensor dfirst = r.state.defined() ? at::empty(r.state.sizes(), f32) : at::empty({0}, f32);
  pla_delta_gradient grad = {};
  grad.d_o = data(go);
  grad.do_batch = go.stride(0), grad.do_token = go.stride(1), grad.do_head = go.stride(2);
  grad.dstate_out = static_cast<const float*>(data(dlast));
  grad.dstate_in = static_cast<float*>(out(dfirst));
  grad.dq = out(dq), grad.dk = out(dk), grad.dv = out(dv), grad.dg = out(dg), grad.dbeta = out(dbeta);
  const Tensor work = delta_workspace(&r.a, q, true);
  check(pla_gated_delta_rule_backward(&r.a, &grad, stream_of(q)), "pla_gated_delta_rule_backward");
  return {dq, dk, dv, dg, dbeta, dfirst};
}

Tensor delta_step_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                       const Tensor& state, double scale) {
  const char* op = "gated_delta_rule_step";
  TORCH_CHECK(q.is_cuda(), op, ": q must be a CUDA tensor");
  pla_delta_step a = {};
  a.dtype = code_of(q, op);
  like_input(q, k, op, "k");
  like_input(q, v, op, "v");
  check_gates(q, g, beta, op);
  TORCH_CHECK(q.dim() == 3 && v.dim() == 3 && k.sizes() == q.sizes() && v.size(0) == q.size(0), op,
              ": q and k must have one shape [sequences, key heads, Dk], v [sequences, value heads, Dv]");
  const int64_t n = q.size(0), Hk = q.size(1), Dk = q.size(2), Hv = v.size(1), Dv = v.size(2);
  TORCH_CHECK(Hk >= 1 && Hv >= 1 && Hv % Hk == 0, op, ": value heads must be a multiple of key heads, got ", Hv, " and ", Hk);
  TORCH_CHECK(Dk >= 1 && Dk <= 256 && Dv >= 1, op, ": Dk from 1 to 256 is supported, got ", Dk);
  for (const Tensor* t : {&g, &beta})
    TORCH_CHECK(t->dim() == 2 && t->size(0) == n && t->size(1) == Hv, op, ": g and beta must have shape [sequences, value heads]");
  on_device(q, state, op, "state");
  TORCH_CHECK(state.scalar_type() == at::kFloat && state.dim() == 4 && state.size(0) == n && state.size(1) == Hv &&
                  state.size(2) == Dk && state.size(3) == Dv,
              op, ": state must be float32 [", n, ", ", Hv, ", ", Dk, ", ", Dv, "], got ", state.sizes());
  TORCH_CHECK(n == 0 || state[0].is_contiguous(), op, ": a sequence's state must be dense (it is updated in place)");
  c10::cuda::CUDAGuard guard(q.device());
  const Tensor qs = dense_rows(q), ks = dense_rows(k), vs = dense_rows(v);
  Tensor o = at::empty(v.sizes(), v.options());
  a.q = data(qs), a.k = data(ks), a.v = data(vs), a.g = data(g), a.beta = data(beta);
  a.q_row = qs.stride(0), a.q_head = qs.stride(1), a.k_row = ks.stride(0), a.k_head = ks.stride(1);
  a.v_row = vs.stride(0), a.v_head = vs.stride(1);
  a.g_row = g.stride(0), a.g_head = g.stride(1), a.beta_row = beta.stride(0), a.beta_head = beta.stride(1);
  a.state = static_cast<float*>(out(state));
  a.state_row = state.stride(0);
  a.o = out(o);
  a.n = as_int(n, op), a.hk = as_int(Hk, op), a.hv = as_int(Hv, op), a.dk = static_cast<int>(Dk), a.dv = as_int(Dv, op);
  a.gates32 = g.scalar_type() == at::kFloat;
  a.scale = static_cast<float>(scale);
  check(pla_gated_delta_rule_step(&a, stream_of(q)), "pla_gated_delta_rule_step");
  return o;
}

// ---- Meta kernels ----------------------------------------------------------
Tensor like_meta(const Tensor& x) { return at::empty_symint(x.sym_sizes(), x.options()); }
Tensor none_meta(const Tensor& x) { return at::empty_symint({0}, x.options()); }
c10::SymInt sequences_meta(const Tensor& x, const optional<Tensor>& cu) {
  return cu && cu->defined() ? cu->sym_size(0) - 1 : x.sym_size(0);
}

std::tuple<Tensor, Tensor> causal_meta(const Tensor& x, const Tensor& weight, const optional<Tensor>&, bool,
                                       const optional<Tensor>& cu, const optional<Tensor>&, bool return_state) {
  TORCH_CHECK(x.dim() == 3, kCausal, ": x must have shape [batch, tokens, channels], got ", x.sym_sizes());
  return {like_meta(x), return_state ? at::empty_symint({sequences_meta(x, cu), weight.sym_size(-1) - 1, x.sym_size(2)}, x.options())
                                     : none_meta(x)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> causal_backward_meta(const Tensor&, const optional<Tensor>&, const Tensor& x,
                                                                const Tensor& weight, const optional<Tensor>& bias, bool,
                                                                const optional<Tensor>&, const optional<Tensor>& state) {
  return {like_meta(x), like_meta(weight), bias && bias->defined() ? like_meta(*bias) : none_meta(x),
          state && state->defined() ? like_meta(*state) : none_meta(x)};
}
Tensor causal_step_meta(const Tensor& x, const Tensor&, const Tensor&, const optional<Tensor>&, bool) { return like_meta(x); }
std::tuple<Tensor, Tensor> norm_meta(const Tensor& q, const Tensor& k, const optional<Tensor>&, const optional<Tensor>&,
                                     const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&, bool, double,
                                     bool) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, kNorm, ": q and k must have shape [batch, tokens, heads, dim]");
  return {like_meta(q), like_meta(k)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> norm_backward_meta(const Tensor&, const Tensor&, const Tensor& q, const Tensor& k,
                                                              const optional<Tensor>& wq, const optional<Tensor>& wk,
                                                              const optional<Tensor>&, const optional<Tensor>&,
                                                              const optional<Tensor>&, bool, double, bool) {
  return {like_meta(q), like_meta(k), wq && wq->defined() ? like_meta(*wq) : none_meta(q),
          wk && wk->defined() ? like_meta(*wk) : none_meta(q)};
}
std::tuple<Tensor, Tensor> delta_meta(const Tensor& q, const Tensor&, const Tensor& v, const Tensor&, const Tensor&, double,
                                      const optional<Tensor>& cu, const optional<Tensor>&, bool return_state) {
  TORCH_CHECK(q.dim() == 4 && v.dim() == 4, kDelta,
              ": q and k must have one shape [batch, tokens, key heads, Dk], v [batch, tokens, value heads, Dv]");
  const auto f32 = q.options().dtype(at::kFloat);
  return {like_meta(v), return_state ? at::empty_symint({sequences_meta(q, cu), v.sym_size(2), q.sym_size(3), v.sym_size(3)}, f32)
                                     : at::empty_symint({0}, f32)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> delta_backward_meta(
    const Tensor&, const optional<Tensor>&, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
    const Tensor& beta, double, const optional<Tensor>&, const optional<Tensor>& state) {
  return {like_meta(q), like_meta(k), like_meta(v), like_meta(g), like_meta(beta),
          state && state->defined() ? like_meta(*state) : at::empty_symint({0}, q.options().dtype(at::kFloat))};
}
Tensor delta_step_meta(const Tensor&, const Tensor&, const Tensor& v, const Tensor&, const Tensor&, const Tensor&, double) {
  return like_meta(v);
}

// ---- autograd --------------------------------------------------------------
// One typed handle per signature (each is used for one op).
template <typename Sig>
const c10::TypedOperatorHandle<Sig>& op_of(const char* name) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
  return op;
}
template <typename... Ts>
bool wants_gradient(const Ts&... ts) {
  const auto one = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>)
      return t.requires_grad();
    else
      return t && t->defined() && t->requires_grad();
  };
  return at::GradMode::is_enabled() && (one(ts) || ...);
}
// There is no forward-mode formula: a tangent raises (it does not ask for a gradient, so it would be dropped).
template <typename... Ts>
void refuse_tangents(const char* op, const Ts&... ts) {
  const auto one = [](const auto& t) {
    if constexpr (std::is_same_v<std::decay_t<decltype(t)>, Tensor>)
      return t._fw_grad(0).defined();
    else
      return t && t->defined() && t->_fw_grad(0).defined();
  };
  TORCH_CHECK_NOT_IMPLEMENTED(!(one(ts) || ...), op, ": forward-mode derivatives are not implemented");
}
Tensor grad_if(const Tensor& g, const Tensor& input) { return input.defined() ? g : Tensor(); }

std::tuple<Tensor, Tensor> causal_below(const Tensor& x, const Tensor& w, const optional<Tensor>& b, bool silu,
                                        const optional<Tensor>& cu, const optional<Tensor>& state, bool return_state) {
  const auto& op = op_of<decltype(causal_cuda)>("pla_b200::causal_depthwise");
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(x, w, b, silu, cu, state, return_state);
}
struct CausalFunction : torch::autograd::Function<CausalFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const optional<Tensor>& b, bool silu,
                               const optional<Tensor>& cu, const optional<Tensor>& state, bool return_state) {
    auto [y, last] = causal_below(x, w, b, silu, cu, state, return_state);
    ctx->save_for_backward({x, w, or_none(b), or_none(cu), or_none(state)});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    if (!return_state) ctx->mark_non_differentiable({last});
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto& op = op_of<decltype(causal_backward_cuda)>("pla_b200::causal_depthwise_backward");
    const Tensor dy = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
    auto [dx, dw, db, dstate] = op.call(dy, as_optional(grads[1]), s[0], s[1], as_optional(s[2]),
                                        ctx->saved_data["silu"].toBool(), as_optional(s[3]), as_optional(s[4]));
    return {dx, dw, grad_if(db, s[2]), Tensor(), Tensor(), grad_if(dstate, s[4]), Tensor()};
  }
};
std::tuple<Tensor, Tensor> causal_autograd(const Tensor& x, const Tensor& w, const optional<Tensor>& b, bool silu,
                                           const optional<Tensor>& cu, const optional<Tensor>& state, bool return_state) {
  refuse_tangents(kCausal, x, w, b, state);
  if (!wants_gradient(x, w, b, state)) return causal_below(x, w, b, silu, cu, state, return_state);
  auto r = CausalFunction::apply(x, w, b, silu, cu, state, return_state);
  return {r[0], r[1]};
}

std::tuple<Tensor, Tensor> norm_below(const Tensor& q, const Tensor& k, const optional<Tensor>& wq, const optional<Tensor>& wk,
                                      const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& pos,
                                      bool l2, double eps, bool interleaved) {
  const auto& op = op_of<decltype(norm_cuda)>("pla_b200::qk_norm_rotate");
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(q, k, wq, wk, cos, sin, pos, l2, eps, interleaved);
}
struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const optional<Tensor>& wq,
                               const optional<Tensor>& wk, const optional<Tensor>& cos, const optional<Tensor>& sin,
                               const optional<Tensor>& pos, bool l2, double eps, bool interleaved) {
    auto [yq, yk] = norm_below(q, k, wq, wk, cos, sin, pos, l2, eps, interleaved);
    ctx->save_for_backward({q, k, or_none(wq), or_none(wk), or_none(cos), or_none(sin), or_none(pos)});
    ctx->saved_data["l2"] = l2;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto& op = op_of<decltype(norm_backward_cuda)>("pla_b200::qk_norm_rotate_backward");
    auto [dq, dk, dwq, dwk] =
        op.call(grads[0], grads[1], s[0], s[1], as_optional(s[2]), as_optional(s[3]), as_optional(s[4]), as_optional(s[5]),
                as_optional(s[6]), ctx->saved_data["l2"].toBool(), ctx->saved_data["eps"].toDouble(),
                ctx->saved_data["interleaved"].toBool());
    return {dq, dk, grad_if(dwq, s[2]), grad_if(dwk, s[3]), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
std::tuple<Tensor, Tensor> norm_autograd(const Tensor& q, const Tensor& k, const optional<Tensor>& wq, const optional<Tensor>& wk,
                                         const optional<Tensor>& cos, const optional<Tensor>& sin, const optional<Tensor>& pos,
                                         bool l2, double eps, bool interleaved) {
  refuse_tangents(kNorm, q, k, wq, wk, cos, sin);
  TORCH_CHECK(!wants_gradient(cos, sin), kNorm, ": the tables have no gradient");
  if (!wants_gradient(q, k, wq, wk)) return norm_below(q, k, wq, wk, cos, sin, pos, l2, eps, interleaved);
  auto r = NormFunction::apply(q, k, wq, wk, cos, sin, pos, l2, eps, interleaved);
  return {r[0], r[1]};
}

std::tuple<Tensor, Tensor> delta_below(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                       double scale, const optional<Tensor>& cu, const optional<Tensor>& state,
                                       bool return_state) {
  const auto& op = op_of<decltype(delta_cuda)>("pla_b200::gated_delta_rule");
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(q, k, v, g, beta, scale, cu, state, return_state);
}
struct DeltaFunction : torch::autograd::Function<DeltaFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                               const Tensor& beta, double scale, const optional<Tensor>& cu, const optional<Tensor>& state,
                               bool return_state) {
    auto [o, last] = delta_below(q, k, v, g, beta, scale, cu, state, return_state);
    ctx->save_for_backward({q, k, v, g, beta, or_none(cu), or_none(state)});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    if (!return_state) ctx->mark_non_differentiable({last});
    return {o, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto& op = op_of<decltype(delta_backward_cuda)>("pla_b200::gated_delta_rule_backward");
    const Tensor d_o = grads[0].defined() ? grads[0] : at::zeros_like(s[2]);
    auto [dq, dk, dv, dg, dbeta, dstate] = op.call(d_o, as_optional(grads[1]), s[0], s[1], s[2], s[3], s[4],
                                                   ctx->saved_data["scale"].toDouble(), as_optional(s[5]), as_optional(s[6]));
    return {dq, dk, dv, dg, dbeta, Tensor(), Tensor(), grad_if(dstate, s[6]), Tensor()};
  }
};
std::tuple<Tensor, Tensor> delta_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                          double scale, const optional<Tensor>& cu, const optional<Tensor>& state,
                                          bool return_state) {
  refuse_tangents(kDelta, q, k, v, g, beta, state);
  if (!wants_gradient(q, k, v, g, beta, state)) return delta_below(q, k, v, g, beta, scale, cu, state, return_state);
  auto r = DeltaFunction::apply(q, k, v, g, beta, scale, cu, state, return_state);
  return {r[0], r[1]};
}

// The single-token forms have no gradient: the call goes through where none is
// asked for, and a result of inputs that ask for one raises when a backward
// pass reaches it.  (An unboxed kernel: the general fallback costs a decoding
// step 1.5 us.)  `state` changes in place, so its version does.
template <typename Sig, typename... Args>
Tensor step_below(const char* name, const Tensor& state, const Args&... args) {
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor out = op_of<Sig>(name).call(args...);
  if (!state.is_inference()) torch::autograd::impl::bump_version(state);
  return out;
}
struct NoGradient : torch::autograd::Function<NoGradient> {
  // what the result depends on
  static Tensor forward(AutogradContext*, const Tensor& result, const Tensor&, const Tensor&, const optional<Tensor>&,
                        const optional<Tensor>&, const optional<Tensor>&) {
    return result;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "pla_b200: the single-token operators have no gradient");
    return {};
  }
};
Tensor causal_step_autograd(const Tensor& x, const Tensor& state, const Tensor& w, const optional<Tensor>& b, bool silu) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && state.requires_grad()),
              "causal_depthwise_step: state is updated in place and must not require grad");
  refuse_tangents("causal_depthwise_step", x, state, w, b);
  Tensor y = step_below<decltype(causal_step_cuda)>("pla_b200::causal_depthwise_step", state, x, state, w, b, silu);
  return wants_gradient(x, w, b) ? NoGradient::apply(y, x, w, b, optional<Tensor>(), optional<Tensor>()) : y;
}
Tensor delta_step_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                           const Tensor& state, double scale) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && state.requires_grad()),
              "gated_delta_rule_step: state is updated in place and must not require grad");
  refuse_tangents("gated_delta_rule_step", q, k, v, g, beta, state);
  Tensor o = step_below<decltype(delta_step_cuda)>("pla_b200::gated_delta_rule_step", state, q, k, v, g, beta, state, scale);
  return wants_gradient(q, k, v, g, beta) ? NoGradient::apply(o, q, k, optional<Tensor>(v), optional<Tensor>(g), optional<Tensor>(beta)) : o;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pla_b200, m) {
  m.def(
      "causal_depthwise(Tensor x, Tensor weight, Tensor? bias, bool silu, Tensor? cu_seqlens, Tensor? state, "
      "bool return_state) -> (Tensor, Tensor)");
  m.def(
      "causal_depthwise_backward(Tensor dy, Tensor? dstate, Tensor x, Tensor weight, Tensor? bias, bool silu, "
      "Tensor? cu_seqlens, Tensor? state) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("causal_depthwise_step(Tensor x, Tensor(a!) state, Tensor weight, Tensor? bias, bool silu) -> Tensor");
  m.def(
      "qk_norm_rotate(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? cos, Tensor? sin, "
      "Tensor? positions, bool l2, float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def(
      "qk_norm_rotate_backward(Tensor dq, Tensor dk, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, "
      "Tensor? cos, Tensor? sin, Tensor? positions, bool l2, float eps, bool interleaved) -> "
      "(Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "gated_delta_rule(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, float scale, Tensor? cu_seqlens, "
      "Tensor? state, bool return_state) -> (Tensor, Tensor)");
  m.def(
      "gated_delta_rule_backward(Tensor d_o, Tensor? dstate, Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, "
      "float scale, Tensor? cu_seqlens, Tensor? state) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "gated_delta_rule_step(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor(a!) state, float scale) -> "
      "Tensor");
}

TORCH_LIBRARY_IMPL(pla_b200, CUDA, m) {
  m.impl("causal_depthwise", &causal_cuda);
  m.impl("causal_depthwise_backward", &causal_backward_cuda);
  m.impl("causal_depthwise_step", &causal_step_cuda);
  m.impl("qk_norm_rotate", &norm_cuda);
  m.impl("qk_norm_rotate_backward", &norm_backward_cuda);
  m.impl("gated_delta_rule", &delta_cuda);
  m.impl("gated_delta_rule_backward", &delta_backward_cuda);
  m.impl("gated_delta_rule_step", &delta_step_cuda);
}

TORCH_LIBRARY_IMPL(pla_b200, Meta, m) {
  m.impl("causal_depthwise", &causal_meta);
  m.impl("causal_depthwise_backward", &causal_backward_meta);
  m.impl("causal_depthwise_step", &causal_step_meta);
  m.impl("qk_norm_rotate", &norm_meta);
  m.impl("qk_norm_rotate_backward", &norm_backward_meta);
  m.impl("gated_delta_rule", &delta_meta);
  m.impl("gated_delta_rule_backward", &delta_backward_meta);
  m.impl("gated_delta_rule_step", &delta_step_meta);
}

TORCH_LIBRARY_IMPL(pla_b200, Autograd, m) {
  m.impl("causal_depthwise", &causal_autograd);
  m.impl("qk_norm_rotate", &norm_autograd);
  m.impl("gated_delta_rule", &delta_autograd);
  m.impl("causal_depthwise_step", &causal_step_autograd);
  m.impl("gated_delta_rule_step", &delta_step_autograd);
  for (const char* op : {"causal_depthwise_backward", "qk_norm_rotate_backward", "gated_delta_rule_backward"})
    m.impl(op, torch::autograd::autogradNotImplementedFallback());
}
