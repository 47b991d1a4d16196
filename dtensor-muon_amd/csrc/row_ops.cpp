// The row operators (include/muon_amd.h) as torch operators of namespace muonium_amd: schemas,
// device implementations on the C ABI, and their gradients.
//
// A training step calls these between a few large products, often on small tensors, where the
// host's time is what counts: as Python autograd Functions around ctypes calls a forward and
// backward pass took 104 to 173 us of it, here 61 (token log probabilities) to 95 (queries and keys,
// with two weights), where a multiplication with its gradient takes 45.
// Arguments are checked in muonium_amd.kernels; the C ABI refuses what would not be safe.
#include <ATen/DeviceGuard.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include "../../include/muon_amd.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::tuple<Tensor, Tensor> Tensor2;
typedef std::tuple<Tensor, Tensor, Tensor> Tensor3;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor> Tensor4;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> Tensor6;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MUON_DT_F32;
    case at::kBFloat16: return MUON_DT_BF16;
    case at::kHalf: return MUON_DT_F16;
    default: TORCH_CHECK_TYPE(false, "muonium_amd: unsupported dtype ", t.scalar_type());
  }
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == MUON_OK, what, " failed (status ", rc, "): ", muon_amd_last_error());
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

template <typename T = void>
T* ptr(const Tensor& t) {
  return (T*)t.data_ptr();
}
template <typename T = void>
T* ptr(const optional<Tensor>& t) {
  return t && t->defined() ? (T*)t->data_ptr() : nullptr;
}

Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, like.options().dtype(type));
}
// Contiguous, whatever the strides of `t`.
Tensor fresh(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
// Scratch from torch's allocator on the current stream: free for reuse there once the launches that
// read it are enqueued.
Tensor scratch(const Tensor& like, int64_t bytes) { return empty(like, {bytes}, at::kByte); }

Tensor unit_last(const Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// What a kernel takes by a plain pointer, contiguous: of one type, so many values, beside `like`.
Tensor plain(const Tensor& t, const Tensor& like, at::ScalarType type, int64_t numel,
             const char* name) {
  TORCH_CHECK(t.scalar_type() == type && t.numel() == numel && t.device() == like.device(),
              "muonium_amd: ", name, " has to be ", numel, " values of ", type, " on ",
              like.device(), "; got ", t.numel(), " of ", t.scalar_type(), " on ", t.device());
  return t.contiguous();
}
optional<Tensor> plain(const optional<Tensor>& t, const Tensor& like, at::ScalarType type,
                       int64_t numel, const char* name) {
  if (!t || !t->defined()) return std::nullopt;
  return plain(*t, like, type, numel, name);
}
// Rows of logits with a contiguous last dimension.
Tensor rows_of(const Tensor& logits) {
  TORCH_CHECK(logits.dim() == 2, "muonium_amd: logits have to be (rows, values); got ",
              logits.sizes());
  return unit_last(logits);
}

// ---- queries and keys -------------------------------------------------------------------

struct QkArgs {
  int64_t strides[12];
  int w_dtype = 0, pos_bits = 64;
  int64_t table_len = 0, pos_stride = 0, batch, tokens, dim, rotary = 0;

  QkArgs(const Tensor& q, const Tensor& k, const optional<Tensor>& qw, const optional<Tensor>& kw,
         const optional<Tensor>& cos, const optional<Tensor>& pos) {
    TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim() && k.size(0) == q.size(0) &&
                    k.size(-3) == q.size(-3) && k.size(-1) == q.size(-1) &&
                    k.scalar_type() == q.scalar_type() && k.device() == q.device() &&
                    (!qw || !kw || qw->scalar_type() == kw->scalar_type()),
                "muonium_amd: q and k, or their weights, do not belong together: ", q.sizes(),
                " and ", k.sizes());
    put(q, 0);
    put(k, 3);
    if (qw) w_dtype = dtype_code(*qw);
    else if (kw) w_dtype = dtype_code(*kw);
    if (cos) {
      table_len = cos->size(0);
      rotary = 2 * cos->size(1);
    }
    if (pos) {
      pos_bits = pos->scalar_type() == at::kLong ? 64 : 32;
      pos_stride = pos->dim() == 2 ? pos->stride(0) : 0;
    }
    batch = q.dim() == 4 ? q.size(0) : 1;
    tokens = q.size(-3);
    dim = q.size(-1);
  }
  void put(const Tensor& t, int at) {
    strides[at] = t.dim() == 4 ? t.stride(0) : 0;
    strides[at + 1] = t.stride(-3);
    strides[at + 2] = t.stride(-2);
  }
};

// The weights, tables and positions of a call, as the kernels take them.
struct QkRest {
  optional<Tensor> qw, kw, cos, sin, pos;

  QkRest(const Tensor& q, const optional<Tensor>& qw_, const optional<Tensor>& kw_,
         const optional<Tensor>& cos_, const optional<Tensor>& sin_, const optional<Tensor>& pos_) {
    if (qw_) qw = plain(qw_, q, qw_->scalar_type(), q.size(-1), "a weight");
    if (kw_) kw = plain(kw_, q, kw_->scalar_type(), q.size(-1), "a weight");
    if (cos_) {
      TORCH_CHECK(sin_ && cos_->dim() == 2, "muonium_amd: cos and sin are two tables");
      cos = plain(cos_, q, at::kFloat, cos_->numel(), "cos");
      sin = plain(sin_, q, at::kFloat, cos_->numel(), "sin");
    }
    if (pos_) {
      const bool each = pos_->dim() == 2;
      const int64_t batch = q.dim() == 4 ? q.size(0) : 1;
      TORCH_CHECK((pos_->scalar_type() == at::kLong || pos_->scalar_type() == at::kInt) &&
                      pos_->dim() >= 1 && pos_->dim() <= 2 && pos_->device() == q.device() &&
                      pos_->size(-1) == q.size(-3) && (!each || pos_->size(0) == batch),
                  "muonium_amd: positions have to be int32 or int64, (tokens,) or (batch, tokens)");
      pos = unit_last(*pos_);
    }
  }
};

Tensor2 qk_forward(const Tensor& q_, const Tensor& k_, const optional<Tensor>& qw_,
                   const optional<Tensor>& kw_, const optional<Tensor>& cos_,
                   const optional<Tensor>& sin_, const optional<Tensor>& pos_, double eps,
                   bool interleaved) {
  const at::DeviceGuard guard(q_.device());
  const Tensor q = unit_last(q_), k = unit_last(k_);
  const auto [qw, kw, cos, sin, pos] = QkRest(q, qw_, kw_, cos_, sin_, pos_);
  Tensor q_out = fresh(q), k_out = fresh(k);
  const QkArgs a(q, k, qw, kw, cos, pos);
  check(muon_qk_norm_rope(ptr(q), ptr(k), a.strides, ptr(qw), ptr(kw), a.w_dtype, ptr<float>(cos),
                          ptr<float>(sin), a.table_len, ptr(pos), a.pos_bits, a.pos_stride,
                          ptr(q_out), ptr(k_out), dtype_code(q), a.batch, a.tokens, q.size(-2),
                          k.size(-2), a.dim, a.rotary, interleaved, (float)eps, stream_of(q)),
        "muon_qk_norm_rope");
  return {q_out, k_out};
}

Tensor4 qk_backward(const Tensor& dq_out, const Tensor& dk_out, const Tensor& q_, const Tensor& k_,
                    const optional<Tensor>& qw_, const optional<Tensor>& kw_,
                    const optional<Tensor>& cos_, const optional<Tensor>& sin_,
                    const optional<Tensor>& pos_, double eps, bool interleaved) {
  const at::DeviceGuard guard(q_.device());
  const Tensor q = unit_last(q_), k = unit_last(k_);
  const auto [qw, kw, cos, sin, pos] = QkRest(q, qw_, kw_, cos_, sin_, pos_);
  TORCH_CHECK(dq_out.sizes() == q.sizes() && dk_out.sizes() == k.sizes() &&
                  dq_out.scalar_type() == q.scalar_type() &&
                  dk_out.scalar_type() == q.scalar_type() && dq_out.device() == q.device() &&
                  dk_out.device() == q.device(),
              "muonium_amd: gradients of q and k are not like them");
  const Tensor gq = unit_last(dq_out), gk = unit_last(dk_out);
  Tensor dq = fresh(q), dk = fresh(k);
  Tensor dqw = qw ? fresh(*qw) : empty(q, {0}, q.scalar_type());
  Tensor dkw = kw ? fresh(*kw) : empty(k, {0}, k.scalar_type());
  QkArgs a(q, k, qw, kw, cos, pos);
  a.put(gq, 6);
  a.put(gk, 9);
  Tensor ws;
  if (qw || kw) ws = scratch(q, muon_qk_norm_rope_workspace_bytes(a.dim));
  check(muon_qk_norm_rope_backward(
            ptr(q), ptr(k), ptr(gq), ptr(gk), a.strides, ptr(qw), ptr(kw), a.w_dtype,
            ptr<float>(cos), ptr<float>(sin), a.table_len, ptr(pos), a.pos_bits, a.pos_stride,
            ptr(dq), ptr(dk), qw ? ptr(dqw) : nullptr, kw ? ptr(dkw) : nullptr,
            ws.defined() ? ptr(ws) : nullptr, dtype_code(q), a.batch, a.tokens, q.size(-2),
            k.size(-2), a.dim, a.rotary, interleaved, (float)eps, stream_of(q)),
        "muon_qk_norm_rope_backward");
  return {dq, dk, dqw, dkw};
}

// ---- routing ----------------------------------------------------------------------------

Tensor6 route_forward(const Tensor& logits_, int64_t top, const optional<Tensor>& mask_,
                      bool normalize) {
  const at::DeviceGuard guard(logits_.device());
  const Tensor logits = rows_of(logits_);
  const int64_t n = logits.size(0), e = logits.size(1);
  const auto mask = plain(mask_, logits, at::kBool, n, "the mask");
  Tensor gates = empty(logits, {n, top}, at::kFloat), experts = empty(logits, {n, top}, at::kLong);
  Tensor counts = empty(logits, {e}, at::kLong);
  Tensor balance = empty(logits, {}, at::kFloat), zloss = empty(logits, {}, at::kFloat);
  Tensor kept = empty(logits, {}, at::kFloat);
  Tensor ws = scratch(logits, muon_route_workspace_bytes(n, e));
  check(muon_route(ptr(logits), dtype_code(logits), logits.stride(0), n, e, top, normalize,
                   ptr(mask), ptr<float>(gates), ptr<int64_t>(experts), ptr<int64_t>(counts),
                   ptr<float>(balance), ptr<float>(zloss), ptr<float>(kept), ptr(ws),
                   stream_of(logits)),
        "muon_route");
  return {gates, experts, counts, balance, zloss, kept};
}

Tensor route_backward(const optional<Tensor>& dgates, const optional<Tensor>& dbalance,
                      const optional<Tensor>& dzloss, const Tensor& logits_,
                      const optional<Tensor>& mask_, const Tensor& experts_, const Tensor& counts_,
                      const Tensor& kept_, bool normalize) {
  const at::DeviceGuard guard(logits_.device());
  const Tensor logits = rows_of(logits_);
  const int64_t n = logits.size(0), e = logits.size(1), top = experts_.size(-1);
  const auto mask = plain(mask_, logits, at::kBool, n, "the mask");
  const Tensor experts = plain(experts_, logits, at::kLong, n * top, "the experts");
  const Tensor counts = plain(counts_, logits, at::kLong, e, "the counts");
  const Tensor kept = plain(kept_, logits, at::kFloat, 1, "the token count");
  const auto dg = plain(dgates, logits, at::kFloat, n * top, "the gates' gradient");
  const auto db = plain(dbalance, logits, at::kFloat, 1, "the balance loss's gradient");
  const auto dz = plain(dzloss, logits, at::kFloat, 1, "the z loss's gradient");
  Tensor dlogits = fresh(logits);
  check(muon_route_backward(ptr(logits), dtype_code(logits), logits.stride(0), n, e, top,
                            normalize, ptr(mask), ptr<int64_t>(experts), ptr<int64_t>(counts),
                            ptr<float>(kept), ptr<float>(dg), ptr<float>(db), ptr<float>(dz),
                            ptr(dlogits), stream_of(logits)),
        "muon_route_backward");
  return dlogits;
}

// ---- log probabilities and the policy loss --------------------------------------------------

Tensor logp_scratch(const Tensor& logits) {
  return scratch(logits, muon_token_logprobs_workspace_bytes(dtype_code(logits), logits.size(0),
                                                             logits.size(1)));
}

Tensor2 logp_forward(const Tensor& logits_, const Tensor& tokens_, double temperature, bool keep) {
  const at::DeviceGuard guard(logits_.device());
  const Tensor logits = rows_of(logits_);
  const int64_t n = logits.size(0);
  const Tensor tokens = plain(tokens_, logits, at::kLong, n, "the tokens");
  Tensor logp = empty(logits, {n}, at::kFloat), stats = empty(logits, {keep ? 2 * n : 0}, at::kFloat);
  Tensor ws = logp_scratch(logits);
  check(muon_token_logprobs(ptr(logits), dtype_code(logits), logits.stride(0), n, logits.size(1),
                            ptr<int64_t>(tokens), (float)temperature, ptr<float>(logp),
                            keep ? ptr<float>(stats) : nullptr, ptr(ws), stream_of(logits)),
        "muon_token_logprobs");
  return {logp, stats};
}

Tensor logp_gradient(const Tensor& dlogp, const float* scale, const Tensor& logits,
                     const Tensor& tokens_, const float* stats, double temperature) {
  const Tensor tokens = plain(tokens_, logits, at::kLong, logits.size(0), "the tokens");
  const Tensor g = plain(dlogp, logits, at::kFloat, logits.size(0), "the gradient");
  Tensor dlogits = fresh(logits);
  check(muon_token_logprobs_backward(ptr(logits), dtype_code(logits), logits.stride(0),
                                     logits.size(0), logits.size(1), ptr<int64_t>(tokens),
                                     (float)temperature, stats, ptr<float>(g), scale, ptr(dlogits),
                                     stream_of(logits)),
        "muon_token_logprobs_backward");
  return dlogits;
}

Tensor logp_backward(const Tensor& dlogp, const Tensor& logits, const Tensor& tokens,
                     const Tensor& stats, double temperature) {
  const at::DeviceGuard guard(logits.device());
  const Tensor kept = plain(stats, logits, at::kFloat, 2 * logits.size(0), "the statistics");
  return logp_gradient(dlogp, nullptr, rows_of(logits), tokens, ptr<float>(kept), temperature);
}

// rows: per row the term, and (keep) the slope and the two statistics that a later gradient
// needs; dlogits: the gradient for a loss gradient of 1 (one_pass), else empty.
Tensor4 policy_forward(const Tensor& logits_, const Tensor& tokens_, const Tensor& old_,
                       const Tensor& advantages_, const Tensor& weights_,
                       const optional<Tensor>& ref_, double clip_low, double clip_high, double kl_coef, double temperature,
                       bool keep, bool one_pass) {
  const at::DeviceGuard guard(logits_.device());
  const Tensor logits = rows_of(logits_);
  const int64_t n = logits.size(0);
  const Tensor tokens = plain(tokens_, logits, at::kLong, n, "the tokens");
  const Tensor old = plain(old_, logits, at::kFloat, n, "the old log probabilities");
  const Tensor advantages = plain(advantages_, logits, at::kFloat, n, "the advantages");
  const Tensor weights = plain(weights_, logits, at::kFloat, n, "the weights");
  const auto ref = plain(ref_, logits, at::kFloat, n, "the reference log probabilities");
  Tensor loss = empty(logits, {}, at::kFloat), logp = empty(logits, {n}, at::kFloat);
  Tensor rows = empty(logits, {keep ? 4 : 1, n}, at::kFloat);
  Tensor dlogits = one_pass ? fresh(logits) : empty(logits, {0}, logits.scalar_type());
  // the ABI takes a null gradient as none asked for: what has no values is none
  const bool made = one_pass && dlogits.numel();
  Tensor ws = made ? Tensor() : logp_scratch(logits);
  float* r = ptr<float>(rows);
  check(muon_policy_loss(ptr(logits), dtype_code(logits), logits.stride(0), n, logits.size(1),
                         ptr<int64_t>(tokens), ptr<float>(old), ptr<float>(advantages),
                         ptr<float>(weights), ptr<float>(ref), (float)clip_low, (float)clip_high,
                         (float)kl_coef, (float)temperature, ptr<float>(loss), ptr<float>(logp),
                         r, keep ? r + 2 * n : nullptr, keep ? r + n : nullptr,
                         made ? ptr(dlogits) : nullptr, made ? nullptr : ptr(ws),
                         stream_of(logits)),
        "muon_policy_loss");
  return {loss, logp, rows, dlogits};
}

Tensor policy_backward(const Tensor& dloss, const Tensor& logits, const Tensor& tokens,
                       const Tensor& rows, double temperature) {
  const at::DeviceGuard guard(logits.device());
  const int64_t n = logits.size(0);
  const Tensor kept = plain(rows, logits, at::kFloat, 4 * n, "the rows' values").view({4, n});
  const Tensor scale = plain(dloss, logits, at::kFloat, 1, "the loss's gradient");
  return logp_gradient(kept.select(0, 1), ptr<float>(scale), rows_of(logits), tokens,
                       ptr<float>(kept) + 2 * n, temperature);
}

// dlogits, as policy_forward's one pass made it of these logits, for a loss gradient of dloss.
void policy_rescale(const Tensor& dlogits, const Tensor& dloss, const Tensor& logits_,
                    const Tensor& tokens_, const Tensor& rows, double temperature) {
  const at::DeviceGuard guard(logits_.device());
  const Tensor logits = rows_of(logits_);
  const int64_t n = logits.size(0);
  TORCH_CHECK(dlogits.sizes() == logits.sizes() && dlogits.is_contiguous() &&
                  dlogits.scalar_type() == logits.scalar_type() &&
                  dlogits.device() == logits.device(),
              "muonium_amd: the gradient is not like its logits");
  const Tensor tokens = plain(tokens_, logits, at::kLong, n, "the tokens");
  const Tensor kept = plain(rows, logits, at::kFloat, 4 * n, "the rows' values");
  const Tensor scale = plain(dloss, logits, at::kFloat, 1, "the loss's gradient");
  const float* r = ptr<float>(kept);
  check(muon_policy_loss_rescale(ptr(logits), dtype_code(logits), logits.stride(0), n,
                                 logits.size(1), ptr<int64_t>(tokens), (float)temperature,
                                 r + 2 * n, r + n, ptr<float>(scale), ptr(dlogits),
                                 stream_of(logits)),
        "muon_policy_loss_rescale");
}

// ---- experts ------------------------------------------------------------------------------

Tensor2 order_forward(const Tensor& experts, int64_t nexperts) {
  const at::DeviceGuard guard(experts.device());
  const int64_t n = experts.numel();
  const Tensor ids = plain(experts, experts, at::kLong, n, "the experts");
  Tensor slots = empty(experts, experts.sizes(), at::kInt);
  Tensor offsets = empty(experts, {nexperts + 1}, at::kInt);
  const int64_t bytes = muon_expert_order_workspace_bytes(n, nexperts);
  Tensor ws = bytes ? scratch(experts, bytes) : Tensor();
  check(muon_expert_order(ptr<int64_t>(ids), n, nexperts, ptr<int32_t>(slots), ptr<int32_t>(offsets),
                          bytes ? ptr(ws) : nullptr, stream_of(experts)),
        "muon_expert_order");
  return {slots, offsets};
}

// (tokens, choices) slots of what is routed.
Tensor slots_of(const Tensor& slots, const Tensor& like) {
  TORCH_CHECK(slots.dim() == 2, "muonium_amd: slots have to be (tokens, choices); got ", slots.sizes());
  return plain(slots, like, at::kInt, slots.numel(), "the slots");
}

Tensor dispatch_forward(const Tensor& x_, const Tensor& slots_) {
  const at::DeviceGuard guard(x_.device());
  const Tensor x = rows_of(x_), slots = slots_of(slots_, x_);
  TORCH_CHECK(slots.size(0) == x.size(0), "muonium_amd: slots of ", slots.size(0), " tokens for ",
              x.size(0));
  Tensor rows = empty(x, {slots.numel(), x.size(1)}, x.scalar_type());
  check(muon_dispatch(ptr(x), dtype_code(x), x.stride(0), x.size(0), slots.size(1), x.size(1),
                      ptr<int32_t>(slots), ptr(rows), stream_of(x)),
        "muon_dispatch");
  return rows;
}

Tensor combine_forward(const Tensor& rows_, const Tensor& slots_, const optional<Tensor>& gates_) {
  const at::DeviceGuard guard(rows_.device());
  const Tensor rows = rows_of(rows_), slots = slots_of(slots_, rows_);
  TORCH_CHECK(rows.size(0) == slots.numel(), "muonium_amd: ", rows.size(0), " rows for ",
              slots.numel(), " choices");
  const auto gates = plain(gates_, rows, at::kFloat, slots.numel(), "the gates");
  Tensor y = empty(rows, {slots.size(0), rows.size(1)}, rows.scalar_type());
  check(muon_combine(ptr(rows), dtype_code(rows), rows.stride(0), slots.size(0), slots.size(1),
                     rows.size(1), ptr<int32_t>(slots), ptr<float>(gates), ptr(y), stream_of(rows)),
        "muon_combine");
  return y;
}

// Gradients that are not asked for come back empty; the rows are needed for the gates' alone.
Tensor2 combine_backward(const Tensor& dy_, const optional<Tensor>& rows_, const Tensor& slots_,
                         const Tensor& gates_, bool rows_wanted, bool gates_wanted) {
  const at::DeviceGuard guard(dy_.device());
  const Tensor dy = rows_of(dy_), slots = slots_of(slots_, dy_);
  TORCH_CHECK(dy.size(0) == slots.size(0), "muonium_amd: the gradient is not like its output");
  const Tensor gates = plain(gates_, dy, at::kFloat, slots.numel(), "the gates");
  Tensor rows;
  if (gates_wanted) {
    TORCH_CHECK(rows_ && rows_->defined(), "muonium_amd: the gates' gradient takes the rows");
    rows = rows_of(*rows_);
    TORCH_CHECK(rows.size(0) == slots.numel() && dy.size(1) == rows.size(1) &&
                    dy.scalar_type() == rows.scalar_type() && dy.device() == rows.device(),
                "muonium_amd: the gradient is not like its output");
  }
  Tensor drows = empty(dy, {rows_wanted ? slots.numel() : 0, dy.size(1)}, dy.scalar_type());
  Tensor dgates = gates_wanted ? empty(dy, slots.sizes(), at::kFloat) : empty(dy, {0}, at::kFloat);
  check(muon_combine_backward(ptr(dy), dy.stride(0), gates_wanted ? ptr(rows) : nullptr,
                              gates_wanted ? rows.stride(0) : 0, dtype_code(dy), slots.size(0),
                              slots.size(1), dy.size(1), ptr<int32_t>(slots), ptr<float>(gates),
                              rows_wanted ? ptr(drows) : nullptr,
                              gates_wanted ? ptr<float>(dgates) : nullptr, stream_of(dy)),
        "muon_combine_backward");
  if (!rows_wanted) drows = empty(dy, {0}, dy.scalar_type());
  return {drows, dgates};
}

// The weights and offsets of a product, and what belongs together.
struct Experts {
  Tensor weight, offsets;
  int64_t n, out, in;

  Experts(const Tensor& like, const Tensor& weight_, const Tensor& offsets_) {
    TORCH_CHECK(weight_.dim() == 3 && weight_.scalar_type() == like.scalar_type() &&
                    weight_.device() == like.device(),
                "muonium_amd: weights have to be (experts, out, in) of the rows' type beside them");
    weight = weight_.contiguous();
    n = weight.size(0);
    out = weight.size(1);
    in = weight.size(2);
    offsets = plain(offsets_, like, at::kInt, n + 1, "the offsets");
  }
};

Tensor linear_forward(const Tensor& rows_, const Tensor& weight, const Tensor& offsets) {
  const at::DeviceGuard guard(rows_.device());
  const Tensor rows = rows_of(rows_);
  const Experts e(rows, weight, offsets);
  TORCH_CHECK(rows.size(1) == e.in, "muonium_amd: rows of ", rows.size(1), " values for weights of ", e.in);
  Tensor y = empty(rows, {rows.size(0), e.out}, rows.scalar_type());
  check(muon_expert_linear(ptr(rows), dtype_code(rows), rows.stride(0), rows.size(0), e.n, e.out, e.in,
                           ptr(e.weight), ptr<int32_t>(e.offsets), ptr(y), stream_of(rows)),
        "muon_expert_linear");
  return y;
}

Tensor linear_backward_rows(const Tensor& dy_, const Tensor& weight, const Tensor& offsets) {
  const at::DeviceGuard guard(dy_.device());
  const Tensor dy = rows_of(dy_);
  const Experts e(dy, weight, offsets);
  TORCH_CHECK(dy.size(1) == e.out, "muonium_amd: the gradient is not like its output");
  Tensor drows = empty(dy, {dy.size(0), e.in}, dy.scalar_type());
  check(muon_expert_linear_backward_rows(ptr(dy), dtype_code(dy), dy.stride(0), dy.size(0), e.n, e.out,
                                         e.in, ptr(e.weight), ptr<int32_t>(e.offsets), ptr(drows),
                                         stream_of(dy)),
        "muon_expert_linear_backward_rows");
  return drows;
}

Tensor linear_backward_weight(const Tensor& dy_, const Tensor& rows_, const Tensor& offsets_) {
  const at::DeviceGuard guard(dy_.device());
  const Tensor dy = rows_of(dy_), rows = rows_of(rows_);
  TORCH_CHECK(dy.size(0) == rows.size(0) && dy.scalar_type() == rows.scalar_type() &&
                  dy.device() == rows.device() && offsets_.numel() > 1,
              "muonium_amd: the gradient is not like its output");
  const int64_t n = offsets_.numel() - 1;
  const Tensor offsets = plain(offsets_, rows, at::kInt, n + 1, "the offsets");
  Tensor dweight = empty(rows, {n, dy.size(1), rows.size(1)}, rows.scalar_type());
  check(muon_expert_linear_backward_weight(ptr(dy), dtype_code(dy), dy.stride(0), ptr(rows),
                                           rows.stride(0), rows.size(0), n, dy.size(1), rows.size(1),
                                           ptr<int32_t>(offsets), ptr(dweight), stream_of(rows)),
        "muon_expert_linear_backward_weight");
  return dweight;
}

// ---- AdamW --------------------------------------------------------------------------------

// One step of all tensors, on one device and of one type; without scales the moments are fp32.
void adamw(at::TensorList params, at::TensorList grads, at::TensorList avgs, at::TensorList sqs,
           at::TensorList avg_scales, at::TensorList sq_scales, at::TensorList steps, int64_t block,
           double lr, double beta1, double beta2, double eps, double weight_decay, bool maximize) {
  const size_t n = params.size();
  const bool fp8 = block != 0;
  TORCH_CHECK(grads.size() == n && avgs.size() == n && sqs.size() == n && steps.size() == n &&
                  avg_scales.size() == (fp8 ? n : 0) && sq_scales.size() == (fp8 ? n : 0),
              "muonium_amd: adamw_ takes one gradient, moment and step for each parameter");
  if (!n) return;
  const at::DeviceGuard guard(params[0].device());
  std::vector<MuonAdamTensor> table(n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor& p = params[i];
    const int64_t numel = p.numel();
    TORCH_CHECK(p.scalar_type() == params[0].scalar_type() && p.device() == params[0].device() &&
                    p.is_non_overlapping_and_dense(),
                "muonium_amd: adamw_'s parameters have to be dense, of one type and on one device");
    TORCH_CHECK(grads[i].scalar_type() == p.scalar_type() && grads[i].device() == p.device() &&
                    grads[i].sizes() == p.sizes() && (numel <= 1 || grads[i].strides() == p.strides()),
                "muonium_amd: a gradient is not laid out like its parameter");
    const auto held = [&](const Tensor& t, at::ScalarType type, int64_t count, const char* name) {
      TORCH_CHECK(t.scalar_type() == type && t.numel() == count && t.device() == p.device() &&
                      t.is_non_overlapping_and_dense(),
                  "muonium_amd: ", name, " has to be ", count, " dense values of ", type, " on ", p.device());
      return t.data_ptr();
    };
    table[i] = {p.data_ptr(), grads[i].data_ptr(), held(avgs[i], fp8 ? at::kByte : at::kFloat, numel, "a mean"),
                held(sqs[i], fp8 ? at::kByte : at::kFloat, numel, "a mean square"),
                fp8 ? (float*)held(avg_scales[i], at::kFloat, numel / block, "a scale") : nullptr,
                fp8 ? (float*)held(sq_scales[i], at::kFloat, numel / block, "a scale") : nullptr,
                (float*)held(steps[i], at::kFloat, 1, "a step"), numel};
  }
  Tensor ws = scratch(params[0], muon_adamw_workspace_bytes((int64_t)n));
  check(muon_adamw((int64_t)n, table.data(), dtype_code(params[0]), block, lr, beta1, beta2, eps,
                   weight_decay, maximize, ptr(ws), stream_of(params[0])),
        "muon_adamw");
  // what saved a parameter for its backward pass finds it changed
  for (const Tensor& p : params)
    if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
}

// ---- gradients --------------------------------------------------------------------------

#define OP(name, impl)                                                                \
  [] {                                                                                \
    static auto h = c10::Dispatcher::singleton()                                      \
                        .findSchemaOrThrow("muonium_amd::" name, "")                  \
                        .typed<decltype(impl)>();                                     \
    return h;                                                                         \
  }()

bool needs(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool needs(const optional<Tensor>& t) { return t && needs(*t); }
template <typename... T>
bool any_needs(const T&... t) {
  return at::GradMode::is_enabled() && (needs(t) || ...);
}

// There is no forward-mode derivative. Below autograd a dual tensor's tangent would be dropped and
// the result pass for a constant; torch itself refuses only where a gradient is asked for too.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const optional<Tensor>& t) { return t && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...),
                              "muonium_amd's row operators have no forward-mode derivative");
}

// Whether somebody records or replaces the operators that run: a tracer or a checkpoint that keeps
// results, by a dispatch mode (over plain tensors too), or a tensor subclass. What it sees has to be
// all that happens.
bool watched() { return c10::impl::TorchDispatchModeTLS::any_modes_set(); }
bool watched(const Tensor& t) { return watched() || t.key_set().has(c10::DispatchKey::Python); }

// Whether launches beside `t` are being recorded into a graph.
bool captured(const Tensor& t) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  C10_HIP_CHECK(hipStreamIsCapturing((hipStream_t)stream_of(t), &status));
  return status != hipStreamCaptureStatusNone;
}

Tensor or_undefined(const optional<Tensor>& t) { return t ? *t : Tensor(); }
optional<Tensor> or_none(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

// Results of a backward pass that is itself differentiated through (create_graph): there is no
// second derivative, and asking for one is an error.
variable_list once(variable_list results, const variable_list& inputs) {
  if (!at::GradMode::is_enabled()) return results;
  bool any = false;
  for (const auto& t : inputs) any = any || needs(t);
  if (!any) return results;
  variable_list outs, marked;
  for (auto& t : results)
    if (t.defined()) marked.push_back(t.detach().set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "muonium_amd's row operators have no second derivative", (int64_t)marked.size());
  marked = (*error)(std::move(marked));
  size_t i = 0;
  for (auto& t : results) outs.push_back(t.defined() ? marked[i++] : Tensor());
  return outs;
}

struct QkFunction : torch::autograd::Function<QkFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const optional<Tensor>& qw, const optional<Tensor>& kw,
                               const optional<Tensor>& cos, const optional<Tensor>& sin,
                               const optional<Tensor>& pos, double eps, bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [a, b] = OP("qk_norm_rope", qk_forward)
                      .call(q, k, qw, kw, cos, sin, pos, eps, interleaved);
    ctx->save_for_backward({q, k, or_undefined(qw), or_undefined(kw), or_undefined(cos),
                            or_undefined(sin), or_undefined(pos)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return {a, b};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto s = ctx->get_saved_variables();
    Tensor4 g;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      g = OP("qk_norm_rope_backward", qk_backward)
              .call(grads[0], grads[1], s[0], s[1], or_none(s[2]), or_none(s[3]), or_none(s[4]),
                    or_none(s[5]), or_none(s[6]), ctx->saved_data["eps"].toDouble(),
                    ctx->saved_data["interleaved"].toBool());
    }
    variable_list in = s;
    in.insert(in.end(), grads.begin(), grads.end());
    return once({std::get<0>(g), std::get<1>(g), s[2].defined() ? std::get<2>(g) : Tensor(),
                 s[3].defined() ? std::get<3>(g) : Tensor(), Tensor(), Tensor(), Tensor(), Tensor(),
                 Tensor()}, in);
  }
};

Tensor2 qk_autograd(const Tensor& q, const Tensor& k, const optional<Tensor>& qw,
                    const optional<Tensor>& kw, const optional<Tensor>& cos,
                    const optional<Tensor>& sin, const optional<Tensor>& pos, double eps,
                    bool interleaved) {
  refuse_tangents(q, k, qw, kw, cos, sin);
  if (any_needs(q, k, qw, kw)) {
    auto out = QkFunction::apply(q, k, qw, kw, cos, sin, pos, eps, interleaved);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("qk_norm_rope", qk_forward).call(q, k, qw, kw, cos, sin, pos, eps, interleaved);
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t top,
                               const optional<Tensor>& mask, bool normalize) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [gates, experts, counts, balance, zloss, kept] =
        OP("route", route_forward).call(logits, top, mask, normalize);
    ctx->save_for_backward({logits, or_undefined(mask), experts, counts, kept});
    ctx->saved_data["normalize"] = normalize;
    ctx->mark_non_differentiable({experts, counts, kept});
    ctx->set_materialize_grads(false);
    return {gates, experts, counts, balance, zloss, kept};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto s = ctx->get_saved_variables();
    Tensor d;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      d = OP("route_backward", route_backward)
              .call(or_none(grads[0]), or_none(grads[3]), or_none(grads[4]), s[0], or_none(s[1]),
                    s[2], s[3], s[4], ctx->saved_data["normalize"].toBool());
    }
    return once({d, Tensor(), Tensor(), Tensor()}, {s[0], grads[0], grads[3], grads[4]});
  }
};

Tensor6 route_autograd(const Tensor& logits, int64_t top, const optional<Tensor>& mask,
                       bool normalize) {
  refuse_tangents(logits);
  if (any_needs(logits)) {
    auto o = RouteFunction::apply(logits, top, mask, normalize);
    return {o[0], o[1], o[2], o[3], o[4], o[5]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("route", route_forward).call(logits, top, mask, normalize);
}

struct LogpFunction : torch::autograd::Function<LogpFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                               double temperature, bool keep) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [logp, stats] = OP("token_logprobs", logp_forward).call(logits, tokens, temperature, true);
    ctx->save_for_backward({logits, tokens, stats});
    ctx->saved_data["temperature"] = temperature;
    if (!keep) stats = empty(logits, {0}, at::kFloat);  // kept for the backward pass alone
    ctx->mark_non_differentiable({stats});
    return {logp, stats};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto s = ctx->get_saved_variables();
    Tensor d;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      d = OP("token_logprobs_backward", logp_backward)
              .call(grads[0], s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble());
    }
    return once({d, Tensor(), Tensor(), Tensor()}, {s[0], grads[0]});
  }
};

Tensor2 logp_autograd(const Tensor& logits, const Tensor& tokens, double temperature, bool keep) {
  refuse_tangents(logits);
  if (any_needs(logits)) {
    auto o = LogpFunction::apply(logits, tokens, temperature, keep);
    return {o[0], o[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("token_logprobs", logp_forward).call(logits, tokens, temperature, keep);
}

struct PolicyFunction : torch::autograd::Function<PolicyFunction> {
  // Whether a gradient of the forward pass waits for the backward pass, and where it was made.
  enum Made { NO, EAGERLY, IN_GRAPH };
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                               const Tensor& old, const Tensor& advantages, const Tensor& weights,
                               const optional<Tensor>& ref, double clip_low, double clip_high,
                               double kl_coef, double temperature, bool keep, bool one_pass) {
    at::AutoDispatchBelowADInplaceOrView below;
    // A gradient made here is the caller's (one_pass), or kept for the backward pass alone. Who
    // watches sees the form whose gradient is an operation of its own on what is saved.
    const bool ours = !one_pass && !watched(logits) &&
                      muon_policy_loss_one_pass(dtype_code(logits), logits.size(1));
    auto [loss, logp, rows, dlogits] =
        OP("policy_loss", policy_forward)
            .call(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
                  temperature, true, one_pass || ours);
    // the gradient too is a saved tensor: hooks move or drop it like the logits
    ctx->save_for_backward({logits, tokens, rows, ours ? dlogits : Tensor()});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["made"] = (int64_t)(!ours ? NO : captured(logits) ? IN_GRAPH : EAGERLY);
    if (ours) dlogits = empty(logits, {0}, logits.scalar_type());
    if (!keep) rows = rows.narrow(0, 0, 1);
    ctx->mark_non_differentiable({logp, rows, dlogits});
    ctx->set_materialize_grads(false);
    return {loss, logp, rows, dlogits};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list none(12);
    if (!grads[0].defined()) return none;
    const auto s = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      // The gradient of the forward pass is handed over once; a second backward pass through the same
      // graph makes its own from the logits, as does one that may run again without its forward
      // pass: one that is watched, or captured alone. What is handed over has a version of its own:
      // what its taker does to it is no change of what this graph saved.
      auto& made = ctx->saved_data["made"];
      if (made.toInt() != NO && !watched() && (made.toInt() == IN_GRAPH || !captured(s[0]))) {
        made = (int64_t)NO;
        none[0] = s[3].variable_data();
        OP("policy_loss_rescale_", policy_rescale)
            .call(none[0], grads[0], s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble());
      } else {
        none[0] = OP("policy_loss_backward", policy_backward)
                      .call(grads[0], s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble());
      }
    }
    return once(none, {s[0], grads[0]});
  }
};

Tensor4 policy_autograd(const Tensor& logits, const Tensor& tokens, const Tensor& old,
                        const Tensor& advantages, const Tensor& weights, const optional<Tensor>& ref,
                        double clip_low, double clip_high, double kl_coef, double temperature,
                        bool keep, bool one_pass) {
  refuse_tangents(logits, old, advantages, weights, ref);
  if (any_needs(logits)) {
    auto o = PolicyFunction::apply(logits, tokens, old, advantages, weights, ref, clip_low,
                                   clip_high, kl_coef, temperature, keep, one_pass);
    return {o[0], o[1], o[2], o[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("policy_loss", policy_forward)
      .call(logits, tokens, old, advantages, weights, ref, clip_low, clip_high, kl_coef,
            temperature, keep, one_pass);
}

struct DispatchFunction : torch::autograd::Function<DispatchFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& slots) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({slots});
    return {OP("dispatch", dispatch_forward).call(x, slots)};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto s = ctx->get_saved_variables();
    Tensor d;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      d = OP("combine", combine_forward).call(grads[0], s[0], std::nullopt);
    }
    return once({d, Tensor()}, grads);
  }
};

Tensor dispatch_autograd(const Tensor& x, const Tensor& slots) {
  refuse_tangents(x);
  if (any_needs(x)) return DispatchFunction::apply(x, slots)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("dispatch", dispatch_forward).call(x, slots);
}

struct CombineFunction : torch::autograd::Function<CombineFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& rows, const Tensor& slots,
                               const optional<Tensor>& gates) {
    at::AutoDispatchBelowADInplaceOrView below;
    // the rows are for the gates' gradient alone; without gates the slots do
    ctx->save_for_backward({needs(gates) ? rows : Tensor(), slots, or_undefined(gates)});
    return {OP("combine", combine_forward).call(rows, slots, gates)};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(3);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      if (!s[2].defined()) {
        out[0] = OP("dispatch", dispatch_forward).call(grads[0], s[1]);
      } else {
        const bool rows = ctx->needs_input_grad(0), gates = ctx->needs_input_grad(2);
        auto [drows, dgates] = OP("combine_backward", combine_backward)
                                   .call(grads[0], or_none(s[0]), s[1], s[2], rows, gates);
        if (rows) out[0] = drows;
        if (gates) out[2] = dgates;
      }
    }
    return once(out, {grads[0], s[0], s[2]});
  }
};

Tensor combine_autograd(const Tensor& rows, const Tensor& slots, const optional<Tensor>& gates) {
  refuse_tangents(rows, gates);
  if (any_needs(rows, gates)) return CombineFunction::apply(rows, slots, gates)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("combine", combine_forward).call(rows, slots, gates);
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weight,
                               const Tensor& offsets) {
    at::AutoDispatchBelowADInplaceOrView below;
    // each is for the other's gradient
    ctx->save_for_backward({needs(weight) ? rows : Tensor(), needs(rows) ? weight : Tensor(), offsets});
    return {OP("expert_linear", linear_forward).call(rows, weight, offsets)};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(3);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      if (ctx->needs_input_grad(0))
        out[0] = OP("expert_linear_backward_rows", linear_backward_rows).call(grads[0], s[1], s[2]);
      if (ctx->needs_input_grad(1))
        out[1] = OP("expert_linear_backward_weight", linear_backward_weight).call(grads[0], s[0], s[2]);
    }
    return once(out, {grads[0], s[0], s[1]});
  }
};

Tensor linear_autograd(const Tensor& rows, const Tensor& weight, const Tensor& offsets) {
  refuse_tangents(rows, weight);
  if (any_needs(rows, weight)) return LinearFunction::apply(rows, weight, offsets)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return OP("expert_linear", linear_forward).call(rows, weight, offsets);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(muonium_amd, m) {
  m.def("sort_by_expert(Tensor experts, int num_experts) -> (Tensor, Tensor)");
  m.def("dispatch(Tensor x, Tensor slots) -> Tensor");
  m.def("combine(Tensor rows, Tensor slots, Tensor? gates) -> Tensor");
  m.def("combine_backward(Tensor dy, Tensor? rows, Tensor slots, Tensor gates, bool rows_wanted, "
        "bool gates_wanted) -> (Tensor, Tensor)");
  m.def("expert_linear(Tensor rows, Tensor weight, Tensor offsets) -> Tensor");
  m.def("expert_linear_backward_rows(Tensor dy, Tensor weight, Tensor offsets) -> Tensor");
  m.def("expert_linear_backward_weight(Tensor dy, Tensor rows, Tensor offsets) -> Tensor");
  m.def("adamw_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, "
        "Tensor(d!)[] avg_scales, Tensor(e!)[] sq_scales, Tensor(f!)[] steps, int block, float lr, "
        "float beta1, float beta2, float eps, float weight_decay, bool maximize) -> ()");
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? cos, "
        "Tensor? sin, Tensor? positions, float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def("qk_norm_rope_backward(Tensor dq_out, Tensor dk_out, Tensor q, Tensor k, "
        "Tensor? q_weight, Tensor? k_weight, Tensor? cos, Tensor? sin, Tensor? positions, "
        "float eps, bool interleaved) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("route(Tensor logits, int top, Tensor? token_mask, bool normalize) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("route_backward(Tensor? dgates, Tensor? dbalance, Tensor? dzloss, Tensor logits, "
        "Tensor? token_mask, Tensor experts, Tensor counts, Tensor kept, bool normalize) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor tokens, float temperature, bool keep) -> "
        "(Tensor, Tensor)");
  m.def("token_logprobs_backward(Tensor dlogp, Tensor logits, Tensor tokens, Tensor stats, "
        "float temperature) -> Tensor");
  m.def("policy_loss(Tensor logits, Tensor tokens, Tensor old, Tensor advantages, "
        "Tensor weights, Tensor? ref, float clip_low, float clip_high, float kl_coef, "
        "float temperature, bool keep, bool one_pass) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("policy_loss_backward(Tensor dloss, Tensor logits, Tensor tokens, Tensor rows, "
        "float temperature) -> Tensor");
  m.def("policy_loss_rescale_(Tensor(a!) dlogits, Tensor dloss, Tensor logits, Tensor tokens, "
        "Tensor rows, float temperature) -> ()");
}

TORCH_LIBRARY_IMPL(muonium_amd, CUDA, m) {
  m.impl("qk_norm_rope", qk_forward);
  m.impl("qk_norm_rope_backward", qk_backward);
  m.impl("route", route_forward);
  m.impl("route_backward", route_backward);
  m.impl("token_logprobs", logp_forward);
  m.impl("token_logprobs_backward", logp_backward);
  m.impl("policy_loss", policy_forward);
  m.impl("policy_loss_backward", policy_backward);
  m.impl("policy_loss_rescale_", policy_rescale);
  m.impl("sort_by_expert", order_forward);
  m.impl("dispatch", dispatch_forward);
  m.impl("combine", combine_forward);
  m.impl("combine_backward", combine_backward);
  m.impl("expert_linear", linear_forward);
  m.impl("expert_linear_backward_rows", linear_backward_rows);
  m.impl("expert_linear_backward_weight", linear_backward_weight);
  m.impl("adamw_", adamw);
}

TORCH_LIBRARY_IMPL(muonium_amd, AutogradCUDA, m) {
  m.impl("qk_norm_rope", qk_autograd);
  m.impl("route", route_autograd);
  m.impl("token_logprobs", logp_autograd);
  m.impl("policy_loss", policy_autograd);
  m.impl("dispatch", dispatch_autograd);
  m.impl("combine", combine_autograd);
  m.impl("expert_linear", linear_autograd);
}
