// The torch op exactsample::verify_out, with the reference's schema
// (csrc/bindings.cpp:139-146), as a thin shim over the C ABI: it checks that
// every tensor is on the logits' CUDA device, describes each tensor as an
// es_tensor, and calls es_verify on the current stream. Every other check
// (dtype, rank, shape, capacity, alignment, aliasing) is the C ABI's, and its
// message becomes the RuntimeError. The row operators (token_logprobs,
// top_logits, policy_loss, distill_loss) are shims of the same kind, which
// also allocate their per-row outputs; their *_tracked forms record the call for
// autograd, whose backward pass calls the same operator with the gradient
// asked for. (A small call with its backward pass takes 72 us of the host's
// time, and 95 through Python's autograd functions.)
#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <array>

#include "exactsample_b200.h"

namespace {
using at::Tensor;
using OptionalTensor = std::optional<Tensor>;

int32_t dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ES_F32;
    case at::kDouble: return ES_F64;
    case at::kHalf: return ES_F16;
    case at::kBFloat16: return ES_BF16;
    case at::kInt: return ES_I32;
    case at::kLong: return ES_I64;
    case at::kByte: return ES_U8;
    default: return -1;
  }
}

es_tensor describe(const Tensor& t) {
  es_tensor e{};
  e.data = t.numel() ? const_cast<void*>(t.const_data_ptr()) : nullptr;
  e.dtype = dtype_of(t);
  e.ndim = int32_t(t.dim());
  for (int d = 0; d < t.dim() && d < 2; ++d) {
    e.size[d] = t.size(d);
    e.stride[d] = t.stride(d);
  }
  if (t.dim() > 2 || t.dim() == 0) e.ndim = -1;  // rejected by the C ABI's rank checks (0 would read as absent)
  return e;
}

void verify_out(const Tensor& logits, const Tensor& cu_rows, const Tensor& draft_ids,
                const OptionalTensor& draft_logits, const Tensor& temperature, const Tensor& top_k,
                const Tensor& top_p, const Tensor& min_p, const Tensor& draft_kind, const Tensor& seeds,
                const Tensor& stream_ids, const Tensor& positions, const OptionalTensor& mask, Tensor workspace,
                Tensor tokens, Tensor accepted_len, Tensor status, Tensor path_used, int64_t mode, int64_t dispatch,
                int64_t max_draft, int64_t list_max) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "target_logits must be a 2D CUDA tensor");
  const auto device = logits.device();
  auto same_device = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.device() == device, name, " has wrong device, dtype or rank");
  };
  same_device(cu_rows, "cu_rows");
  same_device(draft_ids, "draft_ids");
  for (const auto* t : {&temperature, &top_p, &min_p}) same_device(*t, "floating request parameter");
  for (const auto* t : {&top_k, &draft_kind, &seeds, &stream_ids}) same_device(*t, "integer request parameter");
  same_device(positions, "positions");
  if (draft_logits.has_value()) TORCH_CHECK(draft_logits->device() == device, "draft_logits shape/device mismatch");
  if (mask.has_value()) same_device(*mask, "mask");
  same_device(workspace, "workspace");
  same_device(tokens, "tokens");
  for (const auto* t : {&accepted_len, &status, &path_used}) same_device(*t, "output");

  es_args a{};
  a.target_logits = describe(logits);
  a.cu_rows = describe(cu_rows);
  a.draft_ids = describe(draft_ids);
  if (draft_logits.has_value()) a.draft_logits = describe(*draft_logits);
  a.temperature = describe(temperature);
  a.top_k = describe(top_k);
  a.top_p = describe(top_p);
  a.min_p = describe(min_p);
  a.draft_kind = describe(draft_kind);
  a.seeds = describe(seeds);
  a.stream_ids = describe(stream_ids);
  a.positions = describe(positions);
  if (mask.has_value()) a.mask = describe(*mask);
  a.workspace = describe(workspace);
  a.tokens = describe(tokens);
  a.accepted_len = describe(accepted_len);
  a.status = describe(status);
  a.path_used = describe(path_used);
  a.mode = mode;
  a.dispatch = dispatch;
  a.max_draft = max_draft;
  a.list_max = list_max;
  if (a.workspace.ndim == 1 && !workspace.is_contiguous()) a.workspace.stride[0] = 2;  // reported as non-contiguous
  c10::cuda::CUDAGuard guard(device);
  const int result = es_verify(&a, c10::cuda::getCurrentCUDAStream(device.index()).stream());
  TORCH_CHECK(result == ES_SUCCESS, es_last_error());
}

// ---- row operators on logits ----
// The call's device and stream, and its inputs: each is checked to be on the
// device and tied to the stream, so that the allocator does not hand its
// memory on while the call may still read it.
struct RowCall {
  const Tensor& logits;
  c10::cuda::CUDAGuard guard;
  c10::cuda::CUDAStream stream;
  bool capturing;

  static c10::Device device_of(const Tensor& logits) {
    TORCH_CHECK(logits.is_cuda() && logits.dim() == 2, "logits must be a 2D CUDA tensor");
    return logits.device();
  }
  explicit RowCall(const Tensor& l)
      : logits(l), guard(device_of(l)), stream(c10::cuda::getCurrentCUDAStream(l.device().index())),
        // (The default stream is never captured.)
        capturing(stream.stream() != nullptr &&
                  c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {}

  es_tensor use(const Tensor& t, const char* name) const {
    TORCH_CHECK(t.device() == logits.device(), name, " has wrong device, dtype or rank");
    if (!capturing) c10::cuda::CUDACachingAllocator::recordStream(t.unsafeGetTensorImpl()->unsafe_storage().data_ptr(), stream);
    return describe(t);
  }
  es_tensor use(const OptionalTensor& t, const char* name) const {
    return t.has_value() ? use(*t, name) : es_tensor{};
  }
  // A gradient tensor is written: whoever saved it for a backward pass must be able to tell.
  es_tensor write(const OptionalTensor& t, const char* name) const {
    if (t.has_value() && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    return use(t, name);
  }
  es_rows rows(const OptionalTensor& temperature, double temperature_all, const OptionalTensor& mask) const {
    es_rows r{};
    r.logits = use(logits, "logits");
    r.mask = use(mask, "mask");
    r.temperature = use(temperature, "temperature");
    r.temperature_all = temperature_all;
    return r;
  }
  // The call's per-row outputs: `floats` of float32 side by side in one
  // allocation (each starts on 16 bytes), then the statuses in one of their own,
  // since tensors of two types in one storage cannot be saved to one file.
  // (Straight from the allocator: the host's part of a small call is 8.0 us, and
  // was 8.2 with all of them in one at::empty; with a storage for each output a
  // policy loss takes it 12 instead of 10.)
  std::array<Tensor, 5> columns(int floats) const {
    const int64_t rows = logits.size(0), width = (rows + 3) / 4 * 4;
    const auto memory = [](int64_t words) {
      return c10::Storage(c10::Storage::use_byte_size_t(), size_t(words) * 4, c10::cuda::CUDACachingAllocator::get(),
                          /*resizable=*/true);
    };
    const auto column = [rows](c10::Storage storage, int64_t offset, caffe2::TypeMeta type) {
      Tensor t = at::detail::make_tensor<c10::TensorImpl>(std::move(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA), type);
      t.unsafeGetTensorImpl()->set_storage_offset(offset);
      t.unsafeGetTensorImpl()->set_sizes_contiguous({rows});
      return t;
    };
    const c10::Storage all = memory(width * floats);
    std::array<Tensor, 5> out;
    for (int i = 0; i < floats; ++i) out[i] = column(all, width * i, caffe2::TypeMeta::Make<float>());
    out[floats] = column(memory(rows), 0, caffe2::TypeMeta::Make<int32_t>());
    return out;
  }
  static void done(int result) { TORCH_CHECK(result == ES_SUCCESS, es_last_error()); }
};

std::tuple<Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens,
                                                  const OptionalTensor& temperature, double temperature_all,
                                                  const OptionalTensor& mask, const OptionalTensor& grad,
                                                  const OptionalTensor& grad_logprobs,
                                                  const OptionalTensor& grad_entropy) {
  const RowCall call(logits);
  auto [logprobs, entropy, status, _3, _4] = call.columns(2);
  es_logprob_args a{};
  a.in = call.rows(temperature, temperature_all, mask);
  a.tokens = call.use(tokens, "tokens");
  a.logprobs = describe(logprobs);
  a.entropy = describe(entropy);
  a.status = describe(status);
  a.grad = call.write(grad, "grad");
  a.grad_logprobs = call.use(grad_logprobs, "grad_logprobs");
  a.grad_entropy = call.use(grad_entropy, "grad_entropy");
  call.done(es_token_logprobs(&a, call.stream.stream()));
  return {std::move(logprobs), std::move(entropy), std::move(status)};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> top_logits(const Tensor& logits, int64_t k, const OptionalTensor& temperature,
                                                      double temperature_all, const OptionalTensor& mask) {
  const RowCall call(logits);
  TORCH_CHECK(k >= 1 && k <= ES_MAX_TOP, "k must be in [1, 256]");
  Tensor values = at::empty({logits.size(0), k}, logits.options().dtype(at::kFloat));
  Tensor ids = at::empty({logits.size(0), k}, logits.options().dtype(at::kLong));
  auto [rest, status, _2, _3, _4] = call.columns(1);
  es_top_args a{};
  a.in = call.rows(temperature, temperature_all, mask);
  a.values = describe(values);
  a.ids = describe(ids);
  a.rest = describe(rest);
  a.status = describe(status);
  call.done(es_top_logits(&a, call.stream.stream()));
  return {values, ids, rest, status};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> policy_loss(
    const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs, const Tensor& advantages,
    const OptionalTensor& ref_logprobs, const OptionalTensor& weights, const OptionalTensor& temperature,
    double temperature_all, const OptionalTensor& mask, double clip_low, double clip_high, double kl_coef,
    double entropy_coef, const OptionalTensor& grad) {
  const RowCall call(logits);
  auto [loss, logprobs, kl, entropy, status] = call.columns(4);
  es_policy_args a{};
  a.in = call.rows(temperature, temperature_all, mask);
  a.tokens = call.use(tokens, "tokens");
  a.old_logprobs = call.use(old_logprobs, "old_logprobs");
  a.advantages = call.use(advantages, "advantages");
  a.ref_logprobs = call.use(ref_logprobs, "ref_logprobs");
  a.weights = call.use(weights, "weights");
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  a.entropy_coef = entropy_coef;
  a.loss = describe(loss);
  a.logprobs = describe(logprobs);
  a.kl = describe(kl);
  a.entropy = describe(entropy);
  a.status = describe(status);
  a.grad = call.write(grad, "grad");
  call.done(es_policy_loss(&a, call.stream.stream()));
  return {loss, logprobs, kl, entropy, status};
}

std::tuple<Tensor, Tensor> distill_loss(const Tensor& logits, const Tensor& values, const Tensor& ids,
                                        const OptionalTensor& rest, const OptionalTensor& weights,
                                        const OptionalTensor& temperature, double temperature_all,
                                        const OptionalTensor& mask, const OptionalTensor& grad,
                                        const OptionalTensor& teacher_status) {
  const RowCall call(logits);
  auto [loss, status, _2, _3, _4] = call.columns(1);
  es_distill_args a{};
  a.in = call.rows(temperature, temperature_all, mask);
  a.values = call.use(values, "values");
  a.ids = call.use(ids, "ids");
  a.rest = call.use(rest, "rest");
  a.weights = call.use(weights, "weights");
  a.loss = describe(loss);
  a.status = describe(status);
  a.grad = call.write(grad, "grad");
  const es_tensor failed = call.use(teacher_status, "teacher_status");
  call.done(es_distill_loss_status(&a, &failed, call.stream.stream()));
  return {loss, status};
}

// ---- row operators on tensors without memory: what tracing asks for ----
// The checks that the kind of the inputs decides; the results' shapes and types.
struct Traced {
  Tensor column, status;
  explicit Traced(const Tensor& logits) {
    TORCH_CHECK(logits.dim() == 2, "logits must be a 2D CUDA tensor");
    const auto type = logits.scalar_type();
    TORCH_CHECK(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
                "row operators require float16/bfloat16/float32 logits");
    column = at::empty_symint({logits.sym_size(0)}, logits.options().dtype(at::kFloat));
    status = at::empty_symint({logits.sym_size(0)}, logits.options().dtype(at::kInt));
  }
  Tensor one() const { return at::empty_like(column); }
};
std::tuple<Tensor, Tensor, Tensor> token_logprobs_meta(const Tensor& logits, const Tensor&, const OptionalTensor&, double,
                                                       const OptionalTensor&, const OptionalTensor&, const OptionalTensor&,
                                                       const OptionalTensor&) {
  const Traced t(logits);
  return {t.one(), t.one(), t.status};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> top_logits_meta(const Tensor& logits, int64_t k, const OptionalTensor&, double,
                                                           const OptionalTensor&) {
  const Traced t(logits);
  TORCH_CHECK(k >= 1 && k <= ES_MAX_TOP, "k must be in [1, 256]");
  const std::array<c10::SymInt, 2> shape{logits.sym_size(0), k};
  return {at::empty_symint(shape, t.column.options()), at::empty_symint(shape, t.column.options().dtype(at::kLong)), t.one(),
          t.status};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> policy_loss_meta(
    const Tensor& logits, const Tensor&, const Tensor&, const Tensor&, const OptionalTensor&, const OptionalTensor&,
    const OptionalTensor&, double, const OptionalTensor&, double, double, double, double, const OptionalTensor&) {
  const Traced t(logits);
  return {t.one(), t.one(), t.one(), t.one(), t.status};
}
std::tuple<Tensor, Tensor> distill_loss_meta(const Tensor& logits, const Tensor&, const Tensor&, const OptionalTensor&,
                                             const OptionalTensor&, const OptionalTensor&, double, const OptionalTensor&,
                                             const OptionalTensor&, const OptionalTensor&) {
  const Traced t(logits);
  return {t.one(), t.status};
}

// ---- the operators as the dispatcher has them ----
constexpr char TOKEN_LOGPROBS[] = "exactsample::token_logprobs", TOP_LOGITS[] = "exactsample::top_logits",
               POLICY_LOSS[] = "exactsample::policy_loss", DISTILL_LOSS[] = "exactsample::distill_loss";
template <const char* NAME, class F> const c10::TypedOperatorHandle<F>& dispatched() {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(NAME, "").typed<F>();
  return op;
}
// One of them from inside an autograd function: directly, or, for a call that
// is being traced, so that the tracer sees it.
template <const char* NAME, class R, class... A, class... B>
R call_or_trace(R (*f)(A...), const Tensor& logits, B&&... args) {
  const c10::DispatchKeySet traced{c10::DispatchKey::Python, c10::DispatchKey::Functionalize};
  if (c10::impl::dispatch_mode_enabled() || logits.key_set().has_any(traced) || logits.is_meta())
    return dispatched<NAME, R(A...)>().call(logits, std::forward<B>(args)...);
  return f(logits, std::forward<B>(args)...);
}

// ---- row operators under autograd ----
// Of forward-mode derivatives there are none, and a call that ran below
// autograd would return its results with tangents of zero.
template <class T> bool has_tangent(const T&) { return false; }
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptionalTensor& t) { return t.has_value() && has_tangent(*t); }
template <class... A> void refuse_tangents(const A&... args) {
  TORCH_CHECK(!(has_tangent(args) || ...), "row operators have no forward-mode derivative");
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

Tensor or_undefined(const OptionalTensor& t) { return t.value_or(Tensor()); }
OptionalTensor or_none(const Tensor& t) { return t.defined() ? OptionalTensor(t) : std::nullopt; }
// What a backward pass returns: the logits' gradient and nothing for the
// `others`. Where it is itself recorded, the gradient says that it has no
// derivative when one is asked for.
variable_list logits_gradient(Tensor grad, size_t others) {
  if (at::GradMode::is_enabled()) {
    const auto error = std::make_shared<torch::autograd::DelayedError>("row operators are differentiable once", 1);
    grad = (*error)({grad.detach().requires_grad_()})[0];
  }
  variable_list all(1 + others);
  all[0] = std::move(grad);
  return all;
}
// The weights of a backward pass: the call's own times the loss's gradient.
Tensor weighted(const Tensor& weights, const Tensor& grad_loss) { return weights.defined() ? weights * grad_loss : grad_loss; }

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                               const OptionalTensor& temperature, double temperature_all, const OptionalTensor& mask) {
    ctx->save_for_backward({logits, tokens, or_undefined(temperature), or_undefined(mask)});
    ctx->saved_data["temperature"] = temperature_all;
    ctx->set_materialize_grads(false);
    auto [logprobs, entropy, status] =
        call_or_trace<TOKEN_LOGPROBS>(token_logprobs, logits, tokens, temperature, temperature_all, mask, std::nullopt,
                                      std::nullopt, std::nullopt);
    ctx->mark_non_differentiable({status});
    return {logprobs, entropy, status};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& out) {
    if (!out[0].defined() && !out[1].defined()) return variable_list(5);
    const variable_list saved = ctx->get_saved_variables();
    Tensor grad;
    {
      const at::NoGradGuard unrecorded;
      grad = at::empty_like(saved[0]);
      call_or_trace<TOKEN_LOGPROBS>(token_logprobs, saved[0], saved[1], or_none(saved[2]),
                                    ctx->saved_data["temperature"].toDouble(), or_none(saved[3]), grad, or_none(out[0]),
                                    or_none(out[1]));
    }
    return logits_gradient(grad, 4);
  }
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs,
                               const Tensor& advantages, const OptionalTensor& ref_logprobs, const OptionalTensor& weights,
                               const OptionalTensor& temperature, double temperature_all, const OptionalTensor& mask,
                               double clip_low, double clip_high, double kl_coef, double entropy_coef) {
    ctx->save_for_backward({logits, tokens, old_logprobs, advantages, or_undefined(ref_logprobs), or_undefined(weights),
                            or_undefined(temperature), or_undefined(mask)});
    ctx->saved_data["numbers"] = std::vector<double>{temperature_all, clip_low, clip_high, kl_coef, entropy_coef};
    ctx->set_materialize_grads(false);
    auto [loss, logprobs, kl, entropy, status] =
        call_or_trace<POLICY_LOSS>(policy_loss, logits, tokens, old_logprobs, advantages, ref_logprobs, weights, temperature,
                                   temperature_all, mask, clip_low, clip_high, kl_coef, entropy_coef, std::nullopt);
    ctx->mark_non_differentiable({logprobs, kl, entropy, status});
    return {loss, logprobs, kl, entropy, status};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& out) {
    if (!out[0].defined()) return variable_list(13);
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<double> numbers = ctx->saved_data["numbers"].toDoubleVector();
    Tensor grad;
    {
      const at::NoGradGuard unrecorded;
      grad = at::empty_like(saved[0]);
      call_or_trace<POLICY_LOSS>(policy_loss, saved[0], saved[1], saved[2], saved[3], or_none(saved[4]),
                                 weighted(saved[5], out[0]), or_none(saved[6]), numbers[0], or_none(saved[7]), numbers[1],
                                 numbers[2], numbers[3], numbers[4], grad);
    }
    return logits_gradient(grad, 12);
  }
};

struct DistillLoss : torch::autograd::Function<DistillLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& values, const Tensor& ids,
                               const OptionalTensor& rest, const OptionalTensor& weights, const OptionalTensor& temperature,
                               double temperature_all, const OptionalTensor& mask, const OptionalTensor& teacher_status) {
    ctx->save_for_backward({logits, values, ids, or_undefined(rest), or_undefined(weights), or_undefined(temperature),
                            or_undefined(mask)});
    ctx->saved_data["temperature"] = temperature_all;
    ctx->set_materialize_grads(false);
    auto [loss, status] = call_or_trace<DISTILL_LOSS>(distill_loss, logits, values, ids, rest, weights, temperature,
                                                      temperature_all, mask, std::nullopt, teacher_status);
    ctx->mark_non_differentiable({status});
    return {loss, status};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& out) {
    if (!out[0].defined()) return variable_list(9);
    const variable_list saved = ctx->get_saved_variables();
    Tensor grad;
    {
      const at::NoGradGuard unrecorded;
      grad = at::empty_like(saved[0]);
      call_or_trace<DISTILL_LOSS>(distill_loss, saved[0], saved[1], saved[2], or_none(saved[3]), weighted(saved[4], out[0]),
                                  or_none(saved[5]), ctx->saved_data["temperature"].toDouble(), or_none(saved[6]), grad,
                                  std::nullopt);
    }
    return logits_gradient(grad, 8);
  }
};

std::tuple<Tensor, Tensor, Tensor> token_logprobs_tracked(const Tensor& logits, const Tensor& tokens,
                                                          const OptionalTensor& temperature, double temperature_all,
                                                          const OptionalTensor& mask) {
  refuse_tangents(logits, temperature);
  const variable_list out = TokenLogprobs::apply(logits, tokens, temperature, temperature_all, mask);
  return {out[0], out[1], out[2]};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> policy_loss_tracked(
    const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs, const Tensor& advantages,
    const OptionalTensor& ref_logprobs, const OptionalTensor& weights, const OptionalTensor& temperature,
    double temperature_all, const OptionalTensor& mask, double clip_low, double clip_high, double kl_coef,
    double entropy_coef) {
  refuse_tangents(logits, old_logprobs, advantages, ref_logprobs, weights, temperature);
  const variable_list out = PolicyLoss::apply(logits, tokens, old_logprobs, advantages, ref_logprobs, weights, temperature,
                                              temperature_all, mask, clip_low, clip_high, kl_coef, entropy_coef);
  return {out[0], out[1], out[2], out[3], out[4]};
}
std::tuple<Tensor, Tensor> distill_loss_tracked(const Tensor& logits, const Tensor& values, const Tensor& ids,
                                                const OptionalTensor& rest, const OptionalTensor& weights,
                                                const OptionalTensor& temperature, double temperature_all,
                                                const OptionalTensor& mask, const OptionalTensor& teacher_status) {
  refuse_tangents(logits, values, rest, weights, temperature);
  const variable_list out = DistillLoss::apply(logits, values, ids, rest, weights, temperature, temperature_all, mask,
                                               teacher_status);
  return {out[0], out[1]};
}
// ---- the operators as the dispatcher calls them, below autograd ----
template <const char* NAME, class F> struct BelowAutograd;
template <const char* NAME, class R, class... A> struct BelowAutograd<NAME, R(A...)> {
  static R call(c10::DispatchKeySet keys, A... args) {
    refuse_tangents(args...);
    const at::AutoDispatchBelowADInplaceOrView below;
    return dispatched<NAME, R(A...)>().redispatch(keys & c10::after_ADInplaceOrView_keyset, args...);
  }
};
}  // namespace

TORCH_LIBRARY(exactsample, m) {
  m.def(
      "verify_out(Tensor target_logits, Tensor cu_rows, Tensor draft_ids, Tensor? draft_logits, "
      "Tensor temperature, Tensor top_k, Tensor top_p, Tensor min_p, Tensor draft_kind, "
      "Tensor seeds, Tensor stream_ids, Tensor positions, Tensor? mask, "
      "Tensor(a!) workspace, Tensor(b!) tokens, Tensor(c!) accepted_len, Tensor(d!) status, "
      "Tensor(e!) path_used, int mode, int dispatch, int max_draft, int list_max) -> ()");
  m.def(
      "token_logprobs(Tensor logits, Tensor tokens, Tensor? temperature, float temperature_all, Tensor? mask, "
      "Tensor(a!)? grad, Tensor? grad_logprobs, Tensor? grad_entropy) -> (Tensor, Tensor, Tensor)");
  m.def(
      "top_logits(Tensor logits, int k, Tensor? temperature, float temperature_all, Tensor? mask) "
      "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "policy_loss(Tensor logits, Tensor tokens, Tensor old_logprobs, Tensor advantages, Tensor? ref_logprobs, "
      "Tensor? weights, Tensor? temperature, float temperature_all, Tensor? mask, float clip_low, float clip_high, "
      "float kl_coef, float entropy_coef, Tensor(a!)? grad) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "distill_loss(Tensor logits, Tensor values, Tensor ids, Tensor? rest, Tensor? weights, Tensor? temperature, "
      "float temperature_all, Tensor? mask, Tensor(a!)? grad, Tensor? teacher_status=None) -> (Tensor, Tensor)");
  m.def(
      "token_logprobs_tracked(Tensor logits, Tensor tokens, Tensor? temperature, float temperature_all, Tensor? mask) "
      "-> (Tensor, Tensor, Tensor)", &token_logprobs_tracked);
  m.def(
      "policy_loss_tracked(Tensor logits, Tensor tokens, Tensor old_logprobs, Tensor advantages, Tensor? ref_logprobs, "
      "Tensor? weights, Tensor? temperature, float temperature_all, Tensor? mask, float clip_low, float clip_high, "
      "float kl_coef, float entropy_coef) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", &policy_loss_tracked);
  m.def(
      "distill_loss_tracked(Tensor logits, Tensor values, Tensor ids, Tensor? rest, Tensor? weights, "
      "Tensor? temperature, float temperature_all, Tensor? mask, Tensor? teacher_status=None) -> (Tensor, Tensor)",
      &distill_loss_tracked);
}
TORCH_LIBRARY_IMPL(exactsample, CUDA, m) {
  m.impl("verify_out", &verify_out);
  m.impl("token_logprobs", &token_logprobs);
  m.impl("top_logits", &top_logits);
  m.impl("policy_loss", &policy_loss);
  m.impl("distill_loss", &distill_loss);
}
TORCH_LIBRARY_IMPL(exactsample, Autograd, m) {
  m.impl("token_logprobs", &BelowAutograd<TOKEN_LOGPROBS, decltype(token_logprobs)>::call);
  m.impl("top_logits", &BelowAutograd<TOP_LOGITS, decltype(top_logits)>::call);
  m.impl("policy_loss", &BelowAutograd<POLICY_LOSS, decltype(policy_loss)>::call);
  m.impl("distill_loss", &BelowAutograd<DISTILL_LOSS, decltype(distill_loss)>::call);
}
TORCH_LIBRARY_IMPL(exactsample, Meta, m) {
  m.impl("token_logprobs", &token_logprobs_meta);
  m.impl("top_logits", &top_logits_meta);
  m.impl("policy_loss", &policy_loss_meta);
  m.impl("distill_loss", &distill_loss_meta);
}
