// The C ABI of the row operators on logits (include/exactsample_b200.h):
// argument checks, the split of a row, and the launch.
#include <algorithm>
#include <cmath>
#include <exception>

#include "es_host.h"
#include "es_top.cuh"

namespace es {
namespace score {
extern template cudaError_t launch_loss<ES_F32>(const LossParams&, int, cudaStream_t);
extern template cudaError_t launch_loss<ES_F16>(const LossParams&, int, cudaStream_t);
extern template cudaError_t launch_loss<ES_BF16>(const LossParams&, int, cudaStream_t);
extern template cudaError_t launch_top<ES_F32>(const TopParams&, cudaStream_t);
extern template cudaError_t launch_top<ES_F16>(const TopParams&, cudaStream_t);
extern template cudaError_t launch_top<ES_BF16>(const TopParams&, cudaStream_t);
}  // namespace score
}  // namespace es

namespace {
using namespace es::score;
using es::host::check;
using es::host::device_check;
using es::host::disjoint;
using es::host::element_size;
using es::host::fail;
using es::host::g_error;
using es::host::no_internal_overlap;
using es::host::numel;

bool present(const es_tensor& t) { return t.ndim != 0; }

// Offsets inside a tensor stay far from 64-bit overflow in the checks and in the kernels.
bool addressable(const es_tensor& t, const char* name) {
  for (int d = 0; d < t.ndim; ++d)
    if (t.size[d] > INT32_MAX || t.stride[d] > (int64_t(1) << 46) / std::max<int64_t>(t.size[d], 1)) {
      g_error = std::string(name) + " exceeds the kernels' index range";
      return false;
    }
  return true;
}

// The kernels load and store whole elements.
int aligned(const es_tensor& t, const char* name, const char* whose = "its") {
  if (numel(t) == 0 || reinterpret_cast<uintptr_t>(t.data) % element_size(t.dtype) == 0) return ES_SUCCESS;
  return fail(ES_ERR_ALIGNMENT, std::string(name) + " must be aligned to " + whose + " elements");
}

// One call's tensors as they are checked: the inputs and the outputs.
struct Tensors {
  const es_tensor* list[10];
  int count = 0;
  void add(const es_tensor& t) { list[count++] = &t; }
  const es_tensor* const* begin() const { return list; }
  const es_tensor* const* end() const { return list + count; }
};
struct Call {
  const es_rows& in;
  int64_t rows = 0, vocab = 0;
  Tensors inputs, outputs;
  bool in_place = false;  // the gradient is the logits tensor

  // The logits, the mask and the temperatures.
  int begin() {
    const es_tensor& logits = in.logits;
    if (logits.ndim != 2 || logits.size[0] < 0 || logits.size[1] < 0 || (logits.data == nullptr && numel(logits) != 0))
      return fail(ES_ERR_ARGUMENT, "logits must be a 2D CUDA tensor");
    if (logits.dtype != ES_F32 && logits.dtype != ES_F16 && logits.dtype != ES_BF16)
      return fail(ES_ERR_ARGUMENT, "row operators require float16/bfloat16/float32 logits");
    if (logits.stride[0] < 0 || logits.stride[1] < 0) return fail(ES_ERR_ARGUMENT, "logits has a negative stride");
    if (!addressable(logits, "logits")) return ES_ERR_ARGUMENT;
    if (const int e = aligned(logits, "logits", "their"); e != ES_SUCCESS) return e;
    rows = logits.size[0];
    vocab = logits.size[1];
    if (vocab < 1) return fail(ES_ERR_ARGUMENT, "logits must have at least one column");
    inputs.add(logits);
    if (present(in.mask)) {
      if (!check(in.mask, ES_I32, 2, "mask") || !addressable(in.mask, "mask")) return ES_ERR_ARGUMENT;
      if (!(in.mask.size[0] == rows && in.mask.size[1] == (vocab + 31) / 32))
        return fail(ES_ERR_ARGUMENT, "mask shape mismatch");
      if (const int e = aligned(in.mask, "mask"); e != ES_SUCCESS) return e;
      inputs.add(in.mask);
    }
    if (present(in.temperature)) {
      if (const int e = column(in.temperature, ES_F64, "temperature", inputs); e != ES_SUCCESS) return e;
    } else if (!(in.temperature_all > 0 && std::isfinite(in.temperature_all))) {
      return fail(ES_ERR_ARGUMENT, "temperature must be positive and finite");
    }
    return ES_SUCCESS;
  }
  int column(const es_tensor& t, int32_t dtype, const char* name, Tensors& list) {
    if (!check(t, dtype, 1, name) || !addressable(t, name)) return ES_ERR_ARGUMENT;
    if (t.size[0] != rows) return fail(ES_ERR_ARGUMENT, std::string(name) + " must have one value per row");
    list.add(t);
    return aligned(t, name);
  }
  int grid(const es_tensor& t, int32_t dtype, int64_t width, const char* name, Tensors& list) {
    if (!check(t, dtype, 2, name) || !addressable(t, name)) return ES_ERR_ARGUMENT;
    if (t.size[0] != rows || t.size[1] != width) return fail(ES_ERR_ARGUMENT, std::string(name) + " shape mismatch");
    list.add(t);
    return aligned(t, name);
  }
  // A gradient: apart from every other tensor, or the logits tensor itself.
  int gradient(const es_tensor& g) {
    if (!present(g)) return ES_SUCCESS;
    const es_tensor& l = in.logits;
    if (const int e = grid(g, l.dtype, vocab, "grad", outputs); e != ES_SUCCESS) return e;
    if (g.data == l.data && g.stride[0] == l.stride[0] && g.stride[1] == l.stride[1])
      in_place = true;
    return ES_SUCCESS;
  }
  int finish() const {
    for (const es_tensor* const& out : outputs) {
      if (!no_internal_overlap(*out)) return fail(ES_ERR_ALIAS, "output has overlapping strides");
      for (const es_tensor* t : inputs)
        if (!(in_place && t == &in.logits) && !disjoint(*out, *t))
          return fail(ES_ERR_ALIAS, "exactsample input/output aliasing is forbidden");
      for (const es_tensor* const* other = outputs.begin(); other != &out; ++other)
        if (!disjoint(*out, **other)) return fail(ES_ERR_ALIAS, "exactsample outputs alias");
    }
    return ES_SUCCESS;
  }
};

template <class T> Column<T> col(const es_tensor& t) {
  return {present(t) ? static_cast<T*>(t.data) : nullptr, t.stride[0]};
}
template <class T> Grid2<T> grid2(const es_tensor& t) {
  return {present(t) ? static_cast<T*>(t.data) : nullptr, t.stride[0], t.stride[1]};
}

constexpr size_t MAX_SMEM = 227 * 1024;

// Ranks of a row's cluster: slices of about SLICE_BYTES, the fewest ranks
// that allow them, at most 16. The rule sees only the vocabulary and the type, so that a
// row's results do not depend on the batch.
int split(Rows& r, const es_rows& in, size_t slice_bytes, int64_t least, size_t (*smem)(int, int32_t, bool, int), int k, size_t* bytes) {
  const int64_t vocab = in.logits.size[1];
  const int64_t steps = (vocab + SLICE_STEP - 1) / SLICE_STEP;
  const int64_t row_bytes = vocab * int64_t(element_size(in.logits.dtype));
  const int64_t want = std::clamp<int64_t>(std::max((row_bytes + int64_t(slice_bytes) - 1) / int64_t(slice_bytes), least), 1, MAX_RANKS);
  const int64_t slice = (steps + want - 1) / want * SLICE_STEP;
  if (slice > int64_t(MAX_SMEM)) return fail(ES_ERR_UNSUPPORTED, "vocabulary too large for one 16-block cluster's shared memory");
  *bytes = smem(int(slice), in.logits.dtype, present(in.mask), k);
  if (*bytes > MAX_SMEM) return fail(ES_ERR_UNSUPPORTED, "vocabulary too large for one 16-block cluster's shared memory");
  r.logits = in.logits.data;
  r.l_s0 = in.logits.stride[0];
  r.l_s1 = in.logits.stride[1];
  r.mask = grid2<const int32_t>(in.mask);
  r.temperature = col<const double>(in.temperature);
  r.all = scale_of(in.temperature_all);
  r.rows = in.logits.size[0];
  r.vocab = int32_t(vocab);
  r.slice = int32_t(slice);
  r.ranks = int32_t((vocab + slice - 1) / slice);
  if (in.logits.size[0] > INT32_MAX / r.ranks) return fail(ES_ERR_UNSUPPORTED, "too many rows for one launch");
  return ES_SUCCESS;
}

size_t loss_bytes(int slice, int32_t dtype, bool mask, int k) {
  return dtype == ES_F32 ? loss_smem<ES_F32>(slice, mask, k) : loss_smem<ES_F16>(slice, mask, k);
}
// A policy step of 4,096 rows of 151,936 bf16 took, by slice and blocks to an
// SM (runs of 20 on one card): 33 KB, six blocks, 582 us; 38 KB, five, 504; 44
// KB, four, 483; 50 KB, four, 453; 64 KB, three, 483. Nothing else was swept.
constexpr size_t LOSS_SLICE_BYTES = 50 * 1024;

int launched(cudaError_t e) {
  return e == cudaSuccess ? ES_SUCCESS
                          : fail(ES_ERR_LAUNCH, std::string("exactsample kernel launch failed: ") + cudaGetErrorString(e));
}

int run_loss(Call& call, LossParams& p, const es_tensor& grad, int op, cudaStream_t stream) {
  if (const int e = call.gradient(grad); e != ES_SUCCESS) return e;
  if (const int e = call.finish(); e != ES_SUCCESS) return e;
  size_t smem = 0;
  if (const int e = split(p.in, call.in, LOSS_SLICE_BYTES, 1, loss_bytes, p.k, &smem); e != ES_SUCCESS) return e;
  if (call.rows == 0) return ES_SUCCESS;
  if (const int e = device_check(); e != ES_SUCCESS) return e;
  p.grad = present(grad) ? grad.data : nullptr;
  p.g_s0 = grad.stride[0];
  p.g_s1 = grad.stride[1];
  cudaGetLastError();  // clear a stale error so that the check reports this launch's
  switch (call.in.logits.dtype) {
    case ES_F32: return launched(launch_loss<ES_F32>(p, op, stream));
    case ES_F16: return launched(launch_loss<ES_F16>(p, op, stream));
    default: return launched(launch_loss<ES_BF16>(p, op, stream));
  }
}

int token_logprobs(const es_logprob_args* a, cudaStream_t stream) {
  Call call{a->in};
  int e = call.begin();
  if (e == ES_SUCCESS) e = call.column(a->tokens, ES_I64, "tokens", call.inputs);
  if (e == ES_SUCCESS) e = call.column(a->logprobs, ES_F32, "logprobs", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->entropy, ES_F32, "entropy", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->status, ES_I32, "status", call.outputs);
  for (const es_tensor* t : {&a->grad_logprobs, &a->grad_entropy})
    if (e == ES_SUCCESS && present(*t)) {
      if (!present(a->grad)) return fail(ES_ERR_ARGUMENT, "grad_logprobs and grad_entropy need grad");
      e = call.column(*t, ES_F32, t == &a->grad_entropy ? "grad_entropy" : "grad_logprobs", call.inputs);
    }
  if (e != ES_SUCCESS) return e;
  LossParams p{};
  p.tokens = col<const int64_t>(a->tokens);
  p.grad_logprobs = col<const float>(a->grad_logprobs);
  p.grad_entropy = col<const float>(a->grad_entropy);
  p.logprobs = col<float>(a->logprobs);
  p.entropy = col<float>(a->entropy);
  p.status = col<int32_t>(a->status);
  return run_loss(call, p, a->grad, LOGPROB, stream);
}

int policy_loss(const es_policy_args* a, cudaStream_t stream) {
  Call call{a->in};
  int e = call.begin();
  if (e == ES_SUCCESS) e = call.column(a->tokens, ES_I64, "tokens", call.inputs);
  if (e == ES_SUCCESS) e = call.column(a->old_logprobs, ES_F32, "old_logprobs", call.inputs);
  if (e == ES_SUCCESS) e = call.column(a->advantages, ES_F32, "advantages", call.inputs);
  if (e == ES_SUCCESS && present(a->ref_logprobs)) e = call.column(a->ref_logprobs, ES_F32, "ref_logprobs", call.inputs);
  if (e == ES_SUCCESS && present(a->weights)) e = call.column(a->weights, ES_F32, "weights", call.inputs);
  if (e != ES_SUCCESS) return e;
  if (!(a->clip_low >= 0 && a->clip_low <= 1 && a->clip_high >= 0 && std::isfinite(a->clip_high)))
    return fail(ES_ERR_ARGUMENT, "clip_low must be in [0, 1] and clip_high nonnegative and finite");
  if (!(std::isfinite(a->kl_coef) && std::isfinite(a->entropy_coef)))
    return fail(ES_ERR_ARGUMENT, "kl_coef and entropy_coef must be finite");
  if (a->kl_coef != 0 && !present(a->ref_logprobs)) return fail(ES_ERR_ARGUMENT, "kl_coef needs ref_logprobs");
  e = call.column(a->loss, ES_F32, "loss", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->logprobs, ES_F32, "logprobs", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->kl, ES_F32, "kl", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->entropy, ES_F32, "entropy", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->status, ES_I32, "status", call.outputs);
  if (e != ES_SUCCESS) return e;
  LossParams p{};
  p.tokens = col<const int64_t>(a->tokens);
  p.old_logprobs = col<const float>(a->old_logprobs);
  p.advantages = col<const float>(a->advantages);
  p.ref_logprobs = col<const float>(a->ref_logprobs);
  p.weights = col<const float>(a->weights);
  p.ratio_low = 1 - a->clip_low;
  p.ratio_high = 1 + a->clip_high;
  p.kl_coef = a->kl_coef;
  p.entropy_coef = a->entropy_coef;
  p.loss = col<float>(a->loss);
  p.logprobs = col<float>(a->logprobs);
  p.kl = col<float>(a->kl);
  p.entropy = col<float>(a->entropy);
  p.status = col<int32_t>(a->status);
  return run_loss(call, p, a->grad, POLICY, stream);
}

int distill_loss(const es_distill_args* a, const es_tensor* teacher_status, cudaStream_t stream) {
  Call call{a->in};
  int e = call.begin();
  if (e != ES_SUCCESS) return e;
  const int64_t k = a->values.ndim == 2 ? a->values.size[1] : 0;
  if (a->values.ndim == 2 && !(k >= 1 && k <= MAX_TOP)) return fail(ES_ERR_ARGUMENT, "k must be in [1, 256]");
  e = call.grid(a->values, ES_F32, k, "values", call.inputs);
  if (e == ES_SUCCESS) e = call.grid(a->ids, ES_I64, k, "ids", call.inputs);
  if (e == ES_SUCCESS && present(a->rest)) e = call.column(a->rest, ES_F32, "rest", call.inputs);
  if (e == ES_SUCCESS && present(a->weights)) e = call.column(a->weights, ES_F32, "weights", call.inputs);
  const bool of_teacher = teacher_status != nullptr && present(*teacher_status);
  if (e == ES_SUCCESS && of_teacher) e = call.column(*teacher_status, ES_I32, "teacher_status", call.inputs);
  if (e == ES_SUCCESS) e = call.column(a->loss, ES_F32, "loss", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->status, ES_I32, "status", call.outputs);
  if (e != ES_SUCCESS) return e;
  LossParams p{};
  if (of_teacher) p.teacher_status = col<const int32_t>(*teacher_status);
  p.values = grid2<const float>(a->values);
  p.ids = grid2<const int64_t>(a->ids);
  p.rest = col<const float>(a->rest);
  p.weights = col<const float>(a->weights);
  p.k = int32_t(k);
  p.loss = col<float>(a->loss);
  p.status = col<int32_t>(a->status);
  return run_loss(call, p, a->grad, DISTILL, stream);
}

size_t top_bytes(int slice, int32_t, bool, int) { return top_smem(slice); }
// The 64 largest of 2,048 rows of 151,936 bf16 and the 20 largest of 8, whole
// calls: 200 and 10.9 us in slices of 38 KB; 193 and 12.3 of 51 KB; 177 and
// 12.3 of 64 KB; 174 and 15.2 of 102 KB; 174 and 18.5 of 152 KB.
constexpr size_t TOP_SLICE_BYTES = 64 * 1024;

int top_logits(const es_top_args* a, cudaStream_t stream) {
  Call call{a->in};
  int e = call.begin();
  if (e != ES_SUCCESS) return e;
  const int64_t k = a->values.ndim == 2 ? a->values.size[1] : 0;
  if (a->values.ndim == 2 && !(k >= 1 && k <= MAX_TOP)) return fail(ES_ERR_ARGUMENT, "k must be in [1, 256]");
  e = call.grid(a->values, ES_F32, k, "values", call.outputs);
  if (e == ES_SUCCESS) e = call.grid(a->ids, ES_I64, k, "ids", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->rest, ES_F32, "rest", call.outputs);
  if (e == ES_SUCCESS) e = call.column(a->status, ES_I32, "status", call.outputs);
  if (e == ES_SUCCESS) e = call.finish();
  if (e != ES_SUCCESS) return e;
  TopParams p{};
  size_t smem = 0;
  e = split(p.in, a->in, TOP_SLICE_BYTES, (k + 31) / 32, top_bytes, 0, &smem);
  if (e != ES_SUCCESS || call.rows == 0) return e;
  if (e = device_check(); e != ES_SUCCESS) return e;
  p.k = int32_t(k);
  p.values = grid2<float>(a->values);
  p.ids = grid2<int64_t>(a->ids);
  p.rest = col<float>(a->rest);
  p.status = col<int32_t>(a->status);
  cudaGetLastError();
  switch (a->in.logits.dtype) {
    case ES_F32: return launched(launch_top<ES_F32>(p, stream));
    case ES_F16: return launched(launch_top<ES_F16>(p, stream));
    default: return launched(launch_top<ES_BF16>(p, stream));
  }
}

// No exception leaves a C entry point.
template <class A, class F> int guarded(const A* args, void* stream, F f) {
  try {
    g_error.clear();
    if (args == nullptr) return fail(ES_ERR_ARGUMENT, "null arguments");
    return f(args, static_cast<cudaStream_t>(stream));
  } catch (const std::exception&) {
    return ES_ERR_ARGUMENT;  // out of host memory: nothing was enqueued
  }
}
}  // namespace

extern "C" {
int es_token_logprobs(const es_logprob_args* args, void* stream) { return guarded(args, stream, token_logprobs); }
int es_policy_loss(const es_policy_args* args, void* stream) { return guarded(args, stream, policy_loss); }
int es_distill_loss(const es_distill_args* args, void* stream) { return es_distill_loss_status(args, nullptr, stream); }
int es_distill_loss_status(const es_distill_args* args, const es_tensor* teacher_status, void* stream) {
  return guarded(args, stream, [=](const es_distill_args* a, cudaStream_t s) { return distill_loss(a, teacher_status, s); });
}
int es_top_logits(const es_top_args* args, void* stream) { return guarded(args, stream, top_logits); }
}  // extern "C"
