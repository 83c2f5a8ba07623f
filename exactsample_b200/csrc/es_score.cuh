// Row operators on logits: token log-probabilities, the clipped policy loss
// and the distillation loss, each with its gradient (loss_rows), from one
// read of the row.
//
// A row is split over the ranks of one thread-block cluster in contiguous
// slices, and each rank keeps its slice in shared memory (about 38 KB, so
// that five blocks share an SM). The row is read from HBM once: the first
// pass over the slice takes the running maximum and the sums, the ranks
// exchange them, and the gradient is written from the same shared copy. A
// loss with its gradient so moves one read and one write of the row, where a
// row that does not stay on the chip needs two reads and one write.
//
// The split depends on the vocabulary and the type alone, and every thread
// takes the same elements whatever the row's address, so a row's results are
// the same bits in any batch and at any alignment.
#pragma once
#include <atomic>

#include "es_device.cuh"

namespace es {
namespace score {

enum Op { LOGPROB = 0, POLICY = 1, DISTILL = 2 };
constexpr int MAX_RANKS = 16;   // cluster size (beyond 8: non-portable, as for the row kernels)
constexpr int MAX_TOP = ES_MAX_TOP;
constexpr int PIECES = 4;       // bulk copies of a slice, each with its own barrier
constexpr int SLICE_STEP = 128; // slices are a multiple of this many tokens: whole mask words and 16-byte chunks
constexpr float LOWEST = -3.402823466e38f;
// Exponents (base 2) are held at or above this: 2^FAR is 0, and a product of
// it with 0 is 0, where -inf * 0 would be NaN.
constexpr float FAR = -1e4f;
constexpr uint32_t WAIT_LIMIT = 1u << 20;
constexpr double LOG2E = 1.4426950408889634074, LN2 = 0.69314718055994530942;

template <class T> struct Column {  // a strided 1-D tensor; absent when p is null
  T* p;
  int64_t s;
  __device__ __forceinline__ T& operator[](int64_t i) const { return p[i * s]; }
};
template <class T> struct Grid2 {  // a strided 2-D tensor
  T* p;
  int64_t s0, s1;
};

struct Rows {
  const void* logits;
  int64_t l_s0, l_s1;
  Grid2<const int32_t> mask;
  Column<const double> temperature;
  double temperature_all;
  int32_t vocab, ranks, slice;
};

struct LossParams {
  Rows in;
  void* grad;
  int64_t g_s0, g_s1;
  Column<const int64_t> tokens;
  Column<const float> old_logprobs, advantages, ref_logprobs, weights;  // policy; weights: distill too
  Column<const float> grad_logprobs, grad_entropy;                      // logprob
  double ratio_low, ratio_high, kl_coef, entropy_coef;
  Grid2<const float> values;
  Grid2<const int64_t> ids;
  Column<const float> rest;
  int32_t k;
  Column<float> loss, logprobs, kl, entropy;
  Column<int32_t> status;
};

// ---------------------------------------------------------------------------
// Element types. A chunk is 16 bytes of elements; it is unpacked to pairs for
// the packed FP32 instructions.
template <int DT> struct Elem;
template <> struct Elem<ES_F32> {
  using T = float;
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
  static __device__ __forceinline__ float2 unpack(uint32_t a, uint32_t b) {
    return make_float2(__uint_as_float(a), __uint_as_float(b));
  }
};
template <> struct Elem<ES_F16> {
  using T = __half;
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(T v) { return __half2float(v); }
  static __device__ __forceinline__ T put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<ES_BF16> {
  using T = __nv_bfloat16;
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T put(float v) { return __float2bfloat16_rn(v); }
};

template <int DT> __device__ __forceinline__ void unpack(const uint4& q, float2* v) {
  if constexpr (DT == ES_F32) {
    v[0] = Elem<DT>::unpack(q.x, q.y);
    v[1] = Elem<DT>::unpack(q.z, q.w);
  } else {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == ES_BF16) {
        v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      }
    }
  }
}
// Rounded to nearest: the gradient's one rounding to the logits' type.
template <int DT> __device__ __forceinline__ uint4 pack(const float2* v) {
  uint32_t w[4];
  if constexpr (DT == ES_F32) {
    w[0] = __float_as_uint(v[0].x);
    w[1] = __float_as_uint(v[0].y);
    w[2] = __float_as_uint(v[1].x);
    w[3] = __float_as_uint(v[1].y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == ES_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[i].x, v[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[i].x, v[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Packed FP32 pairs (one instruction for two lanes on sm_100).
__device__ __forceinline__ uint64_t bits2(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 pair2(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// max that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---------------------------------------------------------------------------
// The running maximum m of the logits seen, s = sum 2^((z - m) scale) and
// u = sum 2^d d with d = (z - m) scale: everything a row's log-sum and entropy
// need. scale = log2(e) / temperature. The difference is taken before the
// scaling, so that a row of the type's lowest values, or of huge ones, does
// not overflow. s and u are held as two partial sums.
struct Acc {
  float m;
  float2 s, u;
};
__device__ __forceinline__ Acc acc_none() { return {LOWEST, {0.f, 0.f}, {0.f, 0.f}}; }
__device__ __forceinline__ float exponent(float z, float m, float scale) {
  return max_nan(__fmul_rn(__fsub_rn(z, m), scale), FAR);
}
template <bool ENTROPY> __device__ __forceinline__ void acc_raise(Acc& a, float m, float scale) {
  const float d = exponent(a.m, m, scale), f = ex2(d);
  if (ENTROPY) a.u = mul2(both(f), fma2(both(d), a.s, a.u));
  a.s = mul2(both(f), a.s);
  a.m = m;
}
template <int N, bool ENTROPY> __device__ __forceinline__ void acc_chunk(Acc& a, const float2* v, float scale) {
  float top = fmaxf(v[0].x, v[0].y);  // a NaN drops out here and shows up in s
#pragma unroll
  for (int i = 1; i < N / 2; ++i) top = fmaxf(top, fmaxf(v[i].x, v[i].y));
  if (top > a.m) acc_raise<ENTROPY>(a, top, scale);
  const float2 nm = both(-a.m), sc = both(scale);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    float2 d = mul2(add2(v[i], nm), sc);
    if (ENTROPY) d = make_float2(max_nan(d.x, FAR), max_nan(d.y, FAR));
    const float2 e = make_float2(ex2(d.x), ex2(d.y));
    a.s = add2(a.s, e);
    if (ENTROPY) a.u = fma2(e, d, a.u);
  }
}

// What one rank knows of its slice.
struct Record {
  float m, s, u;
  uint32_t bad;  // a NaN or +inf behind the mask, a repeated id, a copy that did not arrive
};
__device__ __forceinline__ Record merge(Record a, Record b, float scale) {
  Record r;
  r.m = fmaxf(a.m, b.m);
  const float da = exponent(a.m, r.m, scale), db = exponent(b.m, r.m, scale);
  const float fa = ex2(da), fb = ex2(db);
  r.s = __fadd_rn(__fmul_rn(fa, a.s), __fmul_rn(fb, b.s));
  r.u = __fadd_rn(__fmul_rn(fa, __fadd_rn(a.u, __fmul_rn(da, a.s))), __fmul_rn(fb, __fadd_rn(b.u, __fmul_rn(db, b.s))));
  r.bad = a.bad | b.bad;
  return r;
}
__device__ __forceinline__ Record shfl_record(Record r, int o) {
  return {shfl_xor(r.m, o), shfl_xor(r.s, o), shfl_xor(r.u, o), shfl_xor(r.bad, o)};
}

// ---------------------------------------------------------------------------
// Cluster barrier halves: between them a rank does work of its own.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// ---------------------------------------------------------------------------
// A rank's slice of the row in shared memory. Element i lies at
// base + shift + i * sizeof(T), where shift is the row's misalignment against
// 16 bytes, so that the aligned middle of the slice comes by bulk copies and
// only the ragged ends by plain loads. Rows without unit stride are gathered.
template <int DT> struct Slice {
  using T = typename Elem<DT>::T;
  static constexpr int N = Elem<DT>::N;
  uint8_t* base;
  uint64_t* bar;
  uint32_t shift, at, piece;  // the bulk part starts at byte `at`, in pieces of `piece` bytes
  int n, chunks, pieces, ready;
  bool late;  // a copy did not arrive in time

  __device__ __forceinline__ T& operator[](int i) const { return reinterpret_cast<T*>(base + shift)[i]; }

  // All threads; ends with a block barrier.
  __device__ __forceinline__ void load(const Rows& in, int64_t row, int begin, int count, uint8_t* buffer, uint64_t* bars) {
    base = buffer;
    bar = bars;
    n = count;
    chunks = (n + N - 1) / N;
    ready = 0;
    late = false;
    const T* src = static_cast<const T*>(in.logits) + row * in.l_s0 + int64_t(begin) * in.l_s1;
    const int tid = threadIdx.x;
    pieces = 0;
    at = 0;
    piece = 4096;
    if (in.l_s1 == 1) {
      const uint32_t bytes = uint32_t(n) * sizeof(T);
      shift = uint32_t(reinterpret_cast<uintptr_t>(src)) & 15;
      const uint32_t lead = min((16 - shift) & 15, bytes), bulk = (bytes - lead) & ~15u;
      at = shift + lead;
      piece = max(4096u, (bulk / PIECES + 4095) & ~4095u);
      pieces = int((bulk + piece - 1) / piece);
      if (tid == 0) {
        for (int i = 0; i < pieces; ++i) mbar_init(bar + i, 1);
        mbar_init_fence();
        const uint8_t* g = reinterpret_cast<const uint8_t*>(src) + lead;
        for (int i = 0; i < pieces; ++i) {
          const uint32_t size = min(piece, bulk - i * piece);
          mbar_arrive_expect_tx(bar + i, size);
          bulk_load(base + at + i * piece, g + i * piece, size, bar + i);
        }
      }
      const int head = int(lead / sizeof(T)), tail = int((lead + bulk) / sizeof(T));
      if (tid < head) (*this)[tid] = src[tid];
      if (tid >= 32 && tail + tid - 32 < n) (*this)[tail + tid - 32] = src[tail + tid - 32];
    } else {
      shift = 0;
      for (int i = tid; i < n; i += THREADS) (*this)[i] = src[i * in.l_s1];
    }
    if (tid < chunks * N - n) (*this)[n + tid] = Elem<DT>::put(-INFINITY);  // the last chunk's unused places
    __syncthreads();
  }
  // Until the first `end` bytes of the buffer are there.
  __device__ __forceinline__ void wait(uint32_t end) {
    while (ready < pieces && at + ready * piece < end) {
      uint32_t spins = 0;
      while (!mbar_try_wait(bar + ready, 0))
        if (++spins >= WAIT_LIMIT) {
          late = true;
          break;
        }
      ++ready;
    }
  }
  __device__ __forceinline__ void wait_all() { wait(0xffffffffu); }
  // Chunk c (elements [c N, c N + N)). A shifted chunk is cut out of two aligned ones.
  __device__ __forceinline__ uint4 chunk(int c) const {
    const uint4* p = reinterpret_cast<const uint4*>(base) + c;
    uint4 a = p[0];
    if (shift) {
      const uint4 b = p[1];
      uint32_t w[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
      uint32_t last = b.w;
      if (shift & 8) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 2];
        w[5] = last;
      }
      if (shift & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
      }
      if (sizeof(T) == 2 && (shift & 2)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
      }
      a = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return a;
  }
  __device__ __forceinline__ void set_chunk(int c, const uint4& q) const {
    if (shift == 0) {
      reinterpret_cast<uint4*>(base)[c] = q;
    } else {
      const T* v = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < N; ++i) (*this)[c * N + i] = v[i];
    }
  }
};

// Masked tokens of a chunk become -inf; returns whether one of them is NaN or +inf.
template <int DT> __device__ __forceinline__ bool mask_chunk(const int32_t* words, int64_t stride, int first, float2* v) {
  constexpr int N = Elem<DT>::N;
  const uint32_t bits = uint32_t(words[(first >> 5) * stride]) >> (first & 31);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    if (!(bits >> (2 * i) & 1)) {
      bad |= !(v[i].x < INFINITY);
      v[i].x = -INFINITY;
    }
    if (!(bits >> (2 * i + 1) & 1)) {
      bad |= !(v[i].y < INFINITY);
      v[i].y = -INFINITY;
    }
  }
  return bad;
}

// ---------------------------------------------------------------------------
// One row's scalars for the gradient: every token's is e (a + b d) with
// d = (z - m) scale and e = 2^d; the row's token has its own.
struct RowScalars {
  float m, a, b, token_grad;
  int32_t zero;  // a row without a gradient
  // Distillation: the kept tokens' gradients are w (q - t).
  double top, log_total, teacher, w;
};

struct Shared {
  uint64_t bar[PIECES];
  Record inbox[MAX_RANKS];
  Record warps[WARPS];
  RowScalars row;
};
// Distillation: the teacher's entries and, a bit per token of the slice, which ids were seen.
struct Kept {
  float value[MAX_TOP], x[MAX_TOP];
  int32_t id[MAX_TOP];  // -1: unused
};

template <int DT> __host__ __device__ constexpr size_t loss_smem(int slice, int op) {
  return sizeof(Shared) + (op == DISTILL ? sizeof(Kept) + size_t(slice) / 8 : 0) + 16 +
         size_t(slice) * sizeof(typename Elem<DT>::T) + 32;
}

__device__ __forceinline__ double warp_sum(double v) {
  return warp_all(v, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ double warp_max(double v) {
  return warp_all(v, [](double a, double b) { return fmax(a, b); });
}

template <int DT, int OP, bool GRAD> struct LossRow {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int N = E::N;
  static constexpr bool ENTROPY = OP != DISTILL;

  const LossParams& p;
  int64_t row;
  int rank, ranks, begin, n, tid;

  __device__ __forceinline__ T logit(int64_t j) const {
    return static_cast<const T*>(p.in.logits)[row * p.in.l_s0 + j * p.in.l_s1];
  }
  __device__ __forceinline__ bool allowed(int64_t j) const {
    return p.in.mask.p == nullptr ||
           (uint32_t(p.in.mask.p[row * p.in.mask.s0 + (j >> 5) * p.in.mask.s1]) >> (j & 31) & 1);
  }
  __device__ __forceinline__ T* grad_at(int64_t j) const {
    return static_cast<T*>(p.grad) + row * p.g_s0 + j * p.g_s1;
  }
  __device__ __forceinline__ bool grad_vector() const {
    return p.g_s1 == 1 && (reinterpret_cast<uintptr_t>(grad_at(begin)) & 15) == 0;
  }

  __device__ __forceinline__ void zero_grad() const {
    if (grad_vector()) {
      uint4* g = reinterpret_cast<uint4*>(grad_at(begin));
      for (int c = tid; c < n / N; c += THREADS) g[c] = make_uint4(0, 0, 0, 0);
      const int i = n / N * N + tid;
      if (i < n) *grad_at(begin + i) = E::put(0.f);
    } else {
      for (int i = tid; i < n; i += THREADS) *grad_at(begin + i) = E::put(0.f);
    }
  }
  __device__ __forceinline__ void outputs(int status, float loss, float logprob, float kl, float entropy) const {
    p.status[row] = status;
    if (OP != LOGPROB) p.loss[row] = loss;
    if (OP != DISTILL) {
      p.logprobs[row] = logprob;
      p.entropy[row] = entropy;
    }
    if (OP == POLICY) p.kl[row] = kl;
  }

  // Warp 0, from the merged records: the token's log-probability and what
  // hangs on it. The row's scalars are in FP64: they cost one warp a few
  // hundred instructions, and differences of logarithms lose no digits.
  __device__ __forceinline__ void token_scalars(Shared& sh, float m, double s, double u, bool bad, double temperature,
                                                int64_t token, float z, bool token_allowed) {
    double log_s = log(s), lp = (double(z) - m) / temperature - log_s, h = log_s - u / s * LN2;
    int status = ES_OK;
    bad |= !(s < double(INFINITY)) || m == INFINITY || token >= p.in.vocab;  // a NaN logit makes s NaN
    double slope = 0, on_entropy = 0, loss = 0, kl = 0;  // of lp and of h
    if (OP == LOGPROB) {
      if (GRAD) {
        slope = p.grad_logprobs.p ? p.grad_logprobs[row] : 0.f;
        on_entropy = p.grad_entropy.p ? p.grad_entropy[row] : 0.f;
      }
    } else {
      const double old = p.old_logprobs[row], adv = p.advantages[row], w = p.weights.p ? p.weights[row] : 1.f;
      const double r = exp(lp - old), plain = r * adv, clipped = fmin(fmax(r, p.ratio_low), p.ratio_high) * adv;
      loss = -fmin(plain, clipped);
      slope = plain <= clipped ? -plain : 0.;
      bad |= !isfinite(old) || !isfinite(adv);
      if (p.ref_logprobs.p) {
        const double ref = p.ref_logprobs[row], d = ref - lp, rise = expm1(d);
        kl = rise - d;
        loss += p.kl_coef * kl;
        slope -= p.kl_coef * rise;
        bad |= !isfinite(ref);
      }
      loss -= p.entropy_coef * h;
      bad |= s > 0 && isfinite(lp) && !(isfinite(float(loss)) && isfinite(float(slope)) && isfinite(float(kl)));
      // Weights multiply as they are: an infinite or NaN one (an overflowed
      // loss scale) shows in the loss and the gradient.
      loss *= w;
      slope *= w;
      on_entropy = -p.entropy_coef * w;
    }
    if (bad) status = ES_INVALID_INPUT;
    else if (s == 0) status = ES_NO_VALID_TOKEN;
    else if (z == -INFINITY || !token_allowed) status = ES_DRAFT_ZERO_PROB;
    if (lane_id() != 0) return;
    const bool ok = status == ES_OK;
    if (rank == 0) outputs(status, ok ? float(loss) : 0.f, ok ? float(lp) : -INFINITY, ok ? float(kl) : 0.f, ok ? float(h) : 0.f);
    if (GRAD) {
      slope /= temperature;
      on_entropy /= temperature;
      RowScalars& r = sh.row;
      r.zero = !ok;
      r.m = m;
      // slope (1[j = t] - p_j) - on_entropy p_j (log p_j + h), with p_j = e / s
      // and log p_j = d ln 2 - log s.
      r.a = float(-(slope + on_entropy * (h - log_s)) / s);
      r.b = float(-on_entropy * LN2 / s);
      r.token_grad = float(-slope * expm1(lp) - on_entropy * exp(lp) * (lp + h));
    }
  }

  // Warp 0, from the merged records of the tokens not kept (m, s): the two
  // distributions over the kept tokens and the bucket.
  __device__ __forceinline__ void distill_scalars(Shared& sh, const Kept& kept, float m, double s, bool bad,
                                                  double temperature) {
    const bool tail = p.rest.p != nullptr;
    const double t_rest = tail ? double(p.rest[row]) : -INFINITY;
    double t_top = t_rest, x_top = s > 0 ? double(m) : -INFINITY;
    for (int k = lane_id(); k < p.k; k += 32)
      if (kept.id[k] >= 0) {
        t_top = fmax(t_top, kept.value[k] / temperature);
        x_top = fmax(x_top, double(kept.x[k]));
      }
    t_top = warp_max(t_top);
    x_top = warp_max(x_top);
    double t_sum = 0, x_sum = 0;
    for (int k = lane_id(); k < p.k; k += 32)
      if (kept.id[k] >= 0) {
        t_sum += exp(kept.value[k] / temperature - t_top);
        x_sum += exp((kept.x[k] - x_top) / temperature);
      }
    const double rest_factor = s > 0 ? exp((m - x_top) / temperature) : 0.;
    t_sum = warp_sum(t_sum) + (tail ? exp(t_rest - t_top) : 0.);
    x_sum = warp_sum(x_sum) + s * rest_factor;
    const double log_t = t_top + log(t_sum), log_x = log(x_sum);
    const double w = p.weights.p ? p.weights[row] : 1.f;
    bad |= !(s < double(INFINITY)) || !isfinite(log_t) || (tail && !(t_rest < INFINITY));
    double loss = 0;
    bool lost = false;  // the student has no mass where the teacher has some
    for (int k = lane_id(); k < p.k; k += 32)
      if (kept.id[k] >= 0) {
        const double lt = kept.value[k] / temperature - log_t, lq = (kept.x[k] - x_top) / temperature - log_x;
        const double t = exp(lt);
        if (t > 0) {
          loss += t * (lt - lq);
          lost |= kept.x[k] == -INFINITY;
        }
      }
    loss = warp_sum(loss);
    lost = __any_sync(0xffffffffu, lost);
    double pull = 1;  // of the tokens not kept: 1 - t_rest / q_rest
    const double lt_rest = t_rest - log_t;
    if (tail && exp(lt_rest) > 0) {
      const double off = lt_rest - (log(s) + (m - x_top) / temperature - log_x);
      loss += exp(lt_rest) * off;
      pull = -expm1(off);
      lost |= !(s > 0);
    }
    int status = ES_OK;
    if (bad) status = ES_INVALID_INPUT;
    else if (x_top == -INFINITY) status = ES_NO_VALID_TOKEN;
    else if (lost) status = ES_DRAFT_ZERO_PROB;
    else if (!isfinite(float(loss))) status = ES_INVALID_INPUT;
    if (lane_id() != 0) return;
    const bool ok = status == ES_OK;
    if (rank == 0) outputs(status, ok ? float(w * loss) : 0.f, 0.f, 0.f, 0.f);
    if (GRAD) {
      RowScalars& r = sh.row;
      r.zero = !ok;
      r.m = m;
      r.a = s > 0 ? float(w / temperature * pull * rest_factor / x_sum) : 0.f;
      r.b = 0.f;
      r.top = x_top;
      r.log_total = log_x;
      r.teacher = log_t;
      r.w = w / temperature;
    }
  }

  // The gradient of this rank's slice from its shared copy.
  template <bool TWO> __device__ __forceinline__ void write_grad(const Slice<DT>& slice, const RowScalars& r, float scale,
                                                                 int token) const {
    const float2 nm = both(-r.m), sc = both(scale), a = both(r.a), b = both(r.b);
    const bool vector = grad_vector();
    for (int c = tid; c < slice.chunks; c += THREADS) {
      float2 v[N / 2];
      unpack<DT>(slice.chunk(c), v);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        float2 d = mul2(add2(v[i], nm), sc);
        if (TWO) d = make_float2(fmaxf(d.x, FAR), fmaxf(d.y, FAR));
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        v[i] = mul2(e, TWO ? fma2(b, d, a) : a);
      }
      if (OP != DISTILL && token / N == c) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          if (token % N == 2 * i) v[i].x = r.token_grad;
          if (token % N == 2 * i + 1) v[i].y = r.token_grad;
        }
      }
      const uint4 q = pack<DT>(v);
      if (vector && (c + 1) * N <= n) {
        *reinterpret_cast<uint4*>(grad_at(begin + c * N)) = q;
      } else if (vector) {
        const T* t = reinterpret_cast<const T*>(&q);
        for (int i = 0; i < n - c * N; ++i) *grad_at(begin + c * N + i) = t[i];
      } else {
        slice.set_chunk(c, q);
      }
    }
    if (vector) return;
    // Gradient rows that do not start on 16 bytes, or have a stride: from
    // shared memory, in whole 16-byte pieces where both sides are aligned alike.
    __syncthreads();
    const bool alike = p.g_s1 == 1 && (reinterpret_cast<uintptr_t>(grad_at(begin)) & 15) == slice.shift;
    if (alike) {
      const int head = min(int((16 - slice.shift) & 15) / int(sizeof(T)), n), whole = (n - head) / N;
      const uint4* s = reinterpret_cast<const uint4*>(&slice[head]);
      uint4* g = reinterpret_cast<uint4*>(grad_at(begin + head));
      for (int c = tid; c < whole; c += THREADS) g[c] = s[c];
      if (tid < head) *grad_at(begin + tid) = slice[tid];
      const int i = head + whole * N + tid;
      if (i < n) *grad_at(begin + i) = slice[i];
    } else {
      for (int i = tid; i < n; i += THREADS) *grad_at(begin + i) = slice[i];
    }
  }

  __device__ __forceinline__ void run(uint8_t* smem) {
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    Kept& kept = *reinterpret_cast<Kept*>(smem + sizeof(Shared));
    uint32_t* seen = reinterpret_cast<uint32_t*>(smem + sizeof(Shared) + sizeof(Kept));
    uint8_t* buffer = smem + ((sizeof(Shared) + (OP == DISTILL ? sizeof(Kept) + size_t(p.in.slice) / 8 : 0) + 15) & ~size_t(15));

    // The row's token, or the teacher's entries; rows without are not read.
    int64_t token = -1;
    float z = 0.f, x = 0.f;
    bool token_allowed = true, bad = false;
    int id = -1;
    if (OP != DISTILL) {
      token = p.tokens[row];
    } else {
      float value = 0.f;
      int64_t wide = -1;
      if (tid < p.k) {
        wide = p.ids.p[row * p.ids.s0 + tid * p.ids.s1];
        value = p.values.p[row * p.values.s0 + tid * p.values.s1];
      }
      if (__syncthreads_or(wide >= 0)) token = 0;
      if (wide >= 0) {
        bad |= wide >= p.in.vocab || !(value < INFINITY);
        id = wide < p.in.vocab ? int(wide) : -1;
      }
      if (tid < p.k) {
        kept.id[tid] = id;
        kept.value[tid] = value;
      }
      for (int i = tid; i < p.in.slice / 32; i += THREADS) seen[i] = 0;
    }
    if (token < 0) {
      if (GRAD) zero_grad();
      if (rank == 0 && tid == 0) outputs(ES_OK, 0.f, 0.f, 0.f, 0.f);
      return;
    }
    cluster_arrive();  // this rank's shared memory may be written from now on
    double temperature = p.in.temperature.p ? p.in.temperature[row] : p.in.temperature_all;
    float scale = float(LOG2E / temperature);
    if (!(temperature > 0 && scale >= 1.17549435e-38f && scale <= 3.402823466e38f)) {
      bad = true;
      temperature = 1;
      scale = float(LOG2E);
    }
    Slice<DT> slice;
    slice.load(p.in, row, begin, n, buffer, sh.bar);
    if (OP != DISTILL) {
      if (warp_id() == 0 && token < p.in.vocab) {
        z = E::get(logit(token));
        token_allowed = allowed(token);
      }
    } else {
      if (id >= 0) {
        x = E::get(logit(id));
        bad |= !(x < INFINITY);
        if (!allowed(id)) x = -INFINITY;
      }
      if (tid < p.k) kept.x[tid] = x;
      slice.wait_all();
      // The kept tokens leave the slice, so that what is summed is the others.
      const int local = id - begin;
      if (id >= 0 && local >= 0 && local < n) {
        bad |= (atomicOr(&seen[local >> 5], 1u << (local & 31)) >> (local & 31)) & 1;
        slice[local] = E::put(-INFINITY);
      }
      __syncthreads();
    }

    Acc acc = acc_none();
    const int32_t* mask = p.in.mask.p ? p.in.mask.p + row * p.in.mask.s0 : nullptr;
    for (int c = tid; c < slice.chunks; c += THREADS) {
      slice.wait(uint32_t(c - tid + THREADS + 1) * 16);
      float2 v[N / 2];
      unpack<DT>(slice.chunk(c), v);
      if (mask) {
        bad |= mask_chunk<DT>(mask, p.in.mask.s1, begin + c * N, v);
        if (GRAD) slice.set_chunk(c, pack<DT>(v));
      }
      acc_chunk<N, ENTROPY>(acc, v, scale);
    }
    slice.wait_all();
    Record rec = {acc.m, __fadd_rn(acc.s.x, acc.s.y), __fadd_rn(acc.u.x, acc.u.y), uint32_t(bad || slice.late)};
#pragma unroll
    for (int o = 16; o; o >>= 1) rec = merge(rec, shfl_record(rec, o), scale);
    if (lane_id() == 0) sh.warps[warp_id()] = rec;
    cluster_wait();  // every rank has started
    __syncthreads();
    if (warp_id() == 0) {
      rec = sh.warps[lane_id() & (WARPS - 1)];
#pragma unroll
      for (int o = WARPS / 2; o; o >>= 1) rec = merge(rec, shfl_record(rec, o), scale);
      if (lane_id() < ranks) cg::this_cluster().map_shared_rank(sh.inbox, lane_id())[rank] = rec;
    }
    cluster_arrive();
    cluster_wait();
    if (!GRAD && rank != 0) return;
    if (warp_id() == 0) {
      const bool mine = lane_id() < ranks;
      rec = mine ? sh.inbox[lane_id()] : Record{LOWEST, 0.f, 0.f, 0u};
      const float m = warp_all(rec.m, [](float a, float b) { return fmaxf(a, b); });
      const float d = exponent(rec.m, m, scale);
      const double f = exp2f(d), s = warp_sum(f * rec.s), u = warp_sum(f * (double(rec.u) + double(d) * rec.s));
      bad = __any_sync(0xffffffffu, rec.bad != 0);
      if (OP == DISTILL) distill_scalars(sh, kept, m, s, bad, temperature);
      else token_scalars(sh, m, s, u, bad, temperature, token, z, token_allowed);
    }
    if (!GRAD) return;
    __syncthreads();
    const RowScalars& r = sh.row;
    if (r.zero) {
      zero_grad();
      return;
    }
    const int64_t local = token - begin;
    const int at = OP != DISTILL && local >= 0 && local < n ? int(local) : -N;
    if (r.b != 0.f) write_grad<true>(slice, r, scale, at);
    else write_grad<false>(slice, r, scale, at);
    if (OP == DISTILL) {
      __syncthreads();  // after the slice's zeros at these places
      const int at_id = id - begin;
      if (id >= 0 && at_id >= 0 && at_id < n) {
        const double q = exp((x - r.top) / temperature - r.log_total), t = exp(kept.value[tid] / temperature - r.teacher);
        *grad_at(id) = E::put(float(r.w * (q - t)));
      }
    }
  }
};

// Five blocks to an SM, so that some load while others exchange or write.
template <int DT, int OP, bool GRAD>
__global__ void __launch_bounds__(THREADS, 4) loss_rows(const __grid_constant__ LossParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = p.in.ranks, rank = int(blockIdx.x % unsigned(ranks));
  const int begin = rank * p.in.slice, n = min(p.in.slice, p.in.vocab - begin);
  LossRow<DT, OP, GRAD> work{p, int64_t(blockIdx.x / unsigned(ranks)), rank, ranks, begin, n, int(threadIdx.x)};
  work.run(smem);
}

// Launches `rows` clusters of `ranks` blocks. A kernel's attributes are set
// once per device, to the most that any call needs.
template <class P>
cudaError_t launch_clusters(void (*kernel)(P), const P& p, int64_t rows, int ranks, size_t smem, cudaStream_t stream,
                            std::atomic<uint64_t>& configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev > 63 || !(configured.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    if (dev <= 63) configured.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(rows * ranks), 1, 1);
  config.blockDim = dim3(THREADS, 1, 1);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, p);
}

template <int DT, int OP, bool GRAD> cudaError_t launch_one(const LossParams& p, int64_t rows, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  return launch_clusters(loss_rows<DT, OP, GRAD>, p, rows, p.in.ranks, loss_smem<DT>(p.in.slice, OP), stream, configured);
}
template <int DT> cudaError_t launch_loss(const LossParams& p, int op, int64_t rows, cudaStream_t stream) {
  const bool grad = p.grad != nullptr;
  switch (op) {
    case LOGPROB: return grad ? launch_one<DT, LOGPROB, true>(p, rows, stream) : launch_one<DT, LOGPROB, false>(p, rows, stream);
    case POLICY: return grad ? launch_one<DT, POLICY, true>(p, rows, stream) : launch_one<DT, POLICY, false>(p, rows, stream);
    default: return grad ? launch_one<DT, DISTILL, true>(p, rows, stream) : launch_one<DT, DISTILL, false>(p, rows, stream);
  }
}

}  // namespace score
}  // namespace es
