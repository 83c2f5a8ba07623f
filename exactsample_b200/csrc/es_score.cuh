// Row operators on logits: token log-probabilities, the clipped policy loss
// and the distillation loss, each with its gradient (loss_rows), from one
// read of the row.
//
// A row is split over the ranks of one thread-block cluster in contiguous
// slices, and each rank keeps its slice in shared memory (about 50 KB, so
// that four blocks share an SM). The row is read from HBM once: the first
// pass over the slice takes the sums, the ranks exchange them, and the
// gradient is written from the same shared copy. A loss with its gradient so
// moves one read and one write of the row, where a row that does not stay on
// the chip needs two reads and one write.
//
// Bounds: the HBM, then the exponentials (two a token, 16 a cycle and SM:
// about 70 % of the time that 2-byte rows take at full HBM rate), then latency
// between the passes. Measured on B200s, 4,096 rows of 151,936 bf16: the
// policy step takes 453 to 476 us in runs of 20, by the card (5.2 to 5.5 TB/s,
// 80 to 84 % of a copy's rate), and 500 to 510 in runs of seconds, whose clocks
// are lower (75 %). Without any exponential the same loops took 408 us where it
// took 453.
//
// The split depends on the vocabulary and the type alone, and every thread
// takes the same elements whatever the row's address, so a row's results are
// the same bits in any batch and at any alignment.
#pragma once
#include <algorithm>
#include <atomic>

#include "es_device.cuh"

namespace es {
namespace score {

enum Op { LOGPROB = 0, POLICY = 1, DISTILL = 2 };
constexpr int THREADS = 128, WARPS = THREADS / 32, BLOCKS = 4;  // blocks: to an SM (see loss_rows)
constexpr int MAX_RANKS = 16;   // cluster size (beyond 8: non-portable, as for the row kernels)
constexpr int MAX_TOP = ES_MAX_TOP;
constexpr int STEP = 4 * THREADS;  // chunks that the block takes at a time, four a thread
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

// 1 / temperature in two floats, and log2(e) / temperature.
struct Scale {
  float log2;      // of the exponents
  float hi, lo;    // 1 / temperature
  bool bad;        // not positive and finite, or beyond float32's range
};
__host__ __device__ inline Scale scale_of(double temperature) {
  const double inv = 1. / temperature;
  Scale s;
  s.log2 = float(LOG2E * inv);
  s.bad = !(s.log2 >= 1.17549435e-38f && s.log2 <= 3.402823466e38f);
  s.hi = float(inv);
  s.lo = float(inv - double(s.hi));
  if (s.bad) s = {float(LOG2E), 1.f, 0.f, true};
  return s;
}

struct Rows {
  const void* logits;
  int64_t l_s0, l_s1;
  Grid2<const int32_t> mask;
  Column<const double> temperature;
  Scale all;  // where the temperature is one number
  int64_t rows;
  int32_t vocab, ranks, slice;
};

__device__ __forceinline__ Scale row_scale(const Rows& in, int64_t row) {
  return in.temperature.p ? scale_of(in.temperature[row]) : in.all;
}

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
  Column<const int32_t> teacher_status;
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
// Sums over logits against a reference m, one of them: s = sum 2^d and u = sum
// 2^d d with d = (z - m) scale: everything a row's log-sum and entropy need.
// scale = log2(e) / temperature. s and u are held as two partial sums.
//
// The fast forms take d = z scale - r in one instruction, with r = m scale
// rounded to 32 bits; acc_exact afterwards makes s and u those of m itself.
// Their m is not the maximum, which took a third of the pass to look for, but
// the largest of a warp's first tokens, and in the thread that has the row's
// token that token's logit if it is larger. d's rounding grows with it, and the
// entropy, log s - u / s, loses what log s and u / s have in common, so that m
// should not lie far below where the mass is. A row whose token has most of it,
// as most rows do, so has the maximum itself for m. (With the first tokens alone
// a row whose peak was 22 nats above the others had an entropy of 7.6e-4 with an
// error of 7e-6, and at 30 nats half of the log-probabilities were above 0.) The
// fast forms leave some rows wrong, and acc_failed tells: sums of MOST and more,
// a -inf beside an entropy (0 * -inf), an r that overflows, and an r so large
// that its rounding moves the exponents. The careful form, which keeps the
// running maximum, subtracts first and holds exponents at FAR, is right for those.
struct Acc {
  float m, r;
  float2 s, u;
};
// At or below this a maximum is none yet: in the fast form a masked token's
// logit lies below it (MASKED), and a real one fails (LARGE_R).
constexpr float NONE = -1e29f;
__device__ __forceinline__ Acc acc_none(float m = -INFINITY) { return {m, 0.f, {0.f, 0.f}, {0.f, 0.f}}; }
__device__ __forceinline__ float exponent(float z, float m, float scale) {
  return max_nan(__fmul_rn(__fsub_rn(z, m), scale), FAR);
}
// The largest of two chunks; a NaN may drop out here, and shows up in s.
template <int DT> __device__ __forceinline__ float chunk_max(const uint4& p, const uint4& q) {
  if constexpr (DT == ES_F32) {
    const float* a = reinterpret_cast<const float*>(&p);
    const float* b = reinterpret_cast<const float*>(&q);
    return fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(b[0], b[1]), fmaxf(b[2], b[3])));
  } else if constexpr (DT == ES_F16) {
    const __half2* a = reinterpret_cast<const __half2*>(&p);
    const __half2* b = reinterpret_cast<const __half2*>(&q);
    const float2 m = __half22float2(__hmax2(__hmax2(__hmax2(a[0], a[1]), __hmax2(a[2], a[3])),
                                            __hmax2(__hmax2(b[0], b[1]), __hmax2(b[2], b[3]))));
    return fmaxf(m.x, m.y);
  } else {
    const __nv_bfloat162* a = reinterpret_cast<const __nv_bfloat162*>(&p);
    const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&q);
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(__hmax2(a[0], a[1]), __hmax2(a[2], a[3])),
                                                __hmax2(__hmax2(b[0], b[1]), __hmax2(b[2], b[3]))));
    return fmaxf(m.x, m.y);
  }
}
// Whether a chunk holds a -inf.
template <int DT> __device__ __forceinline__ bool chunk_has_lowest(const uint4& q) {
  if constexpr (DT == ES_F32) {
    const float* a = reinterpret_cast<const float*>(&q);
    return fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) == -INFINITY;
  } else if constexpr (DT == ES_F16) {
    const __half2* a = reinterpret_cast<const __half2*>(&q);
    const float2 m = __half22float2(__hmin2(__hmin2(a[0], a[1]), __hmin2(a[2], a[3])));
    return fminf(m.x, m.y) == -INFINITY;
  } else {
    const __nv_bfloat162* a = reinterpret_cast<const __nv_bfloat162*>(&q);
    const float2 m = __bfloat1622float2(__hmin2(__hmin2(a[0], a[1]), __hmin2(a[2], a[3])));
    return fminf(m.x, m.y) == -INFINITY;
  }
}
// The largest of a chunk, and NaN if there is one.
template <int DT> __device__ __forceinline__ float chunk_max_nan(const uint4& q) {
  if constexpr (DT == ES_F32) {
    return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
  } else if constexpr (DT == ES_F16) {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m)));
  }
}
template <int N, bool ENTROPY> __device__ __forceinline__ void acc_add(Acc& a, const float2* v, float scale) {
  const float2 nr = both(-a.r), sc = both(scale);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 d = fma2(v[i], sc, nr);
    const float2 e = make_float2(ex2(d.x), ex2(d.y));
    a.s = add2(a.s, e);
    if (ENTROPY) a.u = fma2(e, d, a.u);
  }
}
// Raises the reference to `top` if that is 2^16 above it (masked rows, whose
// first tokens may all be masked).
__device__ __forceinline__ float raise_limit(float m, float scale) { return __fadd_rn(m, __fdividef(16.f, scale)); }
template <bool ENTROPY> __device__ __forceinline__ void acc_raise(Acc& a, float top, float scale, float& limit) {
  if (top > limit) {
    const float r = __fmul_rn(top, scale), d = __fsub_rn(a.r, r), f = a.m <= NONE ? 0.f : ex2(d);
    if (ENTROPY) a.u = mul2(both(f), fma2(both(fmaxf(d, FAR)), a.s, a.u));
    a.s = mul2(both(f), a.s);
    a.m = top;
    a.r = r;
    limit = raise_limit(top, scale);
  }
}
template <int N, bool ENTROPY>
__device__ __forceinline__ void acc_careful(Acc& a, const float2* v, float top, float scale) {
  top = fmaxf(top, LOWEST);
  if (top > a.m) {
    const float d = a.m == -INFINITY ? FAR : exponent(a.m, top, scale), f = ex2(d);
    if (ENTROPY) a.u = mul2(both(f), fma2(both(d), a.s, a.u));
    a.s = mul2(both(f), a.s);
    a.m = top;
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 d = make_float2(exponent(v[i].x, a.m, scale), exponent(v[i].y, a.m, scale));
    const float2 e = make_float2(ex2(d.x), ex2(d.y));
    a.s = add2(a.s, e);
    if (ENTROPY) a.u = fma2(e, d, a.u);
  }
}
// The largest sum of a fast form. With an entropy a sum that large is 17 nats
// above its reference, where log s and u / s are rounded by 1e-6; without one it
// is only to keep a row's coefficient, 1 / s, a normal number.
template <bool ENTROPY> constexpr float MOST = ENTROPY ? 0x1p24f : 0x1p60f;
constexpr float LARGE_R = 65536.f;  // its rounding is 2^-8 at most, which acc_exact takes back
template <bool ENTROPY> __device__ __forceinline__ bool acc_failed(const Acc& a) {
  const float s = a.s.x + a.s.y, u = a.u.x + a.u.y;
  return !(fabsf(a.r) <= LARGE_R) || !(s < MOST<ENTROPY>) || (ENTROPY && !(fabsf(u) < 0x1p67f));
}

// What one rank knows of its slice: s and u against the maximum m.
struct alignas(16) Record {
  float m, s, u;
  uint32_t flags;
};
// BAD: an invalid row (a NaN or +inf, a repeated id, a copy that did not
// arrive). CAREFUL: the gradient needs the careful form too. HELD: it needs
// the slice's -inf held at MASKED. FULL: top_rows'
// lists did not fit.
constexpr uint32_t BAD = 1, CAREFUL = 2, FULL = 4, HELD = 8;

// s and u against m itself: with m scale = r + rest, 2^(z scale - r) is 2^rest
// times too large and its exponent off by rest (at most 2^-8).
template <bool ENTROPY> __device__ __forceinline__ Record acc_exact(const Acc& a, float scale, bool careful) {
  const float rest = careful || a.m <= NONE ? 0.f : __fmaf_rn(a.m, scale, -a.r), f = ex2(-rest);
  const float s = __fadd_rn(a.s.x, a.s.y), u = __fadd_rn(a.u.x, a.u.y);
  return {s == 0.f ? LOWEST : fmaxf(a.m, LOWEST), __fmul_rn(f, s), ENTROPY ? __fmul_rn(f, __fmaf_rn(-rest, s, u)) : 0.f, careful ? CAREFUL : 0u};
}
// The records of LANES neighbouring lanes as one, in every lane. Every warp of
// a block takes it, not in a branch: where the compiler cannot tell that a
// whole warp is there, a shuffle costs about 240 cycles instead of 25 (3,600
// for the 16 of a whole warp's record, measured).
template <bool ENTROPY, int LANES> __device__ __forceinline__ Record lanes_record(Record r, float scale) {
  float m = r.m;
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) m = fmaxf(m, shfl_xor(m, o));
  const float d = exponent(r.m, m, scale), f = ex2(d);
  if (ENTROPY) r.u = __fmul_rn(f, __fmaf_rn(d, r.s, r.u));
  r.s = __fmul_rn(f, r.s);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) {
    r.s = __fadd_rn(r.s, shfl_xor(r.s, o));
    if (ENTROPY) r.u = __fadd_rn(r.u, shfl_xor(r.u, o));
    if (LANES < 32) r.flags |= shfl_xor(r.flags, o);
  }
  if (LANES == 32) r.flags = __reduce_or_sync(0xffffffffu, r.flags);
  r.m = m;
  return r;
}
// `count` records of at most LANES as one, in every lane.
template <bool ENTROPY, int LANES>
__device__ __forceinline__ Record join_records(const Record* records, int count, float scale) {
  const int lane = lane_id() & (LANES - 1);
  const bool mine = lane < count;
  Record r = records[mine ? lane : 0];
  r.m = mine ? r.m : LOWEST;
  r.s = mine ? r.s : 0.f;
  r.u = mine ? r.u : 0.f;
  r.flags = mine ? r.flags : 0u;
  return lanes_record<ENTROPY, LANES>(r, scale);
}

// ---------------------------------------------------------------------------
// Cluster barrier halves: between them a rank does work of its own.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
// Before any access to another rank's memory there is nothing to release but
// the initialisation of barriers, which has its own fence.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }

// A record into another rank's shared memory, counted by that rank's barrier:
// the receiver waits on its own barrier alone, and the sender for nothing.
__device__ __forceinline__ void send_record(Record* to, uint64_t* bar, int rank, const Record& r) {
  uint32_t address, barrier;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(smem_addr(to)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(barrier) : "r"(smem_addr(bar)), "r"(rank));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(address),
               "r"(__float_as_uint(r.m)), "r"(__float_as_uint(r.s)), "r"(__float_as_uint(r.u)), "r"(r.flags), "r"(barrier)
               : "memory");
}
// Whether a barrier's phase completed in time.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity) {
  uint32_t spins = 0;
  while (!mbar_try_wait(bar, parity))
    if (++spins >= WAIT_LIMIT) return false;
  return true;
}

// 16 bytes from global to shared memory, without passing through registers;
// a thread's own copies are there after its copies_done.
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int GROUPS> __device__ __forceinline__ void copies_done() {  // all but the last GROUPS groups
  asm volatile("cp.async.wait_group %0;" ::"n"(GROUPS) : "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// ---------------------------------------------------------------------------
// 16 bytes at `shift` bytes into the 32 of two pieces; shift below 16.
template <int SIZE> __device__ __forceinline__ uint4 shifted_chunk(const uint4& a, const uint4& b, uint32_t shift) {
  uint32_t w[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 2];
    w[5] = b.w;
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (SIZE == 2 && (shift & 2)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Chunk c of n elements that start anywhere and lie `stride` apart, -inf past
// the end. Inside, a chunk that does not start on 16 bytes is cut out of the
// two aligned pieces that it lies in.
template <int DT>
__device__ __forceinline__ uint4 fetch_chunk(const typename Elem<DT>::T* src, int64_t stride, int c, int n) {
  using T = typename Elem<DT>::T;
  constexpr int N = Elem<DT>::N;
  const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(src)) & 15;
  if (stride == 1 && c > 0 && (c + 2) * N <= n) {
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) - shift) + c;
    const uint4 a = from[0], b = from[shift ? 1 : 0];
    return shifted_chunk<sizeof(T)>(a, b, shift);
  }
  uint4 q;
  T* v = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c * N + i < n ? src[(c * N + i) * stride] : Elem<DT>::put(-INFINITY);
  return q;
}

// A rank's slice of the row in shared memory, element i at base + i sizeof(T).
// Chunk c is brought, read and written by thread c mod THREADS alone, so that
// its way needs no barrier. Rows that start on 16 bytes come by asynchronous
// copies of whole chunks, rows that start on 4 by copies of words, and 2-byte
// rows between words by copies of words too, one element off: realign puts
// them right. Rows with a stride pass through registers. (1,001 rows of 50,257
// through distill_loss and its backward pass: float32 207 us, bf16 164; with
// such rows through registers 371 and 238; rows of 50,256 take 174 and 131.)
template <int DT> struct Slice {
  using T = typename Elem<DT>::T;
  static constexpr int N = Elem<DT>::N;
  uint8_t* base;
  int n, chunks, half;  // half: chunks of the first of two groups of copies, all of them whole

  __device__ __forceinline__ T& operator[](int i) const { return reinterpret_cast<T*>(base)[i]; }
  __device__ __forceinline__ uint4& chunk(int c) const { return reinterpret_cast<uint4*>(base)[c]; }

  __device__ __forceinline__ void init(uint8_t* buffer, int count) {
    base = buffer;
    n = count;
    chunks = (n + N - 1) / N;
    half = (chunks + 2 * STEP - 1) / (2 * STEP) * STEP;
    if (half >= chunks) half = 0;
  }
  static __device__ __forceinline__ const T* source(const Rows& in, int64_t row, int begin) {
    return static_cast<const T*>(in.logits) + row * in.l_s0 + int64_t(begin) * in.l_s1;
  }
  // How a row comes: 16 or 4 bytes a copy, 2 for words one element off, 0 for none.
  static __device__ __forceinline__ int width(const Rows& in, const T* src) {
    const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(src)) & 15;
    return in.l_s1 != 1 ? 0 : off == 0 ? 16 : off % 4 == 0 ? 4 : 2;
  }
  // Chunk c of a row that has a width; a whole one.
  __device__ __forceinline__ void copy(int c, const T* src, int width) const {
    uint32_t* to = reinterpret_cast<uint32_t*>(&chunk(c));
    if (width == 16) {
      copy_async(to, reinterpret_cast<const uint4*>(src) + c);
    } else if (width == 4) {
      const uint32_t* from = reinterpret_cast<const uint32_t*>(src) + 4 * c;
#pragma unroll
      for (int i = 0; i < 4; ++i) copy_async4(to + i, from + i);
    } else {
      // Elements N c - 1 to N c + N - 2; the slice's first has none before it.
      const uint32_t* from = reinterpret_cast<const uint32_t*>(src - 1) + 4 * c;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i > 0 || c > 0) copy_async4(to + i, from + i);
      if (c == 0) (*this)[1] = src[0];
    }
  }
  // What whole chunks leave of a row that has a width, by the thread whose
  // place it lies in.
  __device__ __forceinline__ void load_ragged(const T* src, int width) const {
    const int whole = n / N;
    if (int(threadIdx.x) != whole % THREADS) return;
    if (width != 2) {
      if (whole < chunks) chunk(whole) = fetch_chunk<DT>(src, 1, whole, n);
    } else {
      for (int i = whole * N; i <= chunks * N; ++i) (*this)[i] = i > 0 && i <= n ? src[i - 1] : Elem<DT>::put(-INFINITY);
    }
  }
  // All threads: a row of width 2, all there, one element down. A round reads
  // only what no earlier round wrote.
  __device__ __forceinline__ void realign() const {
    __syncthreads();
#pragma unroll 1
    for (int first = 0; first < chunks; first += STEP) {
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = min(first + i * THREADS + int(threadIdx.x), chunks - 1);
        const uint4 a = chunk(c);
        const uint32_t more = reinterpret_cast<const uint32_t*>(&chunk(c + 1))[0];
        q[i] = make_uint4(__funnelshift_r(a.x, a.y, 16), __funnelshift_r(a.y, a.z, 16), __funnelshift_r(a.z, a.w, 16),
                          __funnelshift_r(a.w, more, 16));
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = first + i * THREADS + int(threadIdx.x);
        if (c < chunks) chunk(c) = q[i];
      }
    }
  }
  __device__ __forceinline__ void load(const Rows& in, int64_t row, int begin) const {
    const T* src = source(in, row, begin);
    const int tid = threadIdx.x, whole = n / N, bytes = width(in, src);
    int c = tid;
    if (bytes) {
      for (; c < half; c += THREADS) copy(c, src, bytes);
      copies_end_group();
      for (; c < whole; c += THREADS) copy(c, src, bytes);
      copies_end_group();
      load_ragged(src, bytes);
      return;
    }
    copies_end_group();  // (mask words)
    copies_end_group();
#pragma unroll 1
    for (; c < chunks; c += 4 * THREADS) {
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i * THREADS < chunks) q[i] = fetch_chunk<DT>(src, in.l_s1, c + i * THREADS, n);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i * THREADS < chunks) chunk(c + i * THREADS) = q[i];
    }
  }
  // After this a thread may read its chunks below `half`, and after
  // arrive_rest all of them.
  __device__ __forceinline__ void arrive() const { copies_done<1>(); }
  __device__ __forceinline__ void arrive_rest() const { copies_done<0>(); }
};

// What a masked token's logit becomes in the fast form: 2^d is 0 there, and 0
// times d is too. (Rows with a real logit near it, or a scale that brings it
// near 0, take the careful form: LARGE_R, SMALL_SCALE.) float16 has no such
// number; its masked logits are -inf and held at MASKED in 32 bits.
constexpr float MASKED = -1e30f;
constexpr float SMALL_SCALE = 1e-20f;
// The gradient 2^d (a + b d) is 0 at such a token if b d is finite: in float16
// d is MASKED scale there at the lowest, elsewhere a logit may bring it down to
// the type's lowest number. Rows with a larger b take the careful form, whose
// d stops at FAR (a gradient with an entropy part of 1,024 rows of 151,936
// bf16: 125 us, 129 in the careful form; a product more in every row's fast
// form made a policy step of 4,096 rows 0.5 to 2 % slower).
template <int DT> __device__ __forceinline__ float largest_b(float scale) {
  return DT == ES_F16 ? __fdividef(1e8f, scale) : 0.99f;
}
template <int DT> __device__ __forceinline__ uint32_t masked_word() {
  if constexpr (DT == ES_F32) return __float_as_uint(MASKED);
  const typename Elem<DT>::T v = Elem<DT>::put(MASKED);
  const uint32_t bits = *reinterpret_cast<const uint16_t*>(&v);
  return bits << 16 | bits;
}
// The N mask bits of a chunk that starts at a slice's token `first`.
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* words, int first) { return words[first >> 5] >> (first & 31); }
// Tokens whose bit is clear become `word`'s value.
template <int DT> __device__ __forceinline__ uint4 mask_chunk(const uint4& q, uint32_t bits, uint32_t word) {
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (DT == ES_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t keep = uint32_t(int32_t(bits << (31 - i)) >> 31);
      w[i] = (w[i] & keep) | (word & ~keep);
    }
  } else {
    // Bits 2i and 2i + 1 as the signs of two bytes, each spread over a half word.
    const uint32_t s = (bits & 0x55u) | ((bits & 0xaau) << 7);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t keep;
      asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(keep) : "r"(s << (7 - 2 * i)));  // 8 + b: byte b's sign, eight times
      w[i] = (w[i] & keep) | (word & ~keep);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A chunk's -inf at MASKED (not for float16).
template <int DT> __device__ __forceinline__ uint4 hold_chunk(const uint4& q) {
  uint4 r = q;
  if constexpr (DT == ES_F32) {
    float* v = reinterpret_cast<float*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = max_nan(v[i], MASKED);
  } else if constexpr (DT == ES_BF16) {
    __nv_bfloat162* v = reinterpret_cast<__nv_bfloat162*>(&r);
    const uint32_t word = masked_word<DT>();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmax2_nan(v[i], reinterpret_cast<const __nv_bfloat162&>(word));
  }
  return r;
}
template <int DT> __device__ __forceinline__ uint32_t lowest_word() {  // -inf
  return DT == ES_F32 ? 0xff800000u : DT == ES_F16 ? 0xfc00fc00u : 0xff80ff80u;
}
template <int N> __device__ __forceinline__ float max_of(const float2* v) {
  float top = fmaxf(v[0].x, v[0].y);
#pragma unroll
  for (int i = 1; i < N / 2; ++i) top = fmaxf(top, fmaxf(v[i].x, v[i].y));
  return top;
}

// This thread's share of a slice as a Record: the fast form, or where that
// fails the careful one. The slice has arrived up to `half`. `words`: a
// MASKED_ROW's mask; its masked tokens are masked in the slice too. `token`: the
// row's, if it lies in the slice, or negative. An
// OPEN_ROW's warps that see a -inf among their first tokens (rows that were
// masked before) hold every -inf at MASKED instead; those that meet one later
// take the careful form. (1,024 rows of 151,936 bf16 with a
// fifth of -inf, log-probabilities and policy step: 137 and 191 us in
// the careful form, 81 and 131 so, 74 and 127 without a -inf.)
enum RowKind { OPEN_ROW, MASKED_ROW, HELD_ROW };
template <int DT, bool ENTROPY, int KIND>
__device__ __forceinline__ Record sum_slice(const Slice<DT>& slice, const uint32_t* words, int token, float scale) {
  constexpr int N = Elem<DT>::N;
  constexpr bool HAS_MASK = KIND == MASKED_ROW, RAISE = KIND != OPEN_ROW;
  constexpr bool HOLD = RAISE && ENTROPY && DT == ES_F16;
  const int tid = threadIdx.x, whole = slice.n / N;
  float seen_top = -INFINITY;  // of masked rows' logits, a NaN kept
  uint32_t any = 0;            // mask bits seen, or whether a token is not -inf
  Acc a = acc_none(RAISE ? NONE : -INFINITY);
  // A chunk as it is summed; returns its maximum where that is asked for.
  const auto take = [&](uint4& q, int c) {
    float top = -INFINITY;
    if (KIND == HELD_ROW) {
      top = chunk_max<DT>(q, q);
      any |= top > -INFINITY;
      q = hold_chunk<DT>(q);
    }
    if (HAS_MASK) {
      const uint32_t bits = mask_bits(words, c * N) & ((1u << N) - 1u);
      any |= bits;
      seen_top = max_nan(seen_top, chunk_max_nan<DT>(q));
      q = mask_chunk<DT>(q, bits, masked_word<DT>());
    }
    if (HAS_MASK) slice.chunk(c) = q;
    return top;
  };
  const auto hold = [&](float2* v, int pairs) {
#pragma unroll
    for (int i = 0; i < pairs; ++i) v[i] = make_float2(max_nan(v[i].x, MASKED), max_nan(v[i].y, MASKED));
  };
  bool held = KIND == HELD_ROW;
  bool blank = false;  // no reference among the first tokens
  float limit = NONE;
  if (slice.half == 0) slice.arrive_rest();
  if (KIND == OPEN_ROW) {
    float top = -INFINITY;
    bool lowest = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (tid + i * THREADS < slice.chunks && (i == 0 || slice.half > 0)) {
        const uint4 q = slice.chunk(tid + i * THREADS);
        top = fmaxf(top, chunk_max<DT>(q, q));
        if (ENTROPY) lowest |= chunk_has_lowest<DT>(q);
      }
    if (ENTROPY && __any_sync(0xffffffffu, lowest)) return sum_slice<DT, ENTROPY, ENTROPY ? HELD_ROW : OPEN_ROW>(slice, words, token, scale);
    top = warp_all(top, [](float x, float y) { return fmaxf(x, y); });
    blank = !(top > -INFINITY);
    a.m = blank ? 0.f : top;
    a.r = __fmul_rn(a.m, scale);
  }
  // The thread that has the row's token takes its logit for the reference.
  if (ENTROPY && token >= 0 && token / N % THREADS == tid) {
    if (token / N >= slice.half) slice.arrive_rest();
    const float z = Elem<DT>::get(slice[token]);
    if (z > a.m && (!HAS_MASK || mask_bits(words, token) & 1)) {
      a.m = z;
      a.r = __fmul_rn(z, scale);
      if (RAISE) limit = raise_limit(z, scale);
    }
  }
  // Four chunks a step, for independent loads and exponentials.
  int c = tid;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    if (part) slice.arrive_rest();
    const int end = part ? whole : slice.half;
#pragma unroll 1
    for (; c + 3 * THREADS < end; c += STEP) {
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = slice.chunk(c + i * THREADS);
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, take(q[i], c + i * THREADS));
      if (HAS_MASK) top = fmaxf(chunk_max<DT>(q[0], q[1]), chunk_max<DT>(q[2], q[3]));
      if (RAISE) acc_raise<ENTROPY>(a, top, scale, limit);
      float2 v[2 * N];
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack<DT>(q[i], v + i * N / 2);
      if (HOLD) hold(v, 2 * N);
      acc_add<4 * N, ENTROPY>(a, v, scale);
    }
  }
#pragma unroll 1
  for (; c < slice.chunks; c += THREADS) {
    uint4 q = slice.chunk(c);
    float top = take(q, c);
    if (HAS_MASK) top = chunk_max<DT>(q, q);
    if (RAISE) acc_raise<ENTROPY>(a, top, scale, limit);
    float2 v[N / 2];
    unpack<DT>(q, v);
    if (HOLD || (ENTROPY && c >= whole)) hold(v, N / 2);  // (the last chunk is filled up with -inf)
    if (ENTROPY && c >= whole)
      for (int i = c * N; i < slice.n; ++i) held |= Elem<DT>::get(slice[i]) == -INFINITY;
    acc_add<N, ENTROPY>(a, v, scale);
  }
  // (A thread without chunks has nothing to fail on, and its warp's reference may overflow.)
  const bool failed = blank || acc_failed<ENTROPY>(a) || scale < SMALL_SCALE || (RAISE && any && a.m <= NONE);
  if (failed || tid >= slice.chunks) {
    a = acc_none();
#pragma unroll 1
    for (c = tid; c < slice.chunks; c += THREADS) {
      uint4 q = slice.chunk(c);
      if (HAS_MASK) q = mask_chunk<DT>(q, mask_bits(words, c * N), lowest_word<DT>());
      float2 v[N / 2];
      unpack<DT>(q, v);
      acc_careful<N, ENTROPY>(a, v, max_of<N>(v), scale);
    }
  }
  Record r = acc_exact<ENTROPY>(a, scale, failed && tid < slice.chunks);
  if (HAS_MASK && !(seen_top < INFINITY)) r.flags |= BAD;
  if (held) r.flags |= HELD;
  return r;
}

// ---------------------------------------------------------------------------
// Row scalars. They sit between the row's two passes on one thread, and FP64
// there costs about 4 us a row (FP64 operations are several times slower to
// follow one another than FP32's). Logarithms are held as a float and the
// float it is off by instead, so that differences of them lose no digits.
struct Pair {
  float hi, lo;
};
__device__ __forceinline__ Pair pair_sum(Pair a, Pair b) {
  const float hi = __fadd_rn(a.hi, b.hi), t = __fsub_rn(hi, a.hi);  // hi + rest is a.hi + b.hi exactly
  const float rest = __fadd_rn(__fsub_rn(a.hi, __fsub_rn(hi, t)), __fsub_rn(b.hi, t));
  return {hi, __fadd_rn(rest, __fadd_rn(a.lo, b.lo))};
}
__device__ __forceinline__ Pair negated(Pair a) { return {-a.hi, -a.lo}; }
__device__ __forceinline__ float value_of(Pair a) { return __fadd_rn(a.hi, a.lo); }
// (a - b) / temperature; of finite numbers a finite one (a type's lowest value
// over a temperature below 1 leaves the range, and pairs of infinities are NaN).
__device__ __forceinline__ Pair scaled_gap(float a, float b, const Scale& s) {
  const float hi = __fsub_rn(a, b), t = __fadd_rn(hi, b);
  const float rest = __fsub_rn(__fsub_rn(a, t), __fsub_rn(b, __fsub_rn(t, hi)));  // a - b = hi + rest
  const float p = __fmul_rn(hi, s.hi);
  if (fabsf(p) == INFINITY && fabsf(a) < INFINITY && fabsf(b) < INFINITY) return {copysignf(-LOWEST, hi), 0.f};
  return {p, __fmaf_rn(hi, s.hi, -p) + (hi * s.lo + rest * s.hi)};
}
// log(s) for a positive, normal s, to about 2^-32: with s = 2^k f, f in
// [3/4, 3/2), log f = 2 artanh(q) = 2 (q + q^3 / 3 + q^5 / 5 + ...) at
// q = (f - 1) / (f + 1), |q| <= 1/5.
__device__ __forceinline__ Pair log_pair(float s) {
  const int bits = __float_as_int(s), k = (bits - 0x3f400000) >> 23;
  const float f = __int_as_float(bits - (k << 23));
  const float num = f - 1.f, den = f + 1.f, den_lo = f - (den - 1.f), inv = __frcp_rn(den);
  const float q = __fmul_rn(num, inv), q_lo = (__fmaf_rn(-q, den, num) - q * den_lo) * inv;
  const float u = q * q;
  const float series = q * u * __fmaf_rn(u, __fmaf_rn(u, __fmaf_rn(u, __fmaf_rn(u, 2.f / 11.f, 2.f / 9.f), 2.f / 7.f), 2.f / 5.f), 2.f / 3.f);
  constexpr float LN2_HI = 0.693145751953125f;  // 16 bits: its products with k are exact
  constexpr float LN2_LO = float(LN2 - double(LN2_HI));
  return pair_sum({float(k) * LN2_HI, 0.f}, {2.f * q, __fmaf_rn(2.f, q_lo, __fmaf_rn(float(k), LN2_LO, series))});
}
// exp(x) - 1 - x, from its series where the difference would lose digits.
__device__ __forceinline__ float exp_beyond_first_order(float x, float exp_less_one) {
  if (fabsf(x) >= 1.f) return exp_less_one - x;
  float sum = 1.f / 3628800.f / 132.f;
  constexpr float C[10] = {1.f / 39916800.f, 1.f / 3628800.f, 1.f / 362880.f, 1.f / 40320.f, 1.f / 5040.f,
                           1.f / 720.f, 1.f / 120.f, 1.f / 24.f, 1.f / 6.f, 1.f / 2.f};
#pragma unroll
  for (int i = 0; i < 10; ++i) sum = __fmaf_rn(sum, x, C[i]);
  return sum * x * x;
}

// Above this an exponential of the row's scalars is taken in 64 bits, since
// its product with an advantage or a coefficient may be in float32's range
// where it is not.
constexpr float WIDE = 80.f;

// One row's scalars for the gradient: every token's is 2^d (a + b d), in the
// fast form with d = z scale - r, in the careful form with d = (z - m) scale;
// the row's token has its own.
struct RowScalars {
  float m, r, a, b, token_grad;
  int32_t zero, careful;   // a row without a gradient; the form
  int32_t held;            // -inf is held at MASKED
  float w, inv_q, inv_t;   // distillation: the kept tokens' gradients are w (q inv_q - t inv_t)
};

// Two of what a row writes while slower warps or ranks may still read the row before's.
struct Shared {
  Record inbox[2][MAX_RANKS];
  Record warps[2][WARPS];
  uint64_t bar[2];
  RowScalars row;
  float sums[WARPS][3];  // distillation: kept_sums by warp
};

// Distillation: the teacher's entries, k of each (rounded up to whole warps):
// their ids (-1: unused) and logits, the row's own logits at them, and the
// exponentials of both; then a bit per token of the slice, which ids were seen.
struct Kept {
  int32_t* id;
  float *value, *x, *t, *q;
  uint32_t* seen;
  static constexpr __host__ __device__ size_t bytes(int k, int slice) {
    return size_t((k + 31) / 32 * 32) * 20 + size_t(slice) / 8;
  }
  __device__ Kept(uint8_t* p, int k) {
    const int width = (k + 31) / 32 * 32;
    id = reinterpret_cast<int32_t*>(p);
    value = reinterpret_cast<float*>(id + width);
    x = value + width;
    t = x + width;
    q = t + width;
    seen = reinterpret_cast<uint32_t*>(q + width);
  }
};

constexpr size_t SHARED_BYTES = (sizeof(Shared) + 15) / 16 * 16;
// The buffer of a slice, and a chunk more for rows that land one element off.
template <int DT> __host__ __device__ constexpr size_t slice_bytes(int slice) {
  return size_t(slice) * sizeof(typename Elem<DT>::T) + 16;
}
// Then two rows' mask words, and the distillation's entries.
__host__ __device__ constexpr size_t mask_bytes(int slice) { return size_t(slice) / 8; }
template <int DT> __host__ __device__ constexpr size_t loss_smem(int slice, bool mask, int k) {
  return SHARED_BYTES + slice_bytes<DT>(slice) + (mask ? 2 * mask_bytes(slice) : 0) + (k > 0 ? Kept::bytes(k, slice) : 0);
}

__device__ __forceinline__ float warp_sum(float v) {
  return warp_all(v, [](float a, float b) { return __fadd_rn(a, b); });
}
__device__ __forceinline__ float warp_top(float v) {
  return warp_all(v, [](float a, float b) { return fmaxf(a, b); });
}

// A cluster takes rows at a stride of all clusters. While a row's gradient is
// written, each thread copies the next row's chunks into the places that it
// has done with: the next row's way from HBM costs no time and no memory.
template <int DT, int OP, bool GRAD> struct LossRow {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int N = E::N;
  static constexpr bool ENTROPY = OP != DISTILL;

  const LossParams& p;
  int64_t row, stride;
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

  // What the row's scalars need besides the sums, fetched while the row is on its way.
  struct Inputs {
    int64_t token;
    T raw;          // the token's logit
    uint32_t mask;  // its mask word
    float first, second, ref, w;  // logprob: the two incoming gradients; policy: old log-probability
                                  // and advantage; distillation: the teacher's rest
  };

  // a and b as 2^d (a + b d) needs them: with m scale = r + rest, 2^d of the
  // fast form is 2^rest times 2^((z - m) scale), and its d is off by rest.
  __device__ __forceinline__ void set_scalars(RowScalars& r, float m, float scale, float a, float b, bool careful) const {
    r.m = m;
    r.r = __fmul_rn(m, scale);
    r.careful = careful || !(fabsf(r.r) <= LARGE_R) || fabsf(b) > largest_b<DT>(scale);
    const float rest = r.careful ? 0.f : __fmaf_rn(m, scale, -r.r), x = rest * float(LN2);
    const float f = 1.f - x * (1.f - 0.5f * x);
    r.a = f * (a - b * rest);
    r.b = f * b;
  }

  // One thread, from the merged records: the token's log-probability and what
  // hangs on it.
  __device__ __forceinline__ void token_scalars(Shared& sh, float m, float s, float u, uint32_t flags, const Scale& scale,
                                                const Inputs& in) {
    const float z = E::get(in.raw);
    const Pair log_s = log_pair(s), below = scaled_gap(z, m, scale), lp = pair_sum(below, negated(log_s));
    const float inv_s = __frcp_rn(s), gap = u * inv_s * float(LN2);  // log(s) - h
    // (Neither's rounding may take it past the end of its range.)
    const float h = fmaxf(value_of({log_s.hi, log_s.lo - gap}), 0.f), logprob = fminf(value_of(lp), 0.f);
    const bool mass = z > -INFINITY && (in.mask >> (in.token & 31) & 1);
    // A NaN logit makes s NaN, +inf the maximum.
    bool bad = (flags & BAD) || !(s < INFINITY) || m == INFINITY || in.token >= p.in.vocab;
    float slope = 0.f, on_entropy = 0.f, loss = 0.f, kl = 0.f;  // gradients of lp and of h
    if (OP == LOGPROB) {
      slope = in.first;
      on_entropy = in.second;
    } else {
      const float rise_of_lp = (lp.hi - in.first) + lp.lo;
      // In 64 bits: where the ratio meets a border.
      const double r = rise_of_lp < WIDE ? double(expf(rise_of_lp)) : exp(double(rise_of_lp));
      const double clipped = fmin(fmax(r, p.ratio_low), p.ratio_high);
      const bool through = r * in.second <= clipped * in.second;
      loss = float(through ? -r * in.second : -clipped * in.second);
      slope = through ? loss : 0.f;
      bad |= !isfinite(in.first) || !isfinite(in.second);
      if (p.ref_logprobs.p) {
        const float x = (in.ref - lp.hi) - lp.lo;
        if (x < WIDE) {
          const float rise = expm1f(x);
          kl = exp_beyond_first_order(x, rise);
          loss += float(p.kl_coef) * kl;
          slope -= float(p.kl_coef) * rise;
        } else {
          // (A KL that is only watched is held at the largest number and
          // leaves the loss alone.)
          const double rise = exp(double(x)) - 1., wide = rise - x;
          kl = float(fmin(wide, double(-LOWEST)));
          if (p.kl_coef != 0.) {
            loss += float(p.kl_coef * wide);
            slope -= float(p.kl_coef * rise);
          }
        }
        bad |= !isfinite(in.ref);
      }
      loss -= float(p.entropy_coef) * h;
      // (Of a token without mass there is no loss that could leave the range.)
      bad |= mass && !(isfinite(loss) && isfinite(slope));
      // Weights multiply as they are: an infinite or NaN one (an overflowed
      // loss scale) shows in the loss and the gradient.
      loss *= in.w;
      slope *= in.w;
      on_entropy = -float(p.entropy_coef) * in.w;
    }
    int status = ES_OK;
    if (bad) status = ES_INVALID_INPUT;
    else if (s == 0.f) status = ES_NO_VALID_TOKEN;
    else if (!mass) status = ES_DRAFT_ZERO_PROB;
    const bool ok = status == ES_OK;
    if (rank == 0)
      outputs(status, ok ? loss : 0.f, ok ? logprob : -INFINITY, ok ? kl : 0.f, ok ? h : 0.f);
    if (GRAD) {
      slope *= scale.hi;
      on_entropy *= scale.hi;
      RowScalars& r = sh.row;
      r.zero = !ok;
      // slope (1[j = t] - p_j) - on_entropy p_j (log p_j + h), with p_j = 2^d / s,
      // log p_j = d ln 2 - log s and h = log s - gap.
      set_scalars(r, m, scale.log2, -(slope - on_entropy * gap) * inv_s, -on_entropy * float(LN2) * inv_s,
                  flags & CAREFUL || scale.log2 < SMALL_SCALE);
      r.held = flags & HELD;
      // log p + h without the log(s) that both have.
      r.token_grad = -slope * expm1f(logprob) - on_entropy * expf(logprob) * ((below.hi - gap) + below.lo);
    }
  }

  // Distillation, every thread: the exponentials t and q of both models'
  // logits at the kept tokens, against the maxima over them, and the sums
  //   sum t, sum q, sum t (log t - log q).
  __device__ __forceinline__ void kept_sums(Shared& sh, const Kept& kept, const Scale& scale, float& value_top, float& x_top) const {
    value_top = x_top = -INFINITY;
    for (int k = lane_id(); k < p.k; k += 32)
      if (kept.id[k] >= 0) {
        value_top = fmaxf(value_top, kept.value[k]);
        x_top = fmaxf(x_top, kept.x[k]);
      }
    value_top = warp_top(value_top);
    x_top = warp_top(x_top);
    float t_sum = 0.f, q_sum = 0.f, cross = 0.f;
    for (int k = tid; k < p.k; k += THREADS) {
      float t = 0.f, q = 0.f;
      if (kept.id[k] >= 0) {
        const Pair lt = scaled_gap(kept.value[k], value_top, scale), lq = scaled_gap(kept.x[k], x_top, scale);
        t = kept.value[k] == -INFINITY ? 0.f : expf(lt.hi) * (1.f + lt.lo);
        q = kept.x[k] == -INFINITY ? 0.f : expf(lq.hi) * (1.f + lq.lo);
        if (t > 0.f) cross += kept.x[k] == -INFINITY ? INFINITY : t * ((lt.hi - lq.hi) + (lt.lo - lq.lo));
        t_sum += t;
        q_sum += q;
      }
      kept.t[k] = t;
      kept.q[k] = q;
    }
    t_sum = warp_sum(t_sum);
    q_sum = warp_sum(q_sum);
    cross = warp_sum(cross);
    if (lane_id() == 0) {
      sh.sums[warp_id()][0] = t_sum;
      sh.sums[warp_id()][1] = q_sum;
      sh.sums[warp_id()][2] = cross;
    }
  }

  // A model's total over its entries (their sum `entries`, relative to their
  // maximum) and the others (`others`, relative to theirs, which lies `over`
  // above the entries'): its logarithm relative to both, and the shares that
  // an entry's and another token's relative exponentials are multiplied with.
  struct Total {
    Pair to_entries, to_others;
    float entry_share, other_share, total;
  };
  static __device__ __forceinline__ Total total_of(float entries, float others, Pair over) {
    if (!(others > 0.f)) over = {-INFINITY, 0.f};
    if (!(entries > 0.f)) over = {INFINITY, 0.f};
    const bool above = over.hi > 0.f;  // the others are the reference
    const float f = isfinite(over.hi) ? expf(above ? -over.hi : over.hi) * (1.f + (above ? -over.lo : over.lo)) : 0.f;
    const float f_entries = entries > 0.f ? (above ? f : 1.f) : 0.f, f_others = others > 0.f ? (above ? 1.f : f) : 0.f;
    Total r;
    r.total = entries * f_entries + others * f_others;
    const float inv = __frcp_rn(r.total);
    const Pair log_total = log_pair(r.total);
    r.to_entries = above ? pair_sum(log_total, over) : log_total;
    r.to_others = above ? log_total : pair_sum(log_total, negated(over));
    r.entry_share = f_entries * inv;
    r.other_share = f_others * inv;
    return r;
  }

  // One thread, from the merged records of the tokens not kept (m, s). With T
  // and Q the logs of both totals, relative to the maxima over the entries,
  //   loss = sum_k t (lt - lq) / e^T + (Q - T) sum_k t / e^T + the bucket's term.
  __device__ __forceinline__ void distill_scalars(Shared& sh, float m, float s, uint32_t flags, const Scale& scale,
                                                  const Inputs& in, float value_top, float x_top) {
    const bool tail = p.rest.p != nullptr;
    float t_sum = 0.f, q_sum = 0.f, cross = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      t_sum += sh.sums[w][0];
      q_sum += sh.sums[w][1];
      cross += sh.sums[w][2];
    }
    const Total t = total_of(t_sum, tail && in.first > -INFINITY ? 1.f : 0.f,
                             pair_sum({in.first, 0.f}, negated(scaled_gap(value_top, 0.f, scale))));
    const Total q = total_of(q_sum, s, scaled_gap(m, x_top, scale));
    float loss = 0.f;
    // Of the tokens not kept: their gradient is q_j - t_rest q_j / q_rest, in
    // which their exponential against m is multiplied with this.
    float others = q.other_share;
    bool lost = cross == INFINITY;  // the student has no mass where the teacher has some
    if (t_sum > 0.f) loss = (cross + t_sum * value_of(pair_sum(q.to_entries, negated(t.to_entries)))) * t.entry_share;
    if (t.other_share > 0.f) {
      // log t_rest - log q_rest
      const float off = value_of(pair_sum(pair_sum(q.to_others, negated(t.to_others)), negated(log_pair(s))));
      loss += t.other_share * off;
      // Near t_rest = q_rest the difference would lose its digits. Elsewhere
      // t_rest / q_rest may leave the range where its product with q does not.
      others = fabsf(off) < 1.f ? -expm1f(off) * q.other_share : q.other_share - __fdiv_rn(t.other_share, s);
      lost |= !(s > 0.f);
    }
    const bool bad = (flags & BAD) || !(s < INFINITY) || !(t.total > 0.f && t.total < INFINITY) || (tail && !(in.first < INFINITY));
    int status = ES_OK;
    if (bad) status = ES_INVALID_INPUT;
    else if (!(q_sum > 0.f) && !(s > 0.f)) status = ES_NO_VALID_TOKEN;
    else if (lost) status = ES_DRAFT_ZERO_PROB;
    else if (!isfinite(loss)) status = ES_INVALID_INPUT;
    const bool ok = status == ES_OK;
    // (A KL's rounding may not take it below 0 either.)
    if (rank == 0) outputs(status, ok ? in.w * fmaxf(loss, 0.f) : 0.f, 0.f, 0.f, 0.f);
    if (GRAD) {
      RowScalars& r = sh.row;
      r.zero = !ok;
      r.w = in.w * scale.hi;
      r.inv_q = q.entry_share;
      r.inv_t = t.entry_share;
      set_scalars(r, m, scale.log2, s > 0.f ? r.w * others : 0.f, 0.f, flags & CAREFUL || scale.log2 < SMALL_SCALE);
    }
  }

  // The gradient of chunk c from its logits. FORM 0: 2^d a; 1: 2^d (a + b d);
  // 2: the careful form of the latter. `words`: the mask, where the slice's
  // masked tokens are not yet what the form needs.
  template <int FORM>
  __device__ __forceinline__ uint4 grad_chunk(uint4 q, int c, const uint32_t* words, const RowScalars& r, float scale) const {
    float2 v[N / 2];
    if (FORM == 2 && words) q = mask_chunk<DT>(q, mask_bits(words, c * N), lowest_word<DT>());
    if (FORM == 1 && r.held) q = hold_chunk<DT>(q);
    unpack<DT>(q, v);
    if (FORM == 1 && DT == ES_F16) {
      if (words || r.held) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = make_float2(fmaxf(v[i].x, MASKED), fmaxf(v[i].y, MASKED));
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      float2 d;
      if (FORM == 2) d = make_float2(exponent(v[i].x, r.m, scale), exponent(v[i].y, r.m, scale));
      else d = fma2(v[i], both(scale), both(-r.r));
      const float2 e = make_float2(ex2(d.x), ex2(d.y));
      v[i] = mul2(e, FORM == 0 ? both(r.a) : fma2(both(r.b), d, both(r.a)));
    }
    return pack<DT>(v);
  }

  // The gradient of this rank's slice from its shared copy. `token`: the row's
  // token in it, or negative. `next`: the slice's place in the next row, or null.
  template <int FORM>
  __device__ __forceinline__ void write_grad(const Slice<DT>& slice, const uint32_t* words, const RowScalars& scalars, float scale,
                                             int token, const T* next) const {
    const RowScalars r = scalars;
    if (grad_vector() && (next == nullptr || Slice<DT>::width(p.in, next) == 16)) write_aligned<FORM>(slice, words, r, scale, token, next);
    else write_anywhere<FORM>(slice, words, r, scale, token, next);
  }
  template <int FORM>
  __device__ __forceinline__ void write_aligned(const Slice<DT>& slice, const uint32_t* words, const RowScalars& r, float scale,
                                                int token, const T* next) const {
    uint4* out = reinterpret_cast<uint4*>(grad_at(begin));
    const uint4* from = reinterpret_cast<const uint4*>(next);
    const int whole = n / N;
    int c = tid;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      const int end = part ? whole : slice.half;
#pragma unroll 1
      for (; c + 3 * THREADS < end; c += STEP) {
        uint4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = slice.chunk(c + i * THREADS);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[c + i * THREADS] = grad_chunk<FORM>(q[i], c + i * THREADS, words, r, scale);
        if (next) {
#pragma unroll
          for (int i = 0; i < 4; ++i) copy_async(&slice.chunk(c + i * THREADS), from + c + i * THREADS);
        }
      }
      if (part) {
        for (; c < whole; c += THREADS) {
          out[c] = grad_chunk<FORM>(slice.chunk(c), c, words, r, scale);
          if (next) copy_async(&slice.chunk(c), from + c);
        }
      }
      copies_end_group();
    }
    if (c == whole && whole < slice.chunks) store_elements(grad_chunk<FORM>(slice.chunk(c), c, words, r, scale), c, 0, N);
    if (next) slice.load_ragged(next, 16);
    // The thread that wrote the token's chunk.
    if (OP != DISTILL && token >= 0 && token / N % THREADS == tid) *grad_at(begin + token) = E::put(r.token_grad);
  }
  // Elements [from, to) of chunk c's gradient.
  __device__ __forceinline__ void store_elements(const uint4& q, int c, int from, int to) const {
    const T* v = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i >= from && i < to && c * N + i < n) *grad_at(begin + c * N + i) = v[i];
  }
  // Gradient rows or next rows that do not start on 16 bytes, or have a stride.
  // A warp's 32 chunks go back to their places in the slice and from there out,
  // neighbouring words or elements from neighbouring lanes.
  template <int FORM>
  __device__ __forceinline__ void write_anywhere(const Slice<DT>& slice, const uint32_t* words, const RowScalars& r, float scale,
                                                 int token, const T* next) const {
    const int bytes = next ? Slice<DT>::width(p.in, next) : 0, whole = n / N, lane = lane_id();
    const bool vector = grad_vector();
    // Elements to a store: the most that the row's start allows.
    const int most = p.g_s1 == 1 && reinterpret_cast<uintptr_t>(grad_at(begin)) % 4 == 0 ? 4 / int(sizeof(T)) : 1;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
      const int end = part ? slice.chunks : slice.half;
#pragma unroll 1
      for (int c = (part ? slice.half : 0) + tid; c - lane < end; c += THREADS) {
        if (c < slice.chunks) {
          uint4 g = grad_chunk<FORM>(slice.chunk(c), c, words, r, scale);
          if (OP != DISTILL && token >= 0 && token / N == c) {
            T* v = reinterpret_cast<T*>(&g);
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (token % N == j) v[j] = E::put(r.token_grad);
          }
          if (vector && c < whole) *reinterpret_cast<uint4*>(grad_at(begin + c * N)) = g;
          else slice.chunk(c) = g;
        }
        __syncwarp();
        if (!vector || (c - lane + 32) > whole) {
          const int from = (vector ? max(c - lane, whole) : c - lane) * N, to = min((c - lane + 32) * N, n);
          if (most == 2) {
#pragma unroll 4
            for (int i = from + 2 * lane; i < to; i += 64) {
              if (i + 1 < to) *reinterpret_cast<uint32_t*>(grad_at(begin + i)) = *reinterpret_cast<const uint32_t*>(&slice[i]);
              else *grad_at(begin + i) = slice[i];
            }
          } else {
#pragma unroll 4
            for (int i = from + lane; i < to; i += 32) *grad_at(begin + i) = slice[i];
          }
          __syncwarp();
        }
        if (bytes && c < whole) slice.copy(c, next, bytes);
      }
      copies_end_group();
    }
    if (bytes) slice.load_ragged(next, bytes);
  }
  __device__ __forceinline__ void write_form(const Slice<DT>& slice, const uint32_t* words, const RowScalars& r, float scale,
                                             int token, const T* next) const {
    if (r.careful) write_grad<2>(slice, words, r, scale, token, next);
    else if (ENTROPY && r.b != 0.f) write_grad<1>(slice, words, r, scale, token, next);
    else write_grad<0>(slice, words, r, scale, token, next);
  }

  // The slice's mask words of row `at` into shared memory; there after
  // copies_done and a block barrier.
  __device__ __forceinline__ void load_mask(uint32_t* words, int64_t at) const {
    const int32_t* from = p.in.mask.p + at * p.in.mask.s0 + (begin >> 5) * p.in.mask.s1;
    for (int i = tid; i < (n + 31) / 32; i += THREADS)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(words + i)), "l"(from + i * p.in.mask.s1) : "memory");
  }

  // Distillation: a row's entries into shared memory; false if there are none.
  __device__ __forceinline__ bool load_entries(const Kept& kept, bool& bad) const {
    bool any = false;
    for (int k = tid; k < p.k; k += THREADS) {
      const int64_t id = p.ids.p[row * p.ids.s0 + k * p.ids.s1];
      const float value = p.values.p[row * p.values.s0 + k * p.values.s1];
      any |= id >= 0;
      bad |= id >= p.in.vocab || (id >= 0 && !(value < INFINITY));
      const bool usable = id >= 0 && id < p.in.vocab;
      float x = -INFINITY;
      if (usable) {
        x = E::get(logit(id));
        bad |= !(x < INFINITY);
        if (!allowed(id)) x = -INFINITY;
      }
      kept.id[k] = usable ? int(id) : -1;
      kept.value[k] = value;
      kept.x[k] = x;
    }
    return __syncthreads_or(any);
  }

  __device__ __forceinline__ void run(uint8_t* smem) {
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    uint8_t* buffer = smem + SHARED_BYTES;
    uint32_t* const masks = reinterpret_cast<uint32_t*>(buffer + slice_bytes<DT>(p.in.slice));
    const bool masked = p.in.mask.p != nullptr;
    const Kept kept(buffer + slice_bytes<DT>(p.in.slice) + (masked ? 2 * mask_bytes(p.in.slice) : 0), p.k);
    if (tid == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh.bar[i], 1);
        mbar_arrive_expect_tx(&sh.bar[i], uint32_t(ranks * sizeof(Record)));
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (OP == DISTILL)
      for (int i = tid; i < p.in.slice / 32; i += THREADS) kept.seen[i] = 0;
    __syncthreads();
    cluster_started();
    bool peers = false;  // whether every rank is known to have started

    Slice<DT> slice;
    slice.init(buffer, n);
    bool loaded = false;  // the row's copies are under way
    int turn = 0;         // rows taken so far, those without a token aside
    int64_t next_token = OP != DISTILL ? p.tokens[row] : 0;
    for (; row < p.in.rows; row += stride) {
      // The row's token, or the teacher's entries; rows without are not read.
      Inputs in{};
      bool bad = false;
      in.token = next_token;
      if (OP != DISTILL && row + stride < p.in.rows) next_token = p.tokens[row + stride];
      if (OP == DISTILL) in.token = load_entries(kept, bad) ? 0 : -1;
      if (in.token < 0) {
        if (loaded) {
          copies_done<0>();  // (distillation learns too late that the row is not needed)
          loaded = false;
        }
        if (GRAD) zero_grad();
        if (rank == 0 && tid == 0) {
          // (A teacher's row that failed has no entries either.)
          const int status = OP == DISTILL && p.teacher_status.p ? p.teacher_status[row] : ES_OK;
          outputs(status, 0.f, 0.f, 0.f, 0.f);
        }
        continue;
      }
      uint32_t* const words = masked ? masks + (turn & 1) * (p.in.slice / 32) : nullptr;
      if (!loaded) {
        if (masked) load_mask(words, row);
        slice.load(p.in, row, begin);
      }
      const Scale scale = row_scale(p.in, row);
      bad |= scale.bad;
      if (tid == 0) {
        in.mask = 0xffffffffu;
        if (OP != DISTILL && in.token < p.in.vocab) {
          in.raw = logit(in.token);
          if (p.in.mask.p) in.mask = uint32_t(p.in.mask.p[row * p.in.mask.s0 + (in.token >> 5) * p.in.mask.s1]);
        }
        if (OP == LOGPROB && GRAD) {
          if (p.grad_logprobs.p) in.first = p.grad_logprobs[row];
          if (p.grad_entropy.p) in.second = p.grad_entropy[row];
        }
        if (OP == POLICY) {
          in.first = p.old_logprobs[row];
          in.second = p.advantages[row];
          if (p.ref_logprobs.p) in.ref = p.ref_logprobs[row];
        }
        if (OP == DISTILL && p.rest.p) in.first = p.rest[row];
        if (OP != LOGPROB) in.w = p.weights.p ? p.weights[row] : 1.f;
      }
      float value_top = 0.f, x_top = 0.f;
      if (OP == DISTILL) kept_sums(sh, kept, scale, value_top, x_top);
      slice.arrive();
      if (sizeof(T) == 2 && Slice<DT>::width(p.in, Slice<DT>::source(p.in, row, begin)) == 2) {
        slice.arrive_rest();
        slice.realign();
      }
      if (masked && OP != DISTILL) __syncthreads();  // the mask words come from all threads' first copies
      if (OP == DISTILL) {
        slice.arrive_rest();
        __syncthreads();
        // The kept tokens leave the slice, so that what is summed is the others.
        for (int k = tid; k < p.k; k += THREADS) {
          const int local = kept.id[k] - begin;
          if (kept.id[k] >= 0 && local >= 0 && local < n) {
            bad |= (atomicOr(&kept.seen[local >> 5], 1u << (local & 31)) >> (local & 31)) & 1;
            slice[local] = E::put(-INFINITY);
          }
        }
        __syncthreads();
      }

      const int64_t local = in.token - begin;
      const int at = OP != DISTILL && local >= 0 && local < n ? int(local) : -1;
      Record rec = masked ? sum_slice<DT, ENTROPY, MASKED_ROW>(slice, words, at, scale.log2)
                          : sum_slice<DT, ENTROPY, OPEN_ROW>(slice, nullptr, at, scale.log2);
      // (The token's logit is looked at before this rank says that it has done
      // with the row's memory, which may be the gradient's.)
      if (OP != DISTILL && tid == 0) bad |= isnan(E::get(in.raw));
      if (bad) rec.flags |= BAD;
      const T* next = row + stride < p.in.rows && next_token >= 0 ? Slice<DT>::source(p.in, row + stride, begin) : nullptr;
      if (next && Slice<DT>::width(p.in, next) == 0) next = nullptr;
      rec = lanes_record<ENTROPY, 32>(rec, scale.log2);
      if (lane_id() == 0) sh.warps[turn & 1][warp_id()] = rec;
      if (!peers) cluster_wait();
      peers = true;
      __syncthreads();
      rec = join_records<ENTROPY, WARPS>(sh.warps[turn & 1], WARPS, scale.log2);
      if (tid < ranks) send_record(&sh.inbox[turn & 1][rank], &sh.bar[turn & 1], tid, rec);
      loaded = next != nullptr;
      if (masked && loaded) load_mask(masks + (turn + 1 & 1) * (p.in.slice / 32), row + stride);  // in the first group
      if (!GRAD && loaded) slice.load(p.in, row + stride, begin);
      const bool came = wait_bar(&sh.bar[turn & 1], turn >> 1 & 1);
      if (tid == 0) mbar_arrive_expect_tx(&sh.bar[turn & 1], uint32_t(ranks * sizeof(Record)));  // for the row after the next
      rec = join_records<ENTROPY, MAX_RANKS>(sh.inbox[turn & 1], ranks, scale.log2);
      ++turn;
      if (!came) rec.flags |= BAD;
      if (tid == 0 && (GRAD || rank == 0)) {
        if (OP == DISTILL) distill_scalars(sh, rec.m, rec.s, rec.flags, scale, in, value_top, x_top);
        else token_scalars(sh, rec.m, rec.s, rec.u, rec.flags, scale, in);
      }
      if (GRAD) {
        __syncthreads();
        const RowScalars& r = sh.row;
        if (r.zero) {
          zero_grad();
          if (loaded) slice.load(p.in, row + stride, begin);
        } else {
          write_form(slice, words, r, scale.log2, at, next);
          if (OP == DISTILL) __syncthreads();  // after the slice's zeros at these places
          if (OP == DISTILL)
            for (int k = tid; k < p.k; k += THREADS) {
              const int local_id = kept.id[k] - begin;
              if (kept.id[k] >= 0 && local_id >= 0 && local_id < n)
                *grad_at(kept.id[k]) = E::put(r.w * (kept.q[k] * r.inv_q - kept.t[k] * r.inv_t));
            }
        }
      }
      if (OP == DISTILL)
        for (int k = tid; k < p.k; k += THREADS) {
          const int local = kept.id[k] - begin;
          if (kept.id[k] >= 0 && local >= 0 && local < n) kept.seen[local >> 5] = 0;
        }
    }
    copies_done<0>();
    if (!peers) cluster_wait();
  }
};

template <int DT, int OP, bool GRAD>
__global__ void __launch_bounds__(THREADS, BLOCKS) loss_rows(const __grid_constant__ LossParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = p.in.ranks, rank = int(blockIdx.x % unsigned(ranks));
  const int begin = rank * p.in.slice, n = min(p.in.slice, p.in.vocab - begin);
  LossRow<DT, OP, GRAD> work{p, int64_t(blockIdx.x / unsigned(ranks)), int64_t(gridDim.x / unsigned(ranks)), rank, ranks, begin, n,
                             int(threadIdx.x)};
  work.run(smem);
}

// What a kernel needs to know of each device: whether its attributes are set
// (once, to the most that any call needs), and how many clusters of one shape
// run at a time (a few shapes asked for: the shape in the upper half).
struct Configured {
  std::atomic<uint64_t> devices{0};
  std::atomic<uint64_t> clusters[64][8] = {};
};

// Launches `rows` clusters of `ranks` blocks, or, where they take the rows at a
// stride, no more than run at a time.
template <class P>
cudaError_t launch_clusters(void (*kernel)(P), const P& p, bool strided, int64_t rows, int ranks, int threads, size_t smem,
                            cudaStream_t stream, Configured& configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev < 64;
  const uint64_t bit = 1ull << (dev & 63);
  if (!known || !(configured.devices.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    if (known) configured.devices.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(unsigned(threads), 1, 1);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  if (strided) {
    const uint64_t shape = uint64_t(smem) << 8 | uint64_t(ranks);  // below 2^32
    std::atomic<uint64_t>& slot = configured.clusters[dev & 63][(smem / 512 + ranks) & 7];
    const uint64_t seen = slot.load(std::memory_order_relaxed);
    int most = int(seen & 0xffffffffu);
    if (!known || seen >> 32 != shape) {
      config.gridDim = dim3(unsigned(ranks), 1, 1);
      e = cudaOccupancyMaxActiveClusters(&most, kernel, &config);
      if (e != cudaSuccess) return e;
      most = std::max(most, 1);
      if (known) slot.store(shape << 32 | uint64_t(most), std::memory_order_relaxed);
    }
    rows = std::min<int64_t>(rows, most);
  }
  config.gridDim = dim3(unsigned(rows * ranks), 1, 1);
  return cudaLaunchKernelEx(&config, kernel, p);
}

template <int DT, int OP, bool GRAD> cudaError_t launch_one(const LossParams& p, cudaStream_t stream) {
  static Configured configured;
  return launch_clusters(loss_rows<DT, OP, GRAD>, p, true, p.in.rows, p.in.ranks, THREADS, loss_smem<DT>(p.in.slice, p.in.mask.p != nullptr, p.k), stream, configured);
}
template <int DT> cudaError_t launch_loss(const LossParams& p, int op, cudaStream_t stream) {
  const bool grad = p.grad != nullptr;
  switch (op) {
    case LOGPROB: return grad ? launch_one<DT, LOGPROB, true>(p, stream) : launch_one<DT, LOGPROB, false>(p, stream);
    case POLICY: return grad ? launch_one<DT, POLICY, true>(p, stream) : launch_one<DT, POLICY, false>(p, stream);
    default: return grad ? launch_one<DT, DISTILL, true>(p, stream) : launch_one<DT, DISTILL, false>(p, stream);
  }
}

}  // namespace score
}  // namespace es
