// The k largest logits of each row, sorted, and the log-sum of the rest
// (top_rows): one pass over the row, which never lies in shared memory, so
// that as many blocks as registers allow keep the memory busy.
//
// A row is split over a cluster; a thread goes through every THREADS-th chunk
// of its rank's slice, 32 tokens a step:
//   1. each thread keeps the maximum and the sum of each of its steps;
//   2. each rank finds the ceil(k / ranks)-th largest of its threads' maxima
//      (to 12 bits of its key from the first in which they differ). At least
//      that many of its tokens reach it, so the smallest of the ranks' values
//      is a bound that at least k tokens of the row reach, and few more (a
//      thread rarely holds two of the largest);
//   3. the few steps whose maximum reaches the bound give up their sums.
//      Their tokens are read again, from L2, one to a lane: those at or above
//      the bound are listed, the others summed. So the rest is summed without
//      the largest, and one far below them loses no digits to a subtraction;
//   4. rank 0 has every rank's list, places each entry by the number of larger
//      ones, and adds the entries past the k-th to the rest.
// Entries are 64-bit words, the logit's order key above the complement of its
// id, so that all are distinct and equal logits rank by the lowest id. Where a
// rank lists more than its places on rank 0, rank 0 alone finds the exact
// threshold by a digit-by-digit count over the whole row, 23 passes that load
// single tokens. Two kinds of rows come to that: equal values in numbers, and
// rows where one rank's slice has fewer tokens than it is asked for, since the
// smallest of the ranks' bounds then lets every token through. Masks or -inf
// that leave a part of the vocabulary empty make the second kind: 2,048 rows of
// 151,936 bf16 take 58 ms where a mask allows ids below 3,000, 64 below 100,000,
// 62 with -inf above 100,000 and 68 where all logits are equal, and 8 rows take
// 6 to 7 ms, against 0.18 ms and 16 us for open rows.
//
// Bounds: the latency of the steps after the streaming, each of which waits
// for the other ranks. Measured on a B200: the 64 largest of 2,048 rows of
// 151,936 bf16 take 177 us (3.5 TB/s), of which the first step alone is 129.
// More blocks to an SM hide more of it (six: 204, eight: 177). A row that lay
// in shared memory, for the second look, took 483.
#pragma once
#include "es_score.cuh"

namespace es {
namespace score {

struct TopParams {
  Rows in;
  int32_t k;
  Grid2<float> values;
  Grid2<int64_t> ids;
  Column<float> rest;
  Column<int32_t> status;
};

constexpr int TOP_THREADS = 128, TOP_WARPS = TOP_THREADS / 32;
constexpr int TOP_BLOCKS = 8;  // to an SM (64 of 2,048 rows: 177 us; ten 185, twelve 210: fewer registers for loads in flight)
constexpr uint32_t KEY_NONE = 0x007fffffu;  // the key of -inf: not a token of the row
constexpr int COLLECTED = 1024;             // entries rank 0 takes, an equal share from each rank
constexpr int HOT = 128;                    // steps a warp looks at again
static_assert(COLLECTED >= 2 * MAX_TOP, "a single rank's list holds k entries and more");

struct TopShared {
  Record inbox[MAX_RANKS * TOP_WARPS], bounds[MAX_RANKS];
  uint64_t bar[2];
  uint32_t keys[TOP_THREADS];
  uint16_t hot[TOP_WARPS][HOT];  // steps to look at again
  uint32_t listed, entries;
  uint32_t digits[TOP_WARPS][8];
  alignas(16) uint64_t places[COLLECTED];  // rank 0: each rank's list at its share, then all side by side
  // Maximum and sum of each thread's steps, as many as a slice has; then, on
  // rank 0, when all its warps have done with those, values past the k-th by
  // place. (Memory of its own for each list leaves room for six blocks to an
  // SM: 204 us for 64 of 2,048 rows of 151,936 bf16, against 177.)
  union {
    float2 steps[COLLECTED / 2];
    float beyond[COLLECTED];
  };
};

__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) { return (uint64_t(key) << 32) | (0xffffffffu - uint32_t(id)); }

// Rank 0's barrier: what this thread's block wrote to rank 0 before its last
// block barrier is there when the arrival is seen.
__device__ __forceinline__ void arrive_at(uint64_t* bar, int rank) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(bar)), "r"(rank));
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar) {
  uint32_t spins = 0, done = 0;
  while (true) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar))
        : "memory");
    if (done) return true;
    if (++spins >= WAIT_LIMIT) return false;
  }
}

template <int DT> struct TopRow {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int N = E::N;
  static constexpr int CHUNKS = 32 / N;  // of a step

  const TopParams& p;
  int64_t row;
  int rank, ranks, begin, n, tid;

  __device__ __forceinline__ const T* source() const {
    return static_cast<const T*>(p.in.logits) + row * p.in.l_s0 + int64_t(begin) * p.in.l_s1;
  }
  // Chunk c of the slice. ALIGNED: the slice starts on 16 bytes (c a whole chunk).
  template <bool ALIGNED> __device__ __forceinline__ uint4 chunk(const T* src, int c) const {
    if (ALIGNED) return __ldg(reinterpret_cast<const uint4*>(src) + c);
    return fetch_chunk<DT>(src, p.in.l_s1, c, n);
  }
  // Sets masked tokens to -inf; looks at them first.
  __device__ __forceinline__ void apply_mask(const int32_t* mask, int c, uint4& q, bool& bad) const {
    bad |= !(chunk_max_nan<DT>(q) < INFINITY);
    q = mask_chunk<DT>(q, uint32_t(mask[(c * N >> 5) * p.in.mask.s1]) >> (c * N & 31), lowest_word<DT>());
  }

  // The maximum and the sum of 32 tokens (-inf where there are none).
  __device__ __forceinline__ float2 step_sum(const uint4* q, float scale) const {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < CHUNKS; i += 2) top = fmaxf(top, chunk_max<DT>(q[i], q[i + 1]));
    const float m = fmaxf(top, LOWEST), r = __fmul_rn(m, scale);
    float2 v[16], s = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) unpack<DT>(q[i], v + i * N / 2);
    if (fabsf(r) <= LARGE_R && scale >= SMALL_SCALE) {
      // (r's rounding, at most 2^-24 of it, goes into the sum as a factor.)
      const float rest = __fmaf_rn(m, scale, -r);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 d = fma2(v[i], both(scale), both(-r));
        s = add2(s, make_float2(ex2(d.x), ex2(d.y)));
      }
      return {m, __fmul_rn(__fadd_rn(s.x, s.y), ex2(-rest))};
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s = add2(s, make_float2(ex2(exponent(v[i].x, m, scale)), ex2(exponent(v[i].y, m, scale))));
    return {m, __fadd_rn(s.x, s.y)};
  }
  // Every thread's steps; returns their maximum.
  template <bool ALIGNED>
  __device__ __forceinline__ float sums(TopShared& sh, const T* src, const int32_t* mask, int steps, float scale, bool& bad) const {
    const int chunks = (n + N - 1) / N, whole = ALIGNED ? n / N : chunks;
    const uint4 none = make_uint4(lowest_word<DT>(), lowest_word<DT>(), lowest_word<DT>(), lowest_word<DT>());
    float high = -INFINITY;
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      uint4 q[CHUNKS];
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        const int c = (step * CHUNKS + i) * TOP_THREADS + tid;
        q[i] = none;
        if (c < whole) q[i] = chunk<ALIGNED>(src, c);
        else if (c < chunks) q[i] = chunk<false>(src, c);
      }
      if (mask) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          const int c = (step * CHUNKS + i) * TOP_THREADS + tid;
          if (c < chunks) apply_mask(mask, c, q[i], bad);
        }
      }
      const float2 got = step_sum(q, scale);
      sh.steps[step * TOP_THREADS + tid] = got;
      bad |= !(got.y < INFINITY) || got.x == INFINITY;
      high = fmaxf(high, got.y > 0.f ? got.x : -INFINITY);
    }
    return high;
  }

  // A bound that at least `need` of the threads' keys reach: their common
  // leading bits, then 12 more, one a step. Every warp finds it for itself (in
  // a loop of a fixed length: see lanes_record). 0 if fewer threads than that
  // have any token.
  __device__ __forceinline__ uint32_t thread_bound(const uint32_t* keys, int need) const {
    uint32_t key[TOP_WARPS], low = 0xffffffffu, high = 0;
#pragma unroll
    for (int i = 0; i < TOP_WARPS; ++i) {
      key[i] = keys[i * 32 + lane_id()];
      low = min(low, key[i]);
      high = max(high, key[i]);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    const int differ = 31 - __clz(int((low ^ high) | 1u));
    uint32_t found = differ == 31 ? 0u : high & ~((2u << differ) - 1u);
    int shift = differ - 1;  // two bits a step: three candidates' counts side by side
#pragma unroll
    for (int step = 0; step < 6; ++step, shift -= 2) {
      const int at = max(shift, 0);
      uint32_t above = 0;
#pragma unroll
      for (int i = 0; i < TOP_WARPS; ++i)
        above += (key[i] >= (found | 1u << at)) + ((key[i] >= (found | 2u << at)) << 10) + ((key[i] >= (found | 3u << at)) << 20);
      above = __reduce_add_sync(0xffffffffu, above);
      const uint32_t digit = (int(above & 1023u) >= need) + (int(above >> 10 & 1023u) >= need) + (int(above >> 20) >= need);
      if (shift >= 0) found |= digit << at;
    }
    return need <= TOP_THREADS ? found : 0u;
  }

  __device__ __forceinline__ void write(int64_t at, float value, int64_t id) const {
    p.values.p[row * p.values.s0 + at * p.values.s1] = value;
    p.ids.p[row * p.ids.s0 + at * p.ids.s1] = id;
  }
  // A token of the whole row, as the row's entries see it.
  __device__ __forceinline__ uint64_t entry_at(int j) const {
    const T* src = static_cast<const T*>(p.in.logits) + row * p.in.l_s0 + int64_t(j) * p.in.l_s1;
    const bool allowed = p.in.mask.p == nullptr ||
                         (uint32_t(p.in.mask.p[row * p.in.mask.s0 + (j >> 5) * p.in.mask.s1]) >> (j & 31) & 1);
    const float v = E::get(*src);
    return allowed && v > -INFINITY ? entry_of(order_key(v), j) : 0;
  }

  // Rank 0 alone: the row's k-th largest entry (1 when fewer tokens are
  // valid), three bits of the entry a step.
  __device__ __noinline__ uint64_t exact_threshold(TopShared& sh) const {
    uint64_t found = 0;
    uint32_t need = p.k;
    for (int shift = 63; shift >= 0; shift -= 3) {  // bit 63 alone, then 21 digits of three bits
      uint32_t mine[8] = {};
      for (int j = tid; j < p.in.vocab; j += TOP_THREADS) {
        const uint64_t entry = entry_at(j);
        if (entry != 0 && (shift == 63 || ((entry ^ found) >> (shift + 3)) == 0)) {
#pragma unroll
          for (int d = 0; d < 8; ++d) mine[d] += (int(entry >> shift) & 7) == d;
        }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const uint32_t sum = __reduce_add_sync(0xffffffffu, mine[d]);
        if (lane_id() == 0) sh.digits[warp_id()][d] = sum;
      }
      __syncthreads();
      uint32_t above = 0, digit = 8, at = 0;
      while (digit > 0 && above + at < need) {  // from the largest digit down
        above += at;
        --digit;
        at = 0;
        for (int w = 0; w < TOP_WARPS; ++w) at += sh.digits[w][digit];
      }
      __syncthreads();
      if (above + at < need) return 1;
      need -= above;
      found |= uint64_t(digit) << shift;
    }
    return found;
  }
  // Rank 0 alone: the row's entries at or above the exact threshold, and the
  // sum of the others. Returns how many entries there are.
  __device__ __noinline__ int exact_entries(TopShared& sh, float scale, Record& rest) const {
    const uint64_t least = exact_threshold(sh);
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    Record rec = {LOWEST, 0.f, 0.f, 0u};
    for (int j = tid; j < p.in.vocab; j += TOP_THREADS) {
      const uint64_t entry = entry_at(j);
      if (entry >= least) {
        sh.places[atomicAdd(&sh.listed, 1u)] = entry;
      } else if (entry != 0) {
        const float v = key_value(uint32_t(entry >> 32)), m = fmaxf(rec.m, v);
        rec.s = __fadd_rn(__fmul_rn(ex2(exponent(rec.m, m, scale)), rec.s), ex2(exponent(v, m, scale)));
        rec.m = m;
      }
    }
    __syncthreads();
    rest = rec;
    return int(sh.listed);
  }

  __device__ __forceinline__ void run(TopShared& sh) {
    if (tid == 0) {
      mbar_init(&sh.bar[0], 1);
      mbar_init(&sh.bar[1], ranks * TOP_WARPS);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      mbar_arrive_expect_tx(&sh.bar[0], uint32_t(ranks * sizeof(Record)));
      sh.listed = sh.entries = 0;
    }
    if (rank == 0)
      for (int i = tid; i < COLLECTED; i += TOP_THREADS) sh.places[i] = 0;
    if (rank == 0) cluster_arrive();  // (the cleared places too)
    else cluster_started();
    const Scale temperature = row_scale(p.in, row);
    const float scale = temperature.log2;
    const T* src = source();
    const int32_t* mask = p.in.mask.p ? p.in.mask.p + row * p.in.mask.s0 + (begin >> 5) * p.in.mask.s1 : nullptr;
    bool bad = temperature.bad;
    const bool aligned = p.in.l_s1 == 1 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const int steps = (n + 32 * TOP_THREADS - 1) / (32 * TOP_THREADS);
    const float high = aligned ? sums<true>(sh, src, mask, steps, scale, bad) : sums<false>(sh, src, mask, steps, scale, bad);
    sh.keys[tid] = high > -INFINITY ? order_key(high) : 0u;
    cluster_wait();  // every rank has started
    __syncthreads();

    const uint32_t found = max(thread_bound(sh.keys, (p.k + ranks - 1) / ranks), KEY_NONE + 1);
    if (tid < ranks) send_record(&sh.bounds[rank], &sh.bar[0], tid, Record{0.f, 0.f, 0.f, found});
    if (!wait_bar(&sh.bar[0], 0)) bad = true;
    uint32_t bound = sh.bounds[min(lane_id(), ranks - 1)].flags;
    bound = __reduce_min_sync(0xffffffffu, bound);

    // The steps below the bound add up; the others' tokens are looked at again,
    // a lane each.
    const int share = COLLECTED / ranks;
    uint64_t* places = cg::this_cluster().map_shared_rank(sh.places, 0) + rank * share;
    Record rec = {LOWEST, 0.f, 0.f, 0u};
    bool full = false;
    int count = 0;
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      const float2 got = sh.steps[step * TOP_THREADS + tid];
      const bool some = got.y > 0.f, reaches = some && order_key(got.x) >= bound;
      const uint32_t hot = __ballot_sync(0xffffffffu, reaches);
      const int at = count + __popc(hot & ((1u << lane_id()) - 1));
      if (reaches && at < HOT) sh.hot[warp_id()][at] = uint16_t(step * 32 + lane_id());
      count += __popc(hot);
      const float m = reaches || !some ? rec.m : fmaxf(rec.m, got.x);
      rec.s = __fmul_rn(ex2(exponent(rec.m, m, scale)), rec.s);
      if (some && !reaches) rec.s = __fadd_rn(rec.s, __fmul_rn(ex2(exponent(got.x, m, scale)), got.y));
      rec.m = m;
    }
    if (count > HOT) full = true;  // (they would hardly fit their places either)
    __syncwarp();
#pragma unroll 1
    for (int first = 0; first < min(count, HOT); first += 4) {
      int token[4];
      float v[4], m = rec.m;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t hot = first + i < count ? sh.hot[warp_id()][first + i] : 0u;
        token[i] = (((hot >> 5) * CHUNKS + lane_id() / N) * TOP_THREADS + warp_id() * 32 + (hot & 31)) * N + lane_id() % N;
        v[i] = -INFINITY;
        if (first + i < count && token[i] < n) v[i] = E::get(src[token[i] * p.in.l_s1]);
      }
      if (mask) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v[i] > -INFINITY && !(uint32_t(mask[(token[i] >> 5) * p.in.mask.s1]) >> (token[i] & 31) & 1)) v[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (order_key(v[i]) >= bound) {
          const uint32_t place = atomicAdd(&sh.listed, 1u);
          if (int(place) < share) places[place] = entry_of(order_key(v[i]), begin + token[i]);
          else full = true;
          v[i] = -INFINITY;
        }
        m = fmaxf(m, v[i]);
      }
      rec.s = __fmul_rn(ex2(exponent(rec.m, m, scale)), rec.s);
#pragma unroll
      for (int i = 0; i < 4; ++i) rec.s = __fadd_rn(rec.s, ex2(exponent(v[i], m, scale)));
      rec.m = m;
    }
    rec.flags = (bad ? BAD : 0u) | (full ? FULL : 0u);
    rec = lanes_record<false, 32>(rec, scale);
    if (lane_id() == 0) cg::this_cluster().map_shared_rank(sh.inbox, 0)[rank * TOP_WARPS + warp_id()] = rec;
    __syncwarp();
    if (lane_id() == 0) arrive_at(&sh.bar[1], 0);
    if (rank != 0) return;

    const bool came = wait_cluster(&sh.bar[1]);
    rec = {LOWEST, 0.f, 0.f, 0u};
#pragma unroll
    for (int i = 0; i < MAX_RANKS * TOP_WARPS / 32; ++i) {
      const int at = i * 32 + lane_id();
      if (i * 32 >= ranks * TOP_WARPS) break;
      Record more = sh.inbox[min(at, ranks * TOP_WARPS - 1)];
      if (at >= ranks * TOP_WARPS) more.s = 0.f, more.m = LOWEST;
      const float m = fmaxf(rec.m, more.m);
      rec.s = __fadd_rn(__fmul_rn(ex2(exponent(rec.m, m, scale)), rec.s), __fmul_rn(ex2(exponent(more.m, m, scale)), more.s));
      rec.m = m;
      rec.flags |= more.flags;
    }
    rec = lanes_record<false, 32>(rec, scale);
    bad = (rec.flags & BAD) || !came;
    // The ranks' lists side by side.
    uint64_t mine[COLLECTED / TOP_THREADS];
    count = 0;
#pragma unroll
    for (int i = 0; i < COLLECTED / TOP_THREADS; ++i) {
      mine[i] = sh.places[i * TOP_THREADS + tid];
      count += mine[i] != 0;
    }
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane_id() >= o) upto += below;
    }
    __syncthreads();
    int at = 0;
    if (lane_id() == 31) at = int(atomicAdd(&sh.entries, uint32_t(upto)));
    at = __shfl_sync(0xffffffffu, at, 31) + upto - count;
#pragma unroll
    for (int i = 0; i < COLLECTED / TOP_THREADS; ++i)
      if (mine[i]) sh.places[at++] = mine[i];
    __syncthreads();
    int entries = int(sh.entries);
    Record more = {LOWEST, 0.f, 0.f, 0u};
    if (bad) {
      entries = 0;
    } else if (rec.flags & FULL) {
      entries = exact_entries(sh, scale, more);
      rec = {LOWEST, 0.f, 0.f, 0u};
    }
    // Each entry's place: the larger ones, two at a time (0 is none).
    if (tid == 0) sh.places[min(entries, COLLECTED - 1)] = entries < COLLECTED ? 0 : sh.places[COLLECTED - 1];
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < entries; i += TOP_THREADS) {
      const uint64_t entry = sh.places[i];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < entries; j += 2) {
        const ulonglong2 pair = *reinterpret_cast<const ulonglong2*>(&sh.places[j]);
        place += (pair.x > entry) + (pair.y > entry);
      }
      const float value = key_value(uint32_t(entry >> 32));
      if (place < p.k) write(place, value, int64_t(0xffffffffu - uint32_t(entry)));
      else sh.beyond[place] = value;
    }
    for (int i = entries + tid; i < p.k; i += TOP_THREADS) write(i, -INFINITY, -1);
    __syncthreads();
    for (int i = p.k + tid; i < entries; i += TOP_THREADS) {
      const float m = fmaxf(more.m, sh.beyond[i]);
      more.s = __fadd_rn(__fmul_rn(ex2(exponent(more.m, m, scale)), more.s), ex2(exponent(sh.beyond[i], m, scale)));
      more.m = m;
    }
    more = lanes_record<false, 32>(more, scale);
    if (lane_id() == 0) sh.inbox[warp_id()] = more;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < TOP_WARPS; ++w) {
        const float m = fmaxf(rec.m, sh.inbox[w].m);
        rec.s = __fadd_rn(__fmul_rn(ex2(exponent(rec.m, m, scale)), rec.s), __fmul_rn(ex2(exponent(sh.inbox[w].m, m, scale)), sh.inbox[w].s));
        rec.m = m;
      }
      const bool ok = !bad && entries > 0;
      p.rest[row] = ok && rec.s > 0 ? value_of(pair_sum(scaled_gap(rec.m, 0.f, temperature), log_pair(rec.s))) : -INFINITY;
      p.status[row] = bad ? ES_INVALID_INPUT : ok ? ES_OK : ES_NO_VALID_TOKEN;
    }
  }
};

template <int DT> __global__ void __launch_bounds__(TOP_THREADS, TOP_BLOCKS) top_rows(const __grid_constant__ TopParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = p.in.ranks, rank = int(blockIdx.x % unsigned(ranks));
  const int begin = rank * p.in.slice, n = min(p.in.slice, p.in.vocab - begin);
  TopRow<DT> work{p, int64_t(blockIdx.x / unsigned(ranks)), rank, ranks, begin, n, int(threadIdx.x)};
  work.run(*reinterpret_cast<TopShared*>(smem));
}

inline size_t top_smem(int slice) {
  const size_t steps = size_t((slice + 32 * TOP_THREADS - 1) / (32 * TOP_THREADS)) * TOP_THREADS * sizeof(float2);
  return std::max(sizeof(TopShared), offsetof(TopShared, steps) + steps);
}
template <int DT> cudaError_t launch_top(const TopParams& p, cudaStream_t stream) {
  static Configured configured;
  return launch_clusters(top_rows<DT>, p, false, p.in.rows, p.in.ranks, TOP_THREADS, top_smem(p.in.slice), stream, configured);
}

}  // namespace score
}  // namespace es
