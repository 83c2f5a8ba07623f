// The k largest logits of each row, sorted, and the log-sum of the rest
// (top_rows): one pass over the row, which never lies in shared memory, so
// that as many blocks as registers allow keep the memory busy.
//
// A row is split over a cluster; a thread goes through every THREADS-th chunk
// of its rank's slice:
//   1. each thread takes the maximum and the running sum of its tokens;
//   2. each rank finds the ceil(k / ranks)-th largest of its threads' maxima
//      (to 18 bits of its key). At least that many of its tokens reach it, so
//      the smallest of the ranks' values is a bound that at least k tokens of
//      the row reach, and few more (a thread rarely holds two of the largest);
//   3. the few threads whose maximum reaches the bound give up their sums.
//      Their chunks are read again, from L2: tokens at or above the bound are
//      listed, the others summed. So the rest is summed without the largest,
//      and one far below them loses no digits to a subtraction;
//   4. rank 0 has every rank's list, places each entry by the number of larger
//      ones, and adds the entries past the k-th to the rest.
// Entries are 64-bit words, the logit's order key above the complement of its
// id, so that all are distinct and equal logits rank by the lowest id. Where a
// rank lists more than its places on rank 0 (equal values, in the main), rank
// 0 finds the exact threshold by a digit-by-digit count over the whole row.
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

constexpr int TOP_THREADS = 256, TOP_WARPS = TOP_THREADS / 32;
constexpr uint32_t KEY_NONE = 0x007fffffu;  // the key of -inf: not a token of the row
constexpr int COLLECTED = 2048;             // entries rank 0 takes, an equal share from each rank
static_assert(COLLECTED >= 2 * MAX_TOP, "a single rank's list holds k entries and more");

struct TopShared {
  Record inbox[MAX_RANKS], bounds[MAX_RANKS];
  Record warps[TOP_WARPS];
  uint64_t bar[2];
  uint32_t keys[TOP_THREADS];
  uint32_t hot[TOP_WARPS];   // a bit per thread
  uint16_t owners[TOP_THREADS];
  uint32_t listed, counts[MAX_RANKS];
  uint32_t digits[TOP_WARPS][8];
  uint32_t place[COLLECTED];
  float beyond[COLLECTED];   // values past the k-th, by place
  uint64_t collected[COLLECTED];
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

  const TopParams& p;
  int64_t row;
  int rank, ranks, begin, n, tid;

  __device__ __forceinline__ const T* source() const {
    return static_cast<const T*>(p.in.logits) + row * p.in.l_s0 + int64_t(begin) * p.in.l_s1;
  }
  // Chunk c of the slice, -inf past its end and at masked tokens. ALIGNED: the
  // slice starts on 16 bytes (c a whole chunk).
  template <bool ALIGNED> __device__ __forceinline__ uint4 chunk(const T* src, int c) const {
    if (ALIGNED) return __ldg(reinterpret_cast<const uint4*>(src) + c);
    const uint32_t shift = uint32_t(reinterpret_cast<uintptr_t>(src)) & 15;
    if (p.in.l_s1 == 1 && shift != 0 && c > 0 && (c + 2) * N <= n) {
      // Cut out of the two aligned pieces it lies in, both inside the slice.
      const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) - shift) + c;
      const uint4 pieces[2] = {__ldg(from), __ldg(from + 1)};
      return shifted_chunk<sizeof(T)>(pieces, shift);
    }
    uint4 q;
    T* v = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c * N + i < n ? src[(c * N + i) * p.in.l_s1] : E::put(-INFINITY);
    return q;
  }
  // Sets masked tokens to -inf; looks at them first.
  __device__ __forceinline__ void apply_mask(const int32_t* mask, int c, uint4& q, bool& bad) const {
    bad |= !(chunk_max_nan<DT>(q) < INFINITY);
    q = mask_chunk<DT>(q, uint32_t(mask[(c * N >> 5) * p.in.mask.s1]) >> (c * N & 31), lowest_word<DT>());
  }

  // Every thread's tokens: their maximum and sum.
  template <bool ALIGNED> __device__ __forceinline__ Record sums(const T* src, const int32_t* mask, float scale, bool& bad) const {
    const int chunks = (n + N - 1) / N, whole = ALIGNED ? n / N : chunks;
    Acc a = acc_none();
    int c = tid;
#pragma unroll 1
    for (; c + 3 * TOP_THREADS < whole; c += 4 * TOP_THREADS) {
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = chunk<ALIGNED>(src, c + i * TOP_THREADS);
      if (mask) {
#pragma unroll
        for (int i = 0; i < 4; ++i) apply_mask(mask, c + i * TOP_THREADS, q[i], bad);
      }
      const float top = fmaxf(chunk_max<DT>(q[0], q[1]), chunk_max<DT>(q[2], q[3]));
      float2 v[2 * N];
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack<DT>(q[i], v + i * N / 2);
      acc_fast<4 * N, false>(a, v, top, scale);
    }
#pragma unroll 1
    for (; c < chunks; c += TOP_THREADS) {
      uint4 q = c < whole ? chunk<ALIGNED>(src, c) : chunk<false>(src, c);
      if (mask) apply_mask(mask, c, q, bad);
      float2 v[N / 2];
      unpack<DT>(q, v);
      acc_fast<N, false>(a, v, chunk_max<DT>(q, q), scale);
    }
    const bool failed = acc_failed<false>(a) || scale < SMALL_SCALE;
    if (failed) {
      a = acc_none();
      for (c = tid; c < chunks; c += TOP_THREADS) {
        uint4 q = chunk<false>(src, c);
        if (mask) apply_mask(mask, c, q, bad);
        float2 v[N / 2];
        unpack<DT>(q, v);
        acc_careful<N, false>(a, v, max_of<N>(v), scale);
      }
    }
    return acc_exact<false>(a, scale, failed);
  }

  // A bound that at least `need` of the threads' keys reach, its low 14 bits
  // zero: the keys' common leading bits, then one bit a step. Every warp finds
  // it for itself. 0 if fewer threads than that have any token.
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
    if (need > TOP_THREADS) return 0;
    const int differ = 31 - __clz(int((low ^ high) | 1u));
    uint32_t found = high & ~(differ == 31 ? 0xffffffffu : (2u << differ) - 1u);
    for (int bit = differ; bit >= 14; --bit) {
      const uint32_t least = found | (1u << bit);
      int above = 0;
#pragma unroll
      for (int i = 0; i < TOP_WARPS; ++i) above += key[i] >= least;
      if (int(__reduce_add_sync(0xffffffffu, unsigned(above))) >= need) found = least;
    }
    return found;
  }

  __device__ __forceinline__ Record block_record(TopShared& sh, Record rec, float scale) const {
    rec = lanes_record<false, 32>(rec, scale);
    __syncthreads();
    if (lane_id() == 0) sh.warps[warp_id()] = rec;
    __syncthreads();
    return join_records<false, TOP_WARPS>(sh.warps, TOP_WARPS, scale);
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
        sh.collected[atomicAdd(&sh.listed, 1u)] = entry;
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
      mbar_init(&sh.bar[1], ranks);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      mbar_arrive_expect_tx(&sh.bar[0], uint32_t(ranks * sizeof(Record)));
      sh.listed = 0;
    }
    cluster_started();
    const Scale temperature = row_scale(p.in, row);
    const float scale = temperature.log2;
    const T* src = source();
    const int32_t* mask = p.in.mask.p ? p.in.mask.p + row * p.in.mask.s0 + (begin >> 5) * p.in.mask.s1 : nullptr;
    bool bad = temperature.bad;
    const bool aligned = p.in.l_s1 == 1 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    Record own = aligned ? sums<true>(src, mask, scale, bad) : sums<false>(src, mask, scale, bad);
    bad |= !(own.s < INFINITY) || own.m == INFINITY;
    const uint32_t key = own.s > 0.f ? order_key(own.m) : 0u;
    sh.keys[tid] = key;
    cluster_wait();  // every rank has started
    __syncthreads();

    const uint32_t found = max(thread_bound(sh.keys, (p.k + ranks - 1) / ranks), KEY_NONE + 1);
    if (tid < ranks) send_record(&sh.bounds[rank], &sh.bar[0], tid, Record{0.f, 0.f, 0.f, found});
    if (!wait_bar(&sh.bar[0], 0)) bad = true;
    uint32_t bound = 0xffffffffu;
    for (int r = 0; r < ranks; ++r) bound = min(bound, sh.bounds[r].flags);

    // The threads whose maximum reaches the bound, in order (sums are to have
    // one order too), and their chunks again.
    const uint32_t hot = __ballot_sync(0xffffffffu, key >= bound);
    if (lane_id() == 0) sh.hot[warp_id()] = hot;
    __syncthreads();
    int owners = 0;
    for (int w = 0; w < TOP_WARPS; ++w) {
      if (w == warp_id() && key >= bound) {
        sh.owners[owners + __popc(hot & ((1u << lane_id()) - 1))] = uint16_t(tid);
        own = {LOWEST, 0.f, 0.f, 0u};
      }
      owners += __popc(sh.hot[w]);
    }
    __syncthreads();
    const int share = COLLECTED / ranks, chunks = (n + N - 1) / N, each = (chunks + TOP_THREADS - 1) / TOP_THREADS;
    uint64_t* places = cg::this_cluster().map_shared_rank(sh.collected, 0) + rank * share;
    Acc a = {own.m, 0.f, {own.s, 0.f}, {0.f, 0.f}};
    for (int task = tid; task < owners * each; task += TOP_THREADS) {
      const int c = sh.owners[task / each] + task % each * TOP_THREADS;
      if (c >= chunks) continue;
      uint4 q = aligned && (c + 1) * N <= n ? chunk<true>(src, c) : chunk<false>(src, c);
      if (mask) apply_mask(mask, c, q, bad);
      float2 v[N / 2];
      unpack<DT>(q, v);
      float* f = reinterpret_cast<float*>(v);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (order_key(f[i]) >= bound) {
          const uint32_t at = atomicAdd(&sh.listed, 1u);
          if (int(at) < share) places[at] = entry_of(order_key(f[i]), begin + c * N + i);
          f[i] = -INFINITY;
        }
      }
      acc_careful<N, false>(a, v, max_of<N>(v), scale);
    }
    Record rec = acc_exact<false>(a, scale, true);
    rec.flags = bad ? BAD : 0u;
    rec = block_record(sh, rec, scale);
    if (tid == 0) {
      const uint32_t listed = sh.listed;
      rec.flags |= int(listed) > share ? FULL : 0u;
      cg::this_cluster().map_shared_rank(sh.inbox, 0)[rank] = rec;
      cg::this_cluster().map_shared_rank(sh.counts, 0)[rank] = listed;
      arrive_at(&sh.bar[1], 0);
    }
    if (rank != 0) return;

    const bool came = wait_cluster(&sh.bar[1]);
    rec = join_records<false, MAX_RANKS>(sh.inbox, ranks, scale);
    bad = (rec.flags & BAD) || !came;
    Record more = {LOWEST, 0.f, 0.f, 0u};
    int entries = 0;
    if (!bad && (rec.flags & FULL)) {
      entries = exact_entries(sh, scale, more);
      rec = {LOWEST, 0.f, 0.f, 0u};
    } else if (!bad) {
      // The ranks' lists side by side.
      uint64_t mine[COLLECTED / TOP_THREADS];
#pragma unroll
      for (int i = 0; i < COLLECTED / TOP_THREADS; ++i) {
        const int at = i * TOP_THREADS + tid, r = at / share;
        mine[i] = r < ranks && at % share < int(sh.counts[r]) ? sh.collected[at] : 0;
      }
      if (tid == 0) sh.listed = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < COLLECTED / TOP_THREADS; ++i)
        if (mine[i]) sh.collected[atomicAdd(&sh.listed, 1u)] = mine[i];
      __syncthreads();
      entries = int(sh.listed);
    }
    // Places, several threads to an entry where there are few.
    for (int i = tid; i < entries; i += TOP_THREADS) sh.place[i] = 0;
    __syncthreads();
    const int parts = max(1, TOP_THREADS / max(entries, 1)), length = (entries + parts - 1) / parts;
    for (int i = tid; i < entries * parts; i += TOP_THREADS) {
      const int mine = i % entries, from = i / entries * length, to = min(from + length, entries);
      const uint64_t entry = sh.collected[mine];
      uint32_t larger = 0;
#pragma unroll 4
      for (int j = from; j < to; ++j) larger += sh.collected[j] > entry;
      if (larger) atomicAdd(&sh.place[mine], larger);
    }
    __syncthreads();
    for (int i = tid; i < entries; i += TOP_THREADS) {
      const uint64_t entry = sh.collected[i];
      const float value = key_value(uint32_t(entry >> 32));
      if (int(sh.place[i]) < p.k) {
        write(sh.place[i], value, int64_t(0xffffffffu - uint32_t(entry)));
      } else {
        sh.beyond[sh.place[i]] = value;
      }
    }
    for (int i = entries + tid; i < p.k; i += TOP_THREADS) write(i, -INFINITY, -1);
    __syncthreads();
    for (int i = p.k + tid; i < entries; i += TOP_THREADS) {
      const float m = fmaxf(more.m, sh.beyond[i]);
      more.s = __fadd_rn(__fmul_rn(ex2(exponent(more.m, m, scale)), more.s), ex2(exponent(sh.beyond[i], m, scale)));
      more.m = m;
    }
    more = block_record(sh, more, scale);
    if (tid == 0) {
      const float m = fmaxf(more.m, rec.m);
      const float s = __fadd_rn(__fmul_rn(more.s, ex2(exponent(more.m, m, scale))), __fmul_rn(rec.s, ex2(exponent(rec.m, m, scale))));
      const bool ok = !bad && entries > 0;
      p.rest[row] = ok && s > 0 ? value_of(pair_sum(scaled_gap(m, 0.f, temperature), log_pair(s))) : -INFINITY;
      p.status[row] = bad ? ES_INVALID_INPUT : ok ? ES_OK : ES_NO_VALID_TOKEN;
    }
  }
};

template <int DT> __global__ void __launch_bounds__(TOP_THREADS, 4) top_rows(const __grid_constant__ TopParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = p.in.ranks, rank = int(blockIdx.x % unsigned(ranks));
  const int begin = rank * p.in.slice, n = min(p.in.slice, p.in.vocab - begin);
  TopRow<DT> work{p, int64_t(blockIdx.x / unsigned(ranks)), rank, ranks, begin, n, int(threadIdx.x)};
  work.run(*reinterpret_cast<TopShared*>(smem));
}

template <int DT> cudaError_t launch_top(const TopParams& p, cudaStream_t stream) {
  static Configured configured;
  return launch_clusters(top_rows<DT>, p, false, p.in.rows, p.in.ranks, TOP_THREADS, sizeof(TopShared), stream, configured);
}

}  // namespace score
}  // namespace es
