// The k largest logits of each row, sorted, and the log-sum of the rest
// (top_rows): one read of the row.
//
// A row is split over a cluster and kept in shared memory as in es_score.cuh.
// Selection needs no sort of the row:
//   1. each thread takes the maximum of its tokens as they arrive;
//   2. each rank finds the ceil(k / ranks)-th largest of its threads' maxima
//      (to 16 bits of its key). At least that many of its tokens reach it, so
//      the smallest of the ranks' values is a bound that at least k tokens of
//      the row reach, and few more (a thread rarely holds two of the largest);
//   3. tokens at or above the bound are listed and leave the slice; the pass
//      over what is left sums the rest without them, so that a rest far below
//      the largest logits loses no digits to a subtraction;
//   4. rank 0 gets every rank's list, places each entry by the number of
//      larger ones, and adds the entries past the k-th to the rest.
// Entries are 64-bit words, the logit's order key above the complement of its
// id, so that all are distinct and equal logits rank by the lowest id.
// Rows with too many tokens at the bound (equal values, in the main) take the
// exact threshold from a digit-by-digit count over the cluster instead.
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

constexpr uint32_t KEY_NONE = 0x007fffffu;  // the key of -inf: not a token of the row
constexpr int LISTED = 512;                 // entries a rank lists
constexpr int COLLECTED = 1024;             // entries rank 0 takes

static_assert(THREADS >= 8 * MAX_RANKS, "exact_threshold's exchange has a thread per digit and rank");

struct TopShared {
  Record inbox[MAX_RANKS];
  Record warps[WARPS];
  uint32_t bound[MAX_RANKS];
  uint32_t digits[2][MAX_RANKS][8];
  uint32_t warp_digits[WARPS][8];
  uint32_t listed, total, place;
  uint64_t list[LISTED];
  uint64_t collected[COLLECTED];
};

template <int DT> __host__ __device__ constexpr size_t top_smem(int slice) {
  return (sizeof(TopShared) + 15) / 16 * 16 + slice_bytes<DT>(slice);
}

__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) { return (uint64_t(key) << 32) | (0xffffffffu - uint32_t(id)); }

template <int DT> struct TopRow {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int N = E::N;

  const TopParams& p;
  int64_t row;
  int rank, ranks, begin, n, tid;

  // A bound with 16 zero bits below that at least `need` of the threads' keys
  // reach; 0 if fewer threads than that have any token.
  __device__ __forceinline__ uint32_t thread_bound(uint32_t key, int need) const {
    uint32_t found = 0;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
      if (__syncthreads_count(key >= (found | bit)) >= need) found |= bit;
    return found;
  }

  // The k-th largest entry of the whole row (the smallest possible one when
  // fewer tokens are valid): three bits of the entry a step, counted over the cluster.
  __device__ __noinline__ uint64_t exact_threshold(TopShared& sh, const Slice<DT>& slice) const {
    uint64_t found = 0;
    uint32_t need = p.k;
    int turn = 0;
    for (int shift = 63; shift >= 0; shift -= 3, turn ^= 1) {  // bit 63 alone, then 21 digits of three bits
      uint64_t low = 0, high = 0;  // this thread's counts of the digits 0-3 and 4-7, 16 bits each
      for (int i = tid; i < n; i += THREADS) {
        const uint32_t key = order_key(E::get(slice[i]));
        const uint64_t entry = entry_of(key, begin + i);
        if (key > KEY_NONE && (shift == 63 || ((entry ^ found) >> (shift + 3)) == 0)) {
          const int digit = int(entry >> shift) & 7;
          if (digit < 4) low += 1ull << (16 * digit);
          else high += 1ull << (16 * (digit - 4));
        }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const uint32_t mine = uint32_t((d < 4 ? low : high) >> (16 * (d & 3))) & 0xffff;
        const uint32_t sum = __reduce_add_sync(0xffffffffu, mine);
        if (lane_id() == 0) sh.warp_digits[warp_id()][d] = sum;
      }
      __syncthreads();
      if (tid < 8 * ranks) {
        uint32_t sum = 0;
        for (int w = 0; w < WARPS; ++w) sum += sh.warp_digits[w][tid & 7];
        cg::this_cluster().map_shared_rank(&sh.digits[turn][rank][tid & 7], tid >> 3)[0] = sum;
      }
      cluster_arrive();
      cluster_wait();
      uint32_t above = 0, digit = 8, at = 0;
      while (digit > 0 && above + at < need) {  // from the largest digit down
        above += at;
        --digit;
        at = 0;
        for (int r = 0; r < ranks; ++r) at += sh.digits[turn][r][digit];
      }
      if (above + at < need) return uint64_t(KEY_NONE + 1) << 32;  // every valid token
      need -= above;
      found |= uint64_t(digit) << shift;
      __syncthreads();  // warp_digits are rewritten next
    }
    return found;
  }

  // Lists the tokens at or above `least` and takes them out of the slice. A
  // warp goes through the tokens of each of its threads whose maximum reaches it.
  __device__ __forceinline__ void list_entries(TopShared& sh, uint32_t key, const Slice<DT>& slice, uint64_t least) const {
    uint32_t hot = __ballot_sync(0xffffffffu, key >= uint32_t(least >> 32));
    while (hot) {
      const int owner = warp_id() * 32 + __ffs(hot) - 1;
      hot &= hot - 1;
      for (int first = owner; first < slice.chunks; first += THREADS * (32 / N)) {
        const int i = (first + lane_id() / N * THREADS) * N + lane_id() % N;
        if (i >= n) continue;
        const uint64_t entry = entry_of(order_key(E::get(slice[i])), begin + i);
        if (entry < least) continue;
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < LISTED) {
          sh.list[at] = entry;
          slice[i] = E::put(-INFINITY);
        }
      }
    }
  }

  __device__ __forceinline__ void write(int64_t at, float value, int64_t id) const {
    p.values.p[row * p.values.s0 + at * p.values.s1] = value;
    p.ids.p[row * p.ids.s0 + at * p.ids.s1] = id;
  }

  __device__ __forceinline__ Record block_record(TopShared& sh, Record rec, float scale) const {
    rec = lanes_record<false, 32>(rec, scale);
    __syncthreads();
    if (lane_id() == 0) sh.warps[warp_id()] = rec;
    __syncthreads();
    return join_records<false, WARPS>(sh.warps, WARPS, scale);
  }

  __device__ __forceinline__ void run(uint8_t* smem) {
    TopShared& sh = *reinterpret_cast<TopShared*>(smem);
    uint8_t* buffer = smem + (sizeof(TopShared) + 15) / 16 * 16;
    bool bad = false;
    if (tid == 0) sh.listed = sh.total = 0;
    cluster_arrive();  // this rank's shared memory may be written from now on
    Slice<DT> slice;
    slice.init(buffer, n);
    slice.load(p.in, row, begin);
    const Scale temperature = row_scale(p.in, row);
    const float scale = temperature.log2;
    bad |= temperature.bad;
    slice.arrive();
    slice.arrive_rest();

    // This thread's maximum; masked tokens leave the slice.
    const int32_t* mask = p.in.mask.p ? p.in.mask.p + row * p.in.mask.s0 + (begin >> 5) * p.in.mask.s1 : nullptr;
    float top = -INFINITY;
    if (mask) {
      for (int c = tid; c < slice.chunks; c += THREADS) {
        float2 v[N / 2];
        unpack<DT>(slice.chunk(c), v);
        bad |= chunk_bad<DT>(v);
        mask_chunk<DT>(mask_bits<DT>(mask, p.in.mask.s1, c * N), -INFINITY, v);
        slice.chunk(c) = pack<DT>(v);
        top = fmaxf(top, max_of<N>(v));
      }
    } else {
#pragma unroll 4
      for (int c = tid; c < slice.chunks; c += THREADS) top = max_nan(top, chunk_max_nan<DT>(slice.chunk(c)));
    }
    bad |= !(top < INFINITY);
    const uint32_t key = order_key(top);
    __syncthreads();
    cluster_wait();  // every rank has started

    const uint32_t own = max(thread_bound(key, (p.k + ranks - 1) / ranks), KEY_NONE + 1);
    if (tid < ranks) cg::this_cluster().map_shared_rank(sh.bound, tid)[rank] = own;
    cluster_arrive();
    cluster_wait();
    uint32_t bound = 0xffffffffu;
    for (int r = 0; r < ranks; ++r) bound = min(bound, sh.bound[r]);
    uint64_t least = uint64_t(bound) << 32;

    for (bool exact = false;; exact = true) {
      list_entries(sh, key, slice, least);
      __syncthreads();
      const uint32_t listed = sh.listed;
      const bool fits = listed <= LISTED;
      // Rank 0's places for this rank's entries: asked for now, used after the sums.
      if (tid == 0) sh.place = fits ? atomicAdd(cg::this_cluster().map_shared_rank(&sh.total, 0), listed) : COLLECTED;
      Record rec = {LOWEST, 0.f, 0.f, 0u};
      if (fits) rec = sum_slice<DT, false, false>(slice, nullptr, 0, scale);
      if (bad) rec.flags |= BAD;
      rec = block_record(sh, rec, scale);
      const bool room = sh.place + listed <= COLLECTED;
      rec.flags |= room ? 0 : FULL;
      if (room) {
        uint64_t* to = cg::this_cluster().map_shared_rank(sh.collected, 0) + sh.place;
        for (uint32_t i = tid; i < listed; i += THREADS) to[i] = sh.list[i];
      }
      if (tid < ranks) cg::this_cluster().map_shared_rank(sh.inbox, tid)[rank] = rec;
      cluster_arrive();
      cluster_wait();
      uint32_t flags = 0;
      for (int r = 0; r < ranks; ++r) flags |= sh.inbox[r].flags;
      bad = flags & BAD;
      if (!(flags & FULL) || bad || exact) break;
      // Too many entries: put the listed ones back and take the exact threshold.
      for (uint32_t i = tid; i < min(listed, uint32_t(LISTED)); i += THREADS)
        slice[int(0xffffffffu - uint32_t(sh.list[i])) - begin] = E::put(key_value(uint32_t(sh.list[i] >> 32)));
      if (tid == 0) sh.listed = sh.total = 0;
      __syncthreads();
      least = exact_threshold(sh, slice);
    }
    if (rank != 0) return;

    const int entries = bad ? 0 : int(min(sh.total, uint32_t(COLLECTED)));
    Record rec = {LOWEST, 0.f, 0.f, 0u};
    for (int i = tid; i < entries; i += THREADS) {
      const uint64_t mine = sh.collected[i];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < entries; ++j) place += sh.collected[j] > mine;
      const float value = key_value(uint32_t(mine >> 32));
      if (place < p.k) {
        write(place, value, int64_t(0xffffffffu - uint32_t(mine)));
      } else {
        const float m = fmaxf(rec.m, value);
        rec.s = __fadd_rn(__fmul_rn(ex2(exponent(rec.m, m, scale)), rec.s), ex2(exponent(value, m, scale)));
        rec.m = m;
      }
    }
    for (int i = entries + tid; i < p.k; i += THREADS) write(i, -INFINITY, -1);
    rec = block_record(sh, rec, scale);
    if (tid == 0) {
      float m = rec.m;
      for (int r = 0; r < ranks; ++r) m = fmaxf(m, sh.inbox[r].m);
      float s = rec.s * ex2(exponent(rec.m, m, scale));
      for (int r = 0; r < ranks; ++r) s += sh.inbox[r].s * ex2(exponent(sh.inbox[r].m, m, scale));
      const bool ok = !bad && entries > 0;
      p.rest[row] = ok && s > 0 ? value_of(pair_sum(scaled_gap(m, 0.f, temperature), log_pair(s))) : -INFINITY;
      p.status[row] = bad ? ES_INVALID_INPUT : ok ? ES_OK : ES_NO_VALID_TOKEN;
    }
  }
};

template <int DT> __global__ void __launch_bounds__(THREADS, ES_SCORE_BLOCKS) top_rows(const __grid_constant__ TopParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = p.in.ranks, rank = int(blockIdx.x % unsigned(ranks));
  const int begin = rank * p.in.slice, n = min(p.in.slice, p.in.vocab - begin);
  TopRow<DT> work{p, int64_t(blockIdx.x / unsigned(ranks)), rank, ranks, begin, n, int(threadIdx.x)};
  work.run(smem);
}

template <int DT> cudaError_t launch_top(const TopParams& p, cudaStream_t stream) {
  static Configured configured;
  return launch_clusters(top_rows<DT>, p, false, p.in.rows, p.in.ranks, top_smem<DT>(p.in.slice), stream, configured);
}

}  // namespace score
}  // namespace es
