// The k largest logits of each row, sorted, and the log-sum of the rest
// (top_rows): one read of the row.
//
// A row is split over a cluster and kept in shared memory as in es_score.cuh.
// Selection needs no sort of the row:
//   1. the load pass takes the maximum of every tile of 32 tokens;
//   2. each rank finds the ceil(k / ranks)-th largest of its tile maxima (to
//      18 bits of its key). At least that many of its tokens reach it, so the
//      smallest of the ranks' values is a bound that at least k tokens of the
//      row reach, and few more (a tile rarely holds two of the largest);
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
constexpr int TILE = 32;
constexpr uint32_t BAD = 1, FULL = 2;       // Record::bad: an invalid row, a list that did not fit

struct TopShared {
  uint64_t bar[PIECES];
  Record inbox[MAX_RANKS];
  Record warps[WARPS];
  uint32_t bound[MAX_RANKS];
  uint32_t tiles_above[2][8];
  uint32_t digits[2][MAX_RANKS][8];
  uint32_t warp_digits[WARPS][8];
  uint32_t listed, total, place;
  uint64_t list[LISTED];
  uint64_t collected[COLLECTED];
};

template <int DT> __host__ __device__ constexpr size_t top_smem(int slice) {
  return sizeof(TopShared) + size_t(slice) / TILE * 4 + 16 + size_t(slice) * sizeof(typename Elem<DT>::T) + 32;
}

__device__ __forceinline__ uint64_t entry_of(uint32_t key, int id) { return (uint64_t(key) << 32) | (0xffffffffu - uint32_t(id)); }

template <int DT> struct TopRow {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr int N = E::N;

  const TopParams& p;
  int64_t row;
  int rank, ranks, begin, n, tid;

  // Warps 1..7 count the tiles at or above seven thresholds at once, three
  // bits of the key a step, 18 bits in all. 0: fewer than `need` tiles.
  __device__ __forceinline__ uint32_t tile_bound(TopShared& sh, const uint32_t* tiles, int count, int need) const {
    uint32_t found = 0;
    int turn = 0;
    for (int shift = 29; shift >= 14; shift -= 3, turn ^= 1) {
      if (warp_id() > 0) {
        const uint32_t least = found | (uint32_t(warp_id()) << shift);
        int above = 0;
        for (int t = lane_id(); t < count; t += 32) above += tiles[t] >= least;
        above = __reduce_add_sync(0xffffffffu, above);
        if (lane_id() == 0) sh.tiles_above[turn][warp_id()] = above;
      }
      __syncthreads();
      int digit = 0;
#pragma unroll
      for (int w = 1; w < 8; ++w) digit += sh.tiles_above[turn][w] >= uint32_t(need);
      found |= uint32_t(digit) << shift;
    }
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

  // Lists the tokens at or above `least` and takes them out of the slice.
  __device__ __forceinline__ void list_entries(TopShared& sh, const uint32_t* tiles, int count, const Slice<DT>& slice,
                                               uint64_t least) const {
    const uint32_t least_key = uint32_t(least >> 32);
    for (int base = warp_id() * 32; base < count; base += THREADS) {
      const int t = base + lane_id();
      uint32_t hot = __ballot_sync(0xffffffffu, t < count && tiles[t] >= least_key);
      while (hot) {
        const int i = (base + __ffs(hot) - 1) * TILE + lane_id();
        hot &= hot - 1;
        uint64_t entry = 0;
        if (i < n) entry = entry_of(order_key(E::get(slice[i])), begin + i);
        const bool take = i < n && entry >= least;
        const uint32_t takers = __ballot_sync(0xffffffffu, take);
        uint32_t at = 0;
        if (lane_id() == 0) at = atomicAdd(&sh.listed, uint32_t(__popc(takers)));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(takers & ((1u << lane_id()) - 1));
        if (take && at < LISTED) {
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
#pragma unroll
    for (int o = 16; o; o >>= 1) rec = merge(rec, shfl_record(rec, o), scale);
    __syncthreads();
    if (lane_id() == 0) sh.warps[warp_id()] = rec;
    __syncthreads();
    rec = sh.warps[lane_id() & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o; o >>= 1) rec = merge(rec, shfl_record(rec, o), scale);
    return rec;
  }

  __device__ __forceinline__ void run(uint8_t* smem) {
    TopShared& sh = *reinterpret_cast<TopShared*>(smem);
    uint32_t* tiles = reinterpret_cast<uint32_t*>(smem + sizeof(TopShared));
    uint8_t* buffer = smem + ((sizeof(TopShared) + size_t(p.in.slice) / TILE * 4 + 15) & ~size_t(15));
    const int count = (n + TILE - 1) / TILE;
    bool bad = false;
    double temperature = p.in.temperature.p ? p.in.temperature[row] : p.in.temperature_all;
    float scale = float(LOG2E / temperature);
    if (!(temperature > 0 && scale >= 1.17549435e-38f && scale <= 3.402823466e38f)) {
      bad = true;
      temperature = 1;
      scale = float(LOG2E);
    }
    if (tid == 0) sh.listed = sh.total = 0;
    cluster_arrive();  // this rank's shared memory may be written from now on
    Slice<DT> slice;
    slice.load(p.in, row, begin, n, buffer, sh.bar);

    // Tile maxima: 32 / N neighbouring lanes hold a tile's chunks.
    const int32_t* mask = p.in.mask.p ? p.in.mask.p + row * p.in.mask.s0 : nullptr;
    for (int first = 0; first < slice.chunks; first += THREADS) {
      slice.wait(uint32_t(first + THREADS + 1) * 16);
      const int c = first + tid;
      float top = -INFINITY;
      if (c < slice.chunks) {
        float2 v[N / 2];
        unpack<DT>(slice.chunk(c), v);
        if (mask) {
          bad |= mask_chunk<DT>(mask, p.in.mask.s1, begin + c * N, v);
          slice.set_chunk(c, pack<DT>(v));
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) top = max_nan(top, max_nan(v[i].x, v[i].y));
        bad |= !(top < INFINITY);
      }
#pragma unroll
      for (int o = 1; o < TILE / N; o <<= 1) top = fmaxf(top, shfl_xor(top, o));
      if (c < slice.chunks && c % (TILE / N) == 0) tiles[c / (TILE / N)] = order_key(top);
    }
    slice.wait_all();
    bad |= slice.late;
    cluster_wait();  // every rank has started
    __syncthreads();

    const uint32_t own = max(tile_bound(sh, tiles, count, (p.k + ranks - 1) / ranks), KEY_NONE + 1);
    if (tid < ranks) cg::this_cluster().map_shared_rank(sh.bound, tid)[rank] = own;
    cluster_arrive();
    cluster_wait();
    uint32_t bound = 0xffffffffu;
    for (int r = 0; r < ranks; ++r) bound = min(bound, sh.bound[r]);
    uint64_t least = uint64_t(bound) << 32;

    for (bool exact = false;; exact = true) {
      list_entries(sh, tiles, count, slice, least);
      __syncthreads();
      const uint32_t listed = sh.listed;
      const bool fits = listed <= LISTED;
      // Rank 0's places for this rank's entries: asked for now, used after the sums.
      if (tid == 0) sh.place = fits ? atomicAdd(cg::this_cluster().map_shared_rank(&sh.total, 0), listed) : COLLECTED;
      Acc acc = acc_none();
      if (fits)
        for (int c = tid; c < slice.chunks; c += THREADS) {
          float2 v[N / 2];
          unpack<DT>(slice.chunk(c), v);
          acc_chunk<N, false>(acc, v, scale);
        }
      Record rec = {acc.m, __fadd_rn(acc.s.x, acc.s.y), 0.f, bad ? BAD : 0u};
      rec = block_record(sh, rec, scale);
      const bool room = sh.place + listed <= COLLECTED;
      rec.bad |= room ? 0 : FULL;
      if (room) {
        uint64_t* to = cg::this_cluster().map_shared_rank(sh.collected, 0) + sh.place;
        for (uint32_t i = tid; i < listed; i += THREADS) to[i] = sh.list[i];
      }
      if (tid < ranks) cg::this_cluster().map_shared_rank(sh.inbox, tid)[rank] = rec;
      cluster_arrive();
      cluster_wait();
      uint32_t flags = 0;
      for (int r = 0; r < ranks; ++r) flags |= sh.inbox[r].bad;
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
      for (int j = 0; j < entries; ++j) place += sh.collected[j] > mine;
      const float value = key_value(uint32_t(mine >> 32));
      if (place < p.k) write(place, value, int64_t(0xffffffffu - uint32_t(mine)));
      else rec = merge(rec, Record{value, 1.f, 0.f, 0u}, scale);
    }
    for (int i = entries + tid; i < p.k; i += THREADS) write(i, -INFINITY, -1);
    rec = block_record(sh, rec, scale);
    if (tid == 0) {
      float m = rec.m;
      for (int r = 0; r < ranks; ++r) m = fmaxf(m, sh.inbox[r].m);
      double s = rec.s * exp2(double(exponent(rec.m, m, scale)));
      for (int r = 0; r < ranks; ++r) s += sh.inbox[r].s * exp2(double(exponent(sh.inbox[r].m, m, scale)));
      const bool ok = !bad && entries > 0;
      p.rest[row] = ok && s > 0 ? float(double(m) / temperature + log(s)) : -INFINITY;
      p.status[row] = bad ? ES_INVALID_INPUT : ok ? ES_OK : ES_NO_VALID_TOKEN;
    }
  }
};

template <int DT> __global__ void __launch_bounds__(THREADS, 4) top_rows(const __grid_constant__ TopParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int ranks = p.in.ranks, rank = int(blockIdx.x % unsigned(ranks));
  const int begin = rank * p.in.slice, n = min(p.in.slice, p.in.vocab - begin);
  TopRow<DT> work{p, int64_t(blockIdx.x / unsigned(ranks)), rank, ranks, begin, n, int(threadIdx.x)};
  work.run(smem);
}

template <int DT> cudaError_t launch_top(const TopParams& p, int64_t rows, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  return launch_clusters(top_rows<DT>, p, rows, p.in.ranks, top_smem<DT>(p.in.slice), stream, configured);
}

}  // namespace score
}  // namespace es
