// Eviction from a paged key-value cache by accumulated attention weight.
//
// Two launches: one finds the keys that stay, one moves their rows. (Few small caches: one launch for both.)
//
// Which stay: the weights are ordered as unsigned integers; the weight of the last key to stay is found digit by digit (8
// bits) from histograms in shared memory. Above it all stay, of its equals the first ones. A cluster of C blocks shares a cache,
// its histograms and counts meet through distributed shared memory; digits of 8 bits because reading 2048 bins of eight blocks
// took longer (43 us for 16 caches of 64k keys) than a fourth pass. Bound by the chain of passes and barriers.
//
// Moving: memory bounds it. Into other pages, blocks take stretches of rows and everything is independent. In place, the row that
// goes to place i lies at place i or behind it, so one block moves a column of 32 bytes of all rows in order, reading a round's
// rows before it writes any: columns are independent of each other, and the next round's rows lie behind all places written. A
// row's page and slot are looked up once per round, not by every thread that copies 16 bytes of it.
#include "cluster.cuh"
#include "kv_cache.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kDigits = 4, kBins = 256, kCopies = 2;  // weights crowd into few exponents: lanes count in two copies
constexpr int kCached = 8192;                         // weights of a block that are kept in shared memory
constexpr int kMoveThreads = 256, kMovePieces = 8, kMoveRows = 512;

struct Evict {
  PagedRows rows;
  const int32_t* dst_table;
  int64_t dst_ld;
  char* pool[2];
  const int32_t* lengths;
  int32_t *kept, *new_lengths;
  const float* weights;
  float* weights_out;
  int64_t weights_ld, weights_out_ld;
  int budget, recent, Hk;
  int pieces;        // of a row
  int cols, per_col; // columns that a row is cut into, pieces of a column
  int round;         // rows that are on their way at a time
  int chunk, chunks; // rows of a stretch, stretches
  int pools_in_place, weights_in_place;
};

// weights in the order of unsigned integers; a NaN is the lowest, both zeros are equal
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SelectShared {
  uint32_t hist[kDigits][kCopies][kBins];
  uint32_t cache[kCached];
  uint32_t warp_sum[kBins / 32];
  uint32_t bin, above;                  // the digit that was found, elements with a larger one
  uint32_t stay[kSelWarps], tie[kSelWarps];
  uint32_t block_stay, block_tie;
};

// The largest digit such that at least `want` elements of the cluster have it or a larger one, and the number with a larger one.
template <int C>
__device__ __forceinline__ void find_digit(SelectShared& sm, uint32_t (&hist)[kCopies][kBins], uint32_t want) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t n = 0, incl = 0;
  if (tid < kBins) {  // thread t: the t-th digit from the top
    if constexpr (C > 1) {  // (the copies of a block are its first one by now)
#pragma unroll
      for (int r = 0; r < C; ++r) n += peer_u32<C>(&hist[0][kBins - 1 - tid], r);
    } else {
#pragma unroll
      for (int k = 0; k < kCopies; ++k) n += hist[k][kBins - 1 - tid];
    }
    incl = n;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, x);
      if (lane >= x) incl += y;
    }
    if (lane == 31) sm.warp_sum[warp] = incl;
  }
  __syncthreads();
  if (tid < kBins) {
    const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_sum[lane] : 0u) + incl - n;
    if (before < want && before + n >= want) {
      sm.bin = kBins - 1 - tid;
      sm.above = before;
    }
  }
  __syncthreads();
}

// Positions that stay of the cache of cluster blockIdx.x / C.
template <int C>
__device__ __forceinline__ void select(const Evict& p, SelectShared& sm) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_rank<C>());
  const int seg = blockIdx.x / C, b = seg / p.Hk;
  const int n = p.rows.length(p.lengths, b), keep = min(n, p.budget);
  if (tid == 0 && rank == 0 && seg % p.Hk == 0) p.new_lengths[b] = keep;
  const float* w = p.weights + seg * p.weights_ld;
  int32_t* kept = p.kept + static_cast<int64_t>(seg) * p.budget;
  for (int i = keep + rank * kSelThreads + tid; i < p.budget; i += C * kSelThreads) kept[i] = -1;
  if (n <= p.budget) {  // the whole cluster
    for (int i = rank * kSelThreads + tid; i < n; i += C * kSelThreads) kept[i] = i;
    return;
  }
  const int cand = n - p.recent, want = p.budget - p.recent;
  // contiguous stretches of the sequence, one per warp of the cluster
  const int per = (n + C * kSelWarps * 32 - 1) / (C * kSelWarps * 32) * 32;
  const int j0 = min((rank * kSelWarps + warp) * per, n), j1 = min(j0 + per, n);
  const int c1 = min(j1, cand);
  const bool cached = per * kSelWarps <= kCached;
  uint32_t* mine = sm.cache + warp * per - j0;  // ranks of this warp's stretch, if they fit
  auto rank_at = [&](int j) { return cached ? mine[j] : rank_of(w[j]); };
  for (int i = tid; i < kDigits * kCopies * kBins; i += kSelThreads) (&sm.hist[0][0][0])[i] = 0u;
  __syncthreads();
  uint32_t thr = 0;  // (want 0: nothing but the recent ones stays)
  int ties = 0;
  if (want > 0) {
    uint32_t left = want;
#pragma unroll
    for (int pass = 0; pass < kDigits; ++pass) {
      const int shift = 24 - 8 * pass;
      const uint32_t known = pass == 0 ? 0u : ~0u << (shift + 8);
#pragma unroll 8
      for (int j = j0 + lane; j < c1; j += 32) {
        const uint32_t r = pass == 0 ? rank_of(w[j]) : rank_at(j);
        if (pass == 0 && cached) mine[j] = r;
        if ((r & known) == thr) atomicAdd(&sm.hist[pass][lane % kCopies][(r >> shift) & 255u], 1u);
      }
      if constexpr (C > 1) {
        __syncthreads();
        if (tid < kBins)
#pragma unroll
          for (int k = 1; k < kCopies; ++k) sm.hist[pass][0][tid] += sm.hist[pass][k][tid];
      }
      cluster_barrier<C>();
      find_digit<C>(sm, sm.hist[pass], left);
      thr |= sm.bin << shift;
      left -= sm.above;
    }
    ties = static_cast<int>(left);  // equals of the threshold that stay
  }
  // numbers of keys above the threshold (or recent) and of equals before each warp's stretch
  int stay = max(j1 - max(j0, cand), 0), tie = 0;
  if (want > 0) {
    int s = 0;
#pragma unroll 8
    for (int j = j0 + lane; j < c1; j += 32) {
      const uint32_t r = rank_at(j);
      s += r > thr;
      tie += r == thr;
    }
    stay += __reduce_add_sync(0xffffffffu, s);
    tie = __reduce_add_sync(0xffffffffu, tie);
  }
  if (lane == 0) {
    sm.stay[warp] = stay;
    sm.tie[warp] = tie;
  }
  __syncthreads();
  int stays = __reduce_add_sync(0xffffffffu, lane < warp ? sm.stay[lane] : 0u);
  int tied = __reduce_add_sync(0xffffffffu, lane < warp ? sm.tie[lane] : 0u);
  if constexpr (C > 1) {
    if (warp == 0) {
      const uint32_t a = __reduce_add_sync(0xffffffffu, sm.stay[lane]), t = __reduce_add_sync(0xffffffffu, sm.tie[lane]);
      if (lane == 0) {
        sm.block_stay = a;
        sm.block_tie = t;
      }
    }
    cluster_barrier<C>();
    for (int r = 0; r < rank; ++r) {
      stays += peer_u32<C>(&sm.block_stay, r);
      tied += peer_u32<C>(&sm.block_tie, r);
    }
    cluster_barrier<C>();  // everything is read: a block may leave
  }
  for (int j = j0 + lane; j - lane < j1; j += 32) {
    const uint32_t r = j < c1 && want > 0 ? rank_at(j) : 0u;
    const bool equal = j < c1 && want > 0 && r == thr;
    const bool above = j < j1 && (j >= cand || (want > 0 && r > thr));
    const unsigned em = __ballot_sync(0xffffffffu, equal), am = __ballot_sync(0xffffffffu, above), low = (1u << lane) - 1u;
    const int e = tied + __popc(em & low), a = stays + __popc(am & low);
    if (above || (equal && e < ties)) kept[a + min(e, ties)] = j;
    tied += __popc(em);
    stays += __popc(am);
  }
}

template <int C>
__global__ void __launch_bounds__(kSelThreads)
select_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  extern __shared__ __align__(16) uint8_t smem[];
  select<C>(p, *reinterpret_cast<SelectShared*>(smem));
}

// Places of a round's rows, page and slot, from and to
struct Places {
  int2 from[3][kMoveRows], to[3][kMoveRows];
};

// Moves pieces [c_first, c_first + per_col) of rows [first, last) that stay, NT threads, U pieces of a thread at a time. A round: at
// most `round` rows, whose places one thread each looks up; the next round's are looked up while this one's rows are on their way.
template <typename V, int NT, int U>
__device__ __forceinline__ void move_rows(const Evict& p, Places& at_s, int b, int h, const int32_t* kept, int c_first, int per_col,
                                          int round, int first, int last) {
  const int tid = threadIdx.x;
  const int32_t *src = p.rows.table + b * p.rows.table_ld, *dst = p.dst_table + b * p.dst_ld;
  auto look_up = [&](int r0, int buf) {
    for (int i = tid; i < round && r0 + i < last; i += NT) {
      const int r = r0 + i, j = kept[r];
      int64_t pf = -1, pt = -1;
      int sf = 0, st = 0;
      const bool stays = p.pools_in_place && j == r;  // it lies where it belongs
      if (stays || !p.rows.locate(src, j, pf, sf) || !p.rows.locate(dst, r, pt, st)) pf = pt = -1;
      at_s.from[buf][i] = make_int2(static_cast<int>(pf), sf);
      at_s.to[buf][i] = make_int2(static_cast<int>(pt), st);  // page -1: nothing is moved
    }
  };
  const int row0 = tid / per_col, c0 = tid % per_col, rows_on = NT / per_col, c_on = NT % per_col;
  look_up(first, 0);
  __syncthreads();
  int buf = 0;
  for (int r0 = first; r0 < last; r0 += round) {
    V x[U], y[U];
    const int n = min(round, last - r0);
    int row = row0, c = c0;
    auto on = [&](int k, int2& place, const int2* places) {  // k-th piece of this thread
      if (k == 0) {
        row = row0;
        c = c0;
      } else {
        row += rows_on;
        c += c_on;
        if (c >= per_col) {
          c -= per_col;
          ++row;
        }
      }
      if (row >= n || c_first + c >= p.pieces) return false;
      place = places[row];
      return place.x >= 0;
    };
    int2 at;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (on(k, at, at_s.from[buf])) {
        x[k] = reinterpret_cast<const V*>(p.pool[0] + p.rows.offset(0, at.x, h, at.y))[c_first + c];
        y[k] = reinterpret_cast<const V*>(p.pool[1] + p.rows.offset(1, at.x, h, at.y))[c_first + c];
      }
    const int next = buf == 2 ? 0 : buf + 1;  // (a thread may still store to the places of the round before)
    if (r0 + round < last) look_up(r0 + round, next);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (on(k, at, at_s.to[buf])) {
        reinterpret_cast<V*>(p.pool[0] + p.rows.offset(0, at.x, h, at.y))[c_first + c] = x[k];
        reinterpret_cast<V*>(p.pool[1] + p.rows.offset(1, at.x, h, at.y))[c_first + c] = y[k];
      }
    buf = next;
  }
}

// The weights of rows [first, last) that stay; in order: a round's are read before any is written.
template <int NT, int U>
__device__ __forceinline__ void move_weights(const Evict& p, int seg, const int32_t* kept, int first, int last) {
  const float* w = p.weights + seg * p.weights_ld;
  float* out = p.weights_out + seg * p.weights_out_ld;
  for (int i0 = first; i0 < last; i0 += NT * U) {
    float x[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + k * NT + static_cast<int>(threadIdx.x);
      if (i < last) x[k] = w[kept[i]];
    }
    if (p.weights_in_place) __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + k * NT + static_cast<int>(threadIdx.x);
      if (i < last) out[i] = x[k];
    }
  }
}

// x: segment and column; y: keys and values, or weights; z: stretch of rows.
template <typename V>
__global__ void __launch_bounds__(kMoveThreads, 2)
move_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  __shared__ Places at_s;
  const int seg = blockIdx.x / p.cols, col = blockIdx.x % p.cols, b = seg / p.Hk, h = seg % p.Hk;
  const bool pools = blockIdx.y == 0, ordered = pools ? p.pools_in_place : p.weights_in_place;
  const int keep = min(p.rows.length(p.lengths, b), p.budget);
  const int32_t* kept = p.kept + static_cast<int64_t>(seg) * p.budget;
  if (ordered && blockIdx.z > 0) return;
  const int first = ordered ? 0 : blockIdx.z * p.chunk, last = ordered ? keep : min(keep, first + p.chunk);
  if (first >= last) return;
  if (pools) move_rows<V, kMoveThreads, kMovePieces>(p, at_s, b, h, kept, col * p.per_col, p.per_col, p.round, first, last);
  else if (col == 0) move_weights<kMoveThreads, kMovePieces>(p, seg, kept, first, last);  // in place as rows of one column are
}

// Both at once, a block per cache.
__global__ void __launch_bounds__(kSelThreads)
evict_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  extern __shared__ __align__(16) uint8_t smem[];
  static_assert(sizeof(Places) <= sizeof(SelectShared), "");
  select<1>(p, *reinterpret_cast<SelectShared*>(smem));
  __syncthreads();  // all positions are there, all weights and all of the shared memory have been read
  constexpr int U = 2;
  const int seg = blockIdx.x, b = seg / p.Hk, keep = min(p.rows.length(p.lengths, b), p.budget);
  const int32_t* kept = p.kept + static_cast<int64_t>(seg) * p.budget;
  if (p.weights_out != nullptr) move_weights<kSelThreads, U>(p, seg, kept, 0, keep);
  move_rows<uint4, kSelThreads, U>(p, *reinterpret_cast<Places*>(smem), b, seg % p.Hk, kept, 0, p.pieces,
                                   min(kSelThreads * U / p.pieces, kMoveRows), 0, keep);
}

void launch_select(const Evict& p, int segs, cudaStream_t st) {
  // blocks that share a cache: as many as leave two for each SM and have 4096 keys each
  unsigned c = 8;
  while (c > 1 && (static_cast<int64_t>(segs) * c > 2 * kNumSMs || p.rows.capacity < static_cast<int64_t>(c) * 4096)) c /= 2;
  const dim3 grid(static_cast<unsigned>(segs) * c);
  constexpr size_t smem = sizeof(SelectShared);
  switch (c) {
    case 8: launch_cluster_k(select_kernel<8>, grid, kSelThreads, 8, smem, st, p); break;
    case 4: launch_cluster_k(select_kernel<4>, grid, kSelThreads, 4, smem, st, p); break;
    case 2: launch_cluster_k(select_kernel<2>, grid, kSelThreads, 2, smem, st, p); break;
    default: launch_k(select_kernel<1>, grid, kSelThreads, smem, st, p);
  }
}

}  // namespace
}  // namespace ptj

using namespace ptj;

extern "C" int ptj_kv_evict(const ptj_kv_cache* cache, const int32_t* dst_table, int64_t dst_width, int64_t dst_ld, int64_t budget,
                            int64_t recent, const float* weights, int64_t weights_ld, float* weights_out, int64_t weights_out_ld,
                            int32_t* kept, int32_t* new_lengths, void* stream) {
  Evict p = {};
  const int rc = make_paged_rows(cache, p.rows);
  if (rc != PTJ_OK) return rc;
  if (!dst_table || !weights || !kept || !new_lengths || budget < 1 || budget > (1 << 30) || recent < 0 || recent > budget ||
      dst_width < 1 || dst_ld < dst_width || new_lengths == cache->lengths || pools_overlap(*cache))
    return PTJ_ERR_BAD_SHAPE;
  const int64_t most = budget < p.rows.capacity ? budget : p.rows.capacity;  // keys that a sequence keeps at most
  if (weights_ld < p.rows.capacity || (weights_out && weights_out_ld < most) || dst_width < ceil_div(most, cache->page_size) ||
      (weights_out == weights && weights_out_ld != weights_ld) ||
      (dst_table == cache->table && cache->batch > 1 && dst_ld != cache->table_ld))
    return PTJ_ERR_BAD_SHAPE;
  if (ptj_device_check() != PTJ_OK || (p.rows.fault = tc::fault_word()) == nullptr) return PTJ_ERR_DEVICE;
  p.dst_table = dst_table;
  p.dst_ld = dst_ld;
  p.pool[0] = static_cast<char*>(cache->k);
  p.pool[1] = static_cast<char*>(cache->v);
  p.lengths = cache->lengths;
  p.kept = kept;
  p.new_lengths = new_lengths;
  p.weights = weights;
  p.weights_out = weights_out;
  p.weights_ld = weights_ld;
  p.weights_out_ld = weights_out_ld;
  p.budget = static_cast<int>(budget);
  p.recent = static_cast<int>(recent);
  p.Hk = static_cast<int>(cache->kv_heads);
  const int64_t es = static_cast<int64_t>(dtype_size(cache->dtype));
  const bool wide = paged_rows_aligned(*cache), in_place = dst_table == cache->table;
  const int64_t piece = wide ? 16 : es;
  p.pieces = static_cast<int>(cache->d_head * es / piece);
  const int segs = static_cast<int>(cache->batch * cache->kv_heads);
  p.pools_in_place = in_place;
  p.weights_in_place = weights_out == weights;
  // In place: columns of 32 bytes. Else whole rows, in stretches of a few rounds.
  p.per_col = in_place ? static_cast<int>(32 / piece) : p.pieces;
  if (p.per_col > p.pieces) p.per_col = p.pieces;
  p.cols = static_cast<int>(ceil_div(p.pieces, p.per_col));
  p.round = kMoveThreads * kMovePieces / p.per_col;
  if (p.round > kMoveRows) p.round = kMoveRows;
  // rounds of a block: so many that all blocks are resident (two per SM) where the rows are that many
  const int64_t rounds = ceil_div(most, p.round), least = ceil_div(rounds, 65535);
  int64_t each = ceil_div(rounds * segs, 2 * kNumSMs);
  each = each < 1 ? 1 : (each > 16 ? 16 : each);
  p.chunk = static_cast<int>((each > least ? each : least) * p.round);
  p.chunks = static_cast<int>(ceil_div(most, p.chunk));
  const bool one = in_place && (weights_out == weights || !weights_out);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Few small caches: one launch. A second one takes the caller's thread 3 us, more than a block needs for 96 KB of keys. 8 x 12 bf16
  // caches of 1024 keys of 64 cut to 512: 17.4 us a call with two launches, 15.3 with one (replayed from a graph 14.7 and 13.3); 4 x 8
  // of 2048 of 128 to 1024: 17 and 30 replayed.
  if (wide && segs <= kNumSMs && p.rows.capacity <= 4096 && most * p.rows.row_bytes <= 96 * 1024) {
    launch_k(evict_kernel, dim3(static_cast<unsigned>(segs)), kSelThreads, sizeof(SelectShared), st, p);
    PTJ_CHECK_LAUNCH();
    return PTJ_OK;
  }
  launch_select(p, segs, st);
  PTJ_CHECK_LAUNCH();
  const dim3 grid(static_cast<unsigned>(segs) * p.cols, weights_out ? 2 : 1, one ? 1 : p.chunks);
  if (wide) launch_k(move_kernel<uint4>, grid, kMoveThreads, 0, st, p);
  else if (es == 2) launch_k(move_kernel<uint16_t>, grid, kMoveThreads, 0, st, p);
  else launch_k(move_kernel<uint32_t>, grid, kMoveThreads, 0, st, p);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
