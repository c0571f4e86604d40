// Eviction from a paged key-value cache by accumulated attention weight.
//
// Two launches: one finds the keys that stay, one moves their rows.
//
// Which stay: the weights are ordered as unsigned integers; the weight of the last key to stay is found digit by digit (11, 11
// and 10 bits) from histograms in shared memory. Above it all stay, of its equals the first ones. A cluster of C blocks shares
// a cache, its histograms and counts meet through distributed shared memory. Bound by the chain of barriers and by the histogram
// updates of one SM; the weights themselves are read four times, from L2 after the first.
//
// Moving: memory bounds it. Into other pages, blocks take stretches of rows and everything is independent. In place, the row that
// goes to place i lies at place i or behind it, so one block moves a column of 32 bytes of all rows in order, reading a round's
// rows before it writes any: columns are independent of each other, and the next round's rows lie behind all places written.
#include "cluster.cuh"
#include "kv_cache.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

constexpr int kSelThreads = 1024, kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;

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
  int chunk, chunks; // rows of a stretch, stretches
  int ordered[3];    // keys, values, weights: moved in place
};

// weights in the order of unsigned integers; a NaN is the lowest, both zeros are equal
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SelectShared {
  uint32_t hist[3][kBins];
  uint32_t warp_sum[kSelWarps];
  uint32_t bin, above;                  // the digit that was found, elements with a larger one
  uint32_t stay[kSelWarps], tie[kSelWarps];
  uint32_t block_stay, block_tie;
};

// The largest digit such that at least `want` elements have it or a larger one, and the number with a larger one.
template <int C>
__device__ __forceinline__ void find_digit(SelectShared& sm, const uint32_t* hist, uint32_t want) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // thread t: digits from the top, two each
  uint32_t n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    n[i] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) n[i] += peer_u32<C>(hist + (kBins - 1 - (2 * tid + i)), r);
  }
  uint32_t incl = n[0] + n[1];
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, x);
    if (lane >= x) incl += y;
  }
  if (lane == 31) sm.warp_sum[warp] = incl;
  __syncthreads();
  const uint32_t others = lane < warp ? sm.warp_sum[lane] : 0u;
  uint32_t before = __reduce_add_sync(0xffffffffu, others) + incl - n[0] - n[1];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (before < want && before + n[i] >= want) {
      sm.bin = kBins - 1 - (2 * tid + i);
      sm.above = before;
    }
    before += n[i];
  }
  __syncthreads();
}

template <int C>
__global__ void __launch_bounds__(kSelThreads)
select_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  __shared__ SelectShared sm;
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
  for (int i = tid; i < 3 * kBins; i += kSelThreads) (&sm.hist[0][0])[i] = 0u;
  __syncthreads();
  uint32_t thr = 0;  // (want 0: nothing but the recent ones stays)
  int ties = 0;
  if (want > 0) {
    uint32_t left = want;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const uint32_t mask = pass == 2 ? 1023u : 2047u, known = pass == 0 ? 0u : (pass == 1 ? ~0u << 21 : ~0u << 10);
#pragma unroll 4
      for (int j = j0 + lane; j < c1; j += 32) {
        const uint32_t r = rank_of(w[j]);
        if ((r & known) == thr) atomicAdd(&sm.hist[pass][(r >> shift) & mask], 1u);
      }
      cluster_barrier<C>();
      find_digit<C>(sm, sm.hist[pass], left);
      thr |= sm.bin << shift;
      left -= sm.above;
    }
    ties = static_cast<int>(left);  // equals of the threshold that stay
  }
  // numbers of keys above the threshold (or recent) and of equals before each warp's stretch
  int stay = 0, tie = 0;
#pragma unroll 4
  for (int j = j0 + lane; j < j1; j += 32) {
    const uint32_t r = rank_of(w[j]);
    stay += j >= cand || (want > 0 && r > thr);
    tie += j < cand && want > 0 && r == thr;
  }
  stay = __reduce_add_sync(0xffffffffu, stay);
  tie = __reduce_add_sync(0xffffffffu, tie);
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
    const uint32_t r = j < j1 ? rank_of(w[j]) : 0u;
    const bool equal = j < c1 && want > 0 && r == thr;
    const bool above = j < j1 && (j >= cand || (want > 0 && r > thr));
    const unsigned em = __ballot_sync(0xffffffffu, equal), am = __ballot_sync(0xffffffffu, above), low = (1u << lane) - 1u;
    const int e = tied + __popc(em & low), a = stays + __popc(am & low);
    if (above || (equal && e < ties)) kept[a + min(e, ties)] = j;
    tied += __popc(em);
    stays += __popc(am);
  }
}

// x: segment and column (columns of a row side by side); y: keys, values, weights; z: stretch of rows
template <typename V, int U>
__global__ void __launch_bounds__(kMoveThreads)
move_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  const int kv = blockIdx.y, tid = threadIdx.x;
  const int seg = blockIdx.x / p.cols, col = blockIdx.x % p.cols, b = seg / p.Hk, h = seg % p.Hk;
  const int keep = min(p.rows.length(p.lengths, b), p.budget);
  const int32_t* kept = p.kept + static_cast<int64_t>(seg) * p.budget;
  if (p.ordered[kv] && blockIdx.z > 0) return;
  const int first = p.ordered[kv] ? 0 : blockIdx.z * p.chunk, last = p.ordered[kv] ? keep : min(keep, first + p.chunk);
  if (first >= last) return;
  if (kv == 2) {  // weights: in place they are moved as rows of one column are
    if (col != 0) return;
    const float* w = p.weights + seg * p.weights_ld;
    float* out = p.weights_out + seg * p.weights_out_ld;
    for (int i0 = first; i0 < last; i0 += kMoveThreads * U) {
      float x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * kMoveThreads + tid;
        if (i < last) x[k] = w[kept[i]];
      }
      if (p.ordered[2]) __syncthreads();
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * kMoveThreads + tid;
        if (i < last) out[i] = x[k];
      }
    }
    return;
  }
  const int32_t *from = p.rows.table + b * p.rows.table_ld, *to = p.dst_table + b * p.dst_ld;
  const int row = tid / p.per_col, c = col * p.per_col + tid % p.per_col;  // a thread's row in a round, its piece
  const int step = kMoveThreads / p.per_col;                              // rows of a round
  const bool in = row < step && c < p.pieces;
  for (int r0 = first; r0 < last; r0 += step * U) {
    V x[U];
    V* dst[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int r = r0 + k * step + row;
      dst[k] = nullptr;
      if (!in || r >= last) continue;
      const int j = kept[r];
      if (p.ordered[kv] && j == r) continue;  // it lies where it belongs
      int64_t page;
      int slot;
      if (!p.rows.locate(from, j, page, slot)) continue;
      x[k] = reinterpret_cast<const V*>(p.pool[kv] + p.rows.offset(kv, page, h, slot))[c];
      if (p.rows.locate(to, r, page, slot)) dst[k] = reinterpret_cast<V*>(p.pool[kv] + p.rows.offset(kv, page, h, slot)) + c;
    }
    if (p.ordered[kv]) __syncthreads();
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (dst[k] != nullptr) *dst[k] = x[k];
  }
}

void launch_select(const Evict& p, int segs, cudaStream_t st) {
  // blocks that share a cache: as many as leave two for each SM and have 4096 keys each
  unsigned c = 8;
  while (c > 1 && (static_cast<int64_t>(segs) * c > 2 * kNumSMs || p.rows.capacity < static_cast<int64_t>(c) * 4096)) c /= 2;
  const dim3 grid(static_cast<unsigned>(segs) * c);
  switch (c) {
    case 8: launch_cluster_k(select_kernel<8>, grid, kSelThreads, 8, st, p); break;
    case 4: launch_cluster_k(select_kernel<4>, grid, kSelThreads, 4, st, p); break;
    case 2: launch_cluster_k(select_kernel<2>, grid, kSelThreads, 2, st, p); break;
    default: launch_k(select_kernel<1>, grid, kSelThreads, 0, st, p);
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
      dst_width < 1 || dst_ld < dst_width || new_lengths == cache->lengths)
    return PTJ_ERR_BAD_SHAPE;
  const int64_t most = budget < p.rows.capacity ? budget : p.rows.capacity;  // keys that a sequence keeps at most
  if (weights_ld < p.rows.capacity || (weights_out && weights_out_ld < most) || dst_width < ceil_div(most, cache->page_size) ||
      (weights_out == weights && weights_out_ld != weights_ld))
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
  p.ordered[0] = p.ordered[1] = in_place;
  p.ordered[2] = weights_out == weights;
  constexpr int U = 8;
  // In place: columns of 32 bytes. Else whole rows (a block holds at most 256 pieces), in stretches of a few rounds.
  p.per_col = in_place ? static_cast<int>(32 / piece) : p.pieces;
  if (p.per_col > p.pieces) p.per_col = p.pieces;
  p.cols = static_cast<int>(ceil_div(p.pieces, p.per_col));
  p.chunk = kMoveThreads / p.per_col * U;
  p.chunks = static_cast<int>(ceil_div(most, p.chunk));
  const bool one = in_place && (weights_out == weights || !weights_out);
  if (p.chunks > 65535) {
    p.chunk = static_cast<int>(ceil_div(most, 65535));
    p.chunks = static_cast<int>(ceil_div(most, p.chunk));
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  launch_select(p, segs, st);
  PTJ_CHECK_LAUNCH();
  const dim3 grid(static_cast<unsigned>(segs) * p.cols, weights_out ? 3 : 2, one ? 1 : p.chunks);
  if (wide) launch_k(move_kernel<uint4, U>, grid, kMoveThreads, 0, st, p);
  else if (es == 2) launch_k(move_kernel<uint16_t, U>, grid, kMoveThreads, 0, st, p);
  else launch_k(move_kernel<uint32_t, U>, grid, kMoveThreads, 0, st, p);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
