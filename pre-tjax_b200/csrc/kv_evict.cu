// Eviction from a paged key-value cache by accumulated attention weight.
#include "kv_cache.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

constexpr int kThreads = 1024;

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
  int budget, recent, Hk, pieces;
};

// weights in the order of unsigned integers; a NaN is the lowest, both zeros are equal
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int block_sum_int(int v, int* red) {  // red: 33 ints
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  if (warp == 0) {
    const int t = __reduce_add_sync(0xffffffffu, red[lane]);
    if (lane == 0) red[32] = t;
  }
  __syncthreads();
  return red[32];
}

// A block per sequence and key head. The `want` heaviest of the n candidates are those above a threshold, found bit by bit, and
// the first ones that equal it.
__global__ void __launch_bounds__(kThreads)
select_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  __shared__ int red[33], base[2][33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x / p.Hk;
  const int n = p.rows.length(p.lengths, b), keep = min(n, p.budget);
  if (tid == 0 && blockIdx.x % p.Hk == 0) p.new_lengths[b] = keep;
  const float* w = p.weights + blockIdx.x * p.weights_ld;
  int32_t* kept = p.kept + static_cast<int64_t>(blockIdx.x) * p.budget;
  float* wout = p.weights_out == nullptr ? nullptr : p.weights_out + blockIdx.x * p.weights_out_ld;
  for (int i = keep + tid; i < p.budget; i += kThreads) kept[i] = -1;
  const int cand = n > p.budget ? n - p.recent : 0;  // everything stays in a short sequence
  const int want = n > p.budget ? p.budget - p.recent : 0;
  uint32_t thr = 0;
  int ties = 0;
  if (cand > 0 && want > 0) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = thr | (1u << bit);
      int c = 0;
      for (int j = tid; j < cand; j += kThreads) c += rank_of(w[j]) >= t;
      if (block_sum_int(c, red) >= want) thr = t;
    }
    int above = 0;
    for (int j = tid; j < cand; j += kThreads) above += rank_of(w[j]) > thr;
    ties = want - block_sum_int(above, red);
  }
  int done = 0, tied = 0;  // keys kept and ties met before this round
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + tid;
    const float x = j < n ? w[j] : 0.f;
    const uint32_t r = rank_of(x);
    const bool tie = j < cand && want > 0 && r == thr;
    bool stay = j < n && (j >= cand || (want > 0 && r > thr));
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    __syncthreads();
    if (lane == 0) base[0][warp] = __popc(tie_mask);
    __syncthreads();
    int before = tied, all = 0;
    for (int k = 0; k < kThreads / 32; ++k) {
      if (k < warp) before += base[0][k];
      all += base[0][k];
    }
    tied += all;
    if (tie && before + __popc(tie_mask & ((1u << lane) - 1)) < ties) stay = true;
    const uint32_t mask = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) base[1][warp] = __popc(mask);
    __syncthreads();
    int at = done;
    all = 0;
    for (int k = 0; k < kThreads / 32; ++k) {
      if (k < warp) at += base[1][k];
      all += base[1][k];
    }
    done += all;
    at += __popc(mask & ((1u << lane) - 1));
    if (stay) {
      kept[at] = j;
      if (wout != nullptr) wout[at] = x;  // at <= j: weights that are still to be read lie behind this round's
    }
  }
}

// A block per sequence, key head and pool moves rows in order, a round's rows being read before any of them is written: the row
// that goes to place i lies at place i or behind it.
template <typename V>
__global__ void __launch_bounds__(kThreads)
move_kernel(const __grid_constant__ Evict p) {
  grid_dep_sync();
  const int seg = blockIdx.x >> 1, kv = blockIdx.x & 1, b = seg / p.Hk, h = seg % p.Hk;
  const int keep = min(p.rows.length(p.lengths, b), p.budget);
  const int32_t* kept = p.kept + static_cast<int64_t>(seg) * p.budget;
  const int64_t total = static_cast<int64_t>(keep) * p.pieces;
  for (int64_t i0 = 0; i0 < total; i0 += kThreads) {
    const int64_t i = i0 + threadIdx.x;
    V x = {};
    char* to = nullptr;
    if (i < total) {
      const int r = static_cast<int>(i / p.pieces), c = static_cast<int>(i % p.pieces);
      int64_t page;
      int slot;
      if (p.rows.locate(p.rows.table + b * p.rows.table_ld, kept[r], page, slot)) {
        x = reinterpret_cast<const V*>(p.pool[kv] + p.rows.offset(kv, page, h, slot))[c];
        if (p.rows.locate(p.dst_table + b * p.dst_ld, r, page, slot))
          to = p.pool[kv] + p.rows.offset(kv, page, h, slot) + c * sizeof(V);
      }
    }
    __syncthreads();
    if (to != nullptr) *reinterpret_cast<V*>(to) = x;
    __syncthreads();
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
  const bool wide = paged_rows_aligned(*cache);
  p.pieces = static_cast<int>(wide ? cache->d_head * es / 16 : cache->d_head);
  const int segs = static_cast<int>(cache->batch * cache->kv_heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  launch_k(select_kernel, segs, kThreads, 0, st, p);
  PTJ_CHECK_LAUNCH();
  if (wide) launch_k(move_kernel<uint4>, 2 * segs, kThreads, 0, st, p);
  else if (es == 2) launch_k(move_kernel<uint16_t>, 2 * segs, kThreads, 0, st, p);
  else launch_k(move_kernel<uint32_t>, 2 * segs, kThreads, 0, st, p);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
