// Attention of new tokens over a paged key-value cache.
#include "kv_cache.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

constexpr int kThreads = 256;

struct DecodeAttn {
  PagedRows rows;
  const int32_t *lengths, *counts;
  const char *q, *k, *v;  // pools
  char* out;
  int64_t qs[3], os[3];   // bytes
  const float* weights;
  float* weights_out;
  int64_t weights_ld;
  float scale, keep;
  int Hk, G, T, D;
};

// A block per sequence and key head takes its rows one after the other: maximum and sum of the scores, then the products.
template <typename E>
__global__ void __launch_bounds__(kThreads)
attn_decode_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  __shared__ float qs[kMaxHeadDim], ps[kThreads], red[33];
  __shared__ int64_t voff[kThreads];
  const int tid = threadIdx.x, b = blockIdx.x / p.Hk, h = blockIdx.x % p.Hk;
  const int n = p.rows.length(p.lengths, b), count = p.rows.count(p.counts, p.T, b), first = n - count;
  const int32_t* row = p.rows.table + b * p.rows.table_ld;
  float* w = p.weights_out == nullptr ? nullptr : p.weights_out + blockIdx.x * p.weights_ld;
  if (w != nullptr)
    for (int j = tid; j < n; j += kThreads)
      w[j] = j < first && p.weights != nullptr ? p.weights[blockIdx.x * p.weights_ld + j] : 0.f;
  for (int r = 0; r < p.G * p.T; ++r) {
    const int t = r % p.T, head = h * p.G + r / p.T;
    const int end = t < count ? first + t + 1 : 0;  // keys of this row
    const char* q = p.q + b * p.qs[0] + head * p.qs[1] + t * p.qs[2];
    __syncthreads();
    for (int d = tid; d < p.D; d += kThreads) qs[d] = Elem<E>::load(reinterpret_cast<const E*>(q) + d);
    __syncthreads();
    auto score = [&](int j, int64_t& v_off) {
      int64_t page;
      int slot;
      if (!p.rows.locate(row, j, page, slot)) {
        v_off = -1;
        return -INFINITY;
      }
      v_off = p.rows.offset(1, page, h, slot);
      const E* k = reinterpret_cast<const E*>(p.k + p.rows.offset(0, page, h, slot));
      float s = 0.f;
      for (int d = 0; d < p.D; ++d) s = fmaf(qs[d], Elem<E>::load(k + d), s);
      return s * p.scale;
    };
    float m = -INFINITY;
    int64_t off;
    for (int j = tid; j < end; j += kThreads) {
      const float s = score(j, off);
      if (!(s <= m)) m = s;  // (a NaN stays)
    }
    const bool nan = __syncthreads_or(m != m);
    m = block_max(m, red);
    if (m == -INFINITY) m = 0.f;
    if (nan) m = NAN;
    float sum = 0.f;
    for (int j = tid; j < end; j += kThreads) sum += expf(score(j, off) - m);
    sum = block_sum(sum, red);
    const float inv = end > 0 ? 1.f / sum : 0.f;
    float o = 0.f;
    for (int j0 = 0; j0 < end; j0 += kThreads) {
      const int j = j0 + tid;
      __syncthreads();
      ps[tid] = 0.f;
      voff[tid] = -1;
      if (j < end) {
        ps[tid] = expf(score(j, voff[tid]) - m) * inv;
        if (w != nullptr) w[j] += ps[tid];
      }
      __syncthreads();
      if (tid < p.D)
        for (int i = 0; i < min(kThreads, end - j0); ++i)
          if (voff[i] >= 0) o = fmaf(ps[i], Elem<E>::load(reinterpret_cast<const E*>(p.v + voff[i]) + tid), o);
    }
    if (tid < p.D)
      Elem<E>::store(reinterpret_cast<E*>(p.out + b * p.os[0] + head * p.os[1] + t * p.os[2]) + tid, o * p.keep);
  }
}

}  // namespace
}  // namespace ptj

using namespace ptj;

extern "C" size_t ptj_attn_decode_workspace_bytes(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, int with_weights) {
  (void)cache; (void)tokens; (void)with_weights;
  return 0;
}

extern "C" int ptj_attn_decode(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, float p, const float* weights,
                               float* weights_out, int64_t weights_ld, void* workspace, size_t workspace_bytes, void* stream) {
  DecodeAttn d = {};
  int rc = make_paged_rows(cache, d.rows);
  if (rc == PTJ_OK) rc = check_new_tokens(*cache, tokens, true, false);
  if (rc != PTJ_OK) return rc;
  if (!(p >= 0.f && p <= 1.f) || (weights && !weights_out) || (weights_out && weights_ld < d.rows.capacity)) return PTJ_ERR_BAD_SHAPE;
  if (ptj_device_check() != PTJ_OK || (d.rows.fault = tc::fault_word()) == nullptr) return PTJ_ERR_DEVICE;
  if (tokens->k) {
    rc = ptj_kv_append(cache, tokens, stream);
    if (rc != PTJ_OK) return rc;
  }
  const int64_t es = static_cast<int64_t>(dtype_size(cache->dtype));
  d.lengths = cache->lengths;
  d.counts = tokens->counts;
  d.q = static_cast<const char*>(tokens->q);
  d.k = static_cast<const char*>(cache->k);
  d.v = static_cast<const char*>(cache->v);
  d.out = static_cast<char*>(tokens->out);
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = tokens->q_strides[i] * es;
    d.os[i] = tokens->o_strides[i] * es;
  }
  d.weights = weights;
  d.weights_out = weights_out;
  d.weights_ld = weights_ld;
  d.scale = 1.f / sqrtf(static_cast<float>(cache->d_head));
  d.keep = 1.f - p;
  d.Hk = static_cast<int>(cache->kv_heads);
  d.G = static_cast<int>(tokens->heads / cache->kv_heads);
  d.T = static_cast<int>(tokens->tokens);
  d.D = static_cast<int>(cache->d_head);
  const int grid = static_cast<int>(cache->batch * cache->kv_heads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dtype == PTJ_BF16) launch_k(attn_decode_kernel<__nv_bfloat16>, grid, kThreads, 0, st, d);
  else launch_k(attn_decode_kernel<float>, grid, kThreads, 0, st, d);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
