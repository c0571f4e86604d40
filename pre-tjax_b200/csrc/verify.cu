// Verification of drafted tokens against the target's probabilities, with random numbers that are inputs.
//
// Accepting draft x with probability min(1, p(x) / q(x)) and replacing the first rejected one by a token drawn from
// max(p - q, 0) leaves the target's distribution p unchanged: q(x) min(1, p/q) + (sum of rejections) max(p - q, 0) / total = p(x).
#include "common.cuh"

namespace ptj {
namespace {

constexpr int kThreads = 1024;

struct Verify {
  const void *target, *draft;
  int64_t ts[2], ds[2];
  const int32_t *tokens, *counts;
  const float* uniforms;
  int32_t *out, *accepted;
  int K, V;
};

template <typename E>
__global__ void __launch_bounds__(kThreads)
verify_kernel(const __grid_constant__ Verify p) {
  grid_dep_sync();
  __shared__ double sums[kThreads];
  __shared__ int n_s, pick_s;
  __shared__ float best_s[32];
  __shared__ int arg_s[32];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  const E* target = static_cast<const E*>(p.target) + b * p.ts[0];
  const E* draft = p.draft == nullptr ? nullptr : static_cast<const E*>(p.draft) + b * p.ds[0];
  const int32_t* tokens = p.tokens + b * p.K;
  const float* u = p.uniforms + b * (p.K + 1);
  int count = p.counts == nullptr ? p.K : min(max(p.counts[b], 0), p.K);
  if (tid == 0) {
    int n = 0;
    for (; n < count; ++n) {
      const int x = tokens[n];
      if (x < 0 || x >= p.V) break;
      const double px = Elem<E>::load(target + n * p.ts[1] + x);
      const double qx = draft == nullptr ? 1.0 : static_cast<double>(Elem<E>::load(draft + n * p.ds[1] + x));
      if (!(static_cast<double>(u[n]) * qx < px)) break;
    }
    n_s = n;
    pick_s = 0x7fffffff;
  }
  __syncthreads();
  const int n = n_s;
  const E* row = target + n * p.ts[1];
  const E* sub = n < count && draft != nullptr ? draft + n * p.ds[1] : nullptr;
  const int skip = n < count && draft == nullptr ? tokens[n] : -1;
  auto weight = [&](int j) -> double {
    double w = Elem<E>::load(row + j);
    if (sub != nullptr) w -= static_cast<double>(Elem<E>::load(sub + j));
    return w > 0.0 && j != skip ? w : 0.0;
  };
  const int per = (p.V + kThreads - 1) / kThreads, j0 = min(tid * per, p.V), j1 = min(j0 + per, p.V);
  double s = 0.0;
  for (int j = j0; j < j1; ++j) s += weight(j);
  sums[tid] = s;
  __syncthreads();
  double before = 0.0, total = 0.0;
  for (int i = 0; i < kThreads; ++i) {
    if (i == tid) before = total;
    total += sums[i];
  }
  const double want = static_cast<double>(u[p.K]) * total;
  if (before + s > want) {
    double c = before;
    for (int j = j0; j < j1; ++j) {
      c += weight(j);
      if (c > want) {
        atomicMin(&pick_s, j);
        break;
      }
    }
  }
  // nothing to draw from: the largest probability
  float best = -INFINITY;
  int arg = 0;
  if (!(total > 0.0)) {
    arg = 0x7fffffff;
    for (int j = tid; j < p.V; j += kThreads) {
      const float x = Elem<E>::load(row + j);
      if (x > best) { best = x; arg = j; }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const float v = __shfl_xor_sync(0xffffffffu, best, o);
      const int a = __shfl_xor_sync(0xffffffffu, arg, o);
      if (v > best || (v == best && a < arg)) { best = v; arg = a; }
    }
    if ((tid & 31) == 0) { best_s[tid >> 5] = best; arg_s[tid >> 5] = arg; }
  }
  __syncthreads();
  int32_t* out = p.out + b * (p.K + 1);
  if (tid == 0) {
    int pick = pick_s;
    if (!(total > 0.0)) {
      best = -INFINITY;
      pick = 0x7fffffff;
      for (int i = 0; i < 32; ++i)
        if (best_s[i] > best || (best_s[i] == best && arg_s[i] < pick)) { best = best_s[i]; pick = arg_s[i]; }
    }
    out[n] = pick < p.V ? pick : 0;
    p.accepted[b] = n;
  }
  for (int i = tid; i <= p.K; i += kThreads)
    if (i != n) out[i] = i < n ? tokens[i] : 0;
}

}  // namespace
}  // namespace ptj

using namespace ptj;

extern "C" int ptj_verify_drafts(const void* target, const int64_t target_strides[2], const void* draft,
                                 const int64_t draft_strides[2], const int32_t* tokens, const int32_t* counts,
                                 const float* uniforms, int32_t* out, int32_t* accepted, int64_t batch, int64_t drafts,
                                 int64_t vocab, int dtype, void* stream) {
  if (!target || !target_strides || (draft && !draft_strides) || !uniforms || !out || !accepted || batch < 1 || drafts < 0 ||
      vocab < 1 || batch > (1 << 24) || drafts > 4096 || vocab > (1 << 30) || (drafts > 0 && !tokens))
    return PTJ_ERR_BAD_SHAPE;
  if (dtype != PTJ_F32 && dtype != PTJ_BF16) return PTJ_ERR_DTYPE;
  for (int i = 0; i < 2; ++i)
    if (target_strides[i] < 0 || (draft && draft_strides[i] < 0)) return PTJ_ERR_BAD_SHAPE;
  if (ptj_device_check() != PTJ_OK) return PTJ_ERR_DEVICE;
  Verify p = {};
  p.target = target;
  p.draft = draft;
  for (int i = 0; i < 2; ++i) {
    p.ts[i] = target_strides[i];
    if (draft) p.ds[i] = draft_strides[i];
  }
  p.tokens = tokens;
  p.counts = counts;
  p.uniforms = uniforms;
  p.out = out;
  p.accepted = accepted;
  p.K = static_cast<int>(drafts);
  p.V = static_cast<int>(vocab);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = static_cast<int>(batch);
  if (dtype == PTJ_BF16) launch_k(verify_kernel<__nv_bfloat16>, grid, kThreads, 0, st, p);
  else launch_k(verify_kernel<float>, grid, kThreads, 0, st, p);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
