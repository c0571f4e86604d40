// Verification of drafted tokens against the target's probabilities, with random numbers that are inputs.
//
// Accepting draft x with probability min(1, p(x) / q(x)) and replacing the first rejected one by a token drawn from
// max(p - q, 0) leaves the target's distribution p unchanged: q(x) min(1, p/q) + (sum of rejections) max(p - q, 0) / total = p(x).
//
// Of all the probabilities only one row per sequence (two with a draft's distribution) is read whole: the one the next token is
// drawn from. A cluster of C blocks shares it. Each block sums its slice, the sums meet through distributed shared memory, and
// the block in whose slice the running sum passes the mark looks for the place: a warp's chunk, 256 elements of it, 32, one.
// Sums are float64, products of two float32 in float64 are exact: decisions then agree with a sum in any other order except for
// marks within 1e-13 or so of a border.
#include "cluster.cuh"

namespace ptj {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct Verify {
  const void *target, *draft;
  int64_t ts[2], ds[2];
  const int32_t *tokens, *counts;
  const float* uniforms;
  int32_t *out, *accepted;
  int K, V;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
  return v;
}

// What the next token is drawn from.
template <typename E>
struct Weights {
  const E *row, *sub;  // sub: NULL, or what is taken off
  int skip;            // an element without weight, -1: none
  __device__ __forceinline__ double operator()(int j) const {
    double w = Elem<E>::load(row + j);
    if (sub != nullptr) w -= static_cast<double>(Elem<E>::load(sub + j));
    return w > 0.0 && j != skip ? w : 0.0;  // (a NaN has none)
  }
  // of every 32nd element from j0 + lane on; a batch of loads is under way at a time, the last one too
  template <bool SUB>
  __device__ __forceinline__ double sum(int j0, int j1, int lane) const {
    constexpr int U = 8;
    double s[2] = {0.0, 0.0};
    for (int g = j0 + lane; g < j1; g += 32 * U) {
      float x[U], y[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int j = g + 32 * i;
        x[i] = j < j1 && (SUB || j != skip) ? Elem<E>::load(row + j) : 0.f;
        y[i] = SUB && j < j1 ? Elem<E>::load(sub + j) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const double w = SUB ? static_cast<double>(x[i]) - static_cast<double>(y[i]) : static_cast<double>(x[i]);
        s[i & 1] += w > 0.0 ? w : 0.0;
      }
    }
    return s[0] + s[1];
  }
};

template <typename E, int C>
__global__ void __launch_bounds__(kThreads)
verify_kernel(const __grid_constant__ Verify p) {
  grid_dep_sync();
  __shared__ double chunk_s[kWarps], total_s;
  __shared__ int n_s;
  __shared__ float best_s[kWarps];
  __shared__ int arg_s[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_rank<C>());
  const int64_t b = blockIdx.x / C;
  const E* target = static_cast<const E*>(p.target) + b * p.ts[0];
  const E* draft = p.draft == nullptr ? nullptr : static_cast<const E*>(p.draft) + b * p.ds[0];
  const int32_t* tokens = p.tokens + b * p.K;
  const float* u = p.uniforms + b * (p.K + 1);
  const int count = p.counts == nullptr ? p.K : min(max(p.counts[b], 0), p.K);
  if (warp == 0) {  // every block finds the first rejected draft for itself
    int n = count;
    for (int i0 = 0; i0 < count; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true;
      if (i < count) {
        const int x = tokens[i];
        ok = x >= 0 && x < p.V;
        if (ok) {
          const double px = Elem<E>::load(target + i * p.ts[1] + x);
          const double qx = draft == nullptr ? 1.0 : static_cast<double>(Elem<E>::load(draft + i * p.ds[1] + x));
          ok = static_cast<double>(u[i]) * qx < px;
        }
      }
      const unsigned no = __ballot_sync(0xffffffffu, !ok);
      if (no != 0u) {
        n = i0 + __ffs(no) - 1;
        break;
      }
    }
    if (lane == 0) n_s = n;
  }
  __syncthreads();
  const int n = n_s;
  const bool rejected = n < count;
  Weights<E> weight{target + n * p.ts[1], rejected && draft != nullptr ? draft + n * p.ds[1] : nullptr,
                    rejected && draft == nullptr ? tokens[n] : -1};
  // contiguous chunks, one per warp of the cluster
  const int per = (p.V + C * kWarps * 32 - 1) / (C * kWarps * 32) * 32;
  const int j0 = min((rank * kWarps + warp) * per, p.V), j1 = min(j0 + per, p.V);
  const double s = warp_sum_f64(weight.sub != nullptr ? weight.template sum<true>(j0, j1, lane) : weight.template sum<false>(j0, j1, lane));
  if (lane == 0) chunk_s[warp] = s;
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < kWarps; ++w) t += chunk_s[w];
    total_s = t;
  }
  cluster_barrier<C>();
  double before = 0.0, total = 0.0;
#pragma unroll
  for (int r = 0; r < C; ++r) {
    const double t = peer_f64<C>(&total_s, r);
    if (r < rank) before += t;
    total += t;
  }
  cluster_barrier<C>();  // the sums are read: a block may leave
  int32_t* out = p.out + b * (p.K + 1);
  if (rank == 0) {
    for (int i = tid; i <= p.K; i += kThreads)
      if (i != n) out[i] = i < n ? tokens[i] : 0;
    if (tid == 0) p.accepted[b] = n;
  }
  if (total > 0.0) {
    const float last_u = u[p.K];
    double mark = static_cast<double>(last_u < 1.f ? last_u : 1.f - 5.9604645e-8f) * total;
    if (!(mark >= 0.0)) mark = 0.0;  // (no number, or below 0)
    // the first slice, and in it the first chunk, at whose end the running sum passes the mark
    double end = before + total_s;
    bool mine = before <= mark || rank == 0;
    if (rank < C - 1) mine = mine && end > mark;
    if (!mine) return;
    int w = 0;
    double at = before;
    for (; w < kWarps - 1 && !(at + chunk_s[w] > mark); ++w) at += chunk_s[w];
    // (a mark that rounding puts behind all sums belongs to the last chunk that has any weight)
    while (w > 0 && !(chunk_s[w] > 0.0)) at -= chunk_s[--w];
    if (warp != w) return;
    int pick = -1, last = -1;  // last: the last element with weight so far
    for (int g = j0; g < j1; g += 256) {
      double x[8], sum = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = g + i * 32 + lane;
        x[i] = j < j1 ? weight(j) : 0.0;
        sum += x[i];
      }
      sum = warp_sum_f64(sum);
      const bool here = at + sum > mark;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned some = __ballot_sync(0xffffffffu, x[i] > 0.0);
        if (some != 0u && pick < 0) last = g + i * 32 + 31 - __clz(some);
        if (here && pick < 0) {
          double c = x[i];
#pragma unroll
          for (int k = 1; k < 32; k <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, c, k);
            if (lane >= k) c += y;
          }
          const unsigned over = __ballot_sync(0xffffffffu, at + c > mark && x[i] > 0.0);
          if (over != 0u) pick = g + i * 32 + __ffs(over) - 1;
          at += __shfl_sync(0xffffffffu, c, 31);
        }
      }
      if (pick >= 0 || here) break;
      at += sum;
    }
    if (lane == 0) out[n] = pick >= 0 ? pick : max(last, 0);
    return;
  }
  // nothing to draw from: the largest probability, the first among equals
  if (rank != 0) return;
  float best = -INFINITY;
  int arg = 0x7fffffff;
  auto better = [&](float v, int a) {
    if (v > best || (v == best && a < arg)) {
      best = v;
      arg = a;
    }
  };
  for (int j = tid; j < p.V; j += kThreads) better(Elem<E>::load(weight.row + j), j);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, x);
    better(v, __shfl_xor_sync(0xffffffffu, arg, x));
  }
  if (lane == 0) {
    best_s[warp] = best;
    arg_s[warp] = arg;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) better(best_s[w], arg_s[w]);
    out[n] = arg < p.V ? arg : 0;
  }
}

template <typename E>
void launch_verify(const Verify& p, int64_t batch, cudaStream_t st) {
  // as many blocks per sequence as leave four for each SM, each with a slice worth a few rounds of its threads
  unsigned c = 8;
  while (c > 1 && (batch * c > 4 * kNumSMs || p.V < static_cast<int64_t>(c) * kThreads * 2)) c /= 2;
  const dim3 grid(static_cast<unsigned>(batch) * c);
  switch (c) {
    case 8: launch_cluster_k(verify_kernel<E, 8>, grid, kThreads, 8, 0, st, p); break;
    case 4: launch_cluster_k(verify_kernel<E, 4>, grid, kThreads, 4, 0, st, p); break;
    case 2: launch_cluster_k(verify_kernel<E, 2>, grid, kThreads, 2, 0, st, p); break;
    default: launch_k(verify_kernel<E, 1>, grid, kThreads, 0, st, p);
  }
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
  if (dtype == PTJ_BF16) launch_verify<__nv_bfloat16>(p, batch, st);
  else launch_verify<float>(p, batch, st);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
