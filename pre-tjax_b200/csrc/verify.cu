// Verification of drafted tokens against the target's probabilities, with random numbers that are inputs.
//
// Accepting draft x with probability min(1, p(x) / q(x)) and replacing the first rejected one by a token drawn from
// max(p - q, 0) leaves the target's distribution p unchanged: q(x) min(1, p/q) + (sum of rejections) max(p - q, 0) / total = p(x).
//
// Of all the probabilities only one row per sequence (two with a draft's distribution) is read whole: the one the next token is
// drawn from. A cluster of C blocks shares it, every warp takes a contiguous chunk and keeps the sums of up to 32 groups of it. The
// blocks' sums meet through distributed shared memory; the group in which the running sum passes the mark is found from sums, and
// only its elements (256 of a vocabulary below 500 000) are read again. Bound by the chain of dependent loads, not by bytes: the
// drafts, their probabilities, the row in four or five batches, the group. Sums are float64, products of two float32 in float64 are
// exact: decisions then agree with a sum in any other order except for marks within 1e-13 or so of a border.
#include "cluster.cuh"

namespace ptj {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kGroups = 32, kBatch = 8, kGroup = 32 * kBatch;

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
  // this lane's elements of the kGroup from g on
  template <bool SUB>
  __device__ __forceinline__ void load(int g, int j1, float (&x)[kBatch], float (&y)[kBatch]) const {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int j = g + 32 * i + (threadIdx.x & 31);
      x[i] = j < j1 && (SUB || j != skip) ? Elem<E>::load(row + j) : 0.f;
      y[i] = SUB && j < j1 ? Elem<E>::load(sub + j) : 0.f;
    }
  }
  // sums of the groups of [j0, j1), `size` elements each (a multiple of kGroup); a batch of loads is ahead of the arithmetic
  template <bool SUB>
  __device__ __forceinline__ void sums(int j0, int j1, int size, double* out) const {
    float x[2][kBatch], y[2][kBatch];
    load<SUB>(j0, j1, x[0], y[0]);
    double s = 0.0;
    int group = 0, end = j0 + size;
    auto add = [&](int k, int g) {
      double a[2] = {0.0, 0.0};
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const double w = SUB ? static_cast<double>(x[k][i]) - static_cast<double>(y[k][i]) : static_cast<double>(x[k][i]);
        a[i & 1] += w > 0.0 ? w : 0.0;
      }
      s += a[0] + a[1];
      if (g + kGroup >= end || g + kGroup >= j1) {
        s = warp_sum_f64(s);
        if ((threadIdx.x & 31) == 0) out[group] = s;
        ++group;
        end += size;
        s = 0.0;
      }
    };
    for (int g = j0; g < j1; g += 2 * kGroup) {
      load<SUB>(g + kGroup, j1, x[1], y[1]);
      add(0, g);
      if (g + kGroup >= j1) break;
      load<SUB>(g + 2 * kGroup, j1, x[0], y[0]);
      add(1, g + kGroup);
    }
  }
};

template <typename E, int C>
__global__ void __launch_bounds__(kThreads, 4)
verify_kernel(const __grid_constant__ Verify p) {
  grid_dep_sync();
  __shared__ double group_s[kWarps][kGroups], chunk_s[kWarps], total_s;
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
  // contiguous chunks, one per warp of the cluster, of at most kGroups groups
  const int groups_all = (p.V + kGroup - 1) / kGroup;  // of kGroup elements
  const int per_groups = (groups_all + C * kWarps - 1) / (C * kWarps), size = (per_groups + kGroups - 1) / kGroups * kGroup;
  const int per = per_groups * kGroup;
  const int j0 = static_cast<int>(min(static_cast<int64_t>(rank * kWarps + warp) * per, static_cast<int64_t>(p.V)));
  const int j1 = static_cast<int>(min(static_cast<int64_t>(j0) + per, static_cast<int64_t>(p.V))), groups = (j1 - j0 + size - 1) / size;
  if (weight.sub != nullptr) weight.template sums<true>(j0, j1, size, group_s[warp]);
  else weight.template sums<false>(j0, j1, size, group_s[warp]);
  __syncwarp();
  const double s = warp_sum_f64(lane < groups ? group_s[warp][lane] : 0.0);
  if (lane == 0) chunk_s[warp] = s;
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
#pragma unroll
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
    int k = 0;
    for (; k < groups - 1 && !(at + group_s[w][k] > mark); ++k) at += group_s[w][k];
    while (k > 0 && !(group_s[w][k] > 0.0)) at -= group_s[w][--k];
    int pick = -1, last = -1;  // last: the last element with weight so far
    const int g1 = min(j0 + (k + 1) * size, j1);
    for (int g = j0 + k * size; g < g1 && pick < 0; g += kGroup) {
      double x[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int j = g + i * 32 + lane;
        x[i] = j < g1 ? weight(j) : 0.0;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const unsigned some = __ballot_sync(0xffffffffu, x[i] > 0.0);
        if (pick >= 0 || some == 0u) continue;
        last = g + i * 32 + 31 - __clz(some);
        double c = x[i];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, c, d);
          if (lane >= d) c += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, at + c > mark && x[i] > 0.0);
        if (over != 0u) pick = g + i * 32 + __ffs(over) - 1;
        at += __shfl_sync(0xffffffffu, c, 31);
      }
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
  // as many blocks per sequence as are resident at once (four per SM), each with a slice worth a round of its warps
  unsigned c = 8;
  while (c > 1 && (batch * c > 4 * kNumSMs || p.V < static_cast<int64_t>(c) * kWarps * kGroup)) c /= 2;
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
