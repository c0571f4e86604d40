// Attention of new tokens over a paged cache on CUDA cores, float32 arithmetic: float32 caches and bf16 heads beyond 128.
//
// LPK lanes share a key, 16 bytes of the row each, NV times; 32 / LPK keys stand side by side, KB one behind the other. The lanes'
// parts of KB scores are added with every lane giving half of what it holds away at each exchange: KB - 1 + log2(LPK / KB) shuffles
// for KB scores, after which a lane has one of them, its exponential costs one instruction for all, and KB broadcasts bring them
// back for the products with the values.
#include "attn_decode.cuh"

namespace ptj {
namespace {

template <typename E, int DP, int RB>
struct CoreFma {
  static constexpr int VEC = 16 / static_cast<int>(sizeof(E)), kDim = DP, kRowBytes = DP * static_cast<int>(sizeof(E)), kRows = RB;
  static constexpr int LPK = DP / VEC < 32 ? DP / VEC : 32, NV = DP / (VEC * LPK), KPW = 32 / LPK, W = VEC * NV;
  static constexpr int KS = 4096 / kRowBytes, KB = KS / KPW;  // keys of a step, of a lane
  static constexpr int REP = LPK / KB;                        // lanes that end with the same score
  static constexpr int RG = RB < 4 ? RB : 4;                  // rows whose scores are on their way at a time
  static constexpr int kDepth = 3;
  static constexpr int kBlocks = 2;
  static constexpr bool kParts = false;  // probabilities are multiplied whole
  static constexpr int P = W / 2;  // pairs of elements: products run two elements wide
  uint64_t q[RB][P], o[RB][P];
  float ref[RB], sum[RB], over[RB];  // over: scores beyond it (not scaled) move the reference
  int limit[RB];  // last keys that the rows attend
  int sub_lane, grp;

  __device__ __forceinline__ int elem(int i) const { return (i * LPK + sub_lane) * VEC; }

  __device__ __forceinline__ void init(const DecodeAttn& p, const Segment& sg) {
    const int lane = threadIdx.x & 31;
    sub_lane = lane % LPK;
    grp = lane / LPK;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      ref[r] = kNoRef;
      over[r] = -INFINITY;
      sum[r] = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) q[r][i] = o[r][i] = 0ull;  // (two zeros)
      const int row = sg.rb * kRows + r;
      limit[r] = sg.limit(p, row);
      if (limit[r] < 0) continue;
      const E* src = reinterpret_cast<const E*>(sg.q_row(p, row));
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const int d = elem(i) + e;
          q[r][(i * VEC + e) / 2] = f2_pack(d < p.D ? Elem<E>::load(src + d) : 0.f, d + 1 < p.D ? Elem<E>::load(src + d + 1) : 0.f);
        }
    }
  }

  __device__ __forceinline__ void read(const uint8_t* stage, int r, uint64_t (&out)[P]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(stage + r * kRowBytes + (((i * LPK + sub_lane) ^ swizzle(r % KS)) << 4));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        if constexpr (sizeof(E) == 4) out[i * VEC / 2 + e] = f2_pack(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
        else out[i * VEC / 2 + e] = f2_pack(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
      }
    }
  }

  template <bool>
  __device__ __forceinline__ void step(const DecodeAttn& p, const Segment& sg, int sub, const uint8_t* stage) {
    const int j0 = sub * KS;
    const uint32_t present = present_keys<KS, kRowBytes>(stage);
    const bool edge = j0 + KS > sg.first + 1 || present != (1u << KS) - 1u;  // some rows do not attend all of its keys
    uint64_t k[KB][P], v[KB][P];
#pragma unroll
    for (int e = 0; e < KB; ++e) read(stage, e * KPW + grp, k[e]);
#pragma unroll
    for (int e = 0; e < KB; ++e) read(stage, KS + e * KPW + grp, v[e]);
    const int own = sub_lane / REP * KPW + grp;  // place in the step of the key whose score this lane ends with
    // RG rows side by side: one row's chain of shuffles, exponential and shuffles is long
#pragma unroll
    for (int r0 = 0; r0 < RB; r0 += RG) {
      const int row0 = sg.rb * kRows + r0;
      if (RB > RG && row0 >= p.R) break;
      float s[RG][KB];
#pragma unroll
      for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int e = 0; e < KB; ++e) {
          uint64_t d = f2_mul(q[r0 + r][0], k[e][0]);
#pragma unroll
          for (int i = 1; i < P; ++i) d = f2_fma(q[r0 + r][i], k[e][i], d);
          float lo, hi;
          f2_unpack(d, lo, hi);
          s[r][e] = lo + hi;
        }
      // to one score per lane and row
#pragma unroll
      for (int n = KB / 2, x = LPK / 2; x > 0; n /= 2, x /= 2)
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          if (n > 0) {
            const bool up = sub_lane & x;
#pragma unroll
            for (int e = 0; e < n; ++e) {
              const float give = up ? s[r][e] : s[r][e + n], stay = up ? s[r][e + n] : s[r][e];
              s[r][e] = stay + __shfl_xor_sync(0xffffffffu, give, x);
            }
          } else {
            s[r][0] += __shfl_xor_sync(0xffffffffu, s[r][0], x);
          }
        }
      float mine[RG];
      bool moves = false;
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        mine[r] = s[r][0];
        if (edge && (!((present >> own) & 1u) || j0 + own > limit[r0 + r])) mine[r] = -INFINITY;
        moves |= mine[r] > over[r0 + r];
      }
      if (p.scores != nullptr && sub_lane % REP == 0 && j0 + own < sg.n)
#pragma unroll
        for (int r = 0; r < RG; ++r)
          if (row0 + r < p.R) sg.score_row(p, row0 + r)[j0 + own] = mine[r] * p.scale;
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int r = 0; r < RG; ++r) {
          const float m = fmaxf(warp_max(mine[r]) * p.scale, ref[r0 + r]);
          const float f = rebase(ref[r0 + r], m);
          ref[r0 + r] = m;
          over[r0 + r] = (m + kDecLazy) * p.unscale;
          sum[r0 + r] *= f;
#pragma unroll
          for (int i = 0; i < P; ++i) o[r0 + r][i] = f2_mul(o[r0 + r][i], f2_pack(f, f));
        }
      }
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        mine[r] = ex2(fmaf(mine[r], p.scale, -ref[r0 + r]));
        sum[r0 + r] += mine[r];
      }
#pragma unroll
      for (int r = 0; r < RG; ++r) {
#pragma unroll
        for (int e = 0; e < KB; ++e) s[r][e] = __shfl_sync(0xffffffffu, mine[r], e * REP, LPK);
        if (edge) {  // zero times what is not finite is not zero
#pragma unroll
          for (int e = 0; e < KB; ++e) {
            if (j0 + e * KPW + grp > limit[r0 + r]) continue;
#pragma unroll
            for (int i = 0; i < P; ++i) o[r0 + r][i] = f2_fma(f2_pack(s[r][e], s[r][e]), v[e][i], o[r0 + r][i]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < KB; ++e)
#pragma unroll
            for (int i = 0; i < P; ++i) o[r0 + r][i] = f2_fma(f2_pack(s[r][e], s[r][e]), v[e][i], o[r0 + r][i]);
        }
      }
    }
  }

  // f(row, element, four sums, reference exponent, sum of the row, true for one call per row)
  template <typename F>
  __device__ __forceinline__ void emit(F&& f) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const float l = warp_sum(sum[r]) * (1.f / REP);
#pragma unroll
      for (int x = LPK; x < 32; x <<= 1)
#pragma unroll
        for (int i = 0; i < P; ++i) o[r][i] = f2_add(o[r][i], __shfl_xor_sync(0xffffffffu, o[r][i], x));
      if (grp == 0)
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          float4 x;
          f2_unpack(o[r][i / 2], x.x, x.y);
          f2_unpack(o[r][i / 2 + 1], x.z, x.w);
          f(r, elem(i / VEC) + i % VEC, x, ref[r], l, sub_lane == 0 && i == 0);
        }
    }
  }
};

}  // namespace

int decode_fma_blocks() { return CoreFma<float, 64, 1>::kBlocks; }

int launch_decode_fma(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st) {
  using B = __nv_bfloat16;
  if (pl.es == 2)
    return pl.rows == 1 ? launch_decode<B, CoreFma<B, 256, 1>>(d, pl, st) : launch_decode<B, CoreFma<B, 256, 4>>(d, pl, st);
  switch (pl.dim + pl.rows) {
    case 64 + 1: return launch_decode<float, CoreFma<float, 64, 1>>(d, pl, st);
    case 64 + 4: return launch_decode<float, CoreFma<float, 64, 4>>(d, pl, st);
    case 64 + 8: return launch_decode<float, CoreFma<float, 64, 8>>(d, pl, st);
    case 128 + 1: return launch_decode<float, CoreFma<float, 128, 1>>(d, pl, st);
    case 128 + 4: return launch_decode<float, CoreFma<float, 128, 4>>(d, pl, st);
    case 128 + 8: return launch_decode<float, CoreFma<float, 128, 8>>(d, pl, st);
    case 256 + 1: return launch_decode<float, CoreFma<float, 256, 1>>(d, pl, st);
    default: return launch_decode<float, CoreFma<float, 256, 4>>(d, pl, st);
  }
}

}  // namespace ptj
