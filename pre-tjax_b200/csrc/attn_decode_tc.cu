// Attention of new tokens over a paged cache, bf16 heads of up to 128: tensor cores.
//
// S^T = K Q^T and O^T = V^T P^T with m16n8k16: keys, then head elements, are the 16 rows of a product, eight query rows its columns,
// so one to eight rows cost the same. Which head element sits at which k of a product
// is free as long as Q and K agree, so a lane's 16 bytes of a key are its operands of two products, and its 16 bytes of four
// values turn into operands of four products by picking halves of pairs (the transposition that V needs). P^T comes from S^T by
// transposing 8 x 8 blocks in registers. Probabilities are multiplied in two bf16 parts (16 bits): rounding them to one would
// cost as much accuracy as rounding the output does. Up to four rows take four columns with their first parts and the other four
// with their second ones, so the second part costs nothing; more rows take a second product. The products are not what bounds it (one
// takes 8 cycles of an SM's quarter, 21 in a chain): up to 16 rows memory does (4 x 8 caches of 30k keys of 128, 1, 8 and 16 rows: 89,
// 89 and 92 us, floor 75), 24 rows fill the registers (90 us) and leave nothing for the list of stretches.
#include "attn_decode.cuh"

namespace ptj {
namespace {

template <int DP, int NR, bool HALF = false>
struct CoreTc {
  static_assert(!HALF || NR == 1, "");
  static constexpr int KS = 16, kRows = HALF ? 4 : 8 * NR, kDim = DP, kRowBytes = 2 * DP, KU = DP / 32, VW = DP / 64;
  static constexpr int kDepth = DP == 64 ? (NR == 1 ? 3 : 4) : 3;
  static constexpr bool kParts = true;  // probabilities are multiplied in parts: spoiled()
  static constexpr int kBlocks = DP == 64 ? (NR == 1 ? 4 : 3) : 2;  // resident per SM
  uint4 q[NR][KU];
  float o[NR][DP / 16][4];
  float ref[NR][2], sum[NR][2], over[NR][2];  // over: scores beyond it (not scaled) move the reference
  int g, c;
  uint32_t key_at, value_at[2];  // this lane's pieces in a step
  float* score_at;               // scores of its first column's row, at the first of its keys of step 0; NULL: not wanted
  int limit[NR][2];              // last keys that its columns' rows attend

  __device__ __forceinline__ void init(const DecodeAttn& p, const Segment& sg) {
    const int lane = threadIdx.x & 31;
    g = lane >> 2;
    c = lane & 3;
    key_at = g * kRowBytes + ((c ^ swizzle(g)) << 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) value_at[i] = (KS + 2 * c + i) * kRowBytes + ((g ^ swizzle(2 * c + i)) << 4);
    score_at = p.scores == nullptr || (HALF && c >= 2) ? nullptr : sg.score_row(p, sg.rb * kRows + 2 * c) + g;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = sg.rb * kRows + (HALF ? g & 3 : i * 8 + g);
      const bool on = sg.limit(p, r) >= 0;
      const char* row = on ? sg.q_row(p, r) : nullptr;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int d = 32 * u + 8 * c;
        q[i][u] = make_uint4(0u, 0u, 0u, 0u);
        if (!on) continue;
        if (p.q_wide && d + 8 <= p.D) {
          q[i][u] = *reinterpret_cast<const uint4*>(row + d * 2);
        } else {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(row);
          auto at = [&](int x) { return d + x < p.D ? static_cast<uint32_t>(e[d + x]) : 0u; };
          q[i][u] = make_uint4(at(0) | at(1) << 16, at(2) | at(3) << 16, at(4) | at(5) << 16, at(6) | at(7) << 16);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ref[i][e] = kNoRef;
        over[i][e] = -INFINITY;
        sum[i][e] = 0.f;
        const int row = sg.rb * kRows + row_of(i, e);
        limit[i][e] = sg.limit(p, row);
      }
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
    }
  }

  // row of the block that column 2 c + e of a product belongs to
  __device__ __forceinline__ int row_of(int i, int e) const { return HALF ? 2 * (c & 1) + e : i * 8 + 2 * c + e; }
  // rows of S^T (keys of a step) and k of O^T's products that this lane holds
  __device__ __forceinline__ int key_of(int i) const { return g + 8 * i; }
  __device__ __forceinline__ int value_of(int i) const { return 2 * c + (i & 1) + 8 * (i >> 1); }
  __device__ __forceinline__ uint4 key(const uint8_t* stage, int i, int u) const {
    return *reinterpret_cast<const uint4*>(stage + ((key_at ^ ((u & 1) << 6)) + 8 * i * kRowBytes + (u >> 1) * 128));
  }
  __device__ __forceinline__ uint32_t value_place(int i, int w) const { return value_at[i & 1] + 8 * (i >> 1) * kRowBytes + w * 128; }
  __device__ __forceinline__ uint4 value(const uint8_t* stage, int i, int w) const {
    return *reinterpret_cast<const uint4*>(stage + value_place(i, w));
  }

  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
  }
  static __device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void operands(const uint4 (&v)[4], int j, uint32_t (&a)[4]) {
    const uint32_t v0 = word(v[0], j), v1 = word(v[1], j), v2 = word(v[2], j), v3 = word(v[3], j);
    a[0] = __byte_perm(v0, v1, 0x5410), a[1] = __byte_perm(v0, v1, 0x7632);
    a[2] = __byte_perm(v2, v3, 0x5410), a[3] = __byte_perm(v2, v3, 0x7632);
  }
  static __device__ __forceinline__ void values(float (&acc)[4], const uint4 (&v)[4], int j, const uint32_t (&ph)[2], const uint32_t (&pl)[2]) {
    uint32_t a[4];
    operands(v, j, a);
    mma(acc, a[0], a[1], a[2], a[3], ph[0], ph[1]);
    if constexpr (!HALF) mma(acc, a[0], a[1], a[2], a[3], pl[0], pl[1]);
  }

  // A value that is not finite makes NaN of sums that it does not belong to: of rows that do not attend it, times their zeros, and of
  // those that do, times the second part of a probability (zero, or of either sign). No sum that it meets stays finite, so it is looked
  // for once, in the sums at the end, and costs the steps nothing; where there was one, they run again with CAREFUL.
  __device__ __forceinline__ bool spoiled() const {
    float sizes[4] = {0.f, 0.f, 0.f, 0.f};  // one addition per element; a sum that overflows only costs the second time
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sizes[e] += fabsf(o[i][j][e]);
    return __any_sync(0xffffffffu, !((sizes[0] + sizes[1]) + (sizes[2] + sizes[3]) < INFINITY));
  }

  template <bool CAREFUL>
  __device__ __forceinline__ void step(const DecodeAttn& p, const Segment& sg, int sub, uint8_t* stage) {
    const int j0 = sub * KS;
    const bool edge = j0 + KS > sg.first + 1;  // some rows do not attend all of its keys
    float s[NR][4];
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    float s2[NR][4];  // a second chain of products where there is one column of them
#pragma unroll
    for (int i = 0; i < NR; ++i) s2[i][0] = s2[i][1] = s2[i][2] = s2[i][3] = 0.f;
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const uint4 k0 = key(stage, 0, u), k1 = key(stage, 1, u);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        mma(s[i], k0.x, k1.x, k0.y, k1.y, q[i][u].x, q[i][u].y);
        mma(NR == 1 ? s2[i] : s[i], k0.z, k1.z, k0.w, k1.w, q[i][u].z, q[i][u].w);
      }
    }
    if constexpr (NR == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][e] += s2[0][e];
    }
    const uint32_t present = present_keys<KS, kRowBytes>(stage);
    if (edge || present != 0xffffu) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int j = j0 + key_of(x);
        const bool there = (present >> key_of(x)) & 1u;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!there || j > limit[i][e]) s[i][2 * x + e] = -INFINITY;
      }
    }
    bool moves = false;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) moves |= s[i][e] > over[i][e & 1];
    if (score_at != nullptr) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (sg.rb * kRows + row_of(i, e) < p.R) {
            float* to = score_at + (i * 8 + e) * p.scores_ld + j0;
            if (j0 + g < sg.n) to[0] = s[i][e] * p.scale;
            if (j0 + g + 8 < sg.n) to[8] = s[i][e + 2] * p.scale;
          }
    }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(s[i][e], s[i][e + 2]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
          m = fmaxf(m * p.scale, ref[i][e]);
          const float f = rebase(ref[i][e], m);
          ref[i][e] = m;
          over[i][e] = (m + kDecLazy) * p.unscale;
          sum[i][e] *= f;
#pragma unroll
          for (int j = 0; j < DP / 16; ++j) {
            o[i][j][e] *= f;
            o[i][j][e + 2] *= f;
          }
        }
    }
    uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x0 = ex2(fmaf(s[i][2 * k], p.scale, -ref[i][0])), x1 = ex2(fmaf(s[i][2 * k + 1], p.scale, -ref[i][1]));
        sum[i][0] += x0;
        sum[i][1] += x1;
        const uint32_t hi = pack(x0, x1);
        const uint32_t lo = pack(x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u));
        if constexpr (HALF) {
          ph[i][k] = transpose8(c < 2 ? hi : lo);
        } else {
          ph[i][k] = transpose8(hi);
          pl[i][k] = transpose8(lo);
        }
      }
    if (CAREFUL && not_finite(stage)) infinite_values(p, sg, j0, stage, ph, edge);
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint4 v[4] = {value(stage, 0, w), value(stage, 1, w), value(stage, 2, w), value(stage, 3, w)};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < NR; ++i) values(o[i][w * 4 + j], v, j, ph[i], pl[i]);
    }
  }

  __device__ __forceinline__ bool not_finite(const uint8_t* stage) const {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint4 v = value(stage, i, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = word(v, j);
          bad |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
        }
      }
    return __any_sync(0xffffffffu, bad);
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t x) {  // zero in place of halves that are not
    return ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u);
  }
  // Takes the values of a step that are not finite out of it and adds their products, by the first parts of the probabilities only.
  // At an edge once per new token, with what it does not attend cleared, and to its rows only.
  __device__ __forceinline__ void infinite_values(const DecodeAttn& p, const Segment& sg, int j0, uint8_t* stage, const uint32_t (&ph)[NR][2],
                                                  bool edge) {
    const int tokens = edge ? sg.count : 1;
#pragma unroll 1
    for (int tok = 0; tok < tokens; ++tok)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = !edge || j0 + value_of(i) <= sg.first + tok ? value(stage, i, w) : make_uint4(0u, 0u, 0u, 0u);
          v[i] = make_uint4(v[i].x ^ finite(v[i].x), v[i].y ^ finite(v[i].y), v[i].z ^ finite(v[i].z), v[i].w ^ finite(v[i].w));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t a[4];
            operands(v, j, a);
            mma(acc, a[0], a[1], a[2], a[3], ph[i][0], ph[i][1]);
            if (HALF && c >= 2) continue;  // (columns of second parts)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!edge || limit[i][e & 1] == sg.first + tok) o[i][w * 4 + j][e] += acc[e];
          }
      }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < VW; ++w) {  // (a lane's own pieces: nobody else reads them)
        const uint4 v = value(stage, i, w);
        *reinterpret_cast<uint4*>(stage + value_place(i, w)) = make_uint4(finite(v.x), finite(v.y), finite(v.z), finite(v.w));
      }
  }

  // f(row, element, four sums, reference exponent, sum of the row, true for one call per row)
  template <typename F>
  __device__ __forceinline__ void emit(F&& f) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[i][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        if constexpr (HALF) {  // the parts of a row meet; its two lanes share the elements
#pragma unroll
          for (int j = 0; j < DP / 16; ++j) {
            o[i][j][e] += __shfl_xor_sync(0xffffffffu, o[i][j][e], 2);
            o[i][j][e + 2] += __shfl_xor_sync(0xffffffffu, o[i][j][e + 2], 2);
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const float (&x)[4] = o[i][4 * w], (&y)[4] = o[i][4 * w + 1], (&z)[4] = o[i][4 * w + 2], (&u)[4] = o[i][4 * w + 3];
          if constexpr (HALF) {
            const bool up = c >= 2;
            f(row_of(i, e), 64 * w + 8 * g + (up ? 4 : 0),
              make_float4(up ? z[e] : x[e], up ? z[e + 2] : x[e + 2], up ? u[e] : y[e], up ? u[e + 2] : y[e + 2]), ref[i][e], l,
              w == 0 && g == 0 && !up);
          } else {
            f(row_of(i, e), 64 * w + 8 * g, make_float4(x[e], x[e + 2], y[e], y[e + 2]), ref[i][e], l, w == 0 && g == 0);
            f(row_of(i, e), 64 * w + 8 * g + 4, make_float4(z[e], z[e + 2], u[e], u[e + 2]), ref[i][e], l, false);
          }
        }
      }
  }
};

}  // namespace

int decode_tc_blocks(int dim, int rows) { return dim == 128 ? CoreTc<128, 1>::kBlocks : (rows <= 8 ? CoreTc<64, 1>::kBlocks : CoreTc<64, 2>::kBlocks); }

int launch_decode_tc(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st) {
  using E = __nv_bfloat16;
  switch (pl.dim + pl.rows) {
    case 64 + 4: return launch_decode<E, CoreTc<64, 1, true>>(d, pl, st);
    case 64 + 8: return launch_decode<E, CoreTc<64, 1>>(d, pl, st);
    case 64 + 16: return launch_decode<E, CoreTc<64, 2>>(d, pl, st);
    case 64 + 32: return launch_decode<E, CoreTc<64, 4>>(d, pl, st);
    case 128 + 4: return launch_decode<E, CoreTc<128, 1, true>>(d, pl, st);
    case 128 + 8: return launch_decode<E, CoreTc<128, 1>>(d, pl, st);
    case 128 + 16: return launch_decode<E, CoreTc<128, 2>>(d, pl, st);
    default: return launch_decode<E, CoreTc<128, 3>>(d, pl, st);
  }
}

}  // namespace ptj
