// Attention of new tokens over a paged key-value cache.
//
// out = softmax(q K^T / sqrt(d)) V for the R = group * tokens query rows that share a key head. Every key and value is read once
// and multiplied with a handful of rows: memory bounds it, so the kernel is built to keep loads in flight and to share them
// out evenly.
//
// Work: the keys of every (sequence, key head, block of rows) are cut into tiles of 64; all tiles of the call form one list in
// which lengths, known on the device only, no longer matter, and every worker block takes an equal stretch of it. A worker that
// holds all tiles of a segment writes its output; pieces of a segment (at most two per worker) go to the workspace with their
// maximum and sum and are joined, in order, by a second kernel. Results do not depend on timing.
//
// A warp takes 16 keys at a time. Running sums are kept relative to a reference exponent that only moves when a score outgrows it
// by more than 2^8, so that a tile costs one vote instead of a reduction over lanes.
#include "kv_cache.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kSub = 16, kTile = kSub * kWarps;  // keys of a warp's step and of a block's
constexpr int kJoinThreads = 256;
constexpr float kLazy = 8.f;

struct DecodeAttn {
  PagedRows rows;
  const int32_t *lengths, *counts;
  const char *q, *kn, *vn;   // queries, new rows (NULL: in the pages already)
  char *k, *v, *out;
  int64_t qs[3], os[3], kns[3], vns[3];  // bytes
  const float* weights;
  float* weights_out;
  int64_t weights_ld, scores_ld;
  float *part, *part_ml;     // pieces: [workers][2][block rows][D], [..][2] reference exponent and sum
  float *ml;                 // [segments][block rows][2] of segments that one worker did
  float* scores;             // [batch * key heads][R][scores_ld], log2 units; NULL without weights
  float scale, keep;         // log2(e) / sqrt(d); 1 - p
  int B, Hk, G, T, D, R;
  int nrb;                   // blocks of rows
  int workers, least;        // blocks of the grid; tiles that a worker takes at least
  int q_wide, out_wide;      // 16-byte accesses are aligned
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float base_of(float ref) { return ref == -INFINITY ? 0.f : ref; }
// factor of sums relative to `ref` when they are taken relative to m; sums without any score above -inf are zero (or NaN)
__device__ __forceinline__ float rebase(float ref, float m) { return ref == -INFINITY ? 1.f : ex2(ref - m); }

__device__ __forceinline__ uint4 load16(const char* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// What a block works on: one sequence, key head and block of rows
struct Segment {
  int b, h, rb;
  int n, count, first;  // keys, new tokens, position of the first of them
  const int32_t* table;
  // last key that row r (of all R) attends, -1: none
  __device__ __forceinline__ int limit(const DecodeAttn& p, int r) const {
    const int t = r % p.T;
    return r < p.R && t < count ? first + t : -1;
  }
  __device__ __forceinline__ int64_t index(const DecodeAttn& p) const {
    return (static_cast<int64_t>(b) * p.Hk + h) * p.nrb + rb;
  }
  // keys below this one are in the pages and attended by all rows that attend anything
  __device__ __forceinline__ int plain() const { return max(first, 0); }
  __device__ __forceinline__ const char* q_row(const DecodeAttn& p, int r) const {
    return p.q + b * p.qs[0] + (h * p.G + r / p.T) * p.qs[1] + (r % p.T) * p.qs[2];
  }
};
__device__ __forceinline__ void set_sequence(const DecodeAttn& p, Segment& sg, int b) {
  sg.b = b;
  sg.n = p.rows.length(p.lengths, b);
  sg.count = p.rows.count(p.counts, p.T, b);
  sg.first = sg.n - sg.count;
  sg.table = p.rows.table + b * p.rows.table_ld;
}

// ---- bf16, d_head a multiple of 8 up to 128, aligned rows: tensor cores ----------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T with m16n8k16: keys, then head elements, are the 16 rows, eight query rows the columns, so one to
// eight rows cost the same and sixteen twice that. All fragments come straight from global memory: which head element sits
// at which k of a product is free as long as Q and K agree, so a lane's 16 bytes of a key are its operands of two products, and
// a lane's 16 bytes of four values turn into operands of four products by picking halves of pairs (the transposition that V
// needs). P^T comes from S^T by transposing 8 x 8 blocks in registers. Probabilities are multiplied in two bf16 parts (16 bits);
// the second part's products cost nothing that shows.
template <int DP, int NR>
struct CoreTc {
  static constexpr int kRows = 8 * NR, KU = DP / 32, VW = DP / 64, kDim = DP;
  static constexpr int kBlocks = DP == 64 ? (NR == 1 ? 4 : 3) : 2;  // resident per SM
  struct Tile {
    uint4 k[2][KU], v[4][VW];
    bool ok[2];
  };
  uint4 q[NR][KU];
  float o[NR][DP / 16][4];
  float ref[NR][2], sum[NR][2];
  int g, c;

  __device__ __forceinline__ void init(const DecodeAttn& p, const Segment& sg) {
    const int lane = threadIdx.x & 31;
    g = lane >> 2;
    c = lane & 3;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = sg.rb * kRows + i * 8 + g;
      const bool on = sg.limit(p, r) >= 0;
      const char* row = on ? sg.q_row(p, r) : nullptr;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int d = 32 * u + 8 * c;
        q[i][u] = make_uint4(0u, 0u, 0u, 0u);
        if (on && d < p.D) {
          if (p.q_wide) {
            q[i][u] = *reinterpret_cast<const uint4*>(row + d * 2);
          } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(row) + d;
            q[i][u].x = e[0] | e[1] << 16;
            q[i][u].y = e[2] | e[3] << 16;
            q[i][u].z = e[4] | e[5] << 16;
            q[i][u].w = e[6] | e[7] << 16;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ref[i][e] = -INFINITY;
        sum[i][e] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < DP / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
    }
  }

  __device__ __forceinline__ void load_key(const DecodeAttn& p, Tile& t, int i, const char* row, bool on) const {
#pragma unroll
    for (int u = 0; u < KU; ++u)
      t.k[i][u] = on && 32 * u + 8 * c < p.D ? load16(row + (32 * u + 8 * c) * 2) : make_uint4(0u, 0u, 0u, 0u);
    t.ok[i] = on;
  }
  __device__ __forceinline__ void load_value(const DecodeAttn& p, Tile& t, int i, const char* row, bool on) const {
#pragma unroll
    for (int w = 0; w < VW; ++w)
      t.v[i][w] = on && 64 * w + 8 * g < p.D ? load16(row + (64 * w + 8 * g) * 2) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ int key_of(int i) const { return g + 8 * i; }
  __device__ __forceinline__ int value_of(int i) const { return 2 * c + (i & 1) + 8 * (i >> 1); }

  // 16 keys that are all in the pages
  __device__ __forceinline__ void load(const DecodeAttn& p, const Segment& sg, int sub, Tile& t) const {
    const int j0 = sub * kSub;
    if (p.rows.page_size % kSub == 0) {  // in one page
      int64_t page;
      int slot;
      const bool on = p.rows.locate(sg.table, j0, page, slot);
      const char* k = p.k + p.rows.offset(0, page, sg.h, slot);
      const char* v = p.v + p.rows.offset(1, page, sg.h, slot);
#pragma unroll
      for (int i = 0; i < 2; ++i) load_key(p, t, i, k + key_of(i) * p.rows.slot_stride[0], on);
#pragma unroll
      for (int i = 0; i < 4; ++i) load_value(p, t, i, v + value_of(i) * p.rows.slot_stride[1], on);
    } else {
      int64_t page;
      int slot;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool on = p.rows.locate(sg.table, j0 + key_of(i), page, slot);
        load_key(p, t, i, p.k + p.rows.offset(0, page, sg.h, slot), on);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool on = p.rows.locate(sg.table, j0 + value_of(i), page, slot);
        load_value(p, t, i, p.v + p.rows.offset(1, page, sg.h, slot), on);
      }
    }
  }
  // 16 keys some of which are new, or behind the last one; new rows are put into their pages
  __device__ __forceinline__ void load_edge(const DecodeAttn& p, const Segment& sg, int sub, Tile& t) const {
    const int j0 = sub * kSub;
    auto fetch = [&](int kv, int j, bool& on, bool& fresh, char*& slot_at) -> const char* {
      int64_t page;
      int slot;
      on = j < sg.n;
      const bool placed = on && p.rows.locate(sg.table, j, page, slot);
      fresh = on && j >= sg.first && p.kn != nullptr;
      slot_at = placed ? (kv == 0 ? p.k : p.v) + p.rows.offset(kv, page, sg.h, slot) : nullptr;
      on = placed;
      if (fresh && placed) {
        const int64_t* s = kv == 0 ? p.kns : p.vns;
        return (kv == 0 ? p.kn : p.vn) + sg.b * s[0] + sg.h * s[1] + (j - sg.first) * s[2];
      }
      return slot_at;
    };
    bool on, fresh;
    char* at;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* row = fetch(0, j0 + key_of(i), on, fresh, at);
      load_key(p, t, i, row, on);
      if (fresh && on && sg.rb == 0)
#pragma unroll
        for (int u = 0; u < KU; ++u)
          if (32 * u + 8 * c < p.D) *reinterpret_cast<uint4*>(at + (32 * u + 8 * c) * 2) = t.k[i][u];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* row = fetch(1, j0 + value_of(i), on, fresh, at);
      load_value(p, t, i, row, on);
      if (fresh && on && sg.rb == 0)
#pragma unroll
        for (int w = 0; w < VW; ++w)
          if (64 * w + 8 * g < p.D) *reinterpret_cast<uint4*>(at + (64 * w + 8 * g) * 2) = t.v[i][w];
    }
  }

  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

  // acc += V^T P^T
  template <int N>
  __device__ __forceinline__ void values(float (&acc)[N][DP / 16][4], const Tile& t, const uint32_t (&ph)[NR][2],
                                         const uint32_t (&pl)[NR][2]) const {
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t v0 = word(t.v[0][w], j), v1 = word(t.v[1][w], j), v2 = word(t.v[2][w], j), v3 = word(t.v[3][w], j);
        const uint32_t a0 = __byte_perm(v0, v1, 0x5410), a1 = __byte_perm(v0, v1, 0x7632);
        const uint32_t a2 = __byte_perm(v2, v3, 0x5410), a3 = __byte_perm(v2, v3, 0x7632);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          mma(acc[i][w * 4 + j], a0, a1, a2, a3, ph[i][0], ph[i][1]);
          mma(acc[i][w * 4 + j], a0, a1, a2, a3, pl[i][0], pl[i][1]);
        }
      }
  }

  template <bool EDGE>
  __device__ __forceinline__ void compute(const DecodeAttn& p, const Segment& sg, int sub, const Tile& t) {
    float s[NR][4];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        mma(s[i], t.k[0][u].x, t.k[1][u].x, t.k[0][u].y, t.k[1][u].y, q[i][u].x, q[i][u].y);
        mma(s[i], t.k[0][u].z, t.k[1][u].z, t.k[0][u].w, t.k[1][u].w, q[i][u].z, q[i][u].w);
      }
    }
    bool over = false;
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] *= p.scale;
        bool on = t.ok[e >> 1];
        if (EDGE) on = on && sub * kSub + key_of(e >> 1) <= sg.limit(p, sg.rb * kRows + i * 8 + 2 * c + (e & 1));
        if (!on) s[i][e] = -INFINITY;
        over |= s[i][e] > ref[i][e & 1] + kLazy;
      }
    if (p.scores != nullptr) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = sg.rb * kRows + i * 8 + 2 * c + (e & 1), j = sub * kSub + key_of(e >> 1);
          if (r < p.R && j < sg.n)
            p.scores[((static_cast<int64_t>(sg.b) * p.Hk + sg.h) * p.R + r) * p.scores_ld + j] = s[i][e];
        }
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(s[i][e], s[i][e + 2]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
          m = fmaxf(m, ref[i][e]);
          const float f = rebase(ref[i][e], m);
          ref[i][e] = m;
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
        const float x0 = ex2(s[i][2 * k] - base_of(ref[i][0])), x1 = ex2(s[i][2 * k + 1] - base_of(ref[i][1]));
        sum[i][0] += x0;
        sum[i][1] += x1;
        const uint32_t hi = pack(x0, x1);
        const uint32_t lo = pack(x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u));
        ph[i][k] = transpose8(hi);
        pl[i][k] = transpose8(lo);
      }
    if (EDGE) {
      // a value that some rows of the tile attend and others do not must be finite to be multiplied by the others' zeros
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = word(t.v[i][w], j);
            bad |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
          }
      if (__any_sync(0xffffffffu, bad)) {
        values_by_token(p, sg, sub, t, ph, pl);
        return;
      }
    }
    values(o, t, ph, pl);
  }

  // The products of an edge tile with values that are not finite: once per new token, with what it does not attend cleared, and
  // added to its rows only.
  __device__ __forceinline__ void values_by_token(const DecodeAttn& p, const Segment& sg, int sub, const Tile& t,
                                               const uint32_t (&ph)[NR][2], const uint32_t (&pl)[NR][2]) {
#pragma unroll 1
    for (int tok = 0; tok < sg.count; ++tok) {
      Tile m = t;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (sub * kSub + value_of(i) > sg.first + tok)
#pragma unroll
          for (int w = 0; w < VW; ++w) m.v[i][w] = make_uint4(0u, 0u, 0u, 0u);
      float acc[NR][DP / 16][4];
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
      values(acc, m, ph, pl);
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if ((sg.rb * kRows + i * 8 + 2 * c + e) % p.T == tok)
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
              o[i][j][e] += acc[i][j][e];
              o[i][j][e + 2] += acc[i][j][e + 2];
            }
    }
  }

  // steps s0, s0 + kWarps, .. below s1
  __device__ __forceinline__ void run(const DecodeAttn& p, const Segment& sg, int s0, int s1) {
    const int edge = min(sg.plain() / kSub, s1);
    int s = s0;
    Tile a, b;
    if (s < edge) {
      load(p, sg, s, a);
      for (;;) {
        if (s + kWarps < edge) load(p, sg, s + kWarps, b);
        compute<false>(p, sg, s, a);
        s += kWarps;
        if (s >= edge) break;
        if (s + kWarps < edge) load(p, sg, s + kWarps, a);
        compute<false>(p, sg, s, b);
        s += kWarps;
        if (s >= edge) break;
      }
    }
    for (; s < s1; s += kWarps) {
      load_edge(p, sg, s, a);
      compute<true>(p, sg, s, a);
    }
  }

  // sums of the warp: os [kRows][kDim + 4], ml [kRows][2]
  __device__ __forceinline__ void store(float* os, float* ml) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[i][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        const int r = i * 8 + 2 * c + e;
        if (g == 0) {
          ml[2 * r] = ref[i][e];
          ml[2 * r + 1] = l;
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
            *reinterpret_cast<float4*>(os + r * (kDim + 4) + 64 * w + 8 * g + 4 * hf) =
                make_float4(o[i][w * 4 + 2 * hf][e], o[i][w * 4 + 2 * hf][e + 2], o[i][w * 4 + 2 * hf + 1][e],
                            o[i][w * 4 + 2 * hf + 1][e + 2]);
      }
  }
};

// ---- everything else: float32 arithmetic on CUDA cores ----------------------------------------------------------------------
// LPK lanes share a key, VEC consecutive elements of a row at a time, NV times; 32 / LPK keys side by side, KB of them in flight.
template <typename E, int VEC, int LPK, int NV, int RB>
struct CoreFma {
  static constexpr int kRows = RB, KPW = 32 / LPK, kDim = VEC * LPK * NV;
  static constexpr int W = VEC * NV, KB = W >= 8 || LPK == 8 ? 4 : 8;
  static constexpr int kBlocks = RB * W <= 8 ? 4 : (RB * W <= 16 ? 3 : 2);
  float q[RB][W], o[RB][W];
  float ref[RB], sum[RB];
  int sub_lane, grp;

  static __device__ __forceinline__ void read(const char* row, int d, float* out) {
    if constexpr (VEC == 1) {
      out[0] = Elem<E>::load(reinterpret_cast<const E*>(row) + d);
    } else {
      const uint4 x = load16(row + d * static_cast<int>(sizeof(E)));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (sizeof(E) == 4) out[i] = __uint_as_float(w[i]);
        else out[i] = __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      }
    }
  }
  __device__ __forceinline__ int elem(int i) const { return (i * LPK + sub_lane) * VEC; }

  __device__ __forceinline__ void init(const DecodeAttn& p, const Segment& sg) {
    const int lane = threadIdx.x & 31;
    sub_lane = lane % LPK;
    grp = lane / LPK;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      ref[r] = -INFINITY;
      sum[r] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) q[r][i] = o[r][i] = 0.f;
      const int row = sg.rb * kRows + r;
      if (sg.limit(p, row) < 0) continue;
      const E* src = reinterpret_cast<const E*>(sg.q_row(p, row));
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (elem(i) + e < p.D) q[r][i * VEC + e] = Elem<E>::load(src + elem(i) + e);
    }
  }

  template <bool EDGE>
  __device__ __forceinline__ void batch(const DecodeAttn& p, const Segment& sg, int j0) {
    float k[KB][W], v[KB][W];
    bool ok[KB];
#pragma unroll
    for (int e = 0; e < KB; ++e) {
      const int j = j0 + e * KPW + grp;
      int64_t page;
      int slot;
      ok[e] = (!EDGE || j < sg.n) && p.rows.locate(sg.table, j, page, slot);
      const char *kr = nullptr, *vr = nullptr;
      char *ka = nullptr, *va = nullptr;
      if (ok[e]) {
        ka = p.k + p.rows.offset(0, page, sg.h, slot);
        va = p.v + p.rows.offset(1, page, sg.h, slot);
        kr = ka;
        vr = va;
      }
      const bool fresh = EDGE && ok[e] && j >= sg.first && p.kn != nullptr;
      if (fresh) {
        kr = p.kn + sg.b * p.kns[0] + sg.h * p.kns[1] + (j - sg.first) * p.kns[2];
        vr = p.vn + sg.b * p.vns[0] + sg.h * p.vns[1] + (j - sg.first) * p.vns[2];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = ok[e] && elem(i) < p.D;
        if (in) {
          read(kr, elem(i), k[e] + i * VEC);
          read(vr, elem(i), v[e] + i * VEC);
        } else {
#pragma unroll
          for (int x = 0; x < VEC; ++x) k[e][i * VEC + x] = v[e][i * VEC + x] = 0.f;
        }
        if (fresh && in && sg.rb == 0) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            Elem<E>::store(reinterpret_cast<E*>(ka) + elem(i) + x, k[e][i * VEC + x]);
            Elem<E>::store(reinterpret_cast<E*>(va) + elem(i) + x, v[e][i * VEC + x]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int row = sg.rb * kRows + r;
      if (RB > 1 && row >= p.R) break;
      const int limit = EDGE ? sg.limit(p, row) : 0;
      float s[KB];
#pragma unroll
      for (int e = 0; e < KB; ++e) {
        s[e] = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) s[e] = fmaf(q[r][i], k[e][i], s[e]);
      }
#pragma unroll
      for (int x = LPK / 2; x > 0; x >>= 1)
#pragma unroll
        for (int e = 0; e < KB; ++e) s[e] += __shfl_xor_sync(0xffffffffu, s[e], x);
      bool over = false;
#pragma unroll
      for (int e = 0; e < KB; ++e) {
        const int j = j0 + e * KPW + grp;
        s[e] = ok[e] && (!EDGE || j <= limit) ? s[e] * p.scale : -INFINITY;
        over |= s[e] > ref[r] + kLazy;
        if (p.scores != nullptr && sub_lane == 0 && j < sg.n && row < p.R)
          p.scores[((static_cast<int64_t>(sg.b) * p.Hk + sg.h) * p.R + row) * p.scores_ld + j] = s[e];
      }
      if (__any_sync(0xffffffffu, over)) {
        float m = s[0];
#pragma unroll
        for (int e = 1; e < KB; ++e) m = fmaxf(m, s[e]);
        m = fmaxf(warp_max(m), ref[r]);
        const float f = rebase(ref[r], m);
        ref[r] = m;
        sum[r] *= f;
#pragma unroll
        for (int i = 0; i < W; ++i) o[r][i] *= f;
      }
      const float base = base_of(ref[r]);
#pragma unroll
      for (int e = 0; e < KB; ++e) {
        const float x = ex2(s[e] - base);
        sum[r] += x;
        const bool on = !EDGE || j0 + e * KPW + grp <= limit;  // zero times what is not finite is not zero
#pragma unroll
        for (int i = 0; i < W; ++i) o[r][i] = fmaf(x, on ? v[e][i] : 0.f, o[r][i]);
      }
    }
  }

  __device__ __forceinline__ void run(const DecodeAttn& p, const Segment& sg, int s0, int s1) {
    const int edge = min(sg.plain() / kSub, s1);
    for (int s = s0; s < s1; s += kWarps) {
      if (s < edge) {
#pragma unroll 1
        for (int x = 0; x < kSub; x += KB * KPW) batch<false>(p, sg, s * kSub + x);
      } else {
#pragma unroll 1
        for (int x = 0; x < kSub; x += KB * KPW) batch<true>(p, sg, s * kSub + x);
      }
    }
  }

  __device__ __forceinline__ void store(float* os, float* ml) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float l = sum[r];
#pragma unroll
      for (int x = LPK; x < 32; x <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
        for (int i = 0; i < W; ++i) o[r][i] += __shfl_xor_sync(0xffffffffu, o[r][i], x);
      }
      if (grp == 0) {
        if (sub_lane == 0) {
          ml[2 * r] = ref[r];
          ml[2 * r + 1] = l;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) os[r * (kDim + 4) + elem(i) + e] = o[r][i * VEC + e];
      }
    }
  }
};

// ---- the list of tiles -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int tiles_of(int n) { return (n + kTile - 1) / kTile; }

// Tiles per (key head, block of rows) of all sequences, and of those before each thread's stretch of sequences.
// tot: shared, N / 32 entries; every thread of the block calls.
template <int N>
struct TileList {
  int64_t before, total;  // of this thread's stretch, of all
  int b0, b1;
  __device__ __forceinline__ void build(const DecodeAttn& p, int64_t* tot) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.B + N - 1) / N;
    b0 = min(tid * per, p.B);
    b1 = min(b0 + per, p.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(p.rows.length(p.lengths, b));
    int64_t incl = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, x);
      if (lane >= x) incl += y;
    }
    if (lane == 31) tot[warp] = incl;
    __syncthreads();
    before = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < N / 32; ++w) {
      if (w < warp) before += tot[w];
      total += tot[w];
    }
  }
};

__device__ __forceinline__ int64_t tiles_per_worker(const DecodeAttn& p, int64_t total) {
  const int64_t q = (total * p.Hk * p.nrb + p.workers - 1) / p.workers;
  return q > p.least ? q : p.least;
}

// Sum over the keys' rows of exp2(score - reference) / sum for keys [j0, j1) of a sequence's key head, onto the accumulated
// weights. row_ml(r): reference exponent and sum of row r.
template <int N, typename F>
__device__ __forceinline__ void add_weights(const DecodeAttn& p, const Segment& sg, int j0, int j1, F&& row_ml) {
  const int64_t bh = static_cast<int64_t>(sg.b) * p.Hk + sg.h;
  const float* in = p.weights == nullptr ? nullptr : p.weights + bh * p.weights_ld;
  float* out = p.weights_out + bh * p.weights_ld;
  for (int j = j0 + threadIdx.x; j < j1; j += N) {
    float w = j < sg.first && in != nullptr ? in[j] : 0.f;
    for (int r = 0; r < p.R; ++r) {
      if (sg.limit(p, r) < 0) continue;
      const float2 ml = row_ml(r);
      w += ex2(p.scores[(bh * p.R + r) * p.scores_ld + j] - base_of(ml.x)) / ml.y;
    }
    out[j] = w;
  }
}

template <typename E>
__device__ __forceinline__ void store_out(const DecodeAttn& p, const Segment& sg, int r, int d, const float4& x) {
  char* row = p.out + sg.b * p.os[0] + (sg.h * p.G + r / p.T) * p.os[1] + (r % p.T) * p.os[2];
  const float v[4] = {x.x, x.y, x.z, x.w};
  if (p.out_wide && d + 4 <= p.D) {
    if constexpr (sizeof(E) == 4) {
      *reinterpret_cast<float4*>(row + d * 4) = x;
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
      *reinterpret_cast<uint2*>(row + d * 2) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < p.D) Elem<E>::store(reinterpret_cast<E*>(row) + d + i, v[i]);
  }
}

// SPLIT false: a block per segment, nothing to join.
template <typename E, typename Core, bool SPLIT>
__global__ void __launch_bounds__(kThreads, Core::kBlocks)
attn_decode_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  constexpr int LD = Core::kDim + 4;
  __shared__ __align__(16) float os[kWarps][Core::kRows * LD];
  __shared__ float ml[kWarps][Core::kRows][2];
  __shared__ float fac[kWarps][Core::kRows], fin[Core::kRows][2];
  __shared__ int64_t tot[kWarps];
  __shared__ int64_t start_s[2];
  const int tid = threadIdx.x, warp = tid >> 5;
  Segment sg;
  int64_t left = 1, range0 = 0, at = 0;  // tiles of this worker's stretch, its start, where this segment starts
  int tile = 0, tiles;
  if (SPLIT) {
    TileList<kThreads> list;
    list.build(p, tot);
    const int64_t per_seq = static_cast<int64_t>(p.Hk) * p.nrb, all = list.total * per_seq;
    const int64_t q = tiles_per_worker(p, list.total);
    range0 = blockIdx.x * q;
    left = min(q, all - range0);
    if (left <= 0) return;
    // the thread whose stretch of sequences holds the first tile looks for its sequence
    int64_t acc = list.before * per_seq;
    for (int b = list.b0; b < list.b1; ++b) {
      const int64_t t = tiles_of(p.rows.length(p.lengths, b)) * per_seq;
      if (range0 >= acc && range0 < acc + t) {
        start_s[0] = b;
        start_s[1] = acc;
      }
      acc += t;
    }
    __syncthreads();
    set_sequence(p, sg, static_cast<int>(start_s[0]));
    tiles = tiles_of(sg.n);
    const int64_t in_seq = range0 - start_s[1];
    const int64_t hr = in_seq / tiles;
    tile = static_cast<int>(in_seq - hr * tiles);
    sg.h = static_cast<int>(hr / p.nrb);
    sg.rb = static_cast<int>(hr % p.nrb);
    at = range0 - tile;
  } else {
    const int hr = blockIdx.x % (p.Hk * p.nrb);
    set_sequence(p, sg, blockIdx.x / (p.Hk * p.nrb));
    sg.h = hr / p.nrb;
    sg.rb = hr % p.nrb;
    tiles = tiles_of(sg.n);
  }
  for (;;) {
    const int t1 = SPLIT ? static_cast<int>(min(static_cast<int64_t>(tiles), tile + left)) : tiles;
    {
      Core core;
      core.init(p, sg);
      core.run(p, sg, tile * kWarps + warp, min(t1 * kWarps, (sg.n + kSub - 1) / kSub));
      core.store(os[warp], &ml[warp][0][0]);
    }
    __syncthreads();
    if (tid < Core::kRows) {
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w][tid][0]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        fac[w][tid] = rebase(ml[w][tid][0], m);
        l = fmaf(fac[w][tid], ml[w][tid][1], l);
      }
      fin[tid][0] = m;
      fin[tid][1] = l;
    }
    __syncthreads();
    const bool whole = tile == 0 && t1 == tiles;
    const int rows = min(Core::kRows, p.R - sg.rb * Core::kRows);
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (at <= range0 ? 0 : 1);
    for (int i = tid; i < rows * (Core::kDim / 4); i += kThreads) {
      const int r = i / (Core::kDim / 4), d = i % (Core::kDim / 4) * 4;
      if (d >= p.D) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(&os[w][r * LD + d]);
        const float f = fac[w][r];
        x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
      }
      if (!SPLIT || whole) {
        const int row = sg.rb * Core::kRows + r;
        const float f = p.keep / fin[r][1];
        const bool some = sg.limit(p, row) >= 0;
        x = some ? make_float4(x.x * f, x.y * f, x.z * f, x.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
        store_out<E>(p, sg, row, d, x);
      } else {
        *reinterpret_cast<float4*>(p.part + (slot * Core::kRows + r) * Core::kDim + d) = x;
      }
    }
    if (SPLIT && !whole && tid < rows) {
      p.part_ml[(slot * Core::kRows + tid) * 2] = fin[tid][0];
      p.part_ml[(slot * Core::kRows + tid) * 2 + 1] = fin[tid][1];
    }
    if (SPLIT && whole && p.scores != nullptr && tid < rows) {
      p.ml[(sg.index(p) * Core::kRows + tid) * 2] = fin[tid][0];
      p.ml[(sg.index(p) * Core::kRows + tid) * 2 + 1] = fin[tid][1];
    }
    if (!SPLIT) {
      if (p.scores != nullptr)  // (one block of rows: the host sees to it)
        add_weights<kThreads>(p, sg, 0, sg.n, [&](int r) { return make_float2(fin[r][0], fin[r][1]); });
      return;
    }
    left -= t1 - tile;
    if (left <= 0) return;
    at += tiles;
    tile = 0;
    if (++sg.rb == p.nrb) {
      sg.rb = 0;
      if (++sg.h == p.Hk) {
        sg.h = 0;
        do set_sequence(p, sg, sg.b + 1); while (sg.n == 0);  // (tiles are left: a sequence that has some follows)
        tiles = tiles_of(sg.n);
      }
    }
    __syncthreads();
  }
}

// Blocks [0, rows_blocks): a query row each, joined where several workers hold pieces of it, zero where there is nothing to
// attend. The others: the weights of a stretch of one sequence's and key head's keys.
template <typename E, typename Core>
__global__ void __launch_bounds__(kJoinThreads)
attn_join_kernel(const __grid_constant__ DecodeAttn p, int rows_blocks, int chunk, int chunks) {
  grid_dep_sync();
  constexpr int kVecs = Core::kDim / 4 < kJoinThreads ? Core::kDim / 4 : kJoinThreads, kGroups = kJoinThreads / kVecs;
  static_assert(kGroups * kVecs == kJoinThreads, "");
  __shared__ int64_t tot[kJoinThreads / 32];
  __shared__ int64_t before_s;
  __shared__ float red[33];
  __shared__ float4 part_s[kGroups][kVecs];
  const int tid = threadIdx.x;
  const bool row_block = blockIdx.x < rows_blocks;
  const int64_t id = row_block ? blockIdx.x : (blockIdx.x - rows_blocks) / chunks;
  const int64_t bh = row_block ? id / p.R : id;
  Segment sg;
  set_sequence(p, sg, static_cast<int>(bh / p.Hk));
  sg.h = static_cast<int>(bh % p.Hk);
  TileList<kJoinThreads> list;
  list.build(p, tot);
  if (sg.b >= list.b0 && sg.b < list.b1) {
    int64_t x = list.before;
    for (int b = list.b0; b < sg.b; ++b) x += tiles_of(p.rows.length(p.lengths, b));
    before_s = x;
  }
  __syncthreads();
  const int tiles = tiles_of(sg.n);
  const int64_t q = tiles_per_worker(p, list.total);
  const int64_t t_seq = before_s * p.Hk * p.nrb;
  auto pieces = [&](int rb, int64_t& w0, int64_t& w1, int64_t& t0) {
    t0 = t_seq + (static_cast<int64_t>(sg.h) * p.nrb + rb) * tiles;
    w0 = t0 / q;
    w1 = (t0 + tiles - 1) / q;
  };
  // a segment that starts where a worker's stretch starts is its first piece, as is one that started before
  auto slot_of = [&](int64_t w, int64_t t0) { return w * 2 + (t0 <= w * q ? 0 : 1); };
  if (row_block) {
    const int r = static_cast<int>(id % p.R);
    sg.rb = r / Core::kRows;
    const int rr = r % Core::kRows;
    const int d = tid % kVecs * 4, grp = tid / kVecs;
    int64_t w0 = 0, w1 = 0, t0 = 0;
    if (sg.limit(p, r) < 0 || tiles == 0) {
      if (tid < kVecs && d < p.D) store_out<E>(p, sg, r, d, make_float4(0.f, 0.f, 0.f, 0.f));
      return;
    }
    pieces(sg.rb, w0, w1, t0);
    if (w0 == w1) return;
    float m = -INFINITY;
    for (int64_t w = w0 + tid; w <= w1; w += kJoinThreads) m = fmaxf(m, p.part_ml[(slot_of(w, t0) * Core::kRows + rr) * 2]);
    m = block_max(m, red);
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int64_t w = w0 + grp; w <= w1; w += kGroups) {
      const int64_t s = slot_of(w, t0) * Core::kRows + rr;
      const float f = rebase(p.part_ml[s * 2], m);
      l = fmaf(f, p.part_ml[s * 2 + 1], l);
      if (d < p.D) {
        const float4 y = *reinterpret_cast<const float4*>(p.part + s * Core::kDim + d);
        x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
      }
    }
    part_s[grp][tid % kVecs] = x;
    __syncthreads();
    if (tid % kVecs == 0) red[grp] = l;  // (kGroups <= 32)
    __syncthreads();
    if (grp == 0 && d < p.D) {
      float sum = 0.f;
      x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < kGroups; ++k) {
        const float4 y = part_s[k][tid];
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        sum += red[k];
      }
      const float f = p.keep / sum;
      store_out<E>(p, sg, r, d, make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
    }
    return;
  }
  const int j0 = static_cast<int>((blockIdx.x - rows_blocks) % chunks) * chunk;
  if (j0 >= sg.n) return;
  extern __shared__ float2 row_ml[];  // [R]
  for (int r = tid; r < p.R; r += kJoinThreads) {
    int64_t w0, w1, t0;
    const int rb = r / Core::kRows, rr = r % Core::kRows;
    pieces(rb, w0, w1, t0);
    float m = -INFINITY, l = 0.f;
    if (w0 == w1) {
      const int64_t s = (bh * p.nrb + rb) * Core::kRows + rr;
      m = p.ml[s * 2];
      l = p.ml[s * 2 + 1];
    } else {
      for (int64_t w = w0; w <= w1; ++w) m = fmaxf(m, p.part_ml[(slot_of(w, t0) * Core::kRows + rr) * 2]);
      for (int64_t w = w0; w <= w1; ++w) {
        const int64_t s = slot_of(w, t0) * Core::kRows + rr;
        l = fmaf(rebase(p.part_ml[s * 2], m), p.part_ml[s * 2 + 1], l);
      }
    }
    row_ml[r] = make_float2(m, l);
  }
  __syncthreads();
  add_weights<kJoinThreads>(p, sg, j0, min(j0 + chunk, sg.n), [&](int r) { return row_ml[r]; });
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
constexpr int kMaxRows = 4096;      // query rows of a key head
constexpr int kDirectKeys = 256;    // sequences of at most this many keys are one block's work
constexpr int kLeastTiles = 2;
constexpr int kWorkersPerSm = 4;
constexpr int kWeightsChunk = 4096;

struct Plan {
  int rows, dim;     // of a core: block rows, padded head
  int nrb;
  bool tc, wide, split;
  int workers;
  size_t part_floats, ml_floats, score_floats;
  size_t bytes() const { return (part_floats + ml_floats + score_floats) * 4; }
};

Plan make_plan(const ptj_kv_cache& c, const ptj_new_tokens& t, const PagedRows& rows, bool weights) {
  Plan pl = {};
  const int64_t R = t.heads / c.kv_heads * t.tokens;
  pl.wide = paged_rows_aligned(c);
  pl.tc = c.dtype == PTJ_BF16 && pl.wide && c.d_head <= 128;
  if (pl.tc) {
    pl.dim = c.d_head <= 64 ? 64 : 128;
    pl.rows = R <= 8 ? 8 : 16;
  } else if (!pl.wide) {
    pl.dim = 256;
    pl.rows = 1;
  } else if (c.dtype == PTJ_BF16) {
    pl.dim = 256;
    pl.rows = R <= 1 ? 1 : 4;
  } else {
    pl.dim = c.d_head <= 32 ? 32 : (c.d_head <= 64 ? 64 : (c.d_head <= 128 ? 128 : 256));
    pl.rows = R <= 1 ? 1 : (pl.dim == 256 || R <= 4 ? 4 : 8);
  }
  pl.nrb = static_cast<int>(ceil_div(R, pl.rows));
  pl.split = rows.capacity > kDirectKeys || (weights && pl.nrb > 1);
  pl.workers = kWorkersPerSm * kNumSMs;
  if (pl.split) {
    pl.part_floats = static_cast<size_t>(pl.workers) * 2 * pl.rows * (pl.dim + 2);
    if (weights) pl.ml_floats = static_cast<size_t>(c.batch * c.kv_heads) * pl.nrb * pl.rows * 2;
  }
  if (weights) pl.score_floats = static_cast<size_t>(c.batch * c.kv_heads * R) * rows.capacity;
  pl.part_floats = (pl.part_floats + 3) / 4 * 4;
  pl.ml_floats = (pl.ml_floats + 3) / 4 * 4;
  return pl;
}

template <typename E, typename Core>
int launch(const DecodeAttn& d, const Plan& pl, cudaStream_t st) {
  if (!pl.split) {
    launch_k(attn_decode_kernel<E, Core, false>, d.B * d.Hk * d.nrb, kThreads, 0, st, d);
    PTJ_CHECK_LAUNCH();
    return PTJ_OK;
  }
  launch_k(attn_decode_kernel<E, Core, true>, d.workers, kThreads, 0, st, d);
  PTJ_CHECK_LAUNCH();
  const int64_t rows = static_cast<int64_t>(d.B) * d.Hk * d.R;
  const int64_t chunks = d.scores == nullptr ? 1 : ceil_div(d.rows.capacity, kWeightsChunk);
  const int64_t blocks = rows + (d.scores == nullptr ? 0 : static_cast<int64_t>(d.B) * d.Hk * chunks);
  if (blocks > 0x7fffffff) return PTJ_ERR_BAD_SHAPE;
  launch_k(attn_join_kernel<E, Core>, static_cast<int>(blocks), kJoinThreads, d.scores == nullptr ? 0 : d.R * 8, st, d,
           static_cast<int>(rows), kWeightsChunk, static_cast<int>(chunks));
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}

int dispatch(const DecodeAttn& d, const Plan& pl, int dtype, cudaStream_t st) {
  using B = __nv_bfloat16;
  if (pl.tc) {
    if (pl.dim == 64) return pl.rows == 8 ? launch<B, CoreTc<64, 1>>(d, pl, st) : launch<B, CoreTc<64, 2>>(d, pl, st);
    return pl.rows == 8 ? launch<B, CoreTc<128, 1>>(d, pl, st) : launch<B, CoreTc<128, 2>>(d, pl, st);
  }
  if (!pl.wide) return dtype == PTJ_BF16 ? launch<B, CoreFma<B, 1, 32, 8, 1>>(d, pl, st) : launch<float, CoreFma<float, 1, 32, 8, 1>>(d, pl, st);
  if (dtype == PTJ_BF16)
    return pl.rows == 1 ? launch<B, CoreFma<B, 8, 32, 1, 1>>(d, pl, st) : launch<B, CoreFma<B, 8, 32, 1, 4>>(d, pl, st);
  switch (pl.dim) {
    case 32:
      return pl.rows == 1 ? launch<float, CoreFma<float, 4, 8, 1, 1>>(d, pl, st)
                          : (pl.rows == 4 ? launch<float, CoreFma<float, 4, 8, 1, 4>>(d, pl, st) : launch<float, CoreFma<float, 4, 8, 1, 8>>(d, pl, st));
    case 64:
      return pl.rows == 1 ? launch<float, CoreFma<float, 4, 16, 1, 1>>(d, pl, st)
                          : (pl.rows == 4 ? launch<float, CoreFma<float, 4, 16, 1, 4>>(d, pl, st) : launch<float, CoreFma<float, 4, 16, 1, 8>>(d, pl, st));
    case 128:
      return pl.rows == 1 ? launch<float, CoreFma<float, 4, 32, 1, 1>>(d, pl, st)
                          : (pl.rows == 4 ? launch<float, CoreFma<float, 4, 32, 1, 4>>(d, pl, st) : launch<float, CoreFma<float, 4, 32, 1, 8>>(d, pl, st));
    default:
      return pl.rows == 1 ? launch<float, CoreFma<float, 4, 32, 2, 1>>(d, pl, st) : launch<float, CoreFma<float, 4, 32, 2, 4>>(d, pl, st);
  }
}

int check_decode(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, PagedRows& rows) {
  int rc = make_paged_rows(cache, rows);
  if (rc == PTJ_OK) rc = check_new_tokens(*cache, tokens, true, false);
  if (rc == PTJ_OK && tokens->heads / cache->kv_heads * tokens->tokens > kMaxRows) rc = PTJ_ERR_BAD_SHAPE;
  return rc;
}

}  // namespace
}  // namespace ptj

using namespace ptj;

extern "C" size_t ptj_attn_decode_workspace_bytes(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, int with_weights) {
  PagedRows rows;
  if (check_decode(cache, tokens, rows) != PTJ_OK) return 0;
  return make_plan(*cache, *tokens, rows, with_weights != 0).bytes();
}

extern "C" int ptj_attn_decode(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, float p, const float* weights,
                               float* weights_out, int64_t weights_ld, void* workspace, size_t workspace_bytes, void* stream) {
  DecodeAttn d = {};
  int rc = check_decode(cache, tokens, d.rows);
  if (rc != PTJ_OK) return rc;
  if (!(p >= 0.f && p <= 1.f) || (weights && !weights_out) || (weights_out && weights_ld < d.rows.capacity)) return PTJ_ERR_BAD_SHAPE;
  const Plan pl = make_plan(*cache, *tokens, d.rows, weights_out != nullptr);
  if (static_cast<int64_t>(cache->batch) * cache->kv_heads * pl.nrb > 0x7fffffff) return PTJ_ERR_BAD_SHAPE;
  if (ptj_device_check() != PTJ_OK || (d.rows.fault = tc::fault_word()) == nullptr) return PTJ_ERR_DEVICE;
  if (pl.bytes() > 0) {
    if (!workspace || workspace_bytes < pl.bytes()) return PTJ_ERR_WORKSPACE;
    if (!aligned16(workspace)) return PTJ_ERR_MISALIGNED;
  }
  const int64_t Hk = cache->kv_heads, T = tokens->tokens;
  if (tokens->k) {
    if (!pl.wide || (view_aligned(tokens->k, tokens->k_strides, *cache, Hk, T) && view_aligned(tokens->v, tokens->v_strides, *cache, Hk, T))) {
      d.kn = static_cast<const char*>(tokens->k);
      d.vn = static_cast<const char*>(tokens->v);
    } else if ((rc = ptj_kv_append(cache, tokens, stream)) != PTJ_OK) {  // rows that the kernel could not read 16 bytes at a time
      return rc;
    }
  }
  const int64_t es = static_cast<int64_t>(dtype_size(cache->dtype));
  d.lengths = cache->lengths;
  d.counts = tokens->counts;
  d.q = static_cast<const char*>(tokens->q);
  d.k = static_cast<char*>(cache->k);
  d.v = static_cast<char*>(cache->v);
  d.out = static_cast<char*>(tokens->out);
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = tokens->q_strides[i] * es;
    d.os[i] = tokens->o_strides[i] * es;
    d.kns[i] = tokens->k_strides[i] * es;
    d.vns[i] = tokens->v_strides[i] * es;
  }
  float* ws = static_cast<float*>(workspace);
  d.part = ws;
  d.part_ml = ws + static_cast<size_t>(pl.split ? pl.workers : 0) * 2 * pl.rows * pl.dim;
  d.ml = ws + pl.part_floats;
  d.scores = weights_out == nullptr ? nullptr : ws + pl.part_floats + pl.ml_floats;
  d.scores_ld = d.rows.capacity;
  d.weights = weights;
  d.weights_out = weights_out;
  d.weights_ld = weights_ld;
  d.scale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(cache->d_head)));
  d.keep = 1.f - p;
  d.B = static_cast<int>(cache->batch);
  d.Hk = static_cast<int>(Hk);
  d.G = static_cast<int>(tokens->heads / Hk);
  d.T = static_cast<int>(T);
  d.D = static_cast<int>(cache->d_head);
  d.R = d.G * d.T;
  d.nrb = pl.nrb;
  d.workers = pl.workers;
  d.least = kLeastTiles;
  d.q_wide = view_aligned(tokens->q, tokens->q_strides, *cache, tokens->heads, T);
  d.out_wide = cache->d_head % (16 / es) == 0 && view_aligned(tokens->out, tokens->o_strides, *cache, tokens->heads, T);
  return dispatch(d, pl, cache->dtype, static_cast<cudaStream_t>(stream));
}
