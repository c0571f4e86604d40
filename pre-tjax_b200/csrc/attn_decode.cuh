// Attention of new tokens over a paged key-value cache: the list of work, the ring of keys and values, joining of pieces.
//
// out = softmax(q K^T / sqrt(d)) V for the R = group * tokens query rows that share a key head, in blocks of 1 to 32 rows. Every key
// and value is read once per block of rows and multiplied with a handful of them: memory bounds it, so the kernels are built to keep
// copies in flight and to share them out evenly. (A block goes over all keys of its sequence, the ones that a prompt's earlier rows
// do not attend among them.)
//
// The keys of a segment (sequence, key head, block of rows) are taken in steps of KS = 4 to 16. Two ways to share them out:
//
// * A cluster of one to eight blocks per segment, their warps taking steps in turn and joining their sums in shared memory: one launch
//   and no second pass, unless there are too few segments to fill the GPU that way or sequences are so long that one of them
//   alone could keep its cluster busy long after the others.
// * All steps of the call form one list in which lengths, known on the device only, no longer matter. Every warp of the GPU takes
//   an equal large stretch, three quarters of the list, and then small ones as long as there are some: some SMs get a third less
//   of the memory's rate than others (with equal stretches alone the average SM was busy for 157 k cycles, the last for 207 k:
//   128k keys of 8 heads of 128). A segment within one stretch is written by its warp; pieces of others (at most two per stretch)
//   go to the workspace with their reference exponent and sum and are joined, in order, by a second kernel.
//
// Who computes a stretch does not matter to it: results do not depend on timing. A warp owns a ring of steps in shared memory that
// cp.async fills ahead of the arithmetic, across segments; nothing but the warp itself waits for it. Sums are kept relative to a
// reference exponent that only moves when a score outgrows it by more than 2^8, so that a step costs one vote instead of a reduction
// over lanes.
#pragma once
#include <atomic>
#include <type_traits>

#include "cluster.cuh"
#include "kv_cache.cuh"

namespace ptj {

constexpr int kDecJoinThreads = 256;
constexpr float kDecLazy = 8.f;
constexpr int kDecWarps = 4;
constexpr int kDecDynamicBatch = 512;  // small stretches are cut where this many sequences' places fit into shared memory

struct DecodeAttn {
  PagedRows rows;
  const int32_t *lengths, *counts;
  const char *q, *kn, *vn;   // queries, new rows (NULL: in the pages already)
  char *k, *v, *out;
  int64_t qs[3], os[3], kns[3], vns[3];  // bytes
  const float* weights;
  float* weights_out;
  int64_t weights_ld, scores_ld;
  float *part, *part_ml;     // pieces: [stretches][2][prows][kDim], [..][2] reference exponent and sum
  float* ml;                 // [segments][prows][2] of segments that lie in one stretch
  int64_t* starts;           // [B + 2]: place of each sequence's first step in the list; steps of a large and of a small stretch
  float* scores;             // [batch * key heads][R][scores_ld], log2 units; NULL without weights
  float scale, unscale, keep;  // log2(e) / sqrt(d), its reciprocal; 1 - p
  int B, Hk, G, T, D, R;
  int nrb, prows;            // blocks of rows, rows of a block that exist
  unsigned int* next;        // the next of the small stretches to be taken (zero at the start)
  int workers, small, least; // warps that share the list; number of small stretches at most; steps of a stretch at least
  int wide, q_wide, out_wide;  // 16-byte accesses are aligned: pools and new rows, queries, output
};

struct DecodePlan {
  int rows, dim, es;   // of a core: block rows, padded head, bytes of an element
  int nrb, prows;
  bool split, wide;    // wide: many rows, attn_decode_wide.cu
  int cluster;         // blocks per segment
  int workers, small;
  size_t part, part_ml, ml, starts, scores;  // bytes
  size_t bytes() const { return part + part_ml + ml + starts + scores; }
};
// blocks that an SM holds of the core that takes these
int decode_tc_blocks(int dim, int rows);
int decode_fma_blocks();
int decode_wide_blocks();
int launch_decode_tc(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st);
int launch_decode_fma(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st);
int launch_decode_wide(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st);

namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Reference exponent before any score above -inf: exponentials of -inf relative to it are zero, and so are such sums.
constexpr float kNoRef = -3.402823466e38f;
// factor of sums relative to `ref` when they are taken relative to m
__device__ __forceinline__ float rebase(float ref, float m) { return ex2(ref - m); }

// What a warp works on: one sequence, key head and block of rows
struct Segment {
  int b, h, rb;
  int n, first;  // keys, position of the first new token
  int count;
  const int32_t* table;
  __device__ __forceinline__ void set_sequence(const DecodeAttn& p, int seq) {
    b = seq;
    p.rows.extent(p.lengths, p.counts, p.T, b, n, count);
    first = n - count;
    table = p.rows.table + b * p.rows.table_ld;
  }
  // last key that row r (of all R) attends, -1: none
  __device__ __forceinline__ int limit(const DecodeAttn& p, int r) const {
    const int t = r % p.T;
    return r < p.R && t < count ? first + t : -1;
  }
  __device__ __forceinline__ int64_t index(const DecodeAttn& p) const {
    return (static_cast<int64_t>(b) * p.Hk + h) * p.nrb + rb;
  }
  // What row r's sums are divided by, sum being that of its exponentials. Where that is zero: scores that are all -inf have no softmax,
  // 0 / 0 makes NaN of the row; a row none of whose keys exists attends nothing, 0 / inf makes zeros of it and of its weights.
  __device__ __forceinline__ float divisor(const DecodeAttn& p, int r, float sum) const {
    return sum != 0.f || any_key(p, r) ? sum : INFINITY;
  }
  __device__ __forceinline__ bool any_key(const DecodeAttn& p, int r) const {
    const int last = limit(p, r), pages = last < 0 ? 0 : p.rows.page_of(last) + 1;
    for (int i = 0; i < pages; ++i)
      if (static_cast<unsigned int>(table[i]) < static_cast<unsigned int>(p.rows.pages)) return true;
    return false;
  }
  // scores of row r, and the next row's behind them
  __device__ __forceinline__ float* score_row(const DecodeAttn& p, int r) const {
    return p.scores + ((static_cast<int64_t>(b) * p.Hk + h) * p.R + r) * p.scores_ld;
  }
  __device__ __forceinline__ const char* q_row(const DecodeAttn& p, int r) const {
    return p.q + b * p.qs[0] + (h * p.G + r / p.T) * p.qs[1] + (r % p.T) * p.qs[2];
  }
};

__device__ __forceinline__ void copy16(uint32_t dst, const char* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// on false: the destination is filled with zeros and nothing is read. (A byte count instead of the predicate takes several
// instructions where it is not a constant.)
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const char* src, bool on) {
  asm volatile("{\n\t.reg .pred off;\n\tsetp.eq.u32 off, %2, 0;\n\tcp.async.cg.shared.global [%0], [%1], 16, off;\n\t}"
               ::"r"(dst), "l"(src), "r"(static_cast<uint32_t>(on)) : "memory");
}

// Place of 16-byte piece c of row r of a step: c ^ swizzle(r). Pieces are swapped so that both ways the tensor-core fragments read a
// step (a few pieces of eight consecutive rows, a piece of every second row) touch all banks. swizzle(a ^ b) is swizzle(a) ^
// swizzle(b), so a lane's addresses of all its rows are few registers and constants apart.
__host__ __device__ constexpr int swizzle(int r) { return (((r >> 1) & 3) << 1) ^ ((r & 1) << 2); }

template <int KS, int RB>
__device__ __forceinline__ uint32_t* present_word(uint8_t* stage) { return reinterpret_cast<uint32_t*>(stage + 2 * KS * RB); }
template <int KS, int RB>
__device__ __forceinline__ uint32_t present_keys(const uint8_t* stage) { return *reinterpret_cast<const uint32_t*>(stage + 2 * KS * RB); }

// Copies steps: KS rows of keys, KS rows of values, of RB bytes each, and a word that says which of them exist. Rows the table does
// not place and keys behind the last one become zeros. New rows are taken from where they are; store_new puts them into their
// pages. Short calls are bound by instruction fetches as much as by anything else: one inlined copy of the common case per kernel,
// everything else out of line.
template <int KS, int RB>
struct Fetcher {
  static constexpr int PIECES = RB / 16, ROWS = PIECES >= 32 ? 1 : 32 / PIECES, COLS = PIECES >= 32 ? PIECES / 32 : 1;
  int row0, c0;   // this lane's first row and piece
  uint32_t to;    // its place in a step
  bool dense;     // a step's rows lie in one page
  // Pages of 32 steps to come, one per lane: a look-up in front of every step would be the longest wait of all (800 cycles).
  int ids, base;  // base: the first of them, counted in steps that this warp takes
  const char *k, *v;  // this lane's place in slot row0 of page 0 of the key head
  __device__ __forceinline__ void look_up(const DecodeAttn& p, const int32_t* table, int sub, int stride, int number) {
    const int page = p.rows.page_of((sub + (threadIdx.x & 31) * stride) * KS);
    ids = page < p.rows.capacity_pages ? table[page] : -1;
    base = number;
  }
  __device__ __forceinline__ void init(const DecodeAttn& p) {
    const int lane = threadIdx.x & 31;
    row0 = PIECES >= 32 ? 0 : lane / PIECES;
    c0 = PIECES >= 32 ? lane : lane % PIECES;
    to = row0 * RB + ((c0 ^ swizzle(row0)) << 4);
    dense = p.wide && p.rows.page_size % KS == 0;
  }
  __device__ __forceinline__ void set_head(const DecodeAttn& p, int h) {
    k = p.k + p.rows.offset(0, 0, h, row0) + c0 * 16;
    v = p.v + p.rows.offset(1, 0, h, row0) + c0 * 16;
  }
  // Number of a sequence's first steps that are dense and hold no new key.
  __device__ __forceinline__ int plain_steps(const Segment& sg) const { return dense ? max(sg.first, 0) / KS : 0; }
  // A plain step. sub: its number in its sequence; number: how many this warp took before it, of those that look_up covers.
  // false: its page does not exist, the general way has to take it.
  __device__ __forceinline__ bool plain(const DecodeAttn& p, int sub, int number, uint8_t* stage) const {
    const int page = __shfl_sync(0xffffffffu, ids, number - base);
    if (static_cast<unsigned int>(page) >= static_cast<unsigned int>(p.rows.pages)) return false;
    const int j0 = sub * KS;
    const int slot = p.rows.page_shift >= 0 ? j0 & (p.rows.page_size - 1) : j0 - p.rows.page_of(j0) * p.rows.page_size;
    if ((threadIdx.x & 31) == 0) *present_word<KS, RB>(stage) = (1u << KS) - 1u;
    const char *kr = k + (page * p.rows.page_stride[0] + slot * p.rows.slot_stride[0]);
    const char *vr = v + (page * p.rows.page_stride[1] + slot * p.rows.slot_stride[1]);
    const int64_t ks = ROWS * p.rows.slot_stride[0], vs = ROWS * p.rows.slot_stride[1];
    const uint32_t at = tc::smem_u32(stage);
#pragma unroll
    for (int i = 0; i < KS; i += ROWS) {
#pragma unroll
      for (int x = 0; x < COLS; ++x) {
        if ((c0 + 32 * x) * 16 >= p.rows.row_bytes) continue;  // (zero from the start)
        const uint32_t dst = at + ((to ^ (swizzle(i) << 4)) + i * RB + 512 * x);
        copy16(dst, kr + 512 * x);
        copy16(dst + KS * RB, vr + 512 * x);
      }
      kr += ks;
      vr += vs;
    }
    return true;
  }
  __device__ __forceinline__ void general(const DecodeAttn& p, const Segment& sg, int sub, uint8_t* stage) const {
    if (p.wide) mixed(p, sg, sub * KS, stage);
    else narrow(p, sg, sub * KS, stage);
  }
  // What lies behind narrower rows in a ring is zero: dense steps write their rows only.
  __device__ __forceinline__ void clear(const DecodeAttn& p, uint8_t* ring, int bytes) const {
    if (p.rows.row_bytes == RB) return;
    for (int i = (threadIdx.x & 31) * 16; i < bytes; i += 512) *reinterpret_cast<uint4*>(ring + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
  }
  // Rows here and there: lane r looks row r up, the others get its addresses from it. (Arguments by value: nothing of the caller's
  // is forced into memory.)
  static __device__ __noinline__ void mixed(const DecodeAttn& p, const Segment sg, int j0, uint8_t* stage) {
    const int lane = threadIdx.x & 31, row0 = PIECES >= 32 ? 0 : lane / PIECES, c0 = PIECES >= 32 ? lane : lane % PIECES;
    const int j = j0 + lane;
    int64_t page = 0;
    int slot = 0;
    const bool on = lane < KS && j < sg.n && p.rows.locate(sg.table, j, page, slot);
    const char *k = p.k, *v = p.v;
    if (on) {
      if (j >= sg.first && p.kn != nullptr) {
        k = p.kn + sg.b * p.kns[0] + sg.h * p.kns[1] + (j - sg.first) * p.kns[2];
        v = p.vn + sg.b * p.vns[0] + sg.h * p.vns[1] + (j - sg.first) * p.vns[2];
      } else {
        k += p.rows.offset(0, page, sg.h, slot);
        v += p.rows.offset(1, page, sg.h, slot);
      }
    }
    const uint32_t present = __ballot_sync(0xffffffffu, on);
    if (lane == 0) *present_word<KS, RB>(stage) = present;
    const uint32_t at = tc::smem_u32(stage) + row0 * RB;
#pragma unroll
    for (int i = 0; i < KS; i += ROWS) {
      const int r = i + row0;
      const char* kr = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(k), r));
      const char* vr = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v), r));
#pragma unroll
      for (int x = 0; x < COLS; ++x) {
        const int c = c0 + 32 * x;
        const bool there = (present >> r & 1u) && c * 16 < p.rows.row_bytes;
        const uint32_t dst = at + i * RB + ((c ^ swizzle(r)) << 4);
        copy16_or_zero(dst, kr + c * 16, there);
        copy16_or_zero(dst + KS * RB, vr + c * 16, there);
      }
    }
  }
  // Rows that are not on 16-byte boundaries: by 2 bytes (elements are whole numbers of them), nothing asynchronous.
  static __device__ __noinline__ void narrow(const DecodeAttn& p, const Segment sg, int j0, uint8_t* stage) {
    const int lane = threadIdx.x & 31;
    uint32_t present = 0;
    for (int r = 0; r < KS; ++r) {
      const int j = j0 + r;
      int64_t page = 0;
      int slot = 0;
      const bool on = j < sg.n && p.rows.locate(sg.table, j, page, slot);
      if (on) present |= 1u << r;
      for (int kv = 0; kv < 2; ++kv) {
        const char* src = nullptr;
        if (on) {
          const int64_t* s = kv == 0 ? p.kns : p.vns;
          src = j >= sg.first && p.kn != nullptr ? (kv == 0 ? p.kn : p.vn) + sg.b * s[0] + sg.h * s[1] + (j - sg.first) * s[2]
                                                 : (kv == 0 ? p.k : p.v) + p.rows.offset(kv, page, sg.h, slot);
        }
        for (int e = lane * 2; e < RB; e += 64) {
          const uint16_t val = on && e < p.rows.row_bytes ? *reinterpret_cast<const uint16_t*>(src + e) : 0;
          *reinterpret_cast<uint16_t*>(stage + (kv * KS + r) * RB + (((e >> 4) ^ swizzle(r)) << 4) + (e & 15)) = val;
        }
      }
    }
    if (lane == 0) *present_word<KS, RB>(stage) = present;
  }
  // Puts the new rows of a step that has arrived into their pages.
  __device__ __forceinline__ void store_new(const DecodeAttn& p, const Segment& sg, int sub, const uint8_t* stage) const {
    if (p.kn != nullptr && sg.rb == 0 && (sub + 1) * KS > sg.first) write_new(p, sg, sub * KS, stage);
  }
  static __device__ __noinline__ void write_new(const DecodeAttn& p, const Segment sg, int j0, const uint8_t* stage) {
    const int lane = threadIdx.x & 31, r0 = max(sg.first - j0, 0);
    uint32_t rows = present_keys<KS, RB>(stage) >> r0 << r0;
    int64_t page = 0;
    int slot = 0;
    if (lane < KS && (rows >> lane & 1u)) p.rows.locate(sg.table, j0 + lane, page, slot);  // lane r: row r
    const unsigned long long at[2] = {reinterpret_cast<unsigned long long>(p.k + p.rows.offset(0, page, sg.h, slot)),
                                      reinterpret_cast<unsigned long long>(p.v + p.rows.offset(1, page, sg.h, slot))};
    for (; rows != 0u; rows &= rows - 1u) {
      const int r = __ffs(rows) - 1;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        char* to = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, at[kv], r));
        const uint8_t* row = stage + (kv * KS + r) * RB;
        if (p.wide) {
          for (int c = lane; c * 16 < p.rows.row_bytes; c += 32)
            *reinterpret_cast<uint4*>(to + c * 16) = *reinterpret_cast<const uint4*>(row + ((c ^ swizzle(r)) << 4));
        } else {
          for (int e = lane * 2; e < p.rows.row_bytes; e += 64)
            *reinterpret_cast<uint16_t*>(to + e) = *reinterpret_cast<const uint16_t*>(row + (((e >> 4) ^ swizzle(r)) << 4) + (e & 15));
        }
      }
    }
  }
};

// Sum over the rows of a key of exp2(score - reference) / sum for keys [j0, j1) of a sequence's key head, onto the accumulated
// weights. row_ml(r): reference exponent and reciprocal sum of row r.
template <int N, int U, typename F>
__device__ __forceinline__ void add_weights(const DecodeAttn& p, const Segment& sg, int j0, int j1, F&& row_ml) {
  const int64_t bh = static_cast<int64_t>(sg.b) * p.Hk + sg.h;
  const float* in = p.weights == nullptr ? nullptr : p.weights + bh * p.weights_ld;
  float* out = p.weights_out + bh * p.weights_ld;
  for (int jj = j0 + threadIdx.x; jj < j1; jj += N * U) {
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jj + u * N;
      w[u] = j < j1 && j < sg.first && in != nullptr ? in[j] : 0.f;
    }
    // RB rows' scores are on their way at a time
    const auto rows = [&](auto rb) {
      constexpr int RB = decltype(rb)::value;
      for (int r0 = 0; r0 < p.R; r0 += RB) {
        float s[RB][U];
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int r = min(r0 + i, p.R - 1), j = min(jj + u * N, j1 - 1);
            s[i][u] = __ldcg(p.scores + (bh * p.R + r) * p.scores_ld + j);  // (other blocks' writes: not from L1)
          }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          if (r0 + i >= p.R || sg.limit(p, r0 + i) < 0) continue;
          const float2 ml = row_ml(r0 + i);
#pragma unroll
          for (int u = 0; u < U; ++u) w[u] = fmaf(ex2(s[i][u] - ml.x), ml.y, w[u]);
        }
      }
    };
    if (p.R < 4) rows(std::integral_constant<int, 1>{});
    else rows(std::integral_constant<int, 4>{});
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (jj + u * N < j1) out[jj + u * N] = w[u];
  }
}

template <typename E>
__device__ __forceinline__ void store_out(const DecodeAttn& p, const Segment& sg, int r, int d, const float4& x) {
  char* row = p.out + sg.b * p.os[0] + (sg.h * p.G + r / p.T) * p.os[1] + (r % p.T) * p.os[2];
  const float v[4] = {x.x, x.y, x.z, x.w};
  if (p.out_wide) {
    if (d >= p.D) return;
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
__device__ __forceinline__ float4 scaled(const float4& x, float f) { return make_float4(x.x * f, x.y * f, x.z * f, x.w * f); }

template <typename Core>
constexpr int stage_bytes() { return 2 * Core::KS * Core::kRowBytes + 16; }
template <typename Core>
constexpr int ring_bytes() { return Core::kDepth * stage_bytes<Core>(); }
template <typename Core>
__device__ __forceinline__ int steps_of(int n) { return (n + Core::KS - 1) / Core::KS; }

// A warp's steps s, s + stride, .. below `end` once more, one by one through one place, infinite values with care (Core::spoiled).
// Out of line: the loops that run ahead keep their registers.
template <typename Core>
__device__ __noinline__ Core steps_again(const DecodeAttn& p, const Segment sg, int s, int end, int stride, uint8_t* stage) {
  Fetcher<Core::KS, Core::kRowBytes> fetcher;
  Core core;
  core.init(p, sg);
  for (; s < end; s += stride) {
    __syncwarp();  // all lanes have left the step before
    fetcher.general(p, sg, s, stage);
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();
    core.template step<true>(p, sg, s, stage);
  }
  return core;
}

// ---- a cluster of blocks per segment -----------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned cluster_blocks() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 peer_float4(const float* p, unsigned rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(tc::mapa_shared(tc::smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 peer_float2(const float* p, unsigned rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(tc::mapa_shared(tc::smem_u32(p), rank)) : "memory");
  return v;
}

template <typename E, typename Core>
__global__ void __launch_bounds__(kDecWarps * 32, Core::kBlocks)
attn_decode_direct_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  constexpr int NW = kDecWarps, LD = Core::kDim + 4, D = Core::kDepth;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float ml[NW][Core::kRows][2], fac[NW][Core::kRows];
  __shared__ __align__(8) float top_s[Core::kRows][2];  // of the block: reference exponent, sum
  __shared__ float fin[Core::kRows][2];                 // of the cluster: reference exponent, reciprocal sum
  __shared__ float peer_fac[8][Core::kRows];            // factors of the blocks' sums
  const int tid = threadIdx.x, warp = tid >> 5;
  const unsigned C = cluster_blocks(), rank = tc::cluster_ctarank();
  const int seg = blockIdx.x / C, hr = seg % (p.Hk * p.nrb), b = seg / (p.Hk * p.nrb);
  const int stride = NW * static_cast<int>(C), s0 = static_cast<int>(rank) * NW + warp;
  Fetcher<Core::KS, Core::kRowBytes> fetcher;
  fetcher.look_up(p, p.rows.table + b * p.rows.table_ld, s0, stride, 0);  // (while the length is on its way)
  Segment sg;
  sg.set_sequence(p, b);
  sg.h = hr / p.nrb;
  sg.rb = hr % p.nrb;
  uint8_t* ring = smem + warp * ring_bytes<Core>();
  const int steps = steps_of<Core>(sg.n);
  fetcher.init(p);
  fetcher.set_head(p, sg.h);
  fetcher.clear(p, ring, ring_bytes<Core>());
  Core core;
  const int plain = fetcher.plain_steps(sg);
  core.init(p, sg);
  int slot = 0, free_slot = 0, number = 0;
#pragma unroll 1
  for (int s = s0 - (D - 1) * stride; s < steps; s += stride) {  // (D - 1 rounds ahead: steps to come are fetched only)
    if (s >= 0) {
      cp_async_wait<D - 2>();
      __syncwarp();  // the step is there for all lanes, and all have left the one that is refilled
    }
    const int ahead = s + (D - 1) * stride;
    if (ahead < steps) {
      if (number == fetcher.base + 32) fetcher.look_up(p, sg.table, ahead, stride, number);
      uint8_t* stage = ring + free_slot * stage_bytes<Core>();
      if (ahead >= plain || !fetcher.plain(p, ahead, number, stage)) fetcher.general(p, sg, ahead, stage);
      ++number;
    }
    cp_async_commit();
    free_slot = free_slot + 1 == D ? 0 : free_slot + 1;
    if (s < 0) continue;
    uint8_t* stage = ring + slot * stage_bytes<Core>();
    if (s >= plain) fetcher.store_new(p, sg, s, stage);
    core.template step<false>(p, sg, s, stage);
    slot = slot + 1 == D ? 0 : slot + 1;
  }
  cp_async_wait<0>();
  if constexpr (Core::kParts)
    if (core.spoiled()) core = steps_again<Core>(p, sg, s0, steps, stride, ring);
  __syncthreads();
  // the warps' sums over the rings, then the block's over the first warp's
  float* os = reinterpret_cast<float*>(smem);
  core.emit([&](int r, int d, const float4& x, float ref, float sum, bool first) {
    *reinterpret_cast<float4*>(os + (warp * Core::kRows + r) * LD + d) = x;
    if (first) {
      ml[warp][r][0] = ref;
      ml[warp][r][1] = sum;
    }
  });
  __syncthreads();
  const int rows = min(Core::kRows, p.R - sg.rb * Core::kRows);
  if (tid < rows) {
    float m = kNoRef, l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[w][tid][0]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      fac[w][tid] = rebase(ml[w][tid][0], m);
      l = fmaf(fac[w][tid], ml[w][tid][1], l);
    }
    top_s[tid][0] = m;
    top_s[tid][1] = l;
  }
  __syncthreads();
  for (int i = tid; i < rows * (Core::kDim / 4); i += NW * 32) {
    const int r = i / (Core::kDim / 4), d = i % (Core::kDim / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float4 y = *reinterpret_cast<const float4*>(os + (w * Core::kRows + r) * LD + d);
      const float f = fac[w][r];
      x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
    }
    *reinterpret_cast<float4*>(os + r * LD + d) = x;
  }
  if (C > 1) tc::cluster_sync_all();
  else __syncthreads();
  // (all reads of other blocks are issued before any of them is waited for: one latency, not one per block)
  if (tid < rows) {
    float2 v[8];
#pragma unroll
    for (unsigned k = 0; k < 8; ++k) v[k] = k < C ? peer_float2(top_s[tid], k) : make_float2(kNoRef, 0.f);
    float m = kNoRef, l = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, v[k].x);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = rebase(v[k].x, m);
      peer_fac[k][tid] = f;
      l = fmaf(f, v[k].y, l);
    }
    fin[tid][0] = m;
    fin[tid][1] = 1.f / sg.divisor(p, sg.rb * Core::kRows + tid, l);
  }
  // every block joins its share of the rows' elements
  const int pieces = rows * (Core::kDim / 4);
  for (int i0 = static_cast<int>(rank) * NW * 32; i0 < pieces; i0 += NW * 32 * static_cast<int>(C)) {
    const int i = i0 + tid, r = i / (Core::kDim / 4), d = i % (Core::kDim / 4) * 4, row = sg.rb * Core::kRows + r;
    const bool on = i < pieces && d < p.D;
    float4 y[8];
#pragma unroll
    for (unsigned k = 0; k < 8; ++k) y[k] = on && k < C ? peer_float4(os + r * LD + d, k) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (i0 == static_cast<int>(rank) * NW * 32) __syncthreads();  // the factors (the first round is every thread's)
    if (!on) continue;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (sg.limit(p, row) >= 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = k < static_cast<int>(C) ? peer_fac[k][r] : 0.f;
        x.x = fmaf(f, y[k].x, x.x); x.y = fmaf(f, y[k].y, x.y); x.z = fmaf(f, y[k].z, x.z); x.w = fmaf(f, y[k].w, x.w);
      }
      x = scaled(x, p.keep * fin[r][1]);
    }
    store_out<E>(p, sg, row, d, x);
  }
  __syncthreads();
  if (p.scores != nullptr) {  // (one block of rows: the host sees to it; the scores are this cluster's)
    const int per = (sg.n + static_cast<int>(C) - 1) / static_cast<int>(C), j0 = min(static_cast<int>(rank) * per, sg.n);
    add_weights<NW * 32, 4>(p, sg, j0, min(j0 + per, sg.n), [&](int r) { return make_float2(fin[r][0], fin[r][1]); });
  }
  if (C > 1) tc::cluster_sync_all();  // nobody leaves before its sums are read
}

// ---- stretches of the list ------------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {  // (32 bits where they do: a tenth of the time)
  return ((a | b) >> 31) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
// The list of `all` steps: `workers` large stretches of q1 steps, then small ones of q2.
struct Stretches {
  int64_t q1, q2, edge;
  int workers;
  __device__ __forceinline__ void plan(const DecodeAttn& p, int64_t all) {
    workers = p.workers;
    const int64_t share = divide(all, workers);
    q1 = p.small > 0 ? share - (share >> 2) : share + (share * workers < all);
    if (q1 < p.least) q1 = p.least;
    edge = q1 * workers;
    q2 = 1;
    if (p.small > 0) {
      const int64_t rest = all > edge ? all - edge : 0;
      q2 = divide(rest + p.small - 1, p.small);
      if (q2 < p.least) q2 = p.least;
    }
  }
  __device__ __forceinline__ void load(const DecodeAttn& p) {
    workers = p.workers;
    q1 = p.starts[p.B];
    q2 = p.starts[p.B + 1];
    edge = q1 * workers;
  }
  __device__ __forceinline__ int64_t begin(int64_t w) const { return w < workers ? w * q1 : edge + (w - workers) * q2; }
  __device__ __forceinline__ int64_t of(int64_t t) const { return t < edge ? divide(t, q1) : workers + divide(t - edge, q2); }
};

// A place in the list: the segment, the step in it, where this stretch leaves it, and the steps of the stretch behind that.
template <typename Core>
struct Cursor {
  Segment sg;
  int s, end, steps, left;
  __device__ __forceinline__ void bound(int n) {  // n steps of the stretch from here on
    end = min(steps, s + n);
    left = n - (end - s);
  }
  // to the stretch's next segment (left > 0)
  __device__ __forceinline__ void next_segment(const DecodeAttn& p) {
    s = 0;
    if (++sg.rb == p.nrb) {
      sg.rb = 0;
      if (++sg.h == p.Hk) {
        sg.h = 0;
        do sg.set_sequence(p, sg.b + 1); while (sg.n == 0);  // (steps are left: a sequence that has some follows)
        steps = steps_of<Core>(sg.n);
      }
    }
    bound(left);
  }
  // place `at` of the list, which lies in sequence b whose first step is at place `start`; n steps from there on
  __device__ __forceinline__ void set(const DecodeAttn& p, int b, int64_t start, int64_t at, int64_t n) {
    sg.set_sequence(p, b);
    steps = steps_of<Core>(sg.n);
    const int64_t hr = divide(at - start, steps);
    s = static_cast<int>(at - start - hr * steps);
    sg.h = static_cast<int>(hr) / p.nrb;
    sg.rb = static_cast<int>(hr) - sg.h * p.nrb;
    bound(static_cast<int>(n));
  }
};

// the last sequence that starts at or before a place (empty ones start where the next does)
__device__ __forceinline__ int sequence_at(const int64_t* first, int n, int64_t at) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= at) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename E, typename Core>
__global__ void __launch_bounds__(kDecWarps * 32, Core::kBlocks)
attn_decode_split_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  constexpr int NW = kDecWarps, N = NW * 32, D = Core::kDepth;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t tot[NW], start_s[NW], first_s[kDecDynamicBatch];
  __shared__ int seq_s[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // steps of all sequences, and of those before each thread's stretch of sequences
  const int per = (p.B + N - 1) / N, b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += steps_of<Core>(p.rows.length(p.lengths, b));
  int64_t incl = mine;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, x);
    if (lane >= x) incl += y;
  }
  if (lane == 31) tot[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += tot[w];
    total += tot[w];
  }
  const int64_t heads = static_cast<int64_t>(p.Hk) * p.nrb, all = total * heads;
  Stretches st;
  st.plan(p, all);
  // the thread whose sequences hold the first step of a warp's stretch looks for its sequence
  int64_t acc = before * heads;
  for (int b = b0; b < b1; ++b) {
    const int64_t t = steps_of<Core>(p.rows.length(p.lengths, b)) * heads;
    if (blockIdx.x == 0) p.starts[b] = acc;
    if (p.small > 0) first_s[b] = acc;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int64_t at = (static_cast<int64_t>(blockIdx.x) * NW + w) * st.q1;
      if (at >= acc && at < acc + t) {
        seq_s[w] = b;
        start_s[w] = acc;
      }
    }
    acc += t;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.starts[p.B] = st.q1;
    p.starts[p.B + 1] = st.q2;
  }
  __syncthreads();
  int64_t stretch = static_cast<int64_t>(blockIdx.x) * NW + warp;
  if (st.begin(stretch) >= all) return;
  Cursor<Core> cur;
  cur.set(p, seq_s[warp], start_s[warp], st.begin(stretch), min(st.q1, all - st.begin(stretch)));
  uint8_t* ring = smem + warp * ring_bytes<Core>();
  Fetcher<Core::KS, Core::kRowBytes> fetcher;
  fetcher.init(p);
  fetcher.clear(p, ring, ring_bytes<Core>());
  Cursor<Core> ahead = cur;
  unsigned int ticket = 0;  // lane 0: the small stretch that was taken
  int64_t following = -1;   // the stretch that `ahead` is in, when that is not `cur`'s
  bool asked = p.small == 0, over = asked;
  const int32_t* looked_up = nullptr;  // the sequence whose pages the lanes hold
  int fast = 0;  // steps of `ahead` below this one are plain, covered by look_up and nothing is to be done about what follows them
  // Fetches the step at `ahead` and moves it on, into the next small stretch where its own ends. That one is asked for two steps
  // before: the answer is there in time, and few stretches wait at a slow SM.
  auto fetch_ahead = [&](uint8_t* stage) {
    if (ahead.s < fast && fetcher.plain(p, ahead.s, ahead.s, stage)) {
      ++ahead.s;
      return;
    }
    if (ahead.s == ahead.end) {
      if (ahead.left > 0) {
        ahead.next_segment(p);
      } else {
        if (over) return;
        const int64_t w = st.workers + static_cast<int64_t>(__shfl_sync(0xffffffffu, ticket, 0)), at = st.begin(w);
        if (at >= all) {
          over = true;
          return;
        }
        following = w;
        const int b = sequence_at(first_s, p.B, at);
        ahead.set(p, b, first_s[b], at, min(st.q2, all - at));
        asked = false;
      }
      looked_up = nullptr;
    }
    if (looked_up == nullptr || ahead.s >= fetcher.base + 32) {
      looked_up = ahead.sg.table;
      fetcher.look_up(p, looked_up, ahead.s, 1, ahead.s);
      fetcher.set_head(p, ahead.sg.h);
    }
    if (!asked && ahead.left == 0 && ahead.s + 2 >= ahead.end) {
      if (lane == 0) ticket = atomicAdd(p.next, 1u);
      asked = true;
    }
    const int plain = fetcher.plain_steps(ahead.sg);
    if (ahead.s >= plain || !fetcher.plain(p, ahead.s, ahead.s, stage)) fetcher.general(p, ahead.sg, ahead.s, stage);
    ++ahead.s;
    fast = min(min(plain, fetcher.base + 32), !asked && ahead.left == 0 ? ahead.end - 2 : ahead.end);
  };
  int slot = 0, free_slot = 0, lead = D - 1;  // lead: steps to fetch before the first one is computed
  bool first_piece = true;
  for (;;) {  // segments
    const int s_first = cur.s, cur_plain = fetcher.plain_steps(cur.sg);
    Core core;
    core.init(p, cur.sg);
#pragma unroll 1
    for (;;) {
      if (lead == 0) {
        cp_async_wait<D - 2>();
        __syncwarp();  // the step is there for all lanes, and all have left the one that is refilled
      }
      fetch_ahead(ring + free_slot * stage_bytes<Core>());
      cp_async_commit();
      free_slot = free_slot + 1 == D ? 0 : free_slot + 1;
      if (lead > 0) {
        --lead;
        continue;
      }
      uint8_t* stage = ring + slot * stage_bytes<Core>();
      if (cur.s >= cur_plain) fetcher.store_new(p, cur.sg, cur.s, stage);
      core.template step<false>(p, cur.sg, cur.s, stage);
      slot = slot + 1 == D ? 0 : slot + 1;
      if (++cur.s == cur.end) break;
    }
    if constexpr (Core::kParts)  // (the place that is refilled next is free)
      if (core.spoiled()) core = steps_again<Core>(p, cur.sg, s_first, cur.s, 1, ring + free_slot * stage_bytes<Core>());
    const bool whole = s_first == 0 && cur.s == cur.steps;
    const int64_t piece = stretch * 2 + (first_piece ? 0 : 1);
    const int row0 = cur.sg.rb * Core::kRows;
    core.emit([&](int r, int d, const float4& x, float ref, float sum, bool first) {
      const int row = row0 + r;
      if (row >= p.R || d >= p.D) return;
      if (whole) {
        store_out<E>(p, cur.sg, row, d, cur.sg.limit(p, row) >= 0 ? scaled(x, p.keep / sum) : make_float4(0.f, 0.f, 0.f, 0.f));
      } else {
        *reinterpret_cast<float4*>(p.part + (piece * p.prows + r) * Core::kDim + d) = x;
      }
      if (first && (!whole || p.scores != nullptr)) {
        float* to = whole ? p.ml + (cur.sg.index(p) * p.prows + r) * 2 : p.part_ml + (piece * p.prows + r) * 2;
        *reinterpret_cast<float2*>(to) = make_float2(ref, sum);
      }
    });
    first_piece = false;
    if (cur.left > 0) {
      cur.next_segment(p);
      continue;
    }
    // A stretch ends. `ahead` is in the next one by now, if there is one: no stretch but the list's last is shorter than the ring.
    if (following < 0) break;
    stretch = following;
    following = -1;
    first_piece = true;
    const int64_t at = st.begin(stretch);
    const int b = sequence_at(first_s, p.B, at);
    cur.set(p, b, first_s[b], at, min(st.q2, all - at));
  }
  cp_async_wait<0>();
}

// Pieces of a segment: which stretches hold some, and where.
struct Pieces {
  int64_t w0, w1;
  int second;  // its piece of stretch w0 is that stretch's second
  __device__ __forceinline__ Pieces(const DecodeAttn& p, const Segment& sg, int rb, int steps) {
    Stretches st;
    st.load(p);
    const int64_t t0 = p.starts[sg.b] + (static_cast<int64_t>(sg.h) * p.nrb + rb) * steps;
    w0 = st.of(t0);
    w1 = st.of(t0 + steps - 1);
    // a segment that starts where a stretch starts is its first piece, as is one that started before
    second = t0 > st.begin(w0);
  }
  __device__ __forceinline__ int64_t row(const DecodeAttn& p, int64_t w, int rr) const {
    return (w * 2 + (w == w0 ? second : 0)) * p.prows + rr;
  }
};

// WPR warps per query row, joined where several stretches hold pieces of it, zero where there is nothing to attend.
template <typename E, typename Core, int WPR>
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : kDecJoinThreads)
attn_decode_join_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  constexpr int PER = (WPR > 8 ? WPR : kDecJoinThreads / 32) / WPR, VL = Core::kDim / 32;  // rows of a block, elements of a lane
  const int tid = threadIdx.x, lane = tid & 31;
  Segment sg;
  __shared__ float2 ml_s[PER][WPR];
  __shared__ float part_s[PER][WPR][WPR > 1 ? Core::kDim : 1];
  const int slot = tid / (WPR * 32), wr = tid / 32 % WPR;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * PER + slot;  // row of all
  const bool there = id < static_cast<int64_t>(p.B) * p.Hk * p.R;
  const int bh = there ? static_cast<int>(id / p.R) : 0, r = there ? static_cast<int>(id % p.R) : 0;
  sg.set_sequence(p, bh / p.Hk);
  sg.h = bh % p.Hk;
  sg.rb = r / Core::kRows;
  const int rr = r % Core::kRows, steps = steps_of<Core>(sg.n), d = lane * VL;
  const bool some = there && sg.limit(p, r) >= 0 && steps > 0;
  const Pieces pc(p, sg, sg.rb, steps > 0 ? steps : 1);
  const bool split = some && pc.w0 != pc.w1;
  float m = kNoRef, l = 0.f;
  float x[VL];
#pragma unroll
  for (int k = 0; k < VL; ++k) x[k] = 0.f;
  if (split) {
    for (int64_t base = pc.w0 + wr; base <= pc.w1; base += 32 * WPR) {
      const int64_t w = base + lane * WPR;  // this lane's piece
      float2 ml = make_float2(kNoRef, 0.f);
      if (w <= pc.w1) ml = *reinterpret_cast<const float2*>(p.part_ml + pc.row(p, w, rr) * 2);
      const float top = fmaxf(warp_max(ml.x), m), old = rebase(m, top), f = w <= pc.w1 ? rebase(ml.x, top) : 0.f;
      m = top;
      l = fmaf(l, old, warp_sum(f * ml.y));
#pragma unroll
      for (int k = 0; k < VL; ++k) x[k] *= old;
      const int n = static_cast<int>(min(static_cast<int64_t>(32), (pc.w1 - base) / WPR + 1));
      constexpr int U = VL <= 4 ? 16 : 8;  // pieces that are read at a time
      for (int i0 = 0; i0 < n; i0 += U) {
        float y[U][VL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float* at = p.part + pc.row(p, base + min(i0 + u, n - 1) * WPR, rr) * Core::kDim + d;
          if constexpr (VL == 2) {
            *reinterpret_cast<float2*>(y[u]) = *reinterpret_cast<const float2*>(at);
          } else {
#pragma unroll
            for (int k = 0; k < VL; k += 4) *reinterpret_cast<float4*>(y[u] + k) = *reinterpret_cast<const float4*>(at + k);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float fi = __shfl_sync(0xffffffffu, f, min(i0 + u, 31));
          if (i0 + u >= n) continue;
#pragma unroll
          for (int k = 0; k < VL; ++k) x[k] = fmaf(fi, y[u][k], x[k]);
        }
      }
    }
  }
  if constexpr (WPR > 1) {
#pragma unroll
    for (int k = 0; k < VL; ++k) part_s[slot][wr][d + k] = x[k];
    if (lane == 0) ml_s[slot][wr] = make_float2(m, l);
    __syncthreads();
    if (wr > 0) return;
#pragma unroll
    for (int k = 0; k < WPR; ++k) m = fmaxf(m, ml_s[slot][k].x);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < VL; ++k) x[k] = 0.f;
#pragma unroll 8
    for (int k = 0; k < WPR; ++k) {
      const float f = rebase(ml_s[slot][k].x, m);
      l = fmaf(f, ml_s[slot][k].y, l);
#pragma unroll
      for (int e = 0; e < VL; ++e) x[e] = fmaf(f, part_s[slot][k][d + e], x[e]);
    }
  }
  if (!there || (some && !split && sg.any_key(p, r))) return;
  // (a row that lies in one stretch is there already; where it has no key it is looked at here, the pass has no registers to spare)
  if (some) l = sg.divisor(p, r, l);
  if (some && p.scores != nullptr && lane == 0)
    *reinterpret_cast<float2*>(p.ml + (sg.index(p) * p.prows + rr) * 2) = make_float2(m, l);
  const float f = p.keep / l;
  char* row = p.out + sg.b * p.os[0] + (sg.h * p.G + r / p.T) * p.os[1] + (r % p.T) * p.os[2];
#pragma unroll
  for (int k = 0; k < VL; ++k)
    if (d + k < p.D) Elem<E>::store(reinterpret_cast<E*>(row) + d + k, some ? x[k] * f : 0.f);
}

// The weights of kWeightsChunk of one sequence's and key head's keys, from the rows' statistics that the join left.
constexpr int kWeightsChunk = 1024;

__global__ void __launch_bounds__(kDecJoinThreads)
attn_decode_weights_kernel(const __grid_constant__ DecodeAttn p, int rows_of_block, int chunks) {
  grid_dep_sync();
  extern __shared__ float2 row_ml[];  // [R]
  const int tid = threadIdx.x, id = blockIdx.x / chunks;
  const float* ml = p.ml + static_cast<int64_t>(id) * p.nrb * p.prows * 2;
  for (int r = tid; r < p.R; r += kDecJoinThreads) {
    const float2 x = *reinterpret_cast<const float2*>(ml + (r / rows_of_block * p.prows + r % rows_of_block) * 2);
    row_ml[r] = make_float2(x.x, 1.f / x.y);
  }
  Segment sg;
  sg.set_sequence(p, id / p.Hk);
  sg.h = id % p.Hk;
  __syncthreads();
  const int j0 = blockIdx.x % chunks * kWeightsChunk;
  if (j0 < sg.n)
    add_weights<kDecJoinThreads, kWeightsChunk / kDecJoinThreads>(p, sg, j0, min(j0 + kWeightsChunk, sg.n), [&](int r) { return row_ml[r]; });
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// Needed once per kernel and device (each kernel is launched with one size), not per launch.
template <auto Kernel>
bool set_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    (void)cudaGetLastError();
    return false;
  }
  const uint64_t bit = 1ull << dev;
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    (void)cudaGetLastError();
    return false;
  }
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// Joins the pieces that the stretches left and, where they are wanted, forms the weights.
template <typename E, typename Core>
int launch_join(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st) {
  // warps that join a row: by the pieces to be expected of a segment
  const int64_t rows = static_cast<int64_t>(d.B) * d.Hk * d.R, pieces = (d.workers + d.small) / (static_cast<int64_t>(d.B) * d.Hk * d.nrb);
  const int wpr = pieces <= 3 ? 1 : (pieces <= 32 ? 4 : 16), threads = wpr == 16 ? 512 : kDecJoinThreads;
  const int64_t blocks = ceil_div(rows * wpr * 32, threads);
  if (blocks > 0x7fffffff) return PTJ_ERR_BAD_SHAPE;
  const auto join = wpr == 1 ? attn_decode_join_kernel<E, Core, 1> : (wpr == 4 ? attn_decode_join_kernel<E, Core, 4> : attn_decode_join_kernel<E, Core, 16>);
  launch_k(join, static_cast<int>(blocks), threads, 0, st, d);
  PTJ_CHECK_LAUNCH();
  if (d.scores == nullptr) return PTJ_OK;
  const int64_t chunks = ceil_div(d.rows.capacity, kWeightsChunk);
  if (chunks * d.B * d.Hk > 0x7fffffff) return PTJ_ERR_BAD_SHAPE;
  launch_k(attn_decode_weights_kernel, static_cast<int>(chunks * d.B * d.Hk), kDecJoinThreads, d.R * 8, st, d, pl.rows, static_cast<int>(chunks));
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}

template <typename E, typename Core>
int launch_decode(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st) {
  constexpr int ring = kDecWarps * ring_bytes<Core>(), sums = kDecWarps * Core::kRows * (Core::kDim + 4) * 4;
  if (!pl.split) {
    constexpr int smem = ring > sums ? ring : sums;
    if (!set_smem<attn_decode_direct_kernel<E, Core>>(smem)) return PTJ_ERR_LAUNCH;
    launch_cluster_k(attn_decode_direct_kernel<E, Core>, dim3(static_cast<unsigned>(d.B * d.Hk * d.nrb * pl.cluster)), kDecWarps * 32,
                     pl.cluster, smem, st, d);
    PTJ_CHECK_LAUNCH();
    return PTJ_OK;
  }
  if (d.small > 0 && cudaMemsetAsync(d.next, 0, 4, st) != cudaSuccess) {
    (void)cudaGetLastError();
    return PTJ_ERR_LAUNCH;
  }
  if (!set_smem<attn_decode_split_kernel<E, Core>>(ring)) return PTJ_ERR_LAUNCH;
  launch_k(attn_decode_split_kernel<E, Core>, d.workers / kDecWarps, kDecWarps * 32, ring, st, d);
  PTJ_CHECK_LAUNCH();
  return launch_join<E, Core>(d, pl, st);
}

}  // namespace
}  // namespace ptj
