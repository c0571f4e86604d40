// Attention of new tokens over a paged key-value cache: the list of work, the ring of keys and values, joining of pieces.
//
// out = softmax(q K^T / sqrt(d)) V for the R = group * tokens query rows that share a key head. Every key and value is read once
// and multiplied with a handful of rows: memory bounds it, so the kernels are built to keep copies in flight and to share them out
// evenly.
//
// The keys of a segment (sequence, key head, block of rows) are taken in steps of KS = 4 to 16. Two ways to share them out:
//
// * One block per segment, its 8 or 16 warps taking steps in turn and joining their sums in shared memory: one launch, no second
//   pass, for short caches and for few segments.
// * All steps of the call form one list in which lengths, known on the device only, no longer matter, and every warp of the GPU
//   takes an equal stretch of it. A warp that holds all steps of a segment writes its output; pieces of a segment (at most two
//   per warp) go to the workspace with their reference exponent and sum and are joined, in order, by a second kernel.
//
// Results do not depend on timing. A warp owns a ring of steps in shared memory that cp.async fills ahead of the arithmetic, across
// segments; nothing but the warp itself waits for it. Sums are kept relative to a reference exponent that only moves when a
// score outgrows it by more than 2^8, so that a step costs one vote instead of a reduction over lanes.
#pragma once
#include "kv_cache.cuh"

namespace ptj {

constexpr int kDecJoinThreads = 256;
constexpr float kDecLazy = 8.f;
constexpr int kDecSplitWarps = 4;

struct DecodeAttn {
  PagedRows rows;
  const int32_t *lengths, *counts;
  const char *q, *kn, *vn;   // queries, new rows (NULL: in the pages already)
  char *k, *v, *out;
  int64_t qs[3], os[3], kns[3], vns[3];  // bytes
  const float* weights;
  float* weights_out;
  int64_t weights_ld, scores_ld;
  float *part, *part_ml;     // pieces: [warps][2][prows][kDim], [..][2] reference exponent and sum
  float* ml;                 // [segments][prows][2] of segments that one warp did
  int64_t* starts;           // [B + 1]: place of each sequence's first step in the list; steps of a warp's stretch
  float* scores;             // [batch * key heads][R][scores_ld], log2 units; NULL without weights
  float scale, keep;         // log2(e) / sqrt(d); 1 - p
  int B, Hk, G, T, D, R;
  int nrb, prows;            // blocks of rows, rows of a block that exist
  int workers, least;        // warps that share the list; steps that one takes at least
  int wide, q_wide, out_wide;  // 16-byte accesses are aligned: pools and new rows, queries, output
};

struct DecodePlan {
  int rows, dim, es;   // of a core: block rows, padded head, bytes of an element
  int nrb, prows;
  bool split;
  int workers;
  size_t part, part_ml, ml, starts, scores;  // bytes
  size_t bytes() const { return part + part_ml + ml + starts + scores; }
};
// workers of the split form and keys of a step of the core that takes these (0: there is none)
int decode_tc_blocks(int dim, int rows);
int decode_fma_blocks(int dim, int rows, int es);
int launch_decode_tc(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st);
int launch_decode_fma(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st);

namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float base_of(float ref) { return ref == -INFINITY ? 0.f : ref; }
// factor of sums relative to `ref` when they are taken relative to m; sums without any score above -inf are zero (or NaN)
__device__ __forceinline__ float rebase(float ref, float m) { return ref == -INFINITY ? 1.f : ex2(ref - m); }

// What a warp works on: one sequence, key head and block of rows
struct Segment {
  int b, h, rb;
  int n, first;  // keys, position of the first new token
  int count;
  const int32_t* table;
  __device__ __forceinline__ void set_sequence(const DecodeAttn& p, int seq) {
    b = seq;
    n = p.rows.length(p.lengths, b);
    count = p.rows.count(p.counts, p.T, b);
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
  // scores of row r, and the next row's behind them
  __device__ __forceinline__ float* score_row(const DecodeAttn& p, int r) const {
    return p.scores + ((static_cast<int64_t>(b) * p.Hk + h) * p.R + r) * p.scores_ld;
  }
  __device__ __forceinline__ const char* q_row(const DecodeAttn& p, int r) const {
    return p.q + b * p.qs[0] + (h * p.G + r / p.T) * p.qs[1] + (r % p.T) * p.qs[2];
  }
};

// n: 16, or 0 to fill the destination with zeros (nothing is read then)
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, int n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
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
// not place and keys behind the last one become zeros. New rows are taken from where they are and put into their pages.
template <int KS, int RB>
struct Fetcher {
  static constexpr int PIECES = RB / 16, ROWS = PIECES >= 32 ? 1 : 32 / PIECES, COLS = PIECES >= 32 ? PIECES / 32 : 1;
  int row0, c0;      // this lane's first row and piece
  uint32_t to;       // its place in a step
  bool paged, dense; // a step lies in one page; its rows lie one behind the other
  __device__ __forceinline__ void init(const DecodeAttn& p) {
    const int lane = threadIdx.x & 31;
    row0 = PIECES >= 32 ? 0 : lane / PIECES;
    c0 = PIECES >= 32 ? lane : lane % PIECES;
    to = row0 * RB + ((c0 ^ swizzle(row0)) << 4);
    paged = p.wide && p.rows.page_size % KS == 0;
    dense = p.rows.slot_stride[0] == RB && p.rows.slot_stride[1] == RB;
  }
  // sub: number of the step in its sequence
  __device__ __forceinline__ void fetch(const DecodeAttn& p, const Segment& sg, int sub, uint8_t* stage) const {
    const int j0 = sub * KS;
    if (!paged || j0 + KS > sg.first) {
      mixed(p, sg, j0, stage);
      return;
    }
    int64_t page;
    int slot;
    const bool on = p.rows.locate(sg.table, j0, page, slot);
    if ((threadIdx.x & 31) == 0) *present_word<KS, RB>(stage) = on ? (1u << KS) - 1u : 0u;
    if (!on) page = slot = 0;  // (nothing is read)
    const char* k = p.k + p.rows.offset(0, page, sg.h, slot);
    const char* v = p.v + p.rows.offset(1, page, sg.h, slot);
    if (dense) rows<true>(p, k + (row0 * RB + c0 * 16), v + (row0 * RB + c0 * 16), on, tc::smem_u32(stage));
    else rows<false>(p, k + row0 * p.rows.slot_stride[0] + c0 * 16, v + row0 * p.rows.slot_stride[1] + c0 * 16, on, tc::smem_u32(stage));
  }
  template <bool DENSE>
  __device__ __forceinline__ void rows(const DecodeAttn& p, const char* k, const char* v, bool on, uint32_t stage) const {
    const int64_t ks = ROWS * p.rows.slot_stride[0], vs = ROWS * p.rows.slot_stride[1];
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
      const int n = on && (c0 + 32 * x) * 16 < p.rows.row_bytes ? 16 : 0;
      const char *kr = k + 512 * x, *vr = v + 512 * x;
#pragma unroll
      for (int i = 0; i < KS; i += ROWS) {
        const uint32_t dst = stage + ((to ^ (swizzle(i) << 4)) + i * RB + 512 * x);
        copy16(dst, DENSE ? kr + i * RB : kr, n);
        copy16(dst + KS * RB, DENSE ? vr + i * RB : vr, n);
        if (!DENSE) {
          kr += ks;
          vr += vs;
        }
      }
    }
  }
  // a step that is not all in one page, or holds new keys or the last one (arguments by value: nothing of the caller's is
  // forced into memory)
  static __device__ __noinline__ void mixed(const DecodeAttn& p, const Segment sg, int j0, uint8_t* stage) {
    const int lane = threadIdx.x & 31, row0 = PIECES >= 32 ? 0 : lane / PIECES, c0 = PIECES >= 32 ? lane : lane % PIECES;
    uint32_t present = 0;
#pragma unroll 1
    for (int i = 0; i < KS; i += ROWS) {
      const int r = i + row0, j = j0 + r;
      int64_t page = 0;
      int slot = 0;
      const bool on = j < sg.n && p.rows.locate(sg.table, j, page, slot);
      const bool fresh = on && j >= sg.first && p.kn != nullptr;
      const unsigned lanes = __ballot_sync(0xffffffffu, on);
#pragma unroll
      for (int k = 0; k < ROWS; ++k) present |= (lanes >> (k * (PIECES >= 32 ? 0 : PIECES)) & 1u) << (i + k);
      if (!on) page = slot = 0;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        char* at = (kv == 0 ? p.k : p.v) + p.rows.offset(kv, page, sg.h, slot);
        const int64_t* s = kv == 0 ? p.kns : p.vns;
        const char* src = fresh ? (kv == 0 ? p.kn : p.vn) + sg.b * s[0] + sg.h * s[1] + (j - sg.first) * s[2] : at;
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
          const int c = c0 + 32 * x;
          const int left = on ? p.rows.row_bytes - c * 16 : 0;  // bytes of the row from this piece on
          uint8_t* dst = stage + (kv * KS + r) * RB + ((c ^ swizzle(r)) << 4);
          if (p.wide) {
            copy16(tc::smem_u32(dst), src + c * 16, left > 0 ? 16 : 0);
            if (fresh && left > 0 && sg.rb == 0) *reinterpret_cast<uint4*>(at + c * 16) = *reinterpret_cast<const uint4*>(src + c * 16);
          } else {  // rows that are not on 16-byte boundaries: by 2 bytes (elements are whole numbers of them)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint16_t val = 2 * e < left ? *reinterpret_cast<const uint16_t*>(src + c * 16 + 2 * e) : 0;
              *reinterpret_cast<uint16_t*>(dst + 2 * e) = val;
              if (fresh && 2 * e < left && sg.rb == 0) *reinterpret_cast<uint16_t*>(at + c * 16 + 2 * e) = val;
            }
          }
        }
      }
    }
    if ((threadIdx.x & 31) == 0) *present_word<KS, RB>(stage) = present;
  }
};

// Sum over the rows of a key of exp2(score - reference) / sum for keys [j0, j1) of a sequence's key head, onto the accumulated
// weights. row_ml(r): reference exponent and reciprocal sum of row r.
template <int N, typename F>
__device__ __forceinline__ void add_weights(const DecodeAttn& p, const Segment& sg, int j0, int j1, F&& row_ml) {
  const int64_t bh = static_cast<int64_t>(sg.b) * p.Hk + sg.h;
  const float* in = p.weights == nullptr ? nullptr : p.weights + bh * p.weights_ld;
  float* out = p.weights_out + bh * p.weights_ld;
  constexpr int U = 4;
  for (int jj = j0 + threadIdx.x; jj < j1; jj += N * U) {
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jj + u * N;
      w[u] = j < j1 && j < sg.first && in != nullptr ? in[j] : 0.f;
    }
    for (int r = 0; r < p.R; ++r) {
      if (sg.limit(p, r) < 0) continue;
      const float2 ml = row_ml(r);
      const float base = base_of(ml.x);
      const float* s = p.scores + (bh * p.R + r) * p.scores_ld;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jj + u * N;
        if (j < j1) w[u] = fmaf(ex2(s[j] - base), ml.y, w[u]);
      }
    }
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

// ---- a block per segment -------------------------------------------------------------------------------------------------
template <typename E, typename Core>
__global__ void __launch_bounds__(Core::kDirectWarps * 32, 1)
attn_decode_direct_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  constexpr int NW = Core::kDirectWarps, LD = Core::kDim + 4, D = Core::kDepth;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float ml[NW][Core::kRows][2], fac[NW][Core::kRows], fin[Core::kRows][2];
  const int tid = threadIdx.x, warp = tid >> 5;
  const int hr = blockIdx.x % (p.Hk * p.nrb);
  Segment sg;
  sg.set_sequence(p, blockIdx.x / (p.Hk * p.nrb));
  sg.h = hr / p.nrb;
  sg.rb = hr % p.nrb;
  uint8_t* ring = smem + warp * ring_bytes<Core>();
  const int steps = steps_of<Core>(sg.n);
  Fetcher<Core::KS, Core::kRowBytes> fetcher;
  fetcher.init(p);
#pragma unroll 1
  for (int i = 0; i < D - 1; ++i) {
    if (warp + i * NW < steps) fetcher.fetch(p, sg, warp + i * NW, ring + i * stage_bytes<Core>());
    cp_async_commit();
  }
  Core core;
  core.init(p, sg);
  int slot = 0, free_slot = D - 1;
  for (int s = warp; s < steps; s += NW) {
    cp_async_wait<D - 2>();
    __syncwarp();  // the step is there for all lanes, and all have left the one that is refilled
    const int ahead = s + (D - 1) * NW;
    if (ahead < steps) fetcher.fetch(p, sg, ahead, ring + free_slot * stage_bytes<Core>());
    cp_async_commit();
    core.step(p, sg, s, ring + slot * stage_bytes<Core>());
    slot = slot + 1 == D ? 0 : slot + 1;
    free_slot = free_slot + 1 == D ? 0 : free_slot + 1;
  }
  cp_async_wait<0>();
  __syncthreads();
  // the warps' sums over the rings
  float* os = reinterpret_cast<float*>(smem);
  core.emit([&](int r, int d, const float4& x, float ref, float sum, bool first) {
    *reinterpret_cast<float4*>(os + (warp * Core::kRows + r) * LD + d) = x;
    if (first) {
      ml[warp][r][0] = ref;
      ml[warp][r][1] = sum;
    }
  });
  __syncthreads();
  if (tid < Core::kRows) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[w][tid][0]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      fac[w][tid] = rebase(ml[w][tid][0], m);
      l = fmaf(fac[w][tid], ml[w][tid][1], l);
    }
    fin[tid][0] = m;
    fin[tid][1] = 1.f / l;
  }
  __syncthreads();
  const int rows = min(Core::kRows, p.R - sg.rb * Core::kRows);
  for (int i = tid; i < rows * (Core::kDim / 4); i += NW * 32) {
    const int r = i / (Core::kDim / 4), d = i % (Core::kDim / 4) * 4, row = sg.rb * Core::kRows + r;
    if (d >= p.D) continue;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (sg.limit(p, row) >= 0) {
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(os + (w * Core::kRows + r) * LD + d);
        const float f = fac[w][r];
        x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
      }
      x = scaled(x, p.keep * fin[r][1]);
    }
    store_out<E>(p, sg, row, d, x);
  }
  if (p.scores != nullptr)  // (one block of rows: the host sees to it; the scores are this block's)
    add_weights<NW * 32>(p, sg, 0, sg.n, [&](int r) { return make_float2(fin[r][0], fin[r][1]); });
}

// ---- an equal stretch of the list per warp ----------------------------------------------------------------------------------
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {  // (32 bits where they do: a tenth of the time)
  return ((a | b) >> 31) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
__device__ __forceinline__ int64_t steps_per_worker(const DecodeAttn& p, int64_t total) {
  const int64_t q = divide(total * p.Hk * p.nrb + p.workers - 1, p.workers);
  return q > p.least ? q : p.least;
}

// A place in the list: the segment and the step in it; `left` steps of the stretch from here on.
template <typename Core>
struct Cursor {
  Segment sg;
  int s, steps, left;
  // one step on; false: the stretch ends. `last` says that the step left was its segment's last in the stretch.
  __device__ __forceinline__ bool segment_ends() const { return s + 1 == steps || left == 1; }
  __device__ __forceinline__ void advance(const DecodeAttn& p) {
    --left;
    if (++s < steps || left == 0) return;
    s = 0;
    if (++sg.rb < p.nrb) return;
    sg.rb = 0;
    if (++sg.h < p.Hk) return;
    sg.h = 0;
    do sg.set_sequence(p, sg.b + 1); while (sg.n == 0);  // (steps are left: a sequence that has some follows)
    steps = steps_of<Core>(sg.n);
  }
};

template <typename E, typename Core>
__global__ void __launch_bounds__(kDecSplitWarps * 32, Core::kBlocks)
attn_decode_split_kernel(const __grid_constant__ DecodeAttn p) {
  grid_dep_sync();
  constexpr int NW = kDecSplitWarps, N = NW * 32, D = Core::kDepth;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t tot[NW], start_s[NW][2];
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
  const int64_t q = steps_per_worker(p, total);
  // the thread whose sequences hold the first step of a warp's stretch looks for its sequence
  int64_t acc = before;
  for (int b = b0; b < b1; ++b) {
    const int64_t t = steps_of<Core>(p.rows.length(p.lengths, b));
    if (blockIdx.x == 0) p.starts[b] = acc * heads;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int64_t at = (static_cast<int64_t>(blockIdx.x) * NW + w) * q;
      if (at >= acc * heads && at < (acc + t) * heads) {
        start_s[w][0] = b;
        start_s[w][1] = acc * heads;
      }
    }
    acc += t;
  }
  if (blockIdx.x == 0 && tid == 0) p.starts[p.B] = q;
  __syncthreads();
  const int64_t worker = static_cast<int64_t>(blockIdx.x) * NW + warp, range0 = worker * q;
  Cursor<Core> cur;
  cur.left = static_cast<int>(min(q, all - range0));
  if (range0 >= all) return;
  cur.sg.set_sequence(p, static_cast<int>(start_s[warp][0]));
  cur.steps = steps_of<Core>(cur.sg.n);
  const int64_t in_seq = range0 - start_s[warp][1], hr = divide(in_seq, cur.steps);
  cur.s = static_cast<int>(in_seq - hr * cur.steps);
  cur.sg.h = static_cast<int>(hr) / p.nrb;
  cur.sg.rb = static_cast<int>(hr) - cur.sg.h * p.nrb;
  uint8_t* ring = smem + warp * ring_bytes<Core>();
  Fetcher<Core::KS, Core::kRowBytes> fetcher;
  fetcher.init(p);
  Cursor<Core> ahead = cur;
#pragma unroll 1
  for (int i = 0; i < D - 1; ++i) {
    if (ahead.left > 0) {
      fetcher.fetch(p, ahead.sg, ahead.s, ring + i * stage_bytes<Core>());
      ahead.advance(p);
    }
    cp_async_commit();
  }
  int slot = 0, free_slot = D - 1;
  bool first_piece = true;
  for (;;) {  // segments
    const int s_first = cur.s;
    Core core;
    core.init(p, cur.sg);
    for (;;) {
      cp_async_wait<D - 2>();
      __syncwarp();  // the step is there for all lanes, and all have left the one that is refilled
      if (ahead.left > 0) {
        fetcher.fetch(p, ahead.sg, ahead.s, ring + free_slot * stage_bytes<Core>());
        ahead.advance(p);
      }
      cp_async_commit();
      core.step(p, cur.sg, cur.s, ring + slot * stage_bytes<Core>());
      slot = slot + 1 == D ? 0 : slot + 1;
      free_slot = free_slot + 1 == D ? 0 : free_slot + 1;
      if (cur.segment_ends()) break;
      ++cur.s;
      --cur.left;
    }
    const bool whole = s_first == 0 && cur.s + 1 == cur.steps;
    const int64_t piece = worker * 2 + (first_piece ? 0 : 1);
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
        to[0] = ref;
        to[1] = sum;
      }
    });
    first_piece = false;
    if (cur.left == 1) break;
    cur.advance(p);
  }
  cp_async_wait<0>();
}

// Pieces of a segment: which warps hold some, and where.
struct Pieces {
  int64_t w0, w1, t0, q;
  __device__ __forceinline__ Pieces(const DecodeAttn& p, const Segment& sg, int rb, int steps) {
    q = p.starts[p.B];
    t0 = p.starts[sg.b] + (static_cast<int64_t>(sg.h) * p.nrb + rb) * steps;
    w0 = divide(t0, q);
    w1 = divide(t0 + steps - 1, q);
  }
  // a segment that starts where a warp's stretch starts is its first piece, as is one that started before
  __device__ __forceinline__ int64_t row(const DecodeAttn& p, int64_t w, int rr) const {
    return (w * 2 + (t0 <= w * q ? 0 : 1)) * p.prows + rr;
  }
};

// Blocks [0, rows_blocks): WPR warps per query row, joined where several warps hold pieces of it, zero where there is nothing to
// attend. The others: the weights of a stretch of one sequence's and key head's keys.
template <typename E, typename Core, int WPR>
__global__ void __launch_bounds__(kDecJoinThreads)
attn_decode_join_kernel(const __grid_constant__ DecodeAttn p, int rows_blocks, int chunk, int chunks) {
  grid_dep_sync();
  constexpr int N = kDecJoinThreads, PER = N / 32 / WPR;            // rows of a block
  constexpr int kVecs = Core::kDim / 4, kGroups = WPR * 32 / kVecs > 0 ? WPR * 32 / kVecs : 1, kReach = kVecs > WPR * 32 ? kVecs / (WPR * 32) : 1;
  const int tid = threadIdx.x, lane = tid & 31;
  Segment sg;
  if (blockIdx.x < rows_blocks) {
    __shared__ float2 sums[PER][kGroups];
    __shared__ float4 part_s[PER][kGroups][kVecs];
    const int slot = tid / (WPR * 32), t = tid % (WPR * 32);
    const int64_t id = static_cast<int64_t>(blockIdx.x) * PER + slot;  // row of all
    const bool there = id < static_cast<int64_t>(p.B) * p.Hk * p.R;
    const int bh = there ? static_cast<int>(id / p.R) : 0, r = there ? static_cast<int>(id % p.R) : 0;
    sg.set_sequence(p, bh / p.Hk);
    sg.h = bh % p.Hk;
    sg.rb = r / Core::kRows;
    const int rr = r % Core::kRows, grp = t / kVecs, steps = steps_of<Core>(sg.n);
    const bool some = there && sg.limit(p, r) >= 0 && steps > 0;
    const Pieces pc(p, sg, sg.rb, steps > 0 ? steps : 1);
    const bool split = some && pc.w0 != pc.w1;
    float m = -INFINITY, l = 0.f;
    float4 x[kReach];
#pragma unroll
    for (int k = 0; k < kReach; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (split) {
      // every group of lanes takes every kGroups-th piece, relative to a maximum of its own
#pragma unroll 4
      for (int64_t w = pc.w0 + grp; w <= pc.w1; w += kGroups) m = fmaxf(m, p.part_ml[pc.row(p, w, rr) * 2]);
#pragma unroll 4
      for (int64_t w = pc.w0 + grp; w <= pc.w1; w += kGroups) {
        const int64_t s = pc.row(p, w, rr);
        const float f = rebase(p.part_ml[s * 2], m);
        l = fmaf(f, p.part_ml[s * 2 + 1], l);
#pragma unroll
        for (int k = 0; k < kReach; ++k) {
          const int d = (t % kVecs + k * WPR * 32) * 4;
          if (d < p.D) {
            const float4 y = *reinterpret_cast<const float4*>(p.part + s * Core::kDim + d);
            x[k].x = fmaf(f, y.x, x[k].x); x[k].y = fmaf(f, y.y, x[k].y); x[k].z = fmaf(f, y.z, x[k].z); x[k].w = fmaf(f, y.w, x[k].w);
          }
        }
      }
    }
    if constexpr (kGroups > 1) {
      part_s[slot][grp][t % kVecs] = x[0];
      if (t % kVecs == 0) sums[slot][grp] = make_float2(m, l);
      if constexpr (WPR > 1) __syncthreads();
      else __syncwarp();
      if (grp > 0) return;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) m = fmaxf(m, sums[slot][k].x);
      l = 0.f;
      x[0] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const float f = rebase(sums[slot][k].x, m);
        const float4 y = part_s[slot][k][t % kVecs];
        l = fmaf(f, sums[slot][k].y, l);
        x[0].x = fmaf(f, y.x, x[0].x); x[0].y = fmaf(f, y.y, x[0].y); x[0].z = fmaf(f, y.z, x[0].z); x[0].w = fmaf(f, y.w, x[0].w);
      }
    }
    if (!there || (some && !split)) return;
#pragma unroll
    for (int k = 0; k < kReach; ++k) {
      const int d = (t % kVecs + k * WPR * 32) * 4;
      if (d < p.D) store_out<E>(p, sg, r, d, some ? scaled(x[k], p.keep / l) : make_float4(0.f, 0.f, 0.f, 0.f));
    }
    return;
  }
  const int id = (blockIdx.x - rows_blocks) / chunks;
  sg.set_sequence(p, id / p.Hk);
  sg.h = id % p.Hk;
  const int j0 = (blockIdx.x - rows_blocks) % chunks * chunk, steps = steps_of<Core>(sg.n);
  if (j0 >= sg.n) return;
  extern __shared__ float2 row_ml[];  // [R]
  for (int r = tid >> 5; r < p.R; r += N / 32) {  // a warp per row
    const int rb = r / Core::kRows, rr = r % Core::kRows;
    const Pieces pc(p, sg, rb, steps);
    float m = -INFINITY, l = 0.f;
    if (pc.w0 == pc.w1) {
      const float* s = p.ml + ((static_cast<int64_t>(id) * p.nrb + rb) * p.prows + rr) * 2;
      m = s[0];
      l = s[1];
    } else {
      for (int64_t w = pc.w0 + lane; w <= pc.w1; w += 32) m = fmaxf(m, p.part_ml[pc.row(p, w, rr) * 2]);
      m = warp_max(m);
      for (int64_t w = pc.w0 + lane; w <= pc.w1; w += 32) {
        const float* s = p.part_ml + pc.row(p, w, rr) * 2;
        l = fmaf(rebase(s[0], m), s[1], l);
      }
      l = warp_sum(l);
    }
    if (lane == 0) row_ml[r] = make_float2(m, 1.f / l);
  }
  __syncthreads();
  add_weights<N>(p, sg, j0, min(j0 + chunk, sg.n), [&](int r) { return row_ml[r]; });
}

// ---- host -------------------------------------------------------------------------------------------------------------------
constexpr int kWeightsChunk = 1024;

template <typename K>
bool set_smem(K kernel, int bytes) {
  if (bytes <= 48 * 1024) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess) return true;
  (void)cudaGetLastError();
  return false;
}

template <typename E, typename Core>
int launch_decode(const DecodeAttn& d, bool split, cudaStream_t st) {
  if (!split) {
    constexpr int ring = Core::kDirectWarps * ring_bytes<Core>(), sums = Core::kDirectWarps * Core::kRows * (Core::kDim + 4) * 4;
    constexpr int smem = ring > sums ? ring : sums;
    if (!set_smem(attn_decode_direct_kernel<E, Core>, smem)) return PTJ_ERR_LAUNCH;
    launch_k(attn_decode_direct_kernel<E, Core>, d.B * d.Hk * d.nrb, Core::kDirectWarps * 32, smem, st, d);
    PTJ_CHECK_LAUNCH();
    return PTJ_OK;
  }
  constexpr int smem = kDecSplitWarps * ring_bytes<Core>();
  // rows that many warps hold pieces of are joined by a block each: where there are few rows
  const int64_t rows = static_cast<int64_t>(d.B) * d.Hk * d.R;
  const bool few = rows <= 2 * kNumSMs;
  const int64_t row_blocks = few ? rows : ceil_div(rows, kDecJoinThreads / 32);
  const int64_t chunks = d.scores == nullptr ? 1 : ceil_div(d.rows.capacity, kWeightsChunk);
  const int64_t blocks = row_blocks + (d.scores == nullptr ? 0 : static_cast<int64_t>(d.B) * d.Hk * chunks);
  if (blocks > 0x7fffffff) return PTJ_ERR_BAD_SHAPE;
  if (!set_smem(attn_decode_split_kernel<E, Core>, smem)) return PTJ_ERR_LAUNCH;
  launch_k(attn_decode_split_kernel<E, Core>, d.workers / kDecSplitWarps, kDecSplitWarps * 32, smem, st, d);
  PTJ_CHECK_LAUNCH();
  const auto join = few ? attn_decode_join_kernel<E, Core, kDecJoinThreads / 32> : attn_decode_join_kernel<E, Core, 1>;
  launch_k(join, static_cast<int>(blocks), kDecJoinThreads, d.scores == nullptr ? 0 : d.R * 8, st, d, static_cast<int>(row_blocks),
           kWeightsChunk, static_cast<int>(chunks));
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}

}  // namespace
}  // namespace ptj
