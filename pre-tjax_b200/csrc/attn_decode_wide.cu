// Attention of new tokens over a paged cache, bf16, many query rows per key head (drafted tokens of shared heads): tcgen05.
//
// The kernels with operands in registers run out of registers beyond 16 to 24 rows (attn_decode_tc.cu). Here a block takes 128 keys
// at a time: S^T = K Q^T (128 keys x 32 rows) and O^T += V^T P^T (128 elements x 64 columns: 32 rows' first bf16 parts of the
// probabilities and their second ones) run from shared memory into tensor memory, so that two threads share a key: each has 16 of
// its scores, exponentials and parts, half a row of the product's operand. (One thread with all 32 was a third slower: four warps
// do not hide the chain of a tile.) Keys stand in the 128-byte-swizzled layout with the head
// elements contiguous, which is K-major for the first product and MN-major for the second; cp.async writes it row by row, since
// rows lie in pages. Heads of 64 elements fill half of the second product's rows, what the other half multiplies is not read.
//
// Bound by the chain of a tile (keys arrive, product, scores, parts, product); two blocks per SM run theirs against each other, the
// next tile's keys are on their way from the first product on and its values from the second. 4 x 8 caches of 30k keys of 128,
// 32 rows: 114 us (192 with operands in registers, in two passes; floor 75).
#include "attn_decode.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

using namespace tc;

constexpr int kWideThreads = 256, kWideBlocks = 2;
constexpr uint32_t kWideTmem = 128, kColO = 32;  // columns: 32 of scores, 64 of outputs

template <int DP>
struct CoreWide {
  static constexpr int KS = 128, kRows = 32, kDim = DP;
  static constexpr int DB = DP / 64;  // blocks of 64 elements
  static constexpr int kK = 0, kV = kK + DB * 16384, kP = kV + DB * 16384, kQ = kP + 16384, kX = kQ + DB * 4096;
  static constexpr int kSmem = kX + kRows * DP * 4 + 1024;  // (rounded up to 1024 bytes at run time)
};

// 16-byte piece c of row r of an operand with rows of DP elements in blocks of 64 (`block` bytes each)
__device__ __forceinline__ int place(int r, int c, int block) { return (c >> 3) * block + r * 128 + (((c & 7) ^ (r & 7)) << 4); }

// A value that is not finite makes NaN of sums that it does not belong to: of rows that do not attend it, times their zeros, and of
// those that do, times the second part of a probability (zero, or of either sign). No sum that it meets stays finite, so it is looked
// for once, in the sums of a segment; where there was one, the segment runs again, and of each tile this takes such values out and
// multiplies them by the first parts of the rows that attend them. Out of line: inside the loop it made calls 4 % longer.
template <int DP>
__device__ __noinline__ void take_out(uint8_t* smem, const int* limit_s, int j0) {
  using Core = CoreWide<DP>;
  const int tid = threadIdx.x;
  __syncthreads();  // all values and parts are there
  bool bad = false;
  if (tid < 128)
    for (int c = 0; c < DP / 8; ++c) {
      const uint4 x = *reinterpret_cast<const uint4*>(smem + Core::kV + place(tid, c, 16384));
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
    }
  if (!__syncthreads_or(bad)) return;
  float* x = reinterpret_cast<float*>(smem + Core::kX);  // [rows][DP]
  if (tid < DP)  // a thread per element: this one's column of x, and of the values
    for (int k = 0; k < 128; ++k) {
      uint16_t* v = reinterpret_cast<uint16_t*>(smem + Core::kV + place(k, tid >> 3, 16384)) + (tid & 7);
      if ((*v & 0x7f80u) != 0x7f80u) continue;
      const float val = __uint_as_float(static_cast<uint32_t>(*v) << 16);
      for (int r = 0; r < Core::kRows; ++r)
        if (j0 + k <= limit_s[r]) {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(smem + Core::kP + place(k, r >> 3, 0)) + (r & 7);
          x[r * DP + tid] += __uint_as_float(static_cast<uint32_t>(*h) << 16) * val;
        }
      *v = 0;
    }
}

template <int DP>
__global__ void __launch_bounds__(kWideThreads, kWideBlocks)
attn_decode_wide_kernel(const __grid_constant__ DecodeAttn p) {
  using Core = CoreWide<DP>;
  constexpr int N = kWideThreads, NW = N / 32, R = Core::kRows, RH = R / 2, CH = DP / 8, RPI = 32 / CH;  // pieces of a row, rows of a copy
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  __shared__ uint64_t bars[2];  // scores, outputs
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ __align__(16) float over_s[R], ref_s[R], fac_s[R], red[NW][RH];
  __shared__ uint8_t there_s[2][128];
  __shared__ int limit_s[R];
  __shared__ int64_t tot[NW], start_s;
  __shared__ int seq_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 0) {
    tmem_alloc(&tmem_slot, kWideTmem);
    tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(&bars[0], 1);
    mbar_init(&bars[1], 1);
    fence_barrier_init();
    abort_flag = 0;
  }
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot, lanes = static_cast<uint32_t>(warp & 3) * 32u << 16;
  const int key = (warp & 3) * 32 + lane, r0 = (warp >> 2) * RH;  // this thread's key of a tile (and element of outputs), its rows
  const AbortCtx ctx{&abort_flag, p.rows.fault};
  grid_dep_sync();  // nothing above touches global memory

  // steps of all sequences, and of those before each thread's
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
  const int64_t worker = blockIdx.x, range0 = st.begin(worker);
  int64_t acc = before * heads;
  for (int b = b0; b < b1; ++b) {
    const int64_t t = steps_of<Core>(p.rows.length(p.lengths, b)) * heads;
    if (blockIdx.x == 0) p.starts[b] = acc;
    if (range0 >= acc && range0 < acc + t) {
      seq_s = b;
      start_s = acc;
    }
    acc += t;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.starts[p.B] = st.q1;
    p.starts[p.B + 1] = st.q2;
  }
  __syncthreads();

  uint32_t scores_done = 0, outputs_done = 0;  // parities
  if (range0 < all) {
    Cursor<Core> cur;
    cur.set(p, seq_s, start_s, range0, min(st.q1, all - range0));
    bool first_piece = true, careful = false;  // careful: the segment's sums are not finite, it runs again
    for (;;) {  // segments
      const Segment& sg = cur.sg;
      // the rows' queries
      {
        const int r = tid >> 3, row = sg.rb * R + r, limit = sg.limit(p, row);
        const char* q = limit >= 0 ? sg.q_row(p, row) : nullptr;
#pragma unroll
        for (int c = tid & 7; c < CH; c += 8) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (q != nullptr && p.q_wide && c * 8 + 8 <= p.D) {
            x = *reinterpret_cast<const uint4*>(q + c * 16);
          } else if (q != nullptr) {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(q);
            auto at = [&](int d) { return d < p.D ? static_cast<uint32_t>(e[d]) : 0u; };
            x = make_uint4(at(8 * c) | at(8 * c + 1) << 16, at(8 * c + 2) | at(8 * c + 3) << 16, at(8 * c + 4) | at(8 * c + 5) << 16,
                           at(8 * c + 6) | at(8 * c + 7) << 16);
          }
          *reinterpret_cast<uint4*>(smem + Core::kQ + place(r, c, 4096)) = x;
        }
        if ((tid & 7) == 0) {
          limit_s[r] = limit;
          over_s[r] = -INFINITY;
          ref_s[r] = kNoRef;
        }
      }
      float sum[RH];
#pragma unroll
      for (int i = 0; i < RH; ++i) sum[i] = 0.f;
      if (careful)  // products with values that are not finite
        for (int i = tid; i < R * DP; i += N) reinterpret_cast<float*>(smem + Core::kX)[i] = 0.f;

      // A warp copies 16 keys; lane i < 16 has the address of the i-th key's row, lane 16 + i that of its value's. NULL: absent.
      const int mine16 = warp * 16 + (lane & 15), kv = lane >> 4;
      const char* at = nullptr;
      auto page_at = [&](int j) { return j < sg.n ? sg.table[p.rows.page_of(j)] : 0; };
      auto slot_at = [&](int j, int page) {  // in the pages
        return (kv == 0 ? p.k : p.v) + p.rows.offset(kv, page, sg.h, j - p.rows.page_of(j) * p.rows.page_size);
      };
      auto locate = [&](int tile, int page) {
        const int j = tile * 128 + mine16;
        at = nullptr;
        if (j < sg.n && p.rows.check(page)) {
          const int64_t* st = kv == 0 ? p.kns : p.vns;
          at = j >= sg.first && p.kn != nullptr ? (kv == 0 ? p.kn : p.vn) + sg.b * st[0] + sg.h * st[1] + (j - sg.first) * st[2]
                                                : slot_at(j, page);
        }
        if (kv == 0) there_s[tile & 1][mine16] = at != nullptr;
      };
      auto copy_rows = [&](int which, int where) {
        const uint32_t to = smem_u32(smem + where);
#pragma unroll
        for (int i = 0; i < 16; i += RPI) {
          const int r = i + lane / CH, c = lane % CH;
          const char* row = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at), which * 16 + r));
          copy16_or_zero(to + place(warp * 16 + r, c, 16384), row + c * 16, row != nullptr && c * 16 < p.rows.row_bytes);
        }
        cp_async_commit();
      };
      auto store_new = [&](int which, int j, int page, int where) {  // this lane's row, if it is new, to its page
        if (kv != which || j < sg.first || j >= sg.n || p.kn == nullptr || sg.rb != 0 || !p.rows.check(page)) return;
        char* to = slot_at(j, page);
        for (int c = 0; c * 16 < p.rows.row_bytes; ++c)
          *reinterpret_cast<uint4*>(to + c * 16) = *reinterpret_cast<const uint4*>(smem + where + place(mine16, c, 16384));
      };

      const int s_first = cur.s;
      int page = page_at(s_first * 128 + mine16), page_next = s_first + 1 < cur.end ? page_at(s_first * 128 + 128 + mine16) : 0;
      locate(s_first, page);
      copy_rows(0, Core::kK);
#pragma unroll 1
      for (; cur.s < cur.end; ++cur.s) {
        const int j0 = cur.s * 128, j = j0 + key, j16 = j0 + mine16;
        const bool edge = j0 + 128 > sg.first + 1, news = p.kn != nullptr && j0 + 128 > sg.first;  // edge: not all rows attend all keys
        if (cur.s > s_first) {  // the values' and parts' places are free
          mbar_wait(&bars[1], outputs_done & 1, ctx, 0x3301u);
          ++outputs_done;
        }
        copy_rows(1, Core::kV);
        cp_async_wait<1>();  // the keys
        fence_proxy_async_smem();
        __syncthreads();
        if (news) {
          store_new(0, j16, page, Core::kK);
          __syncthreads();  // (the next keys overwrite what is read here)
        }
        if (warp == 0) {
          tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            mma_bf16_ss_elect(tmem, smem_desc_sw128(smem_u32(smem + Core::kK) + (k >> 2) * 16384 + (k & 3) * 32, 16, 1024),
                              smem_desc_sw128(smem_u32(smem + Core::kQ) + (k >> 2) * 4096 + (k & 3) * 32, 16, 1024),
                              idesc_bf16_f32(128, R, false, false), k > 0);
          mma_commit_elect(&bars[0]);
        }
        const int page_now = page;
        if (cur.s + 1 < cur.end) {  // (looked up a tile ahead)
          page = page_next;
          page_next = cur.s + 2 < cur.end ? page_at(j16 + 256) : 0;
        }
        mbar_wait(&bars[0], scores_done & 1, ctx, 0x3302u);
        ++scores_done;
        tc_fence_after_sync();
        if (cur.s + 1 < cur.end) {
          locate(cur.s + 1, page);
          copy_rows(0, Core::kK);
        } else {
          cp_async_commit();
        }
        const bool there = there_s[cur.s & 1][key];
        uint32_t raw_s[RH];
        tmem_ld_32x16(tmem + lanes + r0, raw_s);
        tmem_ld_wait();
        float s[RH];
#pragma unroll
        for (int i = 0; i < RH; ++i) s[i] = __uint_as_float(raw_s[i]);
        if (edge || !there) {
#pragma unroll
          for (int i = 0; i < RH; ++i)
            if (!there || j > limit_s[r0 + i]) s[i] = -INFINITY;
        }
        if (p.scores != nullptr && j < sg.n) {
          float* to = sg.score_row(p, sg.rb * R + r0) + j;
#pragma unroll
          for (int i = 0; i < RH; ++i)
            if (sg.rb * R + r0 + i < p.R) to[i * p.scores_ld] = s[i] * p.scale;
        }
        bool moves = false;
#pragma unroll
        for (int i = 0; i < RH; i += 4) {
          const float4 o = *reinterpret_cast<const float4*>(over_s + r0 + i);
          moves |= s[i] > o.x || s[i + 1] > o.y || s[i + 2] > o.z || s[i + 3] > o.w;
        }
        if (__syncthreads_or(moves)) {
#pragma unroll
          for (int i = 0; i < RH; ++i) {
            const float m = warp_max(s[i]);
            if (lane == 0) red[warp][i] = m;
          }
          __syncthreads();
          if (tid < R) {
            const int w0 = tid / RH * 4, i = tid % RH;
            const float m = fmaxf(fmaxf(fmaxf(red[w0][i], red[w0 + 1][i]), fmaxf(red[w0 + 2][i], red[w0 + 3][i])) * p.scale, ref_s[tid]);
            fac_s[tid] = rebase(ref_s[tid], m);
            ref_s[tid] = m;
            over_s[tid] = (m + kDecLazy) * p.unscale;
          }
          __syncthreads();
#pragma unroll
          for (int i = 0; i < RH; ++i) sum[i] *= fac_s[r0 + i];
          if (cur.s > s_first) {  // the first four warps rescale the first parts' columns, the others the second parts'
            uint32_t o[32];
            const uint32_t columns = tmem + lanes + kColO + (warp >> 2) * 32;
            tmem_ld_32x32(columns, o);
            tmem_ld_wait();
#pragma unroll
            for (int r = 0; r < R; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * fac_s[r]);
            tmem_st_32x32(columns, o);
            tmem_st_wait();
          }
        }
        // exponentials, their sums, and their parts: half a row of the operand, first parts in the row's first 64 bytes
#pragma unroll
        for (int c = 0; c < RH / 8; ++c) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = c * 8 + 2 * e;
            const float2 ref = *reinterpret_cast<const float2*>(ref_s + r0 + i);
            const float x0 = ex2(fmaf(s[i], p.scale, -ref.x)), x1 = ex2(fmaf(s[i + 1], p.scale, -ref.y));
            sum[i] += x0;
            sum[i + 1] += x1;
            const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
            hi[e] = *reinterpret_cast<const uint32_t*>(&h);
            const __nv_bfloat162 l = __floats2bfloat162_rn(x0 - __uint_as_float(hi[e] << 16), x1 - __uint_as_float(hi[e] & 0xffff0000u));
            lo[e] = *reinterpret_cast<const uint32_t*>(&l);
          }
          const int piece = r0 / 8 + c;
          *reinterpret_cast<uint4*>(smem + Core::kP + place(key, piece, 0)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(smem + Core::kP + place(key, piece + 4, 0)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        cp_async_wait<1>();  // the values
        if (news) {  // (all rows attend a first new key that ends a tile: no edge)
          __syncthreads();
          store_new(1, j16, page_now, Core::kV);
        }
        if (careful) take_out<DP>(smem, limit_s, j0);
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncthreads();
        if (warp == 0) {
          tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_bf16_ss_elect(tmem + kColO, smem_desc_sw128(smem_u32(smem + Core::kV) + k * 2048, 16384, 1024),
                              smem_desc_sw128(smem_u32(smem + Core::kP) + k * 2048, 16384, 1024), idesc_bf16_f32(128, 64, true, true),
                              cur.s > s_first || k > 0);
          mma_commit_elect(&bars[1]);
        }
      }
      cp_async_wait<0>();
      mbar_wait(&bars[1], outputs_done & 1, ctx, 0x3303u);
      ++outputs_done;
      tc_fence_after_sync();
      // sums over the keys, then every thread has an element of its rows
#pragma unroll
      for (int i = 0; i < RH; ++i) {
        const float l = warp_sum(sum[i]);
        if (lane == 0) red[warp][i] = l;
      }
      uint32_t hi[RH], lo[RH];
      tmem_ld_32x16(tmem + lanes + kColO + r0, hi);
      tmem_ld_32x16(tmem + lanes + kColO + 32 + r0, lo);
      tmem_ld_wait();
      tc_fence_before_sync();
      bool spoiled = false;
      if (!careful && key < p.D) {
#pragma unroll
        for (int i = 0; i < RH; ++i) {
          const float o = __uint_as_float(hi[i]) + __uint_as_float(lo[i]);
          spoiled |= !(fabsf(o) < INFINITY) && limit_s[r0 + i] >= 0;
        }
      }
      const bool second = careful;
      careful = __syncthreads_or(spoiled);
      if (careful) {
        cur.s = s_first;
        continue;
      }
      const bool whole = s_first == 0 && cur.s == cur.steps;
      const int64_t piece = worker * 2 + (first_piece ? 0 : 1);
      if (key < p.D) {
        const int w0 = r0 / RH * 4;
#pragma unroll
        for (int i = 0; i < RH; ++i) {
          const int r = r0 + i, row = sg.rb * R + r;
          if (row >= p.R) continue;
          const float l = (red[w0][i] + red[w0 + 1][i]) + (red[w0 + 2][i] + red[w0 + 3][i]);
          float o = __uint_as_float(hi[i]) + __uint_as_float(lo[i]);
          if (second) o += reinterpret_cast<const float*>(smem + Core::kX)[r * DP + key];
          if (whole) {
            char* to = p.out + sg.b * p.os[0] + (sg.h * p.G + row / p.T) * p.os[1] + (row % p.T) * p.os[2];
            reinterpret_cast<__nv_bfloat16*>(to)[key] = __float2bfloat16_rn(limit_s[r] >= 0 ? o * (p.keep / l) : 0.f);
          } else {
            p.part[(piece * p.prows + r) * Core::kDim + key] = o;
          }
          if (key == 0 && (!whole || p.scores != nullptr)) {
            float* to = whole ? p.ml + (sg.index(p) * p.prows + r) * 2 : p.part_ml + (piece * p.prows + r) * 2;
            *reinterpret_cast<float2*>(to) = make_float2(ref_s[r], l);
          }
        }
      }
      first_piece = false;
      __syncthreads();  // what the next segment overwrites has been read
      if (cur.left == 0) break;
      cur.next_segment(p);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == 0) tmem_dealloc(tmem, kWideTmem);
}

template <int DP>
int launch_wide(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st) {
  using Core = CoreWide<DP>;
  if (!set_smem<attn_decode_wide_kernel<DP>>(Core::kSmem)) return PTJ_ERR_LAUNCH;
  launch_k(attn_decode_wide_kernel<DP>, d.workers, kWideThreads, Core::kSmem, st, d);
  PTJ_CHECK_LAUNCH();
  return launch_join<__nv_bfloat16, Core>(d, pl, st);
}

}  // namespace

int decode_wide_blocks() { return kWideBlocks; }
int launch_decode_wide(const DecodeAttn& d, const DecodePlan& pl, cudaStream_t st) {
  return pl.dim == 64 ? launch_wide<64>(d, pl, st) : launch_wide<128>(d, pl, st);
}

}  // namespace ptj
