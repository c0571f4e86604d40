// C entry points of attention over a paged key-value cache: checks, choice of the core and of the way to share the work out.
#include "attn_decode.cuh"
#include "tc_runtime.h"

namespace ptj {
namespace {

constexpr int kMaxRows = 4096;      // query rows of a key head
constexpr int kLeastKeys = 64;      // keys that a stretch of the list has at least
constexpr int kMostPieces = 1024;   // pieces of a sequence of the capacity's length, about

bool new_rows_aligned(const ptj_kv_cache& c, const ptj_new_tokens& t) {
  return !t.k || (view_aligned(t.k, t.k_strides, c, c.kv_heads, t.tokens) && view_aligned(t.v, t.v_strides, c, c.kv_heads, t.tokens));
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// aligned: rows of pools and new tokens are whole 16-byte pieces on 16-byte boundaries
DecodePlan make_plan(const ptj_kv_cache& c, const ptj_new_tokens& t, const PagedRows& rows, bool weights, bool aligned) {
  DecodePlan pl = {};
  const int R = static_cast<int>(t.heads / c.kv_heads * t.tokens);
  pl.es = static_cast<int>(dtype_size(c.dtype));
  const bool tc = c.dtype == PTJ_BF16 && c.d_head <= 128;
  pl.dim = c.d_head <= 64 && (tc || pl.es == 4) ? 64 : (c.d_head <= 128 && (tc || pl.es == 4) ? 128 : 256);
  int64_t segs = 0, longest = 0;
  int per_sm = 0;
  // More rows than the registers' products take in one pass at memory speed, and tiles enough that the tcgen05 kernel's longer chain
  // and its second pass do not show: 32 rows on 32 caches of 30k keys of 128 take 113 us on it, 192 in registers, 24 rows 110 and
  // 90; of 2k keys, 32 rows on 64 caches, 59 and 47; 20 rows of 64 elements, 30k keys, 87 and 94. Where the list of stretches is
  // needed anyway it is taken from fewer rows on: 8 caches of 131k keys of 128, 12, 16 and 20 rows 108, 113 and 116 us on it, 117, 116
  // and 151 in registers; one cache of 30k keys, 20 rows, 22 and 27; but 16 rows of 64 elements, 131k keys, 90 and 72.
  auto share_out = [&](bool wide) {
    pl.wide = wide;
    // the core with the fewest blocks of rows (each reads the keys and values again, mostly from L2), of those the smallest
    if (tc) {
      const int most = pl.dim == 64 ? 32 : 24;
      pl.nrb = static_cast<int>(ceil_div(R, most));
      const int need = static_cast<int>(ceil_div(R, pl.nrb));
      pl.rows = need <= 4 ? 4 : need <= 8 ? 8 : (need <= 16 ? 16 : most);
    } else {
      const int most = pl.dim == 256 ? 4 : 8;
      pl.nrb = static_cast<int>(ceil_div(R, most));
      const int need = static_cast<int>(ceil_div(R, pl.nrb));
      pl.rows = need <= 1 ? 1 : (need <= 4 ? 4 : most);
    }
    if (pl.wide) pl.rows = 32;
    pl.nrb = static_cast<int>(ceil_div(R, pl.rows));
    pl.prows = R < pl.rows ? R : pl.rows;
    segs = c.batch * c.kv_heads * pl.nrb;
    const int ks = pl.wide ? 128 : (tc ? 16 : 4096 / (pl.dim * pl.es));  // keys of a step
    longest = ceil_div(rows.capacity, ks);
    // A cluster per segment, of as many blocks as all fit on the GPU at once and have a step for each of their warps (more come in
    // a second round: 16 x 12 float32 caches of 512 keys 15.5 us with one block each, 22.3 with two; 8 x 12 bf16 caches of 1024 with
    // 1, 2, 4, 8 blocks: 15.6, 12.9, 10.8, 16.0). The list of stretches takes over where that could leave a warp more than 64 steps,
    // or more than 16 with SMs idle.
    per_sm = tc ? decode_tc_blocks(pl.dim, pl.rows) : decode_fma_blocks();
    pl.cluster = 1;
    while (pl.cluster < 8 && segs * pl.cluster * 2 <= per_sm * kNumSMs && longest > kDecWarps * pl.cluster) pl.cluster *= 2;
    const int64_t most = ceil_div(longest, kDecWarps * pl.cluster);  // steps of a warp
    pl.split = pl.wide || most > 64 || (most > 16 && segs * pl.cluster < kNumSMs) || (weights && pl.nrb > 1);
  };
  share_out(tc && aligned && R > (pl.dim == 64 ? 16 : 24) &&
            c.batch * c.kv_heads * ceil_div(R, 32) * ceil_div(rows.capacity, 128) >= 12ll * decode_wide_blocks() * kNumSMs);
  if (tc && aligned && pl.split && R > (pl.dim == 64 ? 16 : 8)) share_out(true);
  if (pl.split) {
    pl.workers = pl.wide ? decode_wide_blocks() * kNumSMs : per_sm * kNumSMs * kDecWarps;
    // small stretches: where sequences may be long enough for 32 steps of a warp, and pieces of a few rows are small beside them
    const int64_t steps = segs * longest;
    pl.small = !pl.wide && c.batch <= kDecDynamicBatch && pl.prows <= 8 && steps >= 32ll * pl.workers ? pl.workers : 0;
    const size_t pieces = static_cast<size_t>(pl.workers + pl.small) * 2 * pl.prows;
    pl.part = pieces * pl.dim * 4;
    pl.part_ml = round16(pieces * 8);
    if (weights) pl.ml = round16(static_cast<size_t>(segs) * pl.prows * 8);
    pl.starts = round16(static_cast<size_t>(c.batch + 2) * 8 + 16);
  }
  if (weights) pl.scores = static_cast<size_t>(c.batch * c.kv_heads * R) * rows.capacity * 4;
  return pl;
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
  // (the size goes by sizes alone, so that a caller can keep it)
  const size_t a = make_plan(*cache, *tokens, rows, with_weights != 0, true).bytes();
  const size_t b = make_plan(*cache, *tokens, rows, with_weights != 0, false).bytes();
  return a > b ? a : b;
}

extern "C" int ptj_attn_decode(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, float p, const float* weights,
                               float* weights_out, int64_t weights_ld, void* workspace, size_t workspace_bytes, void* stream) {
  DecodeAttn d = {};
  const int rc = check_decode(cache, tokens, d.rows);
  if (rc != PTJ_OK) return rc;
  if (!(p >= 0.f && p <= 1.f) || (weights && !weights_out) || (weights_out && weights_ld < d.rows.capacity)) return PTJ_ERR_BAD_SHAPE;
  const DecodePlan pl = make_plan(*cache, *tokens, d.rows, weights_out != nullptr, paged_rows_aligned(*cache) && new_rows_aligned(*cache, *tokens));
  const int64_t Hk = cache->kv_heads, T = tokens->tokens, R = tokens->heads / Hk * T;
  if (cache->batch * Hk * R > 0x7fffffff) return PTJ_ERR_BAD_SHAPE;
  if (pl.bytes() > 0) {
    if (!workspace || workspace_bytes < pl.bytes()) return PTJ_ERR_WORKSPACE;
    if (!aligned16(workspace)) return PTJ_ERR_MISALIGNED;
  }
  if (ptj_device_check() != PTJ_OK || (d.rows.fault = tc::fault_word()) == nullptr) return PTJ_ERR_DEVICE;
  d.lengths = cache->lengths;
  d.counts = tokens->counts;
  d.q = static_cast<const char*>(tokens->q);
  d.kn = static_cast<const char*>(tokens->k);
  d.vn = static_cast<const char*>(tokens->v);
  d.k = static_cast<char*>(cache->k);
  d.v = static_cast<char*>(cache->v);
  d.out = static_cast<char*>(tokens->out);
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = tokens->q_strides[i] * pl.es;
    d.os[i] = tokens->o_strides[i] * pl.es;
    d.kns[i] = tokens->k_strides[i] * pl.es;
    d.vns[i] = tokens->v_strides[i] * pl.es;
  }
  char* ws = static_cast<char*>(workspace);
  d.part = reinterpret_cast<float*>(ws);
  d.part_ml = reinterpret_cast<float*>(ws + pl.part);
  d.ml = reinterpret_cast<float*>(ws + pl.part + pl.part_ml);
  d.starts = reinterpret_cast<int64_t*>(ws + pl.part + pl.part_ml + pl.ml);
  d.next = reinterpret_cast<unsigned int*>(d.starts + cache->batch + 2);
  d.scores = weights_out == nullptr ? nullptr : reinterpret_cast<float*>(ws + pl.part + pl.part_ml + pl.ml + pl.starts);
  d.scores_ld = d.rows.capacity;
  d.weights = weights;
  d.weights_out = weights_out;
  d.weights_ld = weights_ld;
  d.scale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(cache->d_head)));
  d.unscale = 1.f / d.scale;
  d.keep = 1.f - p;
  d.B = static_cast<int>(cache->batch);
  d.Hk = static_cast<int>(Hk);
  d.G = static_cast<int>(tokens->heads / Hk);
  d.T = static_cast<int>(T);
  d.D = static_cast<int>(cache->d_head);
  d.R = static_cast<int>(R);
  d.nrb = pl.nrb;
  d.prows = pl.prows;
  d.workers = pl.workers;
  d.small = pl.small;
  const bool tc = cache->dtype == PTJ_BF16 && cache->d_head <= 128;
  const int ks = pl.wide ? 128 : (tc ? 16 : 4096 / (pl.dim * pl.es));
  const int64_t share = ceil_div(ceil_div(d.rows.capacity, ks), kMostPieces);  // (few segments: a row is not joined from thousands of pieces)
  d.least = static_cast<int>(share > kLeastKeys / ks ? share : (kLeastKeys / ks > 1 ? kLeastKeys / ks : 1));
  d.wide = paged_rows_aligned(*cache);
  if (d.kn && d.wide && !new_rows_aligned(*cache, *tokens)) {
    const int rc2 = ptj_kv_append(cache, tokens, stream);  // new rows that cannot be read 16 bytes at a time
    if (rc2 != PTJ_OK) return rc2;
    d.kn = d.vn = nullptr;
  }
  d.q_wide = view_aligned(tokens->q, tokens->q_strides, *cache, tokens->heads, T);
  d.out_wide = cache->d_head % 4 == 0 && view_aligned(tokens->out, tokens->o_strides, *cache, tokens->heads, T);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pl.wide) return launch_decode_wide(d, pl, st);
  return tc ? launch_decode_tc(d, pl, st) : launch_decode_fma(d, pl, st);
}
