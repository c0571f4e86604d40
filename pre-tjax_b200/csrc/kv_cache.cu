// Paged key-value caches: checks of the descriptors, writing new rows into their pages.
#include "kv_cache.cuh"
#include "tc_runtime.h"

namespace ptj {

int make_paged_rows(const ptj_kv_cache* c, PagedRows& out) {
  if (!c || !c->k || !c->v || !c->table || !c->lengths) return PTJ_ERR_BAD_SHAPE;
  if (c->dtype != PTJ_F32 && c->dtype != PTJ_BF16) return PTJ_ERR_DTYPE;
  if (c->batch < 1 || c->kv_heads < 1 || c->d_head < 1 || c->d_head > kMaxHeadDim || c->pages < 1 || c->page_size < 1 ||
      c->table_width < 1 || c->table_ld < c->table_width)
    return PTJ_ERR_BAD_SHAPE;
  // positions and numbers of rows are 32-bit in the kernels, offsets are 64-bit
  if (c->batch > (1 << 20) || c->kv_heads > (1 << 16) || c->batch * c->kv_heads > (1 << 24) || c->pages > 0x7fffffff ||
      c->page_size > (1 << 24) || c->table_width > (1 << 28) || c->table_width * c->page_size > (1 << 30))
    return PTJ_ERR_BAD_SHAPE;
  out = PagedRows{};
  out.table = c->table;
  out.table_ld = c->table_ld;
  const int64_t es = static_cast<int64_t>(dtype_size(c->dtype));
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i == 0 ? c->k_strides : c->v_strides;
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return PTJ_ERR_BAD_SHAPE;
    out.page_stride[i] = s[0] * es;
    out.head_stride[i] = s[1] * es;
    out.slot_stride[i] = s[2] * es;
  }
  out.pages = static_cast<int>(c->pages);
  out.page_size = static_cast<int>(c->page_size);
  out.page_shift = -1;
  for (int i = 0; i < 25; ++i)
    if (c->page_size == (1ll << i)) out.page_shift = i;
  out.capacity = static_cast<int>(c->table_width * c->page_size);
  out.capacity_pages = static_cast<int>(c->table_width);
  out.row_bytes = static_cast<int>(c->d_head * es);
  return PTJ_OK;
}

static bool strided16(const void* p, const int64_t strides[3], const int64_t sizes[3], int64_t per16) {
  if (!aligned16(p)) return false;
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1 && strides[i] % per16 != 0) return false;
  return true;
}

bool paged_rows_aligned(const ptj_kv_cache& c) {
  const int64_t per16 = 16 / static_cast<int64_t>(dtype_size(c.dtype));
  const int64_t sizes[3] = {c.pages, c.kv_heads, c.page_size};
  return c.d_head % per16 == 0 && strided16(c.k, c.k_strides, sizes, per16) && strided16(c.v, c.v_strides, sizes, per16);
}

bool view_aligned(const void* p, const int64_t strides[3], const ptj_kv_cache& c, int64_t heads, int64_t tokens) {
  const int64_t sizes[3] = {c.batch, heads, tokens};
  return strided16(p, strides, sizes, 16 / static_cast<int64_t>(dtype_size(c.dtype)));
}

bool rows_overlap(const int64_t strides[3], int64_t a, int64_t b, int64_t c) {
  return (a > 1 && strides[0] == 0) || (b > 1 && strides[1] == 0) || (c > 1 && strides[2] == 0);
}

bool pools_overlap(const ptj_kv_cache& c) {
  return rows_overlap(c.k_strides, c.pages, c.kv_heads, c.page_size) || rows_overlap(c.v_strides, c.pages, c.kv_heads, c.page_size);
}

int check_new_tokens(const ptj_kv_cache& c, const ptj_new_tokens* t, bool need_q, bool need_kv) {
  if (!t || t->tokens < 1 || t->tokens > 4096) return PTJ_ERR_BAD_SHAPE;
  if ((t->k == nullptr) != (t->v == nullptr) || (need_kv && !t->k)) return PTJ_ERR_BAD_SHAPE;
  if (need_q && (!t->q || !t->out || t->heads < 1 || t->heads % c.kv_heads != 0 || t->heads > (1 << 16))) return PTJ_ERR_BAD_SHAPE;
  for (int i = 0; i < 3; ++i) {
    if (need_q && (t->q_strides[i] < 0 || t->o_strides[i] < 0)) return PTJ_ERR_BAD_SHAPE;
    if (t->k && (t->k_strides[i] < 0 || t->v_strides[i] < 0)) return PTJ_ERR_BAD_SHAPE;
  }
  // what is written has a place of its own
  if ((need_q && rows_overlap(t->o_strides, c.batch, t->heads, t->tokens)) || (t->k && pools_overlap(c))) return PTJ_ERR_BAD_SHAPE;
  return PTJ_OK;
}

namespace {

constexpr int kAppendThreads = 256;

struct AppendParams {
  PagedRows rows;
  const int32_t *lengths, *counts;
  const char* src[2];
  char* dst[2];
  int64_t src_strides[2][3];  // bytes
  int tokens, heads, pieces;  // pieces of a row
  int64_t total;              // batch * tokens * heads * 2 * pieces
};

// A thread copies one piece V (16 bytes, or an element where rows are not aligned) of a key's or a value's row.
template <typename V>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(const __grid_constant__ AppendParams p) {
  grid_dep_sync();
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kAppendThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x; i < p.total; i += stride) {
    int64_t r = i;
    const int c = static_cast<int>(r % p.pieces); r /= p.pieces;
    const int kv = static_cast<int>(r & 1); r >>= 1;
    const int h = static_cast<int>(r % p.heads); r /= p.heads;
    const int t = static_cast<int>(r % p.tokens);
    const int b = static_cast<int>(r / p.tokens);
    const int count = p.rows.count(p.counts, p.tokens, b);
    const int pos = p.rows.length(p.lengths, b) - count + t;
    if (t >= count || pos < 0) continue;
    int64_t page;
    int slot;
    if (!p.rows.locate(p.rows.table + b * p.rows.table_ld, pos, page, slot)) continue;
    const char* from = p.src[kv] + b * p.src_strides[kv][0] + h * p.src_strides[kv][1] + t * p.src_strides[kv][2];
    char* to = p.dst[kv] + p.rows.offset(kv, page, h, slot);
    reinterpret_cast<V*>(to)[c] = reinterpret_cast<const V*>(from)[c];
  }
}

}  // namespace
}  // namespace ptj

using namespace ptj;

extern "C" int ptj_kv_append(const ptj_kv_cache* cache, const ptj_new_tokens* tokens, void* stream) {
  AppendParams p = {};
  int rc = make_paged_rows(cache, p.rows);
  if (rc == PTJ_OK) rc = check_new_tokens(*cache, tokens, false, true);
  if (rc != PTJ_OK) return rc;
  if (ptj_device_check() != PTJ_OK || (p.rows.fault = tc::fault_word()) == nullptr) return PTJ_ERR_DEVICE;
  const int64_t es = static_cast<int64_t>(dtype_size(cache->dtype));
  const bool wide = paged_rows_aligned(*cache) && view_aligned(tokens->k, tokens->k_strides, *cache, cache->kv_heads, tokens->tokens) &&
                    view_aligned(tokens->v, tokens->v_strides, *cache, cache->kv_heads, tokens->tokens);
  p.lengths = cache->lengths;
  p.counts = tokens->counts;
  for (int i = 0; i < 2; ++i) {
    p.src[i] = static_cast<const char*>(i == 0 ? tokens->k : tokens->v);
    p.dst[i] = static_cast<char*>(i == 0 ? cache->k : cache->v);
    for (int j = 0; j < 3; ++j) p.src_strides[i][j] = (i == 0 ? tokens->k_strides : tokens->v_strides)[j] * es;
  }
  p.tokens = static_cast<int>(tokens->tokens);
  p.heads = static_cast<int>(cache->kv_heads);
  p.pieces = static_cast<int>(wide ? cache->d_head * es / 16 : cache->d_head);
  p.total = cache->batch * tokens->tokens * cache->kv_heads * 2 * p.pieces;
  const int64_t blocks = ceil_div(p.total, kAppendThreads);
  const int grid = static_cast<int>(blocks < 16 * kNumSMs ? blocks : 16 * kNumSMs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (wide) launch_k(append_kernel<uint4>, grid, kAppendThreads, 0, st, p);
  else if (es == 2) launch_k(append_kernel<uint16_t>, grid, kAppendThreads, 0, st, p);
  else launch_k(append_kernel<uint32_t>, grid, kAppendThreads, 0, st, p);
  PTJ_CHECK_LAUNCH();
  return PTJ_OK;
}
