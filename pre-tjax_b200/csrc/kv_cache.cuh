// Addressing of a paged key-value cache, shared by the kernels that read, fill and thin it out.
#pragma once
#include "common.cuh"
#include "tc_common.cuh"

namespace ptj {

constexpr unsigned int kFaultPage = 0x3201u, kFaultLength = 0x3202u;
constexpr int kMaxHeadDim = 256;

// A pool of pages and the table that lists each sequence's. Strides and offsets are in bytes and 64 bits wide: a long cache
// passes 2^31 elements.
struct PagedRows {
  const int32_t* table;
  int64_t table_ld;
  int64_t page_stride[2], head_stride[2], slot_stride[2];  // of the keys' and the values' pool
  unsigned int* fault;
  int pages, page_size, page_shift;  // page_shift: log2 of the page size, -1 where it is no power of two
  int capacity, capacity_pages;      // keys that a row of the table holds, its pages
  int row_bytes;                     // of a key or a value
  // place of key j's page in the table
  __device__ __forceinline__ int page_of(int j) const {
    return page_shift >= 0 ? j >> page_shift : static_cast<int>(static_cast<unsigned int>(j) / static_cast<unsigned int>(page_size));
  }
  __device__ __forceinline__ bool check(int page) const {
    if (static_cast<unsigned int>(page) < static_cast<unsigned int>(pages)) return true;
    tc::record_fault(fault, kFaultPage);
    return false;
  }
  // page and slot of key j; false: the table names no page of the pool
  __device__ __forceinline__ bool locate(const int32_t* row, int j, int64_t& page, int& slot) const {
    const int i = page_of(j), p = row[i];
    slot = j - i * page_size;
    page = p;
    return check(p);
  }
  __device__ __forceinline__ int64_t offset(int kv, int64_t page, int h, int slot) const {  // kv: 0 keys, 1 values
    return page * page_stride[kv] + h * head_stride[kv] + slot * slot_stride[kv];
  }
  __device__ __forceinline__ int length(const int32_t* lengths, int b) const {
    const int n = lengths[b];
    if (n >= 0 && n <= capacity) return n;
    tc::record_fault(fault, kFaultLength);
    return n < 0 ? 0 : capacity;
  }
  // length and count at once: one wait for both
  __device__ __forceinline__ void extent(const int32_t* lengths, const int32_t* counts, int tokens, int b, int& n, int& c) const {
    n = lengths[b];
    c = counts == nullptr ? tokens : counts[b];
    if (n < 0 || n > capacity || c < 0 || c > tokens) {
      tc::record_fault(fault, kFaultLength);
      n = min(max(n, 0), capacity);
      c = min(max(c, 0), tokens);
    }
  }
  __device__ __forceinline__ int count(const int32_t* counts, int tokens, int b) const {
    if (counts == nullptr) return tokens;
    const int n = counts[b];
    if (n >= 0 && n <= tokens) return n;
    tc::record_fault(fault, kFaultLength);
    return n < 0 ? 0 : tokens;
  }
};

// Checks the host can make, and the addressing of `c` for kernels.
int make_paged_rows(const ptj_kv_cache* c, PagedRows& out);
// The rows of both pools start on 16-byte boundaries and are whole 16-byte pieces.
bool paged_rows_aligned(const ptj_kv_cache& c);
// The same for a view [batch, heads, tokens, d_head]; strides of dimensions of size 1 do not matter.
bool view_aligned(const void* p, const int64_t strides[3], const ptj_kv_cache& c, int64_t heads, int64_t tokens);
// Rows that are written must not share a place: a stride of 0 over more than one element.
bool rows_overlap(const int64_t strides[3], int64_t a, int64_t b, int64_t c);
bool pools_overlap(const ptj_kv_cache& c);
// Checks of the new tokens' descriptor; need_q: q and out are given.
int check_new_tokens(const ptj_kv_cache& c, const ptj_new_tokens* t, bool need_q, bool need_kv);

}  // namespace ptj
