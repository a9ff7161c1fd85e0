// What the kernels of the paged key-value cache share: where a slot of a sequence lies, and what is reported when a table or a
// length does not fit the cache.
#pragma once
#include "common.cuh"

namespace tfb {

extern __device__ int g_dev_status;   // the library's status word (status.cu)
constexpr int kBadPage = 0x7200;      // a page id outside the cache
constexpr int kBadLength = 0x7201;    // a length that is negative or more than the sequence's table has room for
constexpr int64_t kCounterBytes = 8192;  // head of a workspace: arrival counters, zero between kernels
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

struct PageMap {
  const int* tables;  // (B, width) page ids, row pitch table_ld
  int64_t table_ld;
  int64_t num_pages;
  int page, width;    // slots of a page, pages of a table
  int64_t s_page, s_head, s_slot;  // element strides of the key and the value pages
  __host__ __device__ int64_t capacity() const { return (int64_t)page * width; }
};

// Page and row of slot `slot` of sequence b; false, and the sticky code, if the table names a page that there is none of.
__device__ __forceinline__ bool find_slot(const PageMap& m, int b, int slot, int& page, int& row) {
  const int i = (int)((unsigned)slot / (unsigned)m.page);
  row = slot - i * m.page;
  page = m.tables[b * m.table_ld + i];
  const bool ok = page >= 0 && page < m.num_pages;
  if (!ok) atomicCAS(&g_dev_status, 0, kBadPage);
  return ok;
}
// Element offset of a row of keys or values.
__device__ __forceinline__ int64_t row_offset(const PageMap& m, int page, int head, int row) {
  return page * m.s_page + head * m.s_head + row * m.s_slot;
}
// Index into the (pages, heads, page) statistics.
__device__ __forceinline__ int64_t stat_offset(const PageMap& m, int page, int heads, int head, int row) {
  return ((int64_t)page * heads + head) * m.page + row;
}

inline int check_pages(const char* what, const PageMap& m, int64_t B, int64_t kv_heads, int64_t hd, int dtype) {
  TFB_REQUIRE(dtype == TFB_F16 || dtype == TFB_BF16, "%s: dtype %d: expected fp16 or bf16", what, dtype);
  if (hd != 32 && hd != 64 && hd != 128) return fail(TFB_ERR_UNSUPPORTED, "%s: Only head_dims of [32,64,128] are supported.", what);
  TFB_REQUIRE(B >= 0 && B < (1 << 20) && kv_heads >= 1 && kv_heads <= 65535, "%s: bad batch or head count", what);
  TFB_REQUIRE(m.page >= 1 && m.width >= 1 && m.capacity() <= (1LL << 30), "%s: a table has 1 to 2^30 slots", what);
  TFB_REQUIRE(m.num_pages >= 1 && m.num_pages < (1LL << 31), "%s: the cache has no pages, or more than 2^31", what);
  TFB_REQUIRE(m.table_ld >= m.width || B <= 1, "%s: the tables' rows overlap", what);
  TFB_REQUIRE(m.s_page % 8 == 0 && m.s_head % 8 == 0 && m.s_slot % 8 == 0, "%s: the pages' rows are not 16-byte aligned", what);
  return TFB_OK;
}

}  // namespace tfb
