// Writing keys and values into a paged cache in 4 bits (sm_100a).
//
// A row of head_dim values becomes codes, the nearest whole numbers to value / scale, and one 16-bit scale, its largest magnitude over 7.
// What is read is 4 times what is written, so the pass is bound by reading the rows once: a row is a line of lanes with 16 bytes each, the
// largest magnitude three to four shuffles away, and a lane's 8 codes are one word of the row.  On request the values that the cache now
// stands for are written out beside it, so that a prompt's own attention can use what later tokens will find.
//
// Measured: 16 sequences of up to 4096 keys, 8 heads of 128, bf16, with what is stored, 84 us, 5.2 TB/s (79% of a copy); 24 warps
// an SM instead of 32 took 90, divisions instead of products 179.  One token: 4.7 us in a graph, the chain of length, table, row
// and scale.
#include "nibbles.cuh"
#include "paged.cuh"

namespace tfb {
namespace {

struct Append4Params {
  PageMap map;  // strides in bytes
  const void *key, *value;
  uint8_t *k, *v;
  uint32_t* scales;  // (pages, heads, page), pairs
  const int *lengths, *counts;  // counts: may be null (all T)
  void *k_stored, *v_stored;    // may be null
  int64_t k_b, k_h, k_t, v_b, v_h, v_t, s_b, s_h, s_t;
  int kv_heads, T;
};

constexpr int A4_ROWS = 64;  // rows of a block

// What codes stand for, rounded to the type.
template <typename T>
__device__ __forceinline__ uint4 restore8(const float (&whole)[8], float scale) {
  float x[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) x[d] = whole[d] * scale;
  return pack8<T>(x);
}

template <typename T>
__device__ __forceinline__ uint4 load_row8(const T* p, bool vec) {
  if (vec) return ld_stream16(p);
  const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
  uint4 v;
  v.x = e[0] | (uint32_t)e[1] << 16;
  v.y = e[2] | (uint32_t)e[3] << 16;
  v.z = e[4] | (uint32_t)e[5] << 16;
  v.w = e[6] | (uint32_t)e[7] << 16;
  return v;
}

// One block: A4_ROWS rows of a (sequence, key head); neighbouring blocks take neighbouring heads, which lie side by side in a
// projection's output.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(256, 4) append_int4_kernel(const Append4Params p) {
  constexpr int LANES = HD / 8, PER = 256 / LANES, N = A4_ROWS / PER;
  __shared__ int sh_page[A4_ROWS], sh_row[A4_ROWS];
  grid_dependency_wait();
  allow_dependents();
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads;
  const int cap = (int)p.map.capacity(), len = p.lengths[b];
  const int want = p.counts ? p.counts[b] : p.T;
  const int start = min(max(len, 0), cap), count = min(min(max(want, 0), p.T), cap - start);
  const int t0 = blockIdx.y * A4_ROWS;
  if (blockIdx.y == 0 && h == 0 && threadIdx.x == 0 && (len < 0 || want < 0 || want > p.T || (int64_t)len + want > cap))
    atomicCAS(&g_dev_status, 0, kBadLength);
  if (t0 >= count) {  // nothing to write but zeros behind the sequence's keys
    if (p.k_stored)
      for (int r = threadIdx.x / LANES; r < A4_ROWS && t0 + r < p.T; r += PER) {
        const int64_t o = b * p.s_b + h * p.s_h + (t0 + r) * p.s_t + threadIdx.x % LANES * 8;
        st_stream16(static_cast<T*>(p.k_stored) + o, make_uint4(0, 0, 0, 0));
        st_stream16(static_cast<T*>(p.v_stored) + o, make_uint4(0, 0, 0, 0));
      }
    return;
  }
  if (threadIdx.x < A4_ROWS) {
    int page = -1, row = 0;
    const int t = t0 + threadIdx.x;
    if (!(t < count && find_slot(p.map, b, start + t, page, row))) page = -1;
    sh_page[threadIdx.x] = page;
    sh_row[threadIdx.x] = row;
  }
  __syncthreads();
  const int c = threadIdx.x % LANES;
  const T* key = static_cast<const T*>(p.key) + b * p.k_b + h * p.k_h + c * 8;
  const T* value = static_cast<const T*>(p.value) + b * p.v_b + h * p.v_h + c * 8;
  uint4 kr[N], vr[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = t0 + i * PER + threadIdx.x / LANES;
    kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
    if (t < count) {
      kr[i] = load_row8<T>(key + t * p.k_t, VEC);
      vr[i] = load_row8<T>(value + t * p.v_t, VEC);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = i * PER + threadIdx.x / LANES, t = t0 + r;
    T ks, vs;
    float kc[8], vc[8];
    const uint32_t kw = quantize8<T, LANES>(kr[i], ks, kc), vw = quantize8<T, LANES>(vr[i], vs, vc);
    if (sh_page[r] >= 0) {
      const int64_t o = row_offset(p.map, sh_page[r], h, sh_row[r]) + c * 4;
      *reinterpret_cast<uint32_t*>(p.k + o) = kw;
      *reinterpret_cast<uint32_t*>(p.v + o) = vw;
      if (c == 0)
        p.scales[stat_offset(p.map, sh_page[r], p.kv_heads, h, sh_row[r])] =
            *reinterpret_cast<const uint16_t*>(&ks) | (uint32_t)*reinterpret_cast<const uint16_t*>(&vs) << 16;
    }
    if (p.k_stored && t < p.T) {
      const int64_t o = b * p.s_b + h * p.s_h + t * p.s_t + c * 8;
      st_stream16(static_cast<T*>(p.k_stored) + o, restore8<T>(kc, Num<T>::to_f(ks)));
      st_stream16(static_cast<T*>(p.v_stored) + o, restore8<T>(vc, Num<T>::to_f(vs)));
    }
  }
}

template <typename T, int HD>
int append4_launch(const Append4Params& p, int64_t B, bool vec, cudaStream_t st) {
  const dim3 grid((unsigned)(B * p.kv_heads), (unsigned)ceil_div(p.T, A4_ROWS));
  launch_overlapped(vec ? append_int4_kernel<T, HD, true> : append_int4_kernel<T, HD, false>, grid, dim3(256), 0, st, p);
  return launched("cache_append_int4");
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int tfb_cache_append_int4(const void* key, const void* value, void* k_pages, void* v_pages, void* scales, const int* tables,
                                     const int* lengths, const int* counts, void* k_stored, void* v_stored, int64_t B,
                                     int64_t kv_heads, int64_t T, int64_t hd, int64_t num_pages, int64_t page, int64_t width,
                                     int64_t table_ld, const int64_t* page_strides, const int64_t* key_strides,
                                     const int64_t* value_strides, const int64_t* stored_strides, int dtype, void* stream) {
  Append4Params p = {};
  TFB_REQUIRE(page >= 1 && page < (1LL << 31) && width >= 1 && width < (1LL << 31), "cache_append_int4: bad page or table size");
  p.map = {tables, table_ld, num_pages, (int)page, (int)width, page_strides[0], page_strides[1], page_strides[2]};
  if (int rc = check_pages("cache_append_int4", p.map, B, kv_heads, hd, dtype)) return rc;
  TFB_REQUIRE(p.map.s_page % 16 == 0 && p.map.s_head % 16 == 0 && p.map.s_slot % 16 == 0,
              "cache_append_int4: the pages' rows are not 16-byte aligned");
  TFB_REQUIRE(T >= 0 && T <= 65535 * (int64_t)A4_ROWS, "cache_append_int4: more than %lld keys", (long long)(65535 * (int64_t)A4_ROWS));
  TFB_REQUIRE(B * kv_heads < (1LL << 31), "cache_append_int4: too many rows of heads");
  TFB_REQUIRE((k_stored == nullptr) == (v_stored == nullptr), "cache_append_int4: stored keys without values, or the other way round");
  if (B == 0 || T == 0) return TFB_OK;
  TFB_REQUIRE(aligned16(k_pages) && aligned16(v_pages), "cache_append_int4: the pages are not 16-byte aligned");
  TFB_REQUIRE(scales && (reinterpret_cast<uintptr_t>(scales) & 3) == 0, "cache_append_int4: the scales are not 4-byte aligned");
  p.key = key;
  p.value = value;
  p.k = static_cast<uint8_t*>(k_pages);
  p.v = static_cast<uint8_t*>(v_pages);
  p.scales = static_cast<uint32_t*>(scales);
  p.lengths = lengths;
  p.counts = counts;
  p.k_stored = k_stored;
  p.v_stored = v_stored;
  p.k_b = key_strides[0];
  p.k_h = key_strides[1];
  p.k_t = key_strides[2];
  p.v_b = value_strides[0];
  p.v_h = value_strides[1];
  p.v_t = value_strides[2];
  if (k_stored) {
    p.s_b = stored_strides[0];
    p.s_h = stored_strides[1];
    p.s_t = stored_strides[2];
    TFB_REQUIRE(aligned16(k_stored) && aligned16(v_stored) && p.s_b % 8 == 0 && p.s_h % 8 == 0 && p.s_t % 8 == 0,
                "cache_append_int4: the stored rows are not 16-byte aligned");
  }
  p.kv_heads = (int)kv_heads;
  p.T = (int)T;
  bool vec = aligned16(key) && aligned16(value);
  for (int i = 0; i < 3; ++i) vec = vec && key_strides[i] % 8 == 0 && value_strides[i] % 8 == 0;
  TFB_DISPATCH_16(dtype, E, {
    if (hd == 32) return append4_launch<E, 32>(p, B, vec, (cudaStream_t)stream);
    if (hd == 64) return append4_launch<E, 64>(p, B, vec, (cudaStream_t)stream);
    return append4_launch<E, 128>(p, B, vec, (cudaStream_t)stream);
  })
}
