// Attention of one new token per sequence over a paged key-value cache in 4 bits (sm_100a): the split, the ring of tiles and the joins of
// paged_attn.cuh, with rows of head_dim / 2 bytes and a pair of 16-bit scales for each.
//
//   s_hj = a_j (q_h . c_j) / sqrt(hd) - slope_h (p - j),  o_h = sum_j softmax_j(s_h) b_j d_j,
//   c_j, d_j whole numbers from -7 to 7 (key and value), a_j, b_j their scales.
//
// The codes go into the products as exact 16-bit numbers, made in registers; a key's scale meets its scores in 32 bits, a value's scale its
// probabilities before they are rounded (to two parts of bf16, so that the weights' rounding does not show).  A word of codes comes out of
// ldmatrix as a lane's share of the instruction: for the keys 8 dims of a key, for the values (transposed as 16-bit units) 4 dims of two
// neighbouring keys, which is the pair that the second product wants.  Tiles come by cp.async: a row is 16 to 64 bytes.
//
// What bounds it is no longer the reading but the instructions: 390 for 16 keys of 128 dims and 8 columns of queries, half of them
// to make codes into numbers, issue slots 58% and the whole-number pipe 54% in use over a launch that lacks a tenth at both ends;
// the copies and the softmax alone take 57 us of the 92 below.  Measured in graphs, in brackets the 16-bit cache: bf16, head_dim
// 128, 32 sequences of up to 16384 keys, 8 key heads of 4 query heads 92 us (169); fp16, head_dim 64, 24 sequences of up to 2048
// keys, 16 heads, slopes 20.4 (25.9); one of 700 keys 8.3 (9.3).  With the new token's row quantized and written, as a generation
// step calls it, on the same inputs each time: 85.8 us for 85.5 without, 20.2 for 19.6, 9.3 for 8.4.  Not kept for the long ones:
// two blocks an SM (113 us, registers spilled), tiles of 32 keys (95 to 109), TMA boxes for the copies (95), 8 warps with three
// tiles ahead (93, the short ones 9.6 and 22.1).
#include "paged_attn.cuh"

namespace tfb {
namespace {

template <typename T, int HD, int G, int BIAS>
int pg4_split(const PgParams& p, cudaStream_t st) {
  using C = PgCfg<HD, G, BIAS, true>;
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(paged_attn_kernel<T, HD, G, BIAS, false, true>, C::SMEM, done, "paged_attention_int4")) return rc;
  const CUtensorMap none = {};
  launch_overlapped(paged_attn_kernel<T, HD, G, BIAS, false, true>, dim3(p.ctas), dim3(C::WARPS * 32), C::SMEM, st, none, none, p);
  return launched("paged_attention_int4");
}
template <typename T, int HD, int G>
int pg4_launch(const PgParams& p, cudaStream_t st) {
  return p.bias_mode == 0 ? pg4_split<T, HD, G, 0>(p, st) : p.bias_mode == 1 ? pg4_split<T, HD, G, 1>(p, st) : pg4_split<T, HD, G, 2>(p, st);
}
template <typename T, int HD>
int pg4_dispatch(const PgParams& p, cudaStream_t st) {
  if (p.group <= 4) return pg4_launch<T, HD, 4>(p, st);
  return p.group <= 8 ? pg4_launch<T, HD, 8>(p, st) : pg4_launch<T, HD, 16>(p, st);
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int tfb_paged_attention_int4(const void* q, const void* k_new, const void* v_new, void* out, void* k_pages, void* v_pages,
                                        void* scales, const int* tables, const int* lengths, const float* slopes, int alibi_round,
                                        int64_t B, int64_t kv_heads, int64_t group, int64_t hd, int64_t num_pages, int64_t page,
                                        int64_t width, int64_t table_ld, const int64_t* page_strides, const int64_t* q_strides,
                                        const int64_t* k_new_strides, const int64_t* v_new_strides, const int64_t* o_strides,
                                        void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  PgParams p = {};
  TFB_REQUIRE(page >= 1 && page < (1LL << 31) && width >= 1 && width < (1LL << 31), "paged_attention_int4: bad page or table size");
  p.map = {tables, table_ld, num_pages, (int)page, (int)width, page_strides[0], page_strides[1], page_strides[2]};
  if (int rc = check_pages("paged_attention_int4", p.map, B, kv_heads, hd, dtype)) return rc;
  TFB_REQUIRE(p.map.s_page % 16 == 0 && p.map.s_head % 16 == 0 && p.map.s_slot % 16 == 0,
              "paged_attention_int4: the pages' rows are not 16-byte aligned");
  TFB_REQUIRE(group >= 1 && group <= 128, "paged_attention_int4: %lld query heads on a key head: expected 1 to 128", (long long)group);
  TFB_REQUIRE(B * kv_heads < (1LL << 31), "paged_attention_int4: too many rows");
  TFB_REQUIRE((k_new == nullptr) == (v_new == nullptr), "paged_attention_int4: a new key without a value, or the other way round");
  TFB_REQUIRE(alibi_round >= 0 && alibi_round <= 2, "paged_attention_int4: alibi_round %d", alibi_round);
  if (B == 0) return TFB_OK;
  TFB_REQUIRE(aligned16(k_pages) && aligned16(v_pages), "paged_attention_int4: the pages are not 16-byte aligned");
  TFB_REQUIRE(scales && (reinterpret_cast<uintptr_t>(scales) & 3) == 0, "paged_attention_int4: the scales are not 4-byte aligned");
  const PgWorkspace s = pg_workspace();
  TFB_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= s.bytes,
              "paged_attention_int4: workspace of %lld bytes, %lld wanted", (long long)workspace_bytes, (long long)s.bytes);
  p.q = q;
  p.k_new = k_new;
  p.v_new = v_new;
  p.out = out;
  p.k = k_pages;
  p.v = v_pages;
  p.scales = scales;
  p.lengths = lengths;
  p.slopes = slopes;
  p.bias_mode = !slopes ? 0 : alibi_round == 0 ? 1 : alibi_round == 1 ? 2 : 4;
  p.q_b = q_strides[0];
  p.q_h = q_strides[1];
  p.o_b = o_strides[0];
  p.o_h = o_strides[1];
  if (k_new) {
    p.kn_b = k_new_strides[0];
    p.kn_h = k_new_strides[1];
    p.vn_b = v_new_strides[0];
    p.vn_h = v_new_strides[1];
    p.new_vec = aligned16(k_new) && aligned16(v_new) && p.kn_b % 8 == 0 && p.kn_h % 8 == 0 && p.vn_b % 8 == 0 && p.vn_h % 8 == 0;
  }
  p.B = (int)B;
  p.kv_heads = (int)kv_heads;
  p.group = (int)group;
  p.row_tiles = (int)ceil_div(group, 16);
  p.ctas = sm_count();
  p.scale = kLog2e / sqrtf((float)hd);
  p.q_pairs = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(p.q_b * 2) | (uintptr_t)(p.q_h * 2)) & 3) == 0;
  char* base = static_cast<char*>(workspace);
  p.arrived = reinterpret_cast<int*>(base);
  p.ml = reinterpret_cast<float2*>(base + s.ml);
  p.acc = reinterpret_cast<float*>(base + s.acc);
  p.heads_acc = reinterpret_cast<float*>(base + s.heads_acc);
  cudaStream_t st = (cudaStream_t)stream;
  TFB_DISPATCH_16(dtype, T, {
    if (hd == 32) return pg4_dispatch<T, 32>(p, st);
    if (hd == 64) return pg4_dispatch<T, 64>(p, st);
    return pg4_dispatch<T, 128>(p, st);
  })
}
