// Attention of one new token per sequence over a paged key-value cache in 16 bits: the kernel of the masses, and the calls.
#include "paged_attn.cuh"

namespace tfb {

// Adds the weights to the masses.  Blocks along (sequence, key head) and shares of its keys; a thread takes MASS_BATCH keys at a
// time, all lookups of a kind together (one after the other the kernel waited for them: 25 us for 2.1 M keys of 8 heads).  V: how
// many of a key's scores are read at once.
constexpr int MASS_BATCH = 4, MASS_THREADS = 128;
template <int V>
__global__ void __launch_bounds__(MASS_THREADS) paged_mass_kernel(const PgParams p) {
  __shared__ __align__(16) float sh_lse[128];
  grid_dependency_wait();
  allow_dependents();
  const int b = blockIdx.x / p.kv_heads, kv = blockIdx.x % p.kv_heads, cap = (int)p.map.capacity();
  constexpr int SPAN = MASS_BATCH * MASS_THREADS;
  const int* table = p.map.tables + b * p.map.table_ld;
  int page[MASS_BATCH], row[MASS_BATCH];
  auto look_up = [&](int slot0) {  // does not wait for the length: entries behind it are read, not used
#pragma unroll
    for (int k = 0; k < MASS_BATCH; ++k) {
      const int slot = min(slot0 + k * MASS_THREADS, cap - 1), i = (int)((unsigned)slot / (unsigned)p.map.page);
      row[k] = slot - i * p.map.page;
      page[k] = table[i];
    }
  };
  const int len = p.lengths[b];
  look_up(blockIdx.y * SPAN + threadIdx.x);
  for (int r = threadIdx.x; r < p.group; r += MASS_THREADS) {
    const float lse = p.lse[((int64_t)b * p.kv_heads + kv) * p.group + r];
    sh_lse[r] = lse == kNone ? INFINITY : lse;  // no weight anywhere: none for the masses either
  }
  const SeqKeys keys = keys_of(p, len);
  if (blockIdx.y * SPAN >= keys.n) return;
  const float* sc = p.scores + ((int64_t)b * p.kv_heads + kv) * p.map.capacity() * p.group;
  __syncthreads();
  for (int slot0 = blockIdx.y * SPAN + threadIdx.x; slot0 < keys.n; slot0 += gridDim.y * SPAN) {
    int64_t at[MASS_BATCH];
    float had[MASS_BATCH], w[MASS_BATCH];
#pragma unroll
    for (int k = 0; k < MASS_BATCH; ++k) {
      // of a slot in use the attention has reported a bad page
      const bool ok = slot0 + k * MASS_THREADS < keys.n && (unsigned)page[k] < (unsigned)p.map.num_pages;
      at[k] = ok ? stat_offset(p.map, page[k], p.kv_heads, kv, row[k]) : -1;
      had[k] = ok ? p.mass[at[k]] : 0.f;
      w[k] = 0.f;
    }
#pragma unroll 2
    for (int r = 0; r < p.group; r += V) {
      float x[MASS_BATCH][V], y[V];
#pragma unroll
      for (int k = 0; k < MASS_BATCH; ++k) {
        const float* mine = sc + (int64_t)min(slot0 + k * MASS_THREADS, keys.n - 1) * p.group + r;
        if constexpr (V == 4) *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(mine);
        else x[k][0] = *mine;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = sh_lse[r + e];
#pragma unroll
      for (int k = 0; k < MASS_BATCH; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) w[k] += ex2(x[k][e] - y[e]);
    }
#pragma unroll
    for (int k = 0; k < MASS_BATCH; ++k) {
      if (at[k] >= 0) p.mass_out[at[k]] = slot0 + k * MASS_THREADS == keys.fresh ? w[k] : had[k] + w[k];
    }
    look_up(slot0 + gridDim.y * SPAN);
  }
}

namespace {

template <typename T, int HD, int G, int BIAS, bool TMA>
int pg_split(const CUtensorMap& tk, const CUtensorMap& tv, const PgParams& p, cudaStream_t st) {
  using C = PgCfg<HD, G, BIAS, false>;
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(paged_attn_kernel<T, HD, G, BIAS, TMA, false>, C::SMEM, done, "paged_attention")) return rc;
  launch_overlapped(paged_attn_kernel<T, HD, G, BIAS, TMA, false>, dim3(p.ctas), dim3(C::WARPS * 32), C::SMEM, st, tk, tv, p);
  return launched("paged_attention");
}

template <typename T, int HD, int G>
int pg_launch(PgParams& p, int dtype, cudaStream_t st) {
  // rows of a box: what divides both a page and a tile, so that a tile is whole boxes and a box lies in one page
  int box = 2048 / HD;
  while (p.map.page % box) box /= 2;
  p.box_log2 = 0;
  while ((1 << p.box_log2) < box) ++p.box_log2;
  CUtensorMap tk = {}, tv = {};
  int rc;
  if (box >= 8) {
    const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)p.map.page, (uint64_t)p.kv_heads, (uint64_t)p.map.num_pages};
    const int64_t s[3] = {p.map.s_slot, p.map.s_head, p.map.s_page};
    uint64_t str[3];
    for (int i = 0; i < 3; ++i) str[i] = dims[i + 1] > 1 ? (uint64_t)s[i] * 2 : (uint64_t)HD * 2;
    const uint32_t shape[4] = {HD < 64 ? (uint32_t)HD : 64u, (uint32_t)box, 1, 1};
    const auto encode = HD == 32 ? encode_tmap_sw64 : encode_tmap_sw128;
    if ((rc = encode(&tk, p.k, dtype, 4, dims, str, shape)) || (rc = encode(&tv, p.v, dtype, 4, dims, str, shape))) return rc;
    rc = p.bias_mode == 0   ? pg_split<T, HD, G, 0, true>(tk, tv, p, st)
         : p.bias_mode == 1 ? pg_split<T, HD, G, 1, true>(tk, tv, p, st)
                            : pg_split<T, HD, G, 2, true>(tk, tv, p, st);
  } else {
    rc = p.bias_mode == 0   ? pg_split<T, HD, G, 0, false>(tk, tv, p, st)
         : p.bias_mode == 1 ? pg_split<T, HD, G, 1, false>(tk, tv, p, st)
                            : pg_split<T, HD, G, 2, false>(tk, tv, p, st);
  }
  if (rc) return rc;
  if (!p.mass_out) return TFB_OK;
  // enough blocks to fill the SMs, none with fewer keys of a full table than its threads take at once
  const int64_t rows = (int64_t)p.B * p.kv_heads, most = ceil_div(p.map.capacity(), MASS_BATCH * MASS_THREADS);
  int64_t shares = ceil_div((int64_t)sm_count() * 32, rows);
  if (shares > most) shares = most;
  const dim3 grid((unsigned)rows, (unsigned)shares);
  if (p.group % 4 == 0) launch_overlapped(paged_mass_kernel<4>, grid, dim3(MASS_THREADS), 0, st, p);
  else launch_overlapped(paged_mass_kernel<1>, grid, dim3(MASS_THREADS), 0, st, p);
  return launched("paged_attention: masses");
}

template <typename T, int HD>
int pg_dispatch(PgParams& p, int dtype, cudaStream_t st) {
  if (p.group <= 4) return pg_launch<T, HD, 4>(p, dtype, st);
  return p.group <= 8 ? pg_launch<T, HD, 8>(p, dtype, st) : pg_launch<T, HD, 16>(p, dtype, st);
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int64_t tfb_paged_attention_workspace_bytes(void) { return pg_workspace().bytes; }

extern "C" int64_t tfb_paged_attention_scratch_bytes(int64_t B, int64_t kv_heads, int64_t group, int64_t capacity) {
  if (B < 0 || kv_heads < 0 || group < 0 || capacity < 0) return 0;
  return up256(B * kv_heads * group * 4) + B * kv_heads * group * capacity * 4;
}

extern "C" int tfb_paged_attention(const void* q, const void* k_new, const void* v_new, void* out, void* k_pages, void* v_pages,
                                   const int* tables, const int* lengths, const int* query_positions, int* positions,
                                   const float* mass, float* mass_out, const float* slopes, int alibi_round, int64_t B,
                                   int64_t kv_heads, int64_t group, int64_t hd, int64_t num_pages, int64_t page, int64_t width,
                                   int64_t table_ld, const int64_t* page_strides, const int64_t* q_strides,
                                   const int64_t* k_new_strides, const int64_t* v_new_strides, const int64_t* o_strides,
                                   void* workspace, int64_t workspace_bytes, void* scratch, int64_t scratch_bytes, int dtype,
                                   void* stream) {
  PgParams p = {};
  TFB_REQUIRE(page >= 1 && page < (1LL << 31) && width >= 1 && width < (1LL << 31), "paged_attention: bad page or table size");
  p.map = {tables, table_ld, num_pages, (int)page, (int)width, page_strides[0], page_strides[1], page_strides[2]};
  if (int rc = check_pages("paged_attention", p.map, B, kv_heads, hd, dtype)) return rc;
  TFB_REQUIRE(group >= 1 && group <= 128, "paged_attention: %lld query heads on a key head: expected 1 to 128", (long long)group);
  TFB_REQUIRE(B * kv_heads < (1LL << 31), "paged_attention: too many rows");
  TFB_REQUIRE((k_new == nullptr) == (v_new == nullptr), "paged_attention: a new key without a value, or the other way round");
  TFB_REQUIRE((mass == nullptr) == (mass_out == nullptr), "paged_attention: mass and mass_out come together");
  TFB_REQUIRE(alibi_round >= 0 && alibi_round <= 2, "paged_attention: alibi_round %d", alibi_round);
  if (B == 0) return TFB_OK;
  TFB_REQUIRE(aligned16(k_pages) && aligned16(v_pages), "paged_attention: the pages are not 16-byte aligned");
  const PgWorkspace s = pg_workspace();
  TFB_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= s.bytes, "paged_attention: workspace of %lld bytes, %lld wanted",
              (long long)workspace_bytes, (long long)s.bytes);
  if (mass) {
    const int64_t want = tfb_paged_attention_scratch_bytes(B, kv_heads, group, p.map.capacity());
    TFB_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= want, "paged_attention: scratch of %lld bytes, %lld wanted",
                (long long)scratch_bytes, (long long)want);
  }
  p.q = q;
  p.k_new = k_new;
  p.v_new = v_new;
  p.out = out;
  p.k = k_pages;
  p.v = v_pages;
  p.lengths = lengths;
  p.query_positions = query_positions;
  p.positions = positions;
  p.mass = mass;
  p.mass_out = mass_out;
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
  if (mass) {
    p.lse = static_cast<float*>(scratch);
    p.scores_stay = B * kv_heads * group * p.map.capacity() * 4 <= (32 << 20);
    p.scores = reinterpret_cast<float*>(static_cast<char*>(scratch) + up256(B * kv_heads * group * 4));
  }
  cudaStream_t st = (cudaStream_t)stream;
  TFB_DISPATCH_16(dtype, T, {
    if (hd == 32) return pg_dispatch<T, 32>(p, dtype, st);
    if (hd == 64) return pg_dispatch<T, 64>(p, dtype, st);
    return pg_dispatch<T, 128>(p, dtype, st);
  })
}
