// Attention of one new token per sequence over a paged key-value cache (sm_100a).
//
//   s_hj = q_h . k_j / sqrt(hd) - slope_h (p - p_j),  w_h = softmax_j(s_h),  o_h = sum_j w_hj v_j,
//   and for eviction  mass_j += sum of w_hj over the query heads h that share the key head.
//
// Every key and value row is used by one group of query heads only, so the pass is bound by reading the rows once; the
// products, padded to the 8 heads of a tensor-core instruction, are far below what the instruction can do.
//
// Split.  The keys of a (sequence, key head, tile of query heads) are cut into tiles of 4 KB of keys and 4 KB of values, all
// tiles of all sequences are numbered in one line, and each warp of the grid takes an equal stretch of that line, wherever
// sequences begin and end: lengths that differ by orders of magnitude leave no SM idle, one sequence alone fills the machine,
// and the lengths never have to be known on the host.  A warp works by itself: its own ring of tiles in shared memory, filled
// ahead and across the borders of sequences, no barrier of the block in the loop.  A row of scores that ends in the warp it
// began in is written out; the pieces of the others meet at the end of the block; what does not begin and end in one block goes
// to a workspace, where the last of its blocks joins the pieces, always in their order (the result does not depend on timing).
// Only masses need a second kernel: a key's weight is known once its row's sum is.
//
// Measured (bf16, head_dim 128): 2 sequences of 49157 keys, 12 heads, 99.7 us, 6.06 TB/s (93% of a copy); 64 sequences of up to 8192
// keys, 8 key heads of 8 query heads, with masses, 214 us, of which the first kernel takes some 190 at 5.8 TB/s.  Head_dim 64, fp16: 24
// sequences of up to 2048 keys, 16 heads, slopes and masses 32.7 us; one of 700 keys, 12 heads, 9.9 us.
//
// Copies.  Where pages and tiles share a divisor of 8 rows or more, TMA boxes of that many rows, which also swizzle the rows
// for ldmatrix; other page sizes take cp.async row by row.
//
// Products.  S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16, keys (or head_dim) along M and query heads along N: a tile
// of 8 heads wastes less than one of 16, and P^T comes out of the first product's registers by a transposition of 8x8
// blocks (movmatrix).  tcgen05 has no place here: its smallest M would be fed from shared memory that the CUDA cores have to
// write P into, and nothing waits for the tensor core.
#include <cfloat>
#include "attn.cuh"
#include "paged.cuh"
#include "tc05.cuh"

namespace tfb {
namespace {

constexpr int PG_WARPS = 8;
// Probabilities are kept relative to a reference that the running maximum may pass by 2^15 before everything is rescaled
// (they then still fit fp16); a new reference is 2^4 below the maximum, so that small ones stay clear of fp16's subnormals.
constexpr float kAhead = 15.f, kBelow = 4.f;
constexpr float kNone = -INFINITY;

// What beginning a row of scores costs a warp, in tiles: rows of a tile or two would otherwise pile up in a few warps.
constexpr int kRowCost = 4;

// G: query heads that a warp takes at once, 4, 8 or 16.
template <int HD, int G, int BIAS> struct PgCfg {
  static constexpr int NT = G == 16 ? 2 : 1;   // blocks of 8 columns in the products
  static constexpr int KEYS = 2048 / HD;       // keys of a tile
  static constexpr int MT = KEYS / 16;
  static constexpr int R = 8 * NT;             // query heads of a head tile
  static constexpr int CHUNKS = HD / 8;        // 16-byte chunks of a row
  static constexpr int RPI = 32 / CHUNKS;      // rows that a warp copies with one cp.async
  static constexpr int ITERS = KEYS / RPI;     // 8
  static constexpr int OWN = (KEYS + 31) / 32; // keys whose place a lane looks up
  static constexpr int TILE = KEYS * HD * 2;   // bytes of the keys of a tile (4096)
  static constexpr int PANELS = HD == 128 ? 2 : 1;  // parts of a row of at most 128 bytes, one after the other
  static constexpr int STAGES = 3;             // what 227 KB hold
  static constexpr int OFF_POS = PG_WARPS * STAGES * 2 * TILE;   // [warp][stage][KEYS] positions
  static constexpr int OFF_ML = OFF_POS + (BIAS ? PG_WARPS * STAGES * KEYS * 4 : 0);  // [warp][2][R] reference and sum of a piece
  static constexpr int OFF_BAR = OFF_ML + PG_WARPS * 2 * R * 8;  // [warp][stage]
  static constexpr int OFF_HEAD = OFF_BAR + 256;  // [warp][R][HD] the piece that a stretch begins in the middle of,
  static constexpr bool HEAD_SMEM = OFF_HEAD + PG_WARPS * R * HD * 4 + 1024 <= 226 * 1024 + 256;  // if that fits (else in scratch)
  static constexpr int SMEM = OFF_HEAD + (HEAD_SMEM ? PG_WARPS * R * HD * 4 : 0) + 1024;
  static_assert(R * HD * 4 <= STAGES * 2 * TILE, "a piece fits its warp's ring");
  static_assert(PG_WARPS * STAGES * 8 <= 256 && SMEM <= 227 * 1024 - 700, "shared memory");
};

struct PgParams {
  PageMap map;
  const void *q, *k_new, *v_new;
  void *out, *k, *v;
  const int *lengths, *query_positions;
  int* positions;
  const float* mass;
  float* mass_out;
  const float* slopes;
  int bias_mode;  // as in AttnArgs: 0 none, 1 exact, 2 / 4 rounded
  int64_t q_b, q_h, kn_b, kn_h, vn_b, vn_h, o_b, o_h;
  int B, kv_heads, group, row_tiles;
  int box_log2;   // rows of a TMA box
  int q_pairs;    // the queries can be read 4 bytes at a time
  int new_vec;    // the new rows can be read 16 bytes at a time
  int ctas;       // of the split kernel's grid
  float scale;    // log2(e) / sqrt(hd)
  int* arrived;     // [ctas] how many blocks have left their pieces of the row that this one begins; zero between calls
  float* lse;       // (B, kv_heads * group) log2 of the sum of exponentials, where masses are wanted
  float2* ml;       // [2 * ctas][R] reference and sum of a piece
  float* acc;       // [2 * ctas][R][hd]
  float* heads_acc; // [ctas][warps][R][hd] the pieces that a warp's stretch begins in the middle of
  float* scores;    // (B, kv_heads, capacity, group) in log2 units, or null
  int scores_stay;  // they fit the L2
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {  // the rest of the 16 is zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A box is read once.  Where the scores stay in the L2 until they are read again, it leaves the L2 before they do (24 sequences of
// up to 2048 keys: 35.1 us without, 33.6 with it); elsewhere that costs (2 of 49157 keys: 100.5 without, 102.4 with it).
__device__ __forceinline__ uint64_t read_once(bool leave) {
  uint64_t first, normal;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
  asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(normal));
  return leave ? first : normal;
}
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6}], [%2], %7;"
      ::"r"(smem_u32(dst)), "l"(m), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An infinite or missing number as the nearest finite one or the lowest: on top of a sum that is not finite either it changes nothing.
__device__ __forceinline__ float finite(float x) { return fminf(fmaxf(x, -FLT_MAX), FLT_MAX); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const typename Num<T>::T2 v = Num<T>::from_f2(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Byte offset of 16-byte chunk `c` of row `row` of a tile, swizzled as TMA does it (128 bytes wide, at head_dim 32 64): the chunk
// number is xor-ed with the row, so that the eight rows of an ldmatrix lie in different banks.
template <int HD> __device__ __forceinline__ uint32_t tile_at(int row, int c) {
  if (HD == 32) return (uint32_t)(row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
  return (uint32_t)((c >> 3) * (2048 / HD) * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

// Keys of a sequence, and the slot of its new one (-1: none; otherwise the last).
struct SeqKeys {
  int n, fresh;
  __device__ __forceinline__ int cached() const { return fresh >= 0 ? fresh : n; }
};
__device__ __forceinline__ SeqKeys keys_of(const PgParams& p, int len) {
  const int cap = (int)p.map.capacity();
  SeqKeys s;
  s.fresh = p.k_new && len >= 0 && len < cap ? len : -1;
  s.n = min(max(len, 0) + (s.fresh >= 0), cap);
  return s;
}

// A place in the line: sequence, (key head, head tile), tile, and its distance from the stretch's beginning.
template <int KEYS>
struct Cursor {
  int b, hr, j, tiles, at;
  SeqKeys keys;
  __device__ __forceinline__ void load(const PgParams& p) {
    keys = keys_of(p, p.lengths[b]);
    tiles = (keys.n + KEYS - 1) / KEYS;
  }
  // to the first tile of the next row of scores; false if there is none
  __device__ __forceinline__ bool next_row(const PgParams& p) {
    at += kRowCost;
    j = 0;
    if (++hr < p.kv_heads * p.row_tiles) return true;
    hr = 0;
    do {
      if (++b >= p.B) return false;
      load(p);
    } while (tiles == 0);
    return true;
  }
  // to the next tile, which there has to be
  __device__ __forceinline__ void step(const PgParams& p) {
    ++at;
    if (++j == tiles) next_row(p);
  }
};

__device__ __forceinline__ int64_t divide(int64_t n, int64_t d) {  // of values that are not negative
  return ((n | d) >> 32) == 0 ? (int64_t)((uint32_t)n / (uint32_t)d) : n / d;
}
// The line has kRowCost units and one for each tile of a row, and is cut into equal stretches, one for each warp (with fewer
// units than warps, of one unit): the first `more` have a unit more than `each`.
struct Line {
  int64_t units, each, more, parts;
  __device__ __forceinline__ Line(int64_t units_, int ctas) : units(units_), parts(min(units_, (int64_t)ctas * PG_WARPS)) {
    each = parts ? divide(units, parts) : 0;
    more = units - each * parts;
  }
  __device__ __forceinline__ int64_t begin(int64_t part) const { return part < parts ? part * each + min(part, more) : units; }
  // the block whose warps have unit t
  __device__ __forceinline__ int block_of(int64_t t) const {
    const int64_t wide = more * (each + 1);
    return (int)((t < wide ? divide(t, each + 1) : more + divide(t - wide, each)) / PG_WARPS);
  }
};
__device__ __forceinline__ int row_units(int tiles) { return tiles ? tiles + kRowCost : 0; }

__device__ __forceinline__ float alibi_rounded_log2(int mode, float slope, float dist) {  // slope already rounded
  const int drop = mode == 2 ? 13 : 16;
  return -round_significand(round_significand(dist, drop) * slope, drop) * kLog2e;
}

// What a block knows of its warps' pieces when it joins them.
struct Pieces {
  int64_t begin[PG_WARPS][2];  // the piece's row's first tile in the line
  int b[PG_WARPS][2], hr[PG_WARPS][2], tiles[PG_WARPS][2];
  uint8_t flags[PG_WARPS];  // bit 0: there is a piece [0], which began before the warp's stretch; 1: a piece [1], which goes on
};                          // behind it; 2: piece [0] is its row's last

}  // namespace

// BIAS: 0 none, 1 exact slopes, 2 slopes rounded as a table's
template <typename T, int HD, int G, int BIAS, bool TMA>
__global__ void __launch_bounds__(PG_WARPS * 32, 1) paged_attn_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                      const __grid_constant__ CUtensorMap tmV, const PgParams p) {
  using C = PgCfg<HD, G, BIAS>;
  constexpr int NT = C::NT, R = C::R, STAGES = C::STAGES, STAGE = 2 * C::TILE, KS = HD / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int64_t sh_scan[PG_WARPS], sh_base[PG_WARPS];
  __shared__ int sh_b[PG_WARPS];
  __shared__ __align__(8) Pieces sh;
  __shared__ int sh_abort, sh_last[2], sh_first[2];
  volatile int* abort_flag = &sh_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.kv_heads * p.row_tiles;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR) + warp * STAGES;

  if (TMA && lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0) sh.flags[warp] = 0;
  if (TMA && threadIdx.x == 32) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  __syncthreads();
  grid_dependency_wait();
  allow_dependents();

  // What one block of the grid does beside its stretches for sequence b: a report, zeros where there are no keys.
  auto look_over = [&](int b, int len, int tiles) {
    if (b % (int)gridDim.x != (int)blockIdx.x) return;
    if (len < 0 || (int64_t)len + (p.k_new ? 1 : 0) > p.map.capacity()) atomicCAS(&g_dev_status, 0, kBadLength);
    if (tiles == 0) {
      T* out = static_cast<T*>(p.out) + b * p.o_b;
      for (int h = 0; h < p.kv_heads * p.group; ++h)
        for (int d = 0; d < HD; ++d) out[h * p.o_h + d] = Num<T>::from_f(0.f);
    }
  };
  // ---- the warps' stretches: a scan over the sequences' units
  const int64_t part = (int64_t)blockIdx.x * PG_WARPS + warp;
  Line line(0, 0);
  int start_b = 0;
  int64_t start_base = 0;  // the units before it
  if (p.B <= 32) {         // each warp by itself: no barrier, one load (one user 10.0 us, with the scan below 10.9)
    const int len = lane < p.B ? p.lengths[lane] : 0;
    const int tiles = lane < p.B ? (keys_of(p, len).n + C::KEYS - 1) / C::KEYS : 0;
    const uint32_t mine = row_units(tiles);
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    line = Line((int64_t)__shfl_sync(0xffffffffu, upto, 31) * heads, p.ctas);
    const unsigned behind = __ballot_sync(0xffffffffu, (int64_t)upto * heads > line.begin(part));
    start_b = behind ? __ffs(behind) - 1 : 0;
    start_base = (int64_t)__shfl_sync(0xffffffffu, upto - mine, start_b) * heads;
    if (warp == 0 && lane < p.B) look_over(lane, len, tiles);
  } else {
    const int per = (p.B + PG_WARPS * 32 - 1) / (PG_WARPS * 32);
    const int b_lo = min((int)threadIdx.x * per, p.B), b_hi = min(b_lo + per, p.B);
    int64_t mine = 0;
    for (int b = b_lo; b < b_hi; ++b) mine += row_units((keys_of(p, p.lengths[b]).n + C::KEYS - 1) / C::KEYS);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sh_scan[warp] = upto;
    __syncthreads();
    int64_t base = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < PG_WARPS; ++w) {
      const int64_t v = sh_scan[w];
      if (w < warp) base += v;
      total += v;
    }
    line = Line(total * heads, p.ctas);
    for (int b = b_lo; b < b_hi; ++b) {
      const int len = p.lengths[b];
      const int tiles = (keys_of(p, len).n + C::KEYS - 1) / C::KEYS;
      look_over(b, len, tiles);
#pragma unroll 1
      for (int w = 0; w < PG_WARPS; ++w) {
        const int64_t f = line.begin((int64_t)blockIdx.x * PG_WARPS + w);
        if (f >= base * heads && f < (base + row_units(tiles)) * heads) {
          sh_b[w] = b;
          sh_base[w] = base * heads;
        }
      }
      base += row_units(tiles);
    }
    __syncthreads();
    start_b = sh_b[warp];
    start_base = sh_base[warp];
  }
  if (line.begin((int64_t)blockIdx.x * PG_WARPS) >= line.units) return;  // nothing for this block
  const int64_t from = line.begin(part);
  const int length = (int)(line.begin(part + 1) - from);

  uint8_t* ring = smem + warp * STAGES * STAGE;
  const uint32_t ring_at = smem_u32(ring);
  uint8_t* places = smem + C::OFF_POS + warp * STAGES * C::KEYS * 4;
  float2* my_ml = reinterpret_cast<float2*>(smem + C::OFF_ML) + warp * 2 * R;
  auto head_piece = [&](int w) {
    return C::HEAD_SMEM ? reinterpret_cast<float*>(smem + C::OFF_HEAD) + w * (R * HD)
                        : p.heads_acc + ((int64_t)blockIdx.x * PG_WARPS + w) * (R * HD);
  };
  const int g8 = lane >> 2, j2 = 2 * (lane & 3);  // row of an 8x8 block, first of its two columns
  // The second product takes the probabilities in two parts of 16 bits: rounded, and what that leaves (64 sequences of 8 query heads a
  // key head: 1.2e-3 off in bf16, its own rounding; 1.6e-3 with the first part alone).  Up to four query heads the instruction's other
  // four columns repeat them and carry the rest; more heads take a second product (that case: 214 us, 219 without it, from a kernel
  // that chose between the two while it ran).
  constexpr bool FINE = G == 4, APART = G == 8;  // APART: in sums of its own, for more than 8 heads there are no registers
  const bool rest = FINE && j2 >= 4;

  Cursor<C::KEYS> cu;
  cu.at = length;
  if (length > 0) {
    cu.b = start_b;
    cu.load(p);
    const int64_t in = from - start_base;  // units of the sequence before the stretch
    const int units = row_units(cu.tiles);
    cu.hr = in < (1LL << 31) ? (int)((uint32_t)in / (uint32_t)units) : (int)(in / units);
    cu.j = (int)(in - (int64_t)cu.hr * units) - kRowCost;
    cu.at = max(-cu.j, 0);
    cu.j = max(cu.j, 0);
  }
  if (cu.at < length) {
    Cursor<C::KEYS> ld = cu;

    // Page and row of what this lane looks up, one tile ahead of the copies: box `lane` of the tile, or keys lane, lane + 32.
    int page[C::OWN], row[C::OWN];
    auto look_up = [&]() {
#pragma unroll
      for (int u = 0; u < (TMA ? 1 : C::OWN); ++u) {
        const int kk = TMA ? lane << p.box_log2 : lane + 32 * u, slot = ld.j * C::KEYS + kk;
        page[u] = -1;
        row[u] = 0;
        if (kk < C::KEYS && slot < ld.keys.cached()) {
          const int i = (int)((unsigned)slot / (unsigned)p.map.page);
          row[u] = slot - i * p.map.page;
          page[u] = p.map.tables[ld.b * p.map.table_ld + i];
        }
      }
    };
    const uint64_t once = read_once(p.scores_stay);
    auto copy = [&](int stage) {
      const int head = ld.hr / p.row_tiles, cached = ld.keys.cached(), slot0 = ld.j * C::KEYS;
      if constexpr (TMA) {
        const int box = 1 << p.box_log2;
        const bool wanted = (lane << p.box_log2) < C::KEYS && slot0 + (lane << p.box_log2) < cached;
        const bool ok = wanted && (unsigned)page[0] < (unsigned)p.map.num_pages;
        const unsigned loads = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) mbar_expect_tx(&full[stage], __popc(loads) * box * HD * 4);
        __syncwarp();
        uint8_t* dst = ring + stage * STAGE + (lane << p.box_log2) * (HD == 32 ? 64 : 128);
        if (ok) {
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c) {
            load_box(dst + c * C::KEYS * 128, &tmK, c * 64, row[0], head, page[0], &full[stage], once);
            load_box(dst + C::TILE + c * C::KEYS * 128, &tmV, c * 64, row[0], head, page[0], &full[stage], once);
          }
        } else if (wanted) {  // no such page: zeros
          atomicCAS(&g_dev_status, 0, kBadPage);
          for (int kk = 0; kk < box; ++kk)
            for (int c = 0; c < C::CHUNKS; ++c) {
              const uint32_t o = stage * STAGE + tile_at<HD>((lane << p.box_log2) + kk, c);
              *reinterpret_cast<uint4*>(ring + o) = make_uint4(0, 0, 0, 0);
              *reinterpret_cast<uint4*>(ring + o + C::TILE) = make_uint4(0, 0, 0, 0);
            }
          fence_proxy_async_smem();
        }
        if (BIAS && p.positions) {
#pragma unroll
          for (int u = 0; u < C::OWN; ++u) {
            const int kk = lane + 32 * u, who = (kk >> p.box_log2) & 31;
            const int pg = __shfl_sync(0xffffffffu, page[0], who), r0 = __shfl_sync(0xffffffffu, row[0], who);
            if (kk < C::KEYS && (loads >> who & 1) != 0)
              cp4(smem_u32(places) + (stage * C::KEYS + kk) * 4,
                  p.positions + stat_offset(p.map, pg, p.kv_heads, head, r0 + (kk & (box - 1))), 4);
          }
          cp_commit();
        }
      } else {
        const uint32_t at = ring_at + stage * STAGE;
        int64_t off[C::OWN];
#pragma unroll
        for (int u = 0; u < C::OWN; ++u) {
          const int kk = lane + 32 * u;
          const bool wanted = kk < C::KEYS && slot0 + kk < cached;
          const bool ok = wanted && (unsigned)page[u] < (unsigned)p.map.num_pages;
          if (wanted && !ok) atomicCAS(&g_dev_status, 0, kBadPage);
          off[u] = ok ? row_offset(p.map, page[u], head, row[u]) : -1;
          if (BIAS && p.positions && kk < C::KEYS)
            cp4(smem_u32(places) + (stage * C::KEYS + kk) * 4,
                ok ? p.positions + stat_offset(p.map, page[u], p.kv_heads, head, row[u]) : p.positions, ok ? 4 : 0);
        }
        const T* k = static_cast<const T*>(p.k) + (lane % C::CHUNKS) * 8;
        const T* v = static_cast<const T*>(p.v) + (lane % C::CHUNKS) * 8;
#pragma unroll
        for (int i = 0; i < C::ITERS; ++i) {
          const int kk = i * C::RPI + lane / C::CHUNKS;
          const int64_t o = __shfl_sync(0xffffffffu, off[(i * C::RPI) / 32], kk & 31);
          const uint32_t dst = at + tile_at<HD>(kk, lane % C::CHUNKS);
          cp16(dst, k + (o < 0 ? 0 : o), o < 0 ? 0 : 16);
          cp16(dst + C::TILE, v + (o < 0 ? 0 : o), o < 0 ? 0 : 16);
        }
        cp_commit();
      }
    };

    look_up();
    int into = 0;
    auto issue = [&]() {  // the next tile, if there is one; groups of cp.async are counted either way
      if (ld.at < length) {
        copy(into);
        if (++into == STAGES) into = 0;
        ld.step(p);
        if (ld.at < length) look_up();
      } else if (!TMA || (BIAS && p.positions)) {
        cp_commit();
      }
    };

    // What a row of scores needs beside its keys is read while the row before it is worked on: the query, the slopes, the
    // query's position, and 16 bytes of the new token's rows with the page that they go to.
    struct Row {
      uint32_t q[NT][KS][2];
      float slope[NT][2];
      int here, page;
      uint4 fresh;
    };
    auto fetch = [&](const Cursor<C::KEYS>& c, Row& w) {
      const int kv = c.hr / p.row_tiles, r0 = (c.hr - kv * p.row_tiles) * R;
      const T* q = static_cast<const T*>(p.q) + c.b * p.q_b;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + (FINE ? g8 & 3 : nt * 8 + g8);
        const T* qr = q + (int64_t)(kv * p.group + r) * p.q_h + j2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t v = 0;
            if (r < p.group) {
              const T* at = qr + ks * 16 + half * 8;
              if (p.q_pairs) v = *reinterpret_cast<const uint32_t*>(at);
              else v = (uint32_t)*reinterpret_cast<const uint16_t*>(at) |
                       (uint32_t)*reinterpret_cast<const uint16_t*>(at + 1) << 16;
            }
            w.q[nt][ks][half] = v;
          }
        if (BIAS)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int rr = r0 + (FINE ? (j2 + e) & 3 : nt * 8 + j2 + e);
            w.slope[nt][e] = rr < p.group ? p.slopes[kv * p.group + rr] : 0.f;
          }
      }
      if (BIAS) w.here = p.query_positions ? p.query_positions[c.b] : c.keys.n - 1;
      w.fresh = make_uint4(0, 0, 0, 0);
      w.page = -1;
      if (c.keys.fresh >= 0) {
        w.page = p.map.tables[c.b * p.map.table_ld + (unsigned)c.keys.fresh / (unsigned)p.map.page];
        if (lane < 2 * C::CHUNKS) {
          const T* at = lane < C::CHUNKS ? static_cast<const T*>(p.k_new) + c.b * p.kn_b + kv * p.kn_h + lane * 8
                                         : static_cast<const T*>(p.v_new) + c.b * p.vn_b + kv * p.vn_h + (lane - C::CHUNKS) * 8;
          if (p.new_vec) w.fresh = *reinterpret_cast<const uint4*>(at);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              reinterpret_cast<uint32_t*>(&w.fresh)[e] = (uint32_t)*reinterpret_cast<const uint16_t*>(at + 2 * e) |
                                                         (uint32_t)*reinterpret_cast<const uint16_t*>(at + 2 * e + 1) << 16;
        }
      }
    };
    Row now, ahead;
    Cursor<C::KEYS> rows = cu;  // the row of `ahead`

    // where ldmatrix reads: chunk 0 of the lane's row; the chunk number's higher bits are xor-ed in
    const int mi = lane >> 3, l8 = lane & 7;
    const uint32_t k_at = tile_at<HD>((mi & 1) * 8 + l8, mi >> 1), v_at = tile_at<HD>((mi >> 1) * 8 + l8, mi & 1) + C::TILE;
    constexpr int PER_PANEL = HD == 32 ? 2 : 4;  // k-steps in a row of at most 128 bytes
    constexpr uint32_t BLOCK16 = 16 * (HD == 32 ? 64 : 128), PANEL = C::KEYS * 128;

    float ref[NT][2], sum[NT][2], o[KS][NT][4], o_rest[APART ? KS : 1][4];
    int first = 0;  // whether the piece began with its row's first tile
    bool begin = true;
    int stage = 0, warm_up = STAGES - 1;  // tiles to copy before the first one is worked on
    int fetches = 2;                      // of the next row's things; for the first row also its own
    uint32_t phase = 0;

    // (Code that runs once or twice in a short call costs its way from the L2 into the instruction cache, so the copies and
    // the fetch stand here once each.)
    for (;;) {
      if (begin && warm_up == 0) {
        begin = false;
        first = cu.j == 0;
#pragma unroll 1
        for (; fetches > 0; --fetches) {
          now = ahead;
          if (fetches == 2 || (cu.at + cu.tiles - cu.j + kRowCost < length && rows.next_row(p))) fetch(rows, ahead);
        }
        fetches = 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (BIAS) {
              float& sl = now.slope[nt][e];
              if (BIAS == 1) sl *= -kLog2e;
              if (p.bias_mode == 2) sl = __half2float(__float2half_rn(sl));
              if (p.bias_mode == 4) sl = __bfloat162float(__float2bfloat16_rn(sl));
            }
            ref[nt][e] = kNone;
            sum[nt][e] = 0.f;
          }
#pragma unroll
        for (int m = 0; m < KS; ++m)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][nt][e] = 0.f;
        if (APART)
#pragma unroll
          for (int m = 0; m < KS; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o_rest[m][e] = 0.f;
      }
      if (warm_up == 0) {
        if (!TMA || (BIAS && p.positions)) cp_wait<STAGES - 2>();
        if (TMA && !__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, 0x9000 | stage, abort_flag))) break;
        __syncwarp();
      }
      issue();  // into the stage that the tile before this one has left
      if (warm_up > 0) {
        --warm_up;
        continue;
      }
      const uint32_t tile = ring_at + stage * STAGE;
      const int slot0 = cu.j * C::KEYS, cached = cu.keys.cached();
      const bool ragged = slot0 + C::KEYS > cached;
      if (ragged) {  // rows behind the last cached key may hold anything; the new token's are not in the pages yet
        const int kv = cu.hr / p.row_tiles;
        uint8_t* at = ring + stage * STAGE;
        for (int i = lane; i < (C::KEYS - (cached - slot0)) * C::CHUNKS; i += 32) {
          const uint32_t dst = tile_at<HD>(cached - slot0 + i / C::CHUNKS, i % C::CHUNKS);
          *reinterpret_cast<uint4*>(at + dst) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(at + dst + C::TILE) = make_uint4(0, 0, 0, 0);
        }
        const int kk = cu.keys.fresh - slot0;  // at least 0, because there is a cached key in every tile before it
        if (cu.keys.fresh >= 0 && kk < C::KEYS) {
          __syncwarp();
          const int c = lane % C::CHUNKS;
          if (lane < 2 * C::CHUNKS) *reinterpret_cast<uint4*>(at + tile_at<HD>(kk, c) + (lane < C::CHUNKS ? 0 : C::TILE)) = now.fresh;
          if (cu.hr == kv * p.row_tiles) {  // one of the row's head tiles writes it into its slot
            const int r0 = cu.keys.fresh % p.map.page;
            if ((unsigned)now.page < (unsigned)p.map.num_pages) {
              if (lane < 2 * C::CHUNKS)
                *reinterpret_cast<uint4*>(static_cast<T*>(lane < C::CHUNKS ? p.k : p.v) + row_offset(p.map, now.page, kv, r0) + c * 8) =
                    now.fresh;
              if (p.positions && lane == 0)
                p.positions[stat_offset(p.map, now.page, p.kv_heads, kv, r0)] =
                    p.query_positions ? p.query_positions[cu.b] : cu.keys.fresh;
            } else {
              atomicCAS(&g_dev_status, 0, kBadPage);
            }
          }
        }
        if (TMA) fence_proxy_async_smem();
        __syncwarp();
      }

      // ---- scores: keys g8 and g8 + 8 of each block of 16, heads j2 and j2 + 1
      float s[C::MT][NT][4];
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[m][nt][e] = 0.f;
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int m = 0; m < C::MT; ++m) {
          uint32_t a[4];
          ldm4(a, tile + (k_at ^ ((ks % PER_PANEL) << 5)) + (ks / PER_PANEL) * PANEL + m * BLOCK16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<T>(s[m][nt], a, now.q[nt][ks][0], now.q[nt][ks][1]);
        }
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = kNone;
      const int* place = reinterpret_cast<const int*>(places) + stage * C::KEYS;
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int kk = m * 16 + half * 8 + g8;
          float dist = 0.f;
          if (BIAS) dist = (float)(now.here - (p.positions ? place[kk] : slot0 + kk));
          if (BIAS && ragged && slot0 + kk == cu.keys.fresh) dist = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = s[m][nt][2 * half + e] * p.scale;
              if (BIAS == 1) x = fmaf(now.slope[nt][e], dist, x);
              if (BIAS == 2) x += alibi_rounded_log2(p.bias_mode, now.slope[nt][e], dist);
              s[m][nt][2 * half + e] = x;
            }
        }
      if (ragged) {
#pragma unroll
        for (int m = 0; m < C::MT; ++m)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            if (slot0 + m * 16 + half * 8 + g8 >= cu.keys.n)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) s[m][nt][2 * half] = s[m][nt][2 * half + 1] = kNone;
      }
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) top[nt][e] = fmaxf(top[nt][e], fmaxf(s[m][nt][e], s[m][nt][2 + e]));
      if (p.scores) {
        const int kv = cu.hr / p.row_tiles, r0 = (cu.hr - kv * p.row_tiles) * R + j2;
        float* sc = p.scores + (((int64_t)cu.b * p.kv_heads + kv) * p.map.capacity() + slot0 + g8) * p.group + r0;
        const int left = ragged ? cu.keys.n - slot0 - g8 : C::KEYS;  // keys from this lane's first on
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (r0 + nt * 8 + e < p.group)
#pragma unroll
              for (int m = 0; m < C::MT; ++m)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                  if (m * 16 + half * 8 < left) sc[(m * 16 + half * 8) * p.group + nt * 8 + e] = s[m][nt][2 * half + e];
      }
      // ---- a new reference where the maximum has run away from the old one
      bool away = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) away |= top[nt][0] > ref[nt][0] + kAhead || top[nt][1] > ref[nt][1] + kAhead;
      if (__any_sync(0xffffffffu, away)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[nt][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            if (x > ref[nt][e] + kAhead) {
              const float f = ref[nt][e] == kNone ? 0.f : ex2(ref[nt][e] - (x - kBelow));
              ref[nt][e] = x - kBelow;
              sum[nt][e] *= f;
#pragma unroll
              for (int m = 0; m < KS; ++m) {
                o[m][nt][e] *= f;
                o[m][nt][2 + e] *= f;
                if (APART) {
                  o_rest[m][e] *= f;
                  o_rest[m][2 + e] *= f;
                }
              }
            }
          }
      }
      // ---- probabilities for the second product: rounded to the values' type (pt), and what that leaves, rounded too (rt); the sum
      // takes them unrounded
      uint32_t pt[C::MT][NT][2], rt[C::MT][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float from_ref[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) from_ref[e] = ref[nt][e] == kNone ? 0.f : ref[nt][e];
#pragma unroll
        for (int m = 0; m < C::MT; ++m)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float w[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              w[e] = ex2(s[m][nt][2 * half + e] - from_ref[e]);
              sum[nt][e] += w[e];
            }
            const uint32_t u = pack2<T>(w[0], w[1]);
            uint32_t left = u;
            if (!FINE || rest) {
              const float2 f = Num<T>::to_f2(*reinterpret_cast<const typename Num<T>::T2*>(&u));
              left = pack2<T>(w[0] - f.x, w[1] - f.y);
            }
            pt[m][nt][half] = transpose8(FINE ? left : u);
            if (!FINE) rt[m][nt][half] = transpose8(left);
          }
      }
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int hm = 0; hm < KS; ++hm) {
          uint32_t a[4];
          ldm4t(a, tile + (v_at ^ ((hm % PER_PANEL) << 5)) + (hm / PER_PANEL) * PANEL + m * BLOCK16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<T>(o[hm][nt], a, pt[m][nt][0], pt[m][nt][1]);
          if (APART) mma<T>(o_rest[hm], a, rt[m][0][0], rt[m][0][1]);
        }
      if (!APART && !FINE) {
        // The rests' products on top, unless a value is infinite: a rest of zero or below would make NaN of that.
        float zero = 0.f;  // NaN if a sum is not finite
#pragma unroll
        for (int m = 0; m < KS; ++m)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) zero = fmaf(o[m][nt][e], 0.f, zero);
        if (!__any_sync(0xffffffffu, zero != zero))
#pragma unroll
          for (int m = 0; m < C::MT; ++m)
#pragma unroll
            for (int hm = 0; hm < KS; ++hm) {
              uint32_t a[4];
              ldm4t(a, tile + (v_at ^ ((hm % PER_PANEL) << 5)) + (hm / PER_PANEL) * PANEL + m * BLOCK16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<T>(o[hm][nt], a, rt[m][nt][0], rt[m][nt][1]);
            }
      }
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }

      // ---- the end of a row of scores, or of the stretch
      const bool last = cu.j + 1 == cu.tiles;
      const int row_at = cu.at - cu.j, row_b = cu.b, row_hr = cu.hr, row_tiles = cu.tiles;
      cu.step(p);
      const bool done = cu.at >= length;
      if (last || done) {
        begin = true;
        const int kv = row_hr / p.row_tiles, r0 = (row_hr - kv * p.row_tiles) * R;
        const bool whole = first && last;
        // a piece: [0] one that began before the stretch, in scratch while the ring is in use; [1] the stretch's last, over the ring
        float* acc = first ? reinterpret_cast<float*>(ring) : head_piece(warp);
        if (!whole) {
          __syncwarp();  // the ring has been read
          if (lane == 0) {
            sh.flags[warp] |= first ? 2 : last ? 5 : 1;
            sh.begin[warp][first] = from + row_at;
            sh.b[warp][first] = row_b;
            sh.hr[warp][first] = row_hr;
            sh.tiles[warp][first] = row_tiles;
          }
        }
        if (FINE) {  // the rests' products
#pragma unroll
          for (int m = 0; m < KS; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][0][e] += finite(__shfl_xor_sync(0xffffffffu, o[m][0][e], 2));
        } else if (APART) {
#pragma unroll
          for (int m = 0; m < KS; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[m][0][e] += finite(o_rest[m][e]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float l = sum[nt][e];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
            const int r = nt * 8 + j2 + e;
            if (r0 + r < p.group) {
              const int64_t head = kv * p.group + r0 + r;
              if (whole) {
                const float inv = l > 0.f ? 1.f / l : l;  // a row whose weights are all zero is zero; NaN stays
                T* out = static_cast<T*>(p.out) + row_b * p.o_b + head * p.o_h;
#pragma unroll
                for (int m = 0; m < KS; ++m) {
                  out[m * 16 + g8] = Num<T>::from_f(o[m][nt][e] * inv);
                  out[m * 16 + 8 + g8] = Num<T>::from_f(o[m][nt][2 + e] * inv);
                }
                if (p.lse && g8 == 0) p.lse[(int64_t)row_b * p.kv_heads * p.group + head] = ref[nt][e] + __log2f(l);
              } else {
#pragma unroll
                for (int m = 0; m < KS; ++m) {
                  acc[r * HD + m * 16 + g8] = o[m][nt][e];
                  acc[r * HD + m * 16 + 8 + g8] = o[m][nt][2 + e];
                }
                if (g8 == 0) my_ml[first * R + r] = make_float2(ref[nt][e], l);
              }
            }
          }
        if (done) break;
      }
    }
    cp_wait<0>();
  }

  // ---- the block joins its warps' pieces
  __syncthreads();
  if (*abort_flag) {
    for (int k = 0; k < 64; ++k) __nanosleep(1000);
    return;
  }
  const float2* ml = reinterpret_cast<const float2*>(smem + C::OFF_ML);
  const uint64_t flags = *reinterpret_cast<const uint64_t*>(sh.flags);
  // bit w: of warp w
  auto bits = [&](int bit) {  // bit `bit` of each byte, gathered
    return (unsigned)(((flags >> bit & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);
  };
  const unsigned has0 = bits(0), has1 = bits(1), ends = bits(2);
  // A chain of pieces starts with a piece [1], or with the piece [0] that has none before it in this block: only the first can.
  const unsigned lead = has0 & (0u - has0);                             // the first warp with a piece [0]
  const bool leads = lead != 0 && (has1 & (lead - 1u)) == 0;            // and nothing goes on into it
  const int chains = __popc(has1) + leads, rows_most = min(R, p.group);
  int open0 = -1, open1 = -1;  // the first warps of the chains that begin, or end, in another block
  auto end_of = [&](int w, int slot) {  // a chain's last warp
    int end = w;
    bool ended = slot == 0 && (ends >> w & 1) != 0;
    while (!ended && end + 1 < PG_WARPS && (has0 >> (end + 1) & 1) != 0) ended = (ends >> ++end & 1) != 0;
    return ended ? end : end | 64;  // 64: the row goes on in the next block
  };
  if (leads) open0 = __ffs(lead) - 1;
  if (has1 != 0) {  // only the last chain can go on
    const int w = 31 - __clz(has1);
    if (end_of(w, 1) & 64) open1 = w;
  }
  for (int job = warp; job < chains * rows_most; job += PG_WARPS) {
    const int chain = job / rows_most, r = job - chain * rows_most;
    const int slot = leads && chain == 0 ? 0 : 1;
    int w = open0;
    if (slot == 1) {
      unsigned left = has1;
      for (int i = chain - leads; i > 0; --i) left &= left - 1u;
      w = __ffs(left) - 1;
    }
    const int end = end_of(w, slot) & 63;
    const bool whole = slot == 1 && w != open1;
    {
      const int b = sh.b[w][slot], hr = sh.hr[w][slot];
      const int kv = hr / p.row_tiles, r0 = (hr - kv * p.row_tiles) * R;
      if (r0 + r < p.group) {
        float m = kNone, l = 0.f, a[HD / 32];
        for (int i = w; i <= end; ++i) m = fmaxf(m, ml[(i * 2 + (i == w ? slot : 0)) * R + r].x);
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) a[e] = 0.f;
#pragma unroll(C::HEAD_SMEM ? 1 : 4)
        for (int i = w; i <= end; ++i) {
          const int which = i == w ? slot : 0;
          const float2 v = ml[(i * 2 + which) * R + r];
          const float* acc = (which ? reinterpret_cast<const float*>(smem + i * STAGES * STAGE) : head_piece(i)) + r * HD;
          const float f = v.x == kNone ? 0.f : ex2(v.x - m);
          l += v.y == v.y ? v.y * f : v.y;
          if (v.x != kNone)
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) a[e] += acc[e * 32 + lane] * f;
        }
        const int64_t head = kv * p.group + r0 + r;
        if (whole) {
          const float inv = l > 0.f ? 1.f / l : l;
          T* out = static_cast<T*>(p.out) + b * p.o_b + head * p.o_h;
#pragma unroll
          for (int e = 0; e < HD / 32; ++e) out[e * 32 + lane] = Num<T>::from_f(a[e] * inv);
          if (p.lse && lane == 0) p.lse[(int64_t)b * p.kv_heads * p.group + head] = m + __log2f(l);
        } else {
          const int64_t piece = 2 * (int64_t)blockIdx.x + slot;
#pragma unroll
          for (int e = 0; e < HD / 32; ++e) p.acc[(piece * R + r) * HD + e * 32 + lane] = a[e];
          if (lane == 0) p.ml[piece * R + r] = make_float2(m, l);
        }
      }
    }
  }
  if (open0 < 0 && open1 < 0) return;

  // ---- rows that several blocks share: the block that comes last joins their pieces.  A block begins at most one such row,
  // whose counter is the block's.
  __syncthreads();
  if (warp < 2 && lane == 0) {
    const int slot = warp, w = slot ? open1 : open0;
    sh_last[slot] = 0;
    if (w >= 0) {
      const int64_t t0 = sh.begin[w][slot];
      const int c0 = line.block_of(t0), c1 = line.block_of(t0 + sh.tiles[w][slot] - 1);
      int before;
      asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrived + c0) : "memory");
      if (before == c1 - c0) {
        p.arrived[c0] = 0;
        sh_last[slot] = c1 - c0 + 1;
        sh_first[slot] = c0;
      }
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int slot = 0; slot < 2; ++slot) {
    const int pieces = sh_last[slot], c0 = sh_first[slot];
    if (!pieces) continue;
    const int w = slot ? open1 : open0, b = sh.b[w][slot], hr = sh.hr[w][slot];
    const int kv = hr / p.row_tiles, r0 = (hr - kv * p.row_tiles) * R, rows = min(R, p.group - r0);
    // threads along (row, 4 columns), and what is left of them along the pieces, up to a share for 8 pieces
    constexpr int N = 8, THREADS = PG_WARPS * 32;
    const int cols = rows * (HD / 4), shares = max(1, min(THREADS / cols, (pieces + N - 1) / N));
    float4* part = reinterpret_cast<float4*>(smem);            // [THREADS]
    float2* part_ml = reinterpret_cast<float2*>(part + THREADS);  // [THREADS]
    for (int i0 = 0; i0 < cols; i0 += THREADS) {
      const int i = shares > 1 ? threadIdx.x % cols : i0 + threadIdx.x, share = shares > 1 ? threadIdx.x / cols : 0;
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float m = kNone, l = 0.f;
      auto add = [&](const float2& v, const float4& x) {  // a piece to what there is
        const float top = fmaxf(m, v.x);
        const float keep = m == kNone ? 0.f : ex2(m - top), f = v.x == kNone ? 0.f : ex2(v.x - top);
        l = (l == l ? l * keep : l) + (v.y == v.y ? v.y * f : v.y);
        a.x = a.x * keep + (v.x == kNone ? 0.f : x.x * f);
        a.y = a.y * keep + (v.x == kNone ? 0.f : x.y * f);
        a.z = a.z * keep + (v.x == kNone ? 0.f : x.z * f);
        a.w = a.w * keep + (v.x == kNone ? 0.f : x.w * f);
        m = top;
      };
      if (i < cols && share < shares) {
#pragma unroll 1
        for (int k0 = share * N; k0 < pieces; k0 += shares * N) {
          float2 v[N];
          float4 x[N];
#pragma unroll
          for (int k = 0; k < N; ++k) {
            v[k] = make_float2(kNone, 0.f);
            if (k0 + k < pieces) {
              const int64_t piece = (int64_t)(2 * (c0 + k0 + k) + (k0 + k == 0)) * R + r;
              v[k] = __ldcg(p.ml + piece);
              x[k] = __ldcg(reinterpret_cast<const float4*>(p.acc + piece * HD + d));
            }
          }
#pragma unroll
          for (int k = 0; k < N; ++k) add(v[k], x[k]);
        }
      }
      if (shares > 1) {
        part[threadIdx.x] = a;
        part_ml[threadIdx.x] = make_float2(m, l);
        __syncthreads();
        if (threadIdx.x < cols)
#pragma unroll 1
          for (int k = 1; k < shares; ++k) add(part_ml[k * cols + i], part[k * cols + i]);
      }
      if (i < cols && share == 0) {
        const int64_t head = kv * p.group + r0 + r;
        T* out = static_cast<T*>(p.out) + b * p.o_b + head * p.o_h + d;
        const float inv = l > 0.f ? 1.f / l : l;
        out[0] = Num<T>::from_f(a.x * inv);
        out[1] = Num<T>::from_f(a.y * inv);
        out[2] = Num<T>::from_f(a.z * inv);
        out[3] = Num<T>::from_f(a.w * inv);
        if (p.lse && d == 0) p.lse[(int64_t)b * p.kv_heads * p.group + head] = m + __log2f(l);
      }
    }
    __syncthreads();
  }
}

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

// Workspace: counters, then the pieces of blocks and warps for the widest rows.  Scratch, for the masses: log-sum-exps, scores.
struct PgWorkspace {
  int64_t ml, acc, heads_acc, bytes;
};
PgWorkspace pg_workspace() {
  const int64_t n = sm_count(), R = 16, hd = 128;
  PgWorkspace s;
  s.ml = kCounterBytes;
  s.acc = s.ml + up256(2 * n * R * 8);
  s.heads_acc = s.acc + up256(2 * n * R * hd * 4);
  s.bytes = s.heads_acc + n * PG_WARPS * R * hd * 4;
  return s;
}

template <typename T, int HD, int G, int BIAS, bool TMA>
int pg_split(const CUtensorMap& tk, const CUtensorMap& tv, const PgParams& p, cudaStream_t st) {
  using C = PgCfg<HD, G, BIAS>;
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(paged_attn_kernel<T, HD, G, BIAS, TMA>, C::SMEM, done, "paged_attention")) return rc;
  launch_overlapped(paged_attn_kernel<T, HD, G, BIAS, TMA>, dim3(p.ctas), dim3(PG_WARPS * 32), C::SMEM, st, tk, tv, p);
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
