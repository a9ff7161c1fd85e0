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
#pragma once
#include <cfloat>
#include <type_traits>

#include "attn.cuh"
#include "nibbles.cuh"
#include "paged.cuh"
#include "tc05.cuh"

namespace tfb {
namespace {

// Probabilities are kept relative to a reference that the running maximum may pass by 2^15 before everything is rescaled
// (they then still fit fp16); a new reference is 2^4 below the maximum, so that small ones stay clear of fp16's subnormals.
constexpr float kAhead = 15.f, kBelow = 4.f;
constexpr float kNone = -INFINITY;

// G: query heads that a warp takes at once, 4, 8 or 16.  Q4: pages in 4 bits.
template <int HD, int G, int BIAS, bool Q4> struct PgCfg {
  // In 4 bits a warp's time is that of making 16-bit numbers, and a third warp for each scheduler fills its waits: one user 9.6
  // -> 8.3 us, 24 sequences of up to 2048 keys 22.1 -> 20.6, long ones the same; 16 warps' registers do not hold a tile's work.
  static constexpr int WARPS = Q4 ? 12 : 8;
  static constexpr int NT = G == 16 ? 2 : 1;   // blocks of 8 columns in the products
  static constexpr int KEYS = Q4 ? 64 : 2048 / HD;  // keys of a tile
  static constexpr int MT = KEYS / 16;
  static constexpr int R = 8 * NT;             // query heads of a head tile
  static constexpr int CHUNKS = HD / (Q4 ? 32 : 8);  // 16-byte chunks of a row
  static constexpr int RPI = 32 / CHUNKS;      // rows that a warp copies with one cp.async
  static constexpr int ITERS = KEYS / RPI;     // 8, and in 4 bits 2 or 4
  static constexpr int OWN = (KEYS + 31) / 32; // keys whose place a lane looks up
  static constexpr int TILE = KEYS * CHUNKS * 16;  // bytes of the keys of a tile (4096, and in 4 bits 1024 to 4096)
  static constexpr int PANELS = HD == 128 ? 2 : 1;  // parts of a row of at most 128 bytes, one after the other
  static constexpr int STAGES = Q4 ? 2 : 3;    // what 227 KB hold
  // What beginning a row of scores costs a warp, in tiles: rows of a tile or two would otherwise pile up in a few warps.  (In 4 bits a tile
  // has more keys and takes longer: 24 sequences of up to 2048 keys 22.2 us, with 4 24.3.)
  static constexpr int ROW_COST = Q4 ? 1 : 4;
  static constexpr int OFF_POS = WARPS * STAGES * 2 * TILE;   // [warp][stage][KEYS] positions, or scales
  static constexpr int OFF_ML = OFF_POS + (BIAS || Q4 ? WARPS * STAGES * KEYS * 4 : 0);  // [warp][2][R] reference and sum of a piece
  static constexpr int OFF_BAR = OFF_ML + WARPS * 2 * R * 8;  // [warp][stage]
  static constexpr int OFF_HEAD = OFF_BAR + 256;  // [warp][R][HD] the piece that a stretch begins in the middle of,
  static constexpr bool HEAD_SMEM = OFF_HEAD + WARPS * R * HD * 4 + 1024 <= 226 * 1024 + 256;  // if that fits (else in scratch)
  static constexpr int SMEM = OFF_HEAD + (HEAD_SMEM ? WARPS * R * HD * 4 : 0) + 1024;
  static_assert(R * HD * 4 <= STAGES * 2 * TILE, "a piece fits its warp's ring");
  static_assert(WARPS * STAGES * 8 <= 256 && SMEM <= 227 * 1024 - 700, "shared memory");
};

struct PgParams {
  PageMap map;           // in 4 bits the strides are in bytes
  const void *q, *k_new, *v_new;
  void *out, *k, *v;
  const int *lengths, *query_positions;
  int* positions;
  void* scales;          // in 4 bits: (pages, heads, page, 2) of keys and values
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
// An infinite or missing number as the nearest finite one or the lowest: on top of a sum that is not finite either it changes nothing.
__device__ __forceinline__ float finite(float x) { return fminf(fmaxf(x, -FLT_MAX), FLT_MAX); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const typename Num<T>::T2 v = Num<T>::from_f2(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Byte offset of 16-byte chunk `c` of row `row` of a tile, swizzled as TMA does it (128 bytes wide, at head_dim 32 64): the chunk
// number is xor-ed with the row, so that the eight rows of an ldmatrix lie in different banks.
template <int HD, bool Q4> __device__ __forceinline__ uint32_t tile_at(int row, int c) {
  if (Q4) return (uint32_t)(row * (HD / 2) + ((c ^ (HD == 32 ? 0 : HD == 64 ? row >> 2 & 1 : row >> 1 & 3)) << 4));
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
template <int KEYS, int ROW_COST>
struct Cursor {
  int b, hr, j, tiles, at;
  SeqKeys keys;
  __device__ __forceinline__ void load(const PgParams& p) {
    keys = keys_of(p, p.lengths[b]);
    tiles = (keys.n + KEYS - 1) / KEYS;
  }
  // to the first tile of the next row of scores; false if there is none
  __device__ __forceinline__ bool next_row(const PgParams& p) {
    at += ROW_COST;
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
// The line has ROW_COST units and one for each tile of a row, and is cut into equal stretches, one for each warp (with fewer
// units than warps, of one unit): the first `more` have a unit more than `each`.
template <int WARPS> struct Line {
  int64_t units, each, more, parts;
  __device__ __forceinline__ Line(int64_t units_, int ctas) : units(units_), parts(min(units_, (int64_t)ctas * WARPS)) {
    each = parts ? divide(units, parts) : 0;
    more = units - each * parts;
  }
  __device__ __forceinline__ int64_t begin(int64_t part) const { return part < parts ? part * each + min(part, more) : units; }
  // the block whose warps have unit t
  __device__ __forceinline__ int block_of(int64_t t) const {
    const int64_t wide = more * (each + 1);
    return (int)((t < wide ? divide(t, each + 1) : more + divide(t - wide, each)) / WARPS);
  }
};
template <int ROW_COST> __device__ __forceinline__ int row_units(int tiles) { return tiles ? tiles + ROW_COST : 0; }

__device__ __forceinline__ float alibi_rounded_log2(int mode, float slope, float dist) {  // slope already rounded
  const int drop = mode == 2 ? 13 : 16;
  return -round_significand(round_significand(dist, drop) * slope, drop) * kLog2e;
}

// What a block knows of its warps' pieces when it joins them.
template <int WARPS> struct Pieces {
  int64_t begin[WARPS][2];  // the piece's row's first tile in the line
  int b[WARPS][2], hr[WARPS][2], tiles[WARPS][2];
  uint8_t flags[WARPS];  // bit 0: there is a piece [0], which began before the warp's stretch; 1: a piece [1], which goes on
};                          // behind it; 2: piece [0] is its row's last

}  // namespace

// BIAS: 0 none, 1 exact slopes, 2 slopes rounded as a table's
template <typename T, int HD, int G, int BIAS, bool TMA, bool Q4>
__global__ void __launch_bounds__(PgCfg<HD, G, BIAS, Q4>::WARPS * 32, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PgParams p) {
  using C = PgCfg<HD, G, BIAS, Q4>;
  constexpr int WARPS = C::WARPS, NT = C::NT, R = C::R, STAGES = C::STAGES, STAGE = 2 * C::TILE, KS = HD / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int64_t sh_scan[WARPS], sh_base[WARPS];
  __shared__ int sh_b[WARPS];
  __shared__ Pieces<WARPS> sh;
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
  const int64_t part = (int64_t)blockIdx.x * WARPS + warp;
  Line<WARPS> line(0, 0);
  int start_b = 0;
  int64_t start_base = 0;  // the units before it
  if (p.B <= 32) {         // each warp by itself: no barrier, one load (one user 10.0 us, with the scan below 10.9)
    const int len = lane < p.B ? p.lengths[lane] : 0;
    const int tiles = lane < p.B ? (keys_of(p, len).n + C::KEYS - 1) / C::KEYS : 0;
    const uint32_t mine = row_units<C::ROW_COST>(tiles);
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    line = Line<WARPS>((int64_t)__shfl_sync(0xffffffffu, upto, 31) * heads, p.ctas);
    const unsigned behind = __ballot_sync(0xffffffffu, (int64_t)upto * heads > line.begin(part));
    start_b = behind ? __ffs(behind) - 1 : 0;
    start_base = (int64_t)__shfl_sync(0xffffffffu, upto - mine, start_b) * heads;
    if (warp == 0 && lane < p.B) look_over(lane, len, tiles);
  } else {
    const int per = (p.B + WARPS * 32 - 1) / (WARPS * 32);
    const int b_lo = min((int)threadIdx.x * per, p.B), b_hi = min(b_lo + per, p.B);
    int64_t mine = 0;
    for (int b = b_lo; b < b_hi; ++b) mine += row_units<C::ROW_COST>((keys_of(p, p.lengths[b]).n + C::KEYS - 1) / C::KEYS);
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
    for (int w = 0; w < WARPS; ++w) {
      const int64_t v = sh_scan[w];
      if (w < warp) base += v;
      total += v;
    }
    line = Line<WARPS>(total * heads, p.ctas);
    for (int b = b_lo; b < b_hi; ++b) {
      const int len = p.lengths[b];
      const int tiles = (keys_of(p, len).n + C::KEYS - 1) / C::KEYS;
      look_over(b, len, tiles);
#pragma unroll 1
      for (int w = 0; w < WARPS; ++w) {
        const int64_t f = line.begin((int64_t)blockIdx.x * WARPS + w);
        if (f >= base * heads && f < (base + row_units<C::ROW_COST>(tiles)) * heads) {
          sh_b[w] = b;
          sh_base[w] = base * heads;
        }
      }
      base += row_units<C::ROW_COST>(tiles);
    }
    __syncthreads();
    start_b = sh_b[warp];
    start_base = sh_base[warp];
  }
  if (line.begin((int64_t)blockIdx.x * WARPS) >= line.units) return;  // nothing for this block
  const int64_t from = line.begin(part);
  const int length = (int)(line.begin(part + 1) - from);

  uint8_t* ring = smem + warp * STAGES * STAGE;
  const uint32_t ring_at = smem_u32(ring);
  uint8_t* places = smem + C::OFF_POS + warp * STAGES * C::KEYS * 4;
  float2* my_ml = reinterpret_cast<float2*>(smem + C::OFF_ML) + warp * 2 * R;
  auto head_piece = [&](int w) {
    return C::HEAD_SMEM ? reinterpret_cast<float*>(smem + C::OFF_HEAD) + w * (R * HD)
                        : p.heads_acc + ((int64_t)blockIdx.x * WARPS + w) * (R * HD);
  };
  const int g8 = lane >> 2, j2 = 2 * (lane & 3);  // row of an 8x8 block, first of its two columns
  // The second product takes the probabilities in two parts of 16 bits: rounded, and what that leaves (64 sequences of 8 query heads a
  // key head: 1.2e-3 off in bf16, its own rounding; 1.6e-3 with the first part alone).  Up to four query heads the instruction's other
  // four columns repeat them and carry the rest; more heads take a second product (that case: 214 us, 219 without it, from a kernel
  // that chose between the two while it ran).
  constexpr bool FINE = G == 4, APART = G == 8 && !Q4;  // APART: in sums of its own, for more than 8 heads there are no registers
  const bool rest = FINE && j2 >= 4;
  // The second product's values: codes are exact in either type, probabilities times scales need bf16's range.
  using V = typename std::conditional<Q4, __nv_bfloat16, T>::type;
  auto dim_at = [&](int m, int half) {  // of row `half` * 8 + g8 of the m-th block of 16 of O^T
    if (!Q4) return m * 16 + half * 8 + g8;
    const int c = HD == 32 ? 0 : m / 4 * 2 + half, n = HD == 32 ? m + 2 * half : m % 4;
    return c * 32 + 8 * (g8 >> 1) + 2 * n + (g8 & 1);
  };

  Cursor<C::KEYS, C::ROW_COST> cu;
  cu.at = length;
  if (length > 0) {
    cu.b = start_b;
    cu.load(p);
    const int64_t in = from - start_base;  // units of the sequence before the stretch
    const int units = row_units<C::ROW_COST>(cu.tiles);
    cu.hr = in < (1LL << 31) ? (int)((uint32_t)in / (uint32_t)units) : (int)(in / units);
    cu.j = (int)(in - (int64_t)cu.hr * units) - C::ROW_COST;
    cu.at = max(-cu.j, 0);
    cu.j = max(cu.j, 0);
  }
  if (cu.at < length) {
    Cursor<C::KEYS, C::ROW_COST> ld = cu;

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
              const uint32_t o = stage * STAGE + tile_at<HD, Q4>((lane << p.box_log2) + kk, c);
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
        using E = typename std::conditional<Q4, uint8_t, T>::type;
        constexpr int PER = 16 / sizeof(E);  // of a chunk
        int64_t off[C::OWN];
#pragma unroll
        for (int u = 0; u < C::OWN; ++u) {
          const int kk = lane + 32 * u;
          const bool wanted = kk < C::KEYS && slot0 + kk < cached;
          const bool ok = wanted && (unsigned)page[u] < (unsigned)p.map.num_pages;
          if (wanted && !ok) atomicCAS(&g_dev_status, 0, kBadPage);
          off[u] = ok ? row_offset(p.map, page[u], head, row[u]) : -1;
          if (Q4 && kk < C::KEYS)  // what is no key has a scale of zero
            cp4(smem_u32(places) + (stage * C::KEYS + kk) * 4,
                static_cast<const uint32_t*>(p.scales) + (ok ? stat_offset(p.map, page[u], p.kv_heads, head, row[u]) : 0), ok ? 4 : 0);
          if (!Q4 && BIAS && p.positions && kk < C::KEYS)
            cp4(smem_u32(places) + (stage * C::KEYS + kk) * 4,
                ok ? p.positions + stat_offset(p.map, page[u], p.kv_heads, head, row[u]) : p.positions, ok ? 4 : 0);
        }
        const E* k = static_cast<const E*>(p.k) + (lane % C::CHUNKS) * PER;
        const E* v = static_cast<const E*>(p.v) + (lane % C::CHUNKS) * PER;
#pragma unroll
        for (int i = 0; i < C::ITERS; ++i) {
          const int kk = i * C::RPI + lane / C::CHUNKS;
          const int64_t o = __shfl_sync(0xffffffffu, off[(i * C::RPI) / 32], kk & 31);
          const uint32_t dst = at + tile_at<HD, Q4>(kk, lane % C::CHUNKS);
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
    auto fetch = [&](const Cursor<C::KEYS, C::ROW_COST>& c, Row& w) {
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
              // in 4 bits the dims of a lane's words: 8 neighbours of every 32, two to a half of an instruction
              const T* at = qr + (Q4 ? ks / 2 * 32 + 3 * j2 + ks % 2 * 4 + half * 2 : ks * 16 + half * 8);
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
        if (lane < HD / 4) {
          const T* at = lane < HD / 8 ? static_cast<const T*>(p.k_new) + c.b * p.kn_b + kv * p.kn_h + lane * 8
                                      : static_cast<const T*>(p.v_new) + c.b * p.vn_b + kv * p.vn_h + (lane - HD / 8) * 8;
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
    Cursor<C::KEYS, C::ROW_COST> rows = cu;  // the row of `ahead`

    // where ldmatrix reads: chunk 0 of the lane's row; the chunk number's higher bits are xor-ed in
    const int mi = lane >> 3, l8 = lane & 7;
    const uint32_t k_at = tile_at<HD, Q4>((mi & 1) * 8 + l8, mi >> 1), v_at = tile_at<HD, Q4>((mi >> 1) * 8 + l8, mi & 1) + C::TILE;
    // in 4 bits: blocks of 8 keys by 32 dims, two of keys by two of dims, or at head_dim 32 four of keys; of keys and of values alike
    const uint32_t at4 = HD == 32 ? tile_at<HD, Q4>(lane, 0) : tile_at<HD, Q4>((mi & 1) * 8 + l8, mi >> 1);
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
          if (fetches == 2 || (cu.at + cu.tiles - cu.j + C::ROW_COST < length && rows.next_row(p))) fetch(rows, ahead);
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
      if (Q4 && ragged) {  // the new token's row is not in the pages yet: as it will be there
        const int kk = cu.keys.fresh - slot0;
        if (cu.keys.fresh >= 0 && kk < C::KEYS) {
          const int kv = cu.hr / p.row_tiles, c = lane % (HD / 8);
          T scale;
          float whole[8];
          const uint32_t word = quantize8<T, HD / 8>(now.fresh, scale, whole);
          const uint32_t mine = *reinterpret_cast<const uint16_t*>(&scale);
          const uint32_t pair = __shfl_sync(0xffffffffu, mine, 0) | __shfl_sync(0xffffffffu, mine, HD / 8) << 16;
          if (lane < HD / 4)
            *reinterpret_cast<uint32_t*>(ring + stage * STAGE + tile_at<HD, Q4>(kk, c / 4) + (lane < HD / 8 ? 0 : C::TILE) + c % 4 * 4) = word;
          if (lane == 0) reinterpret_cast<uint32_t*>(places)[stage * C::KEYS + kk] = pair;
          if (cu.hr == kv * p.row_tiles) {  // one of the row's head tiles writes it into its slot
            const int r0 = cu.keys.fresh % p.map.page;
            if ((unsigned)now.page < (unsigned)p.map.num_pages) {
              if (lane < HD / 4)
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(lane < HD / 8 ? p.k : p.v) + row_offset(p.map, now.page, kv, r0) + c * 4) = word;
              if (lane == 0) static_cast<uint32_t*>(p.scales)[stat_offset(p.map, now.page, p.kv_heads, kv, r0)] = pair;
            } else {
              atomicCAS(&g_dev_status, 0, kBadPage);
            }
          }
        }
        __syncwarp();
      }
      if (!Q4 && ragged) {  // rows behind the last cached key may hold anything; the new token's are not in the pages yet
        const int kv = cu.hr / p.row_tiles;
        uint8_t* at = ring + stage * STAGE;
        for (int i = lane; i < (C::KEYS - (cached - slot0)) * C::CHUNKS; i += 32) {
          const uint32_t dst = tile_at<HD, Q4>(cached - slot0 + i / C::CHUNKS, i % C::CHUNKS);
          *reinterpret_cast<uint4*>(at + dst) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(at + dst + C::TILE) = make_uint4(0, 0, 0, 0);
        }
        const int kk = cu.keys.fresh - slot0;  // at least 0, because there is a cached key in every tile before it
        if (cu.keys.fresh >= 0 && kk < C::KEYS) {
          __syncwarp();
          const int c = lane % C::CHUNKS;
          if (lane < 2 * C::CHUNKS) *reinterpret_cast<uint4*>(at + tile_at<HD, Q4>(kk, c) + (lane < C::CHUNKS ? 0 : C::TILE)) = now.fresh;
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
      const uint32_t* place = reinterpret_cast<const uint32_t*>(places) + stage * C::KEYS;
      if constexpr (Q4) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; c += 2)
#pragma unroll
          for (int m = 0; m < C::MT; m += HD == 32 ? 2 : 1) {
            uint32_t w[4], x[4][4];
            ldm4(w, tile + (at4 ^ (c << 4)) + m * (8 * HD));
#pragma unroll
            for (int i = 0; i < 4; ++i) expand_nibbles<T>(w[i], x[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i)  // chunk c + i, or block m + i
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t a[4] = {x[2 * i][2 * h], x[2 * i + 1][2 * h], x[2 * i][2 * h + 1], x[2 * i + 1][2 * h + 1]};
                const int ks = HD == 32 ? h : (c + i) * 2 + h, mm = HD == 32 ? m + i : m;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma<T>(s[mm][nt], a, now.q[nt][ks][0], now.q[nt][ks][1]);
              }
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int m = 0; m < C::MT; ++m) {
            uint32_t a[4];
            ldm4(a, tile + (k_at ^ ((ks % PER_PANEL) << 5)) + (ks / PER_PANEL) * PANEL + m * BLOCK16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<T>(s[m][nt], a, now.q[nt][ks][0], now.q[nt][ks][1]);
          }
      }
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = kNone;
      float v_scale[C::MT][2];
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int kk = m * 16 + half * 8 + g8;
          float dist = 0.f, scale = p.scale;
          if (Q4) {
            v_scale[m][half] = pair_value<T>(place[kk], 1);
            scale *= pair_value<T>(place[kk], 0);
          }
          if (BIAS) dist = (float)(now.here - (!Q4 && p.positions ? (int)place[kk] : slot0 + kk));
          if (BIAS && ragged && slot0 + kk == cu.keys.fresh) dist = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = s[m][nt][2 * half + e] * scale;
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
      if (!Q4 && p.scores) {
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
              if (Q4) w[e] *= v_scale[m][half];
            }
            const uint32_t u = pack2<V>(w[0], w[1]);
            uint32_t left = u;
            if (!FINE || rest) {
              const float2 f = Num<V>::to_f2(*reinterpret_cast<const typename Num<V>::T2*>(&u));
              left = pack2<V>(w[0] - f.x, w[1] - f.y);
            }
            pt[m][nt][half] = transpose8(FINE ? left : u);
            if (!FINE) rt[m][nt][half] = transpose8(left);
          }
      }
      if constexpr (Q4) {
        // Transposed blocks of 16-bit units: a unit of four dims of two neighbouring keys in a word, nibble by nibble a pair of keys.
#pragma unroll
        for (int c = 0; c < C::CHUNKS; c += 2)
#pragma unroll
          for (int m = 0; m < C::MT; m += HD == 32 ? 2 : 1) {
            uint32_t w[4], x[4][4];
            ldm4t(w, tile + C::TILE + (at4 ^ (c << 4)) + m * (8 * HD));
#pragma unroll
            for (int i = 0; i < 4; ++i) expand_nibbles<V>(w[i], x[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // nibble i of two chunks, or at head_dim 32 nibbles i and i + 2 of one, of block m + i / 2
              const int first = HD == 32 ? i / 2 * 2 : 0, n = HD == 32 ? i % 2 : i, hm = HD == 32 ? n : c * 2 + n;
              const int mm = HD == 32 ? m + i / 2 : m;
              const uint32_t a[4] = {x[first][n], HD == 32 ? x[first][n + 2] : x[2][n], x[first + 1][n], HD == 32 ? x[first + 1][n + 2] : x[3][n]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma<V>(o[hm][nt], a, pt[mm][nt][0], pt[mm][nt][1]);
                if (!FINE) mma<V>(o[hm][nt], a, rt[mm][nt][0], rt[mm][nt][1]);
              }
            }
          }
      } else {
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
      }
      if (!APART && !FINE && !Q4) {
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
                  out[dim_at(m, 0)] = Num<T>::from_f(o[m][nt][e] * inv);
                  out[dim_at(m, 1)] = Num<T>::from_f(o[m][nt][2 + e] * inv);
                }
                if (p.lse && g8 == 0) p.lse[(int64_t)row_b * p.kv_heads * p.group + head] = ref[nt][e] + __log2f(l);
              } else {
#pragma unroll
                for (int m = 0; m < KS; ++m) {
                  acc[r * HD + dim_at(m, 0)] = o[m][nt][e];
                  acc[r * HD + dim_at(m, 1)] = o[m][nt][2 + e];
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
  const int flags = lane < WARPS ? sh.flags[lane] : 0;
  // bit w: of warp w
  const unsigned has0 = __ballot_sync(0xffffffffu, flags & 1), has1 = __ballot_sync(0xffffffffu, flags & 2), ends = __ballot_sync(0xffffffffu, flags & 4);
  // A chain of pieces starts with a piece [1], or with the piece [0] that has none before it in this block: only the first can.
  const unsigned lead = has0 & (0u - has0);                             // the first warp with a piece [0]
  const bool leads = lead != 0 && (has1 & (lead - 1u)) == 0;            // and nothing goes on into it
  const int chains = __popc(has1) + leads, rows_most = min(R, p.group);
  int open0 = -1, open1 = -1;  // the first warps of the chains that begin, or end, in another block
  auto end_of = [&](int w, int slot) {  // a chain's last warp
    int end = w;
    bool ended = slot == 0 && (ends >> w & 1) != 0;
    while (!ended && end + 1 < WARPS && (has0 >> (end + 1) & 1) != 0) ended = (ends >> ++end & 1) != 0;
    return ended ? end : end | 64;  // 64: the row goes on in the next block
  };
  if (leads) open0 = __ffs(lead) - 1;
  if (has1 != 0) {  // only the last chain can go on
    const int w = 31 - __clz(has1);
    if (end_of(w, 1) & 64) open1 = w;
  }
  for (int job = warp; job < chains * rows_most; job += WARPS) {
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
    constexpr int N = 8, THREADS = WARPS * 32;
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

namespace {

// Workspace: counters, then the pieces of blocks and warps for the widest rows.  Scratch, for the masses: log-sum-exps, scores.
struct PgWorkspace {
  int64_t ml, acc, heads_acc, bytes;
};
inline PgWorkspace pg_workspace() {
  const int64_t n = sm_count(), warps = 12, R = 16, hd = 128;
  PgWorkspace s;
  s.ml = kCounterBytes;
  s.acc = s.ml + up256(2 * n * R * 8);
  s.heads_acc = s.acc + up256(2 * n * R * hd * 4);
  s.bytes = s.heads_acc + n * warps * R * hd * 4;
  return s;
}

}  // namespace
}  // namespace tfb
