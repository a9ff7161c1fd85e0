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
// by cp.async two tiles ahead and across the borders of sequences, no barrier of the block anywhere in the loop.  A stretch
// that holds a whole row of scores writes the output; otherwise the reference, sum and accumulator of the piece go to
// scratch, and a second kernel joins the pieces in their order (no atomics: the result does not depend on timing).
//
// Products.  S^T = K Q^T and O^T = V^T P^T by mma.sync m16n8k16, keys (or head_dim) along M and query heads along N: a tile
// of 8 heads wastes less than one of 16, and P^T comes out of the first product's registers by a transposition of 8x8
// blocks (movmatrix).  tcgen05 has no place here: its smallest M would be fed from shared memory that the CUDA cores have to
// write P into, and nothing waits for the tensor core.
#include "attn.cuh"
#include "paged.cuh"

namespace tfb {
namespace {

constexpr int PG_WARPS = 8;
constexpr int PG_STAGES = 3;
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are kept relative to a reference that the running maximum may pass by 2^15 before everything is rescaled
// (they then still fit fp16); a new reference is 2^4 below the maximum, so that small ones stay clear of fp16's subnormals.
constexpr float kAhead = 15.f, kBelow = 4.f;
constexpr float kNone = -INFINITY;

template <int HD> struct PgCfg {
  static constexpr int KEYS = 2048 / HD;       // keys of a tile
  static constexpr int MT = KEYS / 16;
  static constexpr int CHUNKS = HD / 8;        // 16-byte chunks of a row
  static constexpr int RPI = 32 / CHUNKS;      // rows that a warp copies with one instruction
  static constexpr int ITERS = KEYS / RPI;     // 8
  static constexpr int OWN = (KEYS + 31) / 32; // keys whose place a lane looks up
  static constexpr int TILE = KEYS * HD * 2;   // bytes of the keys of a tile (4096)
  static constexpr int STAGE = 2 * TILE + KEYS * 4;  // keys, values, positions
  static constexpr int SMEM = PG_WARPS * PG_STAGES * STAGE;
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
  int new_vec;    // the new rows can be copied 16 bytes at a time
  int warps;      // of the split kernel's grid
  float scale;    // log2(e) / sqrt(hd)
  int64_t* prefix;  // (B + 1) tiles of the sequences before b, per head tile
  float* lse;       // (B, kv_heads * group) log2 of the sum of exponentials, rows that one warp finished
  float2* ml;       // [2 * warps][R] reference and sum of a piece
  float* acc;       // [2 * warps][R][hd]
  float* scores;    // (B, kv_heads * group, capacity) in log2 units, or null
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {  // the rest of the 16 is zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const typename Num<T>::T2 v = Num<T>::from_f2(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Byte offset of 16-byte chunk `c` of row `row` of a tile: the chunk number is xor-ed with the row, so that the eight rows of
// an ldmatrix lie in different banks.
template <int HD> __device__ __forceinline__ uint32_t tile_at(int row, int c) {
  const int x = HD == 32 ? (row >> 1) & 3 : row & 7;
  return (uint32_t)(row * HD * 2 + ((c ^ x) << 4));
}

// Keys of a sequence, and the slot of its new one (-1: none).
struct SeqKeys {
  int n, fresh;
};
__device__ __forceinline__ SeqKeys keys_of(const PgParams& p, int b) {
  const int cap = (int)p.map.capacity(), len = p.lengths[b];
  SeqKeys s;
  s.fresh = p.k_new && len >= 0 && len < cap ? len : -1;
  s.n = min(max(len, 0) + (s.fresh >= 0), cap);
  return s;
}

// The place of a warp's stretch in the line of tiles: sequence, (key head, head tile), tile.
template <int HD>
struct Cursor {
  int b, hr, j, tiles;
  SeqKeys keys;
  __device__ __forceinline__ void load(const PgParams& p) {
    keys = keys_of(p, b);
    tiles = (keys.n + PgCfg<HD>::KEYS - 1) / PgCfg<HD>::KEYS;
  }
  // to the next tile, which there has to be
  __device__ __forceinline__ void step(const PgParams& p) {
    if (++j < tiles) return;
    j = 0;
    if (++hr < p.kv_heads * p.row_tiles) return;
    hr = 0;
    do {
      ++b;
      load(p);
    } while (tiles == 0 && b + 1 < p.B);
  }
};

__device__ __forceinline__ float alibi_log2(int mode, float slope, int dist) {
  const float d = (float)dist;
  if (mode == 1) return -slope * kLog2e * d;
  const int drop = mode == 2 ? 13 : 16;
  return -round_significand(round_significand(d, drop) * slope, drop) * kLog2e;
}

}  // namespace

template <typename T, int HD, int NT, bool BIAS>
__global__ void __launch_bounds__(PG_WARPS * 32, 1) paged_attn_kernel(const PgParams p) {
  using C = PgCfg<HD>;
  constexpr int R = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t sh_scan[PG_WARPS + 1];
  __shared__ int64_t sh_from[PG_WARPS], sh_to[PG_WARPS];
  __shared__ int64_t sh_base[PG_WARPS];
  __shared__ int sh_b[PG_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.kv_heads * p.row_tiles;

  grid_dependency_wait();
  allow_dependents();

  // ---- the block's stretches: a scan over the sequences' tiles
  const int per = (p.B + PG_WARPS * 32 - 1) / (PG_WARPS * 32);
  const int b_lo = min((int)threadIdx.x * per, p.B), b_hi = min(b_lo + per, p.B);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += (keys_of(p, b).n + C::KEYS - 1) / C::KEYS;
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
  // fewer tiles than warps: one tile each, the first warps of all blocks before their second ones
  const int64_t line = total * heads, parts = min(line, (int64_t)p.warps);
  auto part_of = [&](int w) {
    return line < p.warps ? (int64_t)w * gridDim.x + blockIdx.x : (int64_t)blockIdx.x * PG_WARPS + w;
  };
  if (threadIdx.x < PG_WARPS) {
    const int64_t x = part_of(threadIdx.x);
    sh_from[threadIdx.x] = x < parts ? x * line / parts : 0;
    sh_to[threadIdx.x] = x < parts ? (x + 1) * line / parts : 0;
  }
  __syncthreads();
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = p.lengths[b];
    const int tiles = (keys_of(p, b).n + C::KEYS - 1) / C::KEYS;
    if (blockIdx.x == 0) {
      p.prefix[b] = base;
      if (len < 0 || (int64_t)len + (p.k_new ? 1 : 0) > p.map.capacity()) atomicCAS(&g_dev_status, 0, kBadLength);
    }
#pragma unroll
    for (int w = 0; w < PG_WARPS; ++w)
      if (sh_from[w] >= base * heads && sh_from[w] < (base + tiles) * heads) {
        sh_b[w] = b;
        sh_base[w] = base;
      }
    base += tiles;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.prefix[p.B] = total;
  __syncthreads();
  const int64_t from = sh_from[warp];
  const int count = (int)(sh_to[warp] - from);
  if (count <= 0) return;  // no barrier of the block below

  uint8_t* ring = smem + warp * PG_STAGES * C::STAGE;
  const uint32_t ring_at = smem_addr(ring);

  Cursor<HD> ld;
  {
    ld.b = sh_b[warp];
    ld.load(p);
    const int64_t in = from - sh_base[warp] * heads;
    ld.hr = (int)(in / ld.tiles);
    ld.j = (int)(in % ld.tiles);
  }
  Cursor<HD> cu = ld;

  // Page and row of the keys that this lane looks up, one tile ahead of the copies.
  int page[C::OWN], row[C::OWN];
  auto look_up = [&]() {
#pragma unroll
    for (int u = 0; u < C::OWN; ++u) {
      const int kk = lane + 32 * u, slot = ld.j * C::KEYS + kk;
      page[u] = -1;
      row[u] = 0;
      if (kk < C::KEYS && slot < ld.keys.n && slot != ld.keys.fresh) {
        const int i = (int)((unsigned)slot / (unsigned)p.map.page);
        row[u] = slot - i * p.map.page;
        page[u] = p.map.tables[ld.b * p.map.table_ld + i];
      }
    }
  };
  auto copy = [&](int stage) {
    const uint32_t at = ring_at + stage * C::STAGE;
    const int head = ld.hr / p.row_tiles;
    int64_t off[C::OWN];
#pragma unroll
    for (int u = 0; u < C::OWN; ++u) {
      const int kk = lane + 32 * u, slot = ld.j * C::KEYS + kk;
      const bool wanted = kk < C::KEYS && slot < ld.keys.n && slot != ld.keys.fresh;
      const bool ok = wanted && page[u] >= 0 && page[u] < p.map.num_pages;
      if (wanted && !ok) atomicCAS(&g_dev_status, 0, kBadPage);
      off[u] = ok ? row_offset(p.map, page[u], head, row[u]) : slot == ld.keys.fresh ? -2 : -1;
      if (BIAS && p.positions && kk < C::KEYS)
        cp4(at + 2 * C::TILE + kk * 4, ok ? p.positions + stat_offset(p.map, page[u], p.kv_heads, head, row[u]) : p.positions,
            ok ? 4 : 0);
    }
    const T* k = static_cast<const T*>(p.k) + (lane % C::CHUNKS) * 8;
    const T* v = static_cast<const T*>(p.v) + (lane % C::CHUNKS) * 8;
#pragma unroll
    for (int i = 0; i < C::ITERS; ++i) {
      const int kk = i * C::RPI + lane / C::CHUNKS;
      const int64_t o = __shfl_sync(0xffffffffu, off[(i * C::RPI) / 32], kk & 31);
      const uint32_t dst = at + tile_at<HD>(kk, lane % C::CHUNKS);
      if (o != -2) {
        cp16(dst, k + (o < 0 ? 0 : o), o < 0 ? 0 : 16);
        cp16(dst + C::TILE, v + (o < 0 ? 0 : o), o < 0 ? 0 : 16);
      }
    }
    const int kk = ld.keys.fresh - ld.j * C::KEYS;
    if (ld.keys.fresh >= 0 && kk >= 0 && kk < C::KEYS && lane < C::CHUNKS) {  // the new token's row is not in the pages yet
      const T* kn = static_cast<const T*>(p.k_new) + ld.b * p.kn_b + head * p.kn_h + lane * 8;
      const T* vn = static_cast<const T*>(p.v_new) + ld.b * p.vn_b + head * p.vn_h + lane * 8;
      const uint32_t o = stage * C::STAGE + tile_at<HD>(kk, lane);
      if (p.new_vec) {
        cp16(ring_at + o, kn, 16);
        cp16(ring_at + o + C::TILE, vn, 16);
      } else {
        T* dk = reinterpret_cast<T*>(ring + o);
        T* dv = reinterpret_cast<T*>(ring + o + C::TILE);
        for (int e = 0; e < 8; ++e) {
          dk[e] = kn[e];
          dv[e] = vn[e];
        }
      }
    }
  };

  look_up();
  int issued = 0;
  auto issue = [&]() {  // the next tile, if there is one, and always a group
    if (issued < count) {
      copy(issued % PG_STAGES);
      if (++issued < count) {
        ld.step(p);
        look_up();
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < PG_STAGES - 1; ++i) issue();

  const int g8 = lane >> 2, j2 = 2 * (lane & 3);  // row of an 8x8 block, first of its two columns
  uint32_t qf[NT][HD / 16][2];
  float slope[NT][2];
  float ref[NT][2], sum[NT][2], o[HD / 16][NT][4];
  int here = 0, first = 0;  // the query's position; whether the piece began with its row's first tile
  bool begin = true;
  const int mi = lane >> 3, l8 = lane & 7;

  for (int t = 0; t < count; ++t) {
    if (begin) {
      begin = false;
      first = cu.j == 0;
      const int kv = cu.hr / p.row_tiles, r0 = (cu.hr % p.row_tiles) * R;
      const T* q = static_cast<const T*>(p.q) + cu.b * p.q_b;
      const bool pairs = ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)(p.q_b * 2) | (uintptr_t)(p.q_h * 2)) & 3) == 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + nt * 8 + g8;
        const T* qr = q + (int64_t)(kv * p.group + r) * p.q_h + j2;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t v = 0;
            if (r < p.group) {
              const T* at = qr + ks * 16 + half * 8;
              if (pairs) v = *reinterpret_cast<const uint32_t*>(at);
              else v = (uint32_t)*reinterpret_cast<const uint16_t*>(at) |
                       (uint32_t)*reinterpret_cast<const uint16_t*>(at + 1) << 16;
            }
            qf[nt][ks][half] = v;
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rr = r0 + nt * 8 + j2 + e;
          slope[nt][e] = BIAS && rr < p.group ? p.slopes[kv * p.group + rr] : 0.f;
          if (BIAS && p.bias_mode == 2) slope[nt][e] = __half2float(__float2half_rn(slope[nt][e]));
          if (BIAS && p.bias_mode == 4) slope[nt][e] = __bfloat162float(__float2bfloat16_rn(slope[nt][e]));
          ref[nt][e] = kNone;
          sum[nt][e] = 0.f;
        }
      }
      if (BIAS) here = p.query_positions ? p.query_positions[cu.b] : cu.keys.n - 1;
#pragma unroll
      for (int m = 0; m < HD / 16; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[m][nt][e] = 0.f;
    }
    cp_wait<PG_STAGES - 2>();
    __syncwarp();
    issue();  // into the stage that the tile before this one has left
    const uint32_t kt = ring_at + (t % PG_STAGES) * C::STAGE, vt = kt + C::TILE;

    // ---- scores: keys g8 and g8 + 8 of each block of 16, heads j2 and j2 + 1
    float s[C::MT][NT][4];
#pragma unroll
    for (int m = 0; m < C::MT; ++m) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][nt][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t a[4];
        ldm4(a, kt + tile_at<HD>(m * 16 + (mi & 1) * 8 + l8, ks * 2 + (mi >> 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma<T>(s[m][nt], a, qf[nt][ks][0], qf[nt][ks][1]);
      }
    }
    const int slot0 = cu.j * C::KEYS;
    const bool ragged = slot0 + C::KEYS > cu.keys.n;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = kNone;
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int kk = m * 16 + half * 8 + g8, slot = slot0 + kk;
        int dist = 0;
        if (BIAS) {
          const int at = p.positions ? reinterpret_cast<const int*>(ring + (t % PG_STAGES) * C::STAGE + 2 * C::TILE)[kk] : slot;
          dist = slot == cu.keys.fresh ? 0 : here - at;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = s[m][nt][2 * half + e] * p.scale;
            if (BIAS) x += alibi_log2(p.bias_mode, slope[nt][e], dist);
            if (ragged && slot >= cu.keys.n) x = kNone;
            s[m][nt][2 * half + e] = x;
            top[nt][e] = fmaxf(top[nt][e], x);
          }
      }
    if (p.scores) {
      const int kv = cu.hr / p.row_tiles, r0 = (cu.hr % p.row_tiles) * R;
      const int64_t cap = p.map.capacity();
      float* sc = p.scores + ((int64_t)(cu.b * p.kv_heads + kv) * p.group + r0) * cap + slot0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + j2 + e;
          if (r0 + r < p.group)
#pragma unroll
            for (int m = 0; m < C::MT; ++m)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int kk = m * 16 + half * 8 + g8;
                if (slot0 + kk < cu.keys.n) sc[r * cap + kk] = s[m][nt][2 * half + e];
              }
        }
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
            for (int m = 0; m < HD / 16; ++m) {
              o[m][nt][e] *= f;
              o[m][nt][2 + e] *= f;
            }
          }
        }
    }
    // ---- probabilities, rounded to the values' type for the second product; the sum takes them unrounded
    uint32_t pt[C::MT][NT][2];
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[e] = ex2(s[m][nt][2 * half + e] - (ref[nt][e] == kNone ? 0.f : ref[nt][e]));
            sum[nt][e] += w[e];
          }
          pt[m][nt][half] = transpose8(pack2<T>(w[0], w[1]));
        }
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int hm = 0; hm < HD / 16; ++hm) {
        uint32_t a[4];
        ldm4t(a, vt + tile_at<HD>(m * 16 + (mi >> 1) * 8 + l8, hm * 2 + (mi & 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma<T>(o[hm][nt], a, pt[m][nt][0], pt[m][nt][1]);
      }

    // ---- the end of a row of scores, or of the stretch
    const bool last = cu.j + 1 == cu.tiles;
    if (last || t + 1 == count) {
      begin = true;
      const int kv = cu.hr / p.row_tiles, r0 = (cu.hr % p.row_tiles) * R;
      const int64_t piece = 2 * part_of(warp) + first;
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
            if (first && last) {
              const float inv = l > 0.f ? 1.f / l : l;  // a row whose weights are all zero is zero; NaN stays
              T* out = static_cast<T*>(p.out) + cu.b * p.o_b + head * p.o_h;
#pragma unroll
              for (int m = 0; m < HD / 16; ++m) {
                out[m * 16 + g8] = Num<T>::from_f(o[m][nt][e] * inv);
                out[m * 16 + 8 + g8] = Num<T>::from_f(o[m][nt][2 + e] * inv);
              }
              if (g8 == 0) p.lse[(int64_t)cu.b * p.kv_heads * p.group + head] = ref[nt][e] + __log2f(l);
            } else {
              float* acc = p.acc + (piece * R + r) * HD;
#pragma unroll
              for (int m = 0; m < HD / 16; ++m) {
                acc[m * 16 + g8] = o[m][nt][e];
                acc[m * 16 + 8 + g8] = o[m][nt][2 + e];
              }
              if (g8 == 0) p.ml[piece * R + r] = make_float2(ref[nt][e], l);
            }
          }
        }
    }
    if (t + 1 < count) cu.step(p);
  }
  cp_wait<0>();
}

// Joins the pieces of rows that several warps shared, adds the weights to the masses, and writes the new token's row into its
// slot.  One block per (sequence, key head) and share of its keys (blockIdx.y; the first one joins and writes).
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_finish_kernel(const PgParams p, const int R) {
  constexpr int KEYS = PgCfg<HD>::KEYS;
  constexpr int LANES = HD, SHARES = 256 / LANES;
  __shared__ float sh_lse[128], sh_ref[128], sh_inv[128];
  __shared__ float sh_acc[SHARES][HD];
  grid_dependency_wait();
  allow_dependents();
  const int b = blockIdx.x / p.kv_heads, kv = blockIdx.x % p.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SeqKeys keys = keys_of(p, b);
  const int heads = p.kv_heads * p.row_tiles;
  const int64_t line = p.prefix[p.B] * heads, parts = min(line, (int64_t)p.warps), at = p.prefix[b] * heads;
  const int tiles = (keys.n + KEYS - 1) / KEYS;
  const bool join = blockIdx.y == 0;
  T* out = static_cast<T*>(p.out) + b * p.o_b + (int64_t)kv * p.group * p.o_h;

  if (join && keys.fresh >= 0) {
    int page, row;
    if (find_slot(p.map, b, keys.fresh, page, row)) {
      const int64_t o = row_offset(p.map, page, kv, row);
      if (threadIdx.x < HD) {
        static_cast<T*>(p.k)[o + threadIdx.x] = static_cast<const T*>(p.k_new)[b * p.kn_b + kv * p.kn_h + threadIdx.x];
      } else if (threadIdx.x < 2 * HD) {
        const int e = threadIdx.x - HD;
        static_cast<T*>(p.v)[o + e] = static_cast<const T*>(p.v_new)[b * p.vn_b + kv * p.vn_h + e];
      }
      if (p.positions && threadIdx.x == 0)
        p.positions[stat_offset(p.map, page, p.kv_heads, kv, row)] = p.query_positions ? p.query_positions[b] : keys.fresh;
    }
  }
  if (tiles == 0) {  // no keys: zeros
    if (join)
      for (int i = threadIdx.x; i < p.group * HD; i += 256) out[(i / HD) * p.o_h + i % HD] = Num<T>::from_f(0.f);
    return;
  }
  // the stretch that tile t of the line is part of
  auto owner = [&](int64_t t) { return ((t + 1) * parts - 1) / line; };

  // ---- reference and sum of every query head
  for (int r = warp; r < p.group; r += 8) {
    const int64_t t0 = at + ((int64_t)kv * p.row_tiles + r / R) * tiles;
    const int64_t w0 = owner(t0), w1 = owner(t0 + tiles - 1);
    float lse = 0.f, ref = 0.f, inv = -1.f;  // inv < 0: the split kernel has written the row
    if (w0 == w1) {
      if (p.mass_out) lse = p.lse[((int64_t)b * p.kv_heads + kv) * p.group + r];
    } else {
      float m = kNone, l = 0.f;
      for (int64_t w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, p.ml[(2 * w + (w == w0)) * R + r % R].x);
      m = warp_max(m);
      for (int64_t w = w0 + lane; w <= w1; w += 32) {
        const float2 v = p.ml[(2 * w + (w == w0)) * R + r % R];
        l += v.y * (v.x == kNone ? (v.y == v.y ? 0.f : 1.f) : ex2(v.x - m));
      }
      l = warp_sum(l);
      ref = m;
      inv = l > 0.f ? 1.f / l : l == l ? 0.f : l;
      lse = m + __log2f(l);
    }
    if (lane == 0) {
      sh_lse[r] = lse == kNone ? INFINITY : lse;  // no weight anywhere: none for the masses either
      sh_ref[r] = ref;
      sh_inv[r] = inv;
    }
  }
  __syncthreads();
  if (join) {
    const int d = threadIdx.x % LANES, share = threadIdx.x / LANES;
    for (int r = 0; r < p.group; ++r) {
      if (sh_inv[r] < 0.f) continue;
      const int64_t t0 = at + ((int64_t)kv * p.row_tiles + r / R) * tiles;
      const int64_t w0 = owner(t0), w1 = owner(t0 + tiles - 1);
      float a = 0.f;
#pragma unroll 4
      for (int64_t w = w0 + share; w <= w1; w += SHARES) {
        const int64_t piece = (2 * w + (w == w0)) * R + r % R;
        const float2 v = p.ml[piece];
        a += v.x == kNone ? 0.f : p.acc[piece * HD + d] * ex2(v.x - sh_ref[r]);
      }
      sh_acc[share][d] = a;
      __syncthreads();
      if (share == 0) {
#pragma unroll
        for (int i = 1; i < SHARES; ++i) a += sh_acc[i][d];
        out[r * p.o_h + d] = Num<T>::from_f(a * sh_inv[r]);
      }
      __syncthreads();
    }
  }
  // ---- masses
  if (!p.mass_out) return;
  const int64_t cap = p.map.capacity();
  const float* sc = p.scores + ((int64_t)b * p.kv_heads + kv) * p.group * cap;
  for (int slot = blockIdx.y * 256 + threadIdx.x; slot < keys.n; slot += gridDim.y * 256) {
    int page, row;
    if (!find_slot(p.map, b, slot, page, row)) continue;
    const int64_t o = stat_offset(p.map, page, p.kv_heads, kv, row);
    float w = 0.f;
    for (int r = 0; r < p.group; ++r) w += ex2(sc[r * cap + slot] - sh_lse[r]);
    p.mass_out[o] = slot == keys.fresh ? w : p.mass[o] + w;
  }
}

namespace {

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// Scratch: prefix, lse, pieces, scores.
struct PgScratch {
  int64_t lse, ml, acc, scores, bytes;
};
int head_tiles(int64_t group) { return group <= 8 ? 1 : 2; }  // tiles of 8 heads that a warp takes at once
PgScratch pg_scratch(int64_t B, int64_t kv_heads, int64_t group, int64_t hd, int64_t cap, bool mass) {
  const int64_t pieces = 2 * (int64_t)sm_count() * PG_WARPS, R = 8 * head_tiles(group);
  PgScratch s;
  s.lse = up256((B + 1) * 8);
  s.ml = s.lse + up256(B * kv_heads * group * 4);
  s.acc = s.ml + up256(pieces * R * 8);
  s.scores = s.acc + up256(pieces * R * hd * 4);
  s.bytes = s.scores + (mass ? up256(B * kv_heads * group * cap * 4) : 0);
  return s;
}

template <typename T, int HD, int NT, bool BIAS>
int pg_launch(const PgParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(paged_attn_kernel<T, HD, NT, BIAS>, PgCfg<HD>::SMEM, done, "paged_attention")) return rc;
  launch_overlapped(paged_attn_kernel<T, HD, NT, BIAS>, dim3(p.warps / PG_WARPS), dim3(PG_WARPS * 32), PgCfg<HD>::SMEM, st, p);
  if (int rc = launched("paged_attention")) return rc;
  // enough blocks to fill the SMs, none with fewer than 1024 keys of a full table
  int64_t shares = 1;
  if (p.mass_out) {
    const int64_t rows = (int64_t)p.B * p.kv_heads, most = ceil_div(p.map.capacity(), 1024);
    shares = ceil_div((int64_t)sm_count() * 8, rows);
    if (shares > most) shares = most;
  }
  launch_overlapped(paged_finish_kernel<T, HD>, dim3((unsigned)(p.B * p.kv_heads), (unsigned)shares), dim3(256), 0, st, p, 8 * NT);
  return launched("paged_attention: join");
}

template <typename T, int HD>
int pg_dispatch(const PgParams& p, cudaStream_t st) {
  if (p.bias_mode) return head_tiles(p.group) == 1 ? pg_launch<T, HD, 1, true>(p, st) : pg_launch<T, HD, 2, true>(p, st);
  return head_tiles(p.group) == 1 ? pg_launch<T, HD, 1, false>(p, st) : pg_launch<T, HD, 2, false>(p, st);
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int64_t tfb_paged_attention_scratch_bytes(int64_t B, int64_t kv_heads, int64_t group, int64_t hd, int64_t capacity,
                                                     int with_mass) {
  if (B < 0 || kv_heads < 0 || group < 0 || hd < 0 || capacity < 0) return 0;
  return pg_scratch(B, kv_heads, group, hd, capacity, with_mass != 0).bytes;
}

extern "C" int tfb_paged_attention(const void* q, const void* k_new, const void* v_new, void* out, void* k_pages, void* v_pages,
                                   const int* tables, const int* lengths, const int* query_positions, int* positions,
                                   const float* mass, float* mass_out, const float* slopes, int alibi_round, int64_t B,
                                   int64_t kv_heads, int64_t group, int64_t hd, int64_t num_pages, int64_t page, int64_t width,
                                   int64_t table_ld, const int64_t* page_strides, const int64_t* q_strides,
                                   const int64_t* k_new_strides, const int64_t* v_new_strides, const int64_t* o_strides,
                                   void* scratch, int64_t scratch_bytes, int dtype, void* stream) {
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
  const PgScratch s = pg_scratch(B, kv_heads, group, hd, p.map.capacity(), mass != nullptr);
  TFB_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= s.bytes, "paged_attention: scratch of %lld bytes, %lld wanted",
              (long long)scratch_bytes, (long long)s.bytes);
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
  p.row_tiles = (int)ceil_div(group, 8 * head_tiles(group));
  p.warps = sm_count() * PG_WARPS;
  p.scale = kLog2e / sqrtf((float)hd);
  char* base = static_cast<char*>(scratch);
  p.prefix = reinterpret_cast<int64_t*>(base);
  p.lse = reinterpret_cast<float*>(base + s.lse);
  p.ml = reinterpret_cast<float2*>(base + s.ml);
  p.acc = reinterpret_cast<float*>(base + s.acc);
  p.scores = mass ? reinterpret_cast<float*>(base + s.scores) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  TFB_DISPATCH_16(dtype, T, {
    if (hd == 32) return pg_dispatch<T, 32>(p, st);
    if (hd == 64) return pg_dispatch<T, 64>(p, st);
    return pg_dispatch<T, 128>(p, st);
  })
}
