// Attention mass of a prompt's keys on tcgen05 / TMEM: the column sums of the causal softmax map,
//   m_j = sum over the query heads h of j's key head and the queries i >= j, i < count, of exp(s_hij - lse_hi),
// from the log-sum-exp that the attention forward has saved.
//
// With the log-sum-exp at hand one product and one exponential per score are all there is: no maximum, no second product.  The
// product is taken with the keys along the 128 lanes of tensor memory and the queries along its columns, so that a thread
// owns one key and its sum stays in a register from the key tile's first query tile to its last.
//
//   warp 0      TMA producer (K tile of 128 keys into one of two buffers, Q tiles of 256 queries through a ring)
//   warp 1      MMA issuer: M 128 (keys), N 256 (queries), into one of two score buffers of 256 columns
//   warps 4-19  exponentials and sums: four per lane quarter, each with 64 of the 256 queries of a tile.  A lane reads the
//               log-sum-exp of two of the queries, a tile ahead; the warp shares them through shared memory.
//
// Split.  The (key tile, head, query tile) triples of all prompts are numbered in one line, key tile by key tile, and each CTA
// takes an equal stretch of it: the causal triangle and prompts of different lengths leave no CTA with more than one tile
// over another.  Key tiles that several CTAs share leave their sums in a workspace; the last of the CTAs adds them, in order.
//
// Floor: the exponentials, one per score, 16 a clock and SM: 2048 clocks for a tile of 128 x 256, against 512 of the product at
// head_dim 64.  One pair in four goes to the FMA pipe (a polynomial of degree 5 for 2^f, |f| <= 1/2, relative error 2.1e-7 in 32
// bits, the SFU's own being 2.4e-7), which leaves the SFU 1536.  A tile takes about twice that: 42 to 58% of the SFU's and 62 to
// 67% of the issue slots are in use, so nothing is full, and what is waited for (the scores' way out of tensor memory, which a warp
// has nothing to do beside, is the likely cause) has not been measured.  A tile of 128 x 128, with a warp for the terms, took
// longer: the issuing warps' 1.2 k clocks a tile.  Measured: 4 prompts of 2048 tokens, 16 heads of 64, exact slopes 62 us (89 with
// 128 x 128); one of 8192, 12 query heads of 128 on 4 key heads 153 us (264).
#include "attn.cuh"
#include "paged.cuh"
#include "tc05.cuh"
#include <cfloat>
#include <type_traits>

namespace tfb {
namespace {

constexpr int PM_TILE = 128;             // keys of a tile
constexpr int PM_QUERIES = 2 * PM_TILE;  // queries of a tile
constexpr int PM_PARTS = 4;              // warps per lane quarter; each has PM_COLS columns of a tile
constexpr int PM_COLS = PM_QUERIES / PM_PARTS;
// A warp is at most two tiles ahead of another, which may still read the sums of the key tile that ended before those: each of
// the last PM_TURNS key tiles has a place and a barrier of its own.
constexpr int PM_TURNS = 4;

template <int HD> struct PmCfg {
  static constexpr int PANELS = HD / 64;
  static constexpr int K_BYTES = PANELS * 16384, Q_BYTES = 2 * K_BYTES;
  static constexpr int STAGES = HD == 64 ? 4 : 2;
  static constexpr int OFF_K = 0;
  static constexpr int OFF_Q = 2 * K_BYTES;
  static constexpr int OFF_C = OFF_Q + STAGES * Q_BYTES;         // [warp][2][PM_COLS] column terms
  static constexpr int OFF_SUM = OFF_C + 4 * PM_PARTS * 2 * PM_COLS * 4;  // [PM_TURNS][PM_PARTS][128] sums of a key tile
  static constexpr int OFF_BAR = OFF_SUM + PM_TURNS * PM_PARTS * 512;
  static constexpr int SMEM_BYTES = OFF_BAR + 512 + 1024;
  static constexpr int THREADS = 128 + 128 * PM_PARTS;
  static_assert(SMEM_BYTES <= 226 * 1024, "shared memory");
};

struct PmParams {
  const float* lse;
  const int* counts;  // may be null
  const float* slopes;
  float* out;
  int64_t lse_b, lse_h;
  int B, kv_heads, group, T;
  float scale;  // log2(e) / sqrt(hd)
  int ctas;
  int* arrived;     // [ctas] how many CTAs have left their pieces of the key tile that this one begins; zero between calls
  float* pieces;    // [ctas][2][128]
};

__device__ __forceinline__ int pm_count(const PmParams& p, int b) { return p.counts ? min(max(p.counts[b], 0), p.T) : p.T; }
// Query tiles of all m last key tiles of a head: m, m - 1, .. 1 tiles of 128 queries, in pairs.
__device__ __forceinline__ int64_t pm_pairs(int64_t m) { return (m + 1) * (m + 1) / 4; }
__device__ __forceinline__ int64_t pm_tiles(const PmParams& p, int count) {
  return pm_pairs((count + PM_TILE - 1) / PM_TILE) * p.kv_heads * p.group;
}

// A place in the line of tiles.  A run is what a key tile and a head have in common: the query tiles i, i + 2, .. below n.
struct PmCursor {
  int b, kv, j, r, i, n;  // prompt, key head, key tile, query head of the group, query tile (of 128), tiles of the prompt
  __device__ __forceinline__ int64_t start(int64_t j) const { return pm_pairs(n) - pm_pairs(n - j); }  // per head
  __device__ __forceinline__ int64_t key_tile() const { return (int64_t)(n - j + 1) / 2; }            // pairs in a run
  __device__ __forceinline__ void seek(const PmParams& p, int b_, int64_t in) {
    b = b_;
    n = (pm_count(p, b) + PM_TILE - 1) / PM_TILE;
    const int64_t per = pm_pairs(n) * p.group;
    kv = (int)(in / per);
    const int64_t rest = in % per, x = rest / p.group;  // key tile j begins at group * start(j)
    j = n - (int)sqrt(fmax(4.0 * (double)(pm_pairs(n) - x), 0.0));
    j = min(max(j, 0), n - 1);
    while (j > 0 && start(j) > x) --j;
    while (j + 1 < n && start(j + 1) <= x) ++j;
    const int64_t left = rest - start(j) * p.group;
    r = (int)(left / key_tile());
    i = j + 2 * (int)(left % key_tile());
  }
  __device__ __forceinline__ int run(int64_t left) const { return (int)min((int64_t)(n - i + 1) / 2, left); }  // tiles of the run
  __device__ __forceinline__ bool begins() const { return r == 0 && i == j; }
  __device__ __forceinline__ bool ends(const PmParams& p, int tiles) const { return i + 2 * tiles >= n && r + 1 == p.group; }
  // past `tiles` tiles of the run; what follows has to be there
  __device__ __forceinline__ void skip(const PmParams& p, int tiles) {
    i += 2 * tiles;
    if (i < n) return;
    i = j;
    if (++r < p.group) return;
    r = 0;
    i = ++j;
    if (j < n) return;
    i = j = 0;
    if (++kv < p.kv_heads) return;
    kv = 0;
    do {
      ++b;
      n = b < p.B ? (pm_count(p, b) + PM_TILE - 1) / PM_TILE : 1;
    } while (n == 0);
  }
};

__device__ __forceinline__ float at_least(float x, float low) {  // NaN stays
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(low));
  return y;
}
// 2^x of a pair on the FMA pipe: 2^f by a polynomial (minimax of the relative error), times 2^n by its exponent field.
__device__ __forceinline__ uint64_t pm_ex2_fma(uint64_t xp) {
  float x0, x1;
  f2_unpack(xp, x0, x1);
  const uint64_t x = f2_pack(at_least(x0, -127.f), at_least(x1, -127.f));  // 2^-127 is an exponent field of 0: zero
  const uint64_t xr = f2_add(x, f2_pack(12582912.f, 12582912.f));  // n in the low bits
  const uint64_t f = f2_fma(f2_add(xr, f2_pack(-12582912.f, -12582912.f)), f2_pack(-1.f, -1.f), x);
  auto both = [](float c) { return f2_pack(c, c); };
  uint64_t q = f2_fma(f, both(0.0013276472454890609f), both(0.009675540961325169f));
  q = f2_fma(q, f, both(0.05550713092088699f));
  q = f2_fma(q, f, both(0.24022120237350464f));
  q = f2_fma(q, f, both(0.6931469440460205f));
  q = f2_fma(q, f, both(1.0000001192092896f));
  float n0, n1;
  f2_unpack(xr, n0, n1);
  auto power = [](float n) { return __int_as_float((__float_as_int(n) << 23) + 0x3f800000); };
  return f2_mul(q, f2_pack(power(n0), power(n1)));
}

}  // namespace

template <typename T, int HD, int MODE>
__global__ void __launch_bounds__(PmCfg<HD>::THREADS, 1) prompt_mass_kernel(const __grid_constant__ CUtensorMap tmQ,
                                                                            const __grid_constant__ CUtensorMap tmK,
                                                                            const PmParams p) {
  using C = PmCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_full = bars;                  // [2]
  uint64_t* k_empty = k_full + 2;           // [2]
  uint64_t* q_full = k_empty + 2;           // [STAGES]
  uint64_t* q_empty = q_full + C::STAGES;   // [STAGES]
  uint64_t* s_full = q_empty + C::STAGES;   // [2] scores are in tensor memory
  uint64_t* s_empty = s_full + 2;           // [2] and have been read (every warp)
  uint64_t* sum_full = s_empty + 2;         // [PM_TURNS][4 lane quarters] a key tile's sums are in shared memory (PM_PARTS warps)
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sum_full + 4 * PM_TURNS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 * 2 + 2 * 4 + 2 * 2 + 4 * PM_TURNS) * 8 + 8 <= 512, "barriers");
  __shared__ int64_t sh_scan[C::THREADS / 32];
  __shared__ int64_t sh_base, sh_tile[2], sh_row[2];
  __shared__ int sh_b, sh_open[2], sh_key[2], sh_left[2], sh_tiles[2], sh_last[2], sh_first[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 4 * PM_PARTS);
    }
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 4 * PM_TURNS; ++i) mbar_init(&sum_full[i], PM_PARTS);
    mbar_fence_init();
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(tmem_holder, 512);
  }
  grid_dependency_wait();
  allow_dependents();
  if (threadIdx.x == 0) *abort_flag = (*(volatile int*)&g_dev_status != 0) ? 1 : 0;
  if (threadIdx.x < 2) sh_open[threadIdx.x] = 0;

  // ---- the CTA's stretch of the line
  const int per = (p.B + C::THREADS - 1) / C::THREADS;
  const int b_lo = min((int)threadIdx.x * per, p.B), b_hi = min(b_lo + per, p.B);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += pm_tiles(p, pm_count(p, b));
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sh_scan[warp] = upto;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int64_t base = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < C::THREADS / 32; ++w) {
    const int64_t v = sh_scan[w];
    if (w < warp) base += v;
    total += v;
  }
  const int64_t parts = min(total, (int64_t)p.ctas);
  const int64_t from = blockIdx.x < parts ? blockIdx.x * total / parts : 0;
  const int64_t count = blockIdx.x < parts ? (blockIdx.x + 1) * total / parts - from : 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int64_t tiles = pm_tiles(p, pm_count(p, b));
    if (from >= base && from < base + tiles) {
      sh_b = b;
      sh_base = base;
    }
    base += tiles;
  }
  __syncthreads();
  const uint32_t tmem_base = *tmem_holder;
  const bool live = *abort_flag == 0 && count > 0;
  PmCursor cu;
  if (live) cu.seek(p, sh_b, from - sh_base);
  if (*abort_flag == 0 && p.counts)  // keys past the prompts' ends
    for (int row = blockIdx.x; row < p.B * p.kv_heads; row += gridDim.x)
      for (int key = pm_count(p, row / p.kv_heads) + threadIdx.x; key < p.T; key += C::THREADS) p.out[(int64_t)row * p.T + key] = 0.f;

  if (!live) {
  } else if (warp == 0) {
    // --------------------------------------------------------------------- TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      int st = 0, nk = 0;
      uint32_t ph = 0;
      bool ok = true, fresh = true;  // fresh: the key tile has to be read
      for (int64_t left = count; left > 0 && ok;) {
        const int tiles = cu.run(left), head = cu.kv * p.group + cu.r;
        if (fresh || cu.begins()) {
          fresh = false;
          const int kb = nk & 1;
          if (!mbar_wait(&k_empty[kb], ((nk >> 1) & 1) ^ 1, 0x8000 | kb, abort_flag)) break;
          mbar_expect_tx(&k_full[kb], C::K_BYTES);
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c)
            tma_load_4d(smem + C::OFF_K + kb * C::K_BYTES + c * 16384, &tmK, c * 64, cu.j * PM_TILE, cu.kv, cu.b, &k_full[kb]);
          ++nk;
        }
        for (int k = 0; k < tiles; ++k) {
          ok = mbar_wait(&q_empty[st], ph ^ 1, 0x8100 | st, abort_flag);
          if (!ok) break;
          mbar_expect_tx(&q_full[st], C::Q_BYTES);
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c)
            tma_load_4d(smem + C::OFF_Q + st * C::Q_BYTES + c * 32768, &tmQ, c * 64, (cu.i + 2 * k) * PM_TILE, head, cu.b, &q_full[st]);
          if (++st == C::STAGES) { st = 0; ph ^= 1; }
        }
        left -= tiles;
        if (left > 0) cu.skip(p, tiles);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------------- MMA issuer
    constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t idesc = instr_desc_f16(PM_TILE, PM_QUERIES, fmt, 0, 0);
    const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0);
    const uint32_t s0 = smem_u32(smem);
    int st = 0, nk = -1, buf = 0;
    uint32_t ph = 0, sph = 1;
    bool ok = true, fresh = true;
    for (int64_t left = count; left > 0 && ok;) {
      const int tiles = cu.run(left);
      if (fresh || cu.begins()) {
        fresh = false;
        ++nk;
        if (!__all_sync(0xffffffffu, mbar_wait(&k_full[nk & 1], (nk >> 1) & 1, 0x8200 | (nk & 1), abort_flag))) break;
      }
      const bool last = cu.ends(p, tiles);
      const uint64_t dk = smem_desc_sw128(s0 + C::OFF_K + (nk & 1) * C::K_BYTES, 16, 1024);
      for (int k = 0; k < tiles; ++k) {
        ok = mbar_wait(&q_full[st], ph, 0x8300 | st, abort_flag) && mbar_wait(&s_empty[buf], sph, 0x8400 | buf, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dq = smem_desc_sw128(s0 + C::OFF_Q + st * C::Q_BYTES, 16, 1024);
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
          if (elect_one())
            tc_mma_ss(tb + buf * PM_QUERIES, desc_advance(dk, (s / 4) * 16384 + (s % 4) * 32),
                      desc_advance(dq, (s / 4) * 32768 + (s % 4) * 32), idesc, s ? 1u : 0u);
        if (elect_one()) {
          tc_commit(&s_full[buf]);
          tc_commit(&q_empty[st]);
          if (last && k + 1 == tiles) tc_commit(&k_empty[nk & 1]);
        }
        __syncwarp();
        if (++st == C::STAGES) { st = 0; ph ^= 1; }
        if (++buf == 2) { buf = 0; sph ^= 1; }
      }
      left -= tiles;
      if (left > 0) cu.skip(p, tiles);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- exponentials and sums
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    // A thread has rows (keys) g8, g8 + 8, g8 + 16 and g8 + 24 of its quarter and of every 8 columns two: it needs a quarter of
    // the columns' terms, whose way from shared memory would otherwise cost as much as the scores'.
    const int g8 = lane >> 2, j2 = 2 * (lane & 3);
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint64_t scale2 = f2_pack(p.scale, p.scale);
    float* terms = reinterpret_cast<float*>(smem + C::OFF_C) + (warp - 4) * 2 * PM_COLS;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    int turn = 0, buf = 0;
    uint32_t parity = 0;
    bool first = cu.begins(), ok = true;
    int64_t tile_at = from - (cu.r * cu.key_tile() + (cu.i - cu.j) / 2);  // where the key tile begins in the line
    // The log-sum-exps of the next tile are read while a tile is worked on, over the ends of runs too.
    struct Run {
      const float* lse;  // of this lane's first query of the run's first tile
      int left;          // queries from there on to the prompt's end
      float slope;
    };
    auto run_of = [&](const PmCursor& c) {
      const int h = c.kv * p.group + c.r, q = c.i * PM_TILE + part * PM_COLS + lane;
      return Run{p.lse + c.b * p.lse_b + h * p.lse_h + q, pm_count(p, c.b) - q, MODE == 0 ? 0.f : p.slopes[h]};
    };
    float lse[PM_COLS / 32];
    auto fetch = [&](const Run& run, int k) {
#pragma unroll
      for (int e = 0; e < PM_COLS / 32; ++e)
        lse[e] = k * PM_QUERIES + e * 32 < run.left ? run.lse[k * PM_QUERIES + e * 32] : -INFINITY;
    };
    Run run = run_of(cu);
    fetch(run, 0);
    for (int64_t left = count; left > 0 && ok;) {
      const int tiles = cu.run(left);
      const bool last = cu.ends(p, tiles);
      PmCursor next = cu;
      left -= tiles;
      Run after = run;
      if (left > 0) {
        next.skip(p, tiles);
        after = run_of(next);
      }
      const AlibiLog2<MODE> alibi(run.slope);
      int dist = (cu.i - cu.j) * PM_TILE + part * PM_COLS + j2 - quarter * 32 - g8;  // of the first query from the first key
      bool diagonal = cu.i == cu.j;
      for (int k = 0; k < tiles; ++k) {
        // The term of a query's column: -lse * log2(e).  It is -inf, and the column is left out, past the prompt's end and where the
        // row gives no weight; any other one is finite or NaN.  Two buffers in turn, over the ends of runs too: between a tile's reads
        // and the writes two tiles on lies the barrier of the tile between.
        float* mine = terms + buf * PM_COLS;
        bool out = false, in = false;
#pragma unroll
        for (int e = 0; e < PM_COLS / 32; ++e) {
          const bool none = lse[e] == -INFINITY;
          mine[e * 32 + lane] = none ? -INFINITY : at_least(lse[e] * -kLog2e, -FLT_MAX);
          out |= none;
          in |= !none;
        }
        const bool holes = __any_sync(0xffffffffu, out), any = __any_sync(0xffffffffu, in);
        __syncwarp();
        if (k + 1 < tiles) fetch(run, k + 1);
        else if (left > 0) fetch(after, 0);
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf], parity, 0x8500 | buf, abort_flag));
        if (!ok) break;
        tc_fence_after();
        uint64_t acc[4] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        // Distances are exact integers, and one rounding takes their product with the slope into the exponent: parts of it for rows
        // and columns would cancel near the diagonal, where the weights are.
        const float dist_f = (float)dist;
        const uint64_t dist2 = f2_pack(dist_f, dist_f + 1.f);
        // Of a tile whose queries begin before its keys end a warp may have nothing, and has to mask what is below the diagonal.  What is
        // masked or left out is so by selection: its score may be anything, and a NaN or infinite one would outlast a term of -inf.
        const bool none = !any || (diagonal && (part + 1) * PM_COLS <= quarter * 32);
        const bool masked = holes || (diagonal && part * PM_COLS < quarter * 32 + 32);
#pragma unroll
        for (int cc = 0; cc < PM_COLS / 32; ++cc) {  // 32 columns at a time
          uint32_t s[2][16];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tmem_ld_half32(tmem_base + lane_base + ((uint32_t)(16 * h) << 16) + buf * PM_QUERIES + part * PM_COLS + cc * 32, s[h]);
          tc_wait_ld();
          if (cc + 1 == PM_COLS / 32) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_empty[buf]);
          }
          uint64_t term[4];  // of the thread's columns 8 c + j2, 8 c + j2 + 1
#pragma unroll
          for (int c = 0; c < 4; ++c) term[c] = *reinterpret_cast<const uint64_t*>(mine + cc * 32 + c * 8 + j2);
          // the exponents of the columns of block c in row g8 + 8 a
          auto exponent = [&](int c, int a) {
            const uint32_t* v = &s[a / 2][c * 4 + (a % 2) * 2];
            uint64_t x = f2_fma(f2_pack(__uint_as_float(v[0]), __uint_as_float(v[1])), scale2, term[c]);
            if (MODE != 0) {
              const float k = (float)(cc * 32 + c * 8 - 8 * a);
              float d0, d1;
              f2_unpack(f2_add(dist2, f2_pack(k, k)), d0, d1);
              x = alibi.sub_pair(x, d0, d1);
            }
            return x;
          };
          if (!masked) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int a = 0; a < 4; ++a) {
                uint64_t x = exponent(c, a);
                constexpr unsigned kFma = 0x22;  // of eight pairs, those that take the FMA pipe
                if (kFma >> ((c * 4 + a) % 8) & 1) {
                  x = pm_ex2_fma(x);
                } else {
                  float x0, x1;
                  f2_unpack(x, x0, x1);
                  x = f2_pack(ex2(x0), ex2(x1));
                }
                acc[a] = f2_add(acc[a], x);
              }
          } else if (!none) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int a = 0; a < 4; ++a) {
                float x0, x1;
                f2_unpack(exponent(c, a), x0, x1);
                const int d = dist + cc * 32 + c * 8 - 8 * a;
                float t0, t1;
                f2_unpack(term[c], t0, t1);
                if (d < 0 || t0 == -INFINITY) x0 = -INFINITY;
                if (d + 1 < 0 || t1 == -INFINITY) x1 = -INFINITY;
                acc[a] = f2_add(acc[a], f2_pack(ex2(x0), ex2(x1)));
              }
          }
        }
        if (++buf == 2) {
          buf = 0;
          parity ^= 1;
        }
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          float w0, w1;
          f2_unpack(acc[a], w0, w1);
          sum[a] += w0 + w1;
        }
        diagonal = false;
        dist += PM_QUERIES;
      }
      if (ok && (last || left == 0)) {
        // the sums of a key's warps
        const int place = turn % PM_TURNS;
        uint64_t* bar = &sum_full[place * 4 + quarter];
        float* sums = reinterpret_cast<float*>(smem + C::OFF_SUM) + place * PM_PARTS * PM_TILE;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 1);
          sum[a] += __shfl_xor_sync(0xffffffffu, sum[a], 2);
          if (j2 == 0) sums[part * PM_TILE + quarter * 32 + g8 + 8 * a] = sum[a];
          sum[a] = 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        if (part == 0) {
          if (!__all_sync(0xffffffffu, mbar_wait(bar, turn / PM_TURNS & 1, 0x8600 | quarter, abort_flag))) break;
          const int row = quarter * 32 + lane;
          float whole = sums[row];
#pragma unroll
          for (int e = 1; e < PM_PARTS; ++e) whole += sums[e * PM_TILE + row];
          const int key = cu.j * PM_TILE + row, count_of = pm_count(p, cu.b);
          if (first && last) {
            if (key < count_of) p.out[((int64_t)cu.b * p.kv_heads + cu.kv) * p.T + key] = whole;
          } else {
            p.pieces[((int64_t)blockIdx.x * 2 + first) * PM_TILE + row] = whole;
            sh_open[first] = 1;
            sh_row[first] = (int64_t)cu.b * p.kv_heads + cu.kv;
            sh_key[first] = cu.j * PM_TILE;
            sh_left[first] = count_of - cu.j * PM_TILE;
            sh_tile[first] = tile_at;
            sh_tiles[first] = (int)cu.key_tile() * p.group;
          }
        }
        ++turn;
        first = true;  // whatever follows begins with a key tile's first tile
        tile_at += cu.key_tile() * p.group;
      }
      cu = next;
      run = after;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    for (int k = 0; k < 64; ++k) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  if (blockIdx.x == 0 && p.counts)  // at the end, because no CTA begins while the status is set
    for (int b = b_lo; b < b_hi; ++b)
      if (p.counts[b] < 0 || p.counts[b] > p.T) atomicCAS(dev_status(), 0, kBadLength);
  // ---- key tiles that several CTAs share: the last of them adds the pieces.  A CTA begins at most one such tile, whose counter
  // is the CTA's.
  if (*abort_flag || !(sh_open[0] || sh_open[1])) return;
  if (threadIdx.x < 2) {
    const int slot = threadIdx.x;
    sh_last[slot] = 0;
    if (sh_open[slot]) {
      const int64_t t0 = sh_tile[slot], t1 = t0 + sh_tiles[slot] - 1;
      const int c0 = (int)(((t0 + 1) * parts - 1) / total), c1 = (int)(((t1 + 1) * parts - 1) / total);
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
  const int slot = threadIdx.x / PM_TILE, row = threadIdx.x % PM_TILE;
  if (slot < 2 && sh_last[slot] && row < sh_left[slot]) {
    const int c0 = sh_first[slot];
    float sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < sh_last[slot]; ++i) sum += __ldcg(p.pieces + ((int64_t)(c0 + i) * 2 + (i == 0)) * PM_TILE + row);
    p.out[sh_row[slot] * p.T + sh_key[slot] + row] = sum;
  }
}

namespace {

template <typename T, int HD, int MODE>
int pm_launch(const CUtensorMap& tq, const CUtensorMap& tk, const PmParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(prompt_mass_kernel<T, HD, MODE>, PmCfg<HD>::SMEM_BYTES, done, "prompt_mass")) return rc;
  launch_overlapped(prompt_mass_kernel<T, HD, MODE>, dim3(p.ctas), dim3(PmCfg<HD>::THREADS), PmCfg<HD>::SMEM_BYTES, st, tq, tk, p);
  return launched("prompt_mass");
}
template <typename T, int HD>
int pm_dispatch(int mode, const CUtensorMap& tq, const CUtensorMap& tk, const PmParams& p, cudaStream_t st) {
  if (mode == 0) return pm_launch<T, HD, 0>(tq, tk, p, st);
  if (mode == 1) return pm_launch<T, HD, 1>(tq, tk, p, st);
  if (mode == 2) return pm_launch<T, HD, 2>(tq, tk, p, st);
  return pm_launch<T, HD, 4>(tq, tk, p, st);
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int64_t tfb_prompt_mass_workspace_bytes(void) { return kCounterBytes + (int64_t)sm_count() * 2 * PM_TILE * 4; }

extern "C" int tfb_prompt_mass(const void* q, const void* k, const float* lse, const int* counts, const float* slopes,
                               int alibi_round, float* out, int64_t B, int64_t kv_heads, int64_t group, int64_t T, int64_t hd,
                               const int64_t* q_strides, const int64_t* k_strides, const int64_t* lse_strides, void* workspace,
                               int64_t workspace_bytes, int dtype, void* stream) {
  TFB_REQUIRE(dtype == TFB_F16 || dtype == TFB_BF16, "prompt_mass: dtype %d: expected fp16 or bf16", dtype);
  if (hd != 32 && hd != 64 && hd != 128) return fail(TFB_ERR_UNSUPPORTED, "prompt_mass: Only head_dims of [32,64,128] are supported.");
  TFB_REQUIRE(B >= 0 && B < (1 << 20) && kv_heads >= 1 && group >= 1 && kv_heads * group <= 65535, "prompt_mass: bad batch or head count");
  TFB_REQUIRE(T >= 0 && T <= (1 << 23), "prompt_mass: more than 2^23 keys");
  TFB_REQUIRE(B * kv_heads < (1LL << 31), "prompt_mass: too many rows of heads");
  TFB_REQUIRE(alibi_round >= 0 && alibi_round <= 2, "prompt_mass: alibi_round %d", alibi_round);
  if (B == 0 || T == 0) return TFB_OK;
  TFB_REQUIRE(q && k && lse && out, "prompt_mass: a null operand");
  TFB_REQUIRE(aligned16(q) && aligned16(k), "prompt_mass: q and k start on 16-byte boundaries");
  for (int i = 0; i < 3; ++i)
    TFB_REQUIRE(q_strides[i] > 0 && q_strides[i] % 8 == 0 && k_strides[i] > 0 && k_strides[i] % 8 == 0,
                "prompt_mass: strides of q and k are positive multiples of 8 elements");
  TFB_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= tfb_prompt_mass_workspace_bytes(),
              "prompt_mass: workspace of %lld bytes, %lld wanted", (long long)workspace_bytes, (long long)tfb_prompt_mass_workspace_bytes());
  CUtensorMap tq, tk;
  const uint32_t box_q[4] = {64, PM_QUERIES, 1, 1}, box_k[4] = {64, PM_TILE, 1, 1};
  {
    const uint64_t dims[4] = {(uint64_t)hd, (uint64_t)T, (uint64_t)(kv_heads * group), (uint64_t)B};
    const uint64_t st[3] = {(uint64_t)q_strides[2] * 2, (uint64_t)q_strides[1] * 2, (uint64_t)q_strides[0] * 2};
    if (int rc = encode_tmap_sw128(&tq, q, dtype, 4, dims, st, box_q)) return rc;
  }
  {
    const uint64_t dims[4] = {(uint64_t)hd, (uint64_t)T, (uint64_t)kv_heads, (uint64_t)B};
    const uint64_t st[3] = {(uint64_t)k_strides[2] * 2, (uint64_t)k_strides[1] * 2, (uint64_t)k_strides[0] * 2};
    if (int rc = encode_tmap_sw128(&tk, k, dtype, 4, dims, st, box_k)) return rc;
  }
  PmParams p = {};
  p.lse = lse;
  p.counts = counts;
  p.slopes = slopes;
  p.out = out;
  p.lse_b = lse_strides[0];
  p.lse_h = lse_strides[1];
  p.B = (int)B;
  p.kv_heads = (int)kv_heads;
  p.group = (int)group;
  p.T = (int)T;
  p.scale = kLog2e / sqrtf((float)hd);
  const int64_t n = ceil_div(T, PM_TILE), tiles = (n + 1) * (n + 1) / 4 * kv_heads * group * B;
  p.ctas = (int)(tiles < sm_count() ? tiles : sm_count());
  p.arrived = static_cast<int*>(workspace);
  p.pieces = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  const int mode = !slopes ? 0 : alibi_round == 0 ? 1 : alibi_round == 1 ? 2 : 4;
  cudaStream_t st = (cudaStream_t)stream;
  TFB_DISPATCH_16(dtype, E, { return hd <= 64 ? pm_dispatch<E, 64>(mode, tq, tk, p, st) : pm_dispatch<E, 128>(mode, tq, tk, p, st); })
}
