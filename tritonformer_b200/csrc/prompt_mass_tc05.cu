// Attention mass of a prompt's keys on tcgen05 / TMEM: the column sums of the causal softmax map,
//   m_j = sum over the query heads h of j's key head and the queries i >= j, i < count, of exp(s_hij - lse_hi),
// from the log-sum-exp that the attention forward has saved.
//
// With the log-sum-exp at hand one product and one exponential per score are all there is: no maximum, no second product.  The
// product is taken with the keys along the 128 lanes of tensor memory and the queries along its columns, so that a thread
// owns one key and its sum stays in a register from the key tile's first query tile to its last.
//
//   warp 0      TMA producer (K tile of 128 keys into one of two buffers, Q tiles of 128 queries through a ring)
//   warp 1      MMA issuer
//   warp 2      the columns' terms: -lse * log2(e) of 128 queries, -inf for those past the prompt's end, through a ring
//   warps 4-11  exponentials and sums: two per lane quarter, each with 64 of the 128 queries of a tile
//
// Split.  The (key tile, head, query tile) triples of all prompts are numbered in one line, key tile by key tile, and each CTA
// takes an equal stretch of it: the causal triangle and prompts of different lengths leave no CTA with more than one tile
// over another.  Key tiles that several CTAs share leave their sums in scratch, and a second kernel adds them in order.
#include "attn.cuh"
#include "paged.cuh"
#include "tc05.cuh"
#include <type_traits>

namespace tfb {
namespace {

constexpr int PM_TILE = 128;
constexpr int PM_BUFS = 4;  // score buffers of 128 columns
constexpr float kLog2e = 1.4426950408889634f;

template <int HD> struct PmCfg {
  static constexpr int PANELS = HD / 64;
  static constexpr int TILE_BYTES = PANELS * 16384;
  static constexpr int STAGES = HD == 64 ? 4 : 3;
  static constexpr int OFF_K = 0;
  static constexpr int OFF_Q = 2 * TILE_BYTES;
  static constexpr int OFF_C = OFF_Q + STAGES * TILE_BYTES;  // [PM_BUFS][128] column terms
  static constexpr int OFF_BAR = OFF_C + PM_BUFS * 512;
  static constexpr int SMEM_BYTES = OFF_BAR + 256 + 1024;
  static constexpr int THREADS = 384;
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
  int64_t* prefix;  // (B + 1)
  float* halves;    // [2][B][kv_heads][T]
  float* pieces;    // [ctas][2][2][128]
};

__device__ __forceinline__ int pm_count(const PmParams& p, int b) { return p.counts ? min(max(p.counts[b], 0), p.T) : p.T; }
__device__ __forceinline__ int64_t pm_tiles(const PmParams& p, int count) {
  const int64_t n = (count + PM_TILE - 1) / PM_TILE;
  return n * (n + 1) / 2 * p.kv_heads * p.group;
}

// A place in the line of tiles.
struct PmCursor {
  int b, kv, j, r, i, n;  // prompt, key head, key tile, query head of the group, query tile, tiles of the prompt
  __device__ __forceinline__ void seek(const PmParams& p, int b_, int64_t in) {
    b = b_;
    n = (pm_count(p, b) + PM_TILE - 1) / PM_TILE;
    const int64_t per = (int64_t)n * (n + 1) / 2 * p.group;
    kv = (int)(in / per);
    const int64_t rest = in % per, x = rest / p.group;  // key tile j begins at group * (j n - j (j - 1) / 2)
    const double w = 2.0 * n + 1.0;
    j = (int)((w - sqrt(fmax(w * w - 8.0 * (double)x, 0.0))) * 0.5);
    j = min(max(j, 0), n - 1);
    while (j > 0 && start(j) > x) --j;
    while (j + 1 < n && start(j + 1) <= x) ++j;
    const int64_t left = rest - start(j) * p.group;
    r = (int)(left / (n - j));
    i = j + (int)(left % (n - j));
  }
  __device__ __forceinline__ int64_t start(int64_t j) const { return j * n - j * (j - 1) / 2; }
  __device__ __forceinline__ bool begins() const { return r == 0 && i == j; }
  __device__ __forceinline__ bool ends(const PmParams& p) const { return i + 1 == n && r + 1 == p.group; }
  __device__ __forceinline__ void step(const PmParams& p) {
    if (++i < n) return;
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

__device__ __forceinline__ float pm_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  uint64_t* s_full = q_empty + C::STAGES;   // [PM_BUFS] scores are in tensor memory
  uint64_t* s_empty = s_full + PM_BUFS;     // [PM_BUFS] and have been read (8 warps)
  uint64_t* c_full = s_empty + PM_BUFS;     // [PM_BUFS] column terms are in shared memory
  uint64_t* c_empty = c_full + PM_BUFS;     // [PM_BUFS]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(c_empty + PM_BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 * 2 + 2 * 4 + 4 * PM_BUFS) * 8 + 8 <= 256, "barriers");
  __shared__ int64_t sh_scan[C::THREADS / 32];
  __shared__ int64_t sh_base;
  __shared__ int sh_b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < PM_BUFS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 8);
      mbar_init(&c_full[i], 1);
      mbar_init(&c_empty[i], 8);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(tmem_holder, 512);
  }
  grid_dependency_wait();
  allow_dependents();
  if (threadIdx.x == 0) *abort_flag = (*(volatile int*)&g_dev_status != 0) ? 1 : 0;

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
    if (blockIdx.x == 0) {
      p.prefix[b] = base;
      if (p.counts && (p.counts[b] < 0 || p.counts[b] > p.T)) atomicCAS(dev_status(), 0, kBadLength);
    }
    if (from >= base && from < base + tiles) {
      sh_b = b;
      sh_base = base;
    }
    base += tiles;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.prefix[p.B] = total;
  __syncthreads();
  const uint32_t tmem_base = *tmem_holder;
  const bool live = *abort_flag == 0 && count > 0;
  PmCursor cu;
  if (live) cu.seek(p, sh_b, from - sh_base);

  if (!live) {
  } else if (warp == 0) {
    // --------------------------------------------------------------------- TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      int st = 0, nk = 0;
      uint32_t ph = 0;
      for (int64_t t = 0; t < count; ++t) {
        if (t == 0 || cu.begins()) {
          const int kb = nk & 1;
          if (!mbar_wait(&k_empty[kb], ((nk >> 1) & 1) ^ 1, 0x8000 | kb, abort_flag)) break;
          mbar_expect_tx(&k_full[kb], C::TILE_BYTES);
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c)
            tma_load_4d(smem + C::OFF_K + kb * C::TILE_BYTES + c * 16384, &tmK, c * 64, cu.j * PM_TILE, cu.kv, cu.b, &k_full[kb]);
          ++nk;
        }
        if (!mbar_wait(&q_empty[st], ph ^ 1, 0x8100 | st, abort_flag)) break;
        mbar_expect_tx(&q_full[st], C::TILE_BYTES);
#pragma unroll
        for (int c = 0; c < C::PANELS; ++c)
          tma_load_4d(smem + C::OFF_Q + st * C::TILE_BYTES + c * 16384, &tmQ, c * 64, cu.i * PM_TILE, cu.kv * p.group + cu.r, cu.b,
                      &q_full[st]);
        if (++st == C::STAGES) { st = 0; ph ^= 1; }
        if (t + 1 < count) cu.step(p);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------------- MMA issuer
    constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t idesc = instr_desc_f16(PM_TILE, PM_TILE, fmt, 0, 0);
    const uint32_t tb = __shfl_sync(0xffffffffu, tmem_base, 0);
    const uint32_t s0 = smem_u32(smem);
    int st = 0, nk = -1;
    uint32_t ph = 0;
    for (int64_t t = 0; t < count; ++t) {
      const int buf = (int)(t % PM_BUFS);
      bool ok = true;
      if (t == 0 || cu.begins()) {
        ++nk;
        ok = mbar_wait(&k_full[nk & 1], (nk >> 1) & 1, 0x8200 | (nk & 1), abort_flag);
      }
      ok = ok && mbar_wait(&q_full[st], ph, 0x8300 | st, abort_flag);
      ok = ok && mbar_wait(&s_empty[buf], (uint32_t)((t / PM_BUFS) & 1) ^ 1, 0x8400 | buf, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint64_t dk = smem_desc_sw128(s0 + C::OFF_K + (nk & 1) * C::TILE_BYTES, 16, 1024);
      const uint64_t dq = smem_desc_sw128(s0 + C::OFF_Q + st * C::TILE_BYTES, 16, 1024);
#pragma unroll
      for (int s = 0; s < HD / 16; ++s) {
        const uint32_t off = (s / 4) * 16384 + (s % 4) * 32;
        if (elect_one()) tc_mma_ss(tb + buf * PM_TILE, desc_advance(dk, off), desc_advance(dq, off), idesc, s ? 1u : 0u);
      }
      if (elect_one()) {
        tc_commit(&s_full[buf]);
        tc_commit(&q_empty[st]);
        if (cu.ends(p)) tc_commit(&k_empty[nk & 1]);
      }
      __syncwarp();
      if (++st == C::STAGES) { st = 0; ph ^= 1; }
      if (t + 1 < count) cu.step(p);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------------ column terms
    float v[4];
    auto fetch = [&]() {  // of the cursor's tile
      const float* lse = p.lse + cu.b * p.lse_b + (int64_t)(cu.kv * p.group + cu.r) * p.lse_h;
      const int n = pm_count(p, cu.b);
      float slope = 0.f;
      if (MODE == 1) slope = p.slopes[cu.kv * p.group + cu.r] * kLog2e;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = e * 32 + lane, q = cu.i * PM_TILE + c;
        float x = -INFINITY;  // past the end, or a row that gives no weight
        if (q < n) {
          const float l = lse[q];
          x = l == -INFINITY ? -INFINITY : -l * kLog2e - slope * (float)c;
        }
        v[e] = x;
      }
    };
    fetch();
    for (int64_t t = 0; t < count; ++t) {
      const int buf = (int)(t % PM_BUFS);
      const bool ok = mbar_wait(&c_empty[buf], (uint32_t)((t / PM_BUFS) & 1) ^ 1, 0x8500 | buf, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      float* dst = reinterpret_cast<float*>(smem + C::OFF_C) + buf * PM_TILE;
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[e * 32 + lane] = v[e];
      __syncwarp();
      if (lane == 0) mbar_arrive(&c_full[buf]);
      if (t + 1 < count) {
        cu.step(p);
        fetch();
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- exponentials and sums
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const int row = quarter * 32 + lane;  // key of the tile
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint64_t scale2 = f2_pack(p.scale, p.scale);
    float sum = 0.f;
    bool first = cu.begins();
    for (int64_t t = 0; t < count; ++t) {
      const int buf = (int)(t % PM_BUFS);
      const uint32_t par = (uint32_t)((t / PM_BUFS) & 1);
      bool ok = mbar_wait(&c_full[buf], par, 0x8600 | buf, abort_flag);
      ok = ok && mbar_wait(&s_full[buf], par, 0x8700 | buf, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      uint32_t s[64];
      tmem_ld64(tmem_base + lane_base + buf * PM_TILE + half * 64, s);
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_empty[buf]);
      const float4* col = reinterpret_cast<const float4*>(smem + C::OFF_C + buf * 512 + half * 256);
      const int dist = (cu.i - cu.j) * PM_TILE + half * 64 - row;  // of the first of the 64 queries from this thread's key
      float slope = 0.f;
      if (MODE != 0) slope = p.slopes[cu.kv * p.group + cu.r];
      const AlibiLog2<MODE> alibi(slope);
      // exact slopes: the query's place in its tile is in the column's term, the rest is the thread's
      const float shift = MODE == 1 ? -slope * kLog2e * (float)((cu.i - cu.j) * PM_TILE - row) : 0.f;
      const bool diagonal = cu.i == cu.j;
      uint64_t part0 = f2_pack(0.f, 0.f), part1 = part0;
#pragma unroll
      for (int c4 = 0; c4 < 16; ++c4) {
        const float4 a = col[c4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = c4 * 4 + e * 2;
          uint64_t x = f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), scale2, e ? f2_pack(a.z, a.w) : f2_pack(a.x, a.y));
          if (MODE == 1) x = f2_add(x, f2_pack(shift, shift));
          if (MODE > 1) x = alibi.sub_pair(x, (float)(dist + c), (float)(dist + c + 1));
          float x0, x1;
          f2_unpack(x, x0, x1);
          if (diagonal) {
            if (dist + c < 0) x0 = -INFINITY;
            if (dist + c + 1 < 0) x1 = -INFINITY;
          }
          const uint64_t w = f2_pack(pm_ex2(x0), pm_ex2(x1));
          if (e) part1 = f2_add(part1, w);
          else part0 = f2_add(part0, w);
        }
      }
      float w0, w1;
      f2_unpack(f2_add(part0, part1), w0, w1);
      sum += w0 + w1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&c_empty[buf]);
      const bool last = cu.ends(p);
      if (last || t + 1 == count) {
        const int key = cu.j * PM_TILE + row;
        if (first && last) {
          if (key < p.T) p.halves[((int64_t)half * p.B * p.kv_heads + (int64_t)cu.b * p.kv_heads + cu.kv) * p.T + key] = sum;
        } else {
          p.pieces[(((int64_t)blockIdx.x * 2 + first) * 2 + half) * PM_TILE + row] = sum;
        }
        sum = 0.f;
        first = true;  // whatever follows begins with a key tile's first tile
      }
      if (t + 1 < count) cu.step(p);
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
}

// Adds the two halves of each key's sum, or the pieces of a key tile that several CTAs shared; zero past the prompt's end.
__global__ void __launch_bounds__(256) prompt_mass_finish_kernel(const PmParams p) {
  grid_dependency_wait();
  allow_dependents();
  if (*(volatile int*)&g_dev_status != 0) return;
  const int b = blockIdx.x / p.kv_heads, kv = blockIdx.x % p.kv_heads;
  const int key = blockIdx.y * 256 + threadIdx.x;
  if (key >= p.T) return;
  const int count = pm_count(p, b);
  float sum = 0.f;
  const int64_t plane = (int64_t)p.B * p.kv_heads * p.T, at = (int64_t)blockIdx.x * p.T + key;
  if (key < count) {
    const int64_t total = p.prefix[p.B], parts = min(total, (int64_t)p.ctas), n = (count + PM_TILE - 1) / PM_TILE, j = key / PM_TILE;
    const int64_t t0 = p.prefix[b] + (kv * (n * (n + 1) / 2) + j * n - j * (j - 1) / 2) * p.group;
    const int64_t t1 = t0 + (n - j) * p.group - 1;
    const int64_t c0 = ((t0 + 1) * parts - 1) / total, c1 = ((t1 + 1) * parts - 1) / total;
    if (c0 == c1) {
      sum = p.halves[at] + p.halves[plane + at];
    } else {
      for (int64_t c = c0; c <= c1; ++c) {
        const float* piece = p.pieces + (c * 2 + (c == c0)) * 2 * PM_TILE + key % PM_TILE;
        sum += piece[0] + piece[PM_TILE];
      }
    }
  }
  p.out[at] = sum;
}

int encode_tmap_sw128(CUtensorMap* out, const void* base, int dtype, int rank, const uint64_t* dims,
                      const uint64_t* strides_bytes, const uint32_t* box);

namespace {

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
struct PmScratch {
  int64_t halves, pieces, bytes;
};
PmScratch pm_scratch(int64_t B, int64_t kv_heads, int64_t T) {
  PmScratch s;
  s.halves = up256((B + 1) * 8);
  s.pieces = s.halves + up256(2 * B * kv_heads * T * 4);
  s.bytes = s.pieces + (int64_t)sm_count() * 4 * PM_TILE * 4;
  return s;
}

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

extern "C" int64_t tfb_prompt_mass_scratch_bytes(int64_t B, int64_t kv_heads, int64_t T) {
  if (B < 0 || kv_heads < 0 || T < 0) return 0;
  return pm_scratch(B, kv_heads, T).bytes;
}

extern "C" int tfb_prompt_mass(const void* q, const void* k, const float* lse, const int* counts, const float* slopes,
                               int alibi_round, float* out, int64_t B, int64_t kv_heads, int64_t group, int64_t T, int64_t hd,
                               const int64_t* q_strides, const int64_t* k_strides, const int64_t* lse_strides, void* scratch,
                               int64_t scratch_bytes, int dtype, void* stream) {
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
  const PmScratch s = pm_scratch(B, kv_heads, T);
  TFB_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= s.bytes, "prompt_mass: scratch of %lld bytes, %lld wanted",
              (long long)scratch_bytes, (long long)s.bytes);
  CUtensorMap tq, tk;
  const uint32_t box[4] = {64, PM_TILE, 1, 1};
  {
    const uint64_t dims[4] = {(uint64_t)hd, (uint64_t)T, (uint64_t)(kv_heads * group), (uint64_t)B};
    const uint64_t st[3] = {(uint64_t)q_strides[2] * 2, (uint64_t)q_strides[1] * 2, (uint64_t)q_strides[0] * 2};
    if (int rc = encode_tmap_sw128(&tq, q, dtype, 4, dims, st, box)) return rc;
  }
  {
    const uint64_t dims[4] = {(uint64_t)hd, (uint64_t)T, (uint64_t)kv_heads, (uint64_t)B};
    const uint64_t st[3] = {(uint64_t)k_strides[2] * 2, (uint64_t)k_strides[1] * 2, (uint64_t)k_strides[0] * 2};
    if (int rc = encode_tmap_sw128(&tk, k, dtype, 4, dims, st, box)) return rc;
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
  const int64_t n = ceil_div(T, PM_TILE), tiles = n * (n + 1) / 2 * kv_heads * group * B;
  p.ctas = (int)(tiles < sm_count() ? tiles : sm_count());
  char* base = static_cast<char*>(scratch);
  p.prefix = reinterpret_cast<int64_t*>(base);
  p.halves = reinterpret_cast<float*>(base + s.halves);
  p.pieces = reinterpret_cast<float*>(base + s.pieces);
  const int mode = !slopes ? 0 : alibi_round == 0 ? 1 : alibi_round == 1 ? 2 : 4;
  cudaStream_t st = (cudaStream_t)stream;
  int rc = TFB_OK;
  TFB_DISPATCH_16(dtype, E, {
    rc = hd <= 64 ? pm_dispatch<E, 64>(mode, tq, tk, p, st) : pm_dispatch<E, 128>(mode, tq, tk, p, st);
  })
  if (rc) return rc;
  launch_overlapped(prompt_mass_finish_kernel, dim3((unsigned)(B * kv_heads), (unsigned)ceil_div(T, 256)), dim3(256), 0, st, p);
  return launched("prompt_mass: join");
}
