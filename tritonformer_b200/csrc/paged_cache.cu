// Writing prompts into a paged key-value cache, and evicting keys from it by their accumulated attention (sm_100a).
//
// Both move rows of 64 to 256 bytes between places that tables name; what bounds them is the bytes of the rows, so a warp takes
// whole rows in 16-byte chunks, several at a time, and looks the places up beside the copies.
//
// Measured: prompts of up to 4096 keys, 16 x 8 heads of 128 with statistics, 272 MB in and out, 46.0 us (5.9 TB/s; rows stored so that
// they leave the caches first, 48.9 without).  Eviction in place of 4 x 8 heads of 128 from 32768 to 8192 keys 66 us, of which the
// selection takes 31; of 16 x 16 heads of 64 from up to 2048 to 512 keys into other pages 23.7; from 1088 to 1024 keys 10.7.
//
// Eviction has a selection before its copies.  A key's worth is its mass, or infinite while its position is among the
// `recent` last ones; each (sequence, key head) keeps the `keep` worthiest, ties to the lower slot.  With the worth in the upper and
// the inverted slot in the lower half all keys are different 64-bit numbers, and a cluster of one to eight blocks finds the
// keep-th largest by a radix selection, 11 bits a pass.  The passes end as soon as all that is left in a bin stays: after two,
// unless masses are equal, and of a block alone when few are left to be ranked.  The blocks add their histograms through
// distributed shared memory, each a slice of the bins (every block reading every histogram took 5 us a pass of eight blocks, five
// times as long).  Then the keys that go and those that stay behind slot `keep` are numbered in slot order, and a second kernel
// pairs the two: the i-th survivor from behind moves into the i-th slot that becomes free.  So keys that stay in front are not
// touched, no source of a move is the goal of another, and the moves run in any order, in place, all at once.
#include <cooperative_groups.h>
#include "paged.cuh"

namespace tfb {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------------------------------------------------- append
struct AppendParams {
  PageMap map;
  const void *key, *value;
  void *k, *v;
  const int *lengths, *counts, *first;  // counts, first: may be null (all T; the slot's number)
  float* mass;
  int* positions;
  const float* key_mass;
  int64_t k_b, k_h, k_t, v_b, v_h, v_t, m_b, m_h;
  int B, kv_heads, T;
};

constexpr int AP_ROWS = 64;  // rows of a block

// One block: AP_ROWS rows of a (sequence, key head); neighbouring blocks take neighbouring heads, which lie side by side in a
// projection's output.  VEC: 16-byte chunks; otherwise element by element.
template <int HD, bool VEC>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  using E = uint16_t;  // a copy: of the type only the size matters
  constexpr int LANES = HD / 8, PER = 256 / LANES, N = AP_ROWS / PER;
  __shared__ int sh_page[AP_ROWS], sh_row[AP_ROWS];
  grid_dependency_wait();
  allow_dependents();
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads;
  const int cap = (int)p.map.capacity(), len = p.lengths[b];
  const int want = p.counts ? p.counts[b] : p.T;
  const int start = min(max(len, 0), cap), count = min(min(max(want, 0), p.T), cap - start);
  const int t0 = blockIdx.y * AP_ROWS;
  if (blockIdx.y == 0 && h == 0 && threadIdx.x == 0 && (len < 0 || want < 0 || want > p.T || (int64_t)len + want > cap))
    atomicCAS(&g_dev_status, 0, kBadLength);
  if (t0 >= count) return;
  if (threadIdx.x < AP_ROWS) {
    int page = -1, row = 0;
    const int t = t0 + threadIdx.x;
    if (t < count && find_slot(p.map, b, start + t, page, row)) {
      const int64_t o = stat_offset(p.map, page, p.kv_heads, h, row);
      if (p.mass) p.mass[o] = p.key_mass ? p.key_mass[b * p.m_b + h * p.m_h + t] : 0.f;
      if (p.positions) p.positions[o] = (p.first ? p.first[b] : start) + t;
    } else {
      page = -1;
    }
    sh_page[threadIdx.x] = page;
    sh_row[threadIdx.x] = row;
  }
  __syncthreads();
  const E* key = static_cast<const E*>(p.key) + b * p.k_b + h * p.k_h;
  const E* value = static_cast<const E*>(p.value) + b * p.v_b + h * p.v_h;
  const int c = (threadIdx.x % LANES) * 8;
  if constexpr (VEC) {
    uint4 kr[N], vr[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * PER + threadIdx.x / LANES;
      if (sh_page[r] >= 0) {
        kr[i] = ld_stream16(key + (t0 + r) * p.k_t + c);
        vr[i] = ld_stream16(value + (t0 + r) * p.v_t + c);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * PER + threadIdx.x / LANES;
      if (sh_page[r] >= 0) {
        const int64_t o = row_offset(p.map, sh_page[r], h, sh_row[r]) + c;
        st_stream16(static_cast<E*>(p.k) + o, kr[i]);
        st_stream16(static_cast<E*>(p.v) + o, vr[i]);
      }
    }
  } else {
    for (int i = 0; i < N; ++i) {
      const int r = i * PER + threadIdx.x / LANES;
      if (sh_page[r] < 0) continue;
      const int64_t o = row_offset(p.map, sh_page[r], h, sh_row[r]) + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        static_cast<E*>(p.k)[o + e] = key[(t0 + r) * p.k_t + c + e];
        static_cast<E*>(p.v)[o + e] = value[(t0 + r) * p.v_t + c + e];
      }
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- evict
struct EvictParams {
  PageMap map, out_map;
  const void *k, *v;
  void *k_out, *v_out;
  const float* mass;
  const int* positions;
  float* mass_out;
  int* positions_out;
  const int *lengths, *next;  // next: may be null (the length)
  int* left;
  int B, kv_heads, keep, recent;
  int rows_in_place, stats_in_place;  // the outputs are the inputs, slot by slot
  int room;                           // worths that fit shared memory
  int cluster;   // blocks of a (sequence, key head)
  int* moves;    // (B * kv_heads) rows to move
  int* to;       // (B * kv_heads, keep) their goals, ascending
  int* from;     // (B * kv_heads, keep) their sources, ascending
  uint32_t* stay;  // (B * kv_heads, words) bit d: slot d of the first `keep` stays (unset where nothing moves)
  int words;
};

constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_BATCH = 4;  // worths that a thread looks up at a time
constexpr int EV_RANKED = 256;  // of so many keys left, a block alone counts for each how many are above it (a pass saved, with ties three)

// Worths in the order of unsigned numbers; -0 is 0, a mass that is no number is -infinity.
__device__ __forceinline__ uint32_t worth_of(float m) {
  if (m != m) m = -INFINITY;
  const uint32_t u = __float_as_uint(m + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The worths of EV_BATCH slots `EV_THREADS` apart, those from `end` on left out: all lookups of a kind together.
__device__ __forceinline__ void worths_at(const EvictParams& p, int b, int h, int slot, int end, int oldest, uint32_t (&u)[EV_BATCH]) {
  int page[EV_BATCH], row[EV_BATCH], at[EV_BATCH];
  float mass[EV_BATCH];
  const int* table = p.map.tables + b * p.map.table_ld;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < EV_BATCH; ++k) {
    const int s = min(slot + k * EV_THREADS, end - 1), i = (int)((unsigned)s / (unsigned)p.map.page);
    row[k] = s - i * p.map.page;
    page[k] = table[i];
  }
#pragma unroll
  for (int k = 0; k < EV_BATCH; ++k) {
    const bool ok = (unsigned)page[k] < (unsigned)p.map.num_pages;
    bad |= !ok;
    const int64_t o = ok ? stat_offset(p.map, page[k], p.kv_heads, h, row[k]) : 0;
    mass[k] = p.mass[o];
    at[k] = p.positions ? p.positions[o] : slot + k * EV_THREADS;
    if (!ok) at[k] = INT32_MIN, mass[k] = -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < EV_BATCH; ++k) u[k] = worth_of(at[k] >= oldest ? INFINITY : mass[k]);
  if (bad) atomicCAS(&g_dev_status, 0, kBadPage);
}

struct Slot {
  int page, row;
  bool ok;
};
__device__ __forceinline__ Slot slot_at(const PageMap& m, int b, int slot) {  // without a report
  const int i = (int)((unsigned)slot / (unsigned)m.page), page = m.tables[b * m.table_ld + i];
  return {page, slot - i * m.page, (unsigned)page < (unsigned)m.num_pages};
}

// Moves keys, values and statistics of a (sequence, key head): the survivors from behind into the free slots, and where the output
// is another buffer the slots that stay as well.  The block takes every `step`-th batch from `first` on.
template <int HD, int THREADS>
__device__ __forceinline__ void move_rows(const EvictParams& p, int item, int b, int h, int moves, int left, int first, int step) {
  constexpr int ROWS = THREADS / 2, LANES = HD / 8, PER = THREADS / LANES, N = ROWS / PER < 4 ? ROWS / PER : 4;  // N rows at a time
  __shared__ int64_t sh_src[ROWS], sh_dst[ROWS];
  const int* to = p.to + (int64_t)item * p.keep;
  const int* from = p.from + (int64_t)item * p.keep;
  const int batches = (moves + ROWS - 1) / ROWS;
  const int all = batches + (p.rows_in_place ? 0 : (left + ROWS - 1) / ROWS);
  auto stays = [&](int i) { return i < left && (moves == 0 || (p.stay[(int64_t)item * p.words + i / 32] >> (i % 32) & 1) != 0); };
  if (p.rows_in_place && !p.stats_in_place) {  // of slots that stay the statistics alone, all lookups of a kind together
    constexpr int K = 4;
    for (int i0 = first * THREADS * K + threadIdx.x; i0 < left; i0 += step * THREADS * K) {
      int64_t src[K], dst[K];
      float mass[K];
      int position[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = i0 + k * THREADS;
        const Slot a = slot_at(p.map, b, min(i, left - 1)), d = slot_at(p.out_map, b, min(i, left - 1));
        const bool ok = stays(i) && a.ok && d.ok;
        if (i < left && !(a.ok && d.ok)) atomicCAS(&g_dev_status, 0, kBadPage);
        src[k] = ok ? stat_offset(p.map, a.page, p.kv_heads, h, a.row) : -1;
        dst[k] = stat_offset(p.out_map, d.page, p.kv_heads, h, d.row);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        mass[k] = src[k] >= 0 ? p.mass[src[k]] : 0.f;
        position[k] = src[k] >= 0 && p.positions ? p.positions[src[k]] : 0;
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (src[k] >= 0) {
          p.mass_out[dst[k]] = mass[k];
          if (p.positions) p.positions_out[dst[k]] = position[k];
        }
    }
  }
  for (int batch = first; batch < all; batch += step) {
    const bool move = batch < batches;  // otherwise slots that stay
    const bool stats = move || !p.stats_in_place;
    int64_t stat_src = -1, stat_dst = 0;
    __syncthreads();
    if (threadIdx.x < ROWS) {
      const int i = (move ? batch : batch - batches) * ROWS + threadIdx.x;
      int64_t src = -1, dst = 0;
      int source = -1, goal = -1;
      if (move) {
        if (i < moves) {
          source = from[i];
          goal = to[i];
        }
      } else if (stays(i)) {
        source = goal = i;
      }
      int page, row, page2, row2;
      if (source >= 0 && find_slot(p.map, b, source, page, row) && find_slot(p.out_map, b, goal, page2, row2)) {
        src = row_offset(p.map, page, h, row);
        dst = row_offset(p.out_map, page2, h, row2);
        stat_src = stat_offset(p.map, page, p.kv_heads, h, row);
        stat_dst = stat_offset(p.out_map, page2, p.kv_heads, h, row2);
      }
      sh_src[threadIdx.x] = src;
      sh_dst[threadIdx.x] = dst;
    }
    // the statistics' loads go out beside the rows'
    const bool mine = stats && stat_src >= 0;
    float mass = 0.f;
    int position = 0;
    if (mine) {
      mass = p.mass[stat_src];
      if (p.positions) position = p.positions[stat_src];
    }
    __syncthreads();
    const int c = (threadIdx.x % LANES) * 8;
#pragma unroll
    for (int r0 = 0; r0 < ROWS; r0 += PER * N) {
      uint4 kr[N], vr[N];
      int64_t from_row[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        from_row[e] = sh_src[r0 + e * PER + threadIdx.x / LANES];
        if (from_row[e] >= 0) {
          kr[e] = ld_stream16(static_cast<const uint16_t*>(p.k) + from_row[e] + c);
          vr[e] = ld_stream16(static_cast<const uint16_t*>(p.v) + from_row[e] + c);
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int64_t to_row = sh_dst[r0 + e * PER + threadIdx.x / LANES];
        if (from_row[e] >= 0) {
          st_stream16(static_cast<uint16_t*>(p.k_out) + to_row + c, kr[e]);
          st_stream16(static_cast<uint16_t*>(p.v_out) + to_row + c, vr[e]);
        }
      }
    }
    if (mine) {
      p.mass_out[stat_dst] = mass;
      if (p.positions) p.positions_out[stat_dst] = position;
    }
  }
}

// MOVE: the head_dim where the blocks move the rows as well, otherwise 0.
template <int MOVE>
__global__ void __launch_bounds__(EV_THREADS, 2) evict_select_kernel(const EvictParams p) {
  extern __shared__ uint32_t worths[];
  __shared__ __align__(16) int bins[EV_BINS];
  __shared__ int sh_warps[EV_WARPS];
  __shared__ int slice_bins[EV_BINS];  // of this block's slice, all blocks' counts
  __shared__ int sh_slices[2];         // and their sum, in turn: another block may still read the last pass's
  __shared__ int64_t sh_pairs[EV_WARPS], sh_total;
  __shared__ int sh_digit, sh_want, sh_count, sh_found;
  __shared__ uint64_t ranked[EV_RANKED], sh_key;
  cg::cluster_group cluster = cg::this_cluster();
  grid_dependency_wait();
  allow_dependents();
  const int blocks = p.cluster, rank = blockIdx.x % blocks;
  const int item = blockIdx.x / blocks, b = item / p.kv_heads, h = item % p.kv_heads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cap = (int)p.map.capacity(), len = p.lengths[b];
  const int n = min(max(len, 0), cap), keep = min(p.keep, n);
  if (h == 0 && rank == 0 && tid == 0) {
    if (len != n) atomicCAS(&g_dev_status, 0, kBadLength);
    p.left[b] = keep;
  }
  if (n <= keep) {
    if constexpr (MOVE != 0) move_rows<MOVE, EV_THREADS>(p, item, b, h, 0, keep, rank, blocks);
    else if (rank == 0 && tid == 0) p.moves[item] = 0;
    return;
  }
  auto sync = [&]() {
    if (blocks == 1) __syncthreads();
    else cluster.sync();
  };
  const int oldest = (int)max((int64_t)(p.next ? p.next[b] : n) - p.recent, (int64_t)INT32_MIN + 1);
  // the block's slots [base, base + size): whole steps of 32
  const int share = ((n + 31) / 32 + blocks - 1) / blocks * 32;
  const int base = min(rank * share, n), size = min(share, n - base), end = base + size;
  const bool in_smem = share <= p.room;  // else the worths are looked up again in every pass
  if (in_smem)
    for (int i0 = tid; i0 < size; i0 += EV_THREADS * EV_BATCH) {
      uint32_t u[EV_BATCH];
      worths_at(p, b, h, base + i0, end, oldest, u);
#pragma unroll
      for (int k = 0; k < EV_BATCH; ++k)
        if (i0 + k * EV_THREADS < size) worths[i0 + k * EV_THREADS] = u[k];
    }
  // the key of the block's i-th slot; worth and inverted slot
  const int slot_bits = 32 - __clz(n - 1);  // n >= 2
  auto key_of = [&](int i) {
    uint32_t u;
    if (in_smem) {
      u = worths[i];
    } else {
      uint32_t v[EV_BATCH];
      worths_at(p, b, h, base + i, base + i + 1, oldest, v);
      u = v[0];
    }
    return (uint64_t)u << slot_bits | (uint64_t)(n - 1 - (base + i));
  };
  // ---- the keep-th key, as far as it takes: a key stays if its bits in `mask` are at least `prefix`
  uint64_t prefix = 0, mask = 0;
  int want = keep;
#pragma unroll 1
  for (int top = 32 + slot_bits, turn = 0; top > 0; turn ^= 1) {  // top: bits that are not decided yet
    const int shift = max(top - 11, 0), digits = (1 << (top - shift)) - 1;
    top = shift;
    for (int i = tid; i < EV_BINS; i += EV_THREADS) bins[i] = 0;
    if (tid == 0) sh_slices[turn] = sh_found = 0;
    __syncthreads();
    for (int i = tid; i < size; i += EV_THREADS) {
      const uint64_t key = key_of(i);
      if ((key & mask) == prefix) atomicAdd(&bins[(int)(key >> shift) & digits], 1);
    }
    sync();
    const int slice = EV_BINS / blocks;
    int below = 0;  // keys in the slices above the one that the want-th from the top lies in
    int* from_bins = bins;
    if (blocks > 1) {
      int sum = 0;
      for (int i = tid; i < slice; i += EV_THREADS) {
        int c = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < blocks) c += cluster.map_shared_rank(bins, r)[rank * slice + i];
        slice_bins[i] = c;
        sum += c;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0 && sum) atomicAdd(&sh_slices[turn], sum);
      sync();
      int sums[8], owner = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) sums[r] = r < blocks ? *cluster.map_shared_rank(&sh_slices[turn], r) : 0;
      bool found = false;
#pragma unroll
      for (int r = 7; r >= 0; --r)
        if (r < blocks && !found) {
          if (want <= below + sums[r]) {
            owner = r;
            found = true;
          } else {
            below += sums[r];
          }
        }
      from_bins = cluster.map_shared_rank(slice_bins, owner);
      if (tid == 0) sh_digit = owner * slice;
    } else if (tid == 0) {
      sh_digit = 0;
    }
    // the bin in that slice: a thread has up to four, the first thread the top ones
    static_assert(EV_BINS == 4 * EV_THREADS, "bins of a thread");
    const int each = max(slice / EV_THREADS, 1), top_bin = slice - 1 - each * tid;
    int c[4], mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = e < each && top_bin - e >= 0 ? from_bins[top_bin - e] : 0;
      mine += c[e];
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) sh_warps[warp] = upto;
    __syncthreads();
    int before = below + upto - mine;
#pragma unroll
    for (int w = 0; w < EV_WARPS; ++w)
      if (w < warp) before += sh_warps[w];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (before < want && want <= before + c[e]) {
        sh_digit += top_bin - e;
        sh_want = want - before;
        sh_count = c[e];
      }
      before += c[e];
    }
    __syncthreads();
    prefix |= (uint64_t)sh_digit << shift;
    mask |= (uint64_t)digits << shift;
    want = sh_want;
    const int left = sh_count;
    if (left == want) break;  // the whole bin stays
    if (blocks == 1 && left <= EV_RANKED) {  // few enough to be ranked against one another
      for (int i = tid; i < size; i += EV_THREADS) {
        const uint64_t key = key_of(i);
        if ((key & mask) == prefix) ranked[atomicAdd(&sh_found, 1)] = key;
      }
      __syncthreads();
      if (tid < left) {
        const uint64_t key = ranked[tid];
        int above = 0;
        for (int i = 0; i < left; ++i) above += ranked[i] > key;
        if (above == want - 1) sh_key = key;
      }
      __syncthreads();
      prefix = sh_key;
      mask = ~0ull;
      break;
    }
  }
  // ---- number the slots: each warp has a stretch of them, in steps of 32
  const int steps = (size + 31) / 32, per = (steps + EV_WARPS - 1) / EV_WARPS;
  const int lo = min(warp * per, steps), hi = min(lo + per, steps);
  auto stay = [&](int s) {  // which of 32 slots stay
    const int i = s * 32 + lane;
    return __ballot_sync(0xffffffffu, i < size && (key_of(min(i, size - 1)) & mask) >= prefix);
  };
  auto front = [&](int s) {  // those of step s that lie before slot `keep`
    const int f = min(max(keep - base - s * 32, 0), 32);
    return f == 32 ? 0xffffffffu : (1u << f) - 1u;
  };
  int64_t pair = 0;  // slots that become free, and above them (32 bits up) survivors from behind
  for (int s = lo; s < hi; ++s) {
    const unsigned k = stay(s), in_front = front(s);
    pair += __popc(~k & in_front) + ((int64_t)__popc(k & ~in_front) << 32);
  }
  if (lane == 0) sh_pairs[warp] = pair;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < EV_WARPS; ++w) {
    if (w < warp) before += sh_pairs[w];
    total += sh_pairs[w];
  }
  if (blocks > 1) {
    if (tid == 0) sh_total = total;
    cluster.sync();
    total = 0;
    for (int r = 0; r < blocks; ++r) {
      const int64_t y = *cluster.map_shared_rank(&sh_total, r);
      if (r < rank) before += y;
      total += y;
    }
  }
  if (MOVE == 0 && rank == 0 && tid == 0) p.moves[item] = (int)total;
  int hole = (int)before, nth = (int)(before >> 32);
  int* to = p.to + (int64_t)item * p.keep;
  int* from = p.from + (int64_t)item * p.keep;
  for (int s = lo; s < hi; ++s) {
    const unsigned k = stay(s), in_front = front(s), below = (1u << lane) - 1u;
    const unsigned out = ~k & in_front, in = k & ~in_front;
    const int i = base + s * 32 + lane;
    if (out >> lane & 1) to[hole + __popc(out & below)] = i;
    if (in >> lane & 1) from[nth + __popc(in & below)] = i;
    if (lane == 0 && in_front) p.stay[(int64_t)item * p.words + (base / 32 + s)] = k;
    hole += __popc(out);
    nth += __popc(in);
  }
  if (blocks > 1) cluster.sync();  // no block ends while another reads what it counted
  if constexpr (MOVE != 0) {
    if (blocks == 1) __syncthreads();  // the lists are written
    move_rows<MOVE, EV_THREADS>(p, item, b, h, (int)total, keep, rank, blocks);
  }
}

// The moves as a kernel of their own, on more blocks than have selected.
template <int HD>
__global__ void __launch_bounds__(256, 4) evict_move_kernel(const EvictParams p) {
  grid_dependency_wait();
  allow_dependents();
  const int item = blockIdx.x, b = item / p.kv_heads;
  move_rows<HD, 256>(p, item, b, item % p.kv_heads, p.moves[item], p.left[b], blockIdx.y, gridDim.y);
}

constexpr int EV_SMEM = 200 * 1024;  // worths, beside the kernel's own arrays

template <int MOVE>
int evict_select(const EvictParams& p, int64_t smem, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(evict_select_kernel<MOVE>, EV_SMEM, done, "cache_evict")) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.kv_heads * p.cluster));
  cfg.blockDim = dim3(EV_THREADS);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  const int skip = p.cluster == 1 ? 1 : 0;  // a block alone needs no cluster
  cfg.attrs = attr + skip;
  cfg.numAttrs = (g_plain_launch.load(std::memory_order_relaxed) ? 1 : 2) - skip;
  (void)cudaLaunchKernelEx(&cfg, evict_select_kernel<MOVE>, static_cast<const EvictParams>(p));  // error read by launched()
  return launched("cache_evict");
}

template <int HD, bool VEC>
int append_launch(const AppendParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.B * p.kv_heads), (unsigned)ceil_div(p.T, AP_ROWS));
  launch_overlapped(append_kernel<HD, VEC>, grid, dim3(256), 0, st, p);
  return launched("cache_append");
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int tfb_cache_append(const void* key, const void* value, void* k_pages, void* v_pages, const int* tables,
                                const int* lengths, const int* counts, const int* first_positions, float* mass, int* positions,
                                const float* key_mass, int64_t B, int64_t kv_heads, int64_t T, int64_t hd, int64_t num_pages,
                                int64_t page, int64_t width, int64_t table_ld, const int64_t* page_strides,
                                const int64_t* key_strides, const int64_t* value_strides, const int64_t* key_mass_strides,
                                int dtype, void* stream) {
  AppendParams p = {};
  TFB_REQUIRE(page >= 1 && page < (1LL << 31) && width >= 1 && width < (1LL << 31), "cache_append: bad page or table size");
  p.map = {tables, table_ld, num_pages, (int)page, (int)width, page_strides[0], page_strides[1], page_strides[2]};
  if (int rc = check_pages("cache_append", p.map, B, kv_heads, hd, dtype)) return rc;
  TFB_REQUIRE(T >= 0 && T <= 65535 * (int64_t)AP_ROWS, "cache_append: more than %lld keys", (long long)(65535 * (int64_t)AP_ROWS));
  TFB_REQUIRE(B * kv_heads < (1LL << 31), "cache_append: too many rows of heads");
  if (B == 0 || T == 0) return TFB_OK;
  TFB_REQUIRE(aligned16(k_pages) && aligned16(v_pages), "cache_append: the pages are not 16-byte aligned");
  TFB_REQUIRE(!key_mass || mass, "cache_append: masses of the keys without masses of the cache");
  p.key = key;
  p.value = value;
  p.k = k_pages;
  p.v = v_pages;
  p.lengths = lengths;
  p.counts = counts;
  p.first = first_positions;
  p.mass = mass;
  p.positions = positions;
  p.key_mass = key_mass;
  p.k_b = key_strides[0];
  p.k_h = key_strides[1];
  p.k_t = key_strides[2];
  p.v_b = value_strides[0];
  p.v_h = value_strides[1];
  p.v_t = value_strides[2];
  if (key_mass) {
    p.m_b = key_mass_strides[0];
    p.m_h = key_mass_strides[1];
  }
  p.B = (int)B;
  p.kv_heads = (int)kv_heads;
  p.T = (int)T;
  cudaStream_t st = (cudaStream_t)stream;
  bool vec = aligned16(key) && aligned16(value);
  for (int i = 0; i < 3; ++i) vec = vec && key_strides[i] % 8 == 0 && value_strides[i] % 8 == 0;
  if (hd == 32) return vec ? append_launch<32, true>(p, st) : append_launch<32, false>(p, st);
  if (hd == 64) return vec ? append_launch<64, true>(p, st) : append_launch<64, false>(p, st);
  return vec ? append_launch<128, true>(p, st) : append_launch<128, false>(p, st);
}

extern "C" int64_t tfb_cache_evict_scratch_bytes(int64_t B, int64_t kv_heads, int64_t keep) {
  if (B < 0 || kv_heads < 0 || keep < 0) return 0;
  return up256(B * kv_heads * 4) + 2 * up256(B * kv_heads * keep * 4) + up256(B * kv_heads * ((keep + 31) / 32) * 4);
}

extern "C" int tfb_cache_evict(const void* k_pages, const void* v_pages, const float* mass, const int* positions,
                               const int* tables, const int* lengths, const int* next_positions, void* k_out, void* v_out,
                               float* mass_out, int* positions_out, const int* out_tables, int* left, int64_t B,
                               int64_t kv_heads, int64_t hd, int64_t keep, int64_t recent, int64_t page, int64_t num_pages,
                               int64_t width, int64_t table_ld, const int64_t* page_strides, int64_t out_page,
                               int64_t out_num_pages, int64_t out_width, int64_t out_table_ld, const int64_t* out_page_strides,
                               void* scratch, int64_t scratch_bytes, int dtype, void* stream) {
  EvictParams p = {};
  TFB_REQUIRE(page >= 1 && page < (1LL << 31) && width >= 1 && width < (1LL << 31), "cache_evict: bad page or table size");
  TFB_REQUIRE(out_page >= 1 && out_page < (1LL << 31) && out_width >= 1 && out_width < (1LL << 31), "cache_evict: bad page or table size");
  p.map = {tables, table_ld, num_pages, (int)page, (int)width, page_strides[0], page_strides[1], page_strides[2]};
  p.out_map = {out_tables, out_table_ld, out_num_pages, (int)out_page, (int)out_width, out_page_strides[0], out_page_strides[1],
               out_page_strides[2]};
  if (int rc = check_pages("cache_evict", p.map, B, kv_heads, hd, dtype)) return rc;
  if (int rc = check_pages("cache_evict", p.out_map, B, kv_heads, hd, dtype)) return rc;
  TFB_REQUIRE(keep >= 1, "cache_evict: keep %lld: expected at least 1", (long long)keep);
  TFB_REQUIRE(recent >= 0 && recent <= keep, "cache_evict: recent %lld: expected 0 to keep", (long long)recent);
  if (keep > p.map.capacity()) keep = p.map.capacity();
  if (recent > keep) recent = keep;
  TFB_REQUIRE(keep <= p.out_map.capacity(), "cache_evict: %lld keys to keep, and room for %lld", (long long)keep,
              (long long)p.out_map.capacity());
  TFB_REQUIRE(B * kv_heads < (1LL << 28), "cache_evict: too many rows of heads");
  TFB_REQUIRE(mass && mass_out, "cache_evict: no masses");
  TFB_REQUIRE(left && left != lengths, "cache_evict: the new lengths need an array of their own");
  TFB_REQUIRE((positions == nullptr) == (positions_out == nullptr), "cache_evict: positions come with positions for the output");
  TFB_REQUIRE((k_out == k_pages) == (v_out == v_pages), "cache_evict: keys in place and values not, or the other way round");
  const bool stats_shared = mass_out == mass || (positions && positions_out == positions);
  TFB_REQUIRE(out_page == page || (k_out != k_pages && !stats_shared), "cache_evict: the input's own buffers in other shape are no output");
  const int64_t extents[3] = {num_pages < out_num_pages ? num_pages : out_num_pages, kv_heads, page};
  for (int i = 0; i < 3; ++i)
    TFB_REQUIRE(k_out != k_pages || extents[i] == 1 || out_page_strides[i] == page_strides[i],
                "cache_evict: the input's own pages in other shape are no output");
  if (B == 0) return TFB_OK;
  TFB_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && aligned16(k_out) && aligned16(v_out),
              "cache_evict: the pages are not 16-byte aligned");
  TFB_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= tfb_cache_evict_scratch_bytes(B, kv_heads, keep),
              "cache_evict: scratch of %lld bytes, %lld wanted", (long long)scratch_bytes,
              (long long)tfb_cache_evict_scratch_bytes(B, kv_heads, keep));
  p.k = k_pages;
  p.v = v_pages;
  p.k_out = k_out;
  p.v_out = v_out;
  p.mass = mass;
  p.positions = positions;
  p.mass_out = mass_out;
  p.positions_out = positions_out;
  p.lengths = lengths;
  p.next = next_positions;
  p.left = left;
  p.B = (int)B;
  p.kv_heads = (int)kv_heads;
  p.keep = (int)keep;
  p.recent = (int)recent;
  const bool same_tables = out_tables == tables;
  p.rows_in_place = same_tables && k_out == k_pages;
  p.stats_in_place = same_tables && mass_out == mass && positions_out == positions;
  TFB_REQUIRE(same_tables || (k_out != k_pages && mass_out != mass && (!positions || positions_out != positions)),
              "cache_evict: tables of their own need pages of their own");
  TFB_REQUIRE(!same_tables || (mass_out == mass) == (positions_out == positions) || !positions,
              "cache_evict: masses in place and positions not, or the other way round");
  char* base = static_cast<char*>(scratch);
  p.moves = reinterpret_cast<int*>(base);
  p.to = reinterpret_cast<int*>(base + up256(B * kv_heads * 4));
  p.from = reinterpret_cast<int*>(base + up256(B * kv_heads * 4) + up256(B * kv_heads * keep * 4));
  p.stay = reinterpret_cast<uint32_t*>(base + up256(B * kv_heads * 4) + 2 * up256(B * kv_heads * keep * 4));
  p.words = (int)((keep + 31) / 32);
  cudaStream_t st = (cudaStream_t)stream;
  // as many blocks for a (sequence, key head) as the SMs have room for, none with fewer than 2048 slots of a full table
  p.cluster = 1;
  while (p.cluster < 8 && B * kv_heads * p.cluster * 2 <= sm_count() * 2 && p.map.capacity() >= (int64_t)p.cluster * 2 * 2048)
    p.cluster *= 2;
  int64_t smem = (ceil_div(ceil_div(p.map.capacity(), 32), p.cluster) * 32 * 4 + 15) / 16 * 16;
  if (smem > EV_SMEM) smem = EV_SMEM;
  p.room = (int)(smem / 4);
  // Where single blocks select and fill half the SMs they move the rows too: blocks that are done early move while others
  // select, and there is one launch (256 heads of up to 2048 keys into other pages 24.5 us, with two launches 26.3; 96 heads of 1088
  // keys 8 us of the host's time against 13).  Clusters leave the moves to a grid of their own (32 heads of 32768 keys: 68 us, with
  // one launch 71).
  const bool fused = p.cluster == 1 && B * kv_heads * 2 >= sm_count();
  int rc;
  if (!fused) rc = evict_select<0>(p, smem, st);
  else if (hd == 32) rc = evict_select<32>(p, smem, st);
  else if (hd == 64) rc = evict_select<64>(p, smem, st);
  else rc = evict_select<128>(p, smem, st);
  if (rc || fused) return rc;
  // a block for each 128 rows that can move or stay, as far as that takes to fill the SMs
  int64_t shares = ceil_div(keep, 128) * (p.rows_in_place && p.stats_in_place ? 1 : 2);
  const int64_t enough = ceil_div((int64_t)sm_count() * 16, B * kv_heads);
  if (shares > enough) shares = enough;
  const dim3 grid((unsigned)(B * kv_heads), (unsigned)shares);
  if (hd == 32) launch_overlapped(evict_move_kernel<32>, grid, dim3(256), 0, st, p);
  else if (hd == 64) launch_overlapped(evict_move_kernel<64>, grid, dim3(256), 0, st, p);
  else launch_overlapped(evict_move_kernel<128>, grid, dim3(256), 0, st, p);
  return launched("cache_evict: move");
}
