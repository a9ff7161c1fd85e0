// One token per row of logits, drawn with a given uniform number (sm_100a).
//
//   w_i = exp((l_i - max l) / t);  order: larger logits first, equal ones by index;  kept: the first k in that order, of those the
//   first whose predecessors weigh less than p times the sum, of those the ones with w_i >= m;
//   token = the first index j with  sum of the kept w_i, i <= j,  >  u * sum of the kept w_i.
//
// What is kept is a beginning of the order, so it is all logits above a value and some of those equal to it: that cut is what is
// looked for, and nothing is sorted.  All sums are in 64 bits, weights to some 2^-39, the largest exactly 1: a token is the drawn
// one or it is not, and where a sum meets the border between two of 50 thousand tokens, 32 bits would now and then give the
// neighbour.  Sums are taken in a fixed order: the same call gives the same token.
//
// A block or a cluster of blocks has a row; blocks, warps and lanes hold it in the order of its columns, so that the last sums, by
// warps, say which warp has the token.  The cut comes from a list of candidates that are all compared (few of the largest, or of
// the heaviest), from a histogram over all values (16 bits), or from a search (32 bits), below.
//
// Reading the logits is the least of it (13 MB for 128 rows of 50304: 2 us), and no pipe is full: over rows with settings of their
// own issue slots are in use 47 %, the whole-number pipe 30 %, the 64-bit one 8 %.  A call is a chain of steps with a barrier of
// the block or the cluster behind each.  Some are one warp's, while the others wait or have gone (the search for min_p's border,
// the walk through the owner's logits); where many logits are kept each has its exponential once more in the sums by warp, although
// the histogram has their total.  Measured in graphs, fp16 logits: one row of 50304, top_k 40 and top_p 0.95, 14.6 us; 128 rows of
// 50304, temperature alone 28, top_k 40 15, min_p 0.05 18, top_p 0.9 48; bf16, 16 rows of 131071, top_p 0.9 35.
// fp32: 8 rows of 32000, temperature alone 14, top_k 40 31, top_p 0.9 59.
#include <cfloat>
#include <cooperative_groups.h>
#include "common.cuh"

namespace tfb {
namespace {

namespace cg = cooperative_groups;

constexpr int SM_WARPS = 16, SM_THREADS = SM_WARPS * 32, SM_CLUSTER = 8;
constexpr int SM_CUTS = 8;  // values that a round looks at
constexpr double kLog2eD = 1.4426950408889634074;
// The smallest share of the sum that is looked for.  Logits far below the largest weigh some 2^-981 here where 64 bits have
// nothing, and not even a uniform number of zero may draw them: 2^19 of them stay below this.
constexpr double kLeastShare = 0x1p-960;

struct SampleParams {
  const void* logits;
  int64_t ld;
  const float* uniforms;
  const float *temperature, *top_p, *min_p;  // null: the number below for all rows
  const int* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* out;
  int vocab;
  int warp_units;  // 16-byte units of a warp
};

// Whole numbers in the order of 32-bit values; -0 and 0 have one.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? 0u - u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : 0u - k); }
__device__ __forceinline__ void unpack4(const uint4& v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x);
  x[1] = __uint_as_float(v.y);
  x[2] = __uint_as_float(v.z);
  x[3] = __uint_as_float(v.w);
}

// 2^y for y <= 0, by Tang's method (ACM TOMS 15, 1989): 2^(i / 32) from a table, one entry in each lane, times a polynomial for the rest.
// All lanes of the warp take part.
__device__ __forceinline__ double weight_of(double y, double table) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
  constexpr double l = 0.69314718055994530942;
  y = fmax(y, -1021.0);
  const double k = __fma_rn(y, 32.0, kMagic);
  const int n = __double2loint(k);
  const double r = __fma_rn(k - kMagic, -1.0 / 32, y);  // at most 1/64
  double p = __fma_rn(r, l * l * l * l * l / 120, l * l * l * l / 24);
  p = __fma_rn(r, p, l * l * l / 6);
  p = __fma_rn(r, p, l * l / 2);
  p = __fma_rn(r, p, l);
  p = __fma_rn(r, p, 1.0);
  const double s = __shfl_sync(0xffffffffu, table, n & 31) * p;
  return y < -1000.0 ? 0.0 : __hiloint2double(__double2hiint(s) + ((n >> 5) << 20), __double2loint(s));
}

template <typename V> __device__ __forceinline__ V sum_lanes(V v, int from) {
#pragma unroll
  for (int o = from; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Shared {
  double sums[2][SM_CLUSTER][SM_CUTS];
  int counts[2][SM_CLUSTER][SM_CUTS];
  double warp_sums[SM_WARPS][SM_CUTS];
  int warp_counts[SM_WARPS][SM_CUTS];
  float tops[SM_CLUSTER][2];
  int any[SM_CLUSTER];
  float warp_tops[SM_WARPS][2];
  int warp_any[SM_WARPS];
  double all_sums[SM_CLUSTER * SM_WARPS];
  int all_ties[SM_CLUSTER * SM_WARPS];
};

}  // namespace

// ---------------------------------------------------------------------------------------------------------- 32 bits
// The search: a round takes the count and weight above 8 values at once and goes on in the ninth part that holds the border, in
// steps of value and of representation in turn.  The row lies in the cluster's shared memory.
__global__ void __launch_bounds__(SM_THREADS) sample_search_kernel(const SampleParams p) {
  constexpr int W = 4;
  extern __shared__ uint4 units[];
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / blocks;
  const double table = exp2(lane / 32.0);
  if (blocks > 1) cluster.barrier_arrive();  // waited for before the first access to another block's memory
  auto sync = [&]() {
    if (blocks == 1) __syncthreads();
    else cluster.sync();
  };
  grid_dependency_wait();
  allow_dependents();

  // ---- the row's settings
  float t = p.temperature ? p.temperature[row] : p.temperature_all;
  float top_p = p.top_p ? p.top_p[row] : p.top_p_all, min_p = p.min_p ? p.min_p[row] : p.min_p_all;
  int k = p.top_k ? p.top_k[row] : p.top_k_all;
  float u = p.uniforms[row];
  if (!(t > 0.f) || top_p <= 0.f) {
    k = 1;
    t = 1.f;
  }
  if (k <= 0 || k >= p.vocab) k = 0;
  const bool nucleus = top_p < 1.f && k != 1;
  if (!(min_p > 0.f)) min_p = 0.f;
  min_p = fminf(min_p, 1.f);
  u = !(u > 0.f) ? 0.f : fminf(u, 0.99999994f);
  const double per = kLog2eD / (double)t;

  // ---- the warp's part of the row: 16-byte units of memory, with what is not the row's as -infinity
  const float* logits = static_cast<const float*>(p.logits) + row * p.ld;
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(float));
  const uint4* source = reinterpret_cast<const uint4*>(logits - shift);
  const int row_units = (p.vocab + shift + W - 1) / W;
  const int first = (rank * SM_WARPS + warp) * p.warp_units;
  const int mine = max(0, min(p.warp_units, row_units - first));  // of these units there are
  uint4* part = units + warp * p.warp_units;
  float top = -INFINITY, bottom = INFINITY;
  int finite = 0;
  for (int i = lane; i < mine; i += 32) {
    uint4 v = ld_stream16(source + first + i);
    if (first + i == 0 || first + i == row_units - 1) {
      float* e = reinterpret_cast<float*>(&v);
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const int c = (first + i) * W + q - shift;
        if (c < 0 || c >= p.vocab) e[q] = -INFINITY;
      }
    }
    part[i] = v;
    float x[W];
    unpack4(v, x);
#pragma unroll
    for (int q = 0; q < W; ++q) {
      top = fmaxf(top, x[q]);
      if (x[q] > -INFINITY) {
        bottom = fminf(bottom, x[q]);
        ++finite;
      }
    }
  }
  __syncwarp();
  top = warp_max(top);
  bottom = -warp_max(-bottom);
  finite = sum_lanes(finite, 16);
  if (lane == 0) {
    sh.warp_tops[warp][0] = top;
    sh.warp_tops[warp][1] = bottom;
    sh.warp_any[warp] = finite;
  }
  __syncthreads();
  if (blocks > 1) cluster.barrier_wait();
  if (warp == 0) {
    top = warp_max(lane < SM_WARPS ? sh.warp_tops[lane][0] : -INFINITY);
    bottom = -warp_max(lane < SM_WARPS ? -sh.warp_tops[lane][1] : -INFINITY);
    finite = sum_lanes(lane < SM_WARPS ? sh.warp_any[lane] : 0, 16);
    if (lane < blocks) {
      Shared* to = cluster.map_shared_rank(&sh, lane);
      to->tops[rank][0] = top;
      to->tops[rank][1] = bottom;
      to->any[rank] = finite;
    }
  }
  sync();
  top = -INFINITY;
  bottom = INFINITY;
  finite = 0;
  for (int i = 0; i < blocks; ++i) {
    top = fmaxf(top, sh.tops[i][0]);
    bottom = fminf(bottom, sh.tops[i][1]);
    finite += sh.any[i];
  }
  if (finite == 0) {  // nothing is allowed
    if (rank == 0 && tid == 0) p.out[row] = -1;
    return;
  }
  const double peak = (double)top;
  auto weigh = [&](float x) {  // all lanes
    const double w = weight_of(((double)x - peak) * per, table);
    return x == top ? 1.0 : w;
  };

  // Sums over the cluster; every thread gets them.  Two sets of places in turn: one barrier separates the uses of each.
  int parity = 0;
  auto reduce = [&](double (&s)[SM_CUTS], int (&c)[SM_CUTS]) {
    // lanes first: each step halves the values that a lane has
#pragma unroll
    for (int n = SM_CUTS / 2, mask = 16; n > 0; n /= 2, mask /= 2) {
      const bool upper = (lane & mask) != 0;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const double send = upper ? s[i] : s[i + n];
        const int send_c = upper ? c[i] : c[i + n];
        s[i] = (upper ? s[i + n] : s[i]) + __shfl_xor_sync(0xffffffffu, send, mask);
        c[i] = (upper ? c[i + n] : c[i]) + __shfl_xor_sync(0xffffffffu, send_c, mask);
      }
    }
    s[0] = sum_lanes(s[0], 2);
    c[0] = sum_lanes(c[0], 2);
    if ((lane & 3) == 0) {
      const int i = (lane & 16) / 4 + (lane & 8) / 4 + (lane & 4) / 4;
      sh.warp_sums[warp][i] = s[0];
      sh.warp_counts[warp][i] = c[0];
    }
    __syncthreads();
    if (tid < SM_CUTS * blocks) {
      const int i = tid % SM_CUTS;
      double v = 0.0;
      int n = 0;
#pragma unroll
      for (int w = 0; w < SM_WARPS; ++w) {
        v += sh.warp_sums[w][i];
        n += sh.warp_counts[w][i];
      }
      Shared* to = cluster.map_shared_rank(&sh, tid / SM_CUTS);
      to->sums[parity][rank][i] = v;
      to->counts[parity][rank][i] = n;
    }
    sync();
#pragma unroll
    for (int i = 0; i < SM_CUTS; ++i) {
      s[i] = 0.0;
      c[i] = 0;
    }
    for (int b = 0; b < blocks; ++b)
#pragma unroll
      for (int i = 0; i < SM_CUTS; ++i) {
        s[i] += sh.sums[parity][b][i];
        c[i] += sh.counts[parity][b][i];
      }
    parity ^= 1;
  };

  // The cut: all logits above `cut` and the first `ties` of those equal to it.  Below every logit: all of them.
  const uint32_t over = key_of(top) + 1;
  uint32_t low = key_of(bottom) - 1, high = over;  // the search's borders: reached at `low`, not at `high`
  const uint32_t under = low;
  int count_low = finite, count_high = 0;  // logits at or above the two
  double sum_high = 0.0;
  int ties = 0;
  float cuts[SM_CUTS];
  auto place = [&](int round) {  // 8 values between the borders, descending
    const float a = value_of_key(low), b = value_of_key(high);
    const bool even = high - low <= SM_CUTS + 1 || (round & 1) != 0 || !isfinite(b - a);
#pragma unroll
    for (int i = 0; i < SM_CUTS; ++i) {
      uint32_t key;
      if (even) key = high - max((uint32_t)(((uint64_t)(high - low) * (i + 1)) / (SM_CUTS + 1)), 1u);
      else key = key_of(b - (b - a) * ((i + 1) / (float)(SM_CUTS + 1)));
      cuts[i] = value_of_key(min(max(key, low + 1), high - 1));
    }
  };
  auto narrow = [&](int i_low, const double (&s)[SM_CUTS], const int (&c)[SM_CUTS]) {  // the first of the cuts that reaches the goal
    double sum = sum_high;
    int count = count_high;
    uint32_t h = high;
#pragma unroll
    for (int i = 0; i < SM_CUTS; ++i) {
      if (i < i_low) {
        sum = sum_high + s[i];
        count = count_high + c[i];
        h = key_of(cuts[i]);
      }
      if (i == i_low) {
        low = key_of(cuts[i]);
        count_low = count_high + c[i];
      }
    }
    high = h;
    sum_high = sum;
    count_high = count;
  };

  if (k == 1) {
    low = key_of(top);
    ties = 1;
  } else if (k > 0 && k < finite) {
    for (int round = 0; high - low > 1 && round < 64; ++round) {
      place(round);
      const float a = value_of_key(low), b = value_of_key(high);
      const bool open = high == over;  // whose value may be none
      double s[SM_CUTS];
      int c[SM_CUTS];
#pragma unroll
      for (int i = 0; i < SM_CUTS; ++i) {
        s[i] = 0.0;
        c[i] = 0;
      }
      for (int i = lane; i < mine; i += 32) {
        float x[W];
        unpack4(part[i], x);
#pragma unroll
        for (int q = 0; q < W; ++q)
          if (x[q] > a && (open || x[q] < b))
#pragma unroll
            for (int j = 0; j < SM_CUTS; ++j) c[j] += x[q] >= cuts[j];
      }
      reduce(s, c);
      int reached = SM_CUTS;
#pragma unroll
      for (int i = SM_CUTS - 1; i >= 0; --i)
        if (count_high + c[i] >= k) reached = i;
      narrow(reached, s, c);
    }
    ties = k - count_high;
  } else {
    low = under;
  }

  if (nucleus) {
    // of what is left the first whose predecessors weigh less than p times the sum
    const int tied = ties;
    const double low_weight = __shfl_sync(0xffffffffu, weigh(value_of_key(low)), 0);
    const uint32_t floor = low;
    high = over;
    count_high = 0;
    sum_high = 0.0;
    double goal = 0.0;
    for (int round = 0; round == 0 || (high - low > 1 && round < 64); ++round) {
      if (round == 0) {  // by weights, and the last is the sum of all
        const float steps[SM_CUTS] = {0.7f, 1.5f, 2.5f, 4.f, 6.f, 8.5f, 12.f, 0.f};
#pragma unroll
        for (int i = 0; i < SM_CUTS; ++i)
          cuts[i] = value_of_key(min(max(key_of(isfinite(top) ? top - steps[i] * t : top), low + 1), high - 1));
      } else {
        place(round);
      }
      const float a = value_of_key(low), b = value_of_key(high);
      const bool open = high == over;  // whose value may be none
      double s[SM_CUTS];
      int c[SM_CUTS];
#pragma unroll
      for (int i = 0; i < SM_CUTS; ++i) {
        s[i] = 0.0;
        c[i] = 0;
      }
      const int steps = (mine + 31) / 32;
      for (int step = 0; step < steps; ++step) {
        const int i = step * 32 + lane;
        float x[W];
        unpack4(part[min(i, mine - 1)], x);
#pragma unroll
        for (int q = 0; q < W; ++q) {
          const bool in = i < mine && x[q] > a && (open || x[q] < b);
          if (!__any_sync(0xffffffffu, in)) continue;
          const double w = weigh(x[q]);
          if (in) {
#pragma unroll
            for (int j = 0; j < SM_CUTS; ++j)
              if (x[q] >= cuts[j] || (round == 0 && j == SM_CUTS - 1)) {
                s[j] += w;
                ++c[j];
              }
          }
        }
      }
      reduce(s, c);
      if (round == 0) {
        goal = (double)top_p * (s[SM_CUTS - 1] + tied * low_weight);
        cuts[SM_CUTS - 1] = value_of_key(low);  // what lies at `low` or above it reaches the goal
      }
      int reached = SM_CUTS;
#pragma unroll
      for (int i = SM_CUTS - 1; i >= 0; --i)
        if (sum_high + s[i] >= goal && !(round == 0 && i == SM_CUTS - 1)) reached = i;
      if (round == 0 && reached == SM_CUTS) {  // between the last of the cuts and `low`
        const uint32_t keep = low;
        const int had = count_low;
        narrow(SM_CUTS - 1, s, c);
        low = keep;
        count_low = had;
      } else {
        narrow(reached, s, c);
      }
    }
    const double w = __shfl_sync(0xffffffffu, weigh(value_of_key(low)), 0);
    const double fit = ceil((goal - sum_high) / w);
    const int there = low == floor ? tied : count_low - count_high;
    ties = fit < there ? max((int)fit, 1) : there;  // (w = 0: infinite, or NaN)
    if (low == floor && tied == 0) ties = 0;
  }

  // ---- the kept weights of each warp, then the warp that has the token
  const float cut = value_of_key(low);
  const double cut_weight = __shfl_sync(0xffffffffu, weigh(cut), 0);
  const bool ties_kept = ties > 0 && cut_weight >= (double)min_p;
  const int steps = (mine + 31) / 32;
  double sum = 0.0;
  int equal = 0;
  for (int step = 0; step < steps; ++step) {
    const int i = step * 32 + lane;
    float x[W];
    unpack4(part[min(i, mine - 1)], x);
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const bool in = i < mine && x[q] > cut;
      equal += i < mine && x[q] == cut;
      if (!__any_sync(0xffffffffu, in)) continue;
      const double w = weigh(x[q]);
      if (in && w >= (double)min_p) sum += w;
    }
  }
  sum = sum_lanes(sum, 16);
  equal = sum_lanes(equal, 16);
  if (lane < blocks) {
    Shared* to = cluster.map_shared_rank(&sh, lane);
    to->all_sums[rank * SM_WARPS + warp] = sum;
    to->all_ties[rank * SM_WARPS + warp] = equal;
  }
  sync();
  // each warp for itself, in the order of the warps
  double before = 0.0, total = 0.0, here = 0.0;
  int tie_base = 0, last = -1;
  int seen = 0;
  const int me = rank * SM_WARPS + warp;
  for (int i = 0; i < blocks * SM_WARPS; ++i) {
    const int n = sh.all_ties[i], kept = ties_kept ? max(0, min(n, ties - seen)) : 0;
    const double w = sh.all_sums[i] + kept * cut_weight;
    if (i == me) {
      before = total;
      here = w;
      tie_base = seen;
    }
    if (w > 0.0) last = i;
    seen += n;
    total += w;
  }
  const double goal = fmax((double)u, kLeastShare) * total;
  const bool found = here > 0.0 && before <= goal && (before + here > goal || last == me);
  if (!found) return;
  double base = before;
  int token = -1, rank_base = tie_base;
  for (int step = 0; step < steps; ++step) {
    const int i = step * 32 + lane;
    float x[W];
    unpack4(part[min(i, mine - 1)], x);
    int n = 0;
#pragma unroll
    for (int q = 0; q < W; ++q) n += i < mine && x[q] == cut;
    int upto_n = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto_n, o);
      if (lane >= o) upto_n += v;
    }
    int at = rank_base + upto_n - n;
    rank_base += __shfl_sync(0xffffffffu, upto_n, 31);
    double w[W], mine_sum = 0.0;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const bool in = i < mine && x[q] > cut;
      double v = 0.0;
      if (__any_sync(0xffffffffu, in)) v = weigh(x[q]);
      if (!in || v < (double)min_p) v = 0.0;
      if (i < mine && x[q] == cut && ties_kept && at++ < ties) v = cut_weight;
      w[q] = v;
      mine_sum += v;
    }
    double upto = mine_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    double line = base + (upto - mine_sum);
    int hit = -1, back = -1;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      line += w[q];
      if (w[q] > 0.0) {
        back = q;
        if (hit < 0 && line > goal) hit = q;
      }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), backs = __ballot_sync(0xffffffffu, back >= 0);
    if (hits) {
      const int who = __ffs(hits) - 1;
      token = (first + step * 32 + who) * W + __shfl_sync(0xffffffffu, hit, who) - shift;
      break;
    }
    if (backs) {  // where rounding leaves the goal behind the last kept one, that one
      const int who = 31 - __clz(backs);
      token = (first + step * 32 + who) * W + __shfl_sync(0xffffffffu, back, who) - shift;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) p.out[row] = token;
}

// ---------------------------------------------------------------------------------------------------------- 16 bits
// Few candidates.  The k-th largest of the threads' largest logits is not above the k-th largest logit, so what lies below it is
// out; the same holds for each block of a cluster.  What is left, some more than k from each block, is put in a list; up to 256 of
// them are compared each with each, which gives ranks and the weight ahead of each at once (one row, top_k 40: 20 us by the
// histogram, 14.6 so).
//
// Logits of 16 bits have 2^16 values, and equal logits weigh the same: a histogram over all values is all that the cut needs.
// Blocks count their part of the row (a counter of 16 bits for each value, 128 KB of shared memory), the blocks of a cluster add
// theirs up where there is something to add, and a scan over rows of 64 values gives the cut, with an exponential for each value
// that occurs instead of each logit.
// Then the weights of what is kept are summed in the order of the columns.
namespace {

constexpr int H_THREADS = 1024, H_WARPS = 32, H_ROWS = 1024;  // rows of 64 values, two to a word
constexpr int H_UNITS = 8;                                    // 16-byte units of a lane
constexpr int H_FEW = 256;                                    // logits that are compared each with each
// Logits of a block, at most: with one unit of a lane less than there is room for no block of a cluster has 2^16, which a counter
// does not hold.
constexpr int kMostCounted = H_WARPS * (H_UNITS * 32 - 1) * 8 - 8;

// Values in descending order: bin 0 is the last positive NaN, then infinity, .., the lowest, -infinity and the negative NaNs.
template <typename T> struct Bins;
template <> struct Bins<__half> { static constexpr int kTop = 0x03ff, kEnd = 0xfc00; };         // of infinity, of -infinity
template <> struct Bins<__nv_bfloat16> { static constexpr int kTop = 0x007f, kEnd = 0xff80; };
// the two bins of a word of logits; -0 has 0's
template <typename T> __device__ __forceinline__ uint32_t bins_of(uint32_t word) {
  using T2 = typename Num<T>::T2;
  const T2 v = __hadd2(*reinterpret_cast<const T2*>(&word), Num<T>::from_f2(0.f, 0.f));
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&v);
  return u ^ (0x7fff7fffu - ((u >> 15) & 0x00010001u) * 0x7fffu);
}
template <typename T> __device__ __forceinline__ float value_of(int bin) {
  const uint16_t u = (uint16_t)(bin & 0x8000 ? bin : bin ^ 0x7fff);
  return Num<T>::to_f(*reinterpret_cast<const T*>(&u));
}

struct HistShared {
  uint32_t rows[H_WARPS];  // bit i of word w: row 32 i + w has logits
  int counts[H_ROWS];      // of the whole row of logits
  double weights[H_ROWS];
  int warp_counts[H_WARPS];
  double warp_weights[H_WARPS];
  float warp_tops[H_WARPS], warp_lows[H_WARPS], tops[SM_CLUSTER];
  int found, cut, ties, owner, owner_ties, to_last;
  int least;  // the last bin that weighs enough: not in `cut`, which other warps may still be reading while it is found
  double before, owner_before, goal;
  int few[SM_CLUSTER], limits[SM_CLUSTER], total;
  int list_bin[H_FEW], list_col[H_FEW], part_count[4][H_FEW];
  double list_weight[H_FEW], part_weight[4][H_FEW];
  double all_sums[SM_CLUSTER * H_WARPS];
  int all_ties[SM_CLUSTER * H_WARPS];
};

}  // namespace

template <typename T>
__global__ void __launch_bounds__(H_THREADS, 1) sample_hist_kernel(const SampleParams p) {
  using T2 = typename Num<T>::T2;
  constexpr int W = 8;
  extern __shared__ uint4 smem_units[];
  uint32_t* hist = reinterpret_cast<uint32_t*>(smem_units);
  __shared__ HistShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / blocks;
#pragma unroll
  for (int i = 0; i < 8; ++i) smem_units[i * H_THREADS + tid] = make_uint4(0, 0, 0, 0);
  if (tid == 0) sh.found = H_ROWS;
  const double table = exp2(lane / 32.0);
  auto sync = [&]() {
    if (blocks == 1) __syncthreads();
    else cluster.sync();
  };
  grid_dependency_wait();
  allow_dependents();

  // ---- the warp's part of the row: 16-byte units of memory, with what is not the row's as -infinity
  const T* logits = static_cast<const T*>(p.logits) + row * p.ld;
  const int shift = (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  const uint4* source = reinterpret_cast<const uint4*>(logits - shift);
  const int row_units = (p.vocab + shift + W - 1) / W;
  const int first = (rank * H_WARPS + warp) * p.warp_units;
  const int mine = max(0, min(p.warp_units, row_units - first)), steps = (mine + 31) / 32;  // of these units there are
  const T none = Num<T>::from_f(-INFINITY);
  const uint32_t nones = *reinterpret_cast<const uint16_t*>(&none) * 0x10001u;
  const bool edges = first == 0 || first + mine == row_units;  // the row's first or last unit is among them
  auto load_unit = [&](int step) { return step * 32 + lane < mine ? source[first + step * 32 + lane] : make_uint4(nones, nones, nones, nones); };
  auto trim = [&](uint4& x, int step) {
    const int at = first + step * 32 + lane;
    if (at == 0 || at == row_units - 1) {
      uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const int col = at * W + q - shift;
        if (col < 0 || col >= p.vocab) w[q / 2] = q % 2 ? (w[q / 2] & 0xffffu) | (nones & 0xffff0000u) : (w[q / 2] & 0xffff0000u) | (nones & 0xffffu);
      }
      x = make_uint4(w[0], w[1], w[2], w[3]);
    }
  };
  auto unit_at = [&](int step) {
    uint4 x = load_unit(step);
    if (edges) trim(x, step);
    return x;
  };
  uint4 v[H_UNITS];
#pragma unroll
  for (int i = 0; i < H_UNITS; ++i) v[i] = load_unit(i);
  if (edges) {
#pragma unroll
    for (int i = 0; i < H_UNITS; ++i) trim(v[i], i);
  }
  float t = p.temperature ? p.temperature[row] : p.temperature_all;
  float top_p = p.top_p ? p.top_p[row] : p.top_p_all, min_p = p.min_p ? p.min_p[row] : p.min_p_all;
  int k = p.top_k ? p.top_k[row] : p.top_k_all;
  float u = p.uniforms[row];
  if (!(t > 0.f) || top_p <= 0.f) {
    k = 1;
    t = 1.f;
  }
  if (k <= 0 || k >= p.vocab) k = 0;
  const bool nucleus = top_p < 1.f && k != 1;
  if (!(min_p > 0.f)) min_p = 0.f;
  min_p = fminf(min_p, 1.f);
  u = !(u > 0.f) ? 0.f : fminf(u, 0.99999994f);

  // ---- the largest logit of each thread (NaN is none) and of all
  T2 most = *reinterpret_cast<const T2*>(&v[0].x);
#pragma unroll
  for (int i = 0; i < H_UNITS; ++i) {
    most = __hmax2(most, *reinterpret_cast<const T2*>(&v[i].x));
    most = __hmax2(most, *reinterpret_cast<const T2*>(&v[i].y));
    most = __hmax2(most, *reinterpret_cast<const T2*>(&v[i].z));
    most = __hmax2(most, *reinterpret_cast<const T2*>(&v[i].w));
  }
  const float2 pair = Num<T>::to_f2(most);
  const float mine_top = fmaxf(fmaxf(pair.x, pair.y), -INFINITY);
  float top = warp_max(mine_top);
  const float low = -warp_max(-mine_top);  // the smallest of them
  if (lane == 0) {
    sh.warp_tops[warp] = top;
    sh.warp_lows[warp] = low;
  }
  __syncthreads();
  top = warp_max(sh.warp_tops[lane]);
  if (blocks > 1) {
    cluster.sync();  // the others are there
    if (tid < blocks) cluster.map_shared_rank(&sh, tid)->tops[rank] = top;
    cluster.sync();
    for (int b = 0; b < blocks; ++b) top = fmaxf(top, sh.tops[b]);
  }
  if (top == -INFINITY) {  // nothing is allowed
    if (rank == 0 && tid == 0) p.out[row] = -1;
    return;
  }
  auto bin_of = [&](float x) {  // of a value of the type
    const T y = Num<T>::from_f(x + 0.f);
    const int b = *reinterpret_cast<const uint16_t*>(&y);
    return b & 0x8000 ? b : b ^ 0x7fff;
  };
  const int top_bin = bin_of(top);

  // Weights from the difference to the top logit, which is exact in 64 bits: the top one weighs exactly 1, so that sums of equal
  // logits are whole numbers and a border that they meet exactly is met.  (128 rows of 50304 with settings of their own take 45.4
  // us; 45.7 with weights from the logit itself, one sum less each, whose rounding put one token too many into a nucleus of equal
  // logits.)  In the other form where the top logit is infinite, or 32 bits do not tell `lowest` from it.
  const double per = kLog2eD / (double)t, per32 = per * 32.0, peak = (double)top;
  constexpr double kMagic = 6755399441055744.0;  // as in weight_of
  const bool near_by = fabs(peak * per32) < 16384.0;
  const float lowest = top - 680.f * t;  // from there on 2^-981: nothing
  auto weigh_near = [&](float x) {       // all lanes
    constexpr double l = 0.69314718055994530942 / 32;
    const double d = (double)fmaxf(x, lowest) - peak, k_ = __fma_rn(d, per32, kMagic);
    const int n = __double2loint(k_);
    const double r = __fma_rn(d, per32, kMagic - k_);  // at most 1/2; the polynomial leaves 2^-39 of the weight
    const double q = __fma_rn(r, __fma_rn(r, __fma_rn(r, l * l * l * l / 24, l * l * l / 6), l * l / 2), l);
    const double base = __shfl_sync(0xffffffffu, table, n), w = __fma_rn(base, r * q, base);
    return __hiloint2double(__double2hiint(w) + ((n << 15) & 0xfff00000), __double2loint(w));
  };
  auto weigh_far = [&](float x) {
    const double w = weight_of(((double)x - peak) * per, table);
    return x == top ? 1.0 : w;
  };
  auto weigh = [&](float x) { return near_by ? weigh_near(x) : weigh_far(x); };
  // The weights of the warp's logits above a value, and how many are equal to it.
  auto sweep = [&](float above, bool count, int& equal) {
    double sum = 0.0;
    equal = 0;
    uint4 next = unit_at(0);
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      const uint32_t w[4] = {next.x, next.y, next.z, next.w};
      if (step + 1 < steps) next = unit_at(step + 1);
      float x[W];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = Num<T>::to_f2(*reinterpret_cast<const T2*>(&w[q]));
        x[2 * q] = f.x;
        x[2 * q + 1] = f.y;
      }
      float high = x[0];
#pragma unroll
      for (int q = 1; q < W; ++q) high = fmaxf(high, x[q]);
      if (!__any_sync(0xffffffffu, high >= above)) continue;
      if (count) {
#pragma unroll
        for (int q = 0; q < W; ++q) equal += x[q] == above;
      }
      if (!__any_sync(0xffffffffu, high > above)) continue;
      if (near_by) {
#pragma unroll
        for (int q = 0; q < W; ++q) {
          const double y = weigh_near(x[q]);
          if (x[q] > above) sum += y;
        }
      } else {
#pragma unroll
        for (int q = 0; q < W; ++q) {
          const double y = weigh_far(x[q]);
          if (x[q] > above) sum += y;
        }
      }
    }
    sum = sum_lanes(sum, 16);
    equal = __reduce_add_sync(0xffffffffu, equal);
    return sum;
  };
  const int me = rank * H_WARPS + warp;
  auto share = [&](double sum, int equal) {  // each warp's with all blocks
    if (lane < blocks) {
      HistShared* to = cluster.map_shared_rank(&sh, lane);
      to->all_sums[me] = sum;
      to->all_ties[me] = equal;
    }
    sync();
  };

  // ---- Only what may be above the cut is counted: of the k largest none is below the k-th largest of the threads' largest ones.
  int limit = Bins<T>::kEnd - 1;
  if (k > 1 && k <= H_THREADS) {
    const int own = mine_top > -INFINITY ? bin_of(mine_top) : Bins<T>::kEnd;
    const float low = -warp_max(-sh.warp_lows[lane]);
    int lo = top_bin - 1;  // too few up to there
    if (low > -INFINITY) limit = bin_of(low);
    while (limit - lo > 1) {
      const int mid = (lo + limit) / 2;
      if (__syncthreads_count(own <= mid) >= k) limit = mid;
      else lo = mid;
    }
  }

  // ---- Few of them: a list in the order of the columns, each compared with all others.
  const bool threshold = k == 0 && !nucleus && min_p > 0.f;
  if ((k > 1 && k <= H_FEW) || threshold) {
    if (threshold) {  // a little below what weighs enough
      const float least = t * logf(min_p);
      limit = min(bin_of(isfinite(top) ? fmaxf(top + least - 1e-5f * (fabsf(top) - least), -FLT_MAX) : top) + 1, limit);
    }
    uint2* raw = reinterpret_cast<uint2*>(smem_units + H_ROWS * 8);  // the first block's has (bin, column) of each block's, H_FEW to a block
    uint2* to_first = cluster.map_shared_rank(raw, 0) + rank * H_FEW;
    auto few = [&](uint32_t bin) { return bin - Bins<T>::kTop <= (uint32_t)(limit - Bins<T>::kTop); };
    int mine_few = 0;
    uint32_t some = 0;  // units with any in the warp
#pragma unroll
    for (int i = 0; i < H_UNITS; ++i) {
      if (i * 32 >= mine) break;
      const uint32_t words[4] = {bins_of<T>(v[i].x), bins_of<T>(v[i].y), bins_of<T>(v[i].z), bins_of<T>(v[i].w)};
      int n = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) n += few(words[q] & 0xffffu) + few(words[q] >> 16);
      mine_few += n;
      some |= (uint32_t)(__any_sync(0xffffffffu, n != 0) != 0) << i;
    }
    const int warp_few = __reduce_add_sync(0xffffffffu, mine_few);
    if (lane == 0) sh.warp_counts[warp] = warp_few;
    __syncthreads();
    int upto = sh.warp_counts[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    const int block_few = __shfl_sync(0xffffffffu, upto, 31);
    int at = __shfl_sync(0xffffffffu, upto, warp) - warp_few;  // the warp's first place
    if (block_few <= H_FEW) {
#pragma unroll 1
      for (; some != 0; some &= some - 1) {
        const int step = __ffs(some) - 1;
        const uint4 unit = unit_at(step);
        const uint32_t words[4] = {bins_of<T>(unit.x), bins_of<T>(unit.y), bins_of<T>(unit.z), bins_of<T>(unit.w)};
        int n = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) n += few(words[q] & 0xffffu) + few(words[q] >> 16);
        int lanes = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int m = __shfl_up_sync(0xffffffffu, lanes, o);
          if (lane >= o) lanes += m;
        }
        int place = at + lanes - n;
        at += __shfl_sync(0xffffffffu, lanes, 31);
        if (n != 0) {
#pragma unroll
          for (int q = 0; q < W; ++q) {
            const uint32_t bin = q & 1 ? words[q / 2] >> 16 : words[q / 2] & 0xffffu;
            if (few(bin)) {
              to_first[place++] = make_uint2(bin, (first + step * 32 + lane) * W + q - shift);
            }
          }
        }
      }
    }
    if (tid < blocks) {
      HistShared* to = cluster.map_shared_rank(&sh, tid);
      to->few[rank] = block_few;
      to->limits[rank] = limit;
    }
    sync();
    // The first block has those within all blocks' bounds, still in order; if they are too many it says so.
    int total = 0;
    if (rank == 0) {
      bool in[2];
      uint2 entry[2];
      int most = 0, bound = Bins<T>::kEnd;
      for (int b = 0; b < blocks; ++b) {
        most = max(most, sh.few[b]);
        bound = min(bound, sh.limits[b]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int place = 2 * tid + e;
        in[e] = most <= H_FEW && place < blocks * H_FEW && (place & (H_FEW - 1)) < sh.few[place / H_FEW];
        entry[e] = in[e] ? raw[place] : make_uint2(0, 0);
        in[e] = in[e] && (int)entry[e].x <= bound;
      }
      const unsigned ones[2] = {__ballot_sync(0xffffffffu, in[0]), __ballot_sync(0xffffffffu, in[1])}, lt = (1u << lane) - 1;
      if (lane == 0) sh.warp_counts[warp] = __popc(ones[0]) + __popc(ones[1]);
      __syncthreads();
      int warps = sh.warp_counts[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, warps, o);
        if (lane >= o) warps += n;
      }
      total = most <= H_FEW ? __shfl_sync(0xffffffffu, warps, 31) : H_FEW + 1;
      int to = __shfl_sync(0xffffffffu, warps, warp) - (__popc(ones[0]) + __popc(ones[1])) + __popc(ones[0] & lt) + __popc(ones[1] & lt);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (in[e] && to < H_FEW) {
          sh.list_bin[to] = entry[e].x;
          sh.list_col[to++] = entry[e].y;
        }
      if (tid < blocks) cluster.map_shared_rank(&sh, tid)->total = total;
    }
    sync();
    total = sh.total;
    if (total <= H_FEW) {
      if (rank != 0) return;
      const int i = tid & (H_FEW - 1), part = tid / H_FEW;
      const bool real = i < total;
      const int bin = real ? sh.list_bin[i] : Bins<T>::kEnd;
      const double w = weigh(real ? value_of<T>(bin) : top);
      if (part == 0) sh.list_weight[i] = real ? w : 0.0;
      __syncthreads();
      int before = 0;
      double ahead = 0.0;
      for (int j = part * (H_FEW / 4); j < min((part + 1) * (H_FEW / 4), total); ++j) {
        const int other = sh.list_bin[j];
        const bool is = other < bin || (other == bin && j < i);
        before += is;
        if (is) ahead += sh.list_weight[j];
      }
      sh.part_count[part][i] = before;
      sh.part_weight[part][i] = ahead;
      __syncthreads();
      before = 0;
      ahead = 0.0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        before += sh.part_count[q][i];
        ahead += sh.part_weight[q][i];
      }
      const int wanted = k > 0 ? min(k, total) : total;
      if (part == 0 && real && before == wanted - 1) sh.before = ahead + w;
      __syncthreads();
      const double goal = (double)top_p * sh.before, enough = (double)min_p;
      const bool keep = part == 0 && real && before < wanted && (!nucleus || before == 0 || ahead < goal) && w >= enough;
      double line = keep ? w : 0.0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double n = __shfl_up_sync(0xffffffffu, line, o);
        if (lane >= o) line += n;
      }
      if (lane == 31) sh.warp_weights[warp] = line;
      if (tid == 0) sh.owner = -1;
      __syncthreads();
      double all = 0.0, base = 0.0;
#pragma unroll
      for (int q = 0; q < H_FEW / 32; ++q) {
        if (q < warp) base += sh.warp_weights[q];
        all += sh.warp_weights[q];
      }
      line += base;
      // the first whose sum is above the goal; where rounding leaves none, the last
      const double aim = fmax((double)u, kLeastShare) * all;
      if (keep && line > aim) atomicMin(&sh.found, i);
      if (keep) atomicMax(&sh.owner, i);
      __syncthreads();
      if (tid == 0) p.out[row] = sh.list_col[sh.found < H_ROWS ? sh.found : sh.owner];
      return;
    }
    // more than that: as any others, each block by its own bound
    limit = k == 0 ? Bins<T>::kEnd - 1 : limit;
  }

  uint32_t set = 0;  // bit i: row 32 i + lane has logits
  int c[2];
  // counts of a row's two bins of a lane, over the cluster
  auto counts_of = [&](int r) {
    uint32_t word = hist[r * 32 + lane];
    c[0] = word & 0xffffu;
    c[1] = word >> 16;
    for (int b = 1; b < blocks; ++b) {
      word = cluster.map_shared_rank(hist, b == rank ? 0 : b)[r * 32 + lane];
      c[0] += word & 0xffffu;
      c[1] += word >> 16;
    }
  };
  auto row_weight = [&](int r) {  // of the lane's two bins
    const double w0 = weigh(value_of<T>(r * 64 + 2 * lane)), w1 = weigh(value_of<T>(r * 64 + 2 * lane + 1));
    return (c[0] ? c[0] * w0 : 0.0) + (c[1] ? c[1] * w1 : 0.0);
  };
  const bool all_weights = nucleus && k == 0;
  // the logits' counts, and of each row of values how many there are in the cluster; for a nucleus of all logits their weights too
  if (k > 1 || all_weights) {
#pragma unroll
    for (int i = 0; i < H_UNITS; ++i) {
      if (i * 32 >= mine) break;
      const uint32_t words[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t b = bins_of<T>(words[q]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t bin = e ? b >> 16 : b & 0xffffu;
          if (bin - Bins<T>::kTop <= (uint32_t)(limit - Bins<T>::kTop)) atomicAdd(hist + (bin >> 1), 1u + (bin & 1) * 0xffffu);
        }
      }
    }
    sh.counts[tid] = 0;
    sh.weights[tid] = 0.0;
    __syncthreads();
    uint32_t bits = 0;
    for (int i = 0; i * 32 + warp <= limit / 64; ++i) {
      const int r = i * 32 + warp;
      const uint32_t word = hist[r * 32 + lane];
      if (!__any_sync(0xffffffffu, word != 0)) continue;
      bits |= 1u << i;
      if (blocks == 1) {
        counts_of(r);
        const int n = __reduce_add_sync(0xffffffffu, c[0] + c[1]);
        const double sum = all_weights ? sum_lanes(row_weight(r), 16) : 0.0;
        if (lane == 0) {
          sh.counts[r] = n;
          sh.weights[r] = sum;
        }
      }
    }
    if (lane == 0) sh.rows[warp] = bits;
    sync();
    set = 0;
    for (int b = 0; b < blocks; ++b) set |= cluster.map_shared_rank(&sh, b)->rows[lane];
    if (blocks > 1) {
      for (uint32_t todo = __shfl_sync(0xffffffffu, set, warp); todo != 0; todo &= todo - 1) {
        const int i = __ffs(todo) - 1, r = i * 32 + warp;
        if ((i & (blocks - 1)) != rank) continue;
        counts_of(r);
        const double sum = all_weights ? sum_lanes(row_weight(r), 16) : 0.0;
        const int n = __reduce_add_sync(0xffffffffu, c[0] + c[1]);
        if (lane < blocks) {
          HistShared* other = cluster.map_shared_rank(&sh, lane);
          other->counts[r] = n;
          other->weights[r] = sum;
        }
      }
      cluster.sync();
    }
  }
  // sums up to each row, thread by thread
  auto scan = [&](auto upto, auto* warps) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const auto n = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += n;
    }
    if (lane == 31) warps[warp] = upto;
    __syncthreads();
    auto all = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const auto n = __shfl_up_sync(0xffffffffu, all, o);
      if (lane >= o) all += n;
    }
    const auto before = __shfl_sync(0xffffffffu, all, warp ? warp - 1 : 0);
    if (warp) upto += before;
    return upto;
  };
  // the first row whose sum reaches a goal
  auto find_row = [&](bool reached) {
    const unsigned ones = __ballot_sync(0xffffffffu, reached);
    if (ones && lane == __ffs(ones) - 1) atomicMin(&sh.found, tid);
    __syncthreads();
    return sh.found;
  };
  int cut = Bins<T>::kEnd, ties = 0;  // all bins before `cut` are kept, and of it so many
  if (k == 1) {
    cut = top_bin;
    ties = 1;
  } else if (k > 0) {
    const int n = sh.counts[tid], upto = scan(n, sh.warp_counts);
    const int r = find_row(upto >= k);
    if (r < H_ROWS) {
      if (tid == r) sh.ties = k - (upto - n);  // wanted of the row
      __syncthreads();
      if (warp == 0) {
        counts_of(r);
        int lanes = c[0] + c[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v_ = __shfl_up_sync(0xffffffffu, lanes, o);
          if (lane >= o) lanes += v_;
        }
        const int left = sh.ties - (lanes - c[0] - c[1]);  // wanted of this lane's and those behind it
        __syncwarp();
        if (lane == __ffs(__ballot_sync(0xffffffffu, left <= c[0] + c[1])) - 1) {
          const bool second = left > c[0];
          sh.cut = r * 64 + 2 * lane + second;
          sh.ties = left - (second ? c[0] : 0);
          sh.found = H_ROWS;
        }
      }
      __syncthreads();
      cut = sh.cut;
      ties = sh.ties;
    }
  }
  if (nucleus) {
    // of a row's counts what is left
    auto cut_off = [&](int r) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int bin = r * 64 + 2 * lane + e;
        c[e] = bin < cut ? c[e] : bin == cut ? ties : 0;
      }
    };
    if (!all_weights) {
      const int last = min(cut / 64, H_ROWS - 1);
      for (uint32_t todo = __shfl_sync(0xffffffffu, set, warp); todo != 0; todo &= todo - 1) {
        const int r = (__ffs(todo) - 1) * 32 + warp;
        if (r > last) break;
        counts_of(r);
        cut_off(r);
        const double sum = sum_lanes(row_weight(r), 16);
        if (lane == 0) sh.weights[r] = sum;
      }
      __syncthreads();
    }
    const double own = sh.weights[tid], mass = scan(own, sh.warp_weights);
    if (tid == H_THREADS - 1) sh.goal = (double)top_p * mass;
    __syncthreads();
    const double goal = sh.goal;
    const int r = find_row(mass >= goal && own > 0.0);
    if (r < H_ROWS) {  // (else rounding alone has put the goal behind the last)
      if (tid == r) sh.before = mass - own;
      __syncthreads();
      if (warp == 0) {
        counts_of(r);
        cut_off(r);
        const double w0 = weigh(value_of<T>(r * 64 + 2 * lane)), w1 = weigh(value_of<T>(r * 64 + 2 * lane + 1));
        const double m0 = c[0] ? c[0] * w0 : 0.0, m1 = c[1] ? c[1] * w1 : 0.0;
        double lanes = m0 + m1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v_ = __shfl_up_sync(0xffffffffu, lanes, o);
          if (lane >= o) lanes += v_;
        }
        const double ahead = sh.before + (lanes - (m0 + m1));
        const unsigned has = __ballot_sync(0xffffffffu, (c[0] | c[1]) != 0);
        const unsigned over = __ballot_sync(0xffffffffu, (c[0] | c[1]) != 0 && ahead + (m0 + m1) >= goal);
        const int who = over ? __ffs(over) - 1 : 31 - __clz(has);  // by rounding the row's last
        if (lane == who) {
          const bool second = c[0] == 0 || (c[1] != 0 && ahead + m0 < goal);
          const int there = second ? c[1] : c[0];
          const double fit = ceil((goal - ahead - (second ? m0 : 0.0)) / (second ? w1 : w0));
          sh.cut = r * 64 + 2 * lane + second;
          sh.ties = fit < there ? max((int)fit, 1) : there;  // (no weight: infinite, or NaN)
        }
      }
      __syncthreads();
      cut = sh.cut;
      ties = sh.ties;
    }
  }
  if (min_p > 0.f) {  // the last value that weighs enough, 32 at a time
    if (warp == 0) {
      const double enough = (double)min_p;
      int lo = top_bin, hi = Bins<T>::kEnd;  // enough, not enough
      while (hi - lo > 1) {
        const int step = (hi - lo + 32) / 33, bin = min(lo + step * (lane + 1), hi - 1);
        const double w = weigh(value_of<T>(bin));
        const unsigned yes = __ballot_sync(0xffffffffu, w >= enough);
        const int n = yes == 0xffffffffu ? 32 : __ffs(~yes) - 1;  // a beginning of the lanes
        const int next = min(lo + step * (n + 1), hi - 1);
        if (n > 0) lo = min(lo + step * n, hi - 1);
        if (n < 32) hi = next;
      }
      if (lane == 0) sh.least = lo;
    }
    __syncthreads();
    if (sh.least < cut) {
      cut = sh.least + 1;
      ties = 0;
    }
  }

  // ---- the kept weights of each warp, then the warp that has the token
  // as a value (-0 is no bin of any logit: what is above it is above the next one)
  const float above = cut < Bins<T>::kEnd ? value_of<T>(cut == 0x8000 ? 0x8001 : cut) : -INFINITY;
  const double cut_weight = __shfl_sync(0xffffffffu, weigh(above), 0);
  const bool ties_kept = ties > 0;
  {
    int equal;
    const double sum = sweep(above, ties_kept, equal);
    share(sum, equal);
  }
  if (warp == 0) {  // `blocks` neighbours to a lane
    int tied = 0;
    for (int q = 0; q < blocks; ++q) tied += sh.all_ties[lane * blocks + q];
    int tie_base = tied;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, tie_base, o);
      if (lane >= o) tie_base += n;
    }
    tie_base -= tied;
    double weight = 0.0;
    int seen = tie_base;
    auto weight_at = [&](int i, int& ties_before) {  // of a warp of the cluster
      const int n = sh.all_ties[i], some = ties_kept ? max(0, min(n, ties - ties_before)) : 0;
      ties_before += n;
      return sh.all_sums[i] + some * cut_weight;
    };
    for (int q = 0; q < blocks; ++q) weight += weight_at(lane * blocks + q, seen);
    double line = weight;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double n = __shfl_up_sync(0xffffffffu, line, o);
      if (lane >= o) line += n;
    }
    const double goal = fmax((double)u, kLeastShare) * __shfl_sync(0xffffffffu, line, 31);
    line -= weight;
    int owner = 1 << 30, last = -1;
    double owner_before = 0.0;
    seen = tie_base;
    int owner_ties = 0;
    for (int q = 0; q < blocks; ++q) {
      const int i = lane * blocks + q, ties_before = seen;
      const double w = weight_at(i, seen);
      if (w > 0.0) {
        last = i;
        if (owner == 1 << 30 && line + w > goal) {
          owner = i;
          owner_before = line;
          owner_ties = ties_before;
        }
      }
      line += w;
    }
    const unsigned owners = __ballot_sync(0xffffffffu, owner < 1 << 30);
    if (owners) {
      const int who = __ffs(owners) - 1;
      owner = __shfl_sync(0xffffffffu, owner, who);
      owner_before = __shfl_sync(0xffffffffu, owner_before, who);
      owner_ties = __shfl_sync(0xffffffffu, owner_ties, who);
    } else {  // by rounding: the last that has any; its last kept one
      owner = __reduce_max_sync(0xffffffffu, last);
      for (int i = 0; i < owner; ++i) owner_ties += sh.all_ties[i];
      owner_before = -INFINITY;
    }
    if (lane == 0) {
      sh.owner = owner;
      sh.owner_before = owner_before;
      sh.owner_ties = owner_ties;
      sh.goal = goal;
      sh.to_last = owners == 0;
    }
  }
  __syncthreads();
  if (sh.owner != me) return;
  const bool to_last = sh.to_last != 0;
  const double aim = sh.goal;
  double base = sh.owner_before;
  int token = -1, rank_base = sh.owner_ties;
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    const uint4 unit = unit_at(step);
    float x[W];
    unpack8<T>(unit, x);
    int n = 0;
#pragma unroll
    for (int q = 0; q < W; ++q) n += x[q] == above;
    int upto_n = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v_ = __shfl_up_sync(0xffffffffu, upto_n, o);
      if (lane >= o) upto_n += v_;
    }
    int at = rank_base + upto_n - n;
    rank_base += __shfl_sync(0xffffffffu, upto_n, 31);
    double ws[W], here = 0.0;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      double y = 0.0;
      if (__any_sync(0xffffffffu, x[q] > above)) y = weigh(x[q]);
      if (!(x[q] > above)) y = 0.0;
      if (x[q] == above && ties_kept && at++ < ties) y = cut_weight;
      ws[q] = y;
      here += y;
    }
    double sums = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v_ = __shfl_up_sync(0xffffffffu, sums, o);
      if (lane >= o) sums += v_;
    }
    double run = base + (sums - here);
    int hit = -1, back = -1;
#pragma unroll
    for (int q = 0; q < W; ++q) {
      run += ws[q];
      if (ws[q] > 0.0) {
        back = q;
        if (hit < 0 && !to_last && run > aim) hit = q;
      }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), backs = __ballot_sync(0xffffffffu, back >= 0);
    if (hits) {
      const int who = __ffs(hits) - 1;
      token = (first + step * 32 + who) * W + __shfl_sync(0xffffffffu, hit, who) - shift;
      break;
    }
    if (backs) {  // where rounding leaves the goal behind the last kept one, that one
      const int who = 31 - __clz(backs);
      token = (first + step * 32 + who) * W + __shfl_sync(0xffffffffu, back, who) - shift;
    }
    base += __shfl_sync(0xffffffffu, sums, 31);
  }
  if (lane == 0) p.out[row] = token;
}

namespace {

template <typename K>
int sample_start(K kernel, const SampleParams& p, int64_t B, int blocks, int threads, int64_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * blocks));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_plain_launch.load(std::memory_order_relaxed) ? 1 : 2;
  (void)cudaLaunchKernelEx(&cfg, kernel, p);
  return launched("sample");
}

// 16 bits
template <typename T>
int sample_by_histogram(SampleParams p, int64_t B, cudaStream_t st) {
  const int64_t row_units = ceil_div((int64_t)p.vocab + 7, 8);
  int blocks = 1;
  // blocks of a row: what their counters hold, and up to four where they find half of the SMs free (16 rows of 131071: 22 to 34
  // us with 2 or 4 blocks; with 8, whose clusters do not all find room at once, 28 to 51.  One row of 50304, top_k 40: 14.6 us
  // with 4 blocks, 22 with 8, whose own 40 largest are too many together for the list)
  while (blocks < SM_CLUSTER && ((int64_t)p.vocab > (int64_t)kMostCounted * blocks ||
                                 (blocks < 4 && B * blocks * 4 <= sm_count() && row_units > H_THREADS / 2 * blocks)))
    blocks *= 2;
  if ((int64_t)p.vocab > (int64_t)kMostCounted * blocks)
    return fail(TFB_ERR_UNSUPPORTED, "sample: %d logits in a row are more than a cluster has room for", p.vocab);
  p.warp_units = (int)ceil_div(row_units, (int64_t)H_WARPS * blocks);
  static std::atomic<uint64_t> done{0};
  constexpr int smem = H_ROWS * 128 + SM_CLUSTER * H_FEW * 8;
  if (int rc = ensure_dynamic_smem(sample_hist_kernel<T>, smem, done, "sample")) return rc;
  return sample_start(sample_hist_kernel<T>, p, B, blocks, H_THREADS, smem, st);
}

// 32 bits
int sample_by_search(SampleParams p, int64_t B, cudaStream_t st) {
  const int64_t row_units = ceil_div((int64_t)p.vocab + 3, 4);
  int blocks = 1;
  // blocks of a row: what the SMs have room for, and as many as its logits need
  while (blocks < SM_CLUSTER && (B * blocks < sm_count() || ceil_div(row_units, (int64_t)SM_WARPS * blocks) * SM_WARPS * 16 > 104 * 1024) &&
         row_units > (int64_t)SM_THREADS * blocks)
    blocks *= 2;
  p.warp_units = (int)ceil_div(row_units, (int64_t)SM_WARPS * blocks);
  const int64_t smem = (int64_t)p.warp_units * SM_WARPS * 16;
  if (smem > 212 * 1024)
    return fail(TFB_ERR_UNSUPPORTED, "sample: %d logits in a row are more than a cluster has room for", p.vocab);
  static std::atomic<uint64_t> done{0};
  if (int rc = ensure_dynamic_smem(sample_search_kernel, 212 * 1024, done, "sample")) return rc;
  return sample_start(sample_search_kernel, p, B, blocks, SM_THREADS, smem, st);
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int tfb_sample(const void* logits, int64_t ld, const float* uniforms, const float* temperature, float temperature_all,
                          const int* top_k, int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                          int64_t* out, int64_t B, int64_t vocab, int dtype, void* stream) {
  TFB_REQUIRE(B >= 0 && B < (1 << 24) && vocab >= 1 && vocab < (1 << 24), "sample: bad shape");
  TFB_REQUIRE(B <= 1 || ld >= 0, "sample: negative row stride");
  if (B == 0) return TFB_OK;
  TFB_REQUIRE(logits && uniforms && out, "sample: null buffer");
  SampleParams p = {};
  p.logits = logits;
  p.ld = ld;
  p.uniforms = uniforms;
  p.temperature = temperature;
  p.temperature_all = temperature_all;
  p.top_k = top_k;
  p.top_k_all = top_k_all;
  p.top_p = top_p;
  p.top_p_all = top_p_all;
  p.min_p = min_p;
  p.min_p_all = min_p_all;
  p.out = out;
  p.vocab = (int)vocab;
  if (dtype == TFB_F32) return sample_by_search(p, B, (cudaStream_t)stream);
  if (dtype == TFB_F16) return sample_by_histogram<__half>(p, B, (cudaStream_t)stream);
  if (dtype == TFB_BF16) return sample_by_histogram<__nv_bfloat16>(p, B, (cudaStream_t)stream);
  return fail(TFB_ERR_ARG, "sample: dtype %d", dtype);
}
