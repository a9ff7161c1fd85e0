// Products with weights held in 4 bits (sm_100a): y = act(x W + bias) + addend with W[k, n] = s[k / group, n] c[k, n], c a whole
// number from -7 to 7 and s a 16-bit number.
//
// Single tokens and small batches would be bound by reading W once, 4.25 bits a weight at groups of 64.  The packed layout is the
// operand layout of mma.sync m16n8k16: the 16 bytes that a lane loads are its share of 16 columns (along M) by 64 rows (along
// the contraction), so that weights go from global memory to the instruction without shared memory, and 8 rows of x lie along N.
// Products of codes are exact and their sum over a group meets the scale in 32 bits, so no weight is rounded.
// A warp has a strip of 16 columns and a stretch of the contraction; up to 8 warps of a block share a strip where there are few,
// and join their sums in shared memory, in their order: the result does not depend on timing.  More rows go to the tensor cores of
// the library's own matrix product, each weight as the sum of two 16-bit numbers: nothing of it is rounded there either.
//
// Measured in graphs, weights not in the L2, fp16: 1 x 1024 x 1024 1.5 us (1.7 with an addend); 1 x 4096 x 1024 4.2; 4 x 1024 x
// 50304 8.4 (27.7 MB, 3.3 TB/s); 24 x 2048 x 8192 in groups of 32 9.2; 16 x 4096 x 12288 13.1.  No pipe is full there: for the
// 50304 columns and for 24 rows the counters have issue slots at 52 and 33 %, the whole-number pipe, which makes codes into
// numbers, at 45 and 26 %, the tensor pipe at 19 and 21 %.  What is on its way is little: 20 and 14 warps an SM with two units of
// 512 bytes and one, and the rows of x come from the L1 where they are used.
// Two units in flight at a time for up to 8 rows and one for more, in 16 warps an SM at least, were the fastest of 1, 2 and 4 with
// 8 to 32 warps (4 units: 11.5 us for the 50304 columns, one 11.4).  Rings in shared memory, filled by cp.async or bulk copies for
// a block or a warp, were slower throughout (12 to 20 us for the 50304 columns).
#include "nibbles.cuh"

namespace tfb {
namespace {

constexpr int kUnit = 64;  // rows of a unit: what a lane's 16 bytes cover
constexpr int kWarps = 8;  // of a block

struct Int4Params {
  const void* x;
  const uint4* codes;      // (strips, units, 32)
  const uint32_t* scales;  // (strips, groups, 8): of columns r and r + 8
  const void *bias, *addend;
  void* out;
  int64_t x_ld, addend_ld, out_ld;
  int M, K, N, units, groups, strips;
  int parts_log2;  // warps of a strip, which share the contraction
  int x_vec;       // rows of x can be read 16 bytes at a time
  int relu;
};

// Eight values of a row of x from column k on, zeros from column K on.
__device__ __forceinline__ uint4 load_x8(const uint16_t* row, int k, int K) {
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < K) v[e / 2] |= (uint32_t)row[k + e] << (16 * (e % 2));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// A warp: a strip of 16 columns, a stretch of its units, NT * 8 rows of x.  U units at a time: their loads are on their way
// together, the next ones' beside the products.  Rows of x that there are none of repeat the last: a column of the product is a row
// of x, and theirs go nowhere.
// GROUP_LOG2: 5, 6 or 7; groups of 32 are two to a unit, of 128 one for two.
template <typename T, int NT, int GROUP_LOG2>
__global__ void __launch_bounds__(kWarps * 32, 2) int4_linear_kernel(const Int4Params p) {
  constexpr int U = NT == 1 ? 2 : 1, GR = GROUP_LOG2 == 5 ? 2 : 1;
  __shared__ float sums[kWarps][NT * 8][17];  // of the warps that share a strip, columns padded by one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  const int m0 = blockIdx.y * (NT * 8), parts = 1 << p.parts_log2, part = warp & (parts - 1);
  const int strip = (blockIdx.x << (3 - p.parts_log2)) + (warp >> p.parts_log2);
  const int share = (p.units + parts - 1) >> p.parts_log2;
  int u = part * share;
  const int end = strip < p.strips ? min(u + share, p.units) : u;
  const uint4* codes = p.codes + ((int64_t)min(strip, p.strips - 1) * p.units + u) * 32 + lane;
  const uint32_t* scales = p.scales + (int64_t)min(strip, p.strips - 1) * p.groups * 8 + r;
  if (u < end) asm volatile("prefetch.global.L2 [%0];" ::"l"(codes));
  grid_dependency_wait();
  allow_dependents();

  const uint16_t* rows[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) rows[t] = static_cast<const uint16_t*>(p.x) + (int64_t)min(m0 + t * 8 + r, p.M - 1) * p.x_ld + 8 * j;

  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
  // a unit's products, added to acc; b: the lane's two chunks of each row
  auto multiply = [&](const uint4& w, const uint32_t (&sc)[GR], const uint4 (&b)[NT][2]) {
    float sum[GR][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t a[2][4];
      expand_nibbles<T>(h ? w.z : w.x, a[0]);
      expand_nibbles<T>(h ? w.w : w.y, a[1]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (GR == 2 || h == 0) mma_first<T>(sum[GR == 2 ? h : 0][t], a[0], b[t][h].x, b[t][h].y);
        else mma<T>(sum[0][t], a[0], b[t][h].x, b[t][h].y);
        mma<T>(sum[GR == 2 ? h : 0][t], a[1], b[t][h].z, b[t][h].w);
      }
    }
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const float2 f = Num<T>::to_f2(*reinterpret_cast<const typename Num<T>::T2*>(&sc[g]));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        acc[t][0] = fmaf(f.x, sum[g][t][0], acc[t][0]);
        acc[t][1] = fmaf(f.x, sum[g][t][1], acc[t][1]);
        acc[t][2] = fmaf(f.y, sum[g][t][2], acc[t][2]);
        acc[t][3] = fmaf(f.y, sum[g][t][3], acc[t][3]);
      }
    }
  };
  auto load_scales = [&](int unit, uint32_t (&sc)[GR]) {
#pragma unroll
    for (int g = 0; g < GR; ++g) sc[g] = scales[(GROUP_LOG2 == 5 ? 2 * unit + g : GROUP_LOG2 == 6 ? unit : unit >> 1) * 8];
  };
  uint4 w[U];
  uint32_t sc[U][GR];
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      w[i] = ld_stream16(codes + i * 32);
      load_scales(u + i, sc[i]);
    }
  };
  const int quick = p.x_vec ? min(end, p.K / kUnit) : u;  // units whose rows of x are whole vectors
  if (u + U <= quick) load();
#pragma unroll 1
  while (u + U <= quick) {
    uint4 now[U], b[U][NT][2];
    uint32_t sn[U][GR];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      now[i] = w[i];
#pragma unroll
      for (int g = 0; g < GR; ++g) sn[i][g] = sc[i][g];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) b[i][t][h] = *reinterpret_cast<const uint4*>(rows[t] + (u + i) * kUnit + h * 32);
    }
    u += U;
    codes += U * 32;
    if (u + U <= quick) load();
#pragma unroll
    for (int i = 0; i < U; ++i) multiply(now[i], sn[i], b[i]);
  }
  for (; u < end; ++u, codes += 32) {
    uint4 b[NT][2];
    uint32_t sn[GR];
    load_scales(u, sn);
    const uint4 now = ld_stream16(codes);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = u * kUnit + h * 32;
        b[t][h] = p.x_vec && k + 8 * j + 8 <= p.K ? *reinterpret_cast<const uint4*>(rows[t] + k) : load_x8(rows[t], k, p.K - 8 * j);
      }
    multiply(now, sn, b);
  }

  const T* bias = static_cast<const T*>(p.bias);
  const T* addend = static_cast<const T*>(p.addend);
  T* out = static_cast<T*>(p.out);
  auto finish = [&](float v, int m, int n) {
    if (m >= p.M || n >= p.N) return;
    if (bias) v += Num<T>::to_f(bias[n]);
    if (p.relu) v = fmaxf(v, 0.f);  // as the matrix products of more rows
    if (addend) v += Num<T>::to_f(addend[(int64_t)m * p.addend_ld + n]);
    out[(int64_t)m * p.out_ld + n] = Num<T>::from_f(v);
  };
  if (parts == 1) {
    if (strip < p.strips)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) finish(acc[t][e], m0 + t * 8 + 2 * j + (e & 1), strip * 16 + r + 8 * (e >> 1));
    return;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[warp][t * 8 + 2 * j + (e & 1)][r + 8 * (e >> 1)] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < (NT * 128) << (3 - p.parts_log2); i += kWarps * 32) {
    const int s = i / (NT * 128), m = i / 16 % (NT * 8), n = i % 16;
    float v = 0.f;
    for (int k = 0; k < parts; ++k) v += sums[(s << p.parts_log2) + k][m][n];
    finish(v, m0 + m, ((blockIdx.x << (3 - p.parts_log2)) + s) * 16 + n);
  }
}

// ------------------------------------------------------------------------------------------------------- packing
constexpr int QR = 128, QC = 64;  // rows and columns of a block's tile: whole groups, 4 strips by 2 units

template <typename T>
__global__ void __launch_bounds__(256) int4_quantize_kernel(const T* __restrict__ w, int64_t w_k, int64_t w_n, int K, int N, int group,
                                                            int units, int groups, int strips, uint32_t* __restrict__ codes,
                                                            T* __restrict__ scales) {
  __shared__ uint16_t tile[QR][QC + 2];
  __shared__ uint16_t most[QR / 32][QC];  // largest magnitude of 32 rows, as bits: a NaN is above infinity
  __shared__ T scale[QR / 32][QC];
  grid_dependency_wait();
  allow_dependents();
  const int k0 = blockIdx.x * QR, n0 = blockIdx.y * QC;
  const bool along_k = w_k < w_n;
  for (int i = threadIdx.x; i < QR * QC; i += 256) {
    const int k = along_k ? i % QR : i / QC, n = along_k ? i / QR : i % QC;
    T v = Num<T>::from_f(0.f);
    if (k0 + k < K && n0 + n < N) v = w[(int64_t)(k0 + k) * w_k + (int64_t)(n0 + n) * w_n];
    tile[k][n] = *reinterpret_cast<const uint16_t*>(&v);
  }
  __syncthreads();
  {
    const int n = threadIdx.x % QC, part = threadIdx.x / QC;
    uint16_t top = 0;
    for (int k = 0; k < 32; ++k) {
      const uint16_t v = tile[part * 32 + k][n] & 0x7fff;
      top = v > top ? v : top;
    }
    most[part][n] = top;
  }
  __syncthreads();
  const int per = group / 32;  // parts of a group
  {
    const int n = threadIdx.x % QC, part = threadIdx.x / QC, first = part / per * per;
    uint16_t top = 0;
    for (int q = 0; q < per; ++q) top = most[first + q][n] > top ? most[first + q][n] : top;
    const T s = scale_of<T>(top);
    scale[part][n] = s;
    const int g = (k0 + part * 32) / group, column = n0 + n;
    if (part == first && g < groups && column < strips * 16)
      scales[(((int64_t)(column / 16) * groups + g) * 8 + column % 8) * 2 + column / 8 % 2] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < QR * QC / 8; i += 256) {
    const int word = i % 128, t = word % 4, j = word / 4 % 4, r = word / 16, unit = i / 128 % 2, strip = i / 256;
    if (k0 / kUnit + unit >= units || n0 / 16 + strip >= strips) continue;
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = unit * kUnit + t / 2 * 32 + j * 8 + t % 2 * 4 + (e % 4 / 2) * 2 + e / 4, n = strip * 16 + e % 2 * 8 + r;
      const float s = Num<T>::to_f(scale[k / 32][n]);
      v |= (uint32_t)(code_of(Num<T>::to_f(*reinterpret_cast<const T*>(&tile[k][n])), s) + 8) << (4 * e);
    }
    codes[(((int64_t)(n0 / 16 + strip) * units + k0 / kUnit + unit) * 128) + word] = v;
  }
}

// What the product of many rows takes beside the weights: its rows, twice.
struct TwiceParams {
  const void* x;
  void* out;  // (M, 2 * units * 64)
  int64_t ld;
  int M, K, units, vec;  // vec: rows of x can be read 16 bytes at a time
  int blocks;            // of the grid, the first ones
};

// The values of a vector that are finite, zeros for the others.
template <typename T> __device__ __forceinline__ uint32_t finite_pair(uint32_t v) {
  constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  if ((v & kExponent) == kExponent) v &= 0xffff0000u;
  if ((v >> 16 & kExponent) == kExponent) v &= 0xffffu;
  return v;
}

// W in 16 bits, transposed: out (strips * 16, units * 64), so that a lane's codes are eight neighbours.  The product of code and scale
// is rounded to 16 bits here.
// SPLIT: unrounded, as the sum of two 16-bit numbers, out (strips * 16, 2 * units * 64): what the rounding leaves in a row's first
// half, the rounded value in its second.  A scale has 11 significant bits (8 in bf16) and a code three, so the rest is three bits,
// on the grid of the scale: exact.  The rows of x, repeated likewise, then make a product in which no weight is rounded, and the
// smaller sums come first.  Beside the rests what is not finite in x is left out: an infinity times a rest of zero would be NaN.
// Bound by writing: rounded, 1536 x 6144 5.3 us, 1024 x 50304 22.8 (131 MB with the codes, 5.7 TB/s).  A product of 1000 rows of
// 1536 x 6144 with weights in two parts takes 36.8 us, with rounded ones it took 22.5, and was off by 2.7e-4 of the output's norm
// where the output's own rounding is 2.1e-4.
template <typename T, bool SMALL, bool SPLIT>
__global__ void __launch_bounds__(256) int4_expand_kernel(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales, int units,
                                                          int groups, int group_log2, int64_t pieces, T* __restrict__ out,
                                                          const TwiceParams x) {
  grid_dependency_wait();
  allow_dependents();
  if (SPLIT && (int)blockIdx.x < x.blocks) {
    const int per = x.units * 8;  // vectors of a row
    const int64_t all = (int64_t)x.M * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)x.blocks * 256) {
      const int64_t m = i / per;
      const int k = (int)(i - m * per) * 8;
      const uint16_t* row = static_cast<const uint16_t*>(x.x) + m * x.ld;
      const uint4 v = x.vec && k + 8 <= x.K ? *reinterpret_cast<const uint4*>(row + k) : load_x8(row, k, x.K);
      uint4* to = reinterpret_cast<uint4*>(static_cast<uint16_t*>(x.out) + m * per * 16 + k);
      to[0] = make_uint4(finite_pair<T>(v.x), finite_pair<T>(v.y), finite_pair<T>(v.z), finite_pair<T>(v.w));
      to[per] = v;
    }
    return;
  }
  const int block = SPLIT ? blockIdx.x - x.blocks : blockIdx.x, blocks = SPLIT ? gridDim.x - x.blocks : gridDim.x;
  const int64_t pitch = (int64_t)units * kUnit * (SPLIT ? 2 : 1);
  const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  for (int64_t i = (int64_t)block * 8 + (threadIdx.x >> 5); i < pieces; i += (int64_t)blocks * 8) {
    const int strip = (int)(i / units), u = (int)(i - (int64_t)strip * units);
    const uint4 w = ld_stream16(codes + i * 32 + lane);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = SMALL ? 2 * u + h : (u * kUnit) >> group_log2;
      const uint32_t s2 = scales[((int64_t)strip * groups + at) * 8 + r];
      const float2 f = Num<T>::to_f2(*reinterpret_cast<const typename Num<T>::T2*>(&s2));
      uint32_t a[2][4];
      expand_nibbles<T>(h ? w.z : w.x, a[0]);
      expand_nibbles<T>(h ? w.w : w.y, a[1]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float v[8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float2 c = Num<T>::to_f2(*reinterpret_cast<const typename Num<T>::T2*>(&a[t][half + 2 * q]));
            v[t * 4 + q * 2] = c.x * (half ? f.y : f.x);
            v[t * 4 + q * 2 + 1] = c.y * (half ? f.y : f.x);
          }
        const uint4 rounded = pack8<T>(v);
        T* to = out + ((int64_t)strip * 16 + half * 8 + r) * pitch + u * kUnit + h * 32 + j * 8;
        if (SPLIT) {
          float back[8];
          unpack8<T>(rounded, back);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] -= back[e];
          *reinterpret_cast<uint4*>(to) = pack8<T>(v);
          to += (int64_t)units * kUnit;
        }
        *reinterpret_cast<uint4*>(to) = rounded;
      }
    }
  }
}

template <typename T, int NT>
int int4_launch(Int4Params p, int group, cudaStream_t st) {
  const int64_t row_tiles = ceil_div(p.M, NT * 8);
  // warps of a strip: as many as there are SMs for (12 warps each; with 24 the 50304 columns take 9.8 us instead of 8.5), with a
  // unit each at least
  p.parts_log2 = 0;
  while (p.parts_log2 < 3 && (2 << p.parts_log2) <= p.units && ((int64_t)p.strips * row_tiles << p.parts_log2) < sm_count() * 12) ++p.parts_log2;
  const dim3 grid((unsigned)ceil_div(p.strips, kWarps >> p.parts_log2), (unsigned)row_tiles);
  const auto kernel = group == 32   ? int4_linear_kernel<T, NT, 5>
                      : group == 64 ? int4_linear_kernel<T, NT, 6>
                                    : int4_linear_kernel<T, NT, 7>;
  launch_overlapped(kernel, grid, dim3(kWarps * 32), 0, st, p);
  return launched("int4_linear");
}

template <typename T>
int int4_dispatch(const Int4Params& p, int group, cudaStream_t st) {
  return p.M <= 8 ? int4_launch<T, 1>(p, group, st) : p.M <= 16 ? int4_launch<T, 2>(p, group, st) : int4_launch<T, 4>(p, group, st);
}

int check_int4(const char* what, int64_t K, int64_t N, int group) {
  TFB_REQUIRE(K >= 1 && N >= 1 && K < (1LL << 30) && N < (1LL << 30), "%s: bad shape", what);
  TFB_REQUIRE(group == 32 || group == 64 || group == 128, "%s: groups of %d: expected 32, 64 or 128", what, group);
  return TFB_OK;
}
int64_t int4_groups(int64_t K, int group) { return ceil_div(ceil_div(K, kUnit) * kUnit, group); }

template <typename T, bool SPLIT>
int int4_expand_launch(const void* codes, const void* scales, int64_t K, int64_t N, int group, void* out, const TwiceParams& x,
                       cudaStream_t st) {
  const int64_t units = ceil_div(K, kUnit), pieces = units * ceil_div(N, 16);
  const int64_t most = (int64_t)sm_count() * 16, blocks = ceil_div(pieces, 8);
  const int log2 = group == 32 ? 5 : group == 64 ? 6 : 7;
  launch_overlapped(group == 32 ? int4_expand_kernel<T, true, SPLIT> : int4_expand_kernel<T, false, SPLIT>,
                    dim3((unsigned)((blocks < most ? blocks : most) + x.blocks)), dim3(256), 0, st, (const uint4*)codes,
                    (const uint32_t*)scales, (int)units, (int)int4_groups(K, group), log2, pieces, (T*)out, x);
  return launched("int4_expand");
}

}  // namespace
}  // namespace tfb

using namespace tfb;

extern "C" int64_t tfb_int4_codes(int64_t K, int64_t N) { return ceil_div(K, kUnit) * ceil_div(N, 16) * 128; }
extern "C" int64_t tfb_int4_scales(int64_t K, int64_t N, int group) {
  return group > 0 ? int4_groups(K, group) * ceil_div(N, 16) * 16 : 0;
}

extern "C" int tfb_int4_quantize(const void* w, int64_t w_k, int64_t w_n, int64_t K, int64_t N, int group, void* codes, void* scales,
                                 int dtype, void* stream) {
  if (int rc = check_int4("int4_quantize", K, N, group)) return rc;
  TFB_REQUIRE(w && codes && scales, "int4_quantize: null buffer");
  const int64_t strips = ceil_div(N, 16), units = ceil_div(K, kUnit);
  TFB_REQUIRE(ceil_div(N, QC) <= 65535, "int4_quantize: too many columns");
  const dim3 grid((unsigned)ceil_div(K, QR), (unsigned)ceil_div(N, QC));
  TFB_DISPATCH_16(dtype, T, {
    launch_overlapped(int4_quantize_kernel<T>, grid, dim3(256), 0, (cudaStream_t)stream, (const T*)w, w_k, w_n, (int)K, (int)N, group,
                      (int)units, (int)int4_groups(K, group), (int)strips, (uint32_t*)codes, (T*)scales);
    return launched("int4_quantize");
  })
}

extern "C" int tfb_int4_expand(const void* codes, const void* scales, int64_t K, int64_t N, int group, void* out, int dtype, void* stream) {
  if (int rc = check_int4("int4_expand", K, N, group)) return rc;
  TFB_REQUIRE(codes && scales && out && aligned16(codes) && aligned16(scales) && aligned16(out),
              "int4_expand: the buffers are not 16-byte aligned");
  TFB_DISPATCH_16(dtype, T, { return int4_expand_launch<T, false>(codes, scales, K, N, group, out, TwiceParams{}, (cudaStream_t)stream); })
}

extern "C" int tfb_int4_split(const void* codes, const void* scales, int64_t K, int64_t N, int group, void* out, const void* x,
                              int64_t x_ld, int64_t M, void* x_out, int dtype, void* stream) {
  if (int rc = check_int4("int4_split", K, N, group)) return rc;
  TFB_REQUIRE(M >= 0 && M < (1LL << 31), "int4_split: bad row count");
  TFB_REQUIRE(M <= 1 || (x_ld >= 0 && x_ld < (1LL << 40)), "int4_split: bad row stride");
  TFB_REQUIRE(codes && scales && out && aligned16(codes) && aligned16(scales) && aligned16(out),
              "int4_split: the buffers are not 16-byte aligned");
  TFB_REQUIRE(M == 0 || (x && x_out && aligned16(x_out)), "int4_split: the buffers are not 16-byte aligned");
  TwiceParams p = {};
  p.x = x;
  p.out = x_out;
  p.ld = x_ld;
  p.M = (int)M;
  p.K = (int)K;
  p.units = (int)ceil_div(K, kUnit);
  p.vec = aligned16(x) && (M <= 1 || x_ld % 8 == 0);
  const int64_t most = (int64_t)sm_count() * 8, blocks = ceil_div(M * p.units * 8, 256);
  p.blocks = (int)(blocks < most ? blocks : most);
  TFB_DISPATCH_16(dtype, T, { return int4_expand_launch<T, true>(codes, scales, K, N, group, out, p, (cudaStream_t)stream); })
}

extern "C" int tfb_int4_linear(const void* x, int64_t x_ld, const void* codes, const void* scales, const void* bias, const void* addend,
                               int64_t addend_ld, void* out, int64_t out_ld, int64_t M, int64_t K, int64_t N, int group, int relu,
                               int dtype, void* stream) {
  if (int rc = check_int4("int4_linear", K, N, group)) return rc;
  TFB_REQUIRE(M >= 0 && M <= 32 * 65535, "int4_linear: bad row count");
  if (M == 0) return TFB_OK;
  TFB_REQUIRE(x && codes && scales && out && aligned16(codes) && aligned16(scales), "int4_linear: the weights are not 16-byte aligned");
  TFB_REQUIRE((M == 1 || (x_ld >= 0 && x_ld < (1LL << 40))) && out_ld >= N, "int4_linear: row stride smaller than the row");
  Int4Params p = {};
  p.x = x;
  p.codes = static_cast<const uint4*>(codes);
  p.scales = static_cast<const uint32_t*>(scales);
  p.bias = bias;
  p.addend = addend;
  p.out = out;
  p.x_ld = x_ld;
  p.addend_ld = addend_ld;
  p.out_ld = out_ld;
  p.M = (int)M;
  p.K = (int)K;
  p.N = (int)N;
  p.units = (int)ceil_div(K, kUnit);
  p.groups = (int)int4_groups(K, group);
  p.strips = (int)ceil_div(N, 16);
  p.x_vec = aligned16(x) && (M == 1 || x_ld % 8 == 0);
  p.relu = relu;
  TFB_DISPATCH_16(dtype, T, { return int4_dispatch<T>(p, group, (cudaStream_t)stream); })
}
