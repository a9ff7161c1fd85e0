// Products with weights held in 4 bits (sm_100a): y = act(x W + bias) + addend with W[k, n] = s[k / group, n] c[k, n], c a whole
// number from -7 to 7 and s a 16-bit number.
//
// Single tokens and small batches are bound by reading W once, 4.25 bits a weight at groups of 64.  The packed layout is the
// operand layout of mma.sync m16n8k16: the 16 bytes that a lane loads are its share of 16 columns (along M) by 64 rows (along
// the contraction), so that weights go from global memory to the instruction without shared memory, and 8 rows of x lie along N.
// A nibble becomes a 16-bit number by being put below a power of two's exponent (1024 + c in fp16, 128 + c in bf16, exactly) and
// subtracting; products of codes are exact and their sum over a group meets the scale in 32 bits, so no weight is rounded.
// The warps of a block share the contraction and join their sums in shared memory, in their order: the result does not depend on
// timing.  More rows than that go to the tensor cores of the library's own matrix product, on weights expanded to 16 bits.
#include "nibbles.cuh"

namespace tfb {
namespace {

constexpr int kUnit = 64;     // rows of a unit: what a lane's 16 bytes cover
constexpr int kMaxWarps = 16;

struct Int4Params {
  const void* x;
  const uint4* codes;   // (strips, units, 32)
  const uint32_t* scales;  // (strips, groups, 8): of columns r and r + 8
  const void *bias, *addend;
  void* out;
  int64_t x_ld, addend_ld, out_ld;
  int M, K, N, units, groups, group_log2, strips;
  int x_vec;    // rows of x can be read 16 bytes at a time
  int out_vec;  // rows of the output and the addend 4 bytes at a time
  int relu;
};

// Eight values of a row from column k on, zeros from column K on.
__device__ __forceinline__ uint4 load_x8(const uint16_t* row, int k, int K, int vec) {
  if (vec && k + 8 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < K) v[e / 2] |= (uint32_t)row[k + e] << (16 * (e % 2));
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// One block: S strips of 16 columns by NT * 8 rows of x; its warps take the units of the contraction in turn.
// SMALL: groups of 32, two to a unit.
template <typename T, int NT, int S, bool SMALL>
__global__ void __launch_bounds__(kMaxWarps * 32) int4_linear_kernel(const Int4Params p) {
  extern __shared__ float sums[];  // [warps][NT * 8][S * 16 + 1]
  constexpr int LD = S * 16 + 1, GR = SMALL ? 2 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int r = lane >> 2, j = lane & 3;
  const int strip0 = blockIdx.x * S, m0 = blockIdx.y * (NT * 8);
  grid_dependency_wait();
  allow_dependents();

  float acc[S][NT][4];
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[s][t][e] = 0.f;

  uint4 w[S];
  uint32_t sc[S][GR];
  auto load = [&](int u) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int strip = min(strip0 + s, p.strips - 1);
      w[s] = ld_stream16(p.codes + ((int64_t)strip * p.units + u) * 32 + lane);
#pragma unroll
      for (int g = 0; g < GR; ++g) {
        const int at = SMALL ? 2 * u + g : (u * kUnit) >> p.group_log2;
        sc[s][g] = p.scales[((int64_t)strip * p.groups + at) * 8 + r];
      }
    }
  };
  int u = warp;
  if (u < p.units) load(u);
  for (; u < p.units; u += warps) {
    uint4 b[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int m = m0 + t * 8 + r;
      const uint16_t* row = static_cast<const uint16_t*>(p.x) + (int64_t)m * p.x_ld;
#pragma unroll
      for (int h = 0; h < 2; ++h) b[t][h] = m < p.M ? load_x8(row, u * kUnit + 32 * h + 8 * j, p.K, p.x_vec) : make_uint4(0, 0, 0, 0);
    }
    uint4 now[S];
    uint32_t scale[S][GR];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      now[s] = w[s];
#pragma unroll
      for (int g = 0; g < GR; ++g) scale[s][g] = sc[s][g];
    }
    if (u + warps < p.units) load(u + warps);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float part[NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (SMALL || h == 0) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[t][e] = 0.f;
        }
        uint32_t a[4];
        expand_nibbles<T>(h ? now[s].z : now[s].x, a);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma<T>(part[t], a, b[t][h].x, b[t][h].y);
        expand_nibbles<T>(h ? now[s].w : now[s].y, a);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma<T>(part[t], a, b[t][h].z, b[t][h].w);
        if (SMALL || h == 1) {
          const float2 f = Num<T>::to_f2(*reinterpret_cast<const typename Num<T>::T2*>(&scale[s][SMALL ? h : 0]));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[s][t][0] = fmaf(f.x, part[t][0], acc[s][t][0]);
            acc[s][t][1] = fmaf(f.x, part[t][1], acc[s][t][1]);
            acc[s][t][2] = fmaf(f.y, part[t][2], acc[s][t][2]);
            acc[s][t][3] = fmaf(f.y, part[t][3], acc[s][t][3]);
          }
        }
      }
    }
  }
  float* mine = sums + warp * (NT * 8) * LD;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(t * 8 + 2 * j + (e & 1)) * LD + s * 16 + r + 8 * (e >> 1)] = acc[s][t][e];
  __syncthreads();
  const T* bias = static_cast<const T*>(p.bias);
  const T* addend = static_cast<const T*>(p.addend);
  T* out = static_cast<T*>(p.out);
  for (int i = threadIdx.x; i < NT * 8 * S * 16; i += blockDim.x) {
    const int m = i / (S * 16), c = i % (S * 16), n = strip0 * 16 + c;
    if (m0 + m >= p.M || n >= p.N) continue;
    float v = 0.f;
    for (int k = 0; k < warps; ++k) v += sums[(k * NT * 8 + m) * LD + c];
    if (bias) v += Num<T>::to_f(bias[n]);
    if (p.relu) v = v < 0.f ? 0.f : v;  // NaN stays
    if (addend) v += Num<T>::to_f(addend[(int64_t)(m0 + m) * p.addend_ld + n]);
    out[(int64_t)(m0 + m) * p.out_ld + n] = Num<T>::from_f(v);
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

// W in 16 bits, transposed: out (strips * 16, units * 64), so that a lane's codes are eight neighbours.  The product of code and scale
// is rounded to 16 bits here: at most half a step of a weight, where the sums over a thousand rows are not exact to that either.
template <typename T, bool SMALL>
__global__ void __launch_bounds__(256) int4_expand_kernel(const uint4* __restrict__ codes, const uint32_t* __restrict__ scales, int units,
                                                          int groups, int group_log2, int64_t pieces, T* __restrict__ out) {
  grid_dependency_wait();
  allow_dependents();
  const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < pieces; i += (int64_t)gridDim.x * 8) {
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
        *reinterpret_cast<uint4*>(out + ((int64_t)strip * 16 + half * 8 + r) * units * kUnit + u * kUnit + h * 32 + j * 8) = pack8<T>(v);
      }
    }
  }
}

template <typename T, int NT, int S>
int int4_launch(const Int4Params& p, int warps, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.strips, S), (unsigned)ceil_div(p.M, NT * 8));
  const size_t smem = (size_t)warps * NT * 8 * (S * 16 + 1) * 4;
  const auto kernel = p.group_log2 == 5 ? int4_linear_kernel<T, NT, S, true> : int4_linear_kernel<T, NT, S, false>;
  launch_overlapped(kernel, grid, dim3(warps * 32), smem, st, p);
  return launched("int4_linear");
}

template <typename T>
int int4_dispatch(const Int4Params& p, cudaStream_t st) {
  const int nt = p.M <= 8 ? 1 : p.M <= 16 ? 2 : p.M <= 32 ? 4 : 8;
  // strips of a warp: more share their loads of x, as long as there are blocks for all SMs
  int s = nt == 1 ? 4 : nt == 2 ? 2 : 1;
  while (s > 1 && ceil_div(p.strips, s) < 2 * sm_count()) s /= 2;
  const int64_t blocks = ceil_div(p.strips, s) * ceil_div(p.M, nt * 8);
  int warps = 1;
  while (warps < kMaxWarps && warps * 2 <= p.units && blocks * warps < sm_count() * 16) warps *= 2;
  while (warps > 1 && (size_t)warps * nt * 8 * (s * 16 + 1) * 4 > 48 * 1024) warps /= 2;
  if (nt == 1) return s == 4 ? int4_launch<T, 1, 4>(p, warps, st) : s == 2 ? int4_launch<T, 1, 2>(p, warps, st) : int4_launch<T, 1, 1>(p, warps, st);
  if (nt == 2) return s == 2 ? int4_launch<T, 2, 2>(p, warps, st) : int4_launch<T, 2, 1>(p, warps, st);
  if (nt == 4) return int4_launch<T, 4, 1>(p, warps, st);
  return int4_launch<T, 8, 1>(p, warps, st);
}

int check_int4(const char* what, int64_t K, int64_t N, int group) {
  TFB_REQUIRE(K >= 1 && N >= 1 && K < (1LL << 30) && N < (1LL << 30), "%s: bad shape", what);
  TFB_REQUIRE(group == 32 || group == 64 || group == 128, "%s: groups of %d: expected 32, 64 or 128", what, group);
  return TFB_OK;
}
int64_t int4_groups(int64_t K, int group) { return ceil_div(ceil_div(K, kUnit) * kUnit, group); }

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
  TFB_REQUIRE(codes && scales && out && aligned16(codes) && aligned16(scales) && aligned16(out), "int4_expand: the buffers are not 16-byte aligned");
  const int64_t units = ceil_div(K, kUnit), pieces = units * ceil_div(N, 16);
  const int64_t most = (int64_t)sm_count() * 16, blocks = ceil_div(pieces, 8);
  const int log2 = group == 32 ? 5 : group == 64 ? 6 : 7;
  TFB_DISPATCH_16(dtype, T, {
    launch_overlapped(group == 32 ? int4_expand_kernel<T, true> : int4_expand_kernel<T, false>, dim3((unsigned)(blocks < most ? blocks : most)),
                      dim3(256), 0, (cudaStream_t)stream, (const uint4*)codes, (const uint32_t*)scales, (int)units,
                      (int)int4_groups(K, group), log2, pieces, (T*)out);
    return launched("int4_expand");
  })
}

extern "C" int tfb_int4_linear(const void* x, int64_t x_ld, const void* codes, const void* scales, const void* bias, const void* addend,
                               int64_t addend_ld, void* out, int64_t out_ld, int64_t M, int64_t K, int64_t N, int group, int relu,
                               int dtype, void* stream) {
  if (int rc = check_int4("int4_linear", K, N, group)) return rc;
  TFB_REQUIRE(M >= 0 && M <= 64 * 65535, "int4_linear: bad row count");
  if (M == 0) return TFB_OK;
  TFB_REQUIRE(x && codes && scales && out && aligned16(codes) && aligned16(scales), "int4_linear: the weights are not 16-byte aligned");
  TFB_REQUIRE((M == 1 || x_ld >= 0) && out_ld >= N, "int4_linear: row stride smaller than the row");
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
  p.group_log2 = group == 32 ? 5 : group == 64 ? 6 : 7;
  p.strips = (int)ceil_div(N, 16);
  p.x_vec = aligned16(x) && (M == 1 || x_ld % 8 == 0);
  p.relu = relu;
  TFB_DISPATCH_16(dtype, T, { return int4_dispatch<T>(p, (cudaStream_t)stream); })
}
