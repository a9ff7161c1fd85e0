// Whole numbers from -7 to 7 in four bits, as the weights and the caches in 4 bits hold them: how they are made from 16-bit values,
// and how they become 16-bit values again for the tensor cores.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace tfb {

template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first of a chain: nothing to add to.
template <typename T> __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_first<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <> __device__ __forceinline__ void mma_first<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// (v & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t masked_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
  return r;
}

// The eight codes of a word as exact 16-bit numbers: a[i] holds nibbles i and i + 4.  A nibble below the exponent of a power of two
// is that power plus it (1024 in fp16; 128 in bf16, whose seven bits have no room for a nibble four places up); what is added comes
// off again.
template <typename T> __device__ __forceinline__ void expand_nibbles(uint32_t w, uint32_t (&a)[4]);
template <> __device__ __forceinline__ void expand_nibbles<__half>(uint32_t w, uint32_t (&a)[4]) {
  const __half2 off = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f), off16 = __float2half2_rn(-72.f);
#pragma unroll
  for (int i = 0; i < 2; ++i, w >>= 8) {
    const uint32_t lo = masked_or(w, 0x000f000fu, 0x64006400u), hi = masked_or(w, 0x00f000f0u, 0x64006400u);
    const __half2 x = __hadd2(*reinterpret_cast<const __half2*>(&lo), off);
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, off16);
    a[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
    a[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
  }
}
template <> __device__ __forceinline__ void expand_nibbles<__nv_bfloat16>(uint32_t w, uint32_t (&a)[4]) {
  const __nv_bfloat162 off = __float2bfloat162_rn(-136.f);
#pragma unroll
  for (int i = 0; i < 4; ++i, w >>= 4) {
    const uint32_t v = masked_or(w, 0x000f000fu, 0x43004300u);
    const __nv_bfloat162 x = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
    a[i] = *reinterpret_cast<const uint32_t*>(&x);
  }
}

// One of the two 16-bit values of a word.
template <typename T> __device__ __forceinline__ float pair_value(uint32_t w, int which) {
  const uint16_t u = (uint16_t)(which ? w >> 16 : w);
  return Num<T>::to_f(*reinterpret_cast<const T*>(&u));
}

// Scale of a group of 16-bit values whose largest magnitude has the bits `top` (as whole numbers a NaN's are above infinity's), and
// a value's code.  The quotients are rounded as divisions are; neither a scale nor a code then depends on more than the values.
// A seventh of the type's largest values would be rounded up to a scale whose sevenfold is infinite; the one below it is theirs.
template <typename T> constexpr float kLargestScale = std::is_same<T, __half>::value ? 9352.f : 36.25f * 0x1p120f;
template <typename T> __device__ __forceinline__ T scale_of(uint32_t top) {
  const float f = pair_value<T>(top, 0);
  return Num<T>::from_f(isfinite(f) ? fminf(__fdiv_rn(f, 7.f), kLargestScale<T>) : NAN);
}
__device__ __forceinline__ int code_of(float x, float scale) {
  return scale > 0.f ? max(-7, min(7, __float2int_rn(__fdiv_rn(x, scale)))) : 0;
}

// A row of a cache in 4 bits: LANES lanes in a line have 8 neighbouring values each.  Returns a lane's word, dim 2 n + e at bits 4
// n + 16 e; `whole` are its codes.  The same codes and scales as above, without a division (16 sequences of up to 4096 keys, 8
// heads of 128, with what is stored: 179 us with divisions, 84 so).  With values and scales of 11 significant bits, top / 7 is no
// nearer than 2^-15 (relative) to the border between two scales, and a quotient is either half-way between two whole numbers or at
// least 2^-12 away from that: products with reciprocals, 2^-19 off, round to the same, once what is nearer than 2^-14 to a half has
// been made one.
template <typename T, int LANES>
__device__ __forceinline__ uint32_t quantize8(const uint4& v, T& scale, float (&whole)[8]) {
  constexpr float kGrid = 1.5f * (1 << 10), kWhole = 1.5f * (1 << 23);  // adding them rounds to multiples of 2^-13, and of 1
  uint32_t top = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f = pair_value<T>(top, 0);
  scale = Num<T>::from_f(isfinite(f) ? fminf(f * (1.f / 7.f), kLargestScale<T>) : NAN);
  const float s = Num<T>::to_f(scale);
  float x[8];
  unpack8<T>(v, x);
  uint32_t word = 0;
  // a scale that is a subnormal number has fewer bits, and its reciprocal may be none
  if (s >= (std::is_same<T, __half>::value ? 6.2e-5f : 1e-30f)) {
    const float inverse = __fdividef(1.f, s);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const float code = __fadd_rn(__fadd_rn(__fadd_rn(__fmul_rn(x[d], inverse), kGrid), -kGrid), kWhole + 8.f);
      whole[d] = __fadd_rn(code, -kWhole - 8.f);
      const int at = 4 * (d / 2) + 16 * (d % 2);
      word |= (__float_as_uint(code) << at) & (15u << at);
    }
  } else {
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int code = code_of(x[d], s);
      whole[d] = (float)code;
      word |= (uint32_t)(code + 8) << (4 * (d / 2) + 16 * (d % 2));
    }
  }
  return word;
}

}  // namespace tfb
