// What the attention kernels share: vector types, conversions between the
// float types and the 8-bit codes of the K/V cache, and the softmax's moves
// across the lanes of a wave.
#pragma once

#include "common.h"

namespace cowsdm_impl {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kMinusInf = -__builtin_huge_valf();
constexpr float kLeastFloat = -3.402823466e38f;   // the lowest finite number
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kMostCode = 448.0f;         // the largest e4m3 number

// the row widths the cache is laid out for: a head's width is padded with
// zeros to the next one
__host__ __device__ constexpr bool is_cache_width(int64_t w) {
  return w == 32 || w == 64 || w == 96 || w == 128 || w == 192 || w == 256;
}

// x and y exchanged between the halves of the wave, or between its odd and
// even rows of 16 lanes: the largest / the sum over the four lanes that share
// lane % 16.
__device__ __forceinline__ float max_over_rows(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float sum_over_rows(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Of up to 64 numbers below 2^24, lane i's number n, the lane whose number has
// `place` larger ones: the largest first, equal ones by lane.  Lanes from
// `count` on hold none.
__device__ __forceinline__ int lane_by_size(int n, int count, int place) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int key = lane < count ? n * kWave + (kWave - 1 - lane) : -1;
  int rank = 0;
  for (int j = 0; j < count; ++j) rank += __builtin_amdgcn_readlane(key, j) > key ? 1 : 0;
  return __builtin_ctzll(__ballot(lane < count && rank == place));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// eight consecutive elements in float32
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p);
    const f32x4 b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    const vec a = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
  }
}

// eight e4m3 codes times a power of two, in bfloat16: exact (3 bits of
// mantissa, and the scales keep every product a normal number or zero)
__device__ __forceinline__ bf16x8 widen_codes(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x as the sum of N bfloat16 numbers: exact for bfloat16 (N = 1), for float16
// whose 11 bits fit two (N = 2), and to 24 bits for float32 (N = 3)
template <int N>
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&out)[N]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float rest = x[j];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const __bf16 part = static_cast<__bf16>(rest);
      out[n][j] = part;
      if (n + 1 < N) rest -= static_cast<float>(part);
    }
  }
}

// The bfloat16 numbers that carry a query's element, and a probability.  A
// probability takes two at least: one would round it to 8 bits, which shows in
// the output beside its own rounding (an error against 64 bits 20 to 30 %
// larger), and the matrix cores have room for the second product: 64 requests
// of up to 2,560 tokens, 8 key heads, bfloat16: 43.5 us, with one 43.0.
template <typename T>
struct AttentionType;
template <>
struct AttentionType<float> { static constexpr int kParts = 3, kProbParts = 3; };
template <>
struct AttentionType<_Float16> { static constexpr int kParts = 2, kProbParts = 2; };
template <>
struct AttentionType<__bf16> { static constexpr int kParts = 1, kProbParts = 2; };

// four consecutive elements from float32
template <typename T>
__device__ __forceinline__ void store4(T* p, const f32x4 x) {
  typedef T vec __attribute__((ext_vector_type(4)));
  *reinterpret_cast<vec*>(p) = __builtin_convertvector(x, vec);
}

}  // namespace cowsdm_impl
