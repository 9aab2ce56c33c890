// Matrix products with their epilogue: out = residual + activation(x W^T + b).
//
// x [rows, inner] and W [outer, inner] both hold the summed axis last, which
// is the order in which the matrix instructions take either operand: rows of
// both are read 16 bytes at a time and nothing is transposed.  Products are
// computed as W x^T, so that a lane ends with consecutive elements of one
// output row.  Sums, bias, activation and residual are in 32 bits, rounded
// once.

#include <type_traits>

#include "attention.h"

namespace cowsdm_impl {

struct LinearParams {
  const void* x;
  const void* weight;
  const void* bias;
  const void* residual;
  void* out;
  int64_t x_row, weight_row, residual_row;   // strides, in elements
  int32_t rows;
  int32_t inner;
  int32_t outer;
  int32_t activation;
  int32_t wide;                    // epilogue rows move four elements at a time
};

// ------------------------------------------------------- matrix instructions

// 16 bytes of a row of either operand: eight 16-bit numbers or four float32
// ones.  A float32 product takes one of the four at a time, which sums the
// same numbers in another order.
template <typename T>
struct Product {
  typedef typename std::conditional<std::is_same<T, __bf16>::value, bf16x8, f16x8>::type vec;
  static __device__ __forceinline__ f32x16 wide(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (std::is_same<T, __bf16>::value)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vec, a),
                                                     __builtin_bit_cast(vec, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vec, a),
                                                    __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 narrow(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (std::is_same<T, __bf16>::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a),
                                                     __builtin_bit_cast(vec, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a),
                                                    __builtin_bit_cast(vec, b), c, 0, 0, 0);
  }
};

template <>
struct Product<float> {
  static __device__ __forceinline__ f32x16 wide(u32x4 a, u32x4 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0,
                                               0, 0);
    return c;
  }
  static __device__ __forceinline__ f32x4 narrow(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0,
                                               0, 0);
    return c;
  }
};

// --------------------------------------------------------------- epilogue

constexpr float kSqrtHalf = 0.70710678118654752f;

// y Phi(y) for results of 16 bits: max(y, 0) - |y| erfc(|y| / sqrt 2) / 2 with
// the rational approximation 7.1.26 of Abramowitz and Stegun, whose error is
// at most 1.5e-7.  About a third of erff's instructions.
__device__ __forceinline__ float gelu_short(float y) {
  const float a = __builtin_fabsf(y);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.3275911f * kSqrtHalf, 1.0f));
  float s = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  s = __builtin_fmaf(s, t, 1.421413741f);
  s = __builtin_fmaf(s, t, -0.284496736f);
  s = __builtin_fmaf(s, t, 0.254829592f);
  const float e = exp2_fast(y * y * (-0.5f * kLog2E));
  const float h = a < 14.0f ? 0.5f * a * s * t * e : 0.0f;    // 14: below the smallest number
  return (y < 0.0f ? 0.0f : y) - h;
}

// y / (1 + exp(-z))
__device__ __forceinline__ float times_logistic(float y, float z) {
  return y * __builtin_amdgcn_rcpf(1.0f + exp2_fast(-kLog2E * z));
}

template <typename T>
__device__ __forceinline__ f32x4 activated(f32x4 y, int activation) {
  switch (activation) {
    case COWSDM_RELU:
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = y[i] < 0.0f ? 0.0f : y[i];
      break;
    case COWSDM_GELU:
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) y[i] = 0.5f * y[i] * (1.0f + erff(y[i] * kSqrtHalf));
        else y[i] = gelu_short(y[i]);
      }
      break;
    case COWSDM_GELU_TANH:
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = times_logistic(
            y[i], 1.5957691216057308f * (y[i] + 0.044715f * y[i] * y[i] * y[i]));
      break;
    case COWSDM_SILU:
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = times_logistic(y[i], y[i]);
      break;
    default: break;
  }
  return y;
}

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p) {
  typedef T vec __attribute__((ext_vector_type(4)));
  return __builtin_convertvector(*reinterpret_cast<const vec*>(p), f32x4);
}

// Four consecutive elements of an output row, from column n on.
template <typename T>
__device__ __forceinline__ void finish4(const LinearParams& p, int m, int n, f32x4 y) {
  if (m >= p.rows || n >= p.outer) return;
  const T* const bias = static_cast<const T*>(p.bias);
  const T* const residual =
      p.residual ? static_cast<const T*>(p.residual) + m * p.residual_row + n : nullptr;
  T* const out = static_cast<T*>(p.out) + static_cast<int64_t>(m) * p.outer + n;
  if (p.wide) {                    // the outer width is a multiple of four
    if (p.bias) y += load4(bias + n);
    y = activated<T>(y, p.activation);
    if (residual) y = load4(residual) + y;
    store4(out, y);
  } else {
    const int left = p.outer - n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p.bias && i < left) y[i] += static_cast<float>(bias[n + i]);
    y = activated<T>(y, p.activation);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left)
        out[i] = static_cast<T>(residual ? static_cast<float>(residual[i]) + y[i] : y[i]);
  }
}

// -------------------------------------------------------------- many rows

constexpr int kLineBytes = 128;              // of an operand's row in a step
constexpr int kLineChunks = kLineBytes / 16;
constexpr uint32_t kNowhere = 0x80000000u;   // an offset past every buffer: reads 0

// The chunk that place `slot` of a row in LDS holds: the 16 rows that a group
// of lanes reads at once fall on different banks.
__device__ __forceinline__ int line_chunk(int row, int slot) { return slot ^ ((row >> 1) & 7); }

// This thread's chunks of R rows from `first` on, columns from k on; zeros
// past the operand's rows and columns.
template <typename T, int R, int kThreads, bool kAligned>
__device__ __forceinline__ void stage(const T* first, int rows, int64_t stride, int inner, int k,
                                      lds_char* to) {
  constexpr int kEach = 16 / static_cast<int>(sizeof(T));
  const int tid = static_cast<int>(threadIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
#pragma unroll
  for (int i = 0; i < R * kLineChunks / kThreads; ++i) {
    const int q = i * kThreads + tid, row = q / kLineChunks;
    const int column = k + line_chunk(row, q % kLineChunks) * kEach;
    if constexpr (kAligned) {
      const int bytes = static_cast<int>(((rows - 1) * stride + inner) * sizeof(T));
      const uint32_t from =
          column < inner ? static_cast<uint32_t>((row * stride + column) * sizeof(T)) : kNowhere;
      load_to_lds(first, bytes, from, to + (i * kThreads + wave * kWave) * 16);
    } else {
      T v[kEach];
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        v[j] = row < rows && column + j < inner ? first[row * stride + column + j]
                                                : static_cast<T>(0.0f);
      *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(to + q * 16) =
          __builtin_bit_cast(u32x4, v);
    }
  }
}

__device__ __forceinline__ u32x4 line_read(const lds_char* lines, int row, int chunk) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
      lines + row * kLineBytes + line_chunk(row, chunk) * 16);
}

// One workgroup: BM rows of x by BN rows of W; its waves share them as MW by
// NW.  The next step's lines are on their way to LDS while this one's are
// used.
template <typename T, int BM, int BN, int MW, int NW, bool kAligned>
__global__ __launch_bounds__(MW * NW * kWave) void linear_tile_kernel(LinearParams p) {
  constexpr int kThreads = MW * NW * kWave;
  constexpr int MT = BM / MW / 32, NT = BN / NW / 32;     // a wave's tiles of 32 by 32
  constexpr int kEach = kLineBytes / static_cast<int>(sizeof(T));   // columns a step
  extern __shared__ __align__(16) char s_lines[];
  lds_char* const lines = (lds_char*)s_lines;
  constexpr int kBuffer = (BM + BN) * kLineBytes;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int tiles_m = (p.rows + BM - 1) / BM;
  const int tile_n = static_cast<int>(blockIdx.x) / tiles_m;
  const int tile_m = static_cast<int>(blockIdx.x) - tile_n * tiles_m;
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  const T* const x = static_cast<const T*>(p.x) + m0 * p.x_row;
  const T* const w = static_cast<const T*>(p.weight) + n0 * p.weight_row;
  const int x_rows = p.rows - m0 < BM ? p.rows - m0 : BM;
  const int w_rows = p.outer - n0 < BN ? p.outer - n0 : BN;
  const int wm = wave % MW * (BM / MW), wn = wave / MW * (BN / NW);
  f32x16 acc[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
  auto load = [&](int k, int buffer) {
    lds_char* const to = lines + buffer * kBuffer;
    stage<T, BM, kThreads, kAligned>(x, x_rows, p.x_row, p.inner, k, to);
    stage<T, BN, kThreads, kAligned>(w, w_rows, p.weight_row, p.inner, k, to + BM * kLineBytes);
  };
  load(0, 0);
  const int row = lane & 31, half = lane >> 5;
  for (int k = 0, buffer = 0; k < p.inner; k += kEach, buffer ^= 1) {
    __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0): this thread's part has arrived
    __syncthreads();
    if (k + kEach < p.inner) load(k + kEach, buffer ^ 1);
    const lds_char* const xs = lines + buffer * kBuffer;
    const lds_char* const ws = xs + BM * kLineBytes;
#pragma unroll
    for (int s = 0; s < kLineChunks / 2; ++s) {
      u32x4 a[NT], b[MT];
#pragma unroll
      for (int t = 0; t < NT; ++t) a[t] = line_read(ws, wn + t * 32 + row, 2 * s + half);
#pragma unroll
      for (int t = 0; t < MT; ++t) b[t] = line_read(xs, wm + t * 32 + row, 2 * s + half);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = Product<T>::wide(a[t], b[u], acc[t][u]);
    }
  }
  // Through LDS, 32 output rows of this wave at a time, so that a store writes
  // whole rows of its columns; chunks of four are permuted against the banks.
  constexpr int kChunks = NT * 8;
  __syncthreads();
  f32x4* const turned = reinterpret_cast<f32x4*>(s_lines) + wave * 32 * kChunks;
#pragma unroll
  for (int u = 0; u < MT; ++u) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        turned[row * kChunks + ((t * 8 + g * 2 + half) ^ (row & (kChunks - 1)))] =
            f32x4{acc[t][u][4 * g], acc[t][u][4 * g + 1], acc[t][u][4 * g + 2],
                  acc[t][u][4 * g + 3]};
#pragma unroll 2
    for (int r = lane / kChunks; r < 32; r += kWave / kChunks) {
      const int c = lane % kChunks;
      finish4<T>(p, m0 + wm + u * 32 + r, n0 + wn + c * 4,
                 turned[r * kChunks + (c ^ (r & (kChunks - 1)))]);
    }
  }
}

// --------------------------------------------------------------- few rows

typedef __amdgpu_buffer_rsrc_t buffer_t;

__device__ __forceinline__ u32x4 load_chunk(const void* first, int bytes, uint32_t from) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(
      u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                 __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(first), 0, bytes, 0x00020000),
                 from, 0, 0));
#else
  return u32x4{};
#endif
}

// One workgroup: 16 NT rows of W over all of the summed axis, which its waves
// share, by 16 MT rows of x.  Every weight is read once, from memory into
// registers; the waves' sums meet in LDS.
template <typename T, int NT, int MT, int kWaves>
__global__ __launch_bounds__(kWaves * kWave) void linear_few_kernel(LinearParams p) {
  constexpr int kEach = 16 / static_cast<int>(sizeof(T));   // columns a lane
  constexpr int kStep = 4 * kEach;                          // columns a step
  constexpr int kAhead = 4;                                 // steps whose loads go out together
  __shared__ f32x4 s_sums[kWaves][NT * MT][kWave];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int n0 = static_cast<int>(blockIdx.x) * 16 * NT;
  const int m0 = static_cast<int>(blockIdx.y) * 16 * MT;
  const T* const x = static_cast<const T*>(p.x) + m0 * p.x_row;
  const T* const w = static_cast<const T*>(p.weight) + n0 * p.weight_row;
  const int x_rows = p.rows - m0 < 16 * MT ? p.rows - m0 : 16 * MT;
  const int w_rows = p.outer - n0 < 16 * NT ? p.outer - n0 : 16 * NT;
  const int x_bytes = static_cast<int>(((x_rows - 1) * p.x_row + p.inner) * sizeof(T));
  const int w_bytes = static_cast<int>(((w_rows - 1) * p.weight_row + p.inner) * sizeof(T));
  const int row = lane & 15, quarter = lane >> 4;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int a = 0; a < NT; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b) acc[a][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = wave * kAhead * kStep; k < p.inner; k += kWaves * kAhead * kStep) {
    u32x4 a[kAhead][NT], b[kAhead][MT];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int column = k + s * kStep + quarter * kEach;
      const bool in = column < p.inner;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t at = (t * 16 + row) * p.weight_row + column;
        a[s][t] = load_chunk(w, w_bytes, in ? static_cast<uint32_t>(at * sizeof(T)) : kNowhere);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int64_t at = (t * 16 + row) * p.x_row + column;
        b[s][t] = load_chunk(x, x_bytes, in ? static_cast<uint32_t>(at * sizeof(T)) : kNowhere);
      }
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = Product<T>::narrow(a[s][t], b[s][u], acc[t][u]);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) s_sums[wave][t * MT + u][lane] = acc[t][u];
  __syncthreads();
  for (int j = wave; j < NT * MT; j += kWaves) {
    f32x4 y = s_sums[0][j][lane];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) y += s_sums[v][j][lane];
    const int t = j / MT, u = j - t * MT;
    finish4<T>(p, m0 + u * 16 + row, n0 + t * 16 + quarter * 4, y);
  }
}

// ----------------------------------------------------------------- launch

template <typename T, int BM, int BN, int MW, int NW, bool kAligned>
int32_t launch_tiles(const LinearParams& p, hipStream_t s) {
  const int64_t groups = static_cast<int64_t>((p.rows + BM - 1) / BM) * ((p.outer + BN - 1) / BN);
  constexpr int kThreads = MW * NW * kWave;
  if (groups > UINT32_MAX / kThreads) return fail(COWSDM_ELIMIT, "linear: output too large");
  constexpr int kBytes = 2 * (BM + BN) * kLineBytes;
  auto* const kernel = linear_tile_kernel<T, BM, BN, MW, NW, kAligned>;
  if constexpr (kBytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != hipSuccess)
      return fail(static_cast<int32_t>(e), "linear: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), kBytes, s, p);
  return launch_status("linear");
}

template <typename T, int NT, int MT, int kWaves>
int32_t launch_few(const LinearParams& p, hipStream_t s) {
  hipLaunchKernelGGL((linear_few_kernel<T, NT, MT, kWaves>),
                     dim3((p.outer + 16 * NT - 1) / (16 * NT), (p.rows + 16 * MT - 1) / (16 * MT)),
                     dim3(kWaves * kWave), 0, s, p);
  return launch_status("linear");
}

template <typename T>
int32_t launch_linear(const LinearParams& p, bool aligned, hipStream_t s) {
  if (!aligned) return launch_tiles<T, 64, 64, 2, 2, false>(p, s);
  if (p.rows <= 16) return launch_few<T, 1, 1, 8>(p, s);
  if (p.rows <= 32) return launch_few<T, 2, 2, 8>(p, s);
  if (p.rows <= 64) return launch_few<T, 2, 4, 8>(p, s);
  const int64_t large = static_cast<int64_t>((p.rows + 255) / 256) * ((p.outer + 255) / 256);
  if (sizeof(T) == 2 && large >= 256) return launch_tiles<T, 256, 256, 2, 4, true>(p, s);
  return launch_tiles<T, 128, 128, 2, 2, true>(p, s);
}

}  // namespace cowsdm_impl

using namespace cowsdm_impl;

extern "C" int32_t cowsdm_linear(const cowsdm_linear_t* linear, void* stream) {
  if (!linear) return fail(COWSDM_EARG, "linear: null argument");
  const cowsdm_linear_t& l = *linear;
  if (l.rows < 0 || l.inner < 0 || l.outer < 0) return fail(COWSDM_EARG, "linear: negative size");
  if (l.float_type != COWSDM_FLOAT32 && l.float_type != COWSDM_FLOAT16 &&
      l.float_type != COWSDM_BFLOAT16)
    return fail(COWSDM_EARG, "linear: bad float type");
  if (l.activation < COWSDM_NO_ACTIVATION || l.activation > COWSDM_SILU)
    return fail(COWSDM_EARG, "linear: bad activation");
  if (l.x_row < 0 || l.weight_row < 0 || l.residual_row < 0)
    return fail(COWSDM_EARG, "linear: negative stride");
  // a workgroup's rows of an operand lie within 2^31 bytes
  if (l.inner > COWSDM_LINEAR_MOST || l.x_row > COWSDM_LINEAR_MOST ||
      l.weight_row > COWSDM_LINEAR_MOST)
    return fail(COWSDM_ELIMIT, "linear: rows of more than 2^20 elements");
  if (l.rows > INT32_MAX - 256 || l.outer > INT32_MAX - 256)
    return fail(COWSDM_ELIMIT, "linear: too large");
  if (l.rows == 0 || l.outer == 0) return 0;
  if (!l.out || (l.inner > 0 && (!l.x || !l.weight)))
    return fail(COWSDM_EARG, "linear: null pointer argument");
  const int64_t unit = l.float_type == COWSDM_FLOAT32 ? 4 : 8;
  const int64_t size = 16 / unit;
  auto address = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const bool aligned = (address(l.x) | address(l.weight)) % 16 == 0 && l.inner % unit == 0 &&
                       l.x_row % unit == 0 && l.weight_row % unit == 0;
  const bool wide = l.outer % 4 == 0 && l.residual_row % 4 == 0 &&
                    (address(l.out) | address(l.bias) | address(l.residual)) % (4 * size) == 0;
  LinearParams p{l.x, l.weight, l.bias, l.residual, l.out, l.x_row, l.weight_row,
                 l.residual_row, static_cast<int32_t>(l.rows), static_cast<int32_t>(l.inner),
                 static_cast<int32_t>(l.outer), l.activation, wide};
  const auto s = static_cast<hipStream_t>(stream);
  if (l.float_type == COWSDM_FLOAT32) return launch_linear<float>(p, aligned, s);
  if (l.float_type == COWSDM_FLOAT16) return launch_linear<_Float16>(p, aligned, s);
  return launch_linear<__bf16>(p, aligned, s);
}
