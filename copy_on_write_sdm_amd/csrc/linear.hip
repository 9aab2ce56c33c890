// Matrix products with their epilogue: out = residual + activation(x W^T + b).
//
// x [rows, inner] and W [outer, inner] both hold the summed axis last, which
// is the order in which the matrix instructions take either operand: rows of
// both are read 16 bytes at a time and nothing is transposed.  Products are
// computed as W x^T, so that a lane ends with consecutive elements of one
// output row.  Sums, bias, activation and residual are in 32 bits, rounded
// once.  Float32 numbers go through the matrix cores as three of bfloat16.

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
  int32_t splits;                  // of the summed axis; more than one: sums go to `parts`
  int32_t chunk;                   // columns of a split
  float* parts;                    // [splits][rows][outer rounded up to four]
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

// y Phi(y) for results of 16 bits: Phi(-|y|) = erfc(|y| / sqrt 2) / 2 by the
// rational approximation 7.1.26 of Abramowitz and Stegun, whose error is at
// most 1.5e-7.  About a third of erff's instructions.
__device__ __forceinline__ float gelu_short(float y) {
  const float t =
      __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_fabsf(y), 0.3275911f * kSqrtHalf, 1.0f));
  float s = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  s = __builtin_fmaf(s, t, 0.5f * 1.421413741f);
  s = __builtin_fmaf(s, t, 0.5f * -0.284496736f);
  s = __builtin_fmaf(s, t, 0.5f * 0.254829592f);
  const float below = s * t * exp2_fast(y * y * (-0.5f * kLog2E));
  return y * (y > 0.0f ? 1.0f - below : below);
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

// Four elements at any address.
template <typename T>
struct Four {
  typedef T vec __attribute__((ext_vector_type(4)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
};

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p) {
  const typename Four<T>::vec v = *reinterpret_cast<const typename Four<T>::loose*>(p);
  return __builtin_convertvector(v, f32x4);
}

template <typename T>
__device__ __forceinline__ void put4(T* p, f32x4 y) {
  *reinterpret_cast<typename Four<T>::loose*>(p) =
      __builtin_convertvector(y, typename Four<T>::vec);
}

// Columns n to n + 3 of output row m, as far as there are any: nothing past
// the last row and column.
template <typename T>
__device__ __forceinline__ void finish4(const LinearParams& p, int m, int n, f32x4 y) {
  if (m >= p.rows || n >= p.outer) return;
  const T* const bias = static_cast<const T*>(p.bias) + n;
  const T* const residual = static_cast<const T*>(p.residual) + m * p.residual_row + n;
  T* const out = static_cast<T*>(p.out) + static_cast<int64_t>(m) * p.outer + n;
  const int left = p.outer - n;
  if (left >= 4) {
    if (p.bias) y += load4(bias);
    y = activated<T>(y, p.activation);
    if (p.residual) y = load4(residual) + y;
    put4(out, y);
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (p.bias && i < left) y[i] += static_cast<float>(bias[i]);
  y = activated<T>(y, p.activation);
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < left)
      out[i] = static_cast<T>(p.residual ? static_cast<float>(residual[i]) + y[i] : y[i]);
}

// A wave's sums of 32 NT columns by 32 MT rows of the output, as the products
// leave them, through LDS (32 rows of its own at a time, which `put` writes in
// chunks of four columns), so that a store writes whole rows of its columns;
// what other lanes have written is read, and written over, behind a fence of the
// wave.  Chunks are permuted against the banks.  A lane keeps to four columns, whose
// bias it loads once, at whatever address they lie: 1,671 rows by 288 x 11706 in
// bfloat16 take 42 us, and 64 with a column a lane.
template <typename T, int NT, int MT, typename Put>
__device__ __forceinline__ void finish_rows(const LinearParams& p, Put put, f32x4* turned, int m0,
                                            int n0, int split) {
  constexpr int kChunks = NT * 8, kRows = kWave / kChunks;      // rows of a step
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int c = lane % kChunks, n = n0 + c * 4;
  const bool in = n < p.outer, whole = n + 4 <= p.outer;
  f32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.bias && p.splits == 1 && whole) bias = load4(static_cast<const T*>(p.bias) + n);
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    put(u, [&](int r, int chunk) -> f32x4& {
      return turned[r * kChunks + (chunk ^ (r & (kChunks - 1)))];
    });
    wave_lds_sync();
    const int first = m0 + u * 32;
    auto at = [&](int r) { return turned[r * kChunks + (c ^ (r & (kChunks - 1)))]; };
    if (p.splits > 1) {
      const int64_t wide = (p.outer + 3) & ~3;
      float* const to = p.parts + (static_cast<int64_t>(split) * p.rows) * wide + n;
#pragma unroll 4
      for (int r = lane / kChunks; r < 32; r += kRows)
        if (in && first + r < p.rows) *reinterpret_cast<f32x4*>(to + (first + r) * wide) = at(r);
    } else if (!whole) {
      // the last columns, of fewer than four
#pragma unroll 1
      for (int r = lane / kChunks; r < 32; r += kRows) finish4<T>(p, first + r, n, at(r));
    } else if (p.residual) {
      const T* const residual = static_cast<const T*>(p.residual) + n;
#pragma unroll 4
      for (int r = lane / kChunks; r < 32; r += kRows) {
        const int m = first + r;
        if (m >= p.rows) continue;
        const f32x4 more = load4(residual + m * p.residual_row);
        const f32x4 y = activated<T>(at(r) + bias, p.activation);
        put4(static_cast<T*>(p.out) + static_cast<int64_t>(m) * p.outer + n, more + y);
      }
    } else {
#pragma unroll 4
      for (int r = lane / kChunks; r < 32; r += kRows) {
        const int m = first + r;
        const f32x4 y = activated<T>(at(r) + bias, p.activation);
        if (m < p.rows) put4(static_cast<T*>(p.out) + static_cast<int64_t>(m) * p.outer + n, y);
      }
    }
    wave_lds_sync();
  }
}

// The same of sums that lie as products of 32 by 32 leave them.
template <typename T, int NT, int MT>
__device__ __forceinline__ void finish_tile(const LinearParams& p, const f32x16 (&acc)[NT][MT],
                                            f32x4* turned, int m0, int n0, int split) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int row = lane & 31, half = lane >> 5;
  auto put = [&](int u, auto place) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        place(row, t * 8 + g * 2 + half) = f32x4{acc[t][u][4 * g], acc[t][u][4 * g + 1],
                                                 acc[t][u][4 * g + 2], acc[t][u][4 * g + 3]};
  };
  finish_rows<T, NT, MT>(p, put, turned, m0, n0, split);
}

// The splits' sums, added in their order, and the epilogue: a launch and one
// round trip, 3 us after a product of 64 rows by 6144 columns in two splits.
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearParams p) {
  const int wide = (p.outer + 3) & ~3, chunks = wide / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t each = static_cast<int64_t>(p.rows) * wide;
  if (at * 4 >= each) return;
  const int m = static_cast<int>(at / chunks);
  const int n = static_cast<int>(at - m * static_cast<int64_t>(chunks)) * 4;
  const f32x4* const from = reinterpret_cast<const f32x4*>(p.parts) + at;
  f32x4 y = from[0];
#pragma unroll 4
  for (int s = 1; s < p.splits; ++s) y += from[s * (each / 4)];
  finish4<T>(p, m, n, y);
}

// -------------------------------------------------------------- many rows

constexpr int kLineBytes = 128;              // of an operand's row in a step
constexpr int kLineChunks = kLineBytes / 16;
constexpr uint32_t kNowhere = 0x80000000u;   // an offset past every buffer: reads 0

// The chunk that place `slot` of a row in LDS holds: the 16 rows that a group
// of lanes reads at once fall on different banks.
__device__ __forceinline__ int line_chunk(int row, int slot) { return slot ^ ((row >> 1) & 7); }

__device__ __forceinline__ u32x4 line_read(const lds_char* lines, int row, int chunk) {
  return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(
      lines + row * kLineBytes + line_chunk(row, chunk) * 16);
}

// R rows of an operand on their way to LDS, kThreads chunks at a time: where
// this thread's lie.  A thread's chunks are in one place of their rows, as
// kThreads is a multiple of 16 rows.
template <typename T, int R, int kThreads>
struct Lines {
  static constexpr int kLoads = R * kLineChunks / kThreads;
  static_assert(kThreads % (16 * kLineChunks) == 0 && R * kLineChunks % kThreads == 0);
  const T* first;
  int bytes;
  uint32_t from[kLoads];

  __device__ __forceinline__ Lines(const void* base, int64_t stride, int at, int rows, int inner) {
    const int left = rows - at < R ? rows - at : R;
    first = static_cast<const T*>(base) + at * stride;
    bytes = static_cast<int>(((left - 1) * stride + inner) * static_cast<int64_t>(sizeof(T)));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = i * kThreads + static_cast<int>(threadIdx.x), row = q / kLineChunks;
      from[i] = static_cast<uint32_t>(row * stride * static_cast<int64_t>(sizeof(T))) +
                line_chunk(row, q % kLineChunks) * 16;
    }
  }
  // The first column of this thread's chunks in a step.
  static __device__ __forceinline__ int column() {
    const int q = static_cast<int>(threadIdx.x);
    return line_chunk(q / kLineChunks, q % kLineChunks) * (16 / static_cast<int>(sizeof(T)));
  }
  // Loads i to e - 1 of the step from column k on; zeros from column `end` on.
  __device__ __forceinline__ void load(lds_char* to, int k, int end, int i = 0,
                                       int e = kLoads) const {
    const int wave =
        __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const uint32_t at =
        k + column() < end ? static_cast<uint32_t>(k * static_cast<int>(sizeof(T))) : kNowhere;
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      if (n >= i && n < e)
        load_to_lds(first, bytes, from[n] + at, to + (n * kThreads + wave * kWave) * 16);
  }
};

// Waits until at most `kLeft` of this wave's loads are out and its LDS reads
// are in, and then for the workgroup's other waves.  (The builtin barrier
// alone would let the compiler move memory accesses over it, and
// __syncthreads waits for every load.)
template <int kLeft>
__device__ __forceinline__ void arrive() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070 | (kLeft & 15) | ((kLeft >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// A wave's operands of one product step, and the products.
template <typename T, int NT, int MT>
struct Operands {
  u32x4 a[NT], b[MT];
  __device__ __forceinline__ void read(const lds_char* ws, const lds_char* xs, int wn, int wm,
                                       int s) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int row = lane & 31, half = lane >> 5;
#pragma unroll
    for (int t = 0; t < NT; ++t) a[t] = line_read(ws, wn + t * 32 + row, 2 * s + half);
#pragma unroll
    for (int t = 0; t < MT; ++t) b[t] = line_read(xs, wm + t * 32 + row, 2 * s + half);
  }
  __device__ __forceinline__ void multiply(f32x16 (&acc)[NT][MT]) const {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[t][u] = Product<T>::wide(a[t], b[u], acc[t][u]);
  }
};

// The same of float32: half a line's numbers, eight a lane of each row.
template <int NT, int MT>
struct FloatOperands {
  u32x4 a[NT][2], b[MT][2];
  __device__ __forceinline__ void read(const lds_char* ws, const lds_char* xs, int wn, int wm,
                                       int j) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int row = lane & 31, half = lane >> 5;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        a[t][c] = line_read(ws, wn + t * 32 + row, 4 * j + 2 * c + half);
#pragma unroll
      for (int t = 0; t < MT; ++t)
        b[t][c] = line_read(xs, wm + t * 32 + row, 4 * j + 2 * c + half);
    }
  }
  // By float32 products.
  __device__ __forceinline__ void multiply(f32x16 (&acc)[NT][MT]) const {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u)
          acc[t][u] = Product<float>::wide(a[t][c], b[u][c], acc[t][u]);
  }
};

// A float32 number as the sum of three of bfloat16, whose products the matrix
// cores do at sixteen times float32's rate.  Of the nine products of two
// numbers the six that count are taken, smallest first; what is left out is
// within 2^-23 of the product (a third is within 2^-8 of the one before).  A
// number that is not finite, or within 2^-9 of the largest, gives NaN this
// way: such sums are done again by float32 products.  4,000 rows by 4000 x
// 4000, tiles of 256: 579 us, and 911 by float32 products; 2,048 by 2048 x
// 2048, tiles of 128: 96 and 135.
//
// Pairs are rounded together, and a third is taken off as it stands in the
// upper half of a word.
__device__ __forceinline__ void to_thirds(const u32x4 (&v)[2], u32x4 (&out)[3]) {
  typedef float pair __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    pair rest = {__uint_as_float(v[i / 2][i % 2 * 2]), __uint_as_float(v[i / 2][i % 2 * 2 + 1])};
#pragma unroll
    for (int n = 0; n < 3; ++n) {
      const uint32_t part = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, bf16x2));
      out[n][i] = part;
      if (n < 2) {
        rest[0] -= __uint_as_float(part << 16);
        rest[1] -= __uint_as_float(part & 0xffff0000u);
      }
    }
  }
}

// The products that count: which thirds of the left and of the right.
constexpr int kThirds = 6;
constexpr int kOfLeft[kThirds] = {2, 0, 1, 1, 0, 0}, kOfRight[kThirds] = {0, 2, 1, 0, 1, 0};

template <int NT, int MT>
struct Thirds {
  u32x4 a[NT][3], b[MT][3];
  __device__ __forceinline__ void take(const FloatOperands<NT, MT>& raw) {
#pragma unroll
    for (int t = 0; t < NT; ++t) to_thirds(raw.a[t], a[t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) to_thirds(raw.b[t], b[t]);
  }
  __device__ __forceinline__ void multiply(f32x16 (&acc)[NT][MT]) const {
#pragma unroll
    for (int i = 0; i < kThirds; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u)
          acc[t][u] = Product<__bf16>::wide(a[t][kOfLeft[i]], b[u][kOfRight[i]], acc[t][u]);
  }
};

// Whether a sum of the workgroup's is not finite; by way of a word of the LDS
// that its lines have left.
template <typename Acc, int NT, int MT>
__device__ __forceinline__ bool any_not_finite(const Acc (&acc)[NT][MT], int* word) {
  float sum = 0.0f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(Acc) / 4); ++i)
        sum = __builtin_fmaf(acc[t][u][i], 0.0f, sum);
  if (threadIdx.x == 0) *word = 0;
  __syncthreads();
  if (sum != 0.0f) *word = 1;
  __syncthreads();
  const bool any = *word != 0;
  __syncthreads();
  return any;
}

template <typename Acc, int NT, int MT>
__device__ __forceinline__ void clear(Acc (&acc)[NT][MT]) {
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(Acc) / 4); ++i) acc[t][u][i] = 0.0f;
}

constexpr int kSteps = kLineChunks / 2;      // product steps of a line

// Workgroup n runs on XCD n % 8, each of which takes a run of tiles, some rows
// of tiles at a time, so that what an XCD works on at once shares its L2.  Rows
// of 256 at a time (by products of 32 by 32): 7,919 x 4,096 by 16,384 takes 862
// us with 1, 813 with 3, 816 with 4, 842 with 8.  Smaller tiles, 4 against 8:
// 1,024 x 4,096 by 4,096 in 128 x 128 39.4 against 38.9 us, 1,111 x 2,304 by 1,544
// in 64 x 128 17.8 against 17.5, in 64 x 64 17.4 against 16.8.
template <int BM, int BN>
__device__ __forceinline__ void tile_place(const LinearParams& p, int groups, int& m0, int& n0) {
  constexpr int kBand = BM == 256 ? 4 : 8;
  const int tiles_m = (p.rows + BM - 1) / BM, tiles_n = (p.outer + BN - 1) / BN;
  const int side = static_cast<int>(blockIdx.x) % 8, each = groups / 8, rest = groups % 8;
  const int tile = side * each + (side < rest ? side : rest) + static_cast<int>(blockIdx.x) / 8;
  const int band = tile / (kBand * tiles_n), in = tile - band * kBand * tiles_n;
  const int left = tiles_m - band * kBand, high = left < kBand ? left : kBand;
  const int column = in / high;
  m0 = (band * kBand + in - column * high) * BM;
  n0 = column * BN;
}

// One workgroup: 256 rows of x by 256 rows of W, its eight waves 128 by 64
// each.  LDS holds five half tiles (a step's lines of x, or of W): two are
// used, one and a half steps' are on their way.  When a step's lines have all
// been read, W of two steps on takes the place of its x, and x of three steps
// on that of its W.  (With two whole steps in LDS, each waited for as a whole,
// the first case below took a quarter longer; with steps of 64 bytes, or four
// waves of 128 by 128, a sixth.)
//
// Half of a wave's rows of x are multiplied while the other half's next ones
// are read.  The matrix cores bound it, at the clock that the power leaves:
// 7,919 rows by 4096 x 16384 in bfloat16 take 772 us, 1,380 TFLOP/s, with the
// matrix cores busy 64 % of the cycles at 1.9 GHz.  Products of 32 by 32 by 16,
// which do as much a cycle, took 843: 67 % at 1.7 GHz.  GELU in the epilogue adds
// some 40: it fills the vector units, and no other workgroup is on the CU
// meanwhile.
template <typename T>
__global__ __launch_bounds__(512) void linear_large_kernel(LinearParams p) {
  constexpr int B = 256, kThreads = 512, MT = 8, NT = 4, kHalf = MT / 2;
  constexpr int kEach = kLineBytes / static_cast<int>(sizeof(T));   // columns a step
  constexpr int kSlot = B * kLineBytes, kSlots = 5;
  constexpr int kLoads = Lines<T, B, kThreads>::kLoads;
  extern __shared__ __align__(16) char s_lines[];
  lds_char* const lines = (lds_char*)s_lines;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  int m0, n0;
  tile_place<B, B>(p, gridDim.x, m0, n0);
  const int begin = static_cast<int>(blockIdx.y) * p.chunk;
  const int end = p.inner - begin < p.chunk ? p.inner : begin + p.chunk;
  const Lines<T, B, kThreads> x(p.x, p.x_row, m0, p.rows, p.inner);
  const Lines<T, B, kThreads> w(p.weight, p.weight_row, n0, p.outer, p.inner);
  const int wm = wave % 2 * 128, wn = wave / 2 * 64;
  const int row = lane & 15, quarter = lane >> 4;
  f32x4 acc[NT][MT];
  clear(acc);
  u32x4 a[2][NT], b[MT];
  // a wave's rows of W, and half of its rows of x, half a line each
  auto read_w = [&](u32x4 (&to)[NT], int slot, int s) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
      to[t] = line_read(lines + slot * kSlot, wn + t * 16 + row, 4 * s + quarter);
  };
  auto read_x = [&](int half, int slot, int s) {
#pragma unroll
    for (int u = half * kHalf; u < half * kHalf + kHalf; ++u)
      b[u] = line_read(lines + slot * kSlot, wm + u * 16 + row, 4 * s + quarter);
  };
  auto multiply = [&](const u32x4 (&v)[NT], int half) {
#pragma unroll
    for (int u = half * kHalf; u < half * kHalf + kHalf; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][u] = Product<T>::narrow(v[t], b[u], acc[t][u]);
  };
  auto further = [&](int slot) { return slot + 2 < kSlots ? slot + 2 : slot + 2 - kSlots; };
  x.load(lines, begin, end);
  w.load(lines + kSlot, begin, end);
  x.load(lines + 2 * kSlot, begin + kEach, end);
  w.load(lines + 3 * kSlot, begin + kEach, end);
  arrive<2 * kLoads>();
  int xs = 0, ws = 1, spare = 4;           // slots of this step's x and W, and of the last one's W
  read_w(a[0], ws, 0);
  read_x(0, xs, 0);
  read_x(1, xs, 0);
  for (int k = begin; k < end; k += kEach) {
    const int xn = further(xs), wx = further(ws);
    read_w(a[1], ws, 1);
    // not at once with W's, so that those come first
    x.load(lines + spare * kSlot, k + 2 * kEach, end);
    multiply(a[0], 0);
    __builtin_amdgcn_sched_barrier(0);
    read_x(0, xs, 1);
    multiply(a[0], 1);
    __builtin_amdgcn_sched_barrier(0);
    read_x(1, xs, 1);
    multiply(a[1], 0);
    arrive<kLoads>();                      // all but x of two steps on
    read_w(a[0], wx, 0);
    read_x(0, xn, 0);
    w.load(lines + xs * kSlot, k + 2 * kEach, end);
    multiply(a[1], 1);
    __builtin_amdgcn_sched_barrier(0);
    read_x(1, xn, 0);
    spare = ws;
    xs = xn;
    ws = wx;
  }
  arrive<0>();
  auto put = [&](int u, auto place) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int t = 0; t < NT; ++t) place(g * 16 + row, t * 4 + quarter) = acc[t][2 * u + g];
  };
  finish_rows<T, NT / 2, MT / 2>(p, put, reinterpret_cast<f32x4*>(s_lines) + wave * 32 * NT * 4,
                                 m0 + wm, n0 + wn, blockIdx.y);
}

// The same of float32, by thirds: of a line of W's rows at once, and of one row
// of tiles of x's at a time, as registers allow.  Matrix cores and vector units
// (the thirds) bound it: 4,000 rows by 4000 x 4000 take 579 us, 221 TFLOP/s (633
// by products of 32 by 32).
__global__ __launch_bounds__(512) void linear_large_float_kernel(LinearParams p) {
  typedef float T;
  constexpr int B = 256, kThreads = 512, MT = 8, NT = 4;
  constexpr int kEach = kLineBytes / static_cast<int>(sizeof(T));   // columns a step
  constexpr int kSlot = B * kLineBytes, kSlots = 5;
  constexpr int kLoads = Lines<T, B, kThreads>::kLoads;
  extern __shared__ __align__(16) char s_lines[];
  lds_char* const lines = (lds_char*)s_lines;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  int m0, n0;
  tile_place<B, B>(p, gridDim.x, m0, n0);
  const int begin = static_cast<int>(blockIdx.y) * p.chunk;
  const int end = p.inner - begin < p.chunk ? p.inner : begin + p.chunk;
  const Lines<T, B, kThreads> x(p.x, p.x_row, m0, p.rows, p.inner);
  const Lines<T, B, kThreads> w(p.weight, p.weight_row, n0, p.outer, p.inner);
  const int wm = wave % 2 * 128, wn = wave / 2 * 64;
  const int row = lane & 15, quarter = lane >> 4;
  f32x4 acc[NT][MT];
  auto further = [&](int slot) { return slot + 2 < kSlots ? slot + 2 : slot + 2 - kSlots; };
  auto read = [&](u32x4 (&to)[2], int slot, int first) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      to[c] = line_read(lines + slot * kSlot, first + row, 2 * quarter + c);
  };
  auto sums = [&](auto thirds) {
    clear(acc);
    x.load(lines, begin, end);
    w.load(lines + kSlot, begin, end);
    x.load(lines + 2 * kSlot, begin + kEach, end);
    w.load(lines + 3 * kSlot, begin + kEach, end);
    arrive<2 * kLoads>();
    x.load(lines + 4 * kSlot, begin + 2 * kEach, end);
    for (int k = begin, xs = 0, ws = 1; k < end; k += kEach) {
      u32x4 a[NT][2], b[2];
#pragma unroll
      for (int t = 0; t < NT; ++t) read(a[t], ws, wn + t * 16);
      if constexpr (decltype(thirds)::value) {
        u32x4 as[NT][3], bs[3];
#pragma unroll
        for (int t = 0; t < NT; ++t) to_thirds(a[t], as[t]);
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          read(b, xs, wm + u * 16);
          to_thirds(b, bs);
#pragma unroll
          for (int i = 0; i < kThirds; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              acc[t][u] = Product<__bf16>::narrow(as[t][kOfLeft[i]], bs[kOfRight[i]], acc[t][u]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          read(b, xs, wm + u * 16);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              acc[t][u] = Product<float>::narrow(a[t][c], b[c], acc[t][u]);
        }
      }
      arrive<kLoads>();                    // all but x of two steps on
      w.load(lines + xs * kSlot, k + 2 * kEach, end);
      x.load(lines + ws * kSlot, k + 3 * kEach, end);
      xs = further(xs);
      ws = further(ws);
    }
    arrive<0>();
  };
  sums(std::true_type());
  if (any_not_finite(acc, reinterpret_cast<int*>(s_lines))) sums(std::false_type());
  auto put = [&](int u, auto place) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int t = 0; t < NT; ++t) place(g * 16 + row, t * 4 + quarter) = acc[t][2 * u + g];
  };
  finish_rows<T, NT / 2, MT / 2>(p, put, reinterpret_cast<f32x4*>(s_lines) + wave * 32 * NT * 4,
                                 m0 + wm, n0 + wn, blockIdx.y);
}

// One workgroup: BM rows of x by BN rows of W over a split of the summed axis;
// its waves share them as MW by NW.  LDS holds the lines of kStages steps, all
// but one of them on their way.
//
// What a CU takes in from beyond its L2 bounds it where there are few rows, some
// 50 to 60 bytes a nanosecond whatever the stages' number, and else the steps'
// round: 64 rows by 4096 x 6144 in bfloat16, in two splits of 64 x 64, 14.2 us
// with the join; 1,111 rows by 2304 x 1544 in float16, 64 x 128, 18.6 us.
template <typename T, int BM, int BN, int MW, int NW, int kStages>
__global__ __launch_bounds__(MW * NW * kWave) void linear_tile_kernel(LinearParams p) {
  constexpr int kThreads = MW * NW * kWave;
  constexpr int MT = BM / MW / 32, NT = BN / NW / 32;               // a wave's tiles of 32 by 32
  constexpr int kEach = kLineBytes / static_cast<int>(sizeof(T));   // columns a step
  constexpr int kStage = (BM + BN) * kLineBytes;
  constexpr int kLoads = Lines<T, BM, kThreads>::kLoads + Lines<T, BN, kThreads>::kLoads;
  extern __shared__ __align__(16) char s_lines[];
  lds_char* const lines = (lds_char*)s_lines;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  int m0, n0;
  tile_place<BM, BN>(p, gridDim.x, m0, n0);
  const int begin = static_cast<int>(blockIdx.y) * p.chunk;
  const int end = p.inner - begin < p.chunk ? p.inner : begin + p.chunk;
  const Lines<T, BM, kThreads> x(p.x, p.x_row, m0, p.rows, p.inner);
  const Lines<T, BN, kThreads> w(p.weight, p.weight_row, n0, p.outer, p.inner);
  const int wm = wave % MW * (BM / MW), wn = wave / MW * (BN / NW);
  f32x16 acc[NT][MT];
  auto load = [&](int k, int stage) {
    lds_char* const to = lines + stage * kStage;
    x.load(to, k, end);
    w.load(to + BM * kLineBytes, k, end);
  };
  auto start = [&](int stages) {
    clear(acc);
    for (int s = 0; s < stages; ++s) load(begin + s * kEach, s);
  };
  if constexpr (sizeof(T) == 4) {
    // Half a line's products run while the next half's thirds are made of what
    // has been read, and the half after that is read: in one wave, as a CU
    // holds four.
    start(kStages);
    arrive<(kStages - 1) * kLoads>();
    FloatOperands<NT, MT> raw[2];
    Thirds<NT, MT> now[2];
    raw[0].read(lines + BM * kLineBytes, lines, wn, wm, 0);
    raw[1].read(lines + BM * kLineBytes, lines, wn, wm, 1);
    now[0].take(raw[0]);
    for (int k = begin, stage = 0; k < end; k += kEach) {
      arrive<(kStages - 2) * kLoads>();
      load(k + kStages * kEach, stage);
      stage = stage == kStages - 1 ? 0 : stage + 1;
      const lds_char* const from = lines + stage * kStage;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        raw[j].read(from + BM * kLineBytes, from, wn, wm, j);
        now[j ^ 1].take(raw[j ^ 1]);
        now[j].multiply(acc);
        constexpr int kProducts = kThirds * NT * MT, kOthers = 44 * (NT + MT) / kProducts;
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);          // a product
          __builtin_amdgcn_sched_group_barrier(0x002, kOthers, 0);    // vector instructions
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    arrive<0>();
    if (any_not_finite(acc, reinterpret_cast<int*>(s_lines))) {
      start(kStages - 1);
      for (int k = begin, stage = 0; k < end; k += kEach) {
        arrive<(kStages - 2) * kLoads>();
        load(k + (kStages - 1) * kEach, stage == 0 ? kStages - 1 : stage - 1);
        const lds_char* const from = lines + stage * kStage;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          FloatOperands<NT, MT> again;
          again.read(from + BM * kLineBytes, from, wn, wm, j);
          again.multiply(acc);
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
      }
      arrive<0>();
    }
  } else {
    start(kStages - 1);
    arrive<(kStages - 2) * kLoads>();
    Operands<T, NT, MT> now[2];
    now[0].read(lines + BM * kLineBytes, lines, wn, wm, 0);
    int stage = 0;
    for (int k = begin; k < end; k += kEach) {
      const int into = stage == 0 ? kStages - 1 : stage - 1;
      const int after = stage == kStages - 1 ? 0 : stage + 1;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s == 0) load(k + (kStages - 1) * kEach, into);
        if (s == kSteps - 1) arrive<(kStages - 2) * kLoads>();
        const lds_char* const from = lines + (s == kSteps - 1 ? after : stage) * kStage;
        now[(s + 1) & 1].read(from + BM * kLineBytes, from, wn, wm, (s + 1) % kSteps);
        now[s & 1].multiply(acc);
        __builtin_amdgcn_sched_barrier(0);
      }
      stage = after;
    }
    arrive<0>();
  }
  finish_tile<T>(p, acc, reinterpret_cast<f32x4*>(s_lines) + wave * 32 * NT * 8, m0 + wm, n0 + wn,
                 blockIdx.y);
}

// Operands whose rows do not start on 16 bytes: 64 rows of each by a split of
// the summed axis, from memory into registers, which a load of 16 bytes reaches
// from any address, and on into LDS, a step ahead of the products.  What one
// step ahead brings in bounds it: a row by 4095 x 6144 in bfloat16 14.7 us, 64
// rows 30 (4096: 11.7 and 15), 1,111 rows by 2303 x 1544 in float16 34 (2304:
// 18).  Element by element and nothing ahead they took 125, 173 and 117.
template <typename T>
__global__ __launch_bounds__(256) void linear_odd_kernel(LinearParams p) {
  constexpr int B = 64, kThreads = 256;
  constexpr int kEach = 16 / static_cast<int>(sizeof(T)), kColumns = kLineChunks * kEach;
  constexpr int kLoads = B * kLineChunks / kThreads, kStage = 2 * B * kLineBytes;
  __shared__ __align__(16) char s_lines[2 * kStage];
  lds_char* const lines = (lds_char*)s_lines;
  const int tid = static_cast<int>(threadIdx.x);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  int m0, n0;
  tile_place<B, B>(p, gridDim.x, m0, n0);
  const int begin = static_cast<int>(blockIdx.y) * p.chunk;
  const int end = p.inner - begin < p.chunk ? p.inner : begin + p.chunk;
  const int wm = wave % 2 * 32, wn = wave / 2 * 32;
  f32x16 acc[1][1];
  clear(acc);
  u32x4 held[2][kLoads];
  auto load = [&](int of, const void* base, int64_t stride, int first, int rows, int k) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = i * kThreads + tid, row = first + q / kLineChunks;
      const int column = k + line_chunk(q / kLineChunks, q % kLineChunks) * kEach;
      const T* const from = static_cast<const T*>(base) + row * stride + column;
      u32x4 v = {0, 0, 0, 0};
      if (row < rows && column + kEach <= end) {
        __builtin_memcpy(&v, from, 16);
      } else if (row < rows && column < end) {
        T each[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) each[j] = column + j < end ? from[j] : static_cast<T>(0.0f);
        v = __builtin_bit_cast(u32x4, each);
      }
      held[of][i] = v;
    }
  };
  auto load_step = [&](int k) {
    load(0, p.x, p.x_row, m0, p.rows, k);
    load(1, p.weight, p.weight_row, n0, p.outer, k);
  };
  load_step(begin);
  for (int k = begin, stage = 0; k < end; k += kColumns, stage ^= 1) {
    lds_char* const xs = lines + stage * kStage;
    lds_char* const ws = xs + B * kLineBytes;
#pragma unroll
    for (int of = 0; of < 2; ++of)
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(
            (of ? ws : xs) + (i * kThreads + tid) * 16) = held[of][i];
    __syncthreads();
    load_step(k + kColumns);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Operands<T, 1, 1> now;
      now.read(ws, xs, wn, wm, s);
      now.multiply(acc);
    }
  }
  __syncthreads();
  finish_tile<T>(p, acc, reinterpret_cast<f32x4*>(s_lines) + wave * 32 * 8, m0 + wm, n0 + wn,
                 blockIdx.y);
}

// --------------------------------------------------------------- few rows

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

// 16 R rows of an operand, from memory into registers: a lane's four rows'
// worth of 16 bytes in a step.
template <typename T, int R>
struct FewRows {
  const T* first;
  int bytes;
  uint32_t from[R];
  __device__ __forceinline__ FewRows(const void* base, int64_t stride, int at, int rows,
                                     int inner) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int left = rows - at < 16 * R ? rows - at : 16 * R;
    first = static_cast<const T*>(base) + at * stride;
    bytes = static_cast<int>(((left - 1) * stride + inner) * static_cast<int64_t>(sizeof(T)));
#pragma unroll
    for (int t = 0; t < R; ++t)
      from[t] = static_cast<uint32_t>((t * 16 + (lane & 15)) * stride *
                                      static_cast<int64_t>(sizeof(T)));
  }
  __device__ __forceinline__ u32x4 load(int t, uint32_t at) const {
    return load_chunk(first, bytes, from[t] + at);
  }
};

constexpr int kFewWaves = 8;
constexpr int kFewRows = 64;

// One workgroup: 16 rows of W over all of the summed axis, which its waves
// share two steps (128 bytes of a row) at a time, by all of x, 16 MT rows.
// Every weight is read once, from memory into registers, the next ones while
// these are used; the waves' sums meet in LDS.
//
// What a CU can have on its way bounds it: some 36 bytes a nanosecond, of W
// and of x.  bfloat16, a row by 4096 x 6144: 11.7 us, 4.3 TB/s.
template <typename T, int MT>
__global__ __launch_bounds__(kFewWaves * kWave) void linear_few_kernel(LinearParams p) {
  constexpr int kEach = 16 / static_cast<int>(sizeof(T));   // columns a lane
  constexpr int kAhead = 2;                                 // steps whose loads go out together
  constexpr int kSpan = kAhead * 4 * kEach;                 // columns of those
  __shared__ f32x4 s_sums[kFewWaves][MT][kWave];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int n0 = static_cast<int>(blockIdx.x) * 16;
  const FewRows<T, MT> x(p.x, p.x_row, 0, p.rows, p.inner);
  const FewRows<T, 1> w(p.weight, p.weight_row, n0, p.outer, p.inner);
  const int row = lane & 15, quarter = lane >> 4;
  f32x4 acc[MT];
#pragma unroll
  for (int u = 0; u < MT; ++u) acc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Set {
    u32x4 a[kAhead], b[kAhead][MT];
  };
  auto load = [&](Set& set, int k) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int column = k + (s * 4 + quarter) * kEach;
      const uint32_t at = column < p.inner
                              ? static_cast<uint32_t>(column * static_cast<int>(sizeof(T)))
                              : kNowhere;
      set.a[s] = w.load(0, at);
#pragma unroll
      for (int u = 0; u < MT; ++u) set.b[s][u] = x.load(u, at);
    }
  };
  auto multiply = [&](const Set& set) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[u] = Product<T>::narrow(set.a[s], set.b[s][u], acc[u]);
  };
  constexpr int kStride = kFewWaves * kSpan;
  Set one, two;
  load(one, wave * kSpan);
  for (int k = wave * kSpan; k < p.inner; k += 2 * kStride) {
    load(two, k + kStride);                  // past the end: zeros
    __builtin_amdgcn_sched_barrier(0);
    multiply(one);
    load(one, k + 2 * kStride);
    __builtin_amdgcn_sched_barrier(0);
    multiply(two);
  }
#pragma unroll
  for (int u = 0; u < MT; ++u) s_sums[wave][u][lane] = acc[u];
  __syncthreads();
  if (wave < MT) {
    f32x4 y = s_sums[0][wave][lane];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) y += s_sums[v][wave][lane];
    finish4<T>(p, wave * 16 + row, n0 + quarter * 4, y);
  }
}

// ----------------------------------------------------------------- launch

int32_t launch_groups(void (*kernel)(LinearParams), int64_t groups, int splits, int threads,
                      int bytes, const LinearParams& p, hipStream_t s) {
  // a launch counts its threads in 32 bits
  if (groups > UINT32_MAX / threads) return fail(COWSDM_ELIMIT, "linear: output too large");
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess)
      return fail(static_cast<int32_t>(e), "linear: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(groups), static_cast<uint32_t>(splits)),
                     dim3(threads), bytes, s, p);
  return launch_status("linear");
}

constexpr int64_t tiles_of(int64_t rows, int64_t outer, int bm, int bn) {
  return ((rows + bm - 1) / bm) * ((outer + bn - 1) / bn);
}

enum class LinearForm { kOdd, kFew, k64, k64x128, k128, k256 };
struct LinearPlan {
  LinearForm form;
  int splits;
};

template <typename T, int BM, int BN, int MW, int NW, int kStages>
int32_t launch_tiles(const LinearParams& p, hipStream_t s) {
  constexpr int kLines = kStages * (BM + BN) * kLineBytes;
  constexpr int kTurned = MW * NW * 32 * (BN / NW) * 4;
  return launch_groups(&linear_tile_kernel<T, BM, BN, MW, NW, kStages>,
                       tiles_of(p.rows, p.outer, BM, BN), p.splits, MW * NW * kWave,
                       kLines > kTurned ? kLines : kTurned, p, s);
}

template <typename T, int MT>
int32_t launch_few(const LinearParams& p, hipStream_t s) {
  return launch_groups(&linear_few_kernel<T, MT>, (p.outer + 15) / 16, 1, kFewWaves * kWave, 0, p,
                       s);
}

template <typename T>
int32_t launch_linear(LinearParams p, const LinearPlan& plan, hipStream_t s) {
  p.splits = 1;
  p.chunk = p.inner;
  if (plan.splits > 1) {
    constexpr int kEach = kLineBytes / static_cast<int>(sizeof(T));
    const int steps = (p.inner + kEach - 1) / kEach;
    p.splits = plan.splits;
    p.chunk = (steps + plan.splits - 1) / plan.splits * kEach;
  }
  int32_t e = 0;
  switch (plan.form) {
    case LinearForm::kOdd:
      e = launch_groups(&linear_odd_kernel<T>, tiles_of(p.rows, p.outer, 64, 64), p.splits, 256, 0,
                        p, s);
      break;
    case LinearForm::kFew:
      if (p.rows <= 16) return launch_few<T, 1>(p, s);
      if (p.rows <= 32) return launch_few<T, 2>(p, s);
      return launch_few<T, 4>(p, s);
    case LinearForm::k64: e = launch_tiles<T, 64, 64, 2, 2, 4>(p, s); break;
    case LinearForm::k64x128: e = launch_tiles<T, 64, 128, 2, 2, 4>(p, s); break;
    case LinearForm::k128: e = launch_tiles<T, 128, 128, 2, 2, 4>(p, s); break;
    case LinearForm::k256: {
      void (*kernel)(LinearParams) = &linear_large_float_kernel;
      if constexpr (sizeof(T) == 2) kernel = &linear_large_kernel<T>;
      e = launch_groups(kernel, tiles_of(p.rows, p.outer, 256, 256), p.splits, 512,
                        5 * 256 * kLineBytes, p, s);
      break;
    }
  }
  if (e || p.splits == 1) return e;
  const int64_t chunks = static_cast<int64_t>(p.rows) * ((p.outer + 3) / 4);
  return launch_groups(&linear_join_kernel<T>, (chunks + 255) / 256, 1, 256, 0, p, s);
}

// What a form takes of a call's sizes, in microseconds: rounds of workgroups,
// each so long a step of 128 bytes and so long at its ends, or the memory's
// time, and, where the summed axis is split, the join's launch and traffic.
// The least one runs; where rows do not all start on 16 bytes, by their width,
// stride or address, that is the odd form with the best of its own splits (a row
// by 4096 x 1024 in bfloat16 at an odd address 7.8 us in 16 splits, 31.8 in the
// one split of few rows).  The constants are fitted to calls on one MI355X, which
// they give within some 20 %; in bfloat16, by the forms (splits):
//   64 rows, 128 x 384: few 3.2, tiles of 64 3.7; 32 rows, 8192 x 512: few 23,
//   64 (16) 8.9; a row, 4096 x 6144: few 11.7, 64 x 128 (5) 12.7; 64 rows: few
//   38, 64 (2) 15.0, 64 x 128 (4) 15.2, 64 x 128 (1) 25
//   100 rows, 4000 x 100: 64 (16) 7.6, 64 (1) 19
//   2,910 rows, 7848 x 1420: 128 150, 128 (3) 119, 256 150, 256 (3) 80
//   1,111 rows, 2304 x 1544: 64 17.8, 64 x 128 17.9, 128 24, 256 47
//   2,048 rows, 2048 x 2048: 64 31, 64 x 128 32, 128 25, 256 44
//   4,096 rows, 4096 x 4096: 64 206, 64 x 128 197, 128 155, 256 99
//   and in float32 4,000 rows, 4000 x 4000: 64 930, 64 x 128 875, 128 677, 256
//   561; 256 rows, 2048 x 2048: 64 39, 64 (4) 25, 64 x 128 (4) 24; 64 rows, 4096 x
//   6144: few 73, 64 x 128 106, 64 x 128 (5) 34
//   and of rows that are not aligned 64 rows, 4095 x 6144: 49, (2) 30.
struct FormCost {
  LinearForm form;
  int rows, columns;               // of a tile
  float step[2], ends;             // of 16-bit types, and of float32
};
constexpr FormCost kFormCosts[] = {
    {LinearForm::kOdd, 64, 64, {0.45f, 0.8f}, 1.0f},
    {LinearForm::k64, 64, 64, {0.30f, 0.57f}, 1.0f},
    {LinearForm::k64x128, 64, 128, {0.38f, 0.85f}, 1.0f},
    {LinearForm::k128, 128, 128, {0.58f, 1.4f}, 2.5f},
    {LinearForm::k256, 256, 256, {1.45f, 4.55f}, 4.0f},
};
constexpr int64_t kChipCus = 256;
constexpr int kMostSplits = 16;

// `aligned`: both operands' addresses and strides are multiples of 16 bytes.
LinearPlan plan_linear(int64_t rows, int64_t inner, int64_t outer, int size, bool aligned) {
  const float memory =
      static_cast<float>((rows * inner + inner * outer + rows * outer) * size) * (1.0f / 5.0e6f);
  const bool odd = !aligned || inner * size % 16 != 0;
  LinearPlan best{odd ? LinearForm::kOdd : LinearForm::k128, 1};   // of nothing to sum
  float least = 3.0e38f;
  auto consider = [&](LinearForm form, int splits, float us) {
    if (us < least) {
      least = us;
      best = {form, splits};
    }
  };
  if (rows <= kFewRows && !odd) {
    const int64_t rounds = ((outer + 15) / 16 + kChipCus - 1) / kChipCus;
    const float us = static_cast<float>(rounds * (16 + rows) * inner * size) * (1.0f / 36.0e3f);
    consider(LinearForm::kFew, 1, 2.3f + (us > memory ? us : memory));
  }
  const int64_t steps = (inner * size + kLineBytes - 1) / kLineBytes;
  for (const FormCost& f : kFormCosts) {
    if (odd != (f.form == LinearForm::kOdd)) continue;
    const int64_t tiles = tiles_of(rows, outer, f.rows, f.columns);
    const int most = tiles >= kChipCus ? 4 : kMostSplits;
    for (int splits = 1; splits <= most && splits <= steps; ++splits) {
      const int64_t groups = tiles * splits, each = (steps + splits - 1) / splits;
      float step = f.step[size == 4];
      int64_t rounds = (groups + kChipCus - 1) / kChipCus;
      if (f.form == LinearForm::k64 && size == 2 && rounds > 1) {   // two a CU
        rounds = (rounds + 1) / 2;
        step = 0.45f;
      }
      const float us = static_cast<float>(rounds) * (static_cast<float>(each) * step + f.ends);
      const float join =
          splits == 1 ? 0.0f
                      : 3.0f + static_cast<float>(8 * splits * rows * outer) * (1.0f / 4.5e6f);
      consider(f.form, splits, 2.0f + (us > memory ? us : memory) + join);
    }
  }
  // no split is left without columns
  if (best.splits > 1) {
    const int64_t each = (steps + best.splits - 1) / best.splits;
    best.splits = static_cast<int>((steps + each - 1) / each);
  }
  return best;
}

}  // namespace cowsdm_impl

using namespace cowsdm_impl;

namespace {

int64_t workspace_of(const LinearPlan& plan, int64_t rows, int64_t outer) {
  return plan.splits == 1 ? 0 : plan.splits * rows * ((outer + 3) / 4 * 16);
}

// 16-byte loads of both operands, as far as their inner size allows them
bool linear_aligned(const cowsdm_linear_t& l) {
  const int64_t unit = l.float_type == COWSDM_FLOAT32 ? 4 : 8;
  return (reinterpret_cast<uintptr_t>(l.x) | reinterpret_cast<uintptr_t>(l.weight)) % 16 == 0 &&
         l.x_row % unit == 0 && l.weight_row % unit == 0;
}

}  // namespace

extern "C" int32_t cowsdm_linear_plan(int64_t rows, int64_t inner, int64_t outer,
                                      int32_t float_type, int32_t aligned,
                                      cowsdm_linear_plan_t* plan) {
  if (!plan) return fail(COWSDM_EARG, "linear_plan: null argument");
  if (rows < 0 || inner < 0 || outer < 0)
    return fail(COWSDM_EARG, "linear_plan: negative size");
  if (float_type != COWSDM_FLOAT32 && float_type != COWSDM_FLOAT16 &&
      float_type != COWSDM_BFLOAT16)
    return fail(COWSDM_EARG, "linear_plan: bad float type");
  if (inner > COWSDM_LINEAR_MOST || rows > INT32_MAX - 256 || outer > INT32_MAX - 256)
    return fail(COWSDM_ELIMIT, "linear_plan: too large");
  *plan = cowsdm_linear_plan_t{};
  if (rows == 0 || outer == 0) return 0;
  const LinearPlan p =
      plan_linear(rows, inner, outer, float_type == COWSDM_FLOAT32 ? 4 : 2, aligned != 0);
  plan->workspace_bytes = workspace_of(p, rows, outer);
  plan->splits = p.splits;
  if (p.form == LinearForm::kFew) {
    plan->tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : kFewRows;
    plan->tile_columns = 16;
  }
  for (const FormCost& f : kFormCosts) {
    if (f.form != p.form) continue;
    plan->tile_rows = f.rows;
    plan->tile_columns = f.columns;
  }
  return 0;
}

extern "C" int64_t cowsdm_linear_workspace_bytes(int64_t rows, int64_t inner, int64_t outer,
                                                 int32_t float_type) {
  if (rows < 0 || inner < 0 || outer < 0 || rows > INT32_MAX || outer > INT32_MAX) return -1;
  if (rows == 0 || outer == 0) return 0;
  const int size = float_type == COWSDM_FLOAT32 ? 4 : 2;
  const int64_t aligned = workspace_of(plan_linear(rows, inner, outer, size, true), rows, outer);
  const int64_t odd = workspace_of(plan_linear(rows, inner, outer, size, false), rows, outer);
  return aligned > odd ? aligned : odd;
}

extern "C" int32_t cowsdm_linear(const cowsdm_linear_t* linear, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
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
  const int64_t size = l.float_type == COWSDM_FLOAT32 ? 4 : 2;
  auto address = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const LinearPlan plan =
      plan_linear(l.rows, l.inner, l.outer, static_cast<int>(size), linear_aligned(l));
  if (plan.splits > 1) {
    const int64_t need = workspace_of(plan, l.rows, l.outer);
    if (!workspace || workspace_bytes < need)
      return fail(COWSDM_EARG, "linear: workspace of %lld bytes needed",
                  static_cast<long long>(need));
    if (address(workspace) % 16)
      return fail(COWSDM_EARG, "linear: the workspace must be 16-byte aligned");
  }
  LinearParams p{};
  p.x = l.x;
  p.weight = l.weight;
  p.bias = l.bias;
  p.residual = l.residual;
  p.out = l.out;
  p.x_row = l.x_row;
  p.weight_row = l.weight_row;
  p.residual_row = l.residual_row;
  p.rows = static_cast<int32_t>(l.rows);
  p.inner = static_cast<int32_t>(l.inner);
  p.outer = static_cast<int32_t>(l.outer);
  p.activation = l.activation;
  p.parts = static_cast<float*>(workspace);
  const auto s = static_cast<hipStream_t>(stream);
  if (l.float_type == COWSDM_FLOAT32) return launch_linear<float>(p, plan, s);
  if (l.float_type == COWSDM_FLOAT16) return launch_linear<_Float16>(p, plan, s);
  return launch_linear<__bf16>(p, plan, s);
}
