// Query and key heads normed and rotated by position, in one pass.
//
// A position's angle is a fraction of a turn, position * turns[j] modulo
// 2^64: exact in integers however far the position, where 32-bit floating
// angles are off by whole degrees from some 100,000 tokens on.  What remains
// after the nearest quarter turn is at most pi / 4, for which the Taylor
// polynomials to the 9th and 10th power are within 2e-9.

#include <type_traits>

#include "attention.h"

namespace cowsdm_impl {

constexpr int kHeadWaves = 4;
constexpr int kHeadThreads = kHeadWaves * kWave;
constexpr int kHeadMostWidth = 256;
constexpr int kHeadTokens = 16, kHeadBytes = 16384, kHeadGroups = 4096;

struct HeadParams {
  const void* query;
  const void* key;
  int64_t query_row, query_head, key_row, key_head;
  const int32_t* positions;
  const uint64_t* turns;
  const void* query_weight;
  const void* key_weight;
  void* query_out;
  void* key_out;
  int32_t rows;
  int32_t heads;          // of the query
  int32_t all_heads;      // and of the key
  int32_t width;
  int32_t rotated;
  int32_t tokens;         // of a workgroup
  int32_t lanes;          // of a row: a power of two
  float inverse_width;
  float eps;
};

// (cos, sin) of `phase` / 2^64 of a turn.
__device__ __forceinline__ float2 turn_point(uint64_t phase) {
  const uint64_t quarter = (phase + (uint64_t{1} << 61)) >> 62;
  const int32_t rest = static_cast<int32_t>(static_cast<int64_t>(phase - (quarter << 62)) >> 32);
  const float x = static_cast<float>(rest) * 1.4629180792671596e-09f;    // 2 pi / 2^32
  const float z = x * x;
  float s = __builtin_fmaf(z, 2.7557319e-06f, -1.9841270e-04f);
  s = __builtin_fmaf(s, z, 8.3333333e-03f);
  s = __builtin_fmaf(s, z, -1.6666667e-01f);
  s = __builtin_fmaf(s * z, x, x);
  float c = __builtin_fmaf(z, -2.7557319e-07f, 2.4801587e-05f);
  c = __builtin_fmaf(c, z, -1.3888889e-03f);
  c = __builtin_fmaf(c, z, 4.1666667e-02f);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.0f);
  const bool odd = quarter & 1;
  const float a = odd ? s : c, b = odd ? c : s;
  return make_float2(((quarter + 1) & 2) ? -a : a, (quarter & 2) ? -b : b);
}

// C consecutive elements, in float32.
template <typename T, int C>
__device__ __forceinline__ void load_head(const T* p, float (&x)[C]) {
  typedef T vec __attribute__((ext_vector_type(C)));
  const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
  for (int i = 0; i < C; ++i) x[i] = static_cast<float>(v[i]);
}

template <typename T, int C>
__device__ __forceinline__ void store_head(T* p, const float (&x)[C]) {
  typedef T vec __attribute__((ext_vector_type(C)));
  vec v;
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] = static_cast<T>(x[i]);
  *reinterpret_cast<vec*>(p) = v;
}

// A workgroup takes some tokens: their points on the circle go to LDS, one a
// thread, and then every row of a head is a few lanes', each with two chunks
// of C elements that are rotated with each other (or, interleaved, each in
// itself), so that nothing crosses lanes but the norm's sum.  16 bytes a lane
// are read and written where the width allows it.  Memory bounds it from some
// 4,096 tokens on: 16,383 tokens of 40 heads 128 wide in bfloat16 (336 MB read
// and written) take 63 us, 5.3 TB/s, what a large copy reaches.  64 of them
// take 4.6 us: latency of a launch, the positions, the rows and the stores.
template <typename T, int C, bool kInterleaved>
__global__ __launch_bounds__(kHeadThreads) void rotate_heads_kernel(HeadParams p) {
  extern __shared__ __align__(16) char s_heads[];
  float* const s_weight = reinterpret_cast<float*>(s_heads);          // [2][width]
  float2* const s_point = reinterpret_cast<float2*>(s_weight + 2 * p.width);
  const int tid = static_cast<int>(threadIdx.x);
  const int first = static_cast<int>(blockIdx.x) * p.tokens;
  const int tokens = p.rows - first < p.tokens ? p.rows - first : p.tokens;
  const int pairs = p.rotated / 2;
  for (int i = tid; i < tokens * pairs; i += kHeadThreads) {
    const int t = i / pairs, j = i - t * pairs;
    const int64_t position = p.positions[first + t];
    s_point[i] = turn_point(static_cast<uint64_t>(position) * p.turns[j]);
  }
  for (int i = tid; i < 2 * p.width; i += kHeadThreads) {
    const int d = i < p.width ? i : i - p.width;
    const T* const w = static_cast<const T*>(i < p.width ? p.query_weight : p.key_weight);
    s_weight[i] = w ? static_cast<float>(w[d]) : 1.0f;
  }
  __syncthreads();
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  const int at = lane & (p.lanes - 1);                  // this lane's place in its row
  const int each = kWave / p.lanes;                     // rows of a wave's step
  const int swaps = p.rotated / (2 * C);                // lanes whose chunks are rotated
  const int spare = at - swaps;
  const int a = (spare < 0 ? at : 2 * swaps + 2 * spare) * C;
  const int b = spare < 0 ? a + swaps * C : a + C;
  const bool mine = a < p.width;
  const int rows = tokens * p.all_heads;
  for (int r = wave * each + lane / p.lanes; r < rows; r += kHeadWaves * each) {
    const int t = r / p.all_heads, h = r - t * p.all_heads;
    const bool is_key = h >= p.heads;
    const int64_t token = first + t;
    const T* const src =
        is_key ? static_cast<const T*>(p.key) + token * p.key_row + (h - p.heads) * p.key_head
               : static_cast<const T*>(p.query) + token * p.query_row + h * p.query_head;
    const int key_heads = p.all_heads - p.heads;
    T* const dst = is_key ? static_cast<T*>(p.key_out) +
                                (token * key_heads + (h - p.heads)) * p.width
                          : static_cast<T*>(p.query_out) + (token * p.heads + h) * p.width;
    float x[C] = {}, y[C] = {};
    if (mine) {
      load_head<T, C>(src + a, x);
      load_head<T, C>(src + b, y);
    }
    if (is_key ? p.key_weight != nullptr : p.query_weight != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < C; ++i) sum = __builtin_fmaf(x[i], x[i], __builtin_fmaf(y[i], y[i], sum));
      for (int o = p.lanes / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
      const float f = 1.0f / sqrtf(__builtin_fmaf(sum, p.inverse_width, p.eps));
      const float* const w = s_weight + (is_key ? p.width : 0);
      if (mine) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          x[i] = x[i] * f * w[a + i];
          y[i] = y[i] * f * w[b + i];
        }
      }
    }
    if (!mine) continue;
    if (spare < 0) {
      const float2* const point = s_point + t * pairs;
      if constexpr (kInterleaved) {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
          const float2 u = point[(a + i) / 2], v = point[(b + i) / 2];
          const float x0 = x[i], y0 = y[i];
          x[i] = x0 * u.x - x[i + 1] * u.y;
          x[i + 1] = x0 * u.y + x[i + 1] * u.x;
          y[i] = y0 * v.x - y[i + 1] * v.y;
          y[i + 1] = y0 * v.y + y[i + 1] * v.x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const float2 u = point[a + i];
          const float x0 = x[i];
          x[i] = x0 * u.x - y[i] * u.y;
          y[i] = x0 * u.y + y[i] * u.x;
        }
      }
    }
    store_head<T, C>(dst + a, x);
    store_head<T, C>(dst + b, y);
  }
}

template <typename T, int C>
int32_t launch_heads(HeadParams p, bool interleaved, hipStream_t s) {
  const int need = p.width / (2 * C);
  p.lanes = 1;
  while (p.lanes < need) p.lanes *= 2;
  // Tokens of a workgroup: few enough that its waves take their heads in one
  // step (64 tokens of 40 heads 128 wide: 4.6 us with one each, 7.9 with four),
  // but where there are many tokens enough that a workgroup's work outlasts its
  // launch, some 2 ns (65,536 tokens, with one each and with 16 KB read and
  // written each: 6 heads 64 wide in bfloat16 58 and 21 us, 24 heads 80 wide
  // 134 and 104).
  const int bytes_each = 2 * p.all_heads * p.width * static_cast<int>(sizeof(T));
  const int one_step = kHeadWaves * kWave / p.lanes / p.all_heads;
  const int enough = (kHeadBytes + bytes_each - 1) / bytes_each;
  p.tokens = one_step < 1 ? 1 : one_step;
  if (p.rows > kHeadGroups * p.tokens && p.tokens < enough) p.tokens = enough;
  if (p.tokens > kHeadTokens) p.tokens = kHeadTokens;
  const int groups = (p.rows + p.tokens - 1) / p.tokens;
  // a launch counts its threads in 32 bits
  if (groups > static_cast<int>(UINT32_MAX / kHeadThreads))
    return fail(COWSDM_ELIMIT, "rotate_heads: too large");
  const int bytes = 8 * p.width + 4 * p.tokens * p.rotated;
  if (interleaved)
    hipLaunchKernelGGL((rotate_heads_kernel<T, C, true>), dim3(groups), dim3(kHeadThreads), bytes,
                       s, p);
  else
    hipLaunchKernelGGL((rotate_heads_kernel<T, C, false>), dim3(groups), dim3(kHeadThreads),
                       bytes, s, p);
  return launch_status("rotate_heads");
}

}  // namespace cowsdm_impl

using namespace cowsdm_impl;

extern "C" int32_t cowsdm_rotate_heads(const cowsdm_rotate_heads_t* heads, void* stream) {
  if (!heads) return fail(COWSDM_EARG, "rotate_heads: null argument");
  const cowsdm_rotate_heads_t& a = *heads;
  if (a.rows < 0 || a.heads < 0 || a.kv_heads < 0 || a.heads + a.kv_heads <= 0 || a.width <= 0)
    return fail(COWSDM_EARG, "rotate_heads: bad size");
  if (a.width % 8 != 0) return fail(COWSDM_EARG, "rotate_heads: width must be a multiple of 8");
  if (a.rotated < 0 || a.rotated % 8 != 0 || a.rotated > a.width)
    return fail(COWSDM_EARG,
                "rotate_heads: rotated elements must be a multiple of 8, at most the width");
  if (a.width > kHeadMostWidth) return fail(COWSDM_ELIMIT, "rotate_heads: width at most 256");
  if (a.float_type != COWSDM_FLOAT32 && a.float_type != COWSDM_FLOAT16 &&
      a.float_type != COWSDM_BFLOAT16)
    return fail(COWSDM_EARG, "rotate_heads: bad float type");
  if (!(a.eps >= 0.0f) || a.eps > 3.0e38f)
    return fail(COWSDM_EARG, "rotate_heads: eps cannot be negative");
  // counted in 32 bits here, and a launch's threads by its workgroups
  if (a.rows >= (int64_t{1} << 24) * 3 || a.heads > 65535 || a.kv_heads > 65535)
    return fail(COWSDM_ELIMIT, "rotate_heads: too large");
  if (a.rows == 0) return 0;
  if ((a.heads > 0 && (!a.query || !a.query_out)) ||
      (a.kv_heads > 0 && (!a.key || !a.key_out)) ||
      (a.rotated > 0 && (!a.positions || !a.turns)))
    return fail(COWSDM_EARG, "rotate_heads: null pointer argument");
  const int64_t unit = a.float_type == COWSDM_FLOAT32 ? 4 : 8;
  auto address = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  if ((address(a.query) | address(a.key) | address(a.query_out) | address(a.key_out)) % 16 ||
      a.query_row < 0 || a.query_head < 0 || a.key_row < 0 || a.key_head < 0 ||
      (a.query_row | a.query_head | a.key_row | a.key_head) % unit)
    return fail(COWSDM_EARG, "rotate_heads: rows must be 16-byte aligned");
  HeadParams p{};
  p.query = a.query;
  p.key = a.key;
  p.query_row = a.query_row;
  p.query_head = a.query_head;
  p.key_row = a.key_row;
  p.key_head = a.key_head;
  p.positions = a.positions;
  p.turns = a.turns;
  p.query_weight = a.query_weight;
  p.key_weight = a.key_weight;
  p.query_out = a.query_out;
  p.key_out = a.key_out;
  p.rows = static_cast<int32_t>(a.rows);
  p.heads = static_cast<int32_t>(a.heads);
  p.all_heads = static_cast<int32_t>(a.heads + a.kv_heads);
  p.width = static_cast<int32_t>(a.width);
  p.rotated = static_cast<int32_t>(a.rotated);
  p.inverse_width = 1.0f / static_cast<float>(a.width);
  p.eps = a.eps;
  const auto s = static_cast<hipStream_t>(stream);
  const bool by_eight = a.width % 16 == 0 && a.rotated % 16 == 0;
  if (a.float_type == COWSDM_FLOAT32) return launch_heads<float, 4>(p, a.interleaved, s);
  if (a.float_type == COWSDM_FLOAT16)
    return by_eight ? launch_heads<_Float16, 8>(p, a.interleaved, s)
                    : launch_heads<_Float16, 4>(p, a.interleaved, s);
  return by_eight ? launch_heads<__bf16, 8>(p, a.interleaved, s)
                  : launch_heads<__bf16, 4>(p, a.interleaved, s);
}
