// Causal attention over packed prompts with grouped heads.
//
// out[i] = sum_{j <= i} softmax_j(scale q_i . k_j) v_j, in one pass over the
// keys with the running maximum and sum of each row (the online softmax of
// Milakov and Gimelshein, 2018).  Scores are computed
// transposed, S^T = K Q^T, so that a lane holds keys of one query row and its
// probabilities are the right operand of O^T = V^T P^T where they stand:
// neither scores nor probabilities leave the registers.

#include <type_traits>

#include "attention.h"

namespace cowsdm_impl {

constexpr int kPromptWaves = 4;
constexpr int kPromptThreads = kPromptWaves * kWave;

struct PromptParams {
  const void* query;
  const void* key;
  const void* value;
  int64_t query_row, query_head, key_row, key_head, value_row, value_head;
  const int32_t* offsets;
  void* out;
  int32_t rows;
  int32_t sequences;
  int32_t heads;
  int32_t kv_heads;
  int32_t width;
  int32_t blocks;                  // query blocks of a sequence and head in the grid
  int32_t pair_by_pair;            // the grid's order
  float scale;                     // times log2(e)
};

// What a workgroup works on: a sequence, a head, and the first of its query
// blocks (the others are `blocks` further on).
struct PromptWork {
  int sequence, head, kv, block;
};

// Workgroup n runs on XCD n % 8: a pair of a sequence and a key head keeps to
// one XCD where the pairs divide by eight, so that its keys and values stay
// in that XCD's L2.  Later query blocks, which see more keys, come first: of
// all pairs in small grids, where what starts last decides (16 heads of 4,096
// tokens: 91 us, pair by pair 112), and pair by pair in large ones, whose keys
// and values would push each other out (24 prompts of 2,048, 32 heads over 8:
// 909 against 936; 2 x 8,192: 987 against 991).  The grid's size counts
// workgroups that end at once, too: a prompt of 8,192 among 30 of 64 has a
// large grid and little work, and takes 589 pair by pair, 545 the other way.
__device__ __forceinline__ PromptWork prompt_work(const PromptParams& p) {
  const int group = p.heads / p.kv_heads;
  const int pairs = p.sequences * p.kv_heads;
  const int sides = pairs % 8 == 0 ? 8 : 1;
  const int id = static_cast<int>(blockIdx.x) / sides;
  const int own = pairs / sides;              // pairs of this XCD
  int pair, block;
  if (p.pair_by_pair) {
    pair = id / (p.blocks * group);
    block = id / group % p.blocks;
  } else {
    pair = id / group % own;
    block = id / (group * own);
  }
  pair = pair * sides + static_cast<int>(blockIdx.x) % sides;
  PromptWork w;
  w.sequence = pair / p.kv_heads;
  w.kv = pair - w.sequence * p.kv_heads;
  w.block = p.blocks - 1 - block;
  w.head = w.kv * group + id % group;
  return w;
}

// Rows before the first sequence and after the last are 0.
template <typename T>
__device__ void zero_rows(const PromptParams& p, const PromptWork& w) {
  const int first = p.offsets[0], last = p.offsets[p.sequences];
  auto zero = [&](int from, int to) {
    for (int r = from + w.block; r < to; r += p.blocks)
      for (int d = threadIdx.x; d < p.width; d += kPromptThreads)
        static_cast<T*>(p.out)[(static_cast<int64_t>(r) * p.heads + w.head) * p.width + d] =
            static_cast<T>(0.0f);
  };
  if (w.sequence == 0 && first > 0) zero(0, first < p.rows ? first : p.rows);
  if (w.sequence == p.sequences - 1 && last < p.rows) zero(last > 0 ? last : 0, p.rows);
}

__device__ __forceinline__ void sequence_rows(const PromptParams& p, int sequence, int& begin,
                                              int& length) {
  const int a = p.offsets[sequence], b = p.offsets[sequence + 1];
  begin = a < 0 ? 0 : a > p.rows ? p.rows : a;
  const int end = b < begin ? begin : b > p.rows ? p.rows : b;
  length = end - begin;
}

// ------------------------------------------------------------ 16-bit types

template <typename T>
struct Half;
template <>
struct Half<__bf16> {
  typedef bf16x8 vec;
  static constexpr uint32_t kExponent = 0x7f807f80u;
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Half<_Float16> {
  typedef f16x8 vec;
  static constexpr uint32_t kExponent = 0x7c007c00u;
  static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kTileKeys = 64;

// The 16-byte chunk of row `row` of a tile in LDS that holds the row's chunk
// c: chunks are permuted so that the 16 rows of a key read, and the 4 rows by
// 64 bytes of a transposing value read, fall on different banks.
template <int DP>
__device__ __forceinline__ int place(int row, int c) {
  constexpr int chunks = DP / 8;
  if constexpr (chunks % 16 == 0) return c ^ (((row & 3) << 2) | ((row >> 2) & 3));
  else if constexpr (chunks % 8 == 0) return c ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
  else return c ^ ((row >> 2) & 3);
}

// This thread's chunks of a tile into LDS, a wave's side by side.  Rows past
// the sequence's end and columns past the width read as 0.
template <int kLoads, int kThreads>
__device__ __forceinline__ void load_rows(const void* first, int rows, int64_t stride, int width,
                                          const uint32_t (&from)[kLoads], lds_char* to) {
  const int bytes = static_cast<int>((rows - 1) * stride + width) * 2;
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    load_to_lds(first, bytes, from[i], to + i * kThreads * 16);
}

// Four keys of this lane's column from a tile in LDS, each group of 16 lanes
// reading four rows of 16 columns.
__device__ __forceinline__ s16x4 read_turned(const lds_char* __restrict at) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
}

// Of eight 16-bit numbers, whether one is not finite.
template <typename T>
__device__ __forceinline__ bool any_odd(typename Half<T>::vec v) {
  constexpr uint32_t kHigh = Half<T>::kExponent & 0xffff0000u;
  constexpr uint32_t kLow = Half<T>::kExponent & 0xffffu;
  const u32x4 bits = __builtin_bit_cast(u32x4, v);
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    odd |= (bits[j] & kHigh) == kHigh | (bits[j] & kLow) == kLow;
  return odd;
}

constexpr int kOthersMove = 0x406;       // a scheduling barrier that vector and scalar work passes

// Whole: every row sees all of the tile.  Edge: some do not.  Careful: as
// edge, and no value that is not finite reaches a row that does not see it.
enum class PromptTile { kWhole, kEdge, kCareful };

// One wave's 32 query rows of one head: q the rows, acc their products so far,
// transposed, most the maxima that the probabilities are relative to and sum
// their sums (of this lane's keys).
template <typename T, int DP>
struct PromptRows {
  using vec = typename Half<T>::vec;
  static constexpr int KS = DP / 16;       // products along the width
  static constexpr int DT = DP / 32;       // tiles of the output's width
  // steps that operands are read ahead of their products, as registers allow
  static constexpr int kKeysAhead = DP <= 192 ? 3 : 1;
  static constexpr int kValuesAhead = DP <= 192 ? 1 : 0;
  vec q[KS];
  f32x16 acc[DT];
  float most, sum;

  __device__ __forceinline__ void clear() {
    most = kMinusInf;
    sum = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
  }

  // The value operand of step h (16 keys) of column tile d.
  __device__ __forceinline__ vec turned(const lds_char* values, const int (&at)[DT][2], int h,
                                        int d) {
    struct { s16x4 a, b; } both{read_turned(values + at[d][0] + h * 16 * DP * 2),
                                read_turned(values + at[d][1] + h * 16 * DP * 2)};
    return __builtin_bit_cast(vec, both);
  }

  // The maxima grow to `now`.
  __device__ __forceinline__ void rise(float now) {
    const float keep = now == kMinusInf ? 1.0f : exp2_fast(most - now);
    most = now;
    sum *= keep;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] *= keep;
  }

  // One tile of 64 keys from row k0 on.
  template <PromptTile kKind>
  __device__ __forceinline__ void tile(const lds_char* keys, const lds_char* values,
                                       const int (&key_read)[KS],
                                       const int (&value_read)[DT][2], float scale, int k0,
                                       int q0) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int col = lane & 31, half = lane >> 5;
    f32x16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
    // operands are read from LDS some steps before the products that take
    // them, and are kept there: left to itself the compiler reads each at its
    // product, whose wait is longer than the product
    vec key[KS][2];
    auto read_keys = [&](int k) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        key[k][kb] = *reinterpret_cast<const __attribute__((address_space(3))) vec*>(
            keys + key_read[k] + kb * 32 * DP * 2);
    };
#pragma unroll
    for (int k = 0; k < kKeysAhead && k < KS; ++k) read_keys(k);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      if (k + kKeysAhead < KS) read_keys(k + kKeysAhead);
      __builtin_amdgcn_sched_barrier(kOthersMove);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[kb] = Half<T>::mfma(key[k][kb], q[k], s[kb]);
      __builtin_amdgcn_sched_barrier(kOthersMove);
    }
    vec value[4][DT];
    auto read_values = [&](int h) {
#pragma unroll
      for (int d = 0; d < DT; ++d) value[h][d] = turned(values, value_read, h, d);
    };
    if constexpr (kValuesAhead > 0) read_values(0);
    __builtin_amdgcn_sched_barrier(kOthersMove);
    if constexpr (kKind != PromptTile::kWhole) {
      const int row = q0 + col;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + kb * 32 + (i / 4) * 8 + half * 4 + i % 4 > row) s[kb][i] = kMinusInf;
    }
    float top = kMinusInf;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top),
                                                    false, false);
    top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * scale;
    // The maximum that the probabilities are relative to moves only when a
    // row's grows past 2^8 of it: sums of numbers up to 2^8 lose nothing in
    // 32 bits, and a probability keeps its bits in 16.
    if (__any(top > most + 8.0f)) rise(fmaxf(most, top));
    const float shift = most == kMinusInf ? 0.0f : most;
    // A 16-bit product takes its probabilities in 16 bits (the error against 64
    // bits is 0.0020 of the output's size in bfloat16, 0.0016 with
    // probabilities of 32 bits; 0.00025 and 0.00020 in float16); their sum
    // stays in 32.
    vec prob[4];
    float part[4] = {};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = exp2_fast(__builtin_fmaf(s[kb][i], scale, -shift));
        part[i % 4] += e;
        prob[2 * kb + i / 8][i % 8] = static_cast<T>(e);
      }
    sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      if (h + kValuesAhead < 4) read_values(h + kValuesAhead);
      __builtin_amdgcn_sched_barrier(kOthersMove);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        vec v = value[h][d];
        if constexpr (kKind == PromptTile::kCareful) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(__builtin_fabsf(static_cast<float>(v[j])) < __builtin_huge_valf()))
              v[j] = static_cast<T>(0.0f);
        }
        acc[d] = Half<T>::mfma(v, prob[h], acc[d]);
      }
      __builtin_amdgcn_sched_barrier(kOthersMove);
    }
    if constexpr (kKind == PromptTile::kCareful) add_odd(values, value_read, k0, q0);
  }

  // Whether an output of this lane is NaN.
  __device__ __forceinline__ bool any_nan() const {
    bool nan = false;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) nan |= acc[d][i] != acc[d][i];
    return nan;
  }

  // Values that are not finite, for the rows that see them.  Products of ones
  // and zeros count them, and what is counted is added by itself.
  __device__ __forceinline__ void add_odd(const lds_char* values, const int (&value_read)[DT][2],
                                          int k0, int q0) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const int col = lane & 31, half = lane >> 5;
#pragma unroll 1
    for (int h = 0; h < 4; ++h) {
      vec sees;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sees[j] = static_cast<T>(
            k0 + h * 16 + (j / 4) * 8 + half * 4 + j % 4 <= q0 + col ? 1.0f : 0.0f);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const vec v = turned(values, value_read, h, d);
        if (!__any(any_odd<T>(v))) continue;
#pragma unroll 1
        for (int n = 0; n < 3; ++n) {
          vec kind;
          const float sign = n == 1 ? __builtin_huge_valf() : kMinusInf;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = static_cast<float>(v[j]);
            kind[j] = static_cast<T>((n == 0 ? x != x : x == sign) ? 1.0f : 0.0f);
          }
          f32x16 c;
#pragma unroll
          for (int i = 0; i < 16; ++i) c[i] = 0.0f;
          c = Half<T>::mfma(kind, sees, c);
          const float add = n == 0 ? __builtin_nanf("") : sign;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c[i] > 0.0f) acc[d][i] += add;
        }
      }
    }
  }

  // The rows' numbers to and from LDS, a register of the wave's lanes after
  // the other.
  static constexpr int kFloats = (DT * 16 + 2) * kWave;
  typedef __attribute__((address_space(3))) float lds_float;
  __device__ __forceinline__ void give(lds_float* to) const {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) to[(d * 16 + i) * kWave + lane] = acc[d][i];
    to[DT * 16 * kWave + lane] = most;
    to[(DT * 16 + 1) * kWave + lane] = sum;
  }
  __device__ __forceinline__ void join(const lds_float* from) {
    const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
    const float other = from[DT * 16 * kWave + lane];
    rise(fmaxf(most, other));
    const float keep = other == kMinusInf ? 0.0f : exp2_fast(other - most);
    sum += from[(DT * 16 + 1) * kWave + lane] * keep;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] += from[(d * 16 + i) * kWave + lane] * keep;
  }
};

// One workgroup: four waves and 128 query rows of one head, 32 to a wave.
// Keys and values come through LDS, 64 at a time, by loads that go to LDS
// without passing registers; the next tile is on its way while this one is
// used.  KP = 2: 64 rows, of which two waves share 32; one takes the even and
// one the odd tiles, and their sums are joined at the end.  That is for grids
// that the chip holds at once, where the longest row's way through its keys
// counts.
//
// Two prompts of 8,192 tokens, 32 heads over 8, width 128, bfloat16: 975 to
// 990 us, 1,110 to 1,128 TFLOP/s of what causality leaves (a library's
// product of two 8,192 square matrices reaches 1,238 on the same card).  The
// matrix cores are busy 60 % of the cycles and the vector units, whose
// exponentials, maxima, sums and roundings are as long a chain, about as much,
// at the 1.9 GHz that such a load runs at; waits are 16 %, LDS a quarter busy,
// L2 hits 95 %.  24 packed prompts of up to 2,048 take 308 us, 723 TFLOP/s: a
// fifth of their tiles lie on the diagonal, and a workgroup starts and ends,
// with 64 KB from and to memory, around nine tiles (2 us each beside another
// workgroup, and 6 us).
template <typename T, int DP, int KP>
__global__ __launch_bounds__(kPromptThreads, DP <= 128 ? 2 : 1) void prompt_half_kernel(
    PromptParams p) {
  using Rows = PromptRows<T, DP>;
  using vec = typename Half<T>::vec;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  constexpr int KS = Rows::KS, DT = Rows::DT;
  constexpr int kSide = kPromptThreads / KP;           // threads that share a tile
  constexpr int kRows = kSide / 2;
  constexpr int kTileBytes = kTileKeys * DP * 2;
  constexpr int kLoads = kTileBytes / (16 * kSide);
  extern __shared__ __attribute__((aligned(16))) char s_tiles[];   // [KP][2][keys, values]
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int side = KP == 1 ? 0
                           : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kSide);
  const int tid = static_cast<int>(threadIdx.x) - side * kSide;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  lds_char* const tiles = (lds_char*)s_tiles + side * 4 * kTileBytes;
  const int col = lane & 31, half = lane >> 5;
  const PromptWork w = prompt_work(p);
  zero_rows<T>(p, w);
  int begin, length;
  sequence_rows(p, w.sequence, begin, length);
  const T* const query = static_cast<const T*>(p.query) + begin * p.query_row +
                         w.head * p.query_head;
  const T* const key = static_cast<const T*>(p.key) + begin * p.key_row + w.kv * p.key_head;
  const T* const value =
      static_cast<const T*>(p.value) + begin * p.value_row + w.kv * p.value_head;
  // where this thread's chunks of a tile come from, in bytes from its first row
  uint32_t key_from[kLoads], value_from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = i * kSide + tid;
    const int row = at / (DP / 8), c = place<DP>(row, at % (DP / 8));
    const bool inside = c * 8 < p.width;
    key_from[i] = inside ? row * static_cast<uint32_t>(p.key_row * 2) + c * 16 : 0x80000000u;
    value_from[i] = inside ? row * static_cast<uint32_t>(p.value_row * 2) + c * 16 : 0x80000000u;
  }
  auto load_tile = [&](int tile, int buffer) {
    const int first = tile * kTileKeys;
    const int rows = length - first < kTileKeys ? length - first : kTileKeys;
    lds_char* const to = tiles + buffer * 2 * kTileBytes + wave * kWave * 16;
    load_rows<kLoads, kSide>(key + first * p.key_row, rows, p.key_row, p.width, key_from, to);
    load_rows<kLoads, kSide>(value + first * p.value_row, rows, p.value_row, p.width,
                             value_from, to + kTileBytes);
  };
  // this lane's reads of a tile: keys by row col, values turned four keys of
  // 16 columns at a time
  int key_read[KS], value_read[DT][2];
#pragma unroll
  for (int s = 0; s < KS; ++s) key_read[s] = col * DP * 2 + place<DP>(col, 2 * s + half) * 16;
  {
    const int i = lane & 15, b = (lane >> 4) & 1;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 4 * half + 8 * e + i / 4;
        value_read[d][e] = row * DP * 2 + place<DP>(row, d * 4 + b * 2 + (i & 3) / 2) * 16 +
                           (i & 1) * 8;
      }
  }

  for (int block = w.block; block * kRows < length; block += p.blocks) {
    const int q0 = block * kRows + wave * 32;           // this wave's first row
    const int seen = (block + 1) * kRows < length ? (block + 1) * kRows : length;
    const int count = (seen + kTileKeys - 1) / kTileKeys;
    // a turn takes KP tiles, one for each side
    const int turns = (count + KP - 1) / KP;
    auto load_turn = [&](int turn, int buffer) {
      if (KP == 1 || turn * KP + side < count) load_tile(turn * KP + side, buffer);
    };
    auto arrived = [&](int turn, int buffer) {
      __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0): this thread's part has arrived
      __syncthreads();                         // everyone's; the other buffer is used
      if (turn + 1 < turns) load_turn(turn + 1, buffer ^ 1);
    };
    __syncthreads();            // the tiles of the block before are used
    load_turn(0, 0);
    Rows rows;
    {
      const int row = q0 + col;
      const T* const src = query + static_cast<int64_t>(row < length ? row : 0) * p.query_row;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = s * 16 + half * 8;
        rows.q[s] = d < p.width ? *reinterpret_cast<const vec*>(src + d) : vec{};
      }
    }
    rows.clear();
    // Tiles before the block's first row are seen by all of its rows; what
    // follows, to the diagonal, has a loop of its own.  The first go two turns
    // at a time, so that a buffer's address is part of the instructions.
    const int whole = block * (kRows / kTileKeys) / KP / 2 * 2;
    for (int turn = 0; turn < whole; turn += 2) {
#pragma unroll
      for (int buffer = 0; buffer < 2; ++buffer) {
        arrived(turn + buffer, buffer);
        const lds_char* const keys = tiles + buffer * 2 * kTileBytes;
        rows.template tile<PromptTile::kWhole>(keys, keys + kTileBytes, key_read, value_read,
                                               p.scale,
                                               ((turn + buffer) * KP + side) * kTileKeys, q0);
      }
    }
    auto edges = [&](auto kind, int from) {
#pragma unroll 1
      for (int turn = from; turn < turns; ++turn) {
        arrived(turn, turn & 1);
        const int tile = turn * KP + side, k0 = tile * kTileKeys;
        const lds_char* const keys = tiles + (turn & 1) * 2 * kTileBytes;
        if (tile < count && k0 <= q0 + 31 && q0 < length)
          rows.template tile<decltype(kind)::value>(keys, keys + kTileBytes, key_read,
                                                    value_read, p.scale, k0, q0);
      }
    };
    edges(std::integral_constant<PromptTile, PromptTile::kEdge>(), whole);
    // A value that is not finite, times the probability 0 of a row that does
    // not see it, is NaN.  Such values are rare and NaN stays in a sum: a
    // block that has one at its end is done again with care.
    if (__syncthreads_or(rows.any_nan())) {
      rows.clear();
      load_turn(0, 0);
      edges(std::integral_constant<PromptTile, PromptTile::kCareful>(), 0);
      if constexpr (KP == 1) __syncthreads();        // the last tiles are used
    }
    if constexpr (KP == 2) {
      using lds_float = typename Rows::lds_float;
      lds_float* const given = (lds_float*)s_tiles + wave * Rows::kFloats;
      __syncthreads();          // the last tiles are used
      if (side == 1) rows.give(given);
      __syncthreads();
      if (side == 1) continue;
      rows.join(given);
    }
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(rows.sum),
                                                    __float_as_uint(rows.sum), false, false);
    const float inverse = 1.0f / (__uint_as_float(x[0]) + __uint_as_float(x[1]));
    // The rows go out through LDS: as they are, a store would write 16 bytes
    // of each of 32 rows; so, it writes whole rows (24 packed prompts 308 us,
    // 325 without).
    // Its addresses are kept from being worked out before the loop, whose
    // registers they would take.
    int own = lane;
    asm volatile("" : "+v"(own));
    lds_char* const turned =
        (lds_char*)s_tiles + wave * (KP == 1 ? 32 * DP * 2 : Rows::kFloats * 4);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x16& a = rows.acc[d];
        const f32x4 x = f32x4{a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]} * inverse;
        *reinterpret_cast<__attribute__((address_space(3))) vec4*>(
            turned + own % 32 * DP * 2 + place<DP>(own % 32, d * 4 + i) * 16 + own / 32 * 8) =
            __builtin_convertvector(x, vec4);
      }
    wave_lds_sync();            // other lanes' columns
    T* const out = static_cast<T*>(p.out) +
                   ((static_cast<int64_t>(begin) + q0) * p.heads + w.head) * p.width;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int at = i * kWave + own, row = at / (DP / 8), c = at % (DP / 8);
      const vec x = *reinterpret_cast<const __attribute__((address_space(3))) vec*>(
          turned + row * DP * 2 + place<DP>(row, c) * 16);
      if (q0 + row < length && c * 8 < p.width)
        *reinterpret_cast<vec*>(out + static_cast<int64_t>(row) * p.heads * p.width + c * 8) = x;
    }
  }
}

// ----------------------------------------------------------------- float32

constexpr int float_keys(int padded) { return padded <= 64 ? 64 : padded <= 128 ? 32 : 16; }

// Float32 on the float32 matrix instructions: four waves of 16 query rows,
// 16 to 64 keys at a time through LDS.  A sixteenth of the 16-bit products'
// rate leaves the rest of the work small beside them; the next tile's loads
// pass registers while this one is used.  4 prompts of 2,048 tokens, 8 heads
// over 2, width 128: 365 us, 94 TFLOP/s of the 140 that a library's float32
// product reaches; 4 of 128, 4 heads of 32: 8 us, two tiles' round trips.
//
// KP = 2: 32 rows, of which two waves share 16; one takes the even and one the
// odd tiles, as in the 16-bit kernel.
template <int DP, int KP>
__global__ __launch_bounds__(kPromptThreads, DP <= 64 && KP == 1 ? 3 : 2) void prompt_float_kernel(
    PromptParams p) {
  constexpr int kSide = kPromptThreads / KP;           // threads that share a tile
  constexpr int kRows = kSide / 4;
  constexpr int kKeys = float_keys(DP);
  constexpr int KT = kKeys / 16;
  constexpr int KS = DP / 16;
  constexpr int DT = DP / 16;
  constexpr int kStride = DP + 4;      // rows of four apart fall on other banks
  constexpr int kLoads = kKeys * DP / 4 / kSide;
  extern __shared__ __attribute__((aligned(16))) char s_tiles[];
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int side = KP == 1 ? 0
                           : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kSide);
  const int tid = static_cast<int>(threadIdx.x) - side * kSide;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane & 15, quarter = lane >> 4;
  float* const s_key = reinterpret_cast<float*>(s_tiles) + side * 2 * kKeys * kStride;
  float* const s_value = s_key + kKeys * kStride;
  const PromptWork w = prompt_work(p);
  zero_rows<float>(p, w);
  int begin, length;
  sequence_rows(p, w.sequence, begin, length);
  const float* const query =
      static_cast<const float*>(p.query) + begin * p.query_row + w.head * p.query_head;
  const float* const key =
      static_cast<const float*>(p.key) + begin * p.key_row + w.kv * p.key_head;
  const float* const value =
      static_cast<const float*>(p.value) + begin * p.value_row + w.kv * p.value_head;

  for (int block = w.block; block * kRows < length; block += p.blocks) {
    const int q0 = block * kRows + wave * 16;
    const int row = q0 + col;
    const int seen = (block + 1) * kRows < length ? (block + 1) * kRows : length;
    f32x4 next_key[kLoads], next_value[kLoads];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = i * kSide + tid;
        const int r = k0 + at / (DP / 4), c = at % (DP / 4) * 4;
        const bool inside = r < length && c < p.width;
        const int64_t from = inside ? r : 0;
        const int column = inside ? c : 0;
        const f32x4 a = *reinterpret_cast<const f32x4*>(key + from * p.key_row + column);
        const f32x4 b = *reinterpret_cast<const f32x4*>(value + from * p.value_row + column);
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        next_key[i] = inside ? a : zero;
        next_value[i] = inside ? b : zero;
      }
    };
    f32x4 q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + quarter * 4;
      q[s] = d < p.width ? *reinterpret_cast<const f32x4*>(
                               query + static_cast<int64_t>(row < length ? row : 0) *
                                           p.query_row + d)
                         : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    f32x4 acc[DT];
    float most, sum;
    // careful: no value that is not finite reaches a row that does not see it
    auto run = [&](auto careful) {
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      most = kMinusInf;
      sum = 0.0f;
      fetch(side * kKeys);
      // a turn takes KP tiles, one for each side
      for (int first = 0; first < seen; first += KP * kKeys) {
        const int k0 = first + side * kKeys;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int at = i * kSide + tid;
          const int to = at / (DP / 4) * kStride + at % (DP / 4) * 4;
          *reinterpret_cast<f32x4*>(s_key + to) = next_key[i];
          *reinterpret_cast<f32x4*>(s_value + to) = next_value[i];
        }
        __syncthreads();
        if (k0 + KP * kKeys < seen) fetch(k0 + KP * kKeys);
        if (k0 >= seen || k0 > q0 + 15 || q0 >= length) continue;
        f32x4 s[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(s_key + (t * 16 + col) * kStride +
                                                            k * 16 + quarter * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], q[k][j], s[t], 0, 0, 0);
          }
        if (k0 + kKeys - 1 > q0) {
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (k0 + t * 16 + quarter * 4 + i > row) s[t][i] = kMinusInf;
        }
        float top = kMinusInf;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
        top = max_over_rows(top) * p.scale;
        if (__any(top > most)) {
          const float now = fmaxf(most, top);
          const float keep = now == kMinusInf ? 1.0f : exp2_fast(most - now);
          most = now;
          sum *= keep;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] *= keep;
        }
        const float shift = most == kMinusInf ? 0.0f : most;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] = exp2_fast(__builtin_fmaf(s[t][i], p.scale, -shift));
            sum += s[t][i];
          }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              float v = s_value[(t * 16 + quarter * 4 + i) * kStride + d * 16 + col];
              if constexpr (decltype(careful)::value) {
                const float sees = k0 + t * 16 + quarter * 4 + i <= row ? 1.0f : 0.0f;
                const float kind[3] = {v != v ? 1.0f : 0.0f,
                                       v == __builtin_huge_valf() ? 1.0f : 0.0f,
                                       v == kMinusInf ? 1.0f : 0.0f};
                if (!(__builtin_fabsf(v) < __builtin_huge_valf())) v = 0.0f;
#pragma unroll
                for (int n = 0; n < 3; ++n) {
                  f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
                  c = __builtin_amdgcn_mfma_f32_16x16x4f32(kind[n], sees, c, 0, 0, 0);
                  const float add = n == 0 ? __builtin_nanf("")
                                           : n == 1 ? __builtin_huge_valf() : kMinusInf;
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    if (c[j] > 0.0f) acc[d][j] += add;
                }
              }
              acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[t][i], acc[d], 0, 0, 0);
            }
      }
    };
    run(std::false_type());
    // as in the 16-bit kernel
    bool nan = false;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) nan |= acc[d][i] != acc[d][i];
    if (__syncthreads_or(nan)) run(std::true_type());
    sum = sum_over_rows(sum);
    if constexpr (KP == 2) {
      float* const given = reinterpret_cast<float*>(s_tiles) + wave * (DT * 4 + 2) * kWave + lane;
      __syncthreads();          // the last tiles are used
      if (side == 1) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) given[(d * 4 + i) * kWave] = acc[d][i];
        given[DT * 4 * kWave] = most;
        given[(DT * 4 + 1) * kWave] = sum;
      }
      __syncthreads();
      if (side == 1) continue;
      const float other = given[DT * 4 * kWave], now = fmaxf(most, other);
      const float mine = most == kMinusInf ? 0.0f : exp2_fast(most - now);
      const float theirs = other == kMinusInf ? 0.0f : exp2_fast(other - now);
      // a row whose logits are all -inf stays 0 / 0
      sum = sum * mine + given[(DT * 4 + 1) * kWave] * theirs;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[d][i] = acc[d][i] * mine + given[(d * 4 + i) * kWave] * theirs;
    }
    const float inverse = 1.0f / sum;
    if (row < length) {
      float* const out = static_cast<float*>(p.out) +
                         ((static_cast<int64_t>(begin) + row) * p.heads + w.head) * p.width;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int at = d * 16 + quarter * 4;
        if (at < p.width) *reinterpret_cast<f32x4*>(out + at) = acc[d] * inverse;
      }
    }
  }
}

// ---------------------------------------------------------------- launches

// A launch counts its threads in 32 bits.  Far below that it has workgroups
// enough: one that finds no rows takes 1.3 ns, and one that finds several
// blocks takes them in turn, so that a sequence gets no more than its share of
// 2^18, or 1,024 over all heads where that is more.  With 2^20 a prompt of
// 32,768 among 500 of 64, 32 heads of 128, takes 9.8 ms and 8.9 so (14.6 with
// a workgroup for every block); 256 prompts of 128, 64 heads of 64, whose
// longest is left out, 1.4 ms and 0.44 (0.20 where it is given).
constexpr int64_t kMostGroups = (int64_t{1} << 32) / kPromptThreads - 1;
constexpr int64_t kEnoughGroups = 1 << 18;

int32_t launch_prompt_kernel(void (*kernel)(PromptParams), int bytes, int rows, int64_t longest,
                             PromptParams p, hipStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(p.heads) * p.sequences;
  if (pairs > kMostGroups)
    return fail(COWSDM_ELIMIT, "prompt_attention: 2^24 pairs of a head and a sequence or more");
  const int64_t share = kEnoughGroups / pairs, least = (1024 + p.heads - 1) / p.heads;
  const int64_t held = kMostGroups / pairs;
  int64_t blocks = (longest + rows - 1) / rows, most = share > least ? share : least;
  most = most < held ? most : held;
  blocks = blocks < most ? blocks : most;
  p.blocks = static_cast<int32_t>(blocks);
  const int64_t grid = blocks * pairs;
  p.pair_by_pair = grid > 2048;        // four rounds of two workgroups a CU
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess)
      return fail(static_cast<int32_t>(e), "prompt_attention: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grid)), dim3(kPromptThreads), bytes,
                     stream, p);
  return launch_status("prompt_attention");
}

template <int DP>
int32_t launch_prompt_float(const PromptParams& p, int64_t longest, hipStream_t stream) {
  constexpr int kBytes = 2 * float_keys(DP) * (DP + 4) * 4;
  if constexpr (DP < 256) {      // whose registers would not hold another tile
    // Where 64 rows a workgroup leave a CU about one: 4 heads of 4,096 tokens
    // at width 32 take 81 us by 32 rows and 123 by 64, 8 heads of 1,000 at
    // width 64 40 and 56; or two of the narrowest, whose registers allow twice
    // as many (4 heads of 8,192: 211 and 288).  With more workgroups the
    // halves are in each other's way (8 heads of 12 prompts of up to 465: 68
    // and 64), and short rows lose by the join (4 prompts of 128: 11.0 and
    // 10.1; 8 of 256, 14 heads of 32: 17 and 14).
    const int64_t most = (static_cast<int64_t>(p.rows) / 64 + p.sequences) * p.heads;
    if ((most <= 288 && longest >= 4 * float_keys(DP)) ||
        (DP <= 32 && most <= 576 && longest >= 512))
      return launch_prompt_kernel(&prompt_float_kernel<DP, 2>, 2 * kBytes, 32, longest, p,
                                  stream);
  }
  return launch_prompt_kernel(&prompt_float_kernel<DP, 1>, kBytes, 64, longest, p, stream);
}

template <typename T, int DP>
int32_t launch_prompt_half(const PromptParams& p, int64_t longest, hipStream_t stream) {
  constexpr int kTiles = 2 * 2 * kTileKeys * DP * 2;
  if constexpr (DP <= 128) {
    // For grids that are small beside what the chip holds, by the LDS that
    // workgroups of 64 rows take.  The bounds are fitted, on the safe side: a
    // split that is not taken costs less than one too many.  At width 128,
    // where a CU holds one: 8 heads of 1,000 tokens take 19 us so and 22.5 by
    // 128 rows, 18 heads (the bound) 20 and 23, 24 heads 23.7 and 23.0; 16 heads
    // of 600 14.6 and 16.3, and past the bound 24 still 14.9 and 16.8; 4 heads
    // of 4,096 50 and 68, past it 8 heads 59 and 69, 16 heads 114 and 85.
    // Narrower: 8 of 4,096 at width 64 36 and 51, 8 of 8,192 at width 32 69 and
    // 89, 8 prompts of 600 with 8 heads of 32 11 and 12.5.  More workgroups
    // lose by their tiles' traffic (4 of 1,024, 12 heads of 64: 20 and 18; 8 of
    // 600, 8 heads of 64: 16 and 13.5; 2 of 550, 32 heads of 64: 15 and 12.5),
    // and shorter rows gain no more than the join takes (450 tokens, 8 heads of
    // 64: 10.4 and 11.2; 300: 10.4 and 10.5; 4 of 100: 10.9 and 10.8).
    const int64_t most = (static_cast<int64_t>(p.rows) / 64 + p.sequences) * p.heads;
    constexpr int kJoin = 2 * PromptRows<T, DP>::kFloats * 4;
    constexpr int kBytes = 2 * kTiles > kJoin ? 2 * kTiles : kJoin;
    constexpr int kHeld = 160 * 1024 / kBytes < 4 ? 160 * 1024 / kBytes : 4;   // by a CU
    if (most <= (longest >= 1000 ? 288 : 192) * kHeld && longest >= 512)
      return launch_prompt_kernel(&prompt_half_kernel<T, DP, 2>, kBytes, 64, longest, p, stream);
  }
  return launch_prompt_kernel(&prompt_half_kernel<T, DP, 1>, kTiles, 128, longest, p, stream);
}

template <typename T>
int32_t launch_prompt(const PromptParams& p, int64_t longest, hipStream_t stream) {
  const int w = p.width;
  if constexpr (sizeof(T) == 4) {
    if (w <= 32) return launch_prompt_float<32>(p, longest, stream);
    if (w <= 64) return launch_prompt_float<64>(p, longest, stream);
    if (w <= 96) return launch_prompt_float<96>(p, longest, stream);
    if (w <= 128) return launch_prompt_float<128>(p, longest, stream);
    if (w <= 192) return launch_prompt_float<192>(p, longest, stream);
    return launch_prompt_float<256>(p, longest, stream);
  } else {
    if (w <= 32) return launch_prompt_half<T, 32>(p, longest, stream);
    if (w <= 64) return launch_prompt_half<T, 64>(p, longest, stream);
    if (w <= 96) return launch_prompt_half<T, 96>(p, longest, stream);
    if (w <= 128) return launch_prompt_half<T, 128>(p, longest, stream);
    if (w <= 192) return launch_prompt_half<T, 192>(p, longest, stream);
    return launch_prompt_half<T, 256>(p, longest, stream);
  }
}

}  // namespace cowsdm_impl

using namespace cowsdm_impl;

extern "C" int32_t cowsdm_prompt_attention(const cowsdm_prompt_attention_t* attention,
                                           void* stream) {
  if (!attention) return fail(COWSDM_EARG, "prompt_attention: null argument");
  const cowsdm_prompt_attention_t& a = *attention;
  if (a.rows < 0 || a.sequences < 0 || a.longest < 0 || a.heads <= 0 || a.kv_heads <= 0)
    return fail(COWSDM_EARG, "prompt_attention: bad size");
  if (a.heads % a.kv_heads != 0)
    return fail(COWSDM_EARG, "prompt_attention: query heads must be a multiple of key heads");
  if (a.width <= 0 || a.width % 8 != 0)
    return fail(COWSDM_EARG, "prompt_attention: head width must be a multiple of 8");
  if (a.width > 256) return fail(COWSDM_ELIMIT, "prompt_attention: head width at most 256");
  if (a.rows > (1 << 30) || a.sequences > (1 << 30) || a.heads > (1 << 20) ||
      a.query_row >= (1 << 23) || a.key_row >= (1 << 23) || a.value_row >= (1 << 23))
    return fail(COWSDM_ELIMIT, "prompt_attention: too large");
  if (a.float_type != COWSDM_FLOAT32 && a.float_type != COWSDM_FLOAT16 &&
      a.float_type != COWSDM_BFLOAT16)
    return fail(COWSDM_EARG, "prompt_attention: bad float type");
  if (!(a.scale > 0.0f) || a.scale > 3.0e38f)
    return fail(COWSDM_EARG, "prompt_attention: the scale must be positive");
  if (a.rows == 0) return 0;
  if (a.sequences == 0) return fail(COWSDM_EARG, "prompt_attention: rows without a sequence");
  if (!a.query || !a.key || !a.value || !a.offsets || !a.out)
    return fail(COWSDM_EARG, "prompt_attention: null pointer argument");
  const int64_t unit = a.float_type == COWSDM_FLOAT32 ? 4 : 8;
  const int64_t strides[] = {a.query_row, a.query_head, a.key_row,
                             a.key_head,  a.value_row,  a.value_head};
  for (int64_t s : strides)
    if (s < 0 || s % unit != 0)
      return fail(COWSDM_EARG, "prompt_attention: strides must be multiples of 16 bytes");
  const void* pointers[] = {a.query, a.key, a.value, a.out};
  for (const void* x : pointers)
    if (reinterpret_cast<uintptr_t>(x) % 16 != 0)
      return fail(COWSDM_EARG, "prompt_attention: tensors must be 16-byte aligned");
  PromptParams p{};
  p.query = a.query;
  p.key = a.key;
  p.value = a.value;
  p.query_row = a.query_row;
  p.query_head = a.query_head;
  p.key_row = a.key_row;
  p.key_head = a.key_head;
  p.value_row = a.value_row;
  p.value_head = a.value_head;
  p.offsets = a.offsets;
  p.out = a.out;
  p.rows = static_cast<int32_t>(a.rows);
  p.sequences = static_cast<int32_t>(a.sequences);
  p.heads = static_cast<int32_t>(a.heads);
  p.kv_heads = static_cast<int32_t>(a.kv_heads);
  p.width = static_cast<int32_t>(a.width);
  p.scale = a.scale * kLog2E;
  const int64_t longest = a.longest < 1 ? 1 : a.longest < a.rows ? a.longest : a.rows;
  const auto s = static_cast<hipStream_t>(stream);
  if (a.float_type == COWSDM_FLOAT32) return launch_prompt<float>(p, longest, s);
  if (a.float_type == COWSDM_FLOAT16) return launch_prompt<_Float16>(p, longest, s);
  return launch_prompt<__bf16>(p, longest, s);
}
