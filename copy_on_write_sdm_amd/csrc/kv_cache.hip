// The paged K/V cache in 8 bits: page tables and token slots from the
// requests' lengths, release of pages, the write of keys and values, and the
// attention of each request's newest tokens over the cache.
//
// A page holds page_tokens tokens of one request: keys as [page, head, token,
// width] and values transposed, [page, head, width, token], so that the
// attention's two products both read 16 consecutive bytes a lane in the order
// the matrix instructions take them, straight into registers.  Codes are
// float8 e4m3; a page and head has one scale for its keys and one for its
// values, each a power of two: codes keep their bits when a scale grows (but
// for the smallest, which round), and code times scale is exact in bfloat16.

#include <type_traits>

#include "attention.h"

namespace cowsdm_impl {

// ------------------------------------------------------------ page tables

constexpr int kTableThreads = 256;
constexpr int kTableRequests = 4096;       // requests whose prefixes LDS holds
constexpr int kTableTokensPerBlock = 1024;

struct ExtendParams {
  const int32_t* lengths;
  const int32_t* added;
  int32_t* page_tables;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lengths_out;
  int32_t* free_count_out;
  int32_t* offsets;
  int32_t* positions;
  int32_t* slots;
  int32_t* overflow;
  int32_t requests;
  int32_t columns;
  int32_t pages;
  int32_t page_shift;
  int32_t tokens;
};

// Inclusive sum over the wave.
__device__ __forceinline__ int64_t wave_inclusive64(int64_t v) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t u = __shfl_up(v, o, kWave);
    if (lane >= o) v += u;
  }
  return v;
}

// Exclusive sum of v over the workgroup's threads and, in `total`, the sum.
__device__ __forceinline__ int64_t block_exclusive64(int64_t v, int64_t* parts, int64_t& total) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = static_cast<int>(threadIdx.x) / kWave;
  const int64_t in = wave_inclusive64(v);
  __syncthreads();
  if (lane == kWave - 1) parts[wave] = in;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kTableThreads / kWave; ++w) {
    if (w < wave) before += parts[w];
    total += parts[w];
  }
  return before + in - v;
}

// One launch: every workgroup sums the requests' new pages and new tokens
// itself (a few kilobytes, from L2), and then writes its share of the tokens'
// positions and slots.  A request's page j past those it holds is the free
// stack's entry count - 1 - (new pages of the requests before it + j): pops in
// request order, whichever workgroup needs them, with no word exchanged
// between workgroups.  The token that opens a page writes its table entry.
//
// A call's dependent memory round trips bound it: 3.1 us for a token each of
// 64 requests, 9.6 us for 528,000 tokens of 512 (4.4 MB; the sums over the
// requests are most of that, and no more than the host's part of a call).
__global__ __launch_bounds__(kTableThreads) void extend_tables_kernel(ExtendParams p) {
  __shared__ int32_t s_start[kTableRequests];
  __shared__ int32_t s_pages[kTableRequests];   // new pages before the request, less those it holds
  __shared__ int64_t s_parts[2][kTableThreads / kWave];
  __shared__ int32_t s_bad;
  const int tid = static_cast<int>(threadIdx.x);
  const int page = 1 << p.page_shift;
  const bool first = blockIdx.x == 0;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  int64_t tokens = 0, pages = 0;
  for (int at = 0; at < p.requests; at += kTableThreads) {
    const int r = at + tid;
    int64_t n = 0, more = 0, held = 0, need = 0;
    if (r < p.requests) {
      n = p.lengths[r];
      more = p.added[r];
      const int64_t want = (n + more + page - 1) >> p.page_shift;
      held = (n + page - 1) >> p.page_shift;
      if (n < 0 || more < 0 || want > p.columns) {
        atomicOr(&s_bad, 1);
        more = 0;
      } else {
        need = want - held;
      }
    }
    int64_t token_sum, page_sum;
    const int64_t t0 = tokens + block_exclusive64(more, s_parts[0], token_sum);
    const int64_t p0 = pages + block_exclusive64(need, s_parts[1], page_sum);
    if (r < p.requests) {
      s_start[r] = static_cast<int32_t>(t0 < INT32_MAX ? t0 : INT32_MAX);
      s_pages[r] = static_cast<int32_t>(p0 - held);
      if (first) p.offsets[r] = s_start[r];
    }
    tokens += token_sum;
    pages += page_sum;
  }
  __syncthreads();
  const int32_t count = *p.free_count;
  const bool fits = !s_bad && pages <= count && count <= p.pages && tokens <= p.tokens;
  if (first) {
    for (int r = tid; r < p.requests; r += kTableThreads)
      p.lengths_out[r] = p.lengths[r] + (fits ? p.added[r] : 0);
    if (tid == 0) {
      p.offsets[p.requests] = static_cast<int32_t>(tokens < INT32_MAX ? tokens : INT32_MAX);
      *p.free_count_out = fits ? count - static_cast<int32_t>(pages) : count;
      *p.overflow = fits ? 0 : 1;
    }
  }
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * kTableTokensPerBlock;
  for (int64_t t = begin + tid; t < begin + kTableTokensPerBlock && t < p.tokens;
       t += kTableThreads) {
    int32_t position = -1, slot = -1;
    if (fits && t < tokens) {
      // the last request that starts at t or before it: requests without new
      // tokens start where the next one does
      int lo = 0, hi = p.requests - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= t) lo = mid; else hi = mid - 1;
      }
      const int32_t n = p.lengths[lo];
      position = n + static_cast<int32_t>(t - s_start[lo]);
      const int32_t column = position >> p.page_shift;
      const int32_t held = (n + page - 1) >> p.page_shift;
      int32_t* const entry = p.page_tables + static_cast<int64_t>(lo) * p.columns + column;
      int32_t id;
      if (column < held) {
        id = *entry;
      } else {
        id = p.free_pages[count - 1 - (s_pages[lo] + column)];
        if ((position & (page - 1)) == 0) *entry = id;
      }
      // an entry that is no page of the pool gives a slot that is none either
      if (id >= 0 && id <= (INT32_MAX >> p.page_shift))
        slot = (id << p.page_shift) + (position & (page - 1));
    }
    p.positions[t] = position;
    p.slots[t] = slot;
  }
}

// The pages of the named requests go back to the top of the free stack, in
// the order of the list; one workgroup, and a request's pages one after another
// in a thread: 64 requests of 40 pages 45 us, 4 of 8,192 pages 1,180.
__global__ __launch_bounds__(kTableThreads) void release_pages_kernel(
    int32_t* lengths, int32_t* page_tables, int32_t columns, const int32_t* named, int32_t n,
    int32_t requests, int32_t* free_pages, int32_t pages, int32_t* free_count, int page_shift) {
  __shared__ int64_t s_parts[kTableThreads / kWave];
  const int tid = static_cast<int>(threadIdx.x);
  int64_t top = *free_count;
  for (int at = 0; at < n; at += kTableThreads) {
    const int r = at + tid < n ? named[at + tid] : -1;
    int64_t held = 0;
    if (r >= 0 && r < requests) {
      held = (static_cast<int64_t>(lengths[r]) + (1 << page_shift) - 1) >> page_shift;
      held = held < 0 ? 0 : held > columns ? columns : held;
    }
    int64_t sum;
    const int64_t before = top + block_exclusive64(held, s_parts, sum);
    for (int64_t j = 0; j < held; ++j) {
      int32_t* const entry = page_tables + static_cast<int64_t>(r) * columns + j;
      if (before + j >= 0 && before + j < pages) free_pages[before + j] = *entry;
      *entry = -1;
    }
    if (held > 0) lengths[r] = 0;
    top += sum;
  }
  __syncthreads();
  if (tid == 0) *free_count = static_cast<int32_t>(top < pages ? top : pages);
}

// ------------------------------------------------------------------ write

constexpr int kWriteThreads = 256;

struct WriteParams {
  const void* key;
  const void* value;
  int64_t key_row, key_head;       // strides, in elements
  int64_t value_row, value_head;
  const int32_t* slots;
  uint8_t* key_codes;
  float* key_scales;
  uint8_t* value_codes;
  float* value_scales;
  int32_t tokens;
  int32_t heads;
  int32_t width;
  int32_t pages;
  int32_t page_shift;
  int32_t chunk;                   // tokens whose runs one workgroup writes
};

// The least power of two, from 2^-100 to 2^119, by which `most` is at most
// 448 = 1.75 * 2^8.  The bounds keep the scale, its inverse and every code
// times it normal numbers.
__device__ __forceinline__ float power_scale(float most) {
  const uint32_t bits = __float_as_uint(most);
  int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -100 ? -100 : e > 119 ? 119 : e;
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ float power_inverse(float scale) {
  return __uint_as_float((254u << 23) - __float_as_uint(scale));
}

// What is not finite has no code but NaN: the format has no infinity.
__device__ __forceinline__ float code_value(float x, float inverse) {
  const float y = fminf(fmaxf(x * inverse, -kMostCode), kMostCode);
  return __builtin_fabsf(x) < __builtin_huge_valf() ? y : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// Codes under the scale `old` (ratio = old / new, below 1) under the new one.
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float ratio) {
  float x[4];
  x[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0);
  x[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1);
  x[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2);
  x[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3);
  return encode4(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < __builtin_huge_valf() ? a : 0.0f;
}

// Eight elements as loaded: kept packed until they are used.
template <typename T>
struct Eight {
  u32x4 raw[sizeof(T) / 2];
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(raw[j / 4][j % 4]);
    } else {
      const uint32_t pair = raw[0][j / 2];
      return widen_float(j % 2 ? pair >> 16 : pair & 0xffffu,
                         std::is_same<T, __bf16>::value ? COWSDM_BFLOAT16 : COWSDM_FLOAT16);
    }
  }
};

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    e.raw[i] = reinterpret_cast<const u32x4*>(p)[i];
  return e;
}

// Keeps the compiler from holding the elements widened from one use to the
// next: the packed words are half the registers.
template <typename T>
__device__ __forceinline__ void stay_packed(Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t word = e.raw[i][j];
      asm volatile("" : "+v"(word));
      e.raw[i][j] = word;
    }
}

template <typename T>
__device__ __forceinline__ float largest(const Eight<T>& e, float most) {
#pragma unroll
  for (int j = 0; j < 8; ++j) most = fmaxf(most, finite_abs(e[j]));
  return most;
}

// What a workgroup writes: one run of tokens in one page and head.
template <typename T>
struct WriteRun {
  const T* key;          // the run's first row
  const T* value;
  int64_t key_row, value_row;
  uint8_t* kc;           // the page's codes
  uint8_t* vc;
  int columns, wide;     // eights of a row's elements, and of its codes
  int page, first, run;  // tokens of the page, before the run, and of the run

  // Eight elements of key row r; zeros in the padding.
  __device__ __forceinline__ Eight<T> key_at(int r, int c) const {
    return c < columns ? load_eight(key + r * key_row + c * 8) : Eight<T>{};
  }
  __device__ __forceinline__ void put_key(int r, int c, const Eight<T>& e, float inverse) const {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = code_value(e[j], inverse);
    *reinterpret_cast<u32x2*>(kc + (static_cast<int64_t>(first + r) * wide + c) * 8) =
        u32x2{encode4(x[0], x[1], x[2], x[3]), encode4(x[4], x[5], x[6], x[7])};
  }
  // Of the page's four tokens from 4 g on: eight columns of those of the run,
  // and in the result their bytes.
  __device__ __forceinline__ uint32_t values_at(int g, int c, Eight<T> (&e)[4]) const {
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = 4 * g + k - first;
      const bool in = r >= 0 && r < run;
      mine |= in ? 0xffu << (8 * k) : 0u;
      e[k] = in && c < columns ? load_eight(value + r * value_row + c * 8) : Eight<T>{};
    }
    return mine;
  }
  __device__ __forceinline__ uint32_t* value_word(int g, int column) const {
    return reinterpret_cast<uint32_t*>(vc + static_cast<int64_t>(column) * page) + g;
  }
  __device__ __forceinline__ uint32_t value_codes(const Eight<T> (&e)[4], int j,
                                                  float inverse) const {
    return encode4(code_value(e[0][j], inverse),
                   code_value(e[1][j], inverse),
                   code_value(e[2][j], inverse),
                   code_value(e[3][j], inverse));
  }
};

constexpr int kWriteKeys = 4;        // eights of keys that a thread holds

// By the whole workgroup.  Held: a page has at most 8,192 elements (64 tokens
// at width 128), and a run's stay in registers between the maximum and the
// codes; else they are read twice, the second time from cache.
template <typename T, bool kHeld>
__device__ __forceinline__ void write_run(const WriteRun<T>& w, float* key_scale, float* value_scale,
                          float* s_most) {
  const int tid = static_cast<int>(threadIdx.x);
  const int wave = tid / kWave;
  const int g0 = w.first / 4, groups = (w.first + w.run + 3) / 4 - g0;
  const int keys = w.run * w.wide, values = groups * w.wide;
  const int vg = g0 + tid % groups, vcol = tid / groups;
  Eight<T> k[kWriteKeys] = {}, v[4] = {};
  uint32_t mine = 0, other[8] = {};
  float km = 0.0f, vm = 0.0f;
  const float k_old = w.first ? *key_scale : 0.0f;
  const float v_old = w.first ? *value_scale : 0.0f;
  if constexpr (kHeld) {
#pragma unroll
    for (int n = 0; n < kWriteKeys; ++n) {
      const int i = tid + n * kWriteThreads;
      if (i < keys) k[n] = w.key_at(i / w.wide, i % w.wide);
    }
    if (tid < values) {
      mine = w.values_at(vg, vcol, v);
      if (mine != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) other[j] = *w.value_word(vg, vcol * 8 + j);
      }
    }
#pragma unroll
    for (int n = 0; n < kWriteKeys; ++n)
      if (tid + n * kWriteThreads < keys) km = largest(k[n], km);
    if (tid < values) {
#pragma unroll
      for (int n = 0; n < 4; ++n) vm = largest(v[n], vm);
    }
  } else {
    for (int i = tid; i < w.run * w.columns; i += kWriteThreads) {
      const int r = i / w.columns, c = (i - r * w.columns) * 8;
      km = largest(load_eight(w.key + r * w.key_row + c), km);
      vm = largest(load_eight(w.value + r * w.value_row + c), vm);
    }
  }
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    km = fmaxf(km, __shfl_xor(km, o, kWave));
    vm = fmaxf(vm, __shfl_xor(vm, o, kWave));
  }
  if ((tid & (kWave - 1)) == 0) {
    s_most[2 * wave] = km;
    s_most[2 * wave + 1] = vm;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kWriteThreads / kWave; ++n) {
    km = fmaxf(km, s_most[2 * n]);
    vm = fmaxf(vm, s_most[2 * n + 1]);
  }
  if constexpr (kHeld && sizeof(T) == 2) {
#pragma unroll
    for (int n = 0; n < kWriteKeys; ++n) stay_packed(k[n]);
#pragma unroll
    for (int n = 0; n < 4; ++n) stay_packed(v[n]);
  }
  const float k_scale = fmaxf(power_scale(km), k_old), ki = power_inverse(k_scale);
  const float v_scale = fmaxf(power_scale(vm), v_old), vi = power_inverse(v_scale);
  if (tid == 0) {
    *key_scale = k_scale;
    *value_scale = v_scale;
  }
  const bool k_grew = w.first && k_scale > k_old, v_grew = w.first && v_scale > v_old;
  const float k_ratio = k_old * ki, v_ratio = v_old * vi;
  if constexpr (kHeld) {
#pragma unroll
    for (int n = 0; n < kWriteKeys; ++n) {
      const int i = tid + n * kWriteThreads;
      if (i < keys) w.put_key(i / w.wide, i % w.wide, k[n], ki);
    }
    if (tid < values) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t kept = v_grew ? rescale4(other[j], v_ratio) : other[j];
        *w.value_word(vg, vcol * 8 + j) = (w.value_codes(v, j, vi) & mine) | (kept & ~mine);
      }
    }
  } else {
    for (int i = tid; i < keys; i += kWriteThreads)
      w.put_key(i / w.wide, i % w.wide, w.key_at(i / w.wide, i % w.wide), ki);
    for (int i = tid; i < values; i += kWriteThreads) {
      const int g = g0 + i % groups, c = i / groups;
      mine = w.values_at(g, c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t* const word = w.value_word(g, c * 8 + j);
        uint32_t codes = w.value_codes(v, j, vi);
        if (mine != 0xffffffffu) {
          const uint32_t kept = v_grew ? rescale4(*word, v_ratio) : *word;
          codes = (codes & mine) | (kept & ~mine);
        }
        *word = codes;
      }
    }
  }
  // a grown scale takes the page's other codes along: the other rows of keys,
  // and the groups of values outside the run
  if (k_grew) {
    const int row = w.wide * 2;
    for (int i = tid; i < (w.page - w.run) * row; i += kWriteThreads) {
      uint32_t* const word =
          reinterpret_cast<uint32_t*>(w.kc) + (i < w.first * row ? i : i + w.run * row);
      *word = rescale4(*word, k_ratio);
    }
  }
  if (v_grew) {
    const int rest = w.page / 4 - groups;
    for (int i = tid; i < rest * w.wide * 8; i += kWriteThreads) {
      const int g = i % rest;
      uint32_t* const word = w.value_word(g < g0 ? g : g + groups, i / rest);
      *word = rescale4(*word, v_ratio);
    }
  }
  __syncthreads();      // s_most is free for the next run
}

// A run is a stretch of the call's tokens whose slots follow one another in
// one page; the workgroup of its first token's chunk (at most 64 tokens)
// writes it, for one head.  The page's scale needs the whole run's maximum
// before the first code, so that a page and head is the unit of work.
//
// Memory bounds large calls: 45,960 tokens of 8 heads by 128 in bfloat16, 282
// MB read and written, take 64 us, 4.4 TB/s (a copy reaches 5.1); with the
// rows read twice they took 133.  Single tokens take 6.5 us: the slot, the
// rows with the page's scales and words, the maximum across the workgroup, the
// stores.
template <typename T, bool kHeld>
__global__ __launch_bounds__(kWriteThreads) void kv_write_kernel(WriteParams p, int width) {
  __shared__ float s_most[2 * kWriteThreads / kWave];
  __shared__ int s_run;
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & (kWave - 1);
  const int head = blockIdx.y;
  const int page = 1 << p.page_shift;
  const int64_t limit = static_cast<int64_t>(p.pages) << p.page_shift;
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.chunk;
  // every wave finds the chunk's first tokens of runs
  const int64_t mine = begin + lane;
  int slot = -1;
  bool opens = false;
  if (lane < p.chunk && mine < p.tokens) {
    slot = p.slots[mine];
    opens = slot >= 0 && slot < limit &&
            ((slot & (page - 1)) == 0 || mine == 0 || p.slots[mine - 1] != slot - 1);
  }
  for (uint64_t runs = __ballot(opens); runs; runs &= runs - 1) {
    const int from = __builtin_ctzll(runs);
    const int t = static_cast<int>(begin) + from;
    const int at = __builtin_amdgcn_readlane(slot, from);
    const int first = at & (page - 1);
    // the run ends before the first of the page's next slots that is not the
    // next token's
    if (tid == 0) s_run = page - first;
    __syncthreads();
    const int i = tid + 1;
    if (i < page - first && (t + i >= p.tokens || p.slots[t + i] != at + i))
      atomicMin(&s_run, i);
    __syncthreads();
    const int64_t block = static_cast<int64_t>(at >> p.page_shift) * p.heads + head;
    WriteRun<T> w;
    w.key = static_cast<const T*>(p.key) + t * p.key_row + head * p.key_head;
    w.value = static_cast<const T*>(p.value) + t * p.value_row + head * p.value_head;
    w.key_row = p.key_row;
    w.value_row = p.value_row;
    w.kc = p.key_codes + block * page * width;
    w.vc = p.value_codes + block * page * width;
    w.columns = p.width / 8;
    w.wide = width / 8;
    w.page = page;
    w.first = first;
    w.run = s_run;
    write_run<T, kHeld>(w, p.key_scales + block, p.value_scales + block, s_most);
  }
}

template <typename T>
void launch_write(const WriteParams& p, dim3 grid, int width, hipStream_t stream) {
  const bool held = (width << p.page_shift) <= 8 * kWriteKeys * kWriteThreads;
  hipLaunchKernelGGL((held ? &kv_write_kernel<T, true> : &kv_write_kernel<T, false>), grid,
                     dim3(kWriteThreads), 0, stream, p, width);
}

// ------------------------------------------------------- cached attention

constexpr int kCachedTokens = 64;         // tokens a wave takes at a time
constexpr int kCachedRows = 16;           // query rows of a workgroup

struct CachedParams {
  const void* query;
  int64_t query_request, query_token, query_head;   // strides, in elements
  const uint8_t* key_codes;
  const float* key_scales;
  const uint8_t* value_codes;
  const float* value_scales;
  const int32_t* page_tables;
  const int32_t* lengths;
  void* out;                       // [requests, tokens, heads, width]
  float* parts;                    // split: [request, kv head, row tile, split] blocks, or null
  float scale;                     // of the logits, times log2(e)
  int32_t requests;
  int32_t tokens;
  int32_t heads;
  int32_t kv_heads;
  int32_t width;
  int32_t pages;
  int32_t columns;
  int32_t page_shift;
  int32_t chunk;                   // tokens of a split
  int32_t splits;
  int32_t row_tiles;
  int32_t by_length;               // the longest requests come first
};

// A split's block: the 16 rows' largest logits and sums, then their products
// [row][width].
template <int DP>
constexpr int kPartFloats = 2 * kCachedRows + kCachedRows * DP;

typedef const __attribute__((address_space(4))) int32_t* const_int32;

// Number g of four, without a table in memory.
__device__ __forceinline__ int pick4(int g, int a, int b, int c, int d) {
  const int low = (g & 1) ? b : a, high = (g & 1) ? d : c;
  return (g & 2) ? high : low;
}

// A block of 64 tokens as a lane holds it: its quarter of four key rows, 16
// tokens of each of its value columns, and their scales.
template <int DP>
struct Fetched {
  uint32_t kw[4][DP / 16];
  u32x4 vw[DP / 16];
  float ks, vs;
  int base, v_page;
};

// A request's tokens, at most what its page table can hold.
__device__ __forceinline__ int cached_length(const CachedParams& p, int request) {
  const int n = ((const_int32)p.lengths)[request], most = p.columns << p.page_shift;
  return n < 0 ? 0 : n < most ? n : most;
}

// One workgroup: 16 query rows (the tokens and grouped heads of one key head)
// over one split of the cache.  Its NW waves take blocks of 64 tokens in
// turn, the next on its way while one is used.
//
// Scores are computed transposed, S^T = K Q^T, so that a lane ends
// with 16 consecutive tokens of one query row: its probabilities are then the
// right operand of O^T = V^T P^T as they stand, and no score leaves its
// registers.  Key row m of tile t is token (m / 4) * 16 + 4 t + m % 4.
//
// Memory bounds it: two requests of 131,072 tokens, 8 key heads of 128,
// bfloat16, 75 us, 5.6 TB/s.  In float32 at width 128 its 256 registers are
// three words short (12 bytes of scratch a lane): 64 requests of up to 2,560
// tokens take 42 us so, 39 in bfloat16.
template <int DP, typename T, int NW>
__global__ __launch_bounds__(NW * kWave) void cached_attention_kernel(CachedParams p) {
  constexpr int N = AttentionType<T>::kParts;
  constexpr int NP = AttentionType<T>::kProbParts;
  constexpr int KB = DP / 4;            // a lane's bytes of a key row
  constexpr int KS = DP / 32;           // products along the width
  constexpr int DT = DP / 16;           // tiles of the output's width
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave =
      __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int col = lane & 15, row = lane >> 4;
  const int split = blockIdx.x % p.splits;
  const int tile = blockIdx.x / p.splits;
  const int kv = blockIdx.y;
  const int page = 1 << p.page_shift;
  const int group = p.heads / p.kv_heads;
  int request = blockIdx.z, length;
  if (p.by_length) {
    // More workgroups than the chip holds at once: the longest requests come
    // first, so that short ones fill what they leave (64 requests of up to
    // 2,560 tokens, 8 key heads: 43 us, in their own order 46.5).
    const int n = lane < p.requests ? p.lengths[lane] : 0, most = p.columns << p.page_shift;
    const int mine = n < 0 ? 0 : n < most ? n : most;
    request = lane_by_size(mine, p.requests, blockIdx.z);
    length = __builtin_amdgcn_readlane(mine, request);
  } else {
    length = cached_length(p, request);
  }
  const int begin = split * p.chunk;
  if (begin >= length && split > 0) return;
  // the last split takes what a longest length given too short leaves
  const int end = split == p.splits - 1 || length < begin + p.chunk ? length : begin + p.chunk;

  // this lane's query row and the last position that it sees
  const int query_row = tile * kCachedRows + col;
  const bool is_row = query_row < p.tokens * group;
  const int token = is_row ? query_row / group : 0;
  const int head = kv * group + (is_row ? query_row - token * group : 0);
  const int last = is_row ? length - p.tokens + token : -1;
  bf16x8 q[KS][N];
  {
    const T* const src = static_cast<const T*>(p.query) + request * p.query_request +
                         token * p.query_token + head * p.query_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8] = {};
      const int d = row * KB + s * 8;
      if (is_row && d < p.width) load8(src + d, x);
      split_bf16<N>(x, q[s]);
    }
  }

  const const_int32 table =
      (const_int32)(p.page_tables + static_cast<int64_t>(request) * p.columns);
  const int64_t page_bytes = static_cast<int64_t>(page) * DP;
  // a lane's bytes of a block's keys and values, on their way
  auto fetch = [&](int base, Fetched<DP>& f) {
    // the page of the block's tokens 16 g on; columns of tokens before the
    // length are below the table's
    auto page_of = [&](int g) {
      const int column = (base + 16 * g) >> p.page_shift;
      const int id = table[column < p.columns ? column : p.columns - 1];
      return base + 16 * g < end && id >= 0 && id < p.pages ? id : -1;
    };
    const int id0 = page_of(0), id1 = page_of(1), id2 = page_of(2), id3 = page_of(3);
    const int k_page = pick4(col >> 2, id0, id1, id2, id3);
    const int v_page = pick4(row, id0, id1, id2, id3);
    const int k_at = base + (col >> 2) * 16, v_at = base + row * 16;
    const int64_t k_block = static_cast<int64_t>(k_page < 0 ? 0 : k_page) * p.kv_heads + kv;
    const int64_t v_block = static_cast<int64_t>(v_page < 0 ? 0 : v_page) * p.kv_heads + kv;
    const uint8_t* const kp = p.key_codes + k_block * page_bytes +
                              static_cast<int64_t>((k_at & (page - 1)) + (col & 3)) * DP +
                              row * KB;
    const uint8_t* const vp = p.value_codes + v_block * page_bytes +
                              static_cast<int64_t>(col) * page + (v_at & (page - 1));
    f.base = base;
    f.v_page = v_page;
    f.ks = p.key_scales[k_block];
    f.vs = p.value_scales[v_block];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t* const src = kp + t * 4 * DP;
      if constexpr (KB % 16 == 0) {
#pragma unroll
        for (int i = 0; i < KB / 16; ++i)
          *reinterpret_cast<u32x4*>(&f.kw[t][4 * i]) =
              *reinterpret_cast<const u32x4*>(src + 16 * i);
      } else {
#pragma unroll
        for (int i = 0; i < KB / 8; ++i)
          *reinterpret_cast<u32x2*>(&f.kw[t][2 * i]) =
              *reinterpret_cast<const u32x2*>(src + 8 * i);
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
      f.vw[d] = *reinterpret_cast<const u32x4*>(vp + static_cast<int64_t>(d) * 16 * page);
  };

  f32x4 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float most = kMinusInf, sum = 0.0f;     // of logits times scale
  auto use = [&](Fetched<DP>& f) {
    const int base = f.base, v_page = f.v_page, v_at = base + row * 16;
    const float ks = f.ks;
    float vs = f.vs;
    auto& kw = f.kw;
    auto& vw = f.vw;
    f32x4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const bf16x8 a = widen_codes(kw[t][2 * k], kw[t][2 * k + 1], ks);
#pragma unroll
        for (int n = N - 1; n >= 0; --n)
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[k][n], s[t], 0, 0, 0);
      }
    }
    // a block is masked only past the first query token's last position, or
    // where a page is missing
    const bool tail = base + kCachedTokens > length - p.tokens + 1;
    const bool masked = tail || __any(v_page < 0);
    // a row that sees a token has a finite maximum, were its logits all -inf;
    // one that has seen none keeps -inf, and gives 0
    float least = kLeastFloat;
    if (masked) {
      least = v_page < 0 || v_at > last ? kMinusInf : kLeastFloat;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v_page < 0 || v_at + 4 * t + i > last) s[t][i] = kMinusInf;
      // codes of tokens past the length are whatever the page held before;
      // where there is no page, the scale is one that nobody may have written
      const int keep = v_page < 0 ? 0 : length - v_at;
      if (v_page < 0) vs = 1.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = keep - 4 * i;
        const uint32_t mask = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
#pragma unroll
        for (int d = 0; d < DT; ++d) vw[d][i] &= mask;
      }
    }
    float top = kMinusInf;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
    top = max_over_rows(fmaxf(top * p.scale, least));
    if (__any(top > most)) {
      const float now = fmaxf(most, top);
      const float keep = now == kMinusInf ? 1.0f : exp2_fast(most - now);
      most = now;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= keep;
    }
    const float shift = most == kMinusInf ? 0.0f : most;
    float pr[16];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = exp2_fast(__builtin_fmaf(s[t][i], p.scale, -shift));
        pr[4 * t + i] = e;
        sum += e;
      }
    bf16x8 prob[2][NP];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = pr[8 * h + j];
      split_bf16<NP>(x, prob[h]);
    }
    uint32_t poisoned = 0;
    if (masked && p.tokens > 1) {
      // a NaN that only some of the rows see: it must not reach the others
      // through a product with 0
      uint32_t any = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = vw[d][i] & 0x7f7f7f7fu;
          any |= (w + 0x01010101u) & 0x80808080u;
        }
      poisoned = __any(any != 0) ? 1u : 0u;
    }
    if (poisoned) {
      for (int t = 0; t < kCachedTokens; ++t) {
        const int pos = base + t;
        const int word = (t & 15) >> 2, shift8 = 8 * (t & 3);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const uint32_t w = word == 0 ? vw[d][0] : word == 1 ? vw[d][1] : word == 2 ? vw[d][2]
                                                                                 : vw[d][3];
          const int nan = ((w >> shift8) & 0x7fu) == 0x7fu;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (__shfl(nan, (t >> 4) * 16 + row * 4 + i, kWave) && pos <= last)
              acc[d][i] = __uint_as_float(0x7fc00000u);
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (((vw[d][i] >> (8 * b)) & 0x7fu) == 0x7fu) vw[d][i] &= ~(0xffu << (8 * b));
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x8 a = widen_codes(vw[d][2 * h], vw[d][2 * h + 1], vs);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n)
          acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, prob[h][n], acc[d], 0, 0, 0);
      }
    }
  };

  int base = begin + wave * kCachedTokens;
  constexpr int kStep = NW * kCachedTokens;
  if constexpr (DP < 256) {
    // Two blocks in turn.  Past its last block a wave fetches that one again
    // (from cache) and does not use it: a branch there would make every use
    // wait for all that is on its way.
    if (base < end) {
      Fetched<DP> one, two;
      fetch(base, one);
      for (;;) {
        fetch(base + kStep < end ? base + kStep : base, two);
        use(one);
        base += kStep;
        if (base >= end) break;
        fetch(base + kStep < end ? base + kStep : base, one);
        use(two);
        base += kStep;
        if (base >= end) break;
      }
    }
  } else {
    // two blocks of the widest rows do not fit the registers
    for (; base < end; base += kStep) {
      Fetched<DP> one;
      fetch(base, one);
      use(one);
    }
  }
  sum = sum_over_rows(sum);

  // the waves' parts, joined pairwise in a fixed order
  __shared__ __attribute__((aligned(16))) float s_part[NW / 2][DT + 1][kWave * 4];
#pragma unroll
  for (int half = NW / 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
        *reinterpret_cast<f32x4*>(&s_part[wave - half][d][lane * 4]) = acc[d];
      s_part[wave - half][DT][lane * 2] = most;
      s_part[wave - half][DT][lane * 2 + 1] = sum;
    }
    __syncthreads();
    if (wave < half) {
      const float other = s_part[wave][DT][lane * 2];
      const float now = fmaxf(most, other);
      const float a = now == kMinusInf ? 1.0f : exp2_fast(most - now);
      const float b = now == kMinusInf ? 1.0f : exp2_fast(other - now);
      most = now;
      sum = sum * a + s_part[wave][DT][lane * 2 + 1] * b;
#pragma unroll
      for (int d = 0; d < DT; ++d)
        acc[d] = acc[d] * a + *reinterpret_cast<const f32x4*>(&s_part[wave][d][lane * 4]) * b;
    }
    __syncthreads();
  }
  if (wave != 0 || !is_row) return;
  if (p.parts) {
    const int64_t at =
        ((static_cast<int64_t>(request) * p.kv_heads + kv) * p.row_tiles + tile) * p.splits +
        split;
    float* const part = p.parts + at * kPartFloats<DP>;
    if (row == 0) {
      part[col] = most;
      part[kCachedRows + col] = sum;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f32x4*>(part + 2 * kCachedRows + col * DP + d * 16 + row * 4) = acc[d];
    return;
  }
  T* const out = static_cast<T*>(p.out) +
                 ((static_cast<int64_t>(request) * p.tokens + token) * p.heads + head) * p.width;
  const float inverse = 1.0f / sum;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const int at = d * 16 + row * 4;
    if (at < p.width)
      store4(out + at, most == kMinusInf ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc[d] * inverse);
  }
}

// Joins the splits of one query row: every group of DP / 4 lanes takes every
// so many splits, and the groups' sums are added in their order, so that the
// result does not hang on which split ends first.  4 to 5 us, two dependent
// reads; one split after the other in a wave took 13 to 48.
constexpr int kJoinThreads = 256;

template <int DP, typename T>
__global__ __launch_bounds__(kJoinThreads) void cached_join_kernel(CachedParams p) {
  constexpr int kLanes = DP / 4;
  constexpr int kGroups = kJoinThreads / kLanes;
  __shared__ __attribute__((aligned(16))) float s_sum[kGroups][DP + 4];
  __shared__ float s_most[kJoinThreads / kWave];
  const int tid = static_cast<int>(threadIdx.x);
  const int group = p.heads / p.kv_heads;
  const int head = blockIdx.x, token = blockIdx.y, request = blockIdx.z;
  const int kv = head / group;
  const int query_row = token * group + head - kv * group;
  const int tile = query_row / kCachedRows, col = query_row - tile * kCachedRows;
  const int length = cached_length(p, request);
  T* const out = static_cast<T*>(p.out) +
                 ((static_cast<int64_t>(request) * p.tokens + token) * p.heads + head) * p.width;
  const int chunks = (length + p.chunk - 1) / p.chunk;
  const int used = length - p.tokens + token < 0 ? 0 : chunks < p.splits ? chunks : p.splits;
  const float* const parts =
      p.parts + ((static_cast<int64_t>(request) * p.kv_heads + kv) * p.row_tiles + tile) *
                    p.splits * kPartFloats<DP>;
  float most = kMinusInf;
  for (int s = tid; s < used; s += kJoinThreads)
    most = fmaxf(most, parts[static_cast<int64_t>(s) * kPartFloats<DP> + col]);
  most = max_over_rows(most);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, kWave));
  if ((tid & (kWave - 1)) == 0) s_most[tid / kWave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / kWave; ++w) most = fmaxf(most, s_most[w]);
  const int mine = tid / kLanes, at = (tid - mine * kLanes) * 4;
  float sum = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (mine < kGroups) {
#pragma unroll 4
    for (int s = mine; s < used; s += kGroups) {
      const float* const part = parts + static_cast<int64_t>(s) * kPartFloats<DP>;
      const float w = most == kMinusInf ? 1.0f : exp2_fast(part[col] - most);
      sum += part[kCachedRows + col] * w;
      acc += *reinterpret_cast<const f32x4*>(part + 2 * kCachedRows + col * DP + at) * w;
    }
    *reinterpret_cast<f32x4*>(&s_sum[mine][at]) = acc;
    if (at == 0) s_sum[mine][DP] = sum;
  }
  __syncthreads();
  if (tid >= kLanes || at >= p.width) return;
  acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  sum = 0.0f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    acc += *reinterpret_cast<const f32x4*>(&s_sum[g][at]);
    sum += s_sum[g][DP];
  }
  store4(out + at, most == kMinusInf ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / sum));
}

// The waves of a workgroup: eight where the registers of the widths allow two
// on a SIMD.
constexpr int cached_waves(int64_t padded) { return padded <= 128 ? 8 : 4; }

template <int DP, typename T>
void launch_cached(const CachedParams& p, hipStream_t stream) {
  constexpr int NW = cached_waves(DP);
  hipLaunchKernelGGL((cached_attention_kernel<DP, T, NW>),
                     dim3(p.splits * p.row_tiles, p.kv_heads, p.requests), dim3(NW * kWave), 0,
                     stream, p);
  if (p.parts)
    hipLaunchKernelGGL((cached_join_kernel<DP, T>), dim3(p.heads, p.tokens, p.requests),
                       dim3(kJoinThreads), 0, stream, p);
}

template <typename T>
void launch_cached_width(int64_t padded, const CachedParams& p, hipStream_t stream) {
  switch (padded) {
    case 32: return launch_cached<32, T>(p, stream);
    case 64: return launch_cached<64, T>(p, stream);
    case 96: return launch_cached<96, T>(p, stream);
    case 128: return launch_cached<128, T>(p, stream);
    case 192: return launch_cached<192, T>(p, stream);
    default: return launch_cached<256, T>(p, stream);
  }
}

// Workgroups that fill the chip: one a CU, two of the narrowest rows, whose
// registers allow it (10 requests of 65,485 tokens, 7 query tokens, width 32:
// 19 us with two and 25 with one; at width 128 12 of 16,167 take 38 and 29).
constexpr int64_t cached_workgroups(int64_t padded) { return padded <= 32 ? 512 : 256; }

// The splits of the cache that a call's launch makes: enough workgroups to
// fill the chip, none with less than two blocks a wave; and none at all up to
// 2,048 tokens of 131,072 elements of a key head's rows together, for which
// the second launch of a join costs more than the splits give (8 requests of
// 2,048 tokens at width 64: 11 us, 16 in two splits; 4 of 1,500 at width 128,
// past that bound, measure 16 either way).  The lengths are the device's and
// not looked at: one request of 131,072 tokens among 63 of 300, whose rows fill
// the chip by number, is read by a workgroup a key head, 750 us.
int64_t cached_splits(int64_t requests, int64_t kv_heads, int64_t row_tiles, int64_t padded,
                      int64_t longest) {
  if (longest <= 2048 && longest * padded <= 131072) return 1;
  const int64_t least = 2 * cached_waves(padded) * kCachedTokens;
  const int64_t rows = requests * kv_heads * row_tiles;
  const int64_t most = (longest + least - 1) / least;
  int64_t splits = rows > 0 ? (cached_workgroups(padded) + rows - 1) / rows : 1;
  splits = splits < most ? splits : most;
  return splits < 1 ? 1 : splits;
}

int32_t check_cache(const cowsdm_kv_cache_t* c, const char* where, int& shift) {
  if (!c) return fail(COWSDM_EARG, "%s: null cache", where);
  if (c->pages < 0 || c->heads <= 0) return fail(COWSDM_EARG, "%s: bad cache size", where);
  shift = 0;
  while (shift < 8 && (int64_t{1} << shift) < c->page_tokens) ++shift;
  if (c->page_tokens < 16 || (int64_t{1} << shift) != c->page_tokens)
    return fail(COWSDM_EARG, "%s: page tokens must be 16, 32, 64, 128 or 256", where);
  if (!is_cache_width(c->width))
    return fail(COWSDM_EARG, "%s: cache width must be 32, 64, 96, 128, 192 or 256", where);
  if (c->pages * c->page_tokens > INT32_MAX)
    return fail(COWSDM_ELIMIT, "%s: more than 2^31 tokens of pages", where);
  if (c->heads > 65535) return fail(COWSDM_ELIMIT, "%s: at most 65,535 heads", where);
  if (c->pages > 0 && (!c->key_codes || !c->key_scales || !c->value_codes || !c->value_scales))
    return fail(COWSDM_EARG, "%s: null cache tensor", where);
  // codes are loaded 16 bytes at a time
  if ((reinterpret_cast<uintptr_t>(c->key_codes) | reinterpret_cast<uintptr_t>(c->value_codes)) %
      16)
    return fail(COWSDM_EARG, "%s: cache codes must be 16-byte aligned", where);
  return 0;
}

int32_t check_row_width(int64_t width, int64_t padded, const char* where) {
  if (width <= 0 || width % 8 != 0 || width > padded)
    return fail(COWSDM_EARG, "%s: head width must be a multiple of 8, at most the cache's", where);
  return 0;
}

// Rows are loaded 16 bytes at a time.
int32_t check_rows(const void* p, const int64_t* strides, int n, int32_t float_type,
                   const char* where) {
  const int64_t unit = float_type == COWSDM_FLOAT32 ? 4 : 8;
  bool good = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < n; ++i) good = good && strides[i] >= 0 && strides[i] % unit == 0;
  return good ? 0 : fail(COWSDM_EARG, "%s: rows must be 16-byte aligned", where);
}

}  // namespace cowsdm_impl

using namespace cowsdm_impl;

extern "C" int32_t cowsdm_page_tables_extend(
    const int32_t* lengths, const int32_t* added, int64_t requests, int32_t* page_tables,
    int64_t columns, const int32_t* free_pages, int64_t pages, const int32_t* free_count,
    int64_t page_tokens, int64_t tokens, int32_t* lengths_out, int32_t* free_count_out,
    int32_t* offsets, int32_t* positions, int32_t* slots, int32_t* overflow, void* stream) {
  if (requests < 0 || columns < 0 || pages < 0 || tokens < 0)
    return fail(COWSDM_EARG, "page_tables_extend: negative size");
  int shift = 4;
  while (shift < 8 && (int64_t{1} << shift) < page_tokens) ++shift;
  if ((int64_t{1} << shift) != page_tokens)
    return fail(COWSDM_EARG, "page_tables_extend: page tokens must be 16, 32, 64, 128 or 256");
  if (requests > kTableRequests)
    return fail(COWSDM_ELIMIT, "page_tables_extend: at most %d requests", kTableRequests);
  if (pages * page_tokens > INT32_MAX || tokens > INT32_MAX || columns * page_tokens > INT32_MAX)
    return fail(COWSDM_ELIMIT, "page_tables_extend: more than 2^31 tokens");
  if (!free_count || !free_count_out || !offsets || !overflow ||
      (requests > 0 && (!lengths || !added || !lengths_out)) ||
      (requests > 0 && columns > 0 && !page_tables) || (pages > 0 && !free_pages) ||
      (tokens > 0 && (!positions || !slots)))
    return fail(COWSDM_EARG, "page_tables_extend: null pointer argument");
  ExtendParams p{lengths, added, page_tables, free_pages, free_count, lengths_out,
                 free_count_out, offsets, positions, slots, overflow,
                 static_cast<int32_t>(requests), static_cast<int32_t>(columns),
                 static_cast<int32_t>(pages), shift, static_cast<int32_t>(tokens)};
  const int64_t blocks = (tokens + kTableTokensPerBlock - 1) / kTableTokensPerBlock;
  hipLaunchKernelGGL(extend_tables_kernel, dim3(static_cast<uint32_t>(blocks < 1 ? 1 : blocks)),
                     dim3(kTableThreads), 0, static_cast<hipStream_t>(stream), p);
  return launch_status("page_tables_extend");
}

extern "C" int32_t cowsdm_pages_release(int32_t* lengths, int32_t* page_tables, int64_t requests,
                                        int64_t columns, const int32_t* named, int64_t n,
                                        int32_t* free_pages, int64_t pages, int32_t* free_count,
                                        int64_t page_tokens, void* stream) {
  if (requests < 0 || columns < 0 || pages < 0 || n < 0)
    return fail(COWSDM_EARG, "pages_release: negative size");
  int shift = 4;
  while (shift < 8 && (int64_t{1} << shift) < page_tokens) ++shift;
  if ((int64_t{1} << shift) != page_tokens)
    return fail(COWSDM_EARG, "pages_release: page tokens must be 16, 32, 64, 128 or 256");
  if (requests > INT32_MAX || columns > INT32_MAX || pages > INT32_MAX || n > INT32_MAX)
    return fail(COWSDM_ELIMIT, "pages_release: too large");
  if (n == 0) return 0;
  if (!lengths || !page_tables || !named || !free_pages || !free_count)
    return fail(COWSDM_EARG, "pages_release: null pointer argument");
  hipLaunchKernelGGL(release_pages_kernel, dim3(1), dim3(kTableThreads), 0,
                     static_cast<hipStream_t>(stream), lengths, page_tables,
                     static_cast<int32_t>(columns), named, static_cast<int32_t>(n),
                     static_cast<int32_t>(requests), free_pages, static_cast<int32_t>(pages),
                     free_count, shift);
  return launch_status("pages_release");
}

extern "C" int32_t cowsdm_kv_write(const cowsdm_kv_cache_t* cache, const void* key,
                                   int64_t key_row, int64_t key_head, const void* value,
                                   int64_t value_row, int64_t value_head, int32_t float_type,
                                   int64_t width, const int32_t* slots, int64_t tokens,
                                   void* stream) {
  int shift = 0;
  if (int32_t e = check_cache(cache, "kv_write", shift)) return e;
  if (int32_t e = check_row_width(width, cache->width, "kv_write")) return e;
  if (tokens < 0) return fail(COWSDM_EARG, "kv_write: bad token count");
  // a launch counts its threads in 32 bits
  if (tokens >= (int64_t{1} << 30))
    return fail(COWSDM_ELIMIT, "kv_write: 2^30 tokens or more a call");
  if (float_type != COWSDM_FLOAT32 && float_type != COWSDM_FLOAT16 &&
      float_type != COWSDM_BFLOAT16)
    return fail(COWSDM_EARG, "kv_write: bad float type");
  if (tokens == 0 || cache->pages == 0) return 0;
  if (!key || !value || !slots) return fail(COWSDM_EARG, "kv_write: null pointer argument");
  const int64_t strides[] = {key_row, key_head, value_row, value_head};
  if (int32_t e = check_rows(key, strides, 2, float_type, "kv_write")) return e;
  if (int32_t e = check_rows(value, strides + 2, 2, float_type, "kv_write")) return e;
  WriteParams p{};
  p.key = key;
  p.value = value;
  p.key_row = key_row;
  p.key_head = key_head;
  p.value_row = value_row;
  p.value_head = value_head;
  p.slots = slots;
  p.key_codes = static_cast<uint8_t*>(cache->key_codes);
  p.key_scales = cache->key_scales;
  p.value_codes = static_cast<uint8_t*>(cache->value_codes);
  p.value_scales = cache->value_scales;
  p.tokens = static_cast<int32_t>(tokens);
  p.heads = static_cast<int32_t>(cache->heads);
  p.width = static_cast<int32_t>(width);
  p.pages = static_cast<int32_t>(cache->pages);
  p.page_shift = shift;
  // Single tokens are a run each and want a workgroup each; of a prompt's, whose
  // runs are pages, most workgroups would find nothing to open.  The call does
  // not say which it is, so that the token count has to: 8 heads of 128, us by
  // one token and by 64 a workgroup: 512 single tokens 24 and 188, 1,024 41 and
  // 186, 2,048 75 and 185, 4,096 188 and 223; 16 prompts of 64 32 and 10, 4 of
  // 500 21 and 10, 8 of 2,000 341 and 25.  So more than 1,024 single tokens, and
  // prompts of fewer in all, take the slower side.
  p.chunk = tokens <= 1024 ? 1 : kWave;
  const dim3 grid(static_cast<uint32_t>((tokens + p.chunk - 1) / p.chunk),
                  static_cast<uint32_t>(cache->heads));
  const int padded = static_cast<int>(cache->width);
  const auto s = static_cast<hipStream_t>(stream);
  if (float_type == COWSDM_FLOAT32) launch_write<float>(p, grid, padded, s);
  else if (float_type == COWSDM_FLOAT16) launch_write<_Float16>(p, grid, padded, s);
  else launch_write<__bf16>(p, grid, padded, s);
  return launch_status("kv_write");
}

extern "C" int64_t cowsdm_cached_attention_workspace_bytes(int64_t requests, int64_t tokens,
                                                           int64_t heads, int64_t kv_heads,
                                                           int64_t padded_width, int64_t longest) {
  if (requests < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
      !is_cache_width(padded_width) || longest < 0)
    return -1;
  const int64_t tiles = (tokens * (heads / kv_heads) + kCachedRows - 1) / kCachedRows;
  const int64_t splits = cached_splits(requests, kv_heads, tiles, padded_width, longest);
  if (splits == 1) return 0;
  return requests * kv_heads * tiles * splits * (2 * kCachedRows + kCachedRows * padded_width) *
         static_cast<int64_t>(sizeof(float));
}

extern "C" int32_t cowsdm_cached_attention(const cowsdm_kv_cache_t* cache,
                                           const cowsdm_cached_query_t* query, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  int shift = 0;
  if (int32_t e = check_cache(cache, "cached_attention", shift)) return e;
  if (!query) return fail(COWSDM_EARG, "cached_attention: null query");
  const cowsdm_cached_query_t& q = *query;
  if (int32_t e = check_row_width(q.width, cache->width, "cached_attention")) return e;
  if (q.requests < 0 || q.tokens < 0 || q.heads <= 0 || q.columns < 0 || q.longest < 0)
    return fail(COWSDM_EARG, "cached_attention: bad size");
  if (q.heads % cache->heads != 0)
    return fail(COWSDM_EARG, "cached_attention: query heads must be a multiple of the cache's");
  if (q.requests > 65535 || q.tokens > 65535 || q.heads > 65535 ||
      q.columns * cache->page_tokens > (1 << 30) || q.longest > (1 << 30))
    return fail(COWSDM_ELIMIT, "cached_attention: too large");
  if (!(q.scale > 0.0f) || q.scale > 3.0e38f)
    return fail(COWSDM_EARG, "cached_attention: the scale must be positive");
  if (q.float_type != COWSDM_FLOAT32 && q.float_type != COWSDM_FLOAT16 &&
      q.float_type != COWSDM_BFLOAT16)
    return fail(COWSDM_EARG, "cached_attention: bad float type");
  if (q.requests == 0 || q.tokens == 0) return 0;
  if (cache->pages == 0) return fail(COWSDM_EARG, "cached_attention: the cache has no pages");
  if (!q.query || !q.lengths || !q.out || (q.columns > 0 && !q.page_tables))
    return fail(COWSDM_EARG, "cached_attention: null pointer argument");
  const int64_t strides[] = {q.query_request, q.query_token, q.query_head};
  if (int32_t e = check_rows(q.query, strides, 3, q.float_type, "cached_attention")) return e;
  CachedParams p{};
  p.query = q.query;
  p.query_request = q.query_request;
  p.query_token = q.query_token;
  p.query_head = q.query_head;
  p.key_codes = static_cast<const uint8_t*>(cache->key_codes);
  p.key_scales = cache->key_scales;
  p.value_codes = static_cast<const uint8_t*>(cache->value_codes);
  p.value_scales = cache->value_scales;
  p.page_tables = q.page_tables;
  p.lengths = q.lengths;
  p.out = q.out;
  p.scale = q.scale * kLog2E;
  p.requests = static_cast<int32_t>(q.requests);
  p.tokens = static_cast<int32_t>(q.tokens);
  p.heads = static_cast<int32_t>(q.heads);
  p.kv_heads = static_cast<int32_t>(cache->heads);
  p.width = static_cast<int32_t>(q.width);
  p.pages = static_cast<int32_t>(cache->pages);
  p.columns = static_cast<int32_t>(q.columns);
  p.page_shift = shift;
  const int64_t group = q.heads / cache->heads;
  const int64_t tiles = (q.tokens * group + kCachedRows - 1) / kCachedRows;
  p.row_tiles = static_cast<int32_t>(tiles);
  p.splits = static_cast<int32_t>(
      cached_splits(q.requests, cache->heads, tiles, cache->width, q.longest));
  // a launch counts its threads in 32 bits
  if (tiles * p.splits * cached_waves(cache->width) * kWave > UINT32_MAX)
    return fail(COWSDM_ELIMIT, "cached_attention: too many query rows a request");
  const int64_t kBlock = cached_waves(cache->width) * kCachedTokens;
  const int64_t each = (q.longest + p.splits - 1) / p.splits;
  p.chunk = p.splits == 1 ? INT32_MAX / 2
                          : static_cast<int32_t>((each + kBlock - 1) / kBlock * kBlock);
  p.by_length = q.requests > 1 && q.requests <= kWave && p.splits == 1 &&
                q.requests * cache->heads * tiles > cached_workgroups(cache->width) &&
                q.columns * cache->page_tokens < (1 << 24);
  if (p.splits > 1) {
    const int64_t need = cowsdm_cached_attention_workspace_bytes(
        q.requests, q.tokens, q.heads, cache->heads, cache->width, q.longest);
    if (!workspace || workspace_bytes < need)
      return fail(COWSDM_EARG, "cached_attention: workspace of %lld bytes needed",
                  static_cast<long long>(need));
    p.parts = static_cast<float*>(workspace);
  }
  const auto s = static_cast<hipStream_t>(stream);
  if (q.float_type == COWSDM_FLOAT32) launch_cached_width<float>(cache->width, p, s);
  else if (q.float_type == COWSDM_FLOAT16) launch_cached_width<_Float16>(cache->width, p, s);
  else launch_cached_width<__bf16>(cache->width, p, s);
  return launch_status("cached_attention");
}
