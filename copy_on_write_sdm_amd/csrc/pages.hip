// The life of a paged cache's pages besides their extension: requests that
// share the first tokens of others, the return of finished requests' pages,
// the pool's pages in use moved to its lowest numbers, and the copies of
// pages that a fork and a move need.
//
// page_shares[p] counts the requests that hold page p beyond the first, so
// that pages which nothing shares need no care: extension does not write it.
//
// Every operator leaves its inputs as they are and writes new lengths,
// tables, counts and shares, so that a step can be taken back by keeping what
// was there.  Only the free stack is written in place: a release pushes above
// its count, over the numbers that forks and extensions have popped, so that
// after it there is no way back to a larger count.  Each runs in phases that need all of the one before.  Where
// the numbers are few, one workgroup runs them all with the pages' numbers in
// LDS and its entries in registers, so that a phase costs a barrier and not a
// launch or a round trip to memory; else they are launches of their own.

#include "common.h"

namespace cowsdm_impl {

constexpr int kPageThreads = 512;
constexpr int kPageNamed = 4096;       // children of a fork, named requests of a release

// What one workgroup takes: entries of tables and pages (LDS holds two
// numbers a page), and children or named requests.  In us, one workgroup
// against launches of their own: fork of 4 children 3.0 against 4.4, 8,128
// entries over 4,409 pages 6.0 against 5.5; release of 704 entries over 1,327
// pages 4.2 against 9.8, 7,200 entries compacted 9.0 against 12.7.  With 16
// numbers a thread the same release took 5.6 and a compaction of 192 entries
// 7.6 (4.5 with 8), and 12,288 entries 14.8 against 13.1.
constexpr int kOneThreads = 1024;
constexpr int kOneWaves = kOneThreads / kWave;
constexpr int kOneEach = 8;
constexpr int kOneNumbers = kOneThreads * kOneEach;
constexpr int kOnePages = 8192;
constexpr int kOneNamed = 1024;
constexpr int kOneRequests = 4096;

// Exclusive sum of v over the workgroup and, in `total`, the sum.
__device__ __forceinline__ int group_exclusive(int v, int* parts, int& total) {
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wave = static_cast<int>(threadIdx.x) / kWave;
  const int in = wave_inclusive(v);
  __syncthreads();
  if (lane == kWave - 1) parts[wave] = in;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPageThreads / kWave; ++w) {
    if (w < wave) before += parts[w];
    total += parts[w];
  }
  return before + in - v;
}

// Of the numbers counts[0 .. n - 1]: the sum of those before `chunk`, and all.
__device__ __forceinline__ int sum_before(const int32_t* counts, int n, int chunk, int* parts,
                                          int& all) {
  int before = 0, sum = 0;
  for (int c = static_cast<int>(threadIdx.x); c < n; c += kPageThreads) {
    const int v = counts[c];
    sum += v;
    if (c < chunk) before += v;
  }
  int total;
  group_exclusive(before, parts, total);
  group_exclusive(sum, parts, all);
  return total;
}

__device__ __forceinline__ int pages_held(int32_t length, int page_shift, int columns) {
  if (length <= 0) return 0;
  const int n = static_cast<int>((static_cast<uint32_t>(length) + (1u << page_shift) - 1) >>
                                 page_shift);
  return n < columns ? n : columns;
}

// Places in order for one workgroup's numbers, number i * kOneThreads + thread
// being the thread's i-th: s_places[i][wave] becomes how many of the flagged
// (bit i of a thread's `flags`) come before that wave's i-th ones.  Returns
// how many there are.
__device__ __forceinline__ int one_places(uint32_t flags, int (*s_places)[kOneWaves]) {
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (kWave - 1);
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const uint64_t mask = __ballot(flags >> i & 1);
    if (lane == 0) s_places[i][tid / kWave] = __builtin_popcountll(mask);
  }
  __syncthreads();
  constexpr int kCounts = kOneEach * kOneWaves, kMine = kCounts / kWave;
  int* const flat = &s_places[0][0];
  if (tid < kWave) {
    int v[kMine], sum = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) sum += v[j] = flat[tid * kMine + j];
    const int all = wave_inclusive(sum);
    int before = all - sum;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      flat[tid * kMine + j] = before;
      before += v[j];
    }
    if (tid == kWave - 1) s_places[kOneEach][0] = all;
  }
  __syncthreads();
  return s_places[kOneEach][0];
}

// The place of this thread's i-th number among the flagged.
__device__ __forceinline__ int one_place(uint32_t flags, int i,
                                         const int (*s_places)[kOneWaves]) {
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (kWave - 1);
  const uint64_t below = __ballot(flags >> i & 1) & ((uint64_t{1} << lane) - 1);
  return s_places[i][tid / kWave] + __builtin_popcountll(below);
}

// ------------------------------------------------------------------- fork

struct ForkParams {
  const int32_t* lengths;
  const int32_t* page_tables;
  const int32_t* page_shares;
  const int32_t* free_pages;
  const int32_t* free_count;
  const int32_t* parents;
  const int32_t* tokens;
  int32_t* lengths_out;
  int32_t* tables_out;
  int32_t* shares_out;
  int32_t* free_count_out;
  int32_t* sources;
  int32_t* targets;
  int32_t* overflow;
  int32_t requests;
  int32_t columns;
  int32_t pages;
  int32_t children;
  int32_t page_shift;
};

// The new pages, popped from the top of the free stack in the children's
// order, one for every child whose tokens end inside a page.
__device__ void fork_plan(const ForkParams& p, int* parts) {
  const int tid = static_cast<int>(threadIdx.x);
  const int32_t count = *p.free_count;
  int need = 0, bad = 0;
  for (int at = 0; at < p.children; at += kPageThreads) {
    const int i = at + tid;
    int rest = 0, wrong = 0;
    if (i < p.children) {
      const int32_t r = p.parents[i], n = p.tokens[i];
      const bool is = r >= 0 && r < p.requests;
      const int32_t held = is ? p.lengths[r] : -1;
      wrong = n < 0 || n > held || pages_held(n, p.page_shift, INT32_MAX) > p.columns;
      rest = (n & ((1 << p.page_shift) - 1)) != 0;
    }
    int sum, wrongs;
    group_exclusive(rest, parts, sum);
    group_exclusive(wrong, parts, wrongs);
    need += sum;
    bad |= wrongs;
  }
  const bool fits = !bad && need <= count && count <= p.pages;
  int taken = 0;
  for (int at = 0; at < p.children; at += kPageThreads) {
    const int i = at + tid;
    int32_t n = 0, r = 0;
    if (fits && i < p.children) {
      n = p.tokens[i];
      r = p.parents[i];
    }
    const int rest = (n & ((1 << p.page_shift) - 1)) != 0;
    int sum;
    const int before = taken + group_exclusive(rest, parts, sum);
    if (i < p.children) {
      int32_t source = -1, target = -1;
      if (rest) {
        source = p.page_tables[static_cast<int64_t>(r) * p.columns + (n >> p.page_shift)];
        target = p.free_pages[count - 1 - before];
      }
      p.lengths_out[i] = n;
      p.sources[i] = source;
      p.targets[i] = target;
    }
    taken += sum;
  }
  if (tid == 0) {
    *p.free_count_out = fits ? count - need : count;
    *p.overflow = fits ? 0 : 1;
  }
}

__device__ void fork_shares(const ForkParams& p, int block, int blocks) {
  for (int64_t i = static_cast<int64_t>(block) * kPageThreads + threadIdx.x; i < p.pages;
       i += static_cast<int64_t>(blocks) * kPageThreads)
    p.shares_out[i] = p.page_shares[i];
}

// The children's tables: whole pages by number, each with one more sharer.
__device__ void fork_tables(const ForkParams& p, int block, int blocks) {
  const bool fits = *p.overflow == 0;
  const int64_t entries = static_cast<int64_t>(p.children) * p.columns;
  for (int64_t e = static_cast<int64_t>(block) * kPageThreads + threadIdx.x; e < entries;
       e += static_cast<int64_t>(blocks) * kPageThreads) {
    const int i = static_cast<int>(e) / p.columns, j = static_cast<int>(e) - i * p.columns;
    int32_t id = -1;
    if (fits) {
      const int whole = p.tokens[i] >> p.page_shift;
      if (j < whole) {
        id = p.page_tables[static_cast<int64_t>(p.parents[i]) * p.columns + j];
        if (id >= 0 && id < p.pages) atomicAdd(p.shares_out + id, 1);
      } else if (j == whole) {
        id = p.targets[i];
      }
    }
    p.tables_out[e] = id;
  }
}

// The same in one workgroup: a child to a thread, the pages' shares in LDS.
// What bounds it is latency, the dependent loads of a child's parent, its
// length, the tables and the free pages: 3.0 us for 4 children, 4.7 us for 256
// with 5,120 entries, of which a launch by itself is some 2.
__global__ __launch_bounds__(kOneThreads) void fork_one_kernel(ForkParams p) {
  extern __shared__ __align__(16) int32_t s_shares[];             // [pages]
  __shared__ int s_places[2][kOneWaves];
  __shared__ int32_t s_parent[kOneNamed], s_whole[kOneNamed], s_target[kOneNamed];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & (kWave - 1), wave = tid / kWave;
  const int32_t count = *p.free_count;
  int32_t n = 0, r = 0;
  int rest = 0, wrong = 0;
  if (tid < p.children) {
    r = p.parents[tid];
    n = p.tokens[tid];
  }
  for (int i = tid; i < p.pages; i += kOneThreads) s_shares[i] = p.page_shares[i];
  if (tid < p.children) {
    const int32_t held = r >= 0 && r < p.requests ? p.lengths[r] : -1;
    wrong = n < 0 || n > held || pages_held(n, p.page_shift, INT32_MAX) > p.columns;
    rest = (n & ((1 << p.page_shift) - 1)) != 0;
  }
  const uint64_t rests = __ballot(rest);
  if (lane == 0) {
    s_places[0][wave] = __builtin_popcountll(rests);
    s_places[1][wave] = 0;
  }
  if (__ballot(wrong) && lane == 0) s_places[1][wave] = 1;
  __syncthreads();
  int before = 0, need = 0, bad = 0;
#pragma unroll
  for (int w = 0; w < kOneWaves; ++w) {
    if (w < wave) before += s_places[0][w];
    need += s_places[0][w];
    bad |= s_places[1][w];
  }
  before += __builtin_popcountll(rests & ((uint64_t{1} << lane) - 1));
  const bool fits = !bad && need <= count && count <= p.pages;
  if (tid < p.children) {
    int32_t source = -1, target = -1;
    if (fits && rest) {
      source = p.page_tables[static_cast<int64_t>(r) * p.columns + (n >> p.page_shift)];
      target = p.free_pages[count - 1 - before];
    }
    s_parent[tid] = fits ? r : 0;
    s_whole[tid] = fits ? n >> p.page_shift : 0;
    s_target[tid] = target;
    p.lengths_out[tid] = fits ? n : 0;
    p.sources[tid] = source;
    p.targets[tid] = target;
  }
  if (tid == 0) {
    *p.free_count_out = fits ? count - need : count;
    *p.overflow = fits ? 0 : 1;
  }
  __syncthreads();
  const int entries = p.children * p.columns;
#pragma unroll 4
  for (int e = tid; e < entries; e += kOneThreads) {
    const int i = e / p.columns, j = e - i * p.columns, whole = s_whole[i];
    int32_t id = -1;
    if (j < whole) {
      id = p.page_tables[static_cast<int64_t>(s_parent[i]) * p.columns + j];
      if (id >= 0 && id < p.pages) atomicAdd(s_shares + id, 1);
    } else if (j == whole) {
      id = s_target[i];
    }
    p.tables_out[e] = id;
  }
  __syncthreads();
  for (int i = tid; i < p.pages; i += kOneThreads) p.shares_out[i] = s_shares[i];
}

__global__ __launch_bounds__(kPageThreads) void fork_plan_kernel(ForkParams p) {
  __shared__ int s_parts[kPageThreads / kWave];
  if (blockIdx.x == 0) fork_plan(p, s_parts);
  else fork_shares(p, blockIdx.x - 1, gridDim.x - 1);
}

__global__ __launch_bounds__(kPageThreads) void fork_tables_kernel(ForkParams p) {
  fork_tables(p, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------- release

struct ReleaseParams {
  const int32_t* lengths;
  const int32_t* page_tables;
  const int32_t* page_shares;
  const int32_t* free_count;
  const int32_t* named;
  int32_t* free_pages;
  int32_t* lengths_out;
  int32_t* shares_out;
  int32_t* free_count_out;
  int32_t* last;          // [pages] the page's last entry among the named requests'
  int32_t* held;          // [n] pages of each named request; 0 where it is named before
  int32_t* counts;        // freed pages of each chunk of entries
  int32_t requests;
  int32_t columns;
  int32_t pages;
  int32_t n;
  int32_t entries;        // n * columns
  int32_t chunks, chunk;  // of entries, and the entries of one
  int32_t page_shift;
};

// A request counts where it is named first, which is found in LDS, or in the
// new lengths' place where there are more requests.
__device__ void release_plan(const ReleaseParams& p, int32_t* in_lds) {
  const int tid = static_cast<int>(threadIdx.x), step = static_cast<int>(blockDim.x);
  const bool few = p.requests <= kOneRequests;
  int32_t* const first = few ? in_lds : p.lengths_out;
  for (int r = tid; r < p.requests; r += step) first[r] = INT32_MAX;
  if (!few) __threadfence();
  __syncthreads();
  for (int i = tid; i < p.n; i += step) {
    const int32_t r = p.named[i];
    if (r >= 0 && r < p.requests) atomicMin(first + r, i);
  }
  if (!few) __threadfence();
  __syncthreads();
  for (int i = tid; i < p.n; i += step) {
    const int32_t r = p.named[i];
    const bool is = r >= 0 && r < p.requests && first[r] == i;
    p.held[i] = is ? pages_held(p.lengths[r], p.page_shift, p.columns) : 0;
  }
  __syncthreads();
  for (int r = tid; r < p.requests; r += step)
    p.lengths_out[r] = first[r] == INT32_MAX ? p.lengths[r] : 0;
}

__device__ void release_shares(const ReleaseParams& p, int block, int blocks) {
  for (int64_t i = static_cast<int64_t>(block) * kPageThreads + threadIdx.x; i < p.pages;
       i += static_cast<int64_t>(blocks) * kPageThreads) {
    p.shares_out[i] = p.page_shares[i];
    p.last[i] = -1;
  }
}

// The page of entry e of the named requests' tables, or -1.
__device__ __forceinline__ int release_entry(const ReleaseParams& p, int e) {
  if (e >= p.entries) return -1;
  const int i = e / p.columns, j = e - i * p.columns;
  if (j >= p.held[i]) return -1;
  const int32_t id = p.page_tables[static_cast<int64_t>(p.named[i]) * p.columns + j];
  return id >= 0 && id < p.pages ? id : -1;
}

__device__ void release_take(const ReleaseParams& p, int block, int blocks) {
  for (int64_t e = static_cast<int64_t>(block) * kPageThreads + threadIdx.x; e < p.entries;
       e += static_cast<int64_t>(blocks) * kPageThreads) {
    const int id = release_entry(p, static_cast<int>(e));
    if (id < 0) continue;
    atomicSub(p.shares_out + id, 1);
    atomicMax(p.last + id, static_cast<int32_t>(e));
  }
}

// A page is free when more have let it go than shared it; its last entry
// stands for it.
__device__ __forceinline__ int release_freed(const ReleaseParams& p, int e) {
  const int id = release_entry(p, e);
  return id >= 0 && p.last[id] == e && p.shares_out[id] < 0 ? id : -1;
}

__device__ void release_count(const ReleaseParams& p, int* parts) {
  int mine = 0;
  const int from = static_cast<int>(blockIdx.x) * p.chunk + static_cast<int>(threadIdx.x);
  for (int at = 0; at < p.chunk; at += kPageThreads) mine += release_freed(p, from + at) >= 0;
  int total;
  group_exclusive(mine, parts, total);
  if (threadIdx.x == 0) p.counts[blockIdx.x] = total;
}

__device__ void release_push(const ReleaseParams& p, int* parts) {
  const int32_t count = *p.free_count;
  const int c = static_cast<int>(blockIdx.x);
  int all;
  int64_t to = static_cast<int64_t>(count) + sum_before(p.counts, p.chunks, c, parts, all);
  if (c == 0 && threadIdx.x == 0) {
    const int64_t top = static_cast<int64_t>(count) + all;
    *p.free_count_out = static_cast<int32_t>(top < p.pages ? top : p.pages);
  }
  const int from = c * p.chunk + static_cast<int>(threadIdx.x);
  for (int at = 0; at < p.chunk; at += kPageThreads) {
    const int id = release_freed(p, from + at);
    int total;
    const int64_t mine = to + group_exclusive(id >= 0, parts, total);
    if (id >= 0) {
      if (mine >= 0 && mine < p.pages) p.free_pages[mine] = id;
      p.shares_out[id] = 0;
    }
    to += total;
  }
}

// The same in one workgroup: the pages' shares and last entries in LDS, its
// entries in registers.  Latency bounds it: dependent loads of a named request,
// its length and its entries, and eight barriers.
__global__ __launch_bounds__(kOneThreads) void release_one_kernel(ReleaseParams p) {
  extern __shared__ __align__(16) int32_t s_pages[];              // [2][pages]
  __shared__ int32_t s_first[kOneRequests];
  __shared__ int32_t s_row[kOneNamed], s_held[kOneNamed];
  __shared__ int s_places[kOneEach + 1][kOneWaves];
  int32_t* const s_shares = s_pages;
  int32_t* const s_last = s_pages + p.pages;
  const int tid = static_cast<int>(threadIdx.x);
  const int32_t count = *p.free_count;
  const int32_t name = tid < p.n ? p.named[tid] : -1;
  const bool is_name = name >= 0 && name < p.requests;
  const int32_t length = is_name ? p.lengths[name] : 0;
  for (int r = tid; r < p.requests; r += kOneThreads) s_first[r] = INT32_MAX;
  for (int i = tid; i < p.pages; i += kOneThreads) {
    s_shares[i] = p.page_shares[i];
    s_last[i] = -1;
  }
  __syncthreads();
  if (is_name) atomicMin(s_first + name, tid);
  __syncthreads();
  if (tid < p.n) {
    s_row[tid] = name;
    s_held[tid] = is_name && s_first[name] == tid ? pages_held(length, p.page_shift, p.columns) : 0;
  }
  for (int r = tid; r < p.requests; r += kOneThreads)
    p.lengths_out[r] = s_first[r] == INT32_MAX ? p.lengths[r] : 0;
  __syncthreads();
  int32_t id[kOneEach];
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int e = i * kOneThreads + tid;
    id[i] = -1;
    if (e < p.entries) {
      const int named = e / p.columns, j = e - named * p.columns;
      if (j < s_held[named])
        id[i] = p.page_tables[static_cast<int64_t>(s_row[named]) * p.columns + j];
    }
  }
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    if (id[i] < 0 || id[i] >= p.pages) {
      id[i] = -1;
    } else {
      atomicSub(s_shares + id[i], 1);
      atomicMax(s_last + id[i], i * kOneThreads + tid);
    }
  }
  __syncthreads();
  uint32_t freed = 0;
#pragma unroll
  for (int i = 0; i < kOneEach; ++i)
    if (id[i] >= 0 && s_last[id[i]] == i * kOneThreads + tid && s_shares[id[i]] < 0)
      freed |= 1u << i;
  const int all = one_places(freed, s_places);
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int64_t to = static_cast<int64_t>(count) + one_place(freed, i, s_places);
    if (freed >> i & 1) {
      if (to >= 0 && to < p.pages) p.free_pages[to] = id[i];
      s_shares[id[i]] = 0;
    }
  }
  if (tid == 0) {
    const int64_t top = static_cast<int64_t>(count) + all;
    *p.free_count_out = static_cast<int32_t>(top < p.pages ? top : p.pages);
  }
  __syncthreads();
  for (int i = tid; i < p.pages; i += kOneThreads) p.shares_out[i] = s_shares[i];
}

__global__ __launch_bounds__(kPageThreads) void release_plan_kernel(ReleaseParams p) {
  __shared__ int32_t s_first[kOneRequests];
  if (blockIdx.x == 0) release_plan(p, s_first);
  else release_shares(p, blockIdx.x - 1, gridDim.x - 1);
}

__global__ __launch_bounds__(kPageThreads) void release_take_kernel(ReleaseParams p) {
  release_take(p, blockIdx.x, gridDim.x);
}

__global__ __launch_bounds__(kPageThreads) void release_count_kernel(ReleaseParams p) {
  __shared__ int s_parts[kPageThreads / kWave];
  release_count(p, s_parts);
}

__global__ __launch_bounds__(kPageThreads) void release_push_kernel(ReleaseParams p) {
  __shared__ int s_parts[kPageThreads / kWave];
  release_push(p, s_parts);
}

// ---------------------------------------------------------------- compact

struct CompactParams {
  const int32_t* lengths;
  const int32_t* page_tables;
  const int32_t* page_shares;
  int32_t* tables_out;
  int32_t* shares_out;
  int32_t* free_pages;
  int32_t* free_count;
  int32_t* sources;
  int32_t* targets;
  int32_t* used;          // [pages] 1 where a request holds the page; then its rank among the moved
  int32_t* counts;        // pages in use of each chunk
  int32_t requests;
  int32_t columns;
  int32_t pages;
  int32_t entries;
  int32_t chunks, chunk;  // of pages, and the pages of one
  int32_t page_shift;
};

__device__ void compact_clear(const CompactParams& p, int block, int blocks) {
  for (int64_t i = static_cast<int64_t>(block) * kPageThreads + threadIdx.x; i < p.pages;
       i += static_cast<int64_t>(blocks) * kPageThreads) {
    p.used[i] = 0;
    if (i < p.pages / 2) p.sources[i] = p.targets[i] = -1;
  }
}

// The page of entry e, or -1.
__device__ __forceinline__ int compact_entry(const CompactParams& p, int e) {
  const int r = e / p.columns, j = e - r * p.columns;
  if (j >= pages_held(p.lengths[r], p.page_shift, p.columns)) return -1;
  const int32_t id = p.page_tables[e];
  return id >= 0 && id < p.pages ? id : -1;
}

__device__ void compact_mark(const CompactParams& p, int block, int blocks) {
  for (int64_t e = static_cast<int64_t>(block) * kPageThreads + threadIdx.x; e < p.entries;
       e += static_cast<int64_t>(blocks) * kPageThreads) {
    const int id = compact_entry(p, static_cast<int>(e));
    if (id >= 0) p.used[id] = 1;
  }
}

__device__ void compact_count(const CompactParams& p, int* parts) {
  int mine = 0;
  for (int at = 0; at < p.chunk; at += kPageThreads) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * p.chunk + at + threadIdx.x;
    mine += i < p.pages ? p.used[i] : 0;
  }
  int total;
  group_exclusive(mine, parts, total);
  if (threadIdx.x == 0) p.counts[blockIdx.x] = total;
}

// U pages are in use.  The k-th of those numbered U or more goes to the k-th
// number below U that is free: as many of the one as of the other.  Of page i
// with b pages in use before it, i - b are free before it.
__device__ void compact_place(const CompactParams& p, int* parts) {
  const int c = static_cast<int>(blockIdx.x);
  int all;
  int before = sum_before(p.counts, p.chunks, c, parts, all);
  if (c == 0 && threadIdx.x == 0) *p.free_count = p.pages - all;
  // those in use below U
  int low = sum_before(p.counts, p.chunks, all / p.chunk, parts, all);
  {
    int mine = 0, total;
    for (int i = all / p.chunk * p.chunk + static_cast<int>(threadIdx.x); i < all;
         i += kPageThreads)
      mine += p.used[i] != 0;
    group_exclusive(mine, parts, total);
    low += total;
  }
  for (int at = 0; at < p.chunk; at += kPageThreads) {
    const int64_t i = static_cast<int64_t>(c) * p.chunk + at + threadIdx.x;
    const int is = i < p.pages ? p.used[i] : 0;
    int total;
    const int rank = before + group_exclusive(is, parts, total);
    before += total;
    if (is && i >= all) {
      p.sources[rank - low] = static_cast<int32_t>(i);
      p.used[i] = rank - low;          // read by no one before the next phase
    } else if (!is && i < all) {
      p.targets[i - rank] = static_cast<int32_t>(i);
    }
  }
}

__device__ void compact_rewrite(const CompactParams& p, int block, int blocks) {
  const int all = p.pages - *p.free_count;
  const int64_t first = static_cast<int64_t>(block) * kPageThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(blocks) * kPageThreads;
  for (int64_t e = first; e < p.entries; e += step) {
    int id = compact_entry(p, static_cast<int>(e));
    if (id >= all) id = p.targets[p.used[id]];
    p.tables_out[e] = id;
  }
  for (int64_t i = first; i < p.pages; i += step) {
    p.free_pages[i] = i < p.pages - all ? static_cast<int32_t>(p.pages - 1 - i) : -1;
    if (i >= all) p.shares_out[i] = 0;
    else if (p.used[i] != 0) p.shares_out[i] = p.page_shares[i];
    // the other numbers below U get their new page's
    if (i < p.pages / 2 && p.sources[i] >= 0)
      p.shares_out[p.targets[i]] = p.page_shares[p.sources[i]];
  }
}

// The same in one workgroup: what is in use, then the moved pages' ranks and
// the free numbers below U, in LDS.  Latency bounds it, as of a release: 4.5 us
// for 192 entries, 5.2 for 1,280.
__global__ __launch_bounds__(kOneThreads) void compact_one_kernel(CompactParams p) {
  extern __shared__ __align__(16) int32_t s_pages[];              // [2][pages]
  __shared__ int s_places[kOneEach + 1][kOneWaves];
  __shared__ int s_low;
  int32_t* const s_used = s_pages;
  int32_t* const s_targets = s_pages + p.pages;
  const int tid = static_cast<int>(threadIdx.x);
  for (int i = tid; i < p.pages; i += kOneThreads) s_used[i] = 0;
  int32_t id[kOneEach];
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int e = i * kOneThreads + tid;
    id[i] = e < p.entries ? compact_entry(p, e) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOneEach; ++i)
    if (id[i] >= 0) s_used[id[i]] = 1;
  __syncthreads();
  uint32_t used = 0;
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int page = i * kOneThreads + tid;
    if (page < p.pages && s_used[page]) used |= 1u << i;
  }
  const int all = one_places(used, s_places);
  if (tid == 0 && all == p.pages) s_low = all;
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int page = i * kOneThreads + tid, rank = one_place(used, i, s_places);
    if (page == all && all < p.pages) s_low = rank;
    if (page < all && !(used >> i & 1)) {
      s_targets[page - rank] = page;
      p.targets[page - rank] = page;
    }
  }
  __syncthreads();
  const int low = s_low, moves = all - low;
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int page = i * kOneThreads + tid, rank = one_place(used, i, s_places) - low;
    if (page >= p.pages) continue;
    const bool is = used >> i & 1;
    if (is && page >= all) {
      s_used[page] = rank;
      p.sources[rank] = page;
    }
    // every page's shares in their new place
    if (is) p.shares_out[page < all ? page : s_targets[rank]] = p.page_shares[page];
    if (page >= all) p.shares_out[page] = 0;
    p.free_pages[page] = page < p.pages - all ? p.pages - 1 - page : -1;
    if (page >= moves && page < p.pages / 2) p.sources[page] = p.targets[page] = -1;
  }
  if (tid == 0) *p.free_count = p.pages - all;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOneEach; ++i) {
    const int e = i * kOneThreads + tid;
    if (e < p.entries) p.tables_out[e] = id[i] < all ? id[i] : s_targets[s_used[id[i]]];
  }
}

__global__ __launch_bounds__(kPageThreads) void compact_clear_kernel(CompactParams p) {
  compact_clear(p, blockIdx.x, gridDim.x);
}

__global__ __launch_bounds__(kPageThreads) void compact_mark_kernel(CompactParams p) {
  compact_mark(p, blockIdx.x, gridDim.x);
}

__global__ __launch_bounds__(kPageThreads) void compact_count_kernel(CompactParams p) {
  __shared__ int s_parts[kPageThreads / kWave];
  compact_count(p, s_parts);
}

__global__ __launch_bounds__(kPageThreads) void compact_place_kernel(CompactParams p) {
  __shared__ int s_parts[kPageThreads / kWave];
  compact_place(p, s_parts);
}

__global__ __launch_bounds__(kPageThreads) void compact_rewrite_kernel(CompactParams p) {
  compact_rewrite(p, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------- copy

typedef uint32_t page_words __attribute__((ext_vector_type(4)));

constexpr int kCopyThreads = 256;
constexpr int kCopyEach = 4;                                     // 16-byte words of a thread
constexpr int kCopyBytes = kCopyThreads * kCopyEach * 16;        // of a workgroup

struct CopyParams {
  page_words* key_codes;
  page_words* value_codes;
  float* key_scales;
  float* value_scales;
  const int32_t* sources;
  const int32_t* targets;
  int32_t pages;
  int32_t heads;
  int32_t words;          // of a page's keys, and of its values
  int32_t parts;          // workgroups to them
};

// A workgroup copies a part of one page's keys or values in one layer, all of a
// thread's loads before its stores.  Memory bounds it, read and written: 309 MB
// of pages of 64 tokens over four layers (8 heads 128 wide) in 60 us, 5.4 TB/s.
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyParams p) {
  const int copy = static_cast<int>(blockIdx.x) / (2 * p.parts);
  const int part = static_cast<int>(blockIdx.x) - copy * 2 * p.parts;
  const int32_t source = p.sources[copy], target = p.targets[copy];
  if (source < 0 || source >= p.pages || target < 0 || target >= p.pages || source == target)
    return;
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t first = static_cast<int64_t>(blockIdx.y) * p.pages;
  const bool values = part >= p.parts;
  const int at = values ? part - p.parts : part;
  page_words* const codes = values ? p.value_codes : p.key_codes;
  float* const scales = values ? p.value_scales : p.key_scales;
  const page_words* const from = codes + (first + source) * p.words;
  page_words* const to = codes + (first + target) * p.words;
  page_words held[kCopyEach];
  const int begin = at * kCopyThreads * kCopyEach + tid;
#pragma unroll
  for (int n = 0; n < kCopyEach; ++n)
    if (begin + n * kCopyThreads < p.words) held[n] = from[begin + n * kCopyThreads];
  if (at == 0) {
    for (int h = tid; h < p.heads; h += kCopyThreads)
      scales[(first + target) * p.heads + h] = scales[(first + source) * p.heads + h];
  }
#pragma unroll
  for (int n = 0; n < kCopyEach; ++n)
    if (begin + n * kCopyThreads < p.words) to[begin + n * kCopyThreads] = held[n];
}

int32_t page_shift_of(int64_t page_tokens, const char* where, int& shift) {
  shift = 4;
  while (shift < 8 && (int64_t{1} << shift) < page_tokens) ++shift;
  if ((int64_t{1} << shift) != page_tokens)
    return fail(COWSDM_EARG, "%s: page tokens must be 16, 32, 64, 128 or 256", where);
  return 0;
}

constexpr int64_t kMostChunk = int64_t{1} << 22;    // chunk_of(2^31)

// Sizes that every table operator has; n rows of `columns` entries.
int32_t check_tables(int64_t requests, int64_t columns, int64_t pages, int64_t n,
                     int64_t page_tokens, const char* where) {
  if (requests < 0 || columns < 0 || pages < 0 || n < 0)
    return fail(COWSDM_EARG, "%s: negative size", where);
  if (n > kPageNamed)
    return fail(COWSDM_ELIMIT, "%s: at most %d requests a call", where, kPageNamed);
  if (requests > INT32_MAX) return fail(COWSDM_ELIMIT, "%s: too large", where);
  if (pages > INT32_MAX / page_tokens || columns > INT32_MAX / page_tokens)
    return fail(COWSDM_ELIMIT, "%s: more than 2^31 tokens", where);
  const int64_t rows = requests > n ? requests : n;
  if (columns > 0 && rows > (INT32_MAX - kMostChunk) / columns)
    return fail(COWSDM_ELIMIT, "%s: 2^31 table entries or more", where);
  return 0;
}

uint32_t groups_of(int64_t numbers) {
  const int64_t n = (numbers + kPageThreads - 1) / kPageThreads;
  return static_cast<uint32_t>(n < 1 ? 1 : n > 4096 ? 4096 : n);
}

// Numbers that a workgroup counts and then places in order: one a thread, or
// more where 1,024 workgroups would not do, each of which adds up the others'
// counts.
int64_t chunk_of(int64_t numbers) {
  const int64_t each = (numbers + kPageThreads * 1024 - 1) / (kPageThreads * 1024);
  return kPageThreads * (each < 1 ? 1 : each);
}

int64_t chunks_of(int64_t numbers) {
  return numbers <= kPageThreads ? 1 : (numbers + chunk_of(numbers) - 1) / chunk_of(numbers);
}

// Dynamic LDS past what a kernel may have by itself, beside its own.
int32_t allow_lds(const void* kernel, int bytes, const char* where) {
  if (bytes <= 32 * 1024) return 0;
  const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           bytes);
  return e == hipSuccess ? 0
                         : fail(static_cast<int32_t>(e), "%s: %s", where, hipGetErrorString(e));
}

}  // namespace cowsdm_impl

using namespace cowsdm_impl;

extern "C" int32_t cowsdm_page_tables_fork(
    const int32_t* lengths, const int32_t* page_tables, int64_t requests, int64_t columns,
    const int32_t* page_shares, const int32_t* free_pages, int64_t pages,
    const int32_t* free_count, const int32_t* parents, const int32_t* tokens, int64_t children,
    int64_t page_tokens, int32_t* lengths_out, int32_t* tables_out, int32_t* shares_out,
    int32_t* free_count_out, int32_t* sources, int32_t* targets, int32_t* overflow,
    void* stream) {
  int shift;
  if (int32_t e = page_shift_of(page_tokens, "page_tables_fork", shift)) return e;
  if (int32_t e = check_tables(requests, columns, pages, children, page_tokens,
                               "page_tables_fork"))
    return e;
  if (!free_count || !free_count_out || !overflow ||
      (pages > 0 && (!page_shares || !shares_out || !free_pages)) ||
      (children > 0 && (!parents || !tokens || !lengths_out || !sources || !targets ||
                        (columns > 0 && !tables_out))) ||
      (requests > 0 && (!lengths || (columns > 0 && !page_tables))))
    return fail(COWSDM_EARG, "page_tables_fork: null pointer argument");
  ForkParams p{lengths, page_tables, page_shares, free_pages, free_count, parents, tokens,
               lengths_out, tables_out, shares_out, free_count_out, sources, targets, overflow,
               static_cast<int32_t>(requests), static_cast<int32_t>(columns),
               static_cast<int32_t>(pages), static_cast<int32_t>(children), shift};
  const auto s = static_cast<hipStream_t>(stream);
  const int64_t entries = children * columns;
  if (entries <= kOneNumbers && pages <= kOnePages && children <= kOneNamed) {
    const int bytes = static_cast<int>(4 * pages);
    if (int32_t e = allow_lds(reinterpret_cast<const void*>(&fork_one_kernel), bytes,
                              "page_tables_fork"))
      return e;
    hipLaunchKernelGGL(fork_one_kernel, dim3(1), dim3(kOneThreads), bytes, s, p);
    return launch_status("page_tables_fork");
  }
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1 + groups_of(pages)), dim3(kPageThreads), 0, s, p);
  if (int32_t e = launch_status("page_tables_fork")) return e;
  hipLaunchKernelGGL(fork_tables_kernel, dim3(groups_of(entries)), dim3(kPageThreads), 0, s, p);
  return launch_status("page_tables_fork");
}

extern "C" int64_t cowsdm_page_tables_release_workspace_bytes(int64_t pages, int64_t columns,
                                                              int64_t n) {
  if (pages < 0 || columns < 0 || n < 0 || pages > INT32_MAX || columns > INT32_MAX ||
      n > kPageNamed)
    return -1;
  return 4 * (pages + n + chunks_of(n * columns));
}

extern "C" int32_t cowsdm_page_tables_release(
    const int32_t* lengths, const int32_t* page_tables, int64_t requests, int64_t columns,
    const int32_t* page_shares, int32_t* free_pages, int64_t pages, const int32_t* free_count,
    const int32_t* named, int64_t n, int64_t page_tokens, int32_t* lengths_out,
    int32_t* shares_out, int32_t* free_count_out, void* workspace, int64_t workspace_bytes,
    void* stream) {
  int shift;
  if (int32_t e = page_shift_of(page_tokens, "page_tables_release", shift)) return e;
  if (int32_t e = check_tables(requests, columns, pages, n, page_tokens, "page_tables_release"))
    return e;
  const int64_t need = cowsdm_page_tables_release_workspace_bytes(pages, columns, n);
  if (!free_count || !free_count_out || (n > 0 && !named) ||
      (pages > 0 && (!page_shares || !shares_out || !free_pages)) ||
      (requests > 0 && (!lengths || !lengths_out || (columns > 0 && !page_tables))))
    return fail(COWSDM_EARG, "page_tables_release: null pointer argument");
  if (!workspace || workspace_bytes < need)
    return fail(COWSDM_EARG, "page_tables_release: workspace of %lld bytes needed",
                static_cast<long long>(need));
  int32_t* const last = static_cast<int32_t*>(workspace);
  const int64_t entries = n * columns, chunks = chunks_of(entries);
  ReleaseParams p{lengths, page_tables, page_shares, free_count, named, free_pages, lengths_out,
                  shares_out, free_count_out, last, last + pages, last + pages + n,
                  static_cast<int32_t>(requests), static_cast<int32_t>(columns),
                  static_cast<int32_t>(pages), static_cast<int32_t>(n),
                  static_cast<int32_t>(entries), static_cast<int32_t>(chunks),
                  static_cast<int32_t>(chunk_of(entries)), shift};
  const auto s = static_cast<hipStream_t>(stream);
  const auto groups = dim3(static_cast<uint32_t>(p.chunks));
  if (entries <= kOneNumbers && pages <= kOnePages && n <= kOneNamed &&
      requests <= kOneRequests) {
    const int bytes = static_cast<int>(8 * pages);
    if (int32_t e = allow_lds(reinterpret_cast<const void*>(&release_one_kernel), bytes,
                              "page_tables_release"))
      return e;
    hipLaunchKernelGGL(release_one_kernel, dim3(1), dim3(kOneThreads), bytes, s, p);
    return launch_status("page_tables_release");
  }
  hipLaunchKernelGGL(release_plan_kernel, dim3(1 + groups_of(pages)), dim3(kPageThreads), 0, s,
                     p);
  if (int32_t e = launch_status("page_tables_release")) return e;
  hipLaunchKernelGGL(release_take_kernel, dim3(groups_of(entries)), dim3(kPageThreads), 0, s, p);
  if (int32_t e = launch_status("page_tables_release")) return e;
  hipLaunchKernelGGL(release_count_kernel, groups, dim3(kPageThreads), 0, s, p);
  if (int32_t e = launch_status("page_tables_release")) return e;
  hipLaunchKernelGGL(release_push_kernel, groups, dim3(kPageThreads), 0, s, p);
  return launch_status("page_tables_release");
}

extern "C" int64_t cowsdm_page_tables_compact_workspace_bytes(int64_t pages) {
  if (pages < 0 || pages > INT32_MAX) return -1;
  return 4 * (pages + chunks_of(pages));
}

extern "C" int32_t cowsdm_page_tables_compact(
    const int32_t* lengths, const int32_t* page_tables, int64_t requests, int64_t columns,
    const int32_t* page_shares, int64_t pages, int64_t page_tokens, int32_t* tables_out,
    int32_t* shares_out, int32_t* free_pages_out, int32_t* free_count_out, int32_t* sources,
    int32_t* targets, void* workspace, int64_t workspace_bytes, void* stream) {
  int shift;
  if (int32_t e = page_shift_of(page_tokens, "page_tables_compact", shift)) return e;
  if (int32_t e = check_tables(requests, columns, pages, 0, page_tokens, "page_tables_compact"))
    return e;
  const int64_t need = cowsdm_page_tables_compact_workspace_bytes(pages);
  if (!free_count_out || (pages > 0 && (!page_shares || !shares_out || !free_pages_out)) ||
      (pages > 1 && (!sources || !targets)) ||
      (requests > 0 && (!lengths || (columns > 0 && (!page_tables || !tables_out)))))
    return fail(COWSDM_EARG, "page_tables_compact: null pointer argument");
  if (!workspace || workspace_bytes < need)
    return fail(COWSDM_EARG, "page_tables_compact: workspace of %lld bytes needed",
                static_cast<long long>(need));
  int32_t* const used = static_cast<int32_t*>(workspace);
  const int64_t entries = requests * columns, chunks = chunks_of(pages);
  CompactParams p{lengths, page_tables, page_shares, tables_out, shares_out, free_pages_out,
                  free_count_out, sources, targets, used, used + pages,
                  static_cast<int32_t>(requests), static_cast<int32_t>(columns),
                  static_cast<int32_t>(pages), static_cast<int32_t>(entries),
                  static_cast<int32_t>(chunks), static_cast<int32_t>(chunk_of(pages)), shift};
  const auto s = static_cast<hipStream_t>(stream);
  if (entries <= kOneNumbers && pages <= kOnePages) {
    const int bytes = static_cast<int>(8 * pages);
    if (int32_t e = allow_lds(reinterpret_cast<const void*>(&compact_one_kernel), bytes,
                              "page_tables_compact"))
      return e;
    hipLaunchKernelGGL(compact_one_kernel, dim3(1), dim3(kOneThreads), bytes, s, p);
    return launch_status("page_tables_compact");
  }
  const auto groups = dim3(static_cast<uint32_t>(chunks));
  const auto threads = dim3(kPageThreads);
  hipLaunchKernelGGL(compact_clear_kernel, dim3(groups_of(pages)), threads, 0, s, p);
  if (int32_t e = launch_status("page_tables_compact")) return e;
  hipLaunchKernelGGL(compact_mark_kernel, dim3(groups_of(entries)), threads, 0, s, p);
  if (int32_t e = launch_status("page_tables_compact")) return e;
  hipLaunchKernelGGL(compact_count_kernel, groups, threads, 0, s, p);
  if (int32_t e = launch_status("page_tables_compact")) return e;
  hipLaunchKernelGGL(compact_place_kernel, groups, threads, 0, s, p);
  if (int32_t e = launch_status("page_tables_compact")) return e;
  hipLaunchKernelGGL(compact_rewrite_kernel, dim3(groups_of(entries > pages ? entries : pages)),
                     threads, 0, s, p);
  return launch_status("page_tables_compact");
}

extern "C" int32_t cowsdm_pages_copy(const cowsdm_kv_cache_t* cache, int64_t layers,
                                     const int32_t* sources, const int32_t* targets, int64_t n,
                                     void* stream) {
  if (!cache) return fail(COWSDM_EARG, "pages_copy: null cache");
  const cowsdm_kv_cache_t& c = *cache;
  if (layers < 0 || n < 0 || c.pages < 0 || c.heads <= 0 || c.width <= 0)
    return fail(COWSDM_EARG, "pages_copy: bad size");
  int shift;
  if (int32_t e = page_shift_of(c.page_tokens, "pages_copy", shift)) return e;
  if (c.width % 32 != 0 || c.width > 256)
    return fail(COWSDM_EARG, "pages_copy: cache width must be 32, 64, 96, 128, 192 or 256");
  if (c.pages > INT32_MAX / c.page_tokens)
    return fail(COWSDM_ELIMIT, "pages_copy: more than 2^31 tokens of pages");
  if (c.heads > 65535 || layers > 65535)
    return fail(COWSDM_ELIMIT, "pages_copy: at most 65,535 heads and layers");
  if (n == 0 || layers == 0 || c.pages == 0) return 0;
  if (!sources || !targets || !c.key_codes || !c.value_codes || !c.key_scales || !c.value_scales)
    return fail(COWSDM_EARG, "pages_copy: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(c.key_codes) | reinterpret_cast<uintptr_t>(c.value_codes)) % 16)
    return fail(COWSDM_EARG, "pages_copy: cache codes must be 16-byte aligned");
  const int64_t bytes = c.heads * c.page_tokens * c.width;
  const int64_t parts = (bytes + kCopyBytes - 1) / kCopyBytes;
  // a launch counts its threads in 32 bits
  if (2 * parts * n > UINT32_MAX / kCopyThreads)
    return fail(COWSDM_ELIMIT, "pages_copy: too many pages a call");
  CopyParams p{static_cast<page_words*>(c.key_codes), static_cast<page_words*>(c.value_codes),
               c.key_scales, c.value_scales, sources, targets, static_cast<int32_t>(c.pages),
               static_cast<int32_t>(c.heads), static_cast<int32_t>(bytes / 16),
               static_cast<int32_t>(parts)};
  hipLaunchKernelGGL(copy_pages_kernel,
                     dim3(static_cast<uint32_t>(2 * parts * n), static_cast<uint32_t>(layers)),
                     dim3(kCopyThreads), 0, static_cast<hipStream_t>(stream), p);
  return launch_status("pages_copy");
}
