// Pages of a paged cache on gfx950 (MI355X): who holds them, and their copies. HIP kernels and the C ABI of
// the pages section of include/mkmoe.h.
//
// A pool holds for every page how many sequences hold it (refs), and for every block of 1024 pages how many
// are free. A sequence of len tokens holds the pages that the first ceil(len / page_size) entries of its row of
// the table name. Full pages may be held by several sequences; a page that is partly filled by one alone,
// because its next token is written there: fork and trim give a sequence a copy of its own where it
// would be shared. Pages are taken lowest first, in the order of the sequences, whatever the card does first, so
// that the same calls give the same tables.
//
//   k_pages_clear / _hold / _count   a pool from tables (adopt)
//   k_pages_take     the pages that a call takes: grow's whole work, trim's and fork's first half
//   k_pages_trim / _fork / _compact  their second halves: counts, tables, copies of pages
//   k_pages_plan     which pages move where (compact)
//   k_pages_copy     pages that the caller names
//
// A call with few pages is bound by its launches (3 to 7 us each of dependent reads: lengths, counts, pages, tables),
// others by the pages' bytes, read and written once: 301 pages of 24 caches copied in 127 us, 4.8 TB/s, where
// a copy of 2 GiB reaches 4.9 on this card.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/mkmoe.h"

namespace mkmoe_pages {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kBlock = 1024;  // pages a block: 4 a thread
constexpr int kMaxPages = 1 << 22, kMaxBlocks = kMaxPages / kBlock;
constexpr int kMaxSeqs = MKMOE_PAGES_MAX_SEQS;
constexpr int kChunk = 1024;  // 16-byte pieces that a workgroup copies at a time: 4 a thread

// the words at the head of a workspace, behind the error words
struct Head {
  int32_t err[4];
  int32_t arrived;  // workgroups of k_pages_take that are done; 0 between launches
  int32_t moves;    // pages that the launch behind copies: src[i] to dst[i]
  int32_t live;     // compact: pages held
  int32_t missing;  // compact: holders that the table does not have; 0 between calls
  int32_t refused;  // compact: that many, and nothing is moved
};
static_assert(sizeof(Head) <= MKMOE_PAGES_REFS_AT, "the counts follow the head");

enum { kGrow, kTrim, kFork };

struct Params {
  Head* head;
  int32_t* refs;      // [pages]
  int32_t* free_in;   // [blocks]
  int32_t* src;       // [pages]
  int32_t* dst;       // [pages]
  int32_t* rank;      // [pages] compact: a moved page's place in src
  int32_t* old_len;   // [seqs]
  int32_t* new_len;   // [seqs]
  int32_t* new_page;  // [seqs] a page that the sequence got, -1 none
  int32_t* kids;      // [seqs] fork: the rows that go on from a row
  int32_t* held;      // [seqs][max_pages] fork: the table as it was
  int32_t* table;
  int32_t* lens;
  const int32_t* arg;  // grow: added tokens; trim: lengths to keep; fork: parents
  int32_t* slots;
  int32_t* positions;
  int32_t* starts;
  const mkmoe_pages_cache* caches;
  int64_t table_stride;
  int pages, blocks, seqs, max_pages, page_size, shift, ncaches, tokens;
};

__device__ inline void record(Head* h, int code, int where) {
  if (atomicCAS(h->err + MKMOE_PAGES_ERRW_CODE, 0, code) == 0) h->err[MKMOE_PAGES_ERRW_WHERE] = where;
  atomicAdd(h->err + MKMOE_PAGES_ERRW_COUNT, 1);
}
__device__ __forceinline__ int pages_for(const Params& p, int len) { return (int)(((int64_t)len + p.page_size - 1) >> p.shift); }
__device__ __forceinline__ int clamped(const Params& p, int len) {
  return (int)min((int64_t)max(len, 0), (int64_t)p.max_pages << p.shift);
}
// Pages' sequences let go of them, a page a lane (where there is one). The blocks' free pages are counted a wave at a
// time: an atomic addition for each page took 310 us where 98000 that follow each other were freed, so 7
__device__ __forceinline__ void release(const Params& p, bool there, int page, int where) {
  bool freed = false;
  if (there && (uint32_t)page >= (uint32_t)p.pages) {
    record(p.head, MKMOE_PAGES_ERR_PAGE, where);
  } else if (there) {
    const int was = atomicSub(p.refs + page, 1);
    freed = was == 1;
    if (was < 1) {  // nobody held it
      atomicAdd(p.refs + page, 1);
      record(p.head, MKMOE_PAGES_ERR_PAGE, where);
    }
  }
  const int block = page / kBlock;
  for (uint64_t left = __ballot(freed); left != 0;) {
    const int first = __builtin_ctzll(left);
    const uint64_t same = __ballot(freed && block == __builtin_amdgcn_readlane(block, first));
    if ((int)(threadIdx.x & 63) == first) atomicAdd(p.free_in + block, __builtin_popcountll(same));
    left &= ~same;
  }
}

// A held page gets more holders. One that nobody holds stays free: a table may name what it does not hold
__device__ __forceinline__ void hold(const Params& p, int page, int more, int where) {
  int was = __hip_atomic_load(p.refs + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  while (was > 0) {
    const int seen = atomicCAS(p.refs + page, was, was + more);
    if (seen == was) return;
    was = seen;
  }
  record(p.head, MKMOE_PAGES_ERR_PAGE, where);
}

// the sum of v over the threads before this one, and over all of them
template <class T>
__device__ __forceinline__ T scan(T v, T* total, T* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T x = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < wave) before += lds[i];
    all += lds[i];
  }
  *total = all;
  return before + x - v;
}

// ---------------------------------------------------------------- a pool from tables
__global__ __launch_bounds__(kThreads) void k_pages_clear(Params p) {
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < p.pages; i += gridDim.x * kThreads) p.refs[i] = 0;
}
__global__ __launch_bounds__(kThreads) void k_pages_hold(Params p) {
  const int b = blockIdx.x, len = clamped(p, p.lens[b]);
  if (threadIdx.x == 0 && blockIdx.y == 0 && len != p.lens[b]) record(p.head, MKMOE_PAGES_ERR_BOUNDS, b);
  const int n = pages_for(p, len);
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < n; i += gridDim.y * kThreads) {
    const int page = p.table[b * p.table_stride + i];
    if ((uint32_t)page < (uint32_t)p.pages)
      atomicAdd(p.refs + page, 1);
    else
      record(p.head, MKMOE_PAGES_ERR_PAGE, b);
  }
}
// the free pages of each block, and pages that are partly filled and shared
__global__ __launch_bounds__(kThreads) void k_pages_count(Params p) {
  __shared__ int sums[kThreads / 64];
  for (int j = blockIdx.x; j < p.blocks; j += gridDim.x) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int page = j * kBlock + i * kThreads + threadIdx.x;
      n += page < p.pages && p.refs[page] == 0;
    }
    int all;
    (void)scan(n, &all, sums);
    if (threadIdx.x == 0) p.free_in[j] = all;
  }
  for (int b = blockIdx.x * kThreads + threadIdx.x; b < p.seqs; b += gridDim.x * kThreads) {
    const int len = clamped(p, p.lens[b]);
    if ((len & (p.page_size - 1)) == 0) continue;
    const int page = p.table[b * p.table_stride + (len >> p.shift)];
    if ((uint32_t)page < (uint32_t)p.pages && p.refs[page] > 1) record(p.head, MKMOE_PAGES_ERR_SHARED, b);
  }
}

// ---------------------------------------------------------------- pages taken
struct TakeSmem {
  int before[kMaxBlocks];    // free pages before each block
  int first[kMaxSeqs];       // the rank of a sequence's first taken page
  int from[kMaxSeqs + 1];    // grow: its first token
  int len[kMaxSeqs];         // its length
  int to[kMaxSeqs];          // its new length, that it has if it is served
  int lead[kMaxSeqs];        // fork: the first row that goes on from a row; then how many do
  int page[kBlock];          // grow: a block's taken pages
  int at[kBlock];            // the first position of each one's tokens
  int seq[kBlock];
  int64_t sums64[kThreads / 64];
  int sums[kThreads / 64];
  int taken, last;
};

// What each sequence needs and gets: every workgroup finds that out for itself, from the lengths and the
// blocks' free pages, then takes the pages of its own blocks. So a block's counts are read and written by one
// workgroup, and no order of arrival shows in the result. Lengths and the blocks' counts are read by
// all: the last workgroup to be done writes them.
template <int OP>
__global__ __launch_bounds__(kThreads) void k_pages_take(Params p) {
  __shared__ TakeSmem sm;
  const int tid = threadIdx.x;
  // (the first sequences' values, on their way meanwhile)
  const int len0 = tid < p.seqs ? p.lens[tid] : 0, arg0 = tid < p.seqs ? p.arg[tid] : 0;
  // free pages before each block
  int free_pages = 0;
  for (int j0 = 0; j0 < p.blocks; j0 += kThreads) {
    const int j = j0 + tid;
    int all;
    const int before = scan(j < p.blocks ? p.free_in[j] : 0, &all, sm.sums);
    if (j < p.blocks) sm.before[j] = free_pages + before;
    free_pages += all;
  }
  if (tid == 0) sm.taken = 0;
  if constexpr (OP == kFork) {
    for (int b = tid; b < p.seqs; b += kThreads) sm.lead[b] = p.seqs;
    __syncthreads();
    for (int b = tid; b < p.seqs; b += kThreads) {
      const int r = b < kThreads ? arg0 : p.arg[b];
      if ((uint32_t)r < (uint32_t)p.seqs) atomicMin(&sm.lead[r], b);
    }
  }
  __syncthreads();
  // what each sequence needs, in order
  int64_t tokens = 0, needed = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    const bool there = b < p.seqs;
    int len = 0, to = 0, need = 0, add = 0;
    bool room = true;
    if (there) {
      const int raw = b0 == 0 ? len0 : p.lens[b], arg = b0 == 0 ? arg0 : p.arg[b];
      len = to = clamped(p, raw);
      if (len != raw && blockIdx.x == 0) record(p.head, MKMOE_PAGES_ERR_BOUNDS, b);
      if constexpr (OP == kGrow) {
        add = max(arg, 0);
        if (arg < 0 && blockIdx.x == 0) record(p.head, MKMOE_PAGES_ERR_BOUNDS, b);
      } else if constexpr (OP == kTrim) {
        to = min(len, max(arg, 0));
        if (to < len && (to & (p.page_size - 1)) != 0) {
          const int page = p.table[b * p.table_stride + (to >> p.shift)];
          need = (uint32_t)page < (uint32_t)p.pages && p.refs[page] > 1;
        }
      } else {
        const bool some = (uint32_t)arg < (uint32_t)p.seqs;
        if (!some && arg != -1 && blockIdx.x == 0) record(p.head, MKMOE_PAGES_ERR_BOUNDS, b);
        to = some ? clamped(p, p.lens[arg]) : 0;
        need = some && (to & (p.page_size - 1)) != 0 && sm.lead[arg] != b;
      }
    }
    int64_t all;
    if constexpr (OP == kGrow) {
      const int64_t from = tokens + scan((int64_t)add, &all, sm.sums64);
      tokens += all;
      room = (int64_t)len + add <= (int64_t)p.max_pages << p.shift && from + add <= p.tokens;
      if (room) {
        to = len + add;
        need = pages_for(p, to) - pages_for(p, len);
      }
      if (there) {
        sm.from[b] = (int)min(from, (int64_t)p.tokens);
        if (!room && blockIdx.x == 0) record(p.head, MKMOE_PAGES_ERR_ROOM, b);
      }
    }
    const int64_t first = needed + scan((int64_t)need, &all, sm.sums64);
    needed += all;
    const bool full = need > 0 && first + need > free_pages;
    if (there) {
      if (full && blockIdx.x == 0) record(p.head, MKMOE_PAGES_ERR_FULL, b);
      if (full) to = OP == kFork ? -1 : len;
      sm.first[b] = (int)min(first, (int64_t)free_pages);
      sm.len[b] = len;
      sm.to[b] = to;
      if (need > 0 && !full) atomicMax(&sm.taken, (int)(first + need));
    }
  }
  if (OP == kGrow && tid == 0) sm.from[p.seqs] = (int)min(tokens, (int64_t)p.tokens);
  __syncthreads();
  const int taken = sm.taken;

  // the pages of this workgroup's blocks
  for (int j = blockIdx.x; j < p.blocks; j += gridDim.x) {
    const int before = sm.before[j];
    if (before >= taken) break;  // (in order)
    if ((j + 1 < p.blocks ? sm.before[j + 1] : free_pages) == before) continue;
    i32x4 refs = {1, 1, 1, 1};
    const int page0 = j * kBlock + 4 * tid;
    if (page0 + 4 <= p.pages)
      refs = *(const i32x4*)(p.refs + page0);
    else
      for (int i = 0; i < 4; ++i)
        if (page0 + i < p.pages) refs[i] = p.refs[page0 + i];
    int n = 0;
    for (int i = 0; i < 4; ++i) n += refs[i] == 0;
    int all;
    int r = before + scan(n, &all, sm.sums);
    const int count = min(all, taken - before);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (refs[i] != 0) continue;
      const int mine = r++;
      if (mine >= taken) continue;
      int lo = 0, hi = p.seqs - 1;  // the last sequence whose first rank is not past it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sm.first[mid] <= mine) lo = mid; else hi = mid - 1;
      }
      const int page = page0 + i;
      p.refs[page] = 1;
      if constexpr (OP == kGrow) {
        const int entry = pages_for(p, sm.len[lo]) + mine - sm.first[lo];
        p.table[lo * p.table_stride + entry] = page;
        sm.page[mine - before] = page;
        sm.at[mine - before] = entry << p.shift;
        sm.seq[mine - before] = lo;
      } else {
        p.new_page[lo] = page;
        p.dst[mine] = page;
      }
    }
    if constexpr (OP == kGrow) {
      __syncthreads();
      for (int x = tid; x < count << p.shift; x += kThreads) {
        const int i = x >> p.shift, at = sm.at[i] + (x & (p.page_size - 1)), b = sm.seq[i];
        if (at < sm.to[b]) {
          const int t = sm.from[b] + at - sm.len[b];
          p.slots[t] = (sm.page[i] << p.shift) + (x & (p.page_size - 1));
          p.positions[t] = at;
        }
      }
      __syncthreads();
    }
  }

  if constexpr (OP == kGrow) {
    // the tokens that go into the page before, and those that have no place
    for (int t = blockIdx.x * kThreads + tid; t < p.tokens; t += gridDim.x * kThreads) {
      int lo = 0, hi = p.seqs;  // the last sequence that starts at or before it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sm.from[mid] <= t) lo = mid; else hi = mid - 1;
      }
      int slot = -1, at = 0;
      if (lo < p.seqs && sm.to[lo] > sm.len[lo]) {
        at = sm.len[lo] + t - sm.from[lo];
        if (at >= pages_for(p, sm.len[lo]) << p.shift) continue;  // (in a taken page)
        const int page = p.table[lo * p.table_stride + (at >> p.shift)];
        if ((uint32_t)page < (uint32_t)p.pages)
          slot = (page << p.shift) + (at & (p.page_size - 1));
        else
          record(p.head, MKMOE_PAGES_ERR_PAGE, lo);
      }
      p.slots[t] = slot;
      p.positions[t] = at;
    }
    if (blockIdx.x == gridDim.x - 1)
      for (int b = tid; b <= p.seqs; b += kThreads) p.starts[b] = sm.from[b];
  } else if (blockIdx.x == gridDim.x - 1) {
    for (int b = tid; b < p.seqs; b += kThreads) {
      p.old_len[b] = sm.len[b];
      p.new_len[b] = sm.to[b];
      // (no page was taken for it where the next one's first rank is its own)
      if ((b + 1 < p.seqs ? sm.first[b + 1] : taken) <= sm.first[b] || sm.first[b] >= taken) {
        p.new_page[b] = -1;
      } else {
        const int row = OP == kTrim ? b : p.arg[b];
        p.src[sm.first[b]] = p.table[row * p.table_stride + (sm.to[b] >> p.shift)];
      }
    }
    if (tid == 0) p.head->moves = taken;
  }
  if constexpr (OP == kFork) {
    // the rows as they are, for those that go on from them
    for (int b = blockIdx.x; b < p.seqs; b += gridDim.x) {
      const int n = pages_for(p, sm.len[b]);
      for (int i = tid; i < n; i += kThreads) p.held[(int64_t)b * p.max_pages + i] = p.table[b * p.table_stride + i];
    }
    if (blockIdx.x == gridDim.x / 2) {
      for (int b = tid; b < p.seqs; b += kThreads) sm.lead[b] = 0;
      __syncthreads();
      for (int b = tid; b < p.seqs; b += kThreads) {
        const int r = p.arg[b];
        if ((uint32_t)r < (uint32_t)p.seqs && sm.to[b] >= 0) atomicAdd(&sm.lead[r], 1);
      }
      __syncthreads();
      for (int b = tid; b < p.seqs; b += kThreads) p.kids[b] = sm.lead[b];
    }
  }

  // the last one to be done: nobody reads what it writes any more
  __syncthreads();
  if (gridDim.x > 1) {
    if (tid == 0) {
      __threadfence();
      sm.last = atomicAdd(&p.head->arrived, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!sm.last) return;
    __threadfence();
    if (tid == 0) p.head->arrived = 0;
  }
  for (int j = tid; j < p.blocks; j += kThreads) {
    const int before = sm.before[j];
    if (before >= taken) break;
    p.free_in[j] -= min(taken, j + 1 < p.blocks ? sm.before[j + 1] : free_pages) - before;
  }
  if constexpr (OP == kGrow)
    for (int b = tid; b < p.seqs; b += kThreads) p.lens[b] = sm.to[b];
}

// ---------------------------------------------------------------- pages copied
// Pages src[i] to dst[i] of every cache, 16 KB a workgroup and turn; pages outside the pool are left out. The caches'
// chunks follow each other, so that few pages keep every workgroup at work, and the caches' places are in LDS: read one
// after the other, 24 of them took 25 us where there was nothing to copy
constexpr int kCaches = 128;  // places in LDS
__device__ __forceinline__ void copy_pages(const Params& p, const int32_t* src, const int32_t* dst, int n, bool check) {
  __shared__ mkmoe_pages_cache place[kCaches];
  __shared__ int64_t before[kCaches + 1], sums[kThreads / 64];
  if (n == 0) return;
  const int tid = threadIdx.x;
  const int64_t groups = gridDim.x * gridDim.y, me = blockIdx.y * gridDim.x + blockIdx.x;
  for (int c0 = 0; c0 < p.ncaches; c0 += kCaches) {
    const int some = min(kCaches, p.ncaches - c0);
    __syncthreads();
    int64_t mine = 0, all;
    if (tid < some) {
      place[tid] = p.caches[c0 + tid];
      mine = (n * (place[tid].page_bytes / 16) + kChunk - 1) / kChunk;
    }
    const int64_t first = scan(mine, &all, sums);
    if (tid < some) before[tid] = first;
    if (tid == 0) before[some] = all;
    __syncthreads();
    int c = 0;
    for (int64_t k = me; k < all; k += groups) {
      while (before[c + 1] <= k) ++c;
      const mkmoe_pages_cache cache = place[c];
      const uint32_t q = (uint32_t)(cache.page_bytes / 16);
      const int64_t base = (k - before[c]) * kChunk, i0 = base / q;
      const uint32_t rest = (uint32_t)(base - i0 * q);
      // (the places first, then the bytes: loads complete in order, and one behind a place's would wait for it)
      uint32_t part[4];
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = rest + i * kThreads + tid;
        const int64_t at = i0 + x / q;
        part[i] = x % q;
        a[i] = b[i] = -1;
        if (at < n) a[i] = src[at], b[i] = dst[at];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool out = (uint32_t)a[i] >= (uint32_t)p.pages || (uint32_t)b[i] >= (uint32_t)p.pages;
        const int64_t at = i0 + (rest + i * kThreads + tid) / q;
        if (check && out && at < n && part[i] == 0 && c0 + c == 0) record(p.head, MKMOE_PAGES_ERR_PAGE, (int)at);
        if (out) a[i] = -1;
      }
      u32x4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (a[i] >= 0) v[i] = *(const u32x4*)((const uint8_t*)cache.data + a[i] * cache.page_bytes + part[i] * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (a[i] >= 0) *(u32x4*)((uint8_t*)cache.data + b[i] * cache.page_bytes + part[i] * 16) = v[i];
    }
  }
}
__global__ __launch_bounds__(kThreads) void k_pages_copy(Params p, const int32_t* src, const int32_t* dst, int n) {
  copy_pages(p, src, dst, n, true);
}

// ---------------------------------------------------------------- second halves
__global__ __launch_bounds__(kThreads) void k_pages_trim(Params p) {
  const int b = blockIdx.x, len = p.old_len[b], to = p.new_len[b], page = p.new_page[b];
  // entries from the first one that is not kept, or that gets a page of its own
  const int first = pages_for(p, to) - (page >= 0), end = pages_for(p, len);
  for (int i0 = first + blockIdx.y * kThreads; i0 < end; i0 += gridDim.y * kThreads) {
    const int i = i0 + threadIdx.x;
    int32_t* at = p.table + b * p.table_stride + i;
    release(p, i < end, i < end ? *at : 0, b);
    if (page >= 0 && i == first) *at = page;
  }
  if (threadIdx.x == 0 && blockIdx.y == 0) p.lens[b] = to;
  copy_pages(p, p.src, p.dst, p.head->moves, true);
}

__global__ __launch_bounds__(kThreads) void k_pages_fork(Params p) {
  const int b = blockIdx.x;
  // as a parent: its full pages are held by each row that goes on, a last one that is not full by the first
  const int len = p.old_len[b], full = len >> p.shift, end = pages_for(p, len), kids = p.kids[b];
  const int32_t* held = p.held + (int64_t)b * p.max_pages;
  for (int i0 = blockIdx.y * kThreads; i0 < end && kids != 1; i0 += gridDim.y * kThreads) {
    const int i = i0 + threadIdx.x, page = i < end ? held[i] : 0;
    if (kids == 0)
      release(p, i < end, page, b);
    else if (i < full && (uint32_t)page < (uint32_t)p.pages)
      hold(p, page, kids - 1, b);
  }
  // as a row that goes on
  const int to = max(p.new_len[b], 0), own = p.new_page[b], parent = p.arg[b];
  if (parent != b && to > 0) {
    const int32_t* from = p.held + (int64_t)parent * p.max_pages;
    const int n = pages_for(p, to);
    for (int i = blockIdx.y * kThreads + threadIdx.x; i < n; i += gridDim.y * kThreads)
      p.table[b * p.table_stride + i] = own >= 0 && i == n - 1 ? own : from[i];
  }
  if (own >= 0 && parent == b && threadIdx.x == 0 && blockIdx.y == 0) p.table[b * p.table_stride + (to >> p.shift)] = own;
  if (threadIdx.x == 0 && blockIdx.y == 0) p.lens[b] = to;
  copy_pages(p, p.src, p.dst, p.head->moves, true);
}

// Compact: of n pages held, those at n and behind go to the free ones before n, both in order. A workgroup
// finds its blocks' pages and their ranks. The pages' holders are counted against the table's entries: a row that the
// table does not have would be left with pages that are others' afterwards, so then nothing is moved.
__global__ __launch_bounds__(kThreads) void k_pages_plan(Params p) {
  __shared__ int before[kMaxBlocks];
  __shared__ int sums[kThreads / 64];
  const int tid = threadIdx.x;
  int free_pages = 0;
  for (int j0 = 0; j0 < p.blocks; j0 += kThreads) {
    const int j = j0 + tid;
    int all;
    const int at = scan(j < p.blocks ? p.free_in[j] : 0, &all, sums);
    if (j < p.blocks) before[j] = free_pages + at;
    free_pages += all;
  }
  __syncthreads();
  const int live = p.pages - free_pages;
  if (blockIdx.x == 0 && tid == 0) p.head->live = live;
  // the pages' holders, less those that the table has
  int missing = 0;
  for (int b = blockIdx.x; b < p.seqs; b += gridDim.x) {
    const int n = pages_for(p, clamped(p, p.lens[b]));
    for (int i = tid; i < n; i += kThreads) missing -= (uint32_t)p.table[b * p.table_stride + i] < (uint32_t)p.pages;
  }
  for (int j = blockIdx.x; j < p.blocks; j += gridDim.x) {
    int n = 0, used[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int page = j * kBlock + 4 * tid + i, refs = page < p.pages ? p.refs[page] : 0;
      used[i] = page < p.pages ? refs != 0 : 2;
      n += used[i] == 0;
      missing += refs;
    }
    int all;
    int frees = before[j] + scan(n, &all, sums);  // free pages before this one
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int page = j * kBlock + 4 * tid + i;
      if (used[i] == 2) continue;
      // of the pages at live and behind, held ones before this one: all held ones before it, less those before live,
      // of which there are as many as the free ones there are not
      if (page == live) p.head->moves = frees;  // (free pages before live: as many as move)
      if (used[i] == 0) {
        if (page < live) p.dst[frees] = page;
        ++frees;
      } else if (page >= live) {
        // held before it: page - frees; held before live: live - moves. Its rank among those that move is
        // the difference, left for the second half, which knows moves
        p.rank[page] = page - frees - live;
      }
    }
  }
  if (live == p.pages && blockIdx.x == 0 && tid == 0) p.head->moves = 0;
  int all;
  (void)scan(missing, &all, sums);
  if (tid == 0 && all != 0) atomicAdd(&p.head->missing, all);
}
__global__ __launch_bounds__(kThreads) void k_pages_compact(Params p) {
  const int live = p.head->live, moves = p.head->moves, missing = p.head->missing;
  const int groups = gridDim.x * gridDim.y, me = blockIdx.y * gridDim.x + blockIdx.x;
  if (me == 0 && threadIdx.x == 0) p.head->refused = missing;
  if (missing != 0) {
    if (me == 0 && threadIdx.x == 0) record(p.head, MKMOE_PAGES_ERR_TABLE, missing);
    return;
  }
  // (rank + moves: the place among the pages that move)
  for (int page = live + me * kThreads + threadIdx.x; page < p.pages; page += groups * kThreads)
    if (p.refs[page] != 0) p.src[p.rank[page] + moves] = page;
  for (int b = blockIdx.x; b < p.seqs; b += gridDim.x) {
    const int n = pages_for(p, clamped(p, p.lens[b]));
    for (int i = blockIdx.y * kThreads + threadIdx.x; i < n; i += gridDim.y * kThreads) {
      int32_t* at = p.table + b * p.table_stride + i;
      const int page = *at;
      if (page < live && page >= 0) continue;
      const int r = (uint32_t)page < (uint32_t)p.pages && p.refs[page] != 0 ? p.rank[page] + moves : -1;
      if ((uint32_t)r < (uint32_t)moves)
        *at = p.dst[r];
      else
        record(p.head, MKMOE_PAGES_ERR_PAGE, b);
    }
  }
}
// the moved pages' counts and bytes
__global__ __launch_bounds__(kThreads) void k_pages_move(Params p) {
  const int live = p.head->live, moves = p.head->moves;
  const int groups = gridDim.x * gridDim.y, me = blockIdx.y * gridDim.x + blockIdx.x;
  if (me == 0 && threadIdx.x == 0) p.head->missing = 0;
  if (p.head->refused != 0) return;
  for (int i = me * kThreads + threadIdx.x; i < moves; i += groups * kThreads) {
    p.refs[p.dst[i]] = p.refs[p.src[i]];
    p.refs[p.src[i]] = 0;
  }
  for (int j = me * kThreads + threadIdx.x; j < p.blocks; j += groups * kThreads) {
    const int from = j * kBlock, end = min(from + kBlock, p.pages);
    p.free_in[j] = end - max(from, min(live, end));
  }
  copy_pages(p, p.src, p.dst, moves, false);
}

// ---------------------------------------------------------------- host
struct Layout {
  size_t free_in, src, dst, rank, old_len, new_len, new_page, kids, held, bytes;
};
inline Layout layout(int64_t pages, int64_t seqs, int64_t max_pages) {
  Layout l;
  size_t at = MKMOE_PAGES_REFS_AT + pages * 4;
  auto take = [&](size_t words) {
    at = (at + 255) & ~(size_t)255;
    const size_t from = at;
    at += words * 4;
    return from;
  };
  l.free_in = take((pages + kBlock - 1) / kBlock);
  l.src = take(pages);
  l.dst = take(pages);
  l.rank = take(pages);
  l.old_len = take(seqs);
  l.new_len = take(seqs);
  l.new_page = take(seqs);
  l.kids = take(seqs);
  l.held = take(seqs * max_pages);
  l.bytes = (at + 255) & ~(size_t)255;
  return l;
}
inline bool pool_ok(int64_t pages, int64_t seqs, int64_t max_pages) {
  return pages >= 1 && pages <= kMaxPages && seqs >= 1 && seqs <= kMaxSeqs && max_pages >= 1 && max_pages <= kMaxPages;
}
inline bool aligned(const void* q, size_t a) { return ((uintptr_t)q % a) == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? MKMOE_OK : MKMOE_ERR_LAUNCH; }

inline int params(const mkmoe_pages_pool* pool, void* ws, size_t ws_bytes, Params& p) {
  if (!pool || !ws) return MKMOE_ERR_NULL;
  if (!aligned(ws, 256)) return MKMOE_ERR_ALIGN;
  if (!pool_ok(pool->pages, pool->max_seqs, pool->max_pages)) return MKMOE_ERR_ARG;
  if (pool->page_size < 1 || pool->page_size > 1024 || (pool->page_size & (pool->page_size - 1)) != 0) return MKMOE_ERR_ARG;
  if ((int64_t)pool->pages * pool->page_size > 0x7fffffff || (int64_t)pool->max_pages * pool->page_size > 0x7fffffff)
    return MKMOE_ERR_ARG;
  if (pool->ncaches < 0 || (pool->ncaches > 0 && !pool->caches)) return MKMOE_ERR_ARG;
  const Layout l = layout(pool->pages, pool->max_seqs, pool->max_pages);
  if (ws_bytes < l.bytes) return MKMOE_ERR_WORKSPACE;
  uint8_t* at = (uint8_t*)ws;
  auto words = [&](size_t off) { return (int32_t*)(at + off); };
  p = Params{};
  p.head = (Head*)at;
  p.refs = words(MKMOE_PAGES_REFS_AT);
  p.free_in = words(l.free_in);
  p.src = words(l.src);
  p.dst = words(l.dst);
  p.rank = words(l.rank);
  p.old_len = words(l.old_len);
  p.new_len = words(l.new_len);
  p.new_page = words(l.new_page);
  p.kids = words(l.kids);
  p.held = words(l.held);
  p.caches = pool->caches;
  p.pages = pool->pages;
  p.blocks = (pool->pages + kBlock - 1) / kBlock;
  p.page_size = pool->page_size;
  p.shift = __builtin_ctz((unsigned)pool->page_size);
  p.ncaches = pool->ncaches;
  return MKMOE_OK;
}
inline int table_params(const mkmoe_pages_pool* pool, const mkmoe_pages_table* t, Params& p) {
  if (!t || !t->table || !t->lens) return MKMOE_ERR_NULL;
  if (t->seqs < 1 || t->seqs > pool->max_seqs) return MKMOE_ERR_ROWS;
  if (t->max_pages < 1 || t->max_pages > pool->max_pages || t->stride < t->max_pages) return MKMOE_ERR_ARG;
  if (!aligned(t->table, 4) || !aligned(t->lens, 4)) return MKMOE_ERR_ALIGN;
  p.table = t->table;
  p.lens = t->lens;
  p.table_stride = t->stride;
  p.seqs = t->seqs;
  p.max_pages = t->max_pages;
  return MKMOE_OK;
}
inline unsigned rows_y(const Params& p) {  // workgroups a row of the table
  const int y = (p.max_pages + 4 * kThreads - 1) / (4 * kThreads);
  return (unsigned)(y < 16 ? y : 16);
}
// a grid for a table's rows, with enough workgroups for the caches' pages
inline dim3 rows_grid(const Params& p) {
  unsigned y = rows_y(p);
  if (p.ncaches > 0 && y * p.seqs < 2048) y = (2047 + p.seqs) / p.seqs;
  return dim3((unsigned)p.seqs, y);
}
template <int OP>
int take(const Params& p, hipStream_t st) {
  const int64_t by_tokens = OP == kGrow ? p.tokens / (3 * kThreads) : 0, by_rows = OP == kFork ? p.seqs / 8 : 0;
  int64_t n = p.blocks / 16;
  n = n < by_tokens ? by_tokens : n;
  n = n < by_rows ? by_rows : n;
  hipLaunchKernelGGL(k_pages_take<OP>, dim3((unsigned)(n < 1 ? 1 : n > 128 ? 128 : n)), dim3(kThreads), 0, st, p);
  return launched();
}

}  // namespace mkmoe_pages

extern "C" {

int mkmoe_pages_workspace_bytes(int32_t pages, int32_t max_seqs, int32_t max_pages, size_t* bytes) {
  using namespace mkmoe_pages;
  if (!bytes) return MKMOE_ERR_NULL;
  if (!pool_ok(pages, max_seqs, max_pages)) return MKMOE_ERR_ARG;
  *bytes = layout(pages, max_seqs, max_pages).bytes;
  return MKMOE_OK;
}

int mkmoe_pages_adopt(const mkmoe_pages_pool* pool, const mkmoe_pages_table* table, void* ws, size_t ws_bytes, void* stream) {
  using namespace mkmoe_pages;
  Params p;
  if (int rc = params(pool, ws, ws_bytes, p)) return rc;
  if (table)
    if (int rc = table_params(pool, table, p)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const unsigned n = (unsigned)(p.blocks < 512 ? p.blocks : 512);
  hipLaunchKernelGGL(k_pages_clear, dim3(n), dim3(kThreads), 0, st, p);
  if (int rc = launched()) return rc;
  if (table) {
    hipLaunchKernelGGL(k_pages_hold, dim3((unsigned)p.seqs, rows_y(p)), dim3(kThreads), 0, st, p);
    if (int rc = launched()) return rc;
  }
  hipLaunchKernelGGL(k_pages_count, dim3(n), dim3(kThreads), 0, st, p);
  return launched();
}

int mkmoe_pages_grow(const mkmoe_pages_pool* pool, const mkmoe_pages_table* table, const int32_t* add, int32_t tokens,
                     int32_t* slots, int32_t* positions, int32_t* starts, void* ws, size_t ws_bytes, void* stream) {
  using namespace mkmoe_pages;
  Params p;
  if (int rc = params(pool, ws, ws_bytes, p)) return rc;
  if (int rc = table_params(pool, table, p)) return rc;
  if (!add || !starts || (tokens > 0 && (!slots || !positions))) return MKMOE_ERR_NULL;
  if (tokens < 0) return MKMOE_ERR_ROWS;
  if (!aligned(add, 4) || !aligned(slots, 4) || !aligned(positions, 4) || !aligned(starts, 4)) return MKMOE_ERR_ALIGN;
  p.arg = add;
  p.tokens = tokens;
  p.slots = slots;
  p.positions = positions;
  p.starts = starts;
  return take<kGrow>(p, (hipStream_t)stream);
}

int mkmoe_pages_trim(const mkmoe_pages_pool* pool, const mkmoe_pages_table* table, const int32_t* keep, void* ws,
                     size_t ws_bytes, void* stream) {
  using namespace mkmoe_pages;
  Params p;
  if (int rc = params(pool, ws, ws_bytes, p)) return rc;
  if (int rc = table_params(pool, table, p)) return rc;
  if (!keep) return MKMOE_ERR_NULL;
  if (!aligned(keep, 4)) return MKMOE_ERR_ALIGN;
  p.arg = keep;
  if (int rc = take<kTrim>(p, (hipStream_t)stream)) return rc;
  hipLaunchKernelGGL(k_pages_trim, rows_grid(p), dim3(kThreads), 0, (hipStream_t)stream, p);
  return launched();
}

int mkmoe_pages_fork(const mkmoe_pages_pool* pool, const mkmoe_pages_table* table, const int32_t* parents, void* ws,
                     size_t ws_bytes, void* stream) {
  using namespace mkmoe_pages;
  Params p;
  if (int rc = params(pool, ws, ws_bytes, p)) return rc;
  if (int rc = table_params(pool, table, p)) return rc;
  if (!parents) return MKMOE_ERR_NULL;
  if (!aligned(parents, 4)) return MKMOE_ERR_ALIGN;
  p.arg = parents;
  if (int rc = take<kFork>(p, (hipStream_t)stream)) return rc;
  hipLaunchKernelGGL(k_pages_fork, rows_grid(p), dim3(kThreads), 0, (hipStream_t)stream, p);
  return launched();
}

int mkmoe_pages_compact(const mkmoe_pages_pool* pool, const mkmoe_pages_table* table, void* ws, size_t ws_bytes,
                        void* stream) {
  using namespace mkmoe_pages;
  Params p;
  if (int rc = params(pool, ws, ws_bytes, p)) return rc;
  if (int rc = table_params(pool, table, p)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const int plan = p.blocks < p.seqs ? p.seqs : p.blocks;
  hipLaunchKernelGGL(k_pages_plan, dim3((unsigned)(plan < 256 ? plan : 256)), dim3(kThreads), 0, st, p);
  if (int rc = launched()) return rc;
  hipLaunchKernelGGL(k_pages_compact, dim3((unsigned)p.seqs, rows_y(p)), dim3(kThreads), 0, st, p);
  if (int rc = launched()) return rc;
  hipLaunchKernelGGL(k_pages_move, p.ncaches > 0 ? dim3(2048) : dim3(16), dim3(kThreads), 0, st, p);
  return launched();
}

int mkmoe_pages_copy(const mkmoe_pages_pool* pool, const int32_t* src, const int32_t* dst, int32_t count, void* ws,
                     size_t ws_bytes, void* stream) {
  using namespace mkmoe_pages;
  Params p;
  if (int rc = params(pool, ws, ws_bytes, p)) return rc;
  if (count < 0 || count > pool->pages) return MKMOE_ERR_ROWS;
  if (count > 0 && (!src || !dst)) return MKMOE_ERR_NULL;
  if (!aligned(src, 4) || !aligned(dst, 4)) return MKMOE_ERR_ALIGN;
  if (count == 0 || p.ncaches == 0) return MKMOE_OK;
  hipLaunchKernelGGL(k_pages_copy, dim3(2048), dim3(kThreads), 0, (hipStream_t)stream, p, src, dst, count);
  return launched();
}

int mkmoe_pages_read_errors(const void* ws, int32_t* words, int32_t n, void* stream) {
  if (!ws || !words) return MKMOE_ERR_NULL;
  if (n < 1 || n > MKMOE_PAGES_ERRW_WORDS) return MKMOE_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (hipMemcpyAsync(words, ws, (size_t)n * 4, hipMemcpyDeviceToHost, st) != hipSuccess) return MKMOE_ERR_HIP;
  return hipStreamSynchronize(st) == hipSuccess ? MKMOE_OK : MKMOE_ERR_HIP;
}

}  // extern "C"
