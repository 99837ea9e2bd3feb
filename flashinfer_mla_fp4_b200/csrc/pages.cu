// The care of a cache's pages: copying, allocation, forking and freeing of block-table rows, compaction of the pool.
//
// A pool has a reference count per page (0: free) and one or more layers, whose caches hold a page of the same number each: rows, scales
// and, where there is one, the summary.  Which pages move is decided by one CTA from the counts and lengths in device memory (the host is
// not asked, so every call can be captured); the next kernel moves them in every layer.  New pages are the free ones of the lowest
// numbers, in the order in which they are asked for: the same calls give the same tables.
#include <climits>

#include "sparse.cuh"

namespace mla {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;

// pages that `len` tokens take
__device__ __forceinline__ int pages_of(int len, int page_size) { return len > 0 ? (len - 1) / page_size + 1 : 0; }
__device__ __forceinline__ void report(int32_t* status, int code, int which) {
  if (status) {
    status[1] = which;
    status[0] = code;
  }
}

// Sum of the values of the CTA's threads before this one; *total: of all.  warp_s: a word per warp.
template <typename T>
__device__ __forceinline__ T scan_before(T v, T* warp_s, T* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  T sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T up = __shfl_up_sync(0xffffffffu, sum, o);
    sum += lane >= o ? up : 0;
  }
  __syncthreads();
  if (lane == 31) warp_s[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    T w = lane < warps ? warp_s[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T up = __shfl_up_sync(0xffffffffu, w, o);
      w += lane >= o ? up : 0;
    }
    warp_s[lane] = w;
  }
  __syncthreads();
  *total = warp_s[warps - 1];
  return sum - v + (warp ? warp_s[warp - 1] : 0);
}

constexpr int kPerThread = 8;  // counts that a thread of a planning CTA looks at in a round: two loads of 16 bytes
constexpr int kPerRound = kPlanThreads * kPerThread;

// Reference counts first + 8 tid to + 7 (1, in use, behind the last one).
struct Counts {
  int32_t n[kPerThread];
  __device__ __forceinline__ Counts(const int32_t* refcounts, int64_t first, int64_t num_pages) {
    const int64_t at = first + threadIdx.x * kPerThread;
    if (at + kPerThread <= num_pages) {
#pragma unroll
      for (int i = 0; i < kPerThread; i += 4) *reinterpret_cast<int4*>(n + i) = __ldcg(reinterpret_cast<const int4*>(refcounts + at + i));
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) n[i] = at + i < num_pages ? __ldcg(refcounts + at + i) : 1;
    }
  }
};

// Calls take(number, page) for the free pages of the lowest numbers, the first `wanted` of them; returns how many there were.  first: the counts of the
// first round, asked for while something else was waited for.
template <typename Take>
__device__ __forceinline__ int for_free_pages(const int32_t* refcounts, int64_t num_pages, int wanted, int* warp_s, const Counts& first, Take take) {
  int found = 0;
  for (int64_t base = 0; base < num_pages && found < wanted; base += kPerRound) {
    const Counts c = base == 0 ? first : Counts(refcounts, base, num_pages);
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) n += c.n[i] <= 0;
    int total, number = found + scan_before(n, warp_s, &total);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (c.n[i] <= 0) {
        if (number < wanted) take(number, int(base) + int(threadIdx.x) * kPerThread + i);
        ++number;
      }
    found += total;
  }
  return found < wanted ? found : wanted;
}

// ------------------------------------------------------------------------------------------ copying
// Five loads of a thread are on their way before the first store (a page of 64 tokens is five rounds of the CTA).
__device__ __forceinline__ void copy16(void* dst, const void* src, int n16) {
  constexpr int kAhead = 5;
  const uint4* from = static_cast<const uint4*>(src) + threadIdx.x;
  uint4* to = static_cast<uint4*>(dst) + threadIdx.x;
  for (int i = threadIdx.x; i < n16; i += kAhead * kMoveThreads, from += kAhead * kMoveThreads, to += kAhead * kMoveThreads) {
    uint4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k * kMoveThreads < n16) v[k] = __ldcg(from + k * kMoveThreads);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k * kMoveThreads < n16) to[k * kMoveThreads] = v[k];
  }
}
// page `from` of a layer to page `to` of it, by the whole CTA
__device__ __forceinline__ void copy_page(const PageLayer& l, int page_size, int64_t from, int64_t to) {
  const int64_t row = int64_t(page_size) * kRowBytes;
  copy16(l.kv_cache + to * row, l.kv_cache + from * row, int(row / 16));
  copy16(l.kv_cache_sf + to * page_size, l.kv_cache_sf + from * page_size, page_size / 4);
  if (l.summary) {
    copy16(l.summary + to * kQDim, l.summary + from * kQDim, kQDim / 16);
    if (threadIdx.x == 0) l.summary_sf[to] = l.summary_sf[from];
  }
}

__global__ void __launch_bounds__(kMoveThreads) copy_pages_kernel(const __grid_constant__ PageLayers ls, const int32_t* src, const int32_t* dst,
                                                                  int64_t count, int64_t num_pages, int page_size) {
  dependent_launch();
  for (int64_t u = blockIdx.x; u < count * ls.count; u += gridDim.x) {
    const int64_t i = u / ls.count;
    const int64_t from = src[i], to = dst[i];
    if (from >= 0 && from < num_pages && to >= 0 && to < num_pages && from != to) copy_page(ls.layer[u - i * ls.count], page_size, from, to);
  }
}

// ------------------------------------------------------------------------------------------ allocation
__global__ void __launch_bounds__(kPlanThreads, 1) allocate_kernel(PoolParams p, const int32_t* new_lens) {
  __shared__ int warp_s[32];
  __shared__ long long sum_s[32];
  dependent_launch();
  const Counts counts(p.refcounts, 0, p.num_pages);
  int32_t *offset = p.ws, *list = p.ws + p.rows;
  const auto demand = [&](int r) {  // new pages of a row that has room for them in its table, else none
    const int have = pages_of(p.seq_lens[r], p.page_size), want = pages_of(new_lens[r], p.page_size);
    return want <= p.width && want > have ? want - have : 0;
  };
  long long total = 0;  // (rows may ask for more than 32 bits hold)
  for (int base = 0; base < p.rows; base += kPlanThreads) {
    const int r = base + threadIdx.x;
    long long need = 0, sum;
    if (r < p.rows) {
      if (pages_of(new_lens[r], p.page_size) > p.width) report(p.status, kPoolBadRow, r);
      need = demand(r);
    }
    const long long at = total + scan_before(need, sum_s, &sum);
    if (r < p.rows) offset[r] = int(min(at, (long long)(p.num_pages)));
    total += sum;
  }
  const int found = for_free_pages(p.refcounts, p.num_pages, int(min(total, (long long)(p.num_pages))), warp_s, counts, [&](int number, int page) { list[number] = page; });
  // Not enough for all: a row that does not fit (offset -1) leaves what there is to those behind it.  One warp goes over the rows in order, 32 at a time: those
  // up to the first that does not fit are served, then the same again with those behind it that still may.
  if (total > found && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int next = 0;
    for (int base = 0; base < p.rows; base += 32) {
      const int r = base + lane, need = r < p.rows ? demand(r) : 0;
      int at = -1;
      for (uint32_t open = __ballot_sync(0xffffffffu, need > 0); open;) {
        const int left = found - next;
        open = __ballot_sync(0xffffffffu, (open >> lane & 1) && need <= left);
        const long long mine = open >> lane & 1 ? need : 0;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long up = __shfl_up_sync(0xffffffffu, upto, o);
          upto += lane >= o ? up : 0;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, mine > 0 && upto > left);
        const int first = over ? __ffs(over) - 1 : 32;
        if (mine > 0 && lane < first) at = next + int(upto - mine);
        next += int(__shfl_sync(0xffffffffu, over ? upto - mine : upto, over ? first : 31));
        open &= over ? 0xfffffffeu << first : 0u;
      }
      if (r < p.rows) offset[r] = at;
    }
  }
  __syncthreads();
  // A thread writes up to four pages of its row, a warp longer rows in turn (a warp per row: 1024 rows with two new pages each 20.4 us,
  // 64 rows 4.3; so 5.9 and 4.0, and 22.6 and 6.5 from a pool that is short by half).
  constexpr int kFewPages = 4;
  const int lane = threadIdx.x & 31;
  const auto give = [&](int r, int have, int at, int k) {
    const int page = list[at + k];
    p.block_tables[int64_t(r) * p.block_table_stride + have + k] = page;
    p.refcounts[page] = 1;
  };
  for (int base = 0; base < p.rows; base += kPlanThreads) {
    const int r = base + threadIdx.x;
    int have = 0, need = 0, at = 0;
    if (r < p.rows) {
      have = pages_of(p.seq_lens[r], p.page_size);
      need = demand(r);
      at = offset[r];
      if (need > 0 && at < 0) {
        report(p.status, kPoolOutOfPages, r);
        need = 0;
      }
    }
    if (need <= kFewPages)
      for (int k = 0; k < need; ++k) give(r, have, at, k);
    for (uint32_t more = __ballot_sync(0xffffffffu, need > kFewPages); more; more &= more - 1) {
      const int of = __ffs(more) - 1, row = r - lane + of, held = __shfl_sync(0xffffffffu, have, of), start = __shfl_sync(0xffffffffu, at, of),
                pages = __shfl_sync(0xffffffffu, need, of);
      for (int k = lane; k < pages; k += 32) give(row, held, start, k);
    }
  }
}

// ------------------------------------------------------------------------------------------ forking
// Workspace: claim [rows], then for each fork its length (-1: it is not made), the page for its tail (-1: none) and, by number of
// the tail, whose it is.
//
// Up to kFewForks forks have a thread each, and what the threads tell one another goes by way of shared memory, but each looks at all the children named
// before its own.  Us in graphs of forking and freeing, by way of L2 -> so: 1 fork 8.1 -> 7.1, 16 8.8 -> 8.1, 128 9.4 -> 9.1, 256 9.1 -> 10.0.
constexpr int kFewForks = 128;
__global__ void __launch_bounds__(kPlanThreads, 1) fork_plan_kernel(PoolParams p, const int32_t* parents, const int32_t* children, int count) {
  __shared__ int warp_s[32], child_s[kFewForks], page_s[kFewForks];
  dependent_launch();
  const Counts counts(p.refcounts, 0, p.num_pages);
  int32_t *claim = p.ws, *len_of = claim + p.rows, *tail_of = len_of + count, *owner = tail_of + count;
  const auto in_table = [&](int r) { return r >= 0 && r < p.rows; };
  if (count <= kFewForks) {
    const int i = threadIdx.x, child = i < count ? children[i] : -1, parent = i < count ? parents[i] : -1;
    const bool named = in_table(child) && in_table(parent);
    const int held = named ? p.seq_lens[child] : 0, theirs = named ? p.seq_lens[parent] : 0;
    if (i < kFewForks) child_s[i] = named ? child : -1;
    __syncthreads();
    bool again = false;  // the list has named the child before
    if (named)
#pragma unroll 4
      for (int k = 0; k < i; ++k) again |= child_s[k] == child;
    int len = -1, tail = -1;
    if (child >= 0 && parent >= 0) {  // (a negative row is padding)
      if (named && !again && held <= 0 && pages_of(theirs, p.page_size) <= p.width) len = max(theirs, 0);
      else report(p.status, kPoolBadRow, i);
    }
    const int partial = len > 0 && len % p.page_size != 0;
    int tails;
    const int number = scan_before(partial, warp_s, &tails);
    const int found = for_free_pages(p.refcounts, p.num_pages, tails, warp_s, counts, [&](int n, int page) {
      page_s[n] = page;
      p.refcounts[page] = 1;
    });
    __syncthreads();
    if (i >= count) return;
    if (partial && number < found) tail = page_s[number];
    if (partial && number >= found) {  // no page left for the tail
      len = -1;
      report(p.status, kPoolOutOfPages, i);
    }
    len_of[i] = len;
    tail_of[i] = tail;
    return;
  }
  for (int r = threadIdx.x; r < p.rows; r += kPlanThreads) claim[r] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kPlanThreads)
    if (in_table(children[i]) && in_table(parents[i])) atomicMin(&claim[children[i]], i);
  __syncthreads();
  int tails = 0;
  for (int base = 0; base < count; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int len = -1;
    if (i < count && children[i] >= 0 && parents[i] >= 0) {  // (a negative row is padding)
      if (in_table(children[i]) && in_table(parents[i]) && __ldcg(&claim[children[i]]) == i && p.seq_lens[children[i]] <= 0 &&
          pages_of(p.seq_lens[parents[i]], p.page_size) <= p.width)
        len = max(p.seq_lens[parents[i]], 0);
      else
        report(p.status, kPoolBadRow, i);
    }
    const int partial = len > 0 && len % p.page_size != 0;
    int sum;
    const int number = tails + scan_before(partial, warp_s, &sum);
    if (i < count) {
      len_of[i] = len;
      tail_of[i] = -1;
      if (partial) owner[number] = i;
    }
    tails += sum;
  }
  __syncthreads();
  const int found = for_free_pages(p.refcounts, p.num_pages, tails, warp_s, counts, [&](int number, int page) {
    tail_of[owner[number]] = page;
    p.refcounts[page] = 1;
  });
  __syncthreads();
  for (int n = found + threadIdx.x; n < tails; n += kPlanThreads) {  // no page left for these tails
    len_of[owner[n]] = -1;
    report(p.status, kPoolOutOfPages, owner[n]);
  }
}

// The first `count` CTAs write a row each, the others copy the tails, layer by layer.
__global__ void __launch_bounds__(kMoveThreads) fork_kernel(PoolParams p, const __grid_constant__ PageLayers ls, const int32_t* parents,
                                                            const int32_t* children, int count, bool with_rows) {
  dependent_launch();
  const int32_t *len_of = p.ws + p.rows, *tail_of = len_of + count;
  if (with_rows && int(blockIdx.x) < count) {
    const int i = blockIdx.x, len = len_of[i];
    if (len < 0) return;
    const int32_t* from = p.block_tables + int64_t(parents[i]) * p.block_table_stride;
    int32_t* to = p.block_tables + int64_t(children[i]) * p.block_table_stride;
    const int used = pages_of(len, p.page_size), full = len / p.page_size;
    for (int k = threadIdx.x; k < used; k += kMoveThreads) {
      int page = from[k];
      if (k >= full) page = tail_of[i];
      else if (page >= 0 && page < p.num_pages) atomicAdd(&p.refcounts[page], 1);
      to[k] = page;
    }
    if (threadIdx.x == 0) p.seq_lens[children[i]] = len;
    return;
  }
  const int u = int(blockIdx.x) - (with_rows ? count : 0), i = u / ls.count;
  const int to = tail_of[i];
  if (len_of[i] < 0 || to < 0) return;
  const int from = p.block_tables[int64_t(parents[i]) * p.block_table_stride + len_of[i] / p.page_size];
  if (from >= 0 && from < p.num_pages) copy_page(ls.layer[u - i * ls.count], p.page_size, from, to);
}

// ------------------------------------------------------------------------------------------ freeing
__global__ void __launch_bounds__(kMoveThreads) free_kernel(PoolParams p, const int32_t* rows) {
  __shared__ int len_s;
  dependent_launch();
  const int row = rows[blockIdx.x];
  if (row < 0) return;  // padding
  if (row >= p.rows) {
    if (threadIdx.x == 0) report(p.status, kPoolBadRow, blockIdx.x);
    return;
  }
  if (threadIdx.x == 0) len_s = atomicExch(&p.seq_lens[row], 0);  // a row that is named twice is freed once
  __syncthreads();
  const int used = min(pages_of(len_s, p.page_size), p.width);
  for (int k = threadIdx.x; k < used; k += kMoveThreads) {
    const int page = p.block_tables[int64_t(row) * p.block_table_stride + k];
    if (page < 0 || page >= p.num_pages || atomicSub(&p.refcounts[page], 1) > 0) continue;
    atomicAdd(&p.refcounts[page], 1);  // it was free already
    report(p.status, kPoolBadRow, blockIdx.x);
  }
}

// ------------------------------------------------------------------------------------------ compaction
// With n pages in use, the i-th of them whose number is n or more moves into the i-th free page below n.  Workspace: how many move, then
// the holes, then the pages that move.
__global__ void __launch_bounds__(kPlanThreads, 1) compact_plan_kernel(PoolParams p, int32_t* remap) {
  __shared__ int warp_s[32], below_s, hole_s[kPerRound / 2];
  dependent_launch();
  int32_t *hole = p.ws + 4, *high = hole + p.num_pages;
  // One round: the counts stay in registers, the holes in shared memory (170 of 300 pages, two layers 9.0 -> 7.7 us, 2000 of 6000, eight layers 81.7 -> 78.7).
  if (p.num_pages <= kPerRound) {
    const Counts c(p.refcounts, 0, p.num_pages);
    const int at = threadIdx.x * kPerThread;
    uint32_t used = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) used |= uint32_t(c.n[i] > 0 && at + i < p.num_pages) << i;
    int live;
    const int before = scan_before(__popc(used), warp_s, &live);
    // pages in use among those that stay: where the numbers end that the compacted pages have
    if (at <= live && live < at + kPerThread) below_s = before + __popc(used & ((1u << (live - at)) - 1));
    if (threadIdx.x == 0 && live == kPerRound) below_s = live;
    // the i-th free page below that is at place i of the holes, as many pages of higher numbers are in use
    int u = before;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const bool in_use = used >> i & 1;
      if (!in_use && at + i < live) hole_s[at + i - u] = at + i;
      u += in_use;
    }
    __syncthreads();
    u = before - below_s;
    int to[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const bool in_use = used >> i & 1;
      to[i] = in_use ? at + i : -1;
      if (in_use && at + i >= live) {
        to[i] = hole_s[u];
        hole[u] = to[i];
        high[u] = at + i;
        p.refcounts[to[i]] = c.n[i];
        p.refcounts[at + i] = 0;
      }
      u += in_use;
    }
    if (at + kPerThread <= p.num_pages && reinterpret_cast<uintptr_t>(remap) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kPerThread; i += 4) *reinterpret_cast<int4*>(remap + at + i) = make_int4(to[i], to[i + 1], to[i + 2], to[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; ++i)
        if (at + i < p.num_pages) remap[at + i] = to[i];
    }
    if (threadIdx.x == 0) p.ws[0] = live - below_s;
    return;
  }
  int mine = 0, live;
  for (int64_t base = 0; base < p.num_pages; base += kPerRound) {
    const Counts c(p.refcounts, base, p.num_pages);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) mine += c.n[i] > 0 && base + threadIdx.x * kPerThread + i < p.num_pages;
  }
  scan_before(mine, warp_s, &live);
  int holes = 0, highs = 0;
  for (int64_t base = 0; base < p.num_pages; base += kPerRound) {
    const Counts c(p.refcounts, base, p.num_pages);
    const int64_t at = base + threadIdx.x * kPerThread;
    int both = 0;  // holes, and pages that move in the upper half
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const bool used = c.n[i] > 0, low = at + i < live;
      both += (!used && low ? 1 : 0) + (used && !low && at + i < p.num_pages ? 1 << 16 : 0);
    }
    int sum;
    const int before = scan_before(both, warp_s, &sum);
    int h = holes + (before & 0xffff), m = highs + (before >> 16);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (at + i >= p.num_pages) break;
      const bool used = c.n[i] > 0, low = at + i < live;
      if (!used && low) hole[h++] = int(at) + i;
      if (used && !low) high[m++] = int(at) + i;
      remap[at + i] = used ? int(at) + i : -1;
    }
    holes += sum & 0xffff;
    highs += sum >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < highs; i += kPlanThreads) {
    const int from = high[i], to = hole[i];
    remap[from] = to;
    p.refcounts[to] = p.refcounts[from];
    p.refcounts[from] = 0;
  }
  if (threadIdx.x == 0) p.ws[0] = highs;
}

// The first `rows` CTAs (with_rows) rewrite a block-table row each, the others copy.
__global__ void __launch_bounds__(kMoveThreads) compact_kernel(PoolParams p, const __grid_constant__ PageLayers ls, const int32_t* remap, bool with_rows) {
  dependent_launch();
  const int first = with_rows ? p.rows : 0;
  if (int(blockIdx.x) < first) {
    int32_t* row = p.block_tables + int64_t(blockIdx.x) * p.block_table_stride;
    const int used = min(pages_of(p.seq_lens[blockIdx.x], p.page_size), p.width);
    for (int k = threadIdx.x; k < used; k += kMoveThreads) {
      const int page = row[k];
      if (page >= 0 && page < p.num_pages && remap[page] >= 0) row[k] = remap[page];
    }
    return;
  }
  const int32_t *hole = p.ws + 4, *high = hole + p.num_pages;
  const int64_t moves = int64_t(p.ws[0]) * ls.count;
  for (int64_t u = int(blockIdx.x) - first; u < moves; u += int(gridDim.x) - first) {
    const int64_t i = u / ls.count;
    copy_page(ls.layer[u - i * ls.count], p.page_size, high[i], hole[i]);
  }
}

template <typename... Params, typename... Args>
cudaError_t launch_pool(void (*kernel)(Params...), int64_t grid, int threads, cudaStream_t stream, const Args&... args) {
  return launch_dependent(kernel, dim3(unsigned(grid)), threads, 0, stream, args...);
}

// Layers go kMaxLayers at a time; f(layers, whether these are the first) launches.
template <typename F>
cudaError_t by_layers(const PageLayer* layers, int count, F f) {
  PageLayers ls;
  for (int at = 0; at < count; at += kMaxLayers) {
    ls.count = count - at < kMaxLayers ? count - at : kMaxLayers;
    for (int i = 0; i < ls.count; ++i) ls.layer[i] = layers[at + i];
    cudaError_t e = f(ls, at == 0);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
int64_t move_ctas(int64_t units) { return units < 148 * 64 ? units : 148 * 64; }

}  // namespace

cudaError_t launch_copy_pages(const PageLayer* layers, int num_layers, const int32_t* src, const int32_t* dst, int64_t count, int64_t num_pages,
                              int page_size, cudaStream_t stream) {
  return by_layers(layers, num_layers, [&](const PageLayers& ls, bool) {
    return launch_pool(copy_pages_kernel, move_ctas(count * ls.count), kMoveThreads, stream, ls, src, dst, count, num_pages, page_size);
  });
}
cudaError_t launch_pool_allocate(const PoolParams& p, const int32_t* new_lens, cudaStream_t stream) {
  return launch_pool(allocate_kernel, 1, kPlanThreads, stream, p, new_lens);
}
cudaError_t launch_pool_fork(const PoolParams& p, const PageLayer* layers, int num_layers, const int32_t* parents, const int32_t* children, int count,
                             cudaStream_t stream) {
  cudaError_t e = launch_pool(fork_plan_kernel, 1, kPlanThreads, stream, p, parents, children, count);
  if (e != cudaSuccess) return e;
  return by_layers(layers, num_layers, [&](const PageLayers& ls, bool first) {
    return launch_pool(fork_kernel, int64_t(count) * (ls.count + (first ? 1 : 0)), kMoveThreads, stream, p, ls, parents, children, count, first);
  });
}
cudaError_t launch_pool_free(const PoolParams& p, const int32_t* rows, int count, cudaStream_t stream) {
  return launch_pool(free_kernel, count, kMoveThreads, stream, p, rows);
}
cudaError_t launch_pool_compact(const PoolParams& p, const PageLayer* layers, int num_layers, int32_t* remap, cudaStream_t stream) {
  cudaError_t e = launch_pool(compact_plan_kernel, 1, kPlanThreads, stream, p, remap);
  if (e != cudaSuccess) return e;
  return by_layers(layers, num_layers, [&](const PageLayers& ls, bool first) {
    return launch_pool(compact_kernel, (first ? p.rows : 0) + move_ctas(p.num_pages / 2 * ls.count + 1), kMoveThreads, stream, p, ls, remap, first);
  });
}

}  // namespace mla
