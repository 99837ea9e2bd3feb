// Scores of page summaries against queries (mathematics: sparse.cu) on the tensor cores: tcgen05.mma.kind::i8, 128 pages x heads x 576.
//
// Pages are the M axis: a thread of the epilogue has a page (a TMEM lane) and goes over its heads in registers; with the heads on M the
// largest over heads would be a reduction across threads, and fewer than 128 heads would waste half of the MMA or more.
//
// Bound by the gather of the pages' rows: 580 bytes a page and query position, an SM's share of the measured copy rate is a tile (128 pages,
// 74 KB) in 1.7 us, and its 18 MMAs of 128 x 128 x 32 take 0.9.  64 requests of 2048 pages, 128 heads, up to seven tiles a CTA: 18 us, of which 1.8 are
// up to the CTA's share, 3.4 the query and the first tile, 1.9 the conversion, then 1.4 a tile (8 TB/s, the queries and some rows out of L2); 21 where a
// CTA goes on to a second row, whose query waits for the MMAs of the first.  So a CTA per SM walks a contiguous range of the tiles of all
// rows, in two stages of a whole tile each: at least one tile is in flight whatever the other roles do.
// Rows come by cp.async straight into the swizzled operand, 512 contiguous bytes an instruction, 32 bytes a clk and SM; a TMA gather would
// take 160 instructions a tile.
//
// Several query positions of a request look at the same pages: where their heads fit into 128 columns side by side, and there are tiles enough,
// one load of a tile serves them all (Form::kTogether).  Few rows of one tile each (Form::kWhole): a CTA has a row to itself, keeps its keys in
// shared memory and selects too, by counting for each page those before it: no second launch, and nothing that another CTA has to see.
//
// Roles: warps 0-3 take the scores out of TMEM, warp 4 issues the MMAs, warps 5-20 load, and turn a row's query into integers (the B
// operand) while the row's first tile is on its way.  (With eight warps for that instead of sixteen 32 requests of 2048 pages, 128 heads, with
// their attention took 67.7 us instead of 66.0, 64 such selections 28.1 instead of 27.2; one of 16 heads 7.6 instead of 8.0.)  All waits are
// bounded; one that runs out sets the status and ends the CTA, whose keys are then not all written.
#include "common.cuh"
#include "launch.h"
#include "ptx_sm100.cuh"
#include "sparse.cuh"

namespace mla {

namespace {

constexpr int kEpiWarps = 4, kLoadWarps = 16;
constexpr int kMmaWarp = kEpiWarps, kFirstLoad = kEpiWarps + 1;
constexpr int kThreads = 32 * (kEpiWarps + 1 + kLoadWarps);
constexpr int kPages = 128;                       // pages of a tile: the lanes of TMEM
static_assert(kQDim / 16 == 36, "a row is 32 chunks of 16 bytes and four more");
constexpr int kStageBytes = kPages * kQDim;       // an operand of 128 pages (below)
constexpr int kStages = 2;
constexpr int kMaxRows = 1024;                    // rows of a launch (the launcher makes several)
constexpr uint32_t kTmemCols = 256;               // two accumulators of up to 128 columns
constexpr int kWholeKeys = kPages;                // most candidates of a row that a CTA has to itself

// shared memory, from a 1024-byte boundary on: the stages, the query's codes, then
struct Small {
  int candidates[kMaxRows];  // pages that a row scores
  uint16_t request[kMaxRows];  // of a row, counted from the first row's (a division at every tile's page numbers: 1 us for 15 rows of 3750 pages)
  alignas(16) uint32_t keys[kWholeKeys];  // of a row that the CTA has to itself
  int taken[kWholeKeys / 32];
  float unit[4][128];        // 2^-k of the heads, by row: an epilogue may be three tiles, so three rows, behind the loads
  unsigned long long full_a[kStages], empty_a[kStages], full_d[2], empty_d[2], full_b, drained;
  uint32_t tmem;
  int first_row, first_tile, tiles;  // of this CTA
  volatile int abort;
};

__device__ __forceinline__ uint32_t bar(const unsigned long long& b) { return ptx::smem_u32(&b); }

struct Ctx {
  const SelectParams& p;
  Small& s;
};
// Of a whole warp, and bounded: false when it ran out, here or in another role.  The answer is the same in all lanes: one that gave up alone would leave
// the others in front of what a warp does together.
__device__ __forceinline__ bool wait(const Ctx& c, const unsigned long long& b, uint32_t parity) {
  bool there = false;
  for (uint32_t i = 0; i < c.p.wait_polls && !c.s.abort; ++i) {
    there = ptx::mbar_try_wait(bar(b), parity);
    if (there) break;
  }
  if (__all_sync(0xffffffffu, there)) return true;
  if ((threadIdx.x & 31) == 0 && !c.s.abort) {
    c.s.abort = 1;
    report_timeout(c.p.status, bar(b), parity);
  }
  __syncwarp();
  return false;
}

// The tiles of a CTA in order, the same for every role.
struct Walk {
  const int* candidates;
  const uint16_t* request;
  int row, tile, left;
  __device__ __forceinline__ Walk(const Small& s) : candidates(s.candidates), request(s.request), row(s.first_row), tile(s.first_tile), left(s.tiles) {}
  __device__ __forceinline__ bool row_ends() const { return (tile + 1) * kPages >= candidates[row]; }
  __device__ __forceinline__ int next_row() const {  // (there is one where tiles are left)
    int r = row + 1;
    while (candidates[r] == 0) ++r;
    return r;
  }
  __device__ __forceinline__ void next() {  // (behind the last one there is none, however often)
    if (--left <= 0) return;
    if (!row_ends()) ++tile;
    else row = next_row(), tile = 0;
  }
  // block-table entry of page i of the tile, -1 where there is none
  __device__ __forceinline__ int entry(const SelectParams& p, const int32_t* tables, int i) const {
    i += tile * kPages;
    return left > 0 && i < candidates[row] ? __ldcg(tables + int64_t(request[row]) * p.block_table_stride + i) : -1;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// an arrival on the barrier once all copies that this thread has asked for have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// An operand of `rows` rows: four blocks [rows][128 bytes] with the 128-byte swizzle, then one [rows][64 bytes] with the 64-byte swizzle.  (All in blocks of 64
// bytes, eight lanes that store next to one another met in the same banks, and the stores took as long as the MMAs' reads.)
__device__ __forceinline__ uint32_t wide_at(int rows, int row, int chunk) { return uint32_t((chunk >> 3) * (rows * 128) + row * 128 + (((chunk ^ row) & 7) << 4)); }
__device__ __forceinline__ uint32_t tail_at(int rows, int row, int chunk) { return uint32_t(rows * 512 + row * 64 + (((chunk ^ (row >> 1)) & 3) << 4)); }
// Rows `first` to `first + count - 1` of an operand, by a warp: 32 of a row's 36 chunks at a time, a lane each, then the last four of eight rows at a
// time.  src(r): where row first + r comes from, asked by all lanes at once; null: nowhere.  (With the 32 next chunks in the order of their addresses,
// whatever rows they belong to, the instructions that found their places took 4900 clk a tile, whether or not anything was loaded.)
template <typename Src>
__device__ __forceinline__ void copy_rows(uint32_t operand, int rows, int first, int count, Src src) {
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int r = 0; r < count; ++r) {
    const char* from = src(r);
    if (from) cp_async16(operand + wide_at(rows, first + r, lane), from + 16 * lane);
  }
#pragma unroll 1
  for (int h = 0; h < count; h += 8) {
    const int r = h + (lane >> 2);
    const char* from = src(r);
    if (from && r < count) cp_async16(operand + tail_at(rows, first + r, lane), from + 16 * (32 + (lane & 3)));
  }
}

// columns of the MMAs for the heads of a query position
__host__ __device__ __forceinline__ int columns_of(int heads) { return (heads + 15) / 16 * 16; }

// The heads of a row's query, to be the B operand: first fetched as they are, ...  Columns behind the last head repeat head 0, which leaves the
// largest score as it is.  kTogether: of all query positions of the request, `row` being the first.
template <bool kTogether>
__device__ __forceinline__ void fetch_b(const SelectParams& p, uint32_t b_smem, int row, int columns) {
  const int each = columns / kLoadWarps, first = ((threadIdx.x >> 5) - kFirstLoad) * each, batch = row / p.q_len;
  const uint8_t* q = p.q + batch * p.q_stride_batch + (row - batch * p.q_len) * p.q_stride_qpos;
  // 2^16 / the columns of a position, and up to one more: a product with a column is off by less than 2^-8, and a quotient that is not whole has at least 2^-6
  // to the next one
  const int inverse = kTogether ? int(65536.f * __frcp_rn(float(columns_of(p.heads)))) + 1 : 0;
  copy_rows(b_smem, columns, first, each, [&](int r) {
    const int position = kTogether ? (first + r) * inverse >> 16 : 0, head = first + r - position * columns_of(p.heads);
    return reinterpret_cast<const char*>(q + (kTogether ? position * p.q_stride_qpos : 0) + (head < p.heads ? head : 0) * p.q_stride_head);
  });
}
// ... then turned into integers where they lie: eight lanes a head, four heads at a time.  In FP16: an E4M3 value times 2^k is exact, and adding 1536
// rounds it to a whole number (to even, as round() does) that is the low byte of the sum.
__device__ __forceinline__ void convert_b(char* b_smem, float* unit, int columns) {
  constexpr int kMine = 5;  // chunks of a lane; the last one of lanes 0-3 alone
  const int each = columns / kLoadWarps, first = ((threadIdx.x >> 5) - kFirstLoad) * each, lane = threadIdx.x & 31, part = lane & 7;
#pragma unroll 1
  for (int r = lane >> 3; r < (each + 3) / 4 * 4; r += 4) {
    const int head = first + (r < each ? r : 0);
    auto at = [&](int i) { return reinterpret_cast<uint4*>(b_smem + (i < 4 ? wide_at(columns, head, 8 * i + part) : tail_at(columns, head, part))); };
    uint4 v[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) v[i] = i < 4 || part < 4 ? *at(i) : make_uint4(0, 0, 0, 0);
    // the largest magnitude: bytes without their signs, by 16 bits, the upper ones with what lies below them; NaN is 127
    auto top_of = [](uint32_t top, const uint4& x) {
      const uint32_t a = __vmaxu2(x.x & 0x7fff7fff, x.y & 0x7fff7fff), b = __vmaxu2(x.z & 0x7fff7fff, x.w & 0x7fff7fff);
      const uint32_t c = __vmaxu2(x.x & 0x7f007f, x.y & 0x7f007f), d = __vmaxu2(x.z & 0x7f007f, x.w & 0x7f007f);
      return __vmaxu2(__vmaxu2(top, __vmaxu2(a, b) >> 8 & 0x7f007f), __vmaxu2(c, d));
    };
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) top = top_of(top, v[i]);
    if ((top & 0xffff) == 0x7f || top >> 16 == 0x7f) {  // NaN among them: they count as zero
      top = 0;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t nan = ((x[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // the top bit of a byte that is NaN
          x[j] &= ~(nan | (nan - (nan >> 7)));
        }
        v[i] = make_uint4(x[0], x[1], x[2], x[3]);
        top = top_of(top, v[i]);
      }
    }
    __syncwarp();
    uint32_t most = max(top & 0xffff, top >> 16);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int binade = max(int(most >> 3), 1);  // exponent field
    const uint32_t half = uint32_t(15 + 13 - binade) << 10, times = half | half << 16;  // 2^(13 - binade)
    if (r >= each) continue;
    if (part == 0) unit[head] = __uint_as_float(uint32_t(127 + binade - 13) << 23);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = __byte_perm(hfma2(e4m3x2_to_f16x2(x[j] & 0xffff), times, 0x66006600u), hfma2(e4m3x2_to_f16x2(x[j] >> 16), times, 0x66006600u), 0x6420);
      if (i < 4 || part < 4) *at(i) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

// The selection of a row by the CTA that has its keys in shared memory.  The place of a page is the number of those with a larger key, or with the
// same one and nearer the start: 128 compares per thread, with four keys a load that all threads share.
__device__ __forceinline__ void select_whole(const SelectParams& p, Small& s, int row, const Seen& v, int page) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t* table = p.block_tables + int64_t(row / p.q_len) * p.block_table_stride;
  int32_t* out = p.selected + int64_t(row) * p.budget;
  if (v.used <= p.budget) {  // the budget holds them all
    for (int k = tid; k < p.budget; k += kThreads) out[k] = k < v.used ? __ldcg(table + k) : 0;
    if (tid == 0) p.selected_lens[row] = v.len;
    return;
  }
  const int candidates = v.used - p.sink - p.local, wanted = p.budget - p.sink - p.local;
  for (int k = tid; k < p.sink; k += kThreads) out[k] = __ldcg(table + k);
  for (int k = tid; k < p.local; k += kThreads) out[p.budget - p.local + k] = __ldcg(table + v.used - p.local + k);
  if (tid == 0) p.selected_lens[row] = v.len - (v.used - p.budget) * p.page_size;
  bool take = false;
  uint32_t ballot = 0;
  if (warp < kWholeKeys / 32) {
    const uint32_t key = s.keys[tid];
    int before = 0;
#pragma unroll 4
    for (int k = 0; k < candidates; k += 4) {  // (behind the candidates the keys are 0, and their places behind every candidate's)
      const uint4 four = *reinterpret_cast<const uint4*>(s.keys + k);
      before += (four.x > key || (four.x == key && k < tid)) + (four.y > key || (four.y == key && k + 1 < tid)) +
                (four.z > key || (four.z == key && k + 2 < tid)) + (four.w > key || (four.w == key && k + 3 < tid));
    }
    take = tid < candidates && before < wanted;
    ballot = __ballot_sync(0xffffffffu, take);
    if (lane == 0) s.taken[warp] = __popc(ballot);
  }
  __syncthreads();
  if (!take) return;
  int at = p.sink + __popc(ballot & ((1u << lane) - 1));
  for (int w = 0; w < warp; ++w) at += s.taken[w];
  out[at] = page;
}

// kWhole: CTA i has row i and selects; else the CTAs share the tiles of rows row0 to row0 + rows - 1; kTogether: of requests, all of whose query positions
// are scored with one load of a tile.
enum class Form { kRows, kWhole, kTogether };
template <Form kForm>
__global__ void __launch_bounds__(kThreads, 1) score_kernel(SelectParams p, int row0, int rows, int columns) {
  constexpr bool kWhole = kForm == Form::kWhole, kTogether = kForm == Form::kTogether;
  const int positions = kTogether ? p.q_len : 1;  // of a row here
  extern __shared__ char raw[];
  char* a_smem = raw + ((1024 - (ptx::smem_u32(raw) & 1023)) & 1023);
  char* b_smem = a_smem + kStages * kStageBytes;
  Small& s = *reinterpret_cast<Small*>(b_smem + columns * kQDim);
  const Ctx c{p, s};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(bar(s.full_a[i]), 32 * kLoadWarps);
      ptx::mbar_init(bar(s.empty_a[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(s.full_d[i]), 2);
      ptx::mbar_init(bar(s.empty_d[i]), kEpiWarps);
    }
    ptx::mbar_init(bar(s.full_b), kLoadWarps);
    ptx::mbar_init(bar(s.drained), 1);
    s.abort = 0;
    ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(&s.tmem), kTmemCols);
    ptx::tmem_relinquish();
  }
  if constexpr (kWhole) row0 = blockIdx.x;
  const int request0 = kTogether ? row0 : row0 / p.q_len;
  const int32_t* const tables = p.block_tables + int64_t(request0) * p.block_table_stride + p.sink;  // of the first row's request, its candidates
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Seen mine{0, 0};
  int page_of_mine = 0;  // of the candidate that this thread may take
  if constexpr (kWhole) {
    mine = seen(p, row0);
    const int candidates = mine.used > p.budget ? mine.used - p.sink - p.local : 0;
    if (tid == 0) {
      s.candidates[0] = candidates;
      s.request[0] = 0;
      s.first_row = s.first_tile = 0;
      s.tiles = (candidates + kPages - 1) / kPages;
    }
    if (tid < kWholeKeys) {
      s.keys[tid] = 0;
      if (tid < candidates) page_of_mine = __ldcg(tables + tid);
    }
  } else {
    for (int r = tid; r < rows; r += kThreads) {
      const Seen v = seen(p, kTogether ? (row0 + r) * positions + positions - 1 : row0 + r);  // (the last position sees the most)
      s.request[r] = uint16_t(kTogether ? r : (row0 + r) / p.q_len - request0);
      s.candidates[r] = v.used > p.budget ? v.used - p.sink - p.local : 0;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s.tmem;
  if (!kWhole && warp == 0) {  // this CTA's share of all tiles in the order of the rows
    uint32_t total = 0;  // (at most 2^10 rows of 2^31 tokens: 2^31 tiles of 128 pages of 8)
    for (int base = 0; base < rows; base += 32)
      total += __reduce_add_sync(0xffffffffu, base + lane < rows ? (s.candidates[base + lane] + kPages - 1) / kPages : 0);
    const uint32_t each = total / gridDim.x, rest = total - each * gridDim.x;
    const uint32_t lo = each * blockIdx.x + min(blockIdx.x, rest), hi = lo + each + (blockIdx.x < rest);
    uint32_t at = 0;
    for (int base = 0; base < rows && at <= lo && hi > lo; base += 32) {
      const uint32_t mine = base + lane < rows ? (s.candidates[base + lane] + kPages - 1) / kPages : 0;
      uint32_t sum = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
        sum += lane >= o ? up : 0;
      }
      if (at + sum > lo && at + sum - mine <= lo) {
        s.first_row = base + lane;
        s.first_tile = int(lo - (at + sum - mine));
      }
      at += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) s.tiles = int(hi - lo);
  }
  __syncthreads();

  if (s.tiles > 0) {
    if (warp >= kFirstLoad) {
      // ------------------------------------------------------------------ loads
      constexpr int kMine = kPages / kLoadWarps;  // a warp's pages of a tile
      const int first = (warp - kFirstLoad) * kMine;
      const uint32_t a_addr = ptx::smem_u32(a_smem), b_addr = ptx::smem_u32(b_smem);
      Walk k(s);
      // A row's query is fetched once the MMAs of the row before are over, which is known where the tile behind its first one is loaded; the
      // first row's before anything, and converted while the first tile is on its way (behind the second one: 24.4 us instead of 23.6 for 32 rows of
      // 2048 pages).
      fetch_b<kTogether>(p, b_addr, (row0 + k.row) * positions, columns);
      asm volatile("cp.async.commit_group;" ::: "memory");
      // Page numbers are asked for two tiles ahead, and before the rows: behind those they would take as long.
      Walk ahead(s);
      int pages[2];  // of the next two tiles
#pragma unroll
      for (int i = 0; i < 2; ++i, ahead.next()) pages[i] = lane < kMine ? ahead.entry(p, tables, first + lane) : -1;
      int fresh = -1, seg = 0;  // fresh: the row that the last tile was the first of, or -1
      bool ok = true;
      for (int n = 0; ; ++n) {
        const int st = n & 1;
        const bool more = k.left > 0;
        if (n >= kStages && (more || fresh >= 0)) ok = wait(c, s.empty_a[st], ((n >> 1) - 1) & 1);
        if (!ok) break;
        if (fresh >= 0) {
          fetch_b<kTogether>(p, b_addr, (row0 + fresh) * positions, columns);
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const int next_fresh = more && n > 0 && k.tile == 0 ? k.row : -1;
        if (more) {
          k.next();
          const int page = pages[0] < p.num_pages ? pages[0] : -1;
          pages[0] = pages[1];
          pages[1] = lane < kMine ? ahead.entry(p, tables, first + lane) : -1;
          ahead.next();
          // (rows without a page are left as they are: what comes of them nobody reads.  With some page in their place, the same for all, the tiles
          // that are not full had all SMs wait for one line: 148 rows of 57 candidates 21.2 us instead of 11.5.)
          copy_rows(a_addr + st * kStageBytes, kPages, first, kMine, [&](int r) {
            const int from = __shfl_sync(0xffffffffu, page, r);
            return from >= 0 ? reinterpret_cast<const char*>(p.summary + int64_t(from) * kQDim) : nullptr;
          });
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (more) cp_async_arrive(bar(s.full_a[st]));  // (nobody waits here for a tile: its MMAs start when it is there)
        if (n == 0 || fresh >= 0) {
          asm volatile("cp.async.wait_group 1;" ::: "memory");  // the query came first, the tile may still be on its way
          __syncwarp();  // (a lane converts what others have fetched)
          convert_b(b_smem, s.unit[seg++ & 3], columns);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(bar(s.full_b));
        }
        fresh = next_fresh;
        if (!more) break;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kMmaWarp) {
      // ------------------------------------------------------------------ MMAs
      const uint32_t e = ptx::elect_one();
      const uint64_t a0 = ptx::smem_desc(ptx::smem_u32(a_smem), 16, 1024, 2), b0 = ptx::smem_desc(ptx::smem_u32(b_smem), 16, 1024, 2);
      const uint64_t a4 = ptx::smem_desc(ptx::smem_u32(a_smem) + kPages * 512, 16, 512, 4), b4 = ptx::smem_desc(ptx::smem_u32(b_smem) + columns * 512, 16, 512, 4);
      // D: S32; A, B: signed 8-bit, K-major
      const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(columns >> 3) << 17) | (uint32_t(kPages >> 4) << 24);
      int seg = 0;
      bool fresh = true, ok = true;
      Walk k(s);
      for (int n = 0; k.left > 0 && ok; ++n) {
        const int st = n & 1;
        if (fresh) ok = wait(c, s.full_b, seg & 1);
        if (ok && n >= 2) ok = wait(c, s.empty_d[st], ((n >> 1) - 1) & 1);
        if (ok) ok = wait(c, s.full_a[st], (n >> 1) & 1);
        if (!ok) break;
        ptx::fence_proxy_async_smem();  // the copies into the stage were not the async proxy's; the MMAs' reads are
        ptx::tc_fence_after();
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)
          ptx::umma_i8(e, tmem + st * 128, a0 + ((st * kStageBytes + (i >> 2) * (kPages * 128)) >> 4) + 2 * (i & 3),
                       b0 + (((i >> 2) * (columns * 128)) >> 4) + 2 * (i & 3), idesc, i);
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) ptx::umma_i8(e, tmem + st * 128, a4 + ((st * kStageBytes) >> 4) + 2 * i, b4 + 2 * i, idesc, 1u);
        if (e) ptx::umma_commit(bar(s.empty_a[st]));
        if (e) {
          ptx::umma_commit(bar(s.full_d[st]));
          ptx::mbar_arrive(bar(s.full_d[st]));  // (hands on what the load warps have written for the epilogue: the units)
        }
        fresh = k.row_ends();
        seg += fresh;
        k.next();
      }
      // nothing is in flight when TMEM is given back; the MMAs wait for nobody, so this ends whatever the poll budget is
      if (e) ptx::umma_commit(bar(s.drained));
      for (uint32_t i = 0; i < max(p.wait_polls, 1u << 16) && !ptx::mbar_try_wait(bar(s.drained), 0); ++i) {
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------------ scores
      // A page's number is asked for three tiles ahead and its scale two: with everybody loading they take longer than a tile (asked for with the
      // tile before they made an epilogue of 4800 clk of one of 1400).
      Walk k(s), ahead(s);
      auto scale_of = [&](int page) { return page >= 0 && page < p.num_pages ? __ldcg(p.summary_sf + page) : 0.f; };
      int seg = 0, pages[3];
      float scales[2];
#pragma unroll
      for (int i = 0; i < 3; ++i, ahead.next()) pages[i] = ahead.entry(p, tables, tid);
#pragma unroll
      for (int i = 0; i < 2; ++i) scales[i] = scale_of(pages[i]);
      for (int n = 0; k.left > 0; ++n) {
        const int st = n & 1, row = k.row, i = k.tile * kPages + tid, page = pages[0];
        const bool scored = i < k.candidates[row], last = k.row_ends(), there = page >= 0 && page < p.num_pages;
        const float scale = scales[0];
        k.next();
        pages[0] = pages[1];
        pages[1] = pages[2];
        pages[2] = ahead.entry(p, tables, tid);
        ahead.next();
        scales[0] = scales[1];
        scales[1] = scale_of(pages[1]);
        if (!wait(c, s.full_d[st], (n >> 1) & 1)) break;
        const float* unit = s.unit[seg & 3];
        ptx::tc_fence_after();
        float best = __uint_as_float(0xff800000u);
        int position = 0, end = columns_of(p.heads);
#pragma unroll 1
        for (int col = 0; col < columns; col += 16) {
          uint32_t d[16];
          ptx::tmem_ld16(tmem + (uint32_t(warp) << 21) + st * 128 + col, d);
          float u[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(u + 4 * j) = *reinterpret_cast<const float4*>(unit + col + 4 * j);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) best = fmaxf(best, float(int(d[j])) * u[j]);
          if constexpr (kTogether) {
            if (col + 16 < end) continue;
            // (a position that sees fewer pages than the last one has room for the keys all the same, and nobody reads them)
            if (scored) p.keys[(int64_t(row0 + row) * positions + position) * p.key_stride + i] = there ? key_of(best * scale) : 0u;
            ++position;
            end += columns_of(p.heads);
            best = __uint_as_float(0xff800000u);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(s.empty_d[st]));
        if constexpr (!kTogether) {
          const uint32_t key = there ? key_of(best * scale) : 0u;
          if (kWhole && scored) s.keys[i] = key;
          if (!kWhole && scored) p.keys[int64_t(row0 + row) * p.key_stride + i] = key;
        }
        seg += last;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
  if constexpr (kWhole) select_whole(p, s, row0, mine, page_of_mine);
}

size_t smem_bytes(int columns) { return 1024 + size_t(kStages) * kStageBytes + size_t(columns) * kQDim + sizeof(Small); }
static_assert(1024 + kStages * kStageBytes + 128 * kQDim + sizeof(Small) <= 232448, "shared memory of a CTA");

}  // namespace

// Rows with at most 128 candidates have a CTA each that selects too, us in graphs, a launch each for scores and selection -> this: 16 heads, 57
// candidates, 1 row 7.9 -> 5.9, 148 rows 10.8 -> 6.7, 200 12.9 -> 12.6, 296 14.1 -> 13.1, 444 17.8 -> 19.4; 128 heads, 127 candidates, 11.0 -> 8.7,
// 14.9 -> 9.4, 19.0 -> 17.9, 20.5 -> 18.8, 26.2 -> 28.0: so while there are no more rows than two an SM.  With two tiles, and the compares of 256
// keys with one another, one row was 9.6 -> 10.9.
bool scores_and_selects(const SelectParams& p, int sms) { return p.width - p.sink - p.local <= kWholeKeys && p.batch * p.q_len <= 2 * sms; }

cudaError_t launch_score(const SelectParams& p, int sms, cudaStream_t stream) {
  const int rows = p.batch * p.q_len, columns = columns_of(p.heads);
  static std::atomic<bool> allowed[3][64];
  cudaError_t e = allow_smem(score_kernel<Form::kRows>, smem_bytes(128), allowed[0]);
  if (e == cudaSuccess) e = allow_smem(score_kernel<Form::kWhole>, smem_bytes(128), allowed[1]);
  if (e == cudaSuccess) e = allow_smem(score_kernel<Form::kTogether>, smem_bytes(128), allowed[2]);
  if (e != cudaSuccess) return e;
  if (scores_and_selects(p, sms))
    return launch_dependent(score_kernel<Form::kWhole>, dim3(unsigned(rows)), kThreads, smem_bytes(columns), stream, p, 0, 1, columns);
  const int64_t tiles = (p.width - p.sink - p.local + kPages - 1) / kPages;  // of the longest row that the tables can hold
  // Query positions of a request together, where their heads fit side by side, us in graphs, a row each -> together, 16 heads: three positions of 32
  // requests of 2048 pages (1536 tiles of rows) 24.5 -> 17.0, of 8 (384) 13.6 -> 10.8, of 8 of 512 pages (96) 8.5 -> 9.1; two of 8 of 2048 (256) 10.7 -> 10.2;
  // eight of 16 of 512 (512) 14.3 -> 12.1, of 8 of 512 (256) 11.0 -> 11.2; 64 heads, two positions of 32 of 2048 21.6 -> 20.8, of 8 (256) 11.5 -> 12.4: so
  // where the rows have more than two tiles an SM (few tiles leave SMs idle, and each converts all positions' queries).
  const bool together = p.q_len > 1 && p.q_len * columns <= 128 && tiles * rows > 2 * sms;
  const auto kernel = together ? score_kernel<Form::kTogether> : score_kernel<Form::kRows>;
  const int all = together ? p.batch : rows, wide = together ? p.q_len * columns : columns;
  for (int row0 = 0; row0 < all; row0 += kMaxRows) {
    const int n = all - row0 < kMaxRows ? all - row0 : kMaxRows;
    const int64_t most = tiles * n;
    e = launch_dependent(kernel, dim3(unsigned(most < sms ? most : sms)), kThreads, smem_bytes(wide), stream, p, row0, n, wide);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mla
