// Sparse decode over pages that a cheap score selects: the pages' 8-bit summaries, the scores and the selection.  The attention over the
// selected pages is the decode kernel's, over the block table that is written here.
//
// Summary of a full page of n tokens (scales s_t, latent values e_td, RoPE values r_td): its mean key, with the scales taken as
// integers w_t = round(32767 s_t / S), S = max |s_t|, so that every sum is one of integers: exact, whatever its order, and the same
// codes come out wherever a page is summarised.  Latent m_d = S / (32767 n) sum_t w_t e_td, RoPE m_d = 1/n sum_t r_td,
// scale = max_d |m_d| / 127 rounded to FP32, code_d = round(m_d / scale).  What is left of a page (576 values) is done in 64 bits: a
// code next to the middle of two would go either way in 32.
//
// Score of a page for a query: the query's heads as integers q_h = round(q 2^k_h), k_h bringing the head's largest binade to
// [64, 128) (E4M3 values of the three largest binades are exact), dots <q_h, code> in int32 (below 2^24), and
// scale * max_h 2^-k_h <q_h, code> with one rounding at the end.  So scores too are the same wherever they are made, and pages that
// tie do so by value.  The scores are made in score_sm100.cu.
#include <math_constants.h>

#include "sparse.cuh"

namespace mla {

namespace {

// ------------------------------------------------------------------------------------------ summaries
// A CTA per page of 32 tokens or more.  Latent: a thread has eight dims (a 32-bit word of a row) of every fourth pair of tokens; two tokens at a time, their values as
// signed bytes side by side, go through dp2a with the two 16-bit weights.  RoPE: a thread has four dims of every sixteenth token; sums of eight
// values of at most 448 in steps of 2^-9 are exact in FP32, and whole numbers of 2^-9 from there on.
constexpr int kSumThreads = 256, kSumGroups = kSumThreads / 64, kRopeGroups = kSumThreads / 16;

// bytes of b:a by the selector's nibbles, whose highest bit asks for the byte's sign instead
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t selector) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(selector));
  return r;
}
// 8 codes -> twice their values as signed bytes, codes 0-3 and 4-7
__device__ __forceinline__ void e2m1x8_twice(uint32_t w, uint32_t& lo, uint32_t& hi) {
  constexpr uint32_t kP0 = 0x03020100u, kP1 = 0x0C080604u, kN0 = 0xFDFEFF00u, kN1 = 0xF4F8FAFCu;  // 0 1 2 3 4 6 8 12, and negated
  const uint32_t s0 = w & 0x7777u, s1 = (w >> 16) & 0x7777u, x = w << 4;
  const uint32_t m0 = prmt(x, w, 0xD9C8u), m1 = prmt(x, w, 0xFBEAu);  // the signs as byte masks
  lo = (prmt(kP0, kP1, s0) & ~m0) | (prmt(kN0, kN1, s0) & m0);
  hi = (prmt(kP0, kP1, s1) & ~m1) | (prmt(kN0, kN1, s1) & m1);
}
__device__ __forceinline__ int dp2a_lo(int w2, uint32_t b, int c) { return __dp2a_lo(w2, int(b), c); }
__device__ __forceinline__ int dp2a_hi(int w2, uint32_t b, int c) { return __dp2a_hi(w2, int(b), c); }

template <int kPage>
__global__ void __launch_bounds__(kSumThreads) summarize_kernel(SummarizeParams p) {
  constexpr int kWarps = kSumThreads / 32;
  __shared__ __align__(8) int16_t w_s[kPage];
  __shared__ int part_s[kSumGroups][kLatent], rope_s[kRopeGroups][kRope];
  __shared__ float top_s[kWarps];
  __shared__ int most_s[2][kWarps];
  __shared__ int unsound_s;
  __shared__ float scale_s, by_s[2];
  dependent_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int page = page_of_item<kPage>(p, blockIdx.x);
  if (page < 0) return;
  const uint8_t* rows = p.kv_cache + int64_t(page) * kPage * kRowBytes;
  const float s = tid < kPage ? __ldcg(p.kv_cache_sf + int64_t(page) * kPage + tid) : 0.f;
  // all of the page is asked for before anything is done with it
  constexpr int kMine = kPage / 2 / kSumGroups, kRopeMine = kPage / kRopeGroups;
  const int word = tid & 63, group = tid >> 6;
  uint32_t v[kMine][2], rw[kRopeMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int pair = group + i * kSumGroups;
#pragma unroll
    for (int k = 0; k < 2; ++k) v[i][k] = __ldcg(reinterpret_cast<const uint32_t*>(rows + (2 * pair + k) * kRowBytes) + word);
  }
#pragma unroll
  for (int i = 0; i < kRopeMine; ++i) {
    const int t = (tid >> 4) + i * kRopeGroups;
    rw[i] = __ldcg(reinterpret_cast<const uint32_t*>(rows + t * kRowBytes + kLatent / 2) + (tid & 15));
  }
  float top = fabsf(s);
  bool unsound = !(top <= CUDART_MAX_NORMAL_F);
  top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(unsound ? 0.f : top)));  // (non-negative floats order as integers)
  if (tid == 0) unsound_s = 0;
  if (lane == 0) top_s[warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < (kPage + 31) / 32; ++i) top = fmaxf(top, top_s[i]);
  if (unsound) unsound_s = 1;
  if (tid < kPage) w_s[tid] = top > 0.f && !unsound ? int16_t(rint(32767.0 * double(s) / double(top))) : int16_t(0);
  // RoPE meanwhile: nobody waits for the weights
  float sum[4] = {};
#pragma unroll
  for (int i = 0; i < kRopeMine; ++i) {
    const float2 a = e4m3x2_to_float2(rw[i] & 0xffff), b = e4m3x2_to_float2(rw[i] >> 16);
    sum[0] += a.x;
    sum[1] += a.y;
    sum[2] += b.x;
    sum[3] += b.y;
  }
  const bool nan = !(sum[0] == sum[0] && sum[1] == sum[1] && sum[2] == sum[2] && sum[3] == sum[3]);
  if (nan) unsound_s = 1;
  *reinterpret_cast<int4*>(&rope_s[tid >> 4][4 * (tid & 15)]) =
      make_int4(int(512.f * sum[0]), int(512.f * sum[1]), int(512.f * sum[2]), int(512.f * sum[3]));
  __syncthreads();
  int acc[8] = {};
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int pair = group + i * kSumGroups;
    const int w2 = *reinterpret_cast<const int*>(w_s + 2 * pair);
    uint32_t a0, a1, b0, b1;
    e2m1x8_twice(v[i][0], a0, a1);
    e2m1x8_twice(v[i][1], b0, b1);
    const uint32_t p01 = __byte_perm(a0, b0, 0x5140), p23 = __byte_perm(a0, b0, 0x7362), p45 = __byte_perm(a1, b1, 0x5140), p67 = __byte_perm(a1, b1, 0x7362);
    acc[0] = dp2a_lo(w2, p01, acc[0]);
    acc[1] = dp2a_hi(w2, p01, acc[1]);
    acc[2] = dp2a_lo(w2, p23, acc[2]);
    acc[3] = dp2a_hi(w2, p23, acc[3]);
    acc[4] = dp2a_lo(w2, p45, acc[4]);
    acc[5] = dp2a_hi(w2, p45, acc[5]);
    acc[6] = dp2a_lo(w2, p67, acc[6]);
    acc[7] = dp2a_hi(w2, p67, acc[7]);
  }
  // (eight words each: the two halves of a row's words go to the banks side by side)
  *reinterpret_cast<int4*>(&part_s[group][4 * word]) = make_int4(acc[0], acc[1], acc[2], acc[3]);
  *reinterpret_cast<int4*>(&part_s[group][kLatent / 2 + 4 * word]) = make_int4(acc[4], acc[5], acc[6], acc[7]);
  __syncthreads();
  // a thread has dims 8 w + 2 k, + 1 (w, k: its pair's place above), the first 32 threads two of RoPE too
  const int place = 2 * tid;  // in part_s: half h of word w at h * 256 + 4 w + j
  const int dim = place < kLatent / 2 ? (place >> 2) * 8 + (place & 3) : ((place - kLatent / 2) >> 2) * 8 + 4 + (place & 3);
  int2 lat = *reinterpret_cast<const int2*>(&part_s[0][place]), rope = make_int2(0, 0);
#pragma unroll
  for (int g = 1; g < kSumGroups; ++g) {
    const int2 more = *reinterpret_cast<const int2*>(&part_s[g][place]);
    lat.x += more.x;
    lat.y += more.y;
  }
  if (warp == 0)
#pragma unroll
    for (int g = 0; g < kRopeGroups; ++g) {
      const int2 more = *reinterpret_cast<const int2*>(&rope_s[g][2 * tid]);
      rope.x += more.x;
      rope.y += more.y;
    }
  const int most_lat = __reduce_max_sync(0xffffffffu, max(abs(lat.x), abs(lat.y))), most_rope = __reduce_max_sync(0xffffffffu, max(abs(rope.x), abs(rope.y)));
  if (lane == 0) {
    most_s[0][warp] = most_lat;
    most_s[1][warp] = most_rope;
  }
  __syncthreads();
  // One warp makes the scale and what multiplies the sums; the others wait.
  constexpr double kLatUnit = 1.0 / (65534.0 * kPage), kRopeUnit = 1.0 / (512.0 * kPage);
  if (warp == 0) {
    const int ml = __reduce_max_sync(0xffffffffu, most_s[0][lane & (kWarps - 1)]), mr = most_s[1][0];
    const float scale = unsound_s ? CUDART_NAN_F : summary_scale(ml, mr, top, kLatUnit, kRopeUnit);
    if (lane == 0) {
      scale_s = scale;
      by_s[0] = summary_factor(top / scale * float(kLatUnit));
      by_s[1] = summary_factor(float(kRopeUnit) / scale);
    }
  }
  __syncthreads();
  const float scale = scale_s;
  char* out = reinterpret_cast<char*>(p.summary) + int64_t(page) * kQDim;
  const int c[2] = {summary_code(lat.x, scale, by_s[0], top, kLatUnit), summary_code(lat.y, scale, by_s[0], top, kLatUnit)};
  *reinterpret_cast<uint16_t*>(out + dim) = uint16_t((c[0] & 0xff) | (c[1] & 0xff) << 8);
  if (warp == 0) {
    const int r[2] = {summary_code(rope.x, scale, by_s[1], 1.f, kRopeUnit), summary_code(rope.y, scale, by_s[1], 1.f, kRopeUnit)};
    *reinterpret_cast<uint16_t*>(out + kLatent + 2 * lane) = uint16_t((r[0] & 0xff) | (r[1] & 0xff) << 8);
  }
  if (tid == 0) p.summary_sf[page] = scale;
}

// Four pages of 8 or 16 tokens a CTA, 64 threads each: a thread has eight dims of all tokens, so that nothing is added up across threads but RoPE, of
// which it has four dims of every fourth token.
template <int kPage>
__global__ void __launch_bounds__(kSumThreads) summarize_four_kernel(SummarizeParams p, int64_t count) {
  constexpr int kPairs = kPage / 2, kRopeMine = kPage / 4;
  __shared__ __align__(8) int16_t w_s[4][kPage];
  __shared__ float top_s[4];
  __shared__ int rope_s[4][kRope], most_s[4][2], unsound_s[4];
  __shared__ float scale_s[4], by_s[4][2];
  dependent_launch();
  const int tid = threadIdx.x, sub = tid >> 6, t = tid & 63, half = t >> 5, lane = tid & 31;
  const int64_t item = int64_t(blockIdx.x) * 4 + sub;
  const int page = item < count ? page_of_item<kPage>(p, item) : -1;
  const bool there = page >= 0;
  const uint8_t* rows = p.kv_cache + int64_t(there ? page : 0) * kPage * kRowBytes;
  const float* scales = p.kv_cache_sf + int64_t(there ? page : 0) * kPage;
  const float s = there && t < kPage ? __ldcg(scales + t) : 0.f;
  uint32_t rope[kRopeMine];
#pragma unroll
  for (int i = 0; i < kRopeMine; ++i)
    rope[i] = there ? __ldcg(reinterpret_cast<const uint32_t*>(rows + ((t >> 4) + 4 * i) * kRowBytes + kLatent / 2) + (t & 15)) : 0u;
  uint32_t v[kPairs][2];
#pragma unroll
  for (int i = 0; i < kPage; ++i) v[i >> 1][i & 1] = there ? __ldcg(reinterpret_cast<const uint32_t*>(rows + i * kRowBytes) + t) : 0u;
  const bool unsound = !(fabsf(s) <= CUDART_MAX_NORMAL_F);
  // (the page's scales are in its first warp; non-negative floats order as integers)
  float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(unsound ? 0.f : fabsf(s))));
  if (t == 0) unsound_s[sub] = 0;
  if (t == 0) top_s[sub] = top;
  __syncthreads();
  top = top_s[sub];
  if (unsound) unsound_s[sub] = 1;
  if (t < kPage) w_s[sub][t] = top > 0.f && !unsound ? int16_t(rint(32767.0 * double(s) / double(top))) : int16_t(0);
  // RoPE: sums of at most four values of at most 448 in steps of 2^-9 are exact in FP32
  float sum[4] = {};
#pragma unroll
  for (int i = 0; i < kRopeMine; ++i) {
    const float2 a = e4m3x2_to_float2(rope[i] & 0xffff), b = e4m3x2_to_float2(rope[i] >> 16);
    sum[0] += a.x;
    sum[1] += a.y;
    sum[2] += b.x;
    sum[3] += b.y;
  }
  int whole[4];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    nan |= !(sum[i] == sum[i]);
    whole[i] = int(512.f * sum[i]);
    whole[i] += __shfl_xor_sync(0xffffffffu, whole[i], 16);
  }
  if (nan) unsound_s[sub] = 1;
  if (half == 1 && lane < 16) *reinterpret_cast<int4*>(&rope_s[sub][4 * lane]) = make_int4(whole[0], whole[1], whole[2], whole[3]);
  __syncthreads();
  int acc[8] = {};
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int w2 = *reinterpret_cast<const int*>(&w_s[sub][2 * i]);
    uint32_t a0, a1, b0, b1;
    e2m1x8_twice(v[i][0], a0, a1);
    e2m1x8_twice(v[i][1], b0, b1);
    const uint32_t p01 = __byte_perm(a0, b0, 0x5140), p23 = __byte_perm(a0, b0, 0x7362), p45 = __byte_perm(a1, b1, 0x5140), p67 = __byte_perm(a1, b1, 0x7362);
    acc[0] = dp2a_lo(w2, p01, acc[0]);
    acc[1] = dp2a_hi(w2, p01, acc[1]);
    acc[2] = dp2a_lo(w2, p23, acc[2]);
    acc[3] = dp2a_hi(w2, p23, acc[3]);
    acc[4] = dp2a_lo(w2, p45, acc[4]);
    acc[5] = dp2a_hi(w2, p45, acc[5]);
    acc[6] = dp2a_lo(w2, p67, acc[6]);
    acc[7] = dp2a_hi(w2, p67, acc[7]);
  }
  int most = 0, most_rope = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, abs(acc[i]));
  most = __reduce_max_sync(0xffffffffu, most);
  if (half == 0) {  // (lanes 0-15 and 16-31 have the same sums)
    const int4 more = *reinterpret_cast<const int4*>(&rope_s[sub][4 * (lane & 15)]);
    whole[0] += more.x;
    whole[1] += more.y;
    whole[2] += more.z;
    whole[3] += more.w;
    most_rope = __reduce_max_sync(0xffffffffu, max(max(abs(whole[0]), abs(whole[1])), max(abs(whole[2]), abs(whole[3]))));
  }
  if (lane == 0) most_s[sub][half] = most;
  __syncthreads();
  constexpr double kLatUnit = 1.0 / (65534.0 * kPage), kRopeUnit = 1.0 / (512.0 * kPage);
  if (half == 0) {
    const float scale = unsound_s[sub] ? CUDART_NAN_F : summary_scale(max(most_s[sub][0], most_s[sub][1]), most_rope, top, kLatUnit, kRopeUnit);
    if (lane == 0) {
      scale_s[sub] = scale;
      by_s[sub][0] = summary_factor(top / scale * float(kLatUnit));
      by_s[sub][1] = summary_factor(float(kRopeUnit) / scale);
      if (there) p.summary_sf[page] = scale;
    }
  }
  __syncthreads();
  if (!there) return;
  const float scale = scale_s[sub], by = by_s[sub][0];
  int8_t* out = p.summary + int64_t(page) * kQDim;
  uint32_t code[2] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) code[i >> 2] |= uint32_t(summary_code(acc[i], scale, by, top, kLatUnit) & 0xff) << (8 * (i & 3));
  *reinterpret_cast<uint2*>(out + 8 * t) = make_uint2(code[0], code[1]);
  if (half == 0 && lane < 16) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= uint32_t(summary_code(whole[i], scale, by_s[sub][1], 1.f, kRopeUnit) & 0xff) << (8 * i);
    *reinterpret_cast<uint32_t*>(out + kLatent + 4 * lane) = r;
  }
}

// ------------------------------------------------------------------------------------------ selection
// A CTA per row.  A thread has kKeys consecutive keys in registers (and their block-table entries: all loads of a row are on their way at once,
// before its length is known).  The key of the last page that is taken is found by counting the keys' range in 256 buckets, going on with the
// bucket in which the count reaches what is wanted until it holds so few that they are compared with one another: one round where keys
// are spread.  A page's place in the order is its key and, below that, its index from the last one: pages that tie have places of their own.
// Then one scan gives each page that is taken its place in the table.  64 rows of 2048 pages, nothing in L2: 39.8 us by bytes of the keys, whose leading
// byte is nearly everybody's, so that all threads wanted the same counter; 9.8 by halving the range with a barrier each time; 6.7 by buckets down to
// a single key; 5.6 so, of which 1.5 are loads, 0.8 a round, 0.7 the comparing, 0.4 the scan.
// kKeys = 0: more candidates than registers hold; the keys stay in global memory and are read through L2 in each round.
constexpr int kSelMost = 1024, kBuckets = 256, kList = 128;

template <int kKeys>
__global__ void __launch_bounds__(kSelMost) select_kernel(SelectParams p) {
  __shared__ uint32_t range_s[2][32], found_s[3], listed_s;
  __shared__ alignas(16) uint32_t bucket_s[kBuckets];
  __shared__ uint64_t list_s[kList], least_s;
  dependent_launch();
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const uint32_t* keys = p.keys + int64_t(row) * p.key_stride;
  const int32_t* table = p.block_tables + int64_t(row / p.q_len) * p.block_table_stride;
  int32_t* out = p.selected + int64_t(row) * p.budget;
  uint32_t reg[kKeys ? kKeys : 1];
  constexpr bool kPagesToo = kKeys == 4;  // (with sixteen there are no registers for them)
  int32_t page[kPagesToo ? kKeys : 1];
  if constexpr (kKeys > 0) {
#pragma unroll
    for (int i = 0; i < kKeys; i += 4) {  // (a row has room for whole groups of four; what lies behind the candidates is not looked at)
      const int k = tid * kKeys + i;
      if (k >= p.width) break;
      const uint4 four = __ldcg(reinterpret_cast<const uint4*>(keys + k));
      reg[i] = four.x;
      reg[i + 1] = four.y;
      reg[i + 2] = four.z;
      reg[i + 3] = four.w;
      if constexpr (kPagesToo)
#pragma unroll
        for (int j = i; j < i + 4; ++j) page[j] = p.sink + tid * kKeys + j < p.width ? __ldcg(table + p.sink + tid * kKeys + j) : 0;
    }
  }
  for (int k = tid; k < kBuckets; k += blockDim.x) bucket_s[k] = 0;
  if (tid == 0) listed_s = 0;
  const Seen v = seen(p, row);
  if (v.used <= p.budget) {  // the budget holds them all
    for (int k = tid; k < p.budget; k += blockDim.x) out[k] = k < v.used ? __ldcg(table + k) : 0;
    if (tid == 0) p.selected_lens[row] = v.len;
    return;
  }
  const int edges = p.sink + p.local, candidates = v.used - edges, wanted = p.budget - edges;
  // the sink and the local pages: a thread's first one is asked for here and stored at the end
  auto edge_of = [&](int k) { return __ldcg(table + (k < p.sink ? k : v.used - edges + k)); };
  auto store_edge = [&](int k, int32_t page) { out[k < p.sink ? k : p.budget - edges + k] = page; };
  const int32_t edge = tid < edges ? edge_of(tid) : 0;
  const int mine = kKeys ? kKeys : (candidates + int(blockDim.x) - 1) / int(blockDim.x);
  const int first = tid * mine, last = min(first + mine, candidates);
  // f(key of a candidate, its index, i: which of this thread's)
  auto for_keys = [&](auto f) {
    if constexpr (kKeys > 0) {
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if (first + i < candidates) f(reg[i], first + i, i);
    } else {
      for (int k = first; k < last; ++k) f(__ldcg(keys + k), k, k - first);
    }
  };
  auto place_of = [](uint32_t key, int k) { return uint64_t(key) << 32 | uint32_t(~k); };
  // of this thread's count those of the threads before it, too; the last thread's is the sum
  auto scan = [&](uint32_t count) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t down = __shfl_up_sync(0xffffffffu, count, o);
      count += lane >= o ? down : 0;
    }
    if (lane == 31) range_s[0][warp] = count;
    __syncthreads();
    return count + __reduce_add_sync(0xffffffffu, lane < warp ? range_s[0][lane] : 0u);
  };
  if (wanted > 0) {
    uint32_t low = 0xffffffffu, high = 0;
    for_keys([&](uint32_t key, int, int) {
      low = min(low, key);
      high = max(high, key);
    });
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) {
      range_s[0][warp] = low;
      range_s[1][warp] = high;
    }
    __syncthreads();
    low = __reduce_min_sync(0xffffffffu, range_s[0][lane < warps ? lane : 0]);
    high = __reduce_max_sync(0xffffffffu, range_s[1][lane < warps ? lane : 0]);
    // Keys above `high` are fewer than wanted (`above`; none, to begin with), keys from `low` on are enough; `within` lie from low to high.
    uint32_t above = 0, within = candidates;
    while (low < high && within > kList) {
      const int shift = max(0, 24 - __clz(high - low));  // 256 buckets hold the range
      for_keys([&](uint32_t key, int, int) {
        if (key - low <= high - low) atomicAdd(&bucket_s[(key - low) >> shift], 1u);
      });
      __syncthreads();
      if (warp == 0) {  // lane i has the buckets 8 i to 8 i + 7: the one, from above, in which the count reaches what is wanted
        uint4* const eight = reinterpret_cast<uint4*>(bucket_s + 8 * lane);
        const uint4 a = eight[0], b = eight[1];
        eight[0] = eight[1] = make_uint4(0, 0, 0, 0);
        const uint32_t n[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += n[i];
        uint32_t from = sum;  // of this lane and those above it
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_down_sync(0xffffffffu, from, o);
          from += lane + o < 32 ? up : 0;
        }
        uint32_t over = above + from - sum;
        if (over < uint32_t(wanted) && over + sum >= uint32_t(wanted)) {
#pragma unroll
          for (int i = 7; i >= 0; --i) {
            if (over < uint32_t(wanted) && over + n[i] >= uint32_t(wanted)) {
              found_s[0] = 8 * lane + i;
              found_s[1] = over;
              found_s[2] = n[i];
            }
            over += n[i];
          }
        }
      }
      __syncthreads();
      low += found_s[0] << shift;
      above = found_s[1];
      within = found_s[2];
      high = low + min(high - low, (1u << shift) - 1);  // (the bucket's end may lie beyond 32 bits)
    }
    uint64_t least = place_of(low, -1);  // place of the last one that is taken, or below it
    const uint32_t rest = wanted - above;
    if (rest < within) {
      if (within <= kList) {  // few enough to be compared with one another
        uint32_t listed = 0;
        for_keys([&](uint32_t key, int, int) { listed += key - low <= high - low; });
        if (listed) {  // (one counter's answer a thread: an answer takes 200 clk)
          uint64_t* next = list_s + atomicAdd(&listed_s, listed);
          for_keys([&](uint32_t key, int k, int) {
            if (key - low <= high - low) *next++ = place_of(key, k);
          });
        }
        __syncthreads();
        uint64_t some[kList / 32];  // a lane has up to four of them; a warp counts those before one of them at a time
#pragma unroll
        for (int i = 0; i < kList / 32; ++i) some[i] = lane + 32 * i < within ? list_s[lane + 32 * i] : 0;
#pragma unroll 2
        for (uint32_t k = warp; k < within; k += warps) {
          const uint64_t place = list_s[k];
          uint32_t before = 1;
#pragma unroll
          for (int i = 0; i < kList / 32; ++i) before += __popc(__ballot_sync(0xffffffffu, some[i] > place));
          if (before == rest && lane == 0) least_s = place;
        }
      } else {  // all of one key: the first ones
        __syncthreads();  // (where no round was needed, a warp may still be reading the keys' range, whose place the scan takes)
        uint32_t equal = 0;
        for_keys([&](uint32_t key, int, int) { equal += key == low; });
        uint32_t before = scan(equal) - equal;
        for_keys([&](uint32_t key, int k, int) {
          if (key == low && ++before == rest) least_s = place_of(key, k);
        });
      }
      __syncthreads();
      least = least_s;
    }
    // those from `least` on are taken, in the order of their indices
    uint32_t taken = 0, which = 0;  // (which: kKeys > 0, as bits)
    for_keys([&](uint32_t key, int k, int i) {
      const bool take = place_of(key, k) >= least;
      taken += take;
      if constexpr (kKeys > 0) which |= uint32_t(take) << i;
      if constexpr (kKeys > 0 && !kPagesToo)
        if (take) reg[i] = uint32_t(__ldcg(table + p.sink + k));  // (on their way during the scan)
    });
    int32_t* next = out + p.sink + scan(taken) - taken;
    if constexpr (kKeys > 0) {
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if (which >> i & 1) *next++ = kPagesToo ? page[kPagesToo ? i : 0] : int32_t(reg[i]);
    } else {
      for_keys([&](uint32_t key, int k, int) {
        if (place_of(key, k) >= least) *next++ = __ldcg(table + p.sink + k);
      });
    }
  }
  if (tid < edges) store_edge(tid, edge);
  for (int k = tid + blockDim.x; k < edges; k += blockDim.x) store_edge(k, edge_of(k));
  if (tid == 0) p.selected_lens[row] = v.len - (v.used - p.budget) * p.page_size;
}

}  // namespace

// Which kernel, us in graphs of calls on pages that are not in L2, for 4096 / 38000 / 150000 / 300000 tokens (a CTA per page, four pages a CTA, many):
//   pages of   8   3.6 / 16.8 / 59.5 / 116     3.4 /  9.0 / 26.5 / 50.1    (sixteen pages to a tile) 12 / 25 / 65 / 120
//             16   3.7 / 10.4 / 33.5 / 64.3    3.2 /  7.9 / 21.2 / 38.3    (eight) 8.3 / 16.2 / 38.8 / 73.4
//             32   3.0 /  7.4 / 21.3 / 39.6    3.9 /  9.7 / 18.7 / 33.0    6.4 / 10.0 / 18.4 / 31.2
//             64   3.1 /  6.6 / 18.3 / 32.6    5.3 /  9.7 / 17.2 / 29.0    5.2 /  8.3 / 15.5 / 25.0
//            128   3.5 /  6.4 / 17.0 / 28.2    8.4 / 11.2 / 22.6 / 30.3    4.9 /  7.3 / 14.1 / 22.4
// With small pages what is done once a page outweighs its sums, and four share it; with large ones four in turn are longer than one by four groups.
constexpr int64_t kManyTokens = 131072;  // of a call's places for pages (76000: 11.1 with a CTA per page, 11.8)

cudaError_t launch_summarize(const SummarizeParams& p, int64_t count, int sms, cudaStream_t stream) {
  if (p.page_size <= 16) {
    const auto kernel = p.page_size == 8 ? summarize_four_kernel<8> : summarize_four_kernel<16>;
    return launch_dependent(kernel, dim3(unsigned((count + 3) / 4)), kSumThreads, 0, stream, p, count);
  }
  // (its tensor maps want a cache that starts on 32 bytes, its bulk copies scales that start on 16)
  if (count * p.page_size >= kManyTokens && reinterpret_cast<uintptr_t>(p.kv_cache) % 32 == 0 && reinterpret_cast<uintptr_t>(p.kv_cache_sf) % 16 == 0)
    return launch_summarize_many(p, count, sms, stream);
  const auto kernel = p.page_size == 32 ? summarize_kernel<32> : p.page_size == 64 ? summarize_kernel<64> : summarize_kernel<128>;
  return launch_dependent(kernel, dim3(unsigned(count)), kSumThreads, 0, stream, p);
}

cudaError_t launch_select(const SelectParams& p, int sms, cudaStream_t stream) {
  if (p.width > p.budget) {
    cudaError_t e = launch_score(p, sms, stream);
    if (e != cudaSuccess || scores_and_selects(p, sms)) return e;
  }
  // keys of the longest row that the tables can hold: four a thread while there are threads, then sixteen (none where the budget holds every row)
  const int rows = p.batch * p.q_len, most = p.width - p.sink - p.local;
  const int threads = most <= 4 * 256 ? 256 : most <= 4 * 512 ? 512 : kSelMost;
  const auto kernel = p.width <= p.budget ? select_kernel<0> : most <= 4 * kSelMost ? select_kernel<4> : most <= 16 * kSelMost ? select_kernel<16> : select_kernel<0>;
  return launch_dependent(kernel, dim3(unsigned(rows)), threads, 0, stream, p);
}

}  // namespace mla
