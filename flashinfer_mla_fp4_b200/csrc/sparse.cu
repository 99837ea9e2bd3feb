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
constexpr int kSumThreads = 320;  // 256: latent, four groups of tokens x 64 words of a row; 64: RoPE, four groups x 16 words

// twice the value of an E2M1 code
__device__ __forceinline__ int e2m1_twice(uint32_t nibble) {
  const int m = int((0x0C08060403020100ull >> (8 * (nibble & 7))) & 0xff);
  return nibble & 8 ? -m : m;
}
// 512 times the value of an E4M3 byte (not NaN)
__device__ __forceinline__ int e4m3_512(uint32_t b) {
  const int e = (b >> 3) & 15, m = b & 7, v = e ? (8 | m) << (e - 1) : m;
  return b & 0x80 ? -v : v;
}

__global__ void __launch_bounds__(kSumThreads) summarize_kernel(SummarizeParams p) {
  __shared__ int w_s[kTile];
  __shared__ int part_s[4][kQDim];
  __shared__ float top_s[kSumThreads / 32];
  __shared__ double amax_s[kSumThreads / 32];
  __shared__ int unsound_s;
  dependent_launch();
  const int tid = threadIdx.x, n = p.page_size;
  int page = -1;
  if (p.page_ids) {
    page = p.page_ids[blockIdx.x];
  } else {  // the pages that the last new_tokens positions of a request have filled, the newest first
    const int b = blockIdx.x / p.per_request, j = blockIdx.x - b * p.per_request;
    const int len = min(p.seq_lens[b], p.seq_cap), at = len / n - 1 - j;
    if (at >= 0 && (at + 1) * int64_t(n) > int64_t(len) - p.new_tokens) page = p.block_tables[int64_t(b) * p.block_table_stride + at];
  }
  if (page < 0 || page >= p.num_pages) return;
  const uint8_t* rows = p.kv_cache + int64_t(page) * n * kRowBytes;
  const float* sf = p.kv_cache_sf + int64_t(page) * n;
  const float s = tid < n ? sf[tid] : 0.f;
  float top = fabsf(s);
  int unsound = !(top <= CUDART_MAX_NORMAL_F);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tid == 0) unsound_s = 0;
  if ((tid & 31) == 0) top_s[tid >> 5] = top;
  __syncthreads();
  top = 0.f;
  for (int i = 0; i < kSumThreads / 32; ++i) top = fmaxf(top, top_s[i]);
  if (tid < n) w_s[tid] = top > 0.f && !unsound ? int(rint(32767.0 * double(s) / double(top))) : 0;
  if (unsound) unsound_s = 1;
  __syncthreads();
  if (tid < 256) {
    const int c = tid & 63;
    int acc[8] = {};
    for (int t = tid >> 6; t < n; t += 4) {
      const uint32_t v = *reinterpret_cast<const uint32_t*>(rows + t * kRowBytes + 4 * c);
      const int w = w_s[t];
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += w * e2m1_twice(v >> (4 * i));
    }
    for (int i = 0; i < 8; ++i) part_s[tid >> 6][8 * c + i] = acc[i];
  } else {
    const int c = tid & 15, g = (tid - 256) >> 4;
    int acc[4] = {};
    for (int t = g; t < n; t += 4) {
      const uint32_t v = *reinterpret_cast<const uint32_t*>(rows + t * kRowBytes + kLatent / 2 + 4 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = (v >> (8 * i)) & 0xff;
        if ((b & 0x7f) == 0x7f) unsound = 1;
        else acc[i] += e4m3_512(b);
      }
    }
    for (int i = 0; i < 4; ++i) part_s[g][kLatent + 4 * c + i] = acc[i];
    if (unsound) unsound_s = 1;
  }
  __syncthreads();
  const double lat = double(top) / (65534.0 * n), rope = 1.0 / (512.0 * n);
  double mean[2], amax = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = tid + k * kSumThreads;
    mean[k] = d < kQDim ? double(part_s[0][d] + part_s[1][d] + part_s[2][d] + part_s[3][d]) * (d < kLatent ? lat : rope) : 0.0;
    amax = fmax(amax, fabs(mean[k]));
  }
  for (int o = 16; o > 0; o >>= 1) amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((tid & 31) == 0) amax_s[tid >> 5] = amax;
  __syncthreads();
  for (int i = 0; i < kSumThreads / 32; ++i) amax = fmax(amax, amax_s[i]);
  const float scale = float(amax / 127.0);
  const bool sound = !unsound_s && scale <= CUDART_MAX_NORMAL_F;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = tid + k * kSumThreads;
    if (d < kQDim) p.summary[int64_t(page) * kQDim + d] = sound && scale > 0.f ? int8_t(fmin(fmax(rint(mean[k] / double(scale)), -127.0), 127.0)) : int8_t(0);
  }
  if (tid == 0) p.summary_sf[page] = sound ? scale : CUDART_NAN_F;
}

// ------------------------------------------------------------------------------------------ selection
// A CTA per row.  A thread has kKeys consecutive keys in registers; the key of the last page that is taken is found by halving the range of the
// keys until as many lie above the middle as are wanted, which takes about log2(candidates) + 2 counts, 32 where pages tie: a count is a
// compare per key, a reduction in the warp and one across warps behind one barrier.  (By bytes through a histogram in shared memory, whose
// counters of the leading byte everybody wants, 2045 of 64 rows took 39 us.)  Then one scan gives each page that is taken its place.
// kKeys = 0: more candidates than registers hold; the keys stay in global memory, read through L2 at each count.
constexpr int kSelMost = 1024;

template <int kKeys>
__global__ void __launch_bounds__(kSelMost) select_kernel(SelectParams p) {
  __shared__ uint32_t sum_s[2][32], range_s[2][32];
  dependent_launch();
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const uint32_t* keys = p.keys + int64_t(row) * p.key_stride;
  const Seen v = seen(p, row);
  const int32_t* table = p.block_tables + int64_t(row / p.q_len) * p.block_table_stride;
  int32_t* out = p.selected + int64_t(row) * p.budget;
  if (v.used <= p.budget) {  // the budget holds them all
    for (int k = tid; k < p.budget; k += blockDim.x) out[k] = k < v.used ? __ldcg(table + k) : 0;
    if (tid == 0) p.selected_lens[row] = v.len;
    return;
  }
  const int candidates = v.used - p.sink - p.local, wanted = p.budget - p.sink - p.local;
  const int mine = kKeys ? kKeys : (candidates + int(blockDim.x) - 1) / int(blockDim.x);
  const int first = tid * mine, last = min(first + mine, candidates);
  uint32_t reg[kKeys ? kKeys : 1];
  if constexpr (kKeys > 0) {
#pragma unroll
    for (int i = 0; i < kKeys; i += 4) {  // (a row has room for whole groups of four; what lies behind the candidates is not looked at)
      if (first + i >= candidates) break;
      const uint4 four = __ldcg(reinterpret_cast<const uint4*>(keys + first + i));
      reg[i] = four.x;
      reg[i + 1] = four.y;
      reg[i + 2] = four.z;
      reg[i + 3] = four.w;
    }
  }
  auto for_keys = [&](auto f) {  // f(place among the candidates, key)
    if constexpr (kKeys > 0) {
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if (first + i < candidates) f(first + i, reg[i]);
    } else {
      for (int k = first; k < last; ++k) f(k, __ldcg(keys + k));
    }
  };
  for (int k = tid; k < p.sink; k += blockDim.x) out[k] = __ldcg(table + k);
  for (int k = tid; k < p.local; k += blockDim.x) out[p.budget - p.local + k] = __ldcg(table + v.used - p.local + k);
  if (tid == 0) p.selected_lens[row] = v.len - (v.used - p.budget) * p.page_size;
  if (wanted == 0) return;
  uint32_t low = 0xffffffffu, high = 0;
  for_keys([&](int, uint32_t key) {
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
  // Keys above `high` are fewer than wanted (none, to begin with), keys from `low` on are enough.
  uint32_t above = 0;  // keys > high
  for (int turn = 0; low < high; ++turn) {
    const uint32_t middle = low + (high - low) / 2;
    uint32_t n = 0;
    for_keys([&](int, uint32_t key) { n += key > middle; });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sum_s[turn & 1][warp] = n;
    __syncthreads();
    n = __reduce_add_sync(0xffffffffu, lane < warps ? sum_s[turn & 1][lane] : 0u);
    if (n >= uint32_t(wanted)) {
      low = middle + 1;
      if (n == uint32_t(wanted)) {  // these are the ones
        high = middle;
        above = n;
        break;
      }
    } else {
      high = middle;
      above = n;
    }
  }
  // taken: keys > high, and of those equal to it the first wanted - above
  const uint32_t ties = uint32_t(wanted) - above;
  uint32_t more = 0, equal = 0;
  for_keys([&](int, uint32_t key) {
    more += key > high;
    equal += key == high;
  });
  uint32_t more_before = more, equal_before = equal;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, more_before, o), b = __shfl_up_sync(0xffffffffu, equal_before, o);
    more_before += lane >= o ? a : 0;
    equal_before += lane >= o ? b : 0;
  }
  __syncthreads();
  if (lane == 31) {
    range_s[0][warp] = more_before;
    range_s[1][warp] = equal_before;
  }
  __syncthreads();
  more_before += __reduce_add_sync(0xffffffffu, lane < warp ? range_s[0][lane] : 0u) - more;
  equal_before += __reduce_add_sync(0xffffffffu, lane < warp ? range_s[1][lane] : 0u) - equal;
  for_keys([&](int k, uint32_t key) {
    const bool tie = key == high;
    if (key > high || (tie && equal_before < ties)) out[p.sink + more_before + min(equal_before, ties)] = __ldcg(table + p.sink + k);
    more_before += key > high;
    equal_before += tie;
  });
}

}  // namespace

cudaError_t launch_summarize(const SummarizeParams& p, int64_t ctas, cudaStream_t stream) {
  return launch_dependent(summarize_kernel, dim3(unsigned(ctas)), kSumThreads, 0, stream, p);
}

cudaError_t launch_select(const SelectParams& p, int sms, cudaStream_t stream) {
  if (p.width > p.budget) {
    cudaError_t e = launch_score(p, sms, stream);
    if (e != cudaSuccess) return e;
  }
  // keys of the longest row that the tables can hold: four a thread while there are threads, then sixteen
  const int rows = p.batch * p.q_len, most = p.width - p.sink - p.local;
  const int threads = most <= 4 * 256 ? 256 : most <= 4 * 512 ? 512 : kSelMost;
  const auto kernel = most <= 4 * kSelMost ? select_kernel<4> : most <= 16 * kSelMost ? select_kernel<16> : select_kernel<0>;
  return launch_dependent(kernel, dim3(unsigned(rows)), threads, 0, stream, p);
}

}  // namespace mla
