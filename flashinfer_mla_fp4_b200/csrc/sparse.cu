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
constexpr int kSelThreads = 512;

// Sum over the CTA of the values before this thread's; *total: of all.
__device__ __forceinline__ int scan_before(bool flag, int* warp_s, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ballot = __ballot_sync(0xffffffffu, flag);
  __syncthreads();
  if (lane == 0) warp_s[warp] = __popc(ballot);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const int n = warp_s[w];
    before += w < warp ? n : 0;
    all += n;
  }
  *total = all;
  return before + __popc(ballot & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(SelectParams p) {
  __shared__ int hist_s[256], warp_s[kSelThreads / 32];
  __shared__ uint32_t digit_s, above_s;
  dependent_launch();
  const int row = blockIdx.x, tid = threadIdx.x;
  const Seen v = seen(p, row);
  const int32_t* table = p.block_tables + int64_t(row / p.q_len) * p.block_table_stride;
  int32_t* out = p.selected + int64_t(row) * p.budget;
  if (v.used <= p.budget) {  // the budget holds them all
    for (int k = tid; k < p.budget; k += kSelThreads) out[k] = k < v.used ? table[k] : 0;
    if (tid == 0) p.selected_lens[row] = v.len;
    return;
  }
  const int candidates = v.used - p.sink - p.local, wanted = p.budget - p.sink - p.local;
  const uint32_t* keys = p.keys + int64_t(row) * p.width;
  for (int k = tid; k < p.sink; k += kSelThreads) out[k] = table[k];
  for (int k = tid; k < p.local; k += kSelThreads) out[p.budget - p.local + k] = table[v.used - p.local + k];
  if (tid == 0) p.selected_lens[row] = v.len - (v.used - p.budget) * p.page_size;
  if (wanted == 0) return;
  // the key of the last page that is taken, byte by byte; left: how many of the keys with the bytes so far are still wanted
  uint32_t prefix = 0, left = wanted;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int k = tid; k < 256; k += kSelThreads) hist_s[k] = 0;
    __syncthreads();
    for (int k = tid; k < candidates; k += kSelThreads)
      if (shift == 24 || (__ldcg(keys + k) >> (shift + 8)) == prefix) atomicAdd(&hist_s[(__ldcg(keys + k) >> shift) & 255], 1);
    __syncthreads();
    if (tid == 0) {
      uint32_t above = 0;
      int d = 255;
      while (above + hist_s[d] < left) above += hist_s[d--];
      digit_s = d;
      above_s = above;
    }
    __syncthreads();
    prefix = (prefix << 8) | digit_s;
    left -= above_s;
  }
  int taken = 0, ties = 0;
  for (int base = 0; base < candidates; base += kSelThreads) {
    const int k = base + tid;
    const uint32_t key = k < candidates ? __ldcg(keys + k) : 0;
    int n, m;
    const bool tie = k < candidates && key == prefix;
    const int before = scan_before(tie, warp_s, &n);
    const bool take = k < candidates && (key > prefix || (tie && ties + before < int(left)));
    const int at = scan_before(take, warp_s, &m);
    if (take) out[p.sink + taken + at] = table[p.sink + k];
    taken += m;
    ties += n;
  }
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
  return launch_dependent(select_kernel, dim3(unsigned(p.batch * p.q_len)), kSelThreads, 0, stream, p);
}

}  // namespace mla
