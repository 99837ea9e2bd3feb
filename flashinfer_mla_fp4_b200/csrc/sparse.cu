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
// tie do so by value.
#include <math_constants.h>

#include "common.cuh"
#include "launch.h"

namespace mla {

namespace {

__device__ __forceinline__ void dependent_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

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

// ------------------------------------------------------------------------------------------ scores
constexpr int kScoreThreads = 256;
constexpr int kScorePages = 64;             // pages per CTA
constexpr int kWordsQ = kQDim / 4;          // 144 words of four codes
constexpr int kPadWords = kWordsQ + 1;      // a head's row in shared memory, padded against bank conflicts

// What a query position sees of its request.
struct Seen {
  int len, used;  // tokens, pages
};
__device__ __forceinline__ Seen seen(const SelectParams& p, int row) {
  const int b = row / p.q_len, i = row - b * p.q_len;
  int len = min(p.seq_lens[b], p.seq_cap);
  if (p.causal) len -= p.q_len - 1 - i;
  len = max(len, 0);
  return {len, (len - 1 + p.page_size) / p.page_size};
}
// a score as an integer that orders as the score does: NaN first, then by value, zeros of either sign alike
__device__ __forceinline__ uint32_t key_of(float score) {
  if (score != score) return 0xffffffffu;
  const uint32_t u = __float_as_uint(score + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kScoreThreads) score_kernel(SelectParams p) {
  extern __shared__ uint32_t q_s[];  // [heads][kPadWords] codes, then [heads] units, then [8 warps][kWordsQ] a page each
  dependent_launch();
  const int row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Seen v = seen(p, row);
  if (v.used <= p.budget) return;
  const int candidates = v.used - p.sink - p.local, first = blockIdx.x * kScorePages;
  if (first >= candidates) return;
  float* unit_s = reinterpret_cast<float*>(q_s + p.heads * kPadWords);
  uint32_t* page_s = q_s + p.heads * (kPadWords + 1) + warp * kWordsQ;
  const int b = row / p.q_len, i = row - b * p.q_len;
  const uint8_t* q = p.q + b * p.q_stride_batch + i * p.q_stride_qpos;
  for (int h = warp; h < p.heads; h += kScoreThreads / 32) {
    const uint32_t* qh = reinterpret_cast<const uint32_t*>(q + h * p.q_stride_head);
    uint32_t w[5], e = 1;
    for (int k = 0; k < 5; ++k) {
      w[k] = lane + 32 * k < kWordsQ ? qh[lane + 32 * k] : 0;
      for (int j = 0; j < 4; ++j) {
        const uint32_t m = (w[k] >> (8 * j)) & 0x7f;
        if (m != 0x7f) e = max(e, m >> 3);
      }
    }
    e = __reduce_max_sync(0xffffffffu, e);
    for (int k = 0; k < 5; ++k) {
      if (lane + 32 * k >= kWordsQ) break;
      uint32_t out = 0;
      for (int j = 0; j < 4; ++j) {
        const uint32_t byte = (w[k] >> (8 * j)) & 0xff;
        // value * 2^(13 - e), from 512 times the value
        const float x = (byte & 0x7f) == 0x7f ? 0.f : float(e4m3_512(byte)) * __uint_as_float((127 + 4 - e) << 23);
        out |= (uint32_t(__float2int_rn(x)) & 0xff) << (8 * j);
      }
      q_s[h * kPadWords + lane + 32 * k] = out;
    }
    if (lane == 0) unit_s[h] = __uint_as_float((127 + e - 13) << 23);
  }
  __syncthreads();
  const int32_t* table = p.block_tables + int64_t(b) * p.block_table_stride + p.sink;
  for (int c = first + warp; c < min(first + kScorePages, candidates); c += kScoreThreads / 32) {
    const int page = table[c];
    uint32_t key = 0;  // a page outside the pool comes last
    if (page >= 0 && page < p.num_pages) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.summary + int64_t(page) * kQDim);
      __syncwarp();
      for (int k = lane; k < kWordsQ; k += 32) page_s[k] = src[k];
      __syncwarp();
      float best = -CUDART_INF_F;
      for (int h = lane; h < p.heads; h += 32) {
        int dot = 0;
        for (int k = 0; k < kWordsQ; ++k) dot = __dp4a(int(q_s[h * kPadWords + k]), int(page_s[k]), dot);
        best = fmaxf(best, float(dot) * unit_s[h]);
      }
      for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
      key = key_of(best * p.summary_sf[page]);
    }
    if (lane == 0) p.keys[int64_t(row) * p.width + c] = key;
  }
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
      if (shift == 24 || (keys[k] >> (shift + 8)) == prefix) atomicAdd(&hist_s[(keys[k] >> shift) & 255], 1);
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
    const uint32_t key = k < candidates ? keys[k] : 0;
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

template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

cudaError_t launch_summarize(const SummarizeParams& p, int64_t ctas, cudaStream_t stream) {
  return launch_dependent(summarize_kernel, dim3(unsigned(ctas)), kSumThreads, 0, stream, p);
}

cudaError_t launch_select(const SelectParams& p, cudaStream_t stream) {
  const int rows = p.batch * p.q_len, most = p.width - p.sink - p.local;  // candidates of the longest request
  if (p.width > p.budget) {
    const size_t smem = size_t(p.heads) * (kPadWords + 1) * 4 + size_t(kScoreThreads / 32) * kWordsQ * 4;
    cudaError_t e = cudaFuncSetAttribute(score_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    e = launch_dependent(score_kernel, dim3(unsigned((most + kScorePages - 1) / kScorePages), unsigned(rows)), kScoreThreads, smem, stream, p);
    if (e != cudaSuccess) return e;
  }
  return launch_dependent(select_kernel, dim3(unsigned(rows)), kSelThreads, 0, stream, p);
}

}  // namespace mla
