// Summaries of many pages of 32, 64 or 128 tokens (mathematics: sparse.cu) with the latent sums on the tensor cores.
//
// sum_t w_t e_td is a product of the page's latent, transposed, with its weights.  The latent goes to tcgen05.mma.kind::f8f6f4 as the E2M1
// codes that it is (MN-major, by TMA in the MMA's 4-bit form, as in the decode kernel), 128 tokens x 128 dims at a time.  The 15 bits of a
// weight go in as four hexadecimal digits, which E4M3 holds exactly: four columns per page, and zero for the tokens of the tile's other
// pages.  A digit's sum is a whole number of halves below 2^15: exact in the FP32 accumulator, and the sums of the four digits, shifted, are
// the same integer that summarize_kernel (sparse.cu) adds up.
//
// Bound by the copies: 324 bytes a token from HBM, of which the latent comes in pieces of 64 bytes; a tile takes 2300 to 2450 clk, as in the
// decode kernel, where its bytes at the measured rate would take 1800.  What the other kernel spends on taking codes apart (two pages of 64
// tokens: some 8000 warp instructions at 3 a clk) is done by 16 MMAs.  8192 pages of 64 tokens: 54 us there, 39.0 here, floor 27.2.
//
// Roles: warp 0 TMA, warp 1 MMAs, warps 4-7 (front) weights and RoPE sums, warps 8-15 (back) sums out of TMEM, scales, codes; the two
// groups of the back take the tiles in turn (one group: 2900 clk a tile).  Scales and RoPE bytes come with the tile (read by the
// front itself, a tile ahead, they waited behind the rows of all tiles on their way).  Rows brought into L2 ahead of their copies by the same TMA
// unit made no difference.  All waits are bounded; one that runs out sets the status and ends the CTA, whose pages are then not
// all written.
#include <cuda_fp8.h>
#include <math_constants.h>

#include "common.cuh"
#include "launch.h"
#include "ptx_sm100.cuh"
#include "sparse.cuh"

namespace mla {

namespace {

constexpr int kFront = 4, kBack = 8, kBacks = 2;      // first warps of the front's four and of the back's groups of four
constexpr int kThreads = 32 * (kBack + 4 * kBacks);
constexpr int kDigits = 4, kCols = 16;                // of the MMAs: four for each of up to four pages
constexpr int kBlockBytes = kTile * 128;              // 128 tokens x 128 dims in the MMA's 4-bit form
constexpr int kLatBytes = kLatent / 128 * kBlockBytes, kRopeBytes = kTile * kRope, kScaleBytes = kTile * 4, kWeightBytes = kCols * 128;
constexpr int kStages = 3;                            // tiles in shared memory
constexpr int kBufs = 4, kInBufs = 2;                 // between front and back: sums; weights and RoPE sums, which are let go earlier
constexpr int kTmem = kBufs * 4 * kCols;              // tiles x four blocks of dims
constexpr int kRopeParts = 4;                         // partial RoPE sums of a tile, of 32 tokens each
constexpr int kRopeNan = 1 << 27;                     // stands for a partial sum with a NaN: sums without are below 2^25

struct Small {
  int rope[kInBufs][kRopeParts][kRope];
  float top[kBufs][4];       // largest |scale| of a page, +inf where one is not finite
  int page[kBufs][4];        // its number, -1: none
  int stage_page[kStages][4];
  float front_top[2][4];     // of the front's warps
  struct Back {              // what a group of the back hands round
    int most_lat[4][4], most_rope[4][2];
    float scale[4], by_lat[4], by_rope[4];
  } back[kBacks];
  unsigned long long full[kStages], empty[kStages], weights[kBufs], sums[kBufs], free[kBufs], rope_free[kInBufs], drained;
  uint32_t tmem;
  volatile int abort;
};

// shared memory, from a 1024-byte boundary on: latent [3 stages], weights [2], RoPE [3], scales [3], then Small
constexpr size_t kSmemBytes = 1024 + kStages * size_t(kLatBytes + kRopeBytes + kScaleBytes) + kInBufs * size_t(kWeightBytes) + sizeof(Small);
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

__device__ __forceinline__ uint32_t bar(const unsigned long long& b) { return ptx::smem_u32(&b); }

// Of a whole warp, and bounded: false when it ran out, here or in another role.  The lanes vote: one that gave up alone would leave the
// others in front of what a warp does together.  What comes after the first poll is out of line (in line 41.2 us for 8192 pages of 64 tokens, so 39.1).
__device__ __noinline__ bool wait_on(const SummarizeParams& p, Small& s, uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t i = 1; i < p.wait_polls; ++i) {
    if (__any_sync(0xffffffffu, s.abort)) return false;
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  }
  if ((threadIdx.x & 31) == 0) {
    s.abort = 1;
    report_timeout(p.status, bar, parity);
  }
  __syncwarp();
  return false;
}
__device__ __forceinline__ bool wait(const SummarizeParams& p, Small& s, const unsigned long long& b, uint32_t parity) {
  return __all_sync(0xffffffffu, ptx::mbar_try_wait(bar(b), parity)) || wait_on(p, s, bar(b), parity);
}

template <int kPage>
__global__ void __launch_bounds__(kThreads, 1) summarize_many_kernel(SummarizeParams p, int64_t count, const __grid_constant__ CUtensorMap map,
                                                                      const __grid_constant__ CUtensorMap map_rope) {
  static_assert(kPage >= 32 && kTile / kPage * kDigits <= kCols, "pages of a tile");
  constexpr int kPages = kTile / kPage;
  extern __shared__ char raw[];
  char* a_smem = raw + ((1024 - (ptx::smem_u32(raw) & 1023)) & 1023);
  char* b_smem = a_smem + kStages * kLatBytes;
  char* rope_smem = b_smem + kInBufs * kWeightBytes;
  float* scale_smem = reinterpret_cast<float*>(rope_smem + kStages * kRopeBytes);
  Small& s = *reinterpret_cast<Small*>(scale_smem + kStages * kTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kInBufs * kWeightBytes / 16; i += kThreads) reinterpret_cast<uint4*>(b_smem)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(bar(s.full[i]), 1);
      ptx::mbar_init(bar(s.empty[i]), 1 + 4);
    }
    for (int i = 0; i < kBufs; ++i) {
      ptx::mbar_init(bar(s.weights[i]), 4);
      ptx::mbar_init(bar(s.sums[i]), 1);
      ptx::mbar_init(bar(s.free[i]), 4);
    }
    for (int i = 0; i < kInBufs; ++i) ptx::mbar_init(bar(s.rope_free[i]), 4);
    ptx::mbar_init(bar(s.drained), 1);
    s.abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map);
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s.tmem), kTmem);
    ptx::tmem_relinquish();
  }
  ptx::fence_proxy_async_smem();
  ptx::tc_fence_before();
  dependent_launch();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s.tmem;
  const int64_t tiles = (count + kPages - 1) / kPages;
  const int mine = int((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);  // tiles blockIdx.x, + gridDim.x, ...
  auto page_at = [&](int n, int i) {  // page i of this CTA's tile n, -1: none
    const int64_t item = (blockIdx.x + int64_t(n) * gridDim.x) * kPages + i;
    return n < mine && item < count ? page_of_item<kPage>(p, item) : -1;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ latent by TMA
    int page = lane < kPages ? page_at(0, lane) : -1, next = lane < kPages ? page_at(1, lane) : -1, n = 0;
    bool ok = true;
    for (; n < mine; ++n, page = next, next = lane < kPages ? page_at(n + 1, lane) : -1) {
      const int st = n % kStages;
      if (n >= kStages) ok = wait(p, s, s.empty[st], (n / kStages - 1) & 1);
      if (!ok) break;
      const uint32_t there = __ballot_sync(0xffffffffu, page >= 0), full = bar(s.full[st]);
      if (lane < kPages) s.stage_page[st][lane] = page;
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_expect_tx(full, uint32_t(__popc(there)) * kPage * (kLatent / 2 + kRope + 4));
      __syncwarp();
      if (page >= 0) {
        const uint32_t dst = ptx::smem_u32(a_smem) + st * kLatBytes + lane * kPage * 128;
#pragma unroll
        for (int j = 0; j < kLatent / 128; ++j) ptx::tma_load_3d(dst + j * kBlockBytes, &map, full, 128 * j, 0, page);
        ptx::tma_load_3d(ptx::smem_u32(rope_smem) + st * kRopeBytes + lane * kPage * kRope, &map_rope, full, kLatent / 2, 0, page);
        ptx::bulk_load(ptx::smem_u32(scale_smem) + st * kScaleBytes + lane * kPage * 4, p.kv_cache_sf + int64_t(page) * kPage, kPage * 4, full);
      }
    }
    if (!ok && lane == 0)  // copies in flight land before the CTA ends; they wait for nobody
      for (int k = n < kStages ? 0 : n - kStages; k < n; ++k)
        for (uint32_t i = 0; i < (1u << 20) && !ptx::mbar_try_wait(bar(s.full[k % kStages]), (k / kStages) & 1); ++i) {
        }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMAs
    const uint32_t e = ptx::elect_one();
    const uint64_t a0 = ptx::smem_desc(ptx::smem_u32(a_smem), kBlockBytes, 1024, 2);  // MN-major: 32 tokens are four groups of 8 rows
    const uint64_t b0 = ptx::smem_desc(ptx::smem_u32(b_smem), 16, 1024, 2);           // K-major: 128 tokens a row
    constexpr uint32_t kIdesc = ptx::idesc_e4m3(128, kCols, true, false) | (5u << 7);  // A: E2M1
    bool ok = true;
    for (int n = 0; n < mine; ++n) {
      const int st = n % kStages, b = n % kBufs;
      ok = wait(p, s, s.weights[b], (n / kBufs) & 1) && wait(p, s, s.full[st], (n / kStages) & 1);  // (with the weights the accumulator is free too)
      if (!ok) break;
      ptx::tc_fence_after();
#pragma unroll
      for (uint32_t j = 0; j < kLatent / 128; ++j)
#pragma unroll
        for (uint32_t k = 0; k < kTile / 32; ++k)
          ptx::umma_f8(e, tmem + b * (4 * kCols) + j * kCols, a0 + ((st * kLatBytes + j * kBlockBytes) >> 4) + 256 * k, b0 + (((n % kInBufs) * kWeightBytes) >> 4) + 2 * k, kIdesc, k);
      if (e) {
        ptx::umma_commit(bar(s.empty[st]));
        ptx::umma_commit(bar(s.sums[b]));
      }
      __syncwarp();
    }
    // nothing is in flight when TMEM is given back; the MMAs wait for nobody, so this ends whatever the poll budget is
    if (e) ptx::umma_commit(bar(s.drained));
    for (uint32_t i = 0; i < max(p.wait_polls, 1u << 16) && !ptx::mbar_try_wait(bar(s.drained), 0); ++i) {
    }
    __syncwarp();
  } else if (warp >= kFront && warp < kFront + 4) {
    // ------------------------------------------------------------------ front: a thread has a token, and four RoPE dims of sixteen tokens
    const int t = tid - 32 * kFront, in_page = t % kPage, mine_page = t / kPage, part = t >> 4, word = t & 15;
    for (int n = 0; n < mine; ++n) {
      const int st = n % kStages, b = n % kBufs;
      bool ok = wait(p, s, s.full[st], (n / kStages) & 1);
      const char* rows = rope_smem + st * kRopeBytes;
      const int page = s.stage_page[st][mine_page];
      const float scale = page >= 0 ? scale_smem[st * kTile + t] : 0.f;  // (what lies where no page was copied is nothing)
      uint32_t words[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) words[i] = *reinterpret_cast<const uint32_t*>(rows + (16 * part + i) * kRope + 4 * word);
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(s.empty[st]));
      float top = fabsf(scale);
      if (!(top <= CUDART_MAX_NORMAL_F)) top = CUDART_INF_F;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (kPage > 32 && lane == 0) s.front_top[n & 1][warp - kFront] = top;
      // the accumulator, the weights (once the MMAs of the tile that had them are over) and the RoPE sums of that tile
      if (ok && n >= kBufs) ok = wait(p, s, s.free[b], (n / kBufs - 1) & 1);
      if (ok && n >= kInBufs) ok = wait(p, s, s.sums[(n - kInBufs) % kBufs], ((n - kInBufs) / kBufs) & 1) && wait(p, s, s.rope_free[n % kInBufs], (n / kInBufs - 1) & 1);
      if (ptx::bar_or(1, 128, !ok)) break;
      if (kPage > 32) {
#pragma unroll
        for (int i = 0; i < kPage / 32; ++i) top = fmaxf(top, s.front_top[n & 1][mine_page * (kPage / 32) + i]);
      }
      // the weight's digits, with its sign
      const int w = top > 0.f && top <= CUDART_MAX_NORMAL_F ? int(rint(32767.0 * double(scale) / double(top))) : 0;
      const int a = abs(w);
      const uint32_t sign = w < 0 ? 0x8080u : 0u;
      const uint32_t d01 = __nv_cvt_float2_to_fp8x2(make_float2(float(a & 15), float((a >> 4) & 15)), __NV_SATFINITE, __NV_E4M3) | sign;
      const uint32_t d23 = __nv_cvt_float2_to_fp8x2(make_float2(float((a >> 8) & 15), float(a >> 12)), __NV_SATFINITE, __NV_E4M3) | sign;
#pragma unroll
      for (int k = 0; k < kDigits; ++k) {
        const int row = mine_page * kDigits + k;
        b_smem[(n % kInBufs) * kWeightBytes + (row >> 3) * 1024 + (row & 7) * 128 + (((t >> 4) ^ (row & 7)) << 4) + (t & 15)] = char((k < 2 ? d01 : d23) >> (8 * (k & 1)));
      }
      if (in_page == 0) {
        s.top[b][mine_page] = top;
        s.page[b][mine_page] = page;
      }
      ptx::fence_proxy_async_smem();
      // RoPE: sums of 16 values of at most 448 in steps of 2^-9 are exact in FP32
      float sum[4] = {};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = e4m3x2_to_float2(words[i] & 0xffff), y = e4m3x2_to_float2(words[i] >> 16);
        sum[0] += x.x;
        sum[1] += x.y;
        sum[2] += y.x;
        sum[3] += y.y;
      }
      int whole[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        whole[i] = sum[i] == sum[i] ? int(512.f * sum[i]) : kRopeNan;
        whole[i] += __shfl_xor_sync(0xffffffffu, whole[i], 16);  // the warp's other sixteen tokens are of the same page
      }
      if (lane < 16) *reinterpret_cast<int4*>(&s.rope[n % kInBufs][part >> 1][4 * word]) = make_int4(whole[0], whole[1], whole[2], whole[3]);
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(s.weights[b]));
    }
  } else if (warp >= kBack) {
    // ------------------------------------------------------------------ back: a thread has a dim of each block, and a RoPE dim of every other page
    const int group = (warp - kBack) >> 2, t = tid & 127, quarter = warp & 3, half = t >> 6, rope_dim = t & 63;
    auto& g = s.back[group];
    constexpr int kRopeMine = (kPages + 1) / 2, kPagesParts = kRopeParts / kPages;
    constexpr double kLatUnit = 1.0 / (65534.0 * kPage), kRopeUnit = 1.0 / (512.0 * kPage);
    for (int n = group; n < mine; n += kBacks) {
      const int b = n % kBufs;
      const bool ok = wait(p, s, s.weights[b], (n / kBufs) & 1) && wait(p, s, s.sums[b], (n / kBufs) & 1);
      if (ptx::bar_or(2 + group, 128, !ok)) break;
      ptx::tc_fence_after();
      int lat[kPages][4], rope[kRopeMine];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t d[kCols];
        ptx::tmem_ld16(tmem + (uint32_t(quarter) << 21) + b * (4 * kCols) + j * kCols, d);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < kPages; ++i) {
          int sum = 0;
#pragma unroll
          for (int k = kDigits - 1; k >= 0; --k) sum = sum * 16 + __float2int_rn(2.f * __uint_as_float(d[kDigits * i + k]));
          lat[i][j] = sum;
        }
      }
#pragma unroll
      for (int i = 0; i < kPages; ++i) {
        const int most = __reduce_max_sync(0xffffffffu, max(max(abs(lat[i][0]), abs(lat[i][1])), max(abs(lat[i][2]), abs(lat[i][3]))));
        if (lane == 0) g.most_lat[i][quarter] = most;
      }
#pragma unroll
      for (int k = 0; k < kRopeMine; ++k) {
        const int i = 2 * k + half;
        int sum = 0;
        if (i < kPages)
#pragma unroll
          for (int part = 0; part < kPagesParts; ++part) sum += s.rope[n % kInBufs][i * kPagesParts + part][rope_dim];
        rope[k] = sum;
        const int most = __reduce_max_sync(0xffffffffu, abs(sum));
        if (lane == 0 && i < kPages) g.most_rope[i][quarter & 1] = most;
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(s.rope_free[n % kInBufs]));
      ptx::bar_sync(2 + group, 128);
      if (t < kPages) {
        const int ml = max(max(g.most_lat[t][0], g.most_lat[t][1]), max(g.most_lat[t][2], g.most_lat[t][3])), mr = max(g.most_rope[t][0], g.most_rope[t][1]);
        const float top = s.top[b][t];
        float scale = summary_scale(ml, mr, top, kLatUnit, kRopeUnit);
        if (!(top <= CUDART_MAX_NORMAL_F) || mr >= kRopeNan / 2) scale = CUDART_NAN_F;
        g.scale[t] = scale;
        g.by_lat[t] = summary_factor(top / scale * float(kLatUnit));
        g.by_rope[t] = summary_factor(float(kRopeUnit) / scale);
        if (s.page[b][t] >= 0) p.summary_sf[s.page[b][t]] = scale;
      }
      ptx::bar_sync(2 + group, 128);
#pragma unroll
      for (int i = 0; i < kPages; ++i) {
        const int page = s.page[b][i];
        if (page < 0) continue;
        const float scale = g.scale[i], by = g.by_lat[i], top = s.top[b][i];
        int8_t* out = p.summary + int64_t(page) * kQDim;
#pragma unroll
        for (int j = 0; j < 4; ++j) out[128 * j + t] = int8_t(summary_code(lat[i][j], scale, by, top, kLatUnit));
      }
#pragma unroll
      for (int k = 0; k < kRopeMine; ++k) {
        const int i = 2 * k + half, page = i < kPages ? s.page[b][i] : -1;
        if (page >= 0) p.summary[int64_t(page) * kQDim + kLatent + rope_dim] = int8_t(summary_code(rope[k], g.scale[i], g.by_rope[i], 1.f, kRopeUnit));
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(s.free[b]));
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmem);
  }
}

template <int kPage>
cudaError_t launch(const SummarizeParams& p, int64_t count, int sms, cudaStream_t stream) {
  CUtensorMap latent, rope;
  if (!encode_latent_map(p.kv_cache, p.num_pages, kPage, kPage, &latent) || !encode_rope_map(p.kv_cache, p.num_pages, kPage, kPage, false, &rope))
    return cudaErrorInvalidValue;
  static std::atomic<bool> allowed[64];
  cudaError_t e = allow_smem(summarize_many_kernel<kPage>, kSmemBytes, allowed);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (count + kTile / kPage - 1) / (kTile / kPage);
  return launch_dependent(summarize_many_kernel<kPage>, dim3(unsigned(tiles < sms ? tiles : sms)), kThreads, kSmemBytes, stream, p, count, latent, rope);
}

}  // namespace

cudaError_t launch_summarize_many(const SummarizeParams& p, int64_t count, int sms, cudaStream_t stream) {
  return p.page_size == 32 ? launch<32>(p, count, sms, stream) : p.page_size == 64 ? launch<64>(p, count, sms, stream) : launch<128>(p, count, sms, stream);
}

}  // namespace mla
