// What the kernels of sparse decode and of the page pool share.
#pragma once

#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "launch.h"

namespace mla {

// A dependent launch: its CTAs are in place when the kernel before it ends, and so are those of the kernel after it.
__device__ __forceinline__ void dependent_launch() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
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

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two_bytes) {
  uint32_t r;
  asm("{\n\t.reg .b16 b;\n\tcvt.u16.u32 b, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(two_bytes));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two_bytes) {
  const uint32_t h = e4m3x2_to_f16x2(two_bytes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Allows a kernel that much dynamic shared memory, once per device (setting it twice is harmless).
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, size_t bytes, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const bool known = dev >= 0 && dev < 64;
  if (known && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  if (e == cudaSuccess && known) done[dev].store(true, std::memory_order_release);
  return e;
}

// What a query position sees of its request.
struct Seen {
  int len, used;  // tokens, pages
};
__device__ __forceinline__ Seen seen(const SelectParams& p, int row) {
  const int b = row / p.q_len, i = row - b * p.q_len;
  int len = min(__ldcg(p.seq_lens + b), p.seq_cap);
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


// The page of an item of a summary call, -1 where there is none: of the list, or the j-th newest of the pages that the last new_tokens positions of
// a request have filled.
template <int kPage>
__device__ __forceinline__ int page_of_item(const SummarizeParams& p, int64_t item) {
  int page = -1;
  if (p.page_ids) {
    page = __ldcg(p.page_ids + item);
  } else {
    const int b = int(item / p.per_request), j = int(item - int64_t(b) * p.per_request);
    const int len = min(__ldcg(p.seq_lens + b), p.seq_cap), at = len / kPage - 1 - j;
    if (at >= 0 && (at + 1) * int64_t(kPage) > int64_t(len) - p.new_tokens) page = __ldcg(p.block_tables + int64_t(b) * p.block_table_stride + at);
  }
  return page >= 0 && page < p.num_pages ? page : -1;
}
// The scale of a summary, max(most_lat * top * lat_unit, most_rope * rope_unit) / 127 to the nearest FP32 value; NaN where that is not finite.  A quotient
// in FP32, and the exact remainder in 64 bits says whether a neighbour is nearer (a division in 64 bits is several hundred clk;
// a quotient half-way between two FP32 values has more bits than these sums give it).
__device__ __forceinline__ float summary_scale(int most_lat, int most_rope, float top, double lat_unit, double rope_unit) {
  const double largest = fmax(double(most_lat) * (double(top) * lat_unit), double(most_rope) * rope_unit);
  const float q = __double2float_rn(largest * (1.0 / 127.0));
  if (!(q < 3e38f)) return __uint_as_float(0x7fffffffu);
  if (q < 1e-30f) return float(largest / 127.0);  // (where an ulp is not a fixed part of the value)
  const float up = __uint_as_float(__float_as_uint(q) + 1), down = __uint_as_float(__float_as_uint(q) - 1);
  const double off = fma(-127.0, double(q), largest);  // q is the nearest but for the rounding of the product
  return off > 63.5 * double(up - q) ? up : off < -63.5 * double(q - down) ? down : q;
}
// What takes a sum to its code, kept finite: beside a part of the page that outweighs it beyond FP32 it would be infinite, and infinity times a sum of zero
// NaN.  No other sum meets a factor that large: the scale is at least |sum| * top * unit / 127, or half that where it is subnormal.
__device__ __forceinline__ float summary_factor(float by) { return fminf(by, __uint_as_float(0x7f7fffffu)); }
// round(sum * top * unit / scale), within [-127, 127]; 0 where the scale is 0 or NaN.  `by` is top * unit / scale in FP32, and will do unless the
// product is too near the middle of two whole numbers (it is off by less than 2^-14: roundings of 5 * 127 half-ulps of 1): then the
// sum is compared with the middle in 64 bits.
__device__ __forceinline__ int summary_code(int sum, float scale, float by, float top, double unit) {
  const float x = float(sum) * by;
  float whole = rintf(x);
  const float middle = truncf(x) + copysignf(0.5f, x);
  if (!(fabsf(x - middle) > 0x1p-14f)) {
    const double over = fma(double(-middle), double(scale), double(sum) * (double(top) * unit));  // of the middle, times the scale
    const float toward = copysignf(0.5f, x);
    whole = over == 0.0 ? rintf(middle) : (over > 0.0) == (x > 0.f) ? middle + toward : middle - toward;
  }
  return scale > 0.f ? int(fminf(fmaxf(whole, -127.f), 127.f)) : 0;
}

// what a bounded wait that ran out leaves in the status words: the first one's record, as in the decode kernel
__device__ __forceinline__ void report_timeout(int32_t* status, uint32_t bar, uint32_t parity) {
  if (!status || atomicCAS(status, 0, MLA_FP4_ERR_DEVICE_TIMEOUT) != 0) return;
  status[1] = int(bar);
  status[2] = blockIdx.x;
  status[3] = threadIdx.x;
  status[4] = int(parity);
}

}  // namespace mla
