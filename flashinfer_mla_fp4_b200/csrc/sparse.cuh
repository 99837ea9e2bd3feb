// What the kernels of sparse decode and of the page pool share.
#pragma once

#include <cuda_fp16.h>

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

}  // namespace mla
