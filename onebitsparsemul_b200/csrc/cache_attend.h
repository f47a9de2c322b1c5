// What the two cache attention kernels share. Internal header.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace ob {

// many query rows per cache head (cache_attend_sm100.cu)
int64_t cache_attend_many_workspace(const CacheAttendCall& c);
cudaError_t launch_cache_attend_many(const CacheAttendCall& c, void* workspace, cudaStream_t stream);

}  // namespace ob

namespace ob_block {

// two e4m3 bytes (low or high half of a word) -> two fp16, exact
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

}  // namespace ob_block
