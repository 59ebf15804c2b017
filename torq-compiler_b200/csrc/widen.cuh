// Shared memory by address, and bytes widened for the tensor cores.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace tb200 {

// four int8 -> four bf16, exact: 0x4300 | the low seven bits is 128 + those bits, and 128 comes off again, or 256 where the byte is negative
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t low = w & 0x7f7f7f7fu, off = w & 0x80808080u;
  const uint32_t a0 = __byte_perm(low, 0x43434343u, 0x4140), a1 = __byte_perm(low, 0x43434343u, 0x4342);
  const uint32_t c0 = __byte_perm(off, 0x43434343u, 0x4140), c1 = __byte_perm(off, 0x43434343u, 0x4342);
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(a0), "r"(c0));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(a1), "r"(c1));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {  // zeros when not valid
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

}  // namespace tb200
