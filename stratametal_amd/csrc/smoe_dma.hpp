// stratametal_amd/csrc/smoe_dma.hpp - buffer loads that write LDS directly, and the wait for them (gfx950).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace smoe {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

// Raw buffer resource over [base, base + bytes) (no swizzle, no stride; out-of-range lanes read nothing).
__device__ __forceinline__ i32x4 buffer_rsrc(const void* base, uint32_t bytes) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    return i32x4{(int)(uint32_t)b, (int)(uint32_t)(b >> 32), (int)bytes, 0x00020000};
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const lds_u8*)p; }
constexpr uint32_t kOob = 0x80000000u;  // an offset beyond any such buffer: zeros are written, no memory is read
// M0 is written one instruction before the load that reads it (one wait state for LDS DMA).
__device__ __forceinline__ void dma16(uint32_t lds, uint32_t voff, i32x4 rsrc, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(voff),
                 "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void vmcnt() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace smoe
