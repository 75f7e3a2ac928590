// lds_copy.hpp -- copies from memory into LDS that pass no registers, and the buffer descriptors they read through.
#pragma once
#include "common.hpp"

typedef int i4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// Raw buffer of `bytes` bytes at a wave-uniform base; reads past it give zero.  The lane's and the scalar offset
// count together (measured: a scalar offset at the end or past it leaves no lane in range).
__device__ __forceinline__ i4v buffer_at(const void* base, uint32_t bytes) {
  const uint64_t b = (uint64_t)(uintptr_t)base;
  return i4v{__builtin_amdgcn_readfirstlane((int)(uint32_t)b), __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xffff),
             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// Global -> LDS copies as inline asm, so that the compiler adds no waits for them at LDS reads: the
// kernel's own vmcnt waits and barriers order them.  Lane l's bytes land at m0 + 16 l (4 l).
// A vector-memory read of a scalar register needs five wait states after the vector unit has written it, as
// buffer_at does and the restoring of a spilled descriptor; the compiler does not look for that in here.
// The write of m0 and s_nop 3 are five whatever stands in front.  Over s_nop 0 they cost 0 to 3%, in turn: gated
// 4,616 x 2,048 x 768 20.7 to 21.0 us, 24,288 x 113 x 3,936 in f32 57.9 to 59.4, 16,391 x 8,192 x 4,096 in bf16 nothing.
__device__ __forceinline__ void lds_copy16(i4v rsrc, uint32_t voff, uint32_t soff, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(m0)
               : "memory", "m0");
}
__device__ __forceinline__ void lds_copy4(i4v rsrc, uint32_t voff, uint32_t soff, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff),
               "s"(m0)
               : "memory", "m0");
}
constexpr uint32_t kOutside = 0x7fffffffu;  // past every descriptor's range
