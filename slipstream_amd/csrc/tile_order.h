// Device helpers shared by the kernels that write their order out: loops unrolled at compile time, waits for
// DMAs, LDS addresses as numbers.
#pragma once
#include <type_traits>
#include <utility>

#include "w8a8_common.h"

namespace ss {
namespace {

template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// Until at most N of the wave's DMAs (and other vector memory instructions) are on their way
template <int N>
__device__ __forceinline__ void wait_dma() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

typedef __attribute__((address_space(3))) const u32x4* LdsWords;
__device__ __forceinline__ uint32_t lds_address(char* p) { return (uint32_t)(uintptr_t)(LdsBytes)p; }
__device__ __forceinline__ u32x4 lds_word(uint32_t at) { return *(LdsWords)(uintptr_t)at; }
__device__ __forceinline__ float lds_float(uint32_t at) {
  return *(__attribute__((address_space(3))) const float*)(uintptr_t)at;
}

// As dma_b128, four bytes a lane
__device__ __forceinline__ void dma_b32(i32x4 rs, uint32_t lds, int voff, int soff) {
  asm volatile("s_nop 1\n\tbuffer_load_dword %0, %1, %2 offen lds"
               :
               : "v"(voff), "s"(rs), "s"(soff), "{m0}"(lds)
               : "memory");
}

}  // namespace
}  // namespace ss
