// mm.hpp -- what the product kernels of operands laid out for the matrix unit share:
// unrolling, tiles for XCDs, loads from memory into LDS.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

namespace acfun {

typedef __attribute__((address_space(3))) void lds_void;

// f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>)
template <class F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F f) { each_of(f, std::make_integer_sequence<int, N>{}); }

// XCD x (workgroup id mod 8) owns a contiguous run of the `total` tiles: the number
// of this workgroup's, or `total` if it has none.
__device__ __forceinline__ unsigned xcd_tile(unsigned total) {
    const unsigned x = blockIdx.x & 7;
    auto first = [&](unsigned y) { return y * (total >> 3) + (y * (total & 7) >> 3); };
    const unsigned l = first(x) + (blockIdx.x >> 3);
    return l < first(x + 1) ? l : total;
}

// ReLU where lo is 0, nothing where it is -infinity; NaN stays NaN.
__device__ __forceinline__ float at_least(float v, float lo) { return __builtin_elementwise_maximum(v, lo); }

// s_waitcnt vmcnt(n), n < 64
constexpr int vm_count(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }

// 64 times 16 (or 4) bytes from q into LDS; nothing is read unless `live`.
__device__ __forceinline__ void lds_dma16(const void* q, bool live, char* lds, unsigned voff, unsigned soff) {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)q, (short)0, live ? 0x7fffffff : 0, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void lds_dma4(const void* q, bool live, char* lds, unsigned voff, unsigned soff) {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)q, (short)0, live ? 0x7fffffff : 0, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds, 4, voff, soff, 0, 0);
}

}  // namespace acfun
