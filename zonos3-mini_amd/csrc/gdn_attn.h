// What the attention kernels share: tiles of K and V rows in LDS, loads straight into them, MFMA fragments.
#pragma once

#include <atomic>

#include "gdn_common.h"

namespace zgdn {

typedef __bf16 abf16x8 __attribute__((ext_vector_type(8)));
typedef float af32x4 __attribute__((ext_vector_type(4)));
typedef float af32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 abf16x2 __attribute__((ext_vector_type(2)));
typedef short ashort4 __attribute__((ext_vector_type(4)));

// Rows of ROWB bytes (128, 256 or 512) in LDS, 16-byte chunk c of row r at place c ^ mask(r), so that what is read at a time
// spreads over the banks (256 bytes). Row fragments: 16 rows at one chunk; all masks give 16 neighbouring rows different
// places. Values, for products of M x M tiles: bf16, transposing reads, by 32 lanes 8 rows by 2 chunks (M = 16) or 4 rows by 4
// chunks (M = 32); fp32, single floats, 4 rows 4 apart by 4 chunks (M = 16) or 2 rows 4 apart by 8 chunks (M = 32).
template <int ROWB, typename T, int M>
__device__ __forceinline__ constexpr int swizzle(int r) {
  constexpr int n = ROWB / 16;
  if (sizeof(T) == 4) return M == 16 ? r & 15 : (r & 3) | (r >> 3 & 1) << 2 | (r >> 2 & 1) << 3;
  if (M == 16) return n == 16 ? (r & 7) << 1 | (r >> 3 & 1) : (r >> 1) & 7;
  return n == 16 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3);
}
template <int ROWB, typename T, int M>
__device__ __forceinline__ int row_chunk(int r, int c) {
  return r * ROWB + ((c ^ swizzle<ROWB, T, M>(r)) << 4);
}

// Four rows by 16 columns of 16-bit entries, transposed: in each group of 16 lanes, lane s gives the address of 4 entries of
// row s / 4, columns 4 (s % 4) .., and gets the 4 rows' entries of column s.
__device__ __forceinline__ uint2 lds_transposed(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ashort4*)p));
}

// Reads by an address within LDS.
typedef uint32_t au32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) const au32x4* LdsPieces;
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)p; }  // (the low half)
__device__ __forceinline__ uint4 lds_piece(uint32_t at) {
  return __builtin_bit_cast(uint4, *(LdsPieces)(uintptr_t)at);
}
__device__ __forceinline__ uint2 lds_transposed(uint32_t at) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ashort4*)(uintptr_t)at));
}

// 16 bytes a lane straight into LDS, lane i at lds + 16 i (lds: an address within LDS, wave-uniform), from the lane's own
// address, or from a uniform one and the lane's offset. As for load_lds (gdn_common.h): in assembly, so that the kernel's own
// waits count it; a wait state behind M0's move. `nt`: the rows of a cache are not read again before others of their size.
__device__ __forceinline__ void load_lds_from(const void* p, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(p), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void load_lds_from(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}
static __device__ __attribute__((aligned(16))) const uint32_t zeros16[4] = {0, 0, 0, 0};  // where loads of no row go
// At most N of the wave's own loads still on their way.
template <int N>
__device__ __forceinline__ void wait_own_loads() {
  static_assert(N < 64, "counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Largest value of lanes l, l ^ 16, l ^ 32, l ^ 48, and their sum.
__device__ __forceinline__ float max_over_groups(float x) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // (one instruction; below 2^-126: 0)

// Lets `kernel` have `bytes` of dynamic LDS on the current device, once a device; false where the device refuses.
constexpr int MAX_DEVICES = 64;
inline bool lds_ready(const void* kernel, int bytes, std::atomic<signed char>* ready) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return false;
  const signed char was = ready[dev].load(std::memory_order_acquire);
  if (was != 0) return was > 0;
  const bool ok = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
  if (!ok) (void)hipGetLastError();
  ready[dev].store(ok ? 1 : -1, std::memory_order_release);
  return ok;
}

constexpr float LOG2E = 1.44269504088896340736f;

}  // namespace zgdn
