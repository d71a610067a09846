// Elements of 32 or 16 bits in 16-byte pieces, for the operators that take fp32, bf16 and fp16 (ORCA_F32 / BF16 / F16).
#pragma once
#include "common.h"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// gfx950 loads and stores 16 bytes at any even address in one instruction (amdhsa runs with unaligned access on): rows of odd widths
// and tensors inside a flat buffer need no path of their own
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <class T> constexpr int elems16 = 16 / (int)sizeof(T);

__device__ __forceinline__ u32x4 load16(const void* p) { return *reinterpret_cast<const u32x4_any*>(p); }
__device__ __forceinline__ void store16(void* p, u32x4 v) { *reinterpret_cast<u32x4_any*>(p) = v; }
// the same past the caches (non-temporal).  The choice has to be a template's: the compiler merges the two sides of a branch on a
// run-time flag into one plain access.
__device__ __forceinline__ u32x4 load16_past(const void* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p)); }
__device__ __forceinline__ void store16_past(void* p, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p)); }

template <class T> __device__ __forceinline__ void unpack16(u32x4 r, float (&f)[elems16<T>]) {
  T e[elems16<T>];
  __builtin_memcpy(e, &r, 16);
#pragma unroll
  for (int j = 0; j < elems16<T>; ++j) f[j] = (float)e[j];
}
template <class T> __device__ __forceinline__ u32x4 pack16(const float* f) {      // rounds to nearest even
  T e[elems16<T>];
#pragma unroll
  for (int j = 0; j < elems16<T>; ++j) e[j] = (T)f[j];
  u32x4 r;
  __builtin_memcpy(&r, e, 16);
  return r;
}
