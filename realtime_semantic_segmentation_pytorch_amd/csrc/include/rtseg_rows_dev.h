// Loads and stores of rows in device memory without a branch a load: as bounded buffers where rows are
// 16-byte aligned, from clamped addresses where they are not.
#pragma once

#include <type_traits>

#include "rtseg_common.h"

namespace rtseg {
namespace rows {

// 16 bytes of operand: 8 (bf16 / fp16) or 4 (fp32) consecutive k
template <typename T> constexpr int kPer16 = 16 / static_cast<int>(sizeof(T));

// A range of a tensor as a buffer: loads past `bytes` read 0 and stores there are dropped, so the rows
// that a tile does not have cost no branch.  kOut as an offset, and the 128 bytes behind it, are past every range.
constexpr uint32_t kOut = 0xffffff40u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t range(const void* p, int64_t bytes) {
  const uint32_t n = bytes < 0 ? 0u : bytes > 0xffffff00ll ? 0xffffff00u : static_cast<uint32_t>(bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(n), 0x00020000);
}
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
// `off` alone decides whether an access is in range; `base` (uniform, added to it) only moves along a row,
// between columns that the caller has checked, so that a range has to end at the last row and no sooner
__device__ __forceinline__ uint4 buf16(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t base = 0) {
  return __builtin_bit_cast(
      uint4, static_cast<u32x4_t>(__builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(off), static_cast<int>(base), 0)));
}
__device__ __forceinline__ uint8_t buf1(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t base = 0) {
  return static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(r, static_cast<int>(off), static_cast<int>(base), 0));
}
__device__ __forceinline__ float buf_f32(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, static_cast<int>(off), 0, 0));
}
__device__ __forceinline__ uint2 buf8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(uint2, static_cast<u32x2_t>(__builtin_amdgcn_raw_buffer_load_b64(r, static_cast<int>(off), 0, 0)));
}
__device__ __forceinline__ void put16(__amdgpu_buffer_rsrc_t r, uint32_t off, uint4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), r, static_cast<int>(off), 0, 0);
}
__device__ __forceinline__ void put8(__amdgpu_buffer_rsrc_t r, uint32_t off, uint2 v) {
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, v), r, static_cast<int>(off), 0, 0);
}
// A launch holds fewer than 2^32 threads: 2^24 - 1 blocks of 256.
constexpr int64_t kMaxBlocks = (1 << 24) - 1;
template <typename P>
P* ahead(P* p, int64_t bytes) {  // null stays null
  using Byte = std::conditional_t<std::is_const_v<P>, const char, char>;
  return p == nullptr ? nullptr : reinterpret_cast<P*>(reinterpret_cast<Byte*>(p) + bytes);
}
inline int size_of(int dt) { return dt == kF32 ? 4 : 2; }
inline bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Rows of any alignment.  The load is issued without a branch, from inside the tensor: p[i] where 16 bytes
// fit behind it, else from its last 16 bytes (the tensor has at least that many where a row does; rows that
// are shorter are left to settle16).  A value for which fewer than 16 bytes exist is settled when it is
// used, after the wait: 0 where nothing exists, a row's last elements one by one.
template <typename T>
__device__ __forceinline__ uint4 any16(const T* p, int64_t i, int64_t size) {
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  const int64_t last = size - kPer16<T>;
  if (last >= 0) __builtin_memcpy(&q, p + (i < last ? i : last), 16);
  return q;
}
// 16 bytes of any alignment that are all there
template <typename T>
__device__ __forceinline__ uint4 here16(const T* p, uint32_t i) {
  uint4 q;
  __builtin_memcpy(&q, p + i, 16);
  return q;
}
template <typename T>
__device__ __forceinline__ uint4 settle16(uint4 q, const T* p, int64_t i, int n) {
  if (n <= 0) return make_uint4(0u, 0u, 0u, 0u);
  if (n < kPer16<T>) {
    T t[kPer16<T>];
#pragma unroll
    for (int e = 0; e < kPer16<T>; ++e) {
      t[e] = T(0);
      if (e < n) t[e] = p[i + e];
    }
    __builtin_memcpy(&q, t, 16);
  }
  return q;
}

// ---- eight consecutive channels of a row, as raw bits and as floats ----------------------------
template <typename T> struct Raw8 { uint4 q[sizeof(T) / 2]; };

template <typename T>
__device__ __forceinline__ void unraw8(const Raw8<T>& r, float* v) {
  T t[8];
  __builtin_memcpy(t, &r, sizeof(t));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Io<T>::ld(t + i);
}
template <typename T>
__device__ __forceinline__ Raw8<T> raw8(const float* v) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16)) {
    r.q[0] = make_uint4(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]),
                        f32x2_to_bf16x2(v[6], v[7]));
  } else {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) Io<T>::st(t + i, v[i]);
    __builtin_memcpy(&r, t, sizeof(t));
  }
  return r;
}

// `size` elements from p on, read and written 8 at a time; a null or empty range (size <= 0) reads as 0.
// e: the first element, n: how many from it on are wanted (<= 0: none, read as 0 and not written).
// VEC: p and every e are 16-byte aligned and n is a multiple of 8; what lies past `size` reads as 0.
// Otherwise e + n <= size where n > 0, and a value is settled in front of its use, after the loads' wait.
template <typename T, bool VEC>
struct Span {
  T* p;
  int64_t size;
  __device__ __forceinline__ Span(const void* t, int64_t first, int64_t total)
      : p(static_cast<T*>(const_cast<void*>(t)) + (t != nullptr ? first : 0)), size(t != nullptr ? total - first : 0) {}
  __device__ __forceinline__ Raw8<T> load(uint32_t e, int n) const {
    Raw8<T> r;
    if constexpr (VEC) {
      const auto b = range(p, size * static_cast<int64_t>(sizeof(T)));
      const uint32_t off = n > 0 ? e * static_cast<uint32_t>(sizeof(T)) : kOut;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.q[i] = buf16(b, off + 16 * i);
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        r.q[i] = any16<T>(p, static_cast<int64_t>(n > 0 ? e : 0) + i * kPer16<T>, size);
    }
    return r;
  }
  __device__ __forceinline__ void settle(Raw8<T>& r, uint32_t e, int n) const {
    if constexpr (!VEC) {
      if (size <= 0) n = 0;  // an empty range is not read here either
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
        r.q[i] = settle16<T>(r.q[i], p, static_cast<int64_t>(e) + i * kPer16<T>, n - i * kPer16<T>);
    }
  }
  __device__ __forceinline__ void store(uint32_t e, int n, const Raw8<T>& r) const {
    if constexpr (VEC) {
      const auto b = range(p, size * static_cast<int64_t>(sizeof(T)));
      const uint32_t off = n > 0 ? e * static_cast<uint32_t>(sizeof(T)) : kOut;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) put16(b, off + 16 * i, r.q[i]);
    } else if (n >= 8) {
      __builtin_memcpy(p + e, &r, sizeof(r));
    } else {
      T t[8];
      __builtin_memcpy(t, &r, sizeof(t));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[e + i] = t[i];
    }
  }
};

}  // namespace rows
}  // namespace rtseg
