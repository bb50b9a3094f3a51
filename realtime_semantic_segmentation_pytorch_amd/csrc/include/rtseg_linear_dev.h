// Device helpers of the checkpointing linear layer's kernels (linear_ckpt8_*.hip): activation, operand
// loads and conversions, matrix instructions, LDS layouts.
//
//   forward   y = act(x) w^T + b          codes = checkpoint of x (rtseg_ckpt8.h)
//   dgrad     dx = (dy w) * act'(z)       z = the checkpoint's values
//   wgrad     dw = dy^T act(z), db = sum_rows dy
//
// bf16 / fp16 operands feed v_mfma_f32_16x16x32, fp32 ones v_mfma_f32_16x16x4_f32; sums are fp32.
// Operands are of x's type, and two are rounded to it: act = gelu, computed in fp32 and rounded in front of the
// product, and fp32 weights beside a 16-bit x (cast by the caller, binding_ckpt8.cpp).  Both are what a separate
// activation layer and autocast hand to a linear layer; a second product for the rest of each would double the
// MFMA work.  Relative to the formula with exact operands, bf16 (fp16: an eighth), 256 to 64: y is off by 2.4e-3
// with fp32 weights and 2.9e-3 behind gelu as well, of which 1.7e-3 are the rounding of y itself; dw of fp32
// weights is off by 1.7e-3 behind gelu and by fp32 sums (7e-8) without it, since a checkpoint's values are exact.
#pragma once

#include "rtseg_ckpt8.h"
#include "rtseg_launch.h"
#include "rtseg_mfma_dev.h"
#include "rtseg_rows_dev.h"

namespace rtseg {
namespace lin {

using namespace ckpt8;
using namespace rows;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Phi(-a), the normal tail, for a >= 0: log2 Phi(-a) is smooth, and a polynomial of degree 7 (minimax over
// [0, 9], the error weighted by Phi and, up to a = 6.5, by itself; -inf beyond) gives Phi within 3e-7, and
// within 2^-11.8 of its own value where it is small.
__device__ __forceinline__ float normal_tail(float a) {
  float q = __builtin_fmaf(a, -7.709749070272665e-07f, 4.193515997030772e-05f);
  q = __builtin_fmaf(a, q, -0.0007947825361043215f);
  q = __builtin_fmaf(a, q, 0.008072120137512684f);
  q = __builtin_fmaf(a, q, -0.05329299345612526f);
  q = __builtin_fmaf(a, q, -0.4589170515537262f);
  q = __builtin_fmaf(a, q, -1.151143193244934f);
  return __builtin_amdgcn_exp2f(__builtin_fmaf(a, q, -0.9999992251396179f));
}
// gelu(x) = x Phi(x) = max(x, 0) - |x| Phi(-|x|), gelu'(x) = Phi(x) + x phi(x).  16-bit operands take the tail
// above (10 full-rate instructions and one quarter-rate; erff costs five times that, and the activation is
// what bounds the wide layers' forward); fp32 ones erff.  max and min work on the bits: the float forms
// spend an instruction each to quiet a NaN, which here comes through the tail.
template <typename T>
__device__ __forceinline__ float gelu(float x) {
  if constexpr (sizeof(T) == 4) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  const int bits = __float_as_int(x);
  // The factor of a positive x is cut off at 64, where the tail is 0: gelu(inf) = inf - 64 * 0.  As integers the
  // negative ones are below that and pass: gelu(-inf) = -inf * 0, a NaN as in every other form.
  const float a = __int_as_float(min(bits, 0x42800000));
  return __builtin_fmaf(-fabsf(a), normal_tail(fabsf(x)), __int_as_float(max(bits, 0)));
}
template <typename T>
__device__ __forceinline__ float gelu_slope(float x) {
  if constexpr (sizeof(T) == 4)
    return 0.5f * (1.f + erff(x * 0.70710678118654752f)) + x * 0.39894228040143268f * __expf(-0.5f * x * x);
  const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f), tail = normal_tail(fabsf(x));
  return __builtin_fmaf(x * 0.39894228040143268f, e, x >= 0.f ? 1.f - tail : tail);
}

template <typename T>
__device__ __forceinline__ void unpack16(uint4 q, float* v) {
  T t[kPer16<T>];
  __builtin_memcpy(t, &q, 16);
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i) v[i] = Io<T>::ld(t + i);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  T t[kPer16<T>];
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i) Io<T>::st(t + i, v[i]);
  uint4 q;
  __builtin_memcpy(&q, t, 16);
  return q;
}
template <>
__device__ __forceinline__ uint4 pack16<uint16_t>(const float* v) {
  return make_uint4(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]),
                    f32x2_to_bf16x2(v[6], v[7]));
}

// four values of a 16-bit T
template <typename T>
__device__ __forceinline__ uint2 pack8(const float* v) {
  if constexpr (__is_same(T, _Float16)) {
    const _Float16 t[4] = {static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]),
                           static_cast<_Float16>(v[3])};
    return __builtin_bit_cast(uint2, t);
  } else {
    return make_uint2(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]));
  }
}

// columns of a row of any alignment: W values from p on, of which n exist
template <typename T, int W>
__device__ __forceinline__ void put_any(T* p, int n, const float* v) {
  constexpr int C = W % kPer16<T> == 0 ? kPer16<T> : 4;  // a store's
  static_assert(W % C == 0, "whole stores");
#pragma unroll
  for (int e = 0; e < W; e += C) {
    if (e + C <= n) {
      if constexpr (C == kPer16<T>) {
        const uint4 q = pack16<T>(v + e);
        __builtin_memcpy(p + e, &q, 16);
      } else {
        const uint2 q = pack8<T>(v + e);
        __builtin_memcpy(p + e, &q, 8);
      }
    } else {
#pragma unroll
      for (int i = e; i < e + C; ++i)
        if (i < n) Io<T>::st(p + i, v[i]);
    }
  }
}

// largest of the chunk's absolute values as the bits of an fp32, NaN above infinity above every number
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint4 q, const float* v) {
  if constexpr (sizeof(T) == 4) {
    return max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
  } else {
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
    auto half = [](uint32_t w) { return __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu); };
    const u16x2_t m = __builtin_elementwise_max(__builtin_elementwise_max(half(q.x), half(q.y)),
                                                __builtin_elementwise_max(half(q.z), half(q.w)));
    const unsigned short top = m.x > m.y ? m.x : m.y;
    if constexpr (__is_same(T, _Float16)) return __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, top)));
    else return static_cast<uint32_t>(top) << 16;
  }
}

// one 16x16 tile step over 64 bytes of k a row: lane (g = lane / 16) holds k = g * kPer16 .. + kPer16 - 1
// of its row, for A and B alike
template <typename T>
__device__ __forceinline__ f32x4_t mma16(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (sizeof(T) == 4) {
    float x[4], y[4];
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &b, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(mdev::as_frag(a), mdev::as_frag(b), c, 0, 0, 0);
  }
}

__device__ __forceinline__ uint2 tr_read(const void* p) {
  auto q = (__attribute__((address_space(3))) mdev::i16x4_t*)((__attribute__((address_space(3))) void*)const_cast<void*>(p));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(q));
}

// LDS rows of an operand whose sum runs along them: 8 chunks of 16 bytes, chunk ^ (row & 7), which spreads
// the 16 rows of a fragment read over the banks
__device__ __forceinline__ int swz_a(int row) { return row & 7; }

template <class F>
void by_type(int dt, F f) {
  if (dt == kF32) f(float{});
  else if (dt == kBF16) f(uint16_t{});
  else f(_Float16{});
}
// Blocks that the whole device holds at once, for kernels whose blocks walk over several tiles.
template <class K>
int resident_blocks(K kernel, int threads) {
  int a_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&a_cu, kernel, threads, 0) != hipSuccess || a_cu < 1) a_cu = 2;
  return 256 * a_cu;
}
// A grid of at most that many blocks, a multiple of ntiles, each with the same number of row tiles: one
// block more than fit would cost as long again as all the others.
inline unsigned one_wave_grid(int resident, int mtiles, int ntiles) {
  const int most = resident / ntiles > 0 ? resident / ntiles : 1, each = (mtiles + most - 1) / most;
  return static_cast<unsigned>((mtiles + each - 1) / each * ntiles);
}

}  // namespace lin
}  // namespace rtseg
