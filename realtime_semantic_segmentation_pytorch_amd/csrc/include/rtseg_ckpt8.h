// 8-bit activation checkpoints: the format, and its device-side coding.
//
// A [rows, C] activation is held as int8 codes [rows, Cp] (Cp = C rounded up to 32; the codes behind
// C are 0) and one scale byte per block of 32 consecutive channels of a row, [rows, Cp / 32]:
//     e = the smallest integer >= -126 with max |x| <= 127 * 2^e,   q = rne(x / 2^e),   byte = e + 127.
// The scale is a power of two, so dividing by it is exact (one rounding in all, at most half of 2^e)
// and q * 2^e fits the type of the tensor exactly: a matrix product reads the checkpoint through bf16
// MFMA with no further rounding.  The one value that does not fit is 64 * 2^e of the type's largest
// scale, which what lies in the last half step below infinity rounds up to: it decodes to the type's
// largest finite value, which is nearer still to what was packed (`hold`).  A block that holds an infinity or a NaN gets the scale
// byte 255 and codes 0, which decode to 0 * inf = NaN: an overflowed activation still shows in the
// gradients that are computed from it (the loss scaler of fp16 training looks for exactly that).
#pragma once

#include "rtseg_common.h"

namespace rtseg {
namespace ckpt8 {

constexpr int kBlock = 32;  // channels per scale
__host__ __device__ inline int64_t padded(int64_t c) { return (c + kBlock - 1) / kBlock * kBlock; }

// largest |v| as bits: the integer order of the bits puts NaN above infinity above every number
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// block maximum (abs_bits) -> scale byte.  max = m * 2^(E-127) with m in [1, 2): e = E - 127 - 6 holds
// it iff m <= 127 / 64, whose fraction bits are 0x7e0000.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;
  const int e = static_cast<int>(amax >> 23) - 6 + ((amax & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return static_cast<uint32_t>(e < 1 ? 1 : e);
}
// 2^-(byte - 127); byte is in [1, 249] or 255 (whose codes are 0 whatever this is)
__device__ __forceinline__ float inv_scale(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }  // 255: inf

// four values -> four code bytes: adding 1.5 * 2^23 rounds to an integer (to nearest, ties to even)
// whose two's complement is the low byte of the sum
__device__ __forceinline__ uint32_t code4(const float* v, float inv, bool bad) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__builtin_fmaf(v[i], inv, 12582912.f));
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return bad ? 0u : (lo | hi);
}
// four code bytes -> values
__device__ __forceinline__ void decode4(uint32_t w, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * scale;
}

// The last scale byte of T's blocks, and the largest finite value: max = f * 2^(byte - 127) with f in (63.5, 64).
template <typename T>
constexpr uint32_t kTopByte = __is_same(T, _Float16) ? 137u : 249u;
template <typename T>
constexpr uint32_t kTopBits = __is_same(T, _Float16) ? 0x477fe000u : sizeof(T) == 2 ? 0x7f7f0000u : 0x7f7fffffu;
// N values that were decoded with this scale byte, held in T's range.  A branch and not a clamp of each value: next to
// no block takes it, and its values are numbers (a NaN would be clamped to one).
template <typename T, int N>
__device__ __forceinline__ void hold(uint32_t byte, float* v) {
  if (byte == kTopByte<T>) {
    const float top = __uint_as_float(kTopBits<T>);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fminf(fmaxf(v[i], -top), top);
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {  // over 4 consecutive lanes
  const uint32_t a = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
  return max(a, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(a), 0x4E, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t oct_max(uint32_t v) {  // over 8 consecutive lanes
  const uint32_t a = quad_max(v);
  return max(a, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(a), 0x141, 0xF, 0xF, true)));
}

// 8 consecutive channels held by each of 4 consecutive lanes = one block: this lane's 8 code bytes
// and the block's scale byte (the same in all 4 lanes, every one of which has to execute this)
__device__ __forceinline__ uint2 encode8(const float* v, uint32_t& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
  byte = scale_byte(quad_max(m));
  const float inv = inv_scale(byte);
  return make_uint2(code4(v, inv, byte == 255u), code4(v + 4, inv, byte == 255u));
}

}  // namespace ckpt8
}  // namespace rtseg
