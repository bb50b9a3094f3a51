// Layer norm over the last axis: what the forward and the backward kernel (layer_norm_fwd.hip,
// layer_norm_bwd.hip) share -- the rows' layout over lanes, the branch beside the stream, the row sums.
//
//   s = x + r (rounded to the stream's type)      mean, var over the C channels of a row
//   h = (s - mean) * rstd, rstd = (var + eps)^-1/2         y = h * w + b
//   g = dy * w      dx = rstd * (g - mean(g) - h * mean(g * h)) + ds       dr = dx
//   dw = sum_rows dy * h        db = sum_rows dy
//
// Statistics, row sums and weight gradients are fp32 whatever the tensors' types; the variance and what the
// mean's sum left out are a second pass over (s - mean) in registers, so a large mean costs no digits (0.3 us
// of a row's latency, nothing measurable of a large tensor's time).
//
// Both kernels are bound by HBM: every tensor is read or written once.  A row is held in registers by
// G lanes (4 .. 64 of a wave, or all 256 of a block) of NV vectors of 8 channels each, which is what
// lets narrow rows (C = 32: 4 lanes) fill a wave with 16 rows and wide ones (C <= 8192) stay on chip.
// The weight gradients: each lane adds up its own channels over the rows of a grid-stride loop, the
// block joins its lanes in LDS and writes one partial row, and a second kernel sums those rows -- no
// atomics, the same bits on every run.
#pragma once

#include <type_traits>

#include "rtseg_ckpt8.h"
#include "rtseg_launch.h"
#include "rtseg_rows_dev.h"

namespace rtseg {
namespace ln {

using namespace ckpt8;
using namespace rows;

constexpr int kThreads = 256;
constexpr int kMaxNV = 4;

// rows of a tensor beside the stream: of the stream's type TX, or, where that is fp32, of any type `dt`
template <typename TX, bool VEC>
struct Branch {
  const void* t;
  int dt;
  int64_t first, total;
  __device__ __forceinline__ Raw8<TX> load(uint32_t e, int n) const {
    if constexpr (sizeof(TX) == 2) return Span<TX, VEC>(t, first, total).load(e, n);
    if (dt == kF32) return Span<TX, VEC>(t, first, total).load(e, n);
    Raw8<TX> r;
    r.q[0] = Span<uint16_t, VEC>(t, first, total).load(e, n).q[0];
    r.q[sizeof(TX) / 2 - 1] = make_uint4(0u, 0u, 0u, 0u);
    return r;
  }
  __device__ __forceinline__ void values(Raw8<TX> r, uint32_t e, int n, float* v) const {
    if (sizeof(TX) == 2 || dt == kF32) {
      Span<TX, VEC>(t, first, total).settle(r, e, n);
      unraw8<TX>(r, v);
      return;
    }
    Raw8<uint16_t> h;
    h.q[0] = r.q[0];
    Span<uint16_t, VEC>(t, first, total).settle(h, e, n);
    if (dt == kBF16) unraw8<uint16_t>(h, v);
    else unraw8<_Float16>(__builtin_bit_cast(Raw8<_Float16>, h), v);
  }
  __device__ __forceinline__ void store(uint32_t e, int n, const float* v) const {  // 16 bits beside an fp32 stream
    if (dt == kBF16) Span<uint16_t, VEC>(t, first, total).store(e, n, raw8<uint16_t>(v));
    else Span<_Float16, VEC>(t, first, total).store(e, n, raw8<_Float16>(v));
  }
};

// sum over the G lanes of a row; G == kThreads joins the block's waves through LDS (red: 2 x 4 floats,
// used alternately so that one barrier a call is enough)
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, int G, float (*red)[4], int& turn) {
  if constexpr (!BLOCK) {
    for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
  } else {
    v = wave_sum(v);
    float* r = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    return (r[0] + r[1]) + (r[2] + r[3]);
  }
}

// Lanes a row and vectors a lane: of the pairs that hold the row, the one with the fewest idle slots
// (C = 160, 20 vectors of 8: 8 lanes x 3 rather than 32 x 1), the wider row on a tie.
struct LnPlan { int lanes, nv; };
inline LnPlan ln_plan(int C) {
  const int need = static_cast<int>(padded(C) / 8);
  LnPlan best{kThreads, kMaxNV};
  int waste = 1 << 30;
  for (int g : {64, 32, 16, 8, 4}) {
    const int nv = (need + g - 1) / g;
    if (nv <= kMaxNV && g * nv - need < waste) {
      waste = g * nv - need;
      best = {g, nv};
    }
  }
  if (waste == 1 << 30) best.nv = (need + kThreads - 1) / kThreads;
  return best;
}

// f(lanes' vectors, a block a row?): a block a row only past 64 lanes x 4 vectors
template <class F>
void by_plan(const LnPlan& p, F f) {
  using std::integral_constant;
  const auto wave = std::false_type{};
  if (p.lanes == kThreads) {
    if (p.nv <= 2) f(integral_constant<int, 2>{}, std::true_type{});
    else f(integral_constant<int, 4>{}, std::true_type{});
  } else if (p.nv == 1) f(integral_constant<int, 1>{}, wave);
  else if (p.nv == 2) f(integral_constant<int, 2>{}, wave);
  else if (p.nv == 3) f(integral_constant<int, 3>{}, wave);
  else f(integral_constant<int, 4>{}, wave);
}
template <class F>
void by_flag(bool v, F f) {
  if (v) f(std::true_type{});
  else f(std::false_type{});
}

// the output is the stream's type, fp32 behind a 16-bit stream, or 16 bits behind an fp32 one
template <class F>
void by_types(int tx, int to, F f) {
  if (tx == kF32) {
    if (to == kF32) f(float{}, float{});
    else if (to == kBF16) f(float{}, uint16_t{});
    else f(float{}, _Float16{});
  } else if (tx == kBF16) {
    if (to == kF32) f(uint16_t{}, float{});
    else f(uint16_t{}, uint16_t{});
  } else {
    if (to == kF32) f(_Float16{}, float{});
    else f(_Float16{}, _Float16{});
  }
}

}  // namespace ln
}  // namespace rtseg
