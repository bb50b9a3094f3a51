// Layer norm over the last axis, forward (rtseg_ln_dev.h has the mathematics and the rows' layout).
#include "rtseg_ln_dev.h"

namespace rtseg {
namespace ln {
namespace {

// One row (or 4 .. 64 rows a block) and out: the many blocks' loads hide each other's wait, and weight and bias
// come from L2 while the row sums are formed.  Bound by HBM: 262144 x 64 of an fp32 stream with a bf16 branch in
// 34 us, 32768 x 320 of bf16 with its checkpoint in 20 us (with a branch around each load: 45 and 27 us).
template <typename TX, typename TO, int NV, bool BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) ln_fwd_kernel(const LnFwdArgs a) {
  __shared__ float red[2][4];
  int turn = 0;
  const int G = BLOCK ? kThreads : a.lanes, rpb = kThreads / G;
  const int lane = threadIdx.x & (G - 1), rl = threadIdx.x / G;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * rpb, left = a.rows - r0;  // rows past `left`: no row
  const bool live = rl < left;
  const int64_t first = r0 * a.C, total = a.rows * a.C;
  const Span<TX, VEC> x(a.x, first, total), s(a.s, first, total);
  const Span<TO, VEC> y(a.y, first, total);
  const Branch<TX, VEC> r{a.r, a.r_dtype, first, total};
  const Span<float, VEC> ws(a.w, 0, a.C), bs(a.b, 0, a.C);

  uint32_t e[NV];
  int n[NV];
  Raw8<TX> xr[NV], rr[NV];
  Raw8<float> wr[NV], br[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8;
    e[j] = static_cast<uint32_t>(rl * a.C + c);
    n[j] = live ? a.C - c : 0;
    xr[j] = x.load(e[j], n[j]);
  }
  if (a.r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) rr[j] = r.load(e[j], n[j]);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8;
    wr[j] = ws.load(c, a.C - c);
    br[j] = bs.load(c, a.C - c);
  }
  float v[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    x.settle(xr[j], e[j], n[j]);
    unraw8<TX>(xr[j], v[j]);
  }
  if (a.r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float t[8];
      r.values(rr[j], e[j], n[j], t);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] += t[i];
      // the stream is a tensor of its own type: the norm sees the sum as rounded to it
      const Raw8<TX> sr = raw8<TX>(v[j]);
      unraw8<TX>(sr, v[j]);
      if (a.s != nullptr) s.store(e[j], n[j], sr);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[j][i];  // channels past C were loaded as 0
  const float inv_c = 1.f / static_cast<float>(a.C);
  // The sum's roundings leave the mean off by up to 41 of its own; the differences from it, small and nearly exact where
  // that matters, give back what is missing: the mean of equal values is that value, and a row of a large mean keeps
  // its digits.  The variance is taken around the first mean and moved by the square of the second.
  const float first_mean = row_sum<BLOCK>(sum, G, red, turn) * inv_c;
  float sd = 0.f, sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = (VEC ? n[j] > 0 : i < n[j]) ? v[j][i] - first_mean : 0.f;
      sd += d;
      sq += d * d;
    }
  }
  const float rest = row_sum<BLOCK>(sd, G, red, turn) * inv_c;
  const float mean = first_mean + rest;
  // fused: the square, of no more than the other term, is not rounded to an infinity by itself
  const float var = fmaxf(__builtin_fmaf(-rest, rest, row_sum<BLOCK>(sq, G, red, turn) * inv_c), 0.f);
  const float rstd = 1.f / sqrtf(var + a.eps);

  if (live && lane == 0 && a.mean != nullptr) {
    a.mean[r0 + rl] = mean;
    a.rstd[r0 + rl] = rstd;
  }
  if (a.codes != nullptr) {  // every lane: the block maximum crosses lanes
    const auto codes = range(a.codes + r0 * a.Cp, left * a.Cp);
    uint8_t* scales = a.scales + r0 * (a.Cp / kBlock);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * 8;
      const uint32_t o = static_cast<uint32_t>(rl * a.Cp + c);
      uint32_t byte;
      const uint2 code = encode8(v[j], byte);
      put8(codes, c < a.Cp ? o : kOut, code);
      if (live && c < a.Cp && (lane & 3) == 0) scales[o / kBlock] = static_cast<uint8_t>(byte);
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8;
    float w[8], b[8], o[8];
    ws.settle(wr[j], c, a.C - c);
    bs.settle(br[j], c, a.C - c);
    unraw8<float>(wr[j], w);
    unraw8<float>(br[j], b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float h = (v[j][i] - mean) * rstd;
      o[i] = a.w != nullptr ? __builtin_fmaf(h, w[i], b[i]) : h + b[i];
    }
    y.store(e[j], n[j], raw8<TO>(o));
  }
}

}  // namespace
}  // namespace ln

int layer_norm_max_channels() { return ln::kThreads * ln::kMaxNV * 8; }

void launch_layer_norm_fwd(LnFwdArgs a, hipStream_t st) {
  using namespace ln;
  if (a.rows == 0) return;
  const LnPlan p = ln_plan(a.C);
  a.lanes = p.lanes;
  const bool vec = a.C % 8 == 0 && al16(a.x) && al16(a.r) && al16(a.s) && al16(a.y) && al16(a.w) && al16(a.b);
  const int64_t rpb = kThreads / a.lanes;
  if (a.rows > rpb * kMaxBlocks) {  // more than one launch holds
    const int64_t rows = a.rows, first = rpb * kMaxBlocks / 64 * 64, n = first * a.C;
    a.rows = first;
    launch_layer_norm_fwd(a, st);
    a.x = ahead(a.x, n * size_of(a.x_dtype));
    a.r = ahead(a.r, n * size_of(a.r_dtype));
    a.s = ahead(a.s, n * size_of(a.x_dtype));
    a.y = ahead(a.y, n * size_of(a.y_dtype));
    a.mean = ahead(a.mean, first * 4);
    a.rstd = ahead(a.rstd, first * 4);
    a.codes = ahead(a.codes, first * a.Cp);
    a.scales = ahead(a.scales, first * (a.Cp / kBlock));
    a.rows = rows - first;
    launch_layer_norm_fwd(a, st);
    return;
  }
  const unsigned grid = static_cast<unsigned>((a.rows + rpb - 1) / rpb);
  by_types(a.x_dtype, a.y_dtype, [&](auto tx, auto to) {
    by_plan(p, [&](auto nv, auto block) {
      by_flag(vec, [&](auto v) {
        constexpr auto kernel =
            &ln_fwd_kernel<decltype(tx), decltype(to), decltype(nv)::value, decltype(block)::value, decltype(v)::value>;
        kernel<<<grid, kThreads, 0, st>>>(a);
      });
    });
  });
}

}  // namespace rtseg
