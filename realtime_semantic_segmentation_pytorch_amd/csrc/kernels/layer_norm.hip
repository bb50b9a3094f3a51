// Layer norm over the last axis, forward and backward, with an optional residual sum in front and an
// optional 8-bit checkpoint (rtseg_ckpt8.h) of the normalised tensor in place of the tensor itself.
//
//   s = x + r (rounded to the stream's type)      mean, var over the C channels of a row
//   h = (s - mean) * rstd, rstd = (var + eps)^-1/2         y = h * w + b
//   g = dy * w      dx = rstd * (g - mean(g) - h * mean(g * h)) + ds       dr = dx
//   dw = sum_rows dy * h        db = sum_rows dy
//
// Statistics, row sums and weight gradients are fp32 whatever the tensors' types; the variance is the
// second pass over (s - mean) in registers, so a large mean costs no digits.
//
// Both kernels are bound by HBM: every tensor is read or written once.  A row is held in registers by
// G lanes (4 .. 64 of a wave, or all 256 of a block) of NV vectors of 8 channels each, which is what
// lets narrow rows (C = 32: 4 lanes) fill a wave with 16 rows and wide ones (C <= 8192) stay on chip.
// The weight gradients: each lane adds up its own channels over the rows of a grid-stride loop, the
// block joins its lanes in LDS and writes one partial row, and a second kernel sums those rows -- no
// atomics, the same bits on every run.
#include "rtseg_ckpt8.h"
#include "rtseg_launch.h"

namespace rtseg {
namespace {

using namespace ckpt8;

constexpr int kThreads = 256;
constexpr int kMaxNV = 4;

// a tensor of one of two types: the stream's T, or (a branch under autocast) a 16-bit type
struct AnyRaw { uint4 q[2]; };
__device__ __forceinline__ AnyRaw load_any(const void* p, int dt, int64_t off, int n, bool vec) {
  AnyRaw a;
  if (dt == kF32) {
    const Raw8<float> r = load8<float>(static_cast<const float*>(p) + off, n, vec);
    a.q[0] = r.q[0];
    a.q[1] = r.q[1];
  } else {
    a.q[0] = load8<uint16_t>(static_cast<const uint16_t*>(p) + off, n, vec).q[0];
    a.q[1] = make_uint4(0u, 0u, 0u, 0u);
  }
  return a;
}
__device__ __forceinline__ void unraw_any(const AnyRaw& a, int dt, float* v) {
  if (dt == kF32) {
    Raw8<float> r;
    r.q[0] = a.q[0];
    r.q[1] = a.q[1];
    unraw8<float>(r, v);
  } else if (dt == kBF16) {
    Raw8<uint16_t> r;
    r.q[0] = a.q[0];
    unraw8<uint16_t>(r, v);
  } else {
    Raw8<_Float16> r;
    r.q[0] = a.q[0];
    unraw8<_Float16>(r, v);
  }
}
__device__ __forceinline__ void store_any(void* p, int dt, int64_t off, const float* v, int n, bool vec) {
  if (dt == kF32) store8<float>(static_cast<float*>(p) + off, raw8<float>(v), n, vec);
  else if (dt == kBF16) store8<uint16_t>(static_cast<uint16_t*>(p) + off, raw8<uint16_t>(v), n, vec);
  else store8<_Float16>(static_cast<_Float16*>(p) + off, raw8<_Float16>(v), n, vec);
}

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

template <typename TX, typename TO, int NV, bool BLOCK>
__global__ void __launch_bounds__(kThreads) ln_fwd_kernel(const LnFwdArgs a) {
  __shared__ float red[2][4];
  int turn = 0;
  const int G = BLOCK ? kThreads : a.lanes;
  const int lane = threadIdx.x & (G - 1);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  const bool live = row0 < a.rows;
  const int64_t row = live ? row0 : 0;
  const int64_t base = row * a.C;
  const TX* x = static_cast<const TX*>(a.x);

  Raw8<TX> xr[NV];
  AnyRaw rr[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8;
    xr[j] = load8<TX>(x + base + c, a.C - c, a.vec);
  }
  if (a.r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * 8;
      rr[j] = load_any(a.r, a.r_dtype, base + c, a.C - c, a.vec);
    }
  }
  float v[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) unraw8<TX>(xr[j], v[j]);
  if (a.r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * 8;
      float t[8];
      unraw_any(rr[j], a.r_dtype, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] += t[i];
      // the stream is a tensor of its own type: the norm sees the sum as rounded to it
      const Raw8<TX> sr = raw8<TX>(v[j]);
      unraw8<TX>(sr, v[j]);
      if (live && a.s != nullptr) store8<TX>(static_cast<TX*>(a.s) + base + c, sr, a.C - c, a.vec);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[j][i];  // channels past C were loaded as 0
  const float inv_c = 1.f / static_cast<float>(a.C);
  const float mean = row_sum<BLOCK>(sum, G, red, turn) / static_cast<float>(a.C);  // exact for a constant row
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int n = a.C - (j * G + lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = v[j][i] - mean;
      if (i < n) sq += d * d;
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<BLOCK>(sq, G, red, turn) * inv_c + a.eps);

  if (live && lane == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8, n = a.C - c;
    if (a.codes != nullptr) {  // every lane: the block maximum crosses lanes
      uint32_t byte;
      const uint2 code = encode8(v[j], byte);
      if (live && c < a.Cp) {
        const int64_t o = row * a.Cp + c;
        *reinterpret_cast<uint2*>(a.codes + o) = code;
        if ((lane & 3) == 0) a.scales[o / kBlock] = static_cast<uint8_t>(byte);
      }
    }
    float w[8], b[8], o[8];
    const Raw8<float> wr = load8<float>(a.w + c, a.w != nullptr ? n : 0, a.wvec);
    const Raw8<float> br = load8<float>(a.b + c, a.b != nullptr ? n : 0, a.wvec);
    unraw8<float>(wr, w);
    unraw8<float>(br, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float h = (v[j][i] - mean) * rstd;
      o[i] = a.w != nullptr ? __builtin_fmaf(h, w[i], b[i]) : h + b[i];
    }
    if (live) store8<TO>(static_cast<TO*>(a.y) + base + c, raw8<TO>(o), n, a.vec);
  }
}

template <typename TX, typename TO, int NV, bool BLOCK, bool CK>
__global__ void __launch_bounds__(kThreads) ln_bwd_kernel(const LnBwdArgs a) {
  __shared__ float red[2][4];
  __shared__ float col[BLOCK ? 1 : 2 * kMaxNV * 64 * 8];
  int turn = 0;
  const int G = BLOCK ? kThreads : a.lanes;
  const int lane = threadIdx.x & (G - 1);
  const int rpb = kThreads / G;
  const float inv_c = 1.f / static_cast<float>(a.C);

  float w[NV][8], aw[NV][8], ab[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8;
    const Raw8<float> wr = load8<float>(a.w + c, a.w != nullptr ? a.C - c : 0, a.wvec);
    unraw8<float>(wr, w[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (a.w == nullptr) w[j][i] = 1.f;
      aw[j][i] = ab[j][i] = 0.f;
    }
  }
  // every thread of a block makes the same number of turns: the row sums cross lanes
  const int64_t stride = static_cast<int64_t>(gridDim.x) * rpb;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * rpb; r0 < a.rows; r0 += stride) {
    const int64_t want = r0 + threadIdx.x / G;
    const bool live = want < a.rows;
    const int64_t row = live ? want : 0;
    const int64_t base = row * a.C;
    Raw8<TO> yr[NV];
    Raw8<TX> xr[NV], dr[NV];
    uint2 cr[NV];
    uint8_t sb[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * 8, n = live ? a.C - c : 0;
      yr[j] = load8<TO>(static_cast<const TO*>(a.dy) + base + c, n, a.vec);
      if constexpr (CK) {
        const bool in = live && c < a.Cp;
        const int64_t o = row * a.Cp + c;
        cr[j] = in ? *reinterpret_cast<const uint2*>(a.codes + o) : make_uint2(0u, 0u);
        sb[j] = in ? a.scales[o / kBlock] : 0;
      } else {
        xr[j] = load8<TX>(static_cast<const TX*>(a.x) + base + c, n, a.vec);
      }
      if (a.ds != nullptr) dr[j] = load8<TX>(static_cast<const TX*>(a.ds) + base + c, n, a.vec);
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[NV][8], h[NV][8];
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = live ? a.C - (j * G + lane) * 8 : 0;
      float t[8];
      if constexpr (CK) {
        const float s = scale_of(sb[j]);
        decode4(cr[j].x, s, t);
        decode4(cr[j].y, s, t + 4);
      } else {
        unraw8<TX>(xr[j], t);
      }
      unraw8<TO>(yr[j], g[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[j][i] = i < n ? (t[i] - mean) * rstd : 0.f;
        aw[j][i] += g[j][i] * h[j][i];
        ab[j][i] += g[j][i];
        g[j][i] *= w[j][i];
        c1 += g[j][i];
        c2 += g[j][i] * h[j][i];
      }
    }
    c1 = row_sum<BLOCK>(c1, G, red, turn) * inv_c;
    c2 = row_sum<BLOCK>(c2, G, red, turn) * inv_c;
    if (live) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + lane) * 8, n = a.C - c;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = rstd * (g[j][i] - c1 - h[j][i] * c2);
        if (a.ds != nullptr) {
          float t[8];
          unraw8<TX>(dr[j], t);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] += t[i];
        }
        if (a.dx != nullptr) store8<TX>(static_cast<TX*>(a.dx) + base + c, raw8<TX>(o), n, a.vec);
        if (a.dr != nullptr) store_any(a.dr, a.r_dtype, base + c, o, n, a.vec);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.C;
  if constexpr (BLOCK) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < a.C) {
          part[c + i] = aw[j][i];
          part[a.C + c + i] = ab[j][i];
        }
    }
  } else {
    // the wave's rows first, then its 4 waves one after the other
    const int width = NV * G * 8;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        for (int o = G; o < kWave; o <<= 1) {
          aw[j][i] += __shfl_xor(aw[j][i], o, kWave);
          ab[j][i] += __shfl_xor(ab[j][i], o, kWave);
        }
    for (int wv = 0; wv < kThreads / kWave; ++wv) {
      if (threadIdx.x / kWave == wv && (threadIdx.x & 63) < G) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = (j * G + lane) * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            col[c + i] = wv == 0 ? aw[j][i] : col[c + i] + aw[j][i];
            col[width + c + i] = wv == 0 ? ab[j][i] : col[width + c + i] + ab[j][i];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      part[c] = col[c];
      part[a.C + c] = col[width + c];
    }
  }
}

// part [nb, 2, C] -> dw, db: 16 columns x 64 row lanes a block
__global__ void __launch_bounds__(1024) ln_bwd_join_kernel(const float* __restrict__ part, int nb, int C, float* dw,
                                                           float* db) {
  __shared__ float sm[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cl;
  float s = 0.f;
  if (c < 2 * C)
    for (int r = rl; r < nb; r += 64) s += part[static_cast<int64_t>(r) * 2 * C + c];
  sm[rl][cl] = s;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (rl < o) sm[rl][cl] += sm[rl + o][cl];
    __syncthreads();
  }
  if (rl == 0 && c < 2 * C) {
    if (c < C) dw[c] = sm[0][cl];
    else db[c - C] = sm[0][cl];
  }
}

// Lanes a row and vectors a lane: of the pairs that hold the row, the one with the fewest idle slots
// (C = 160, 20 vectors of 8: 8 lanes x 3 rather than 32 x 1), the wider row on a tie.
struct LnPlan { int lanes, nv; };
LnPlan ln_plan(int C) {
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

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename TX, typename TO, int NV>
void fwd_nv(const LnFwdArgs& a, hipStream_t st) {
  const int64_t rpb = kThreads / a.lanes;
  const unsigned grid = static_cast<unsigned>((a.rows + rpb - 1) / rpb);
  if constexpr (NV > 1) {  // a block a row only past 64 lanes x 4 vectors
    if (a.lanes == kThreads) {
      ln_fwd_kernel<TX, TO, NV, true><<<grid, kThreads, 0, st>>>(a);
      return;
    }
  }
  ln_fwd_kernel<TX, TO, NV, false><<<grid, kThreads, 0, st>>>(a);
}
template <typename TX, typename TO>
void fwd_t(const LnFwdArgs& a, int nv, hipStream_t st) {
  switch (nv) {
    case 1: fwd_nv<TX, TO, 1>(a, st); break;
    case 2: fwd_nv<TX, TO, 2>(a, st); break;
    case 3: fwd_nv<TX, TO, 3>(a, st); break;
    default: fwd_nv<TX, TO, 4>(a, st); break;
  }
}
template <typename TX, typename TO, int NV>
void bwd_nv(const LnBwdArgs& a, hipStream_t st) {
  const bool ck = a.codes != nullptr;
  if constexpr (NV > 1) {
    if (a.lanes == kThreads) {
      if (ck) ln_bwd_kernel<TX, TO, NV, true, true><<<a.blocks, kThreads, 0, st>>>(a);
      else ln_bwd_kernel<TX, TO, NV, true, false><<<a.blocks, kThreads, 0, st>>>(a);
      return;
    }
  }
  if (ck) ln_bwd_kernel<TX, TO, NV, false, true><<<a.blocks, kThreads, 0, st>>>(a);
  else ln_bwd_kernel<TX, TO, NV, false, false><<<a.blocks, kThreads, 0, st>>>(a);
}
template <typename TX, typename TO>
void bwd_t(const LnBwdArgs& a, int nv, hipStream_t st) {
  switch (nv) {
    case 1: bwd_nv<TX, TO, 1>(a, st); break;
    case 2: bwd_nv<TX, TO, 2>(a, st); break;
    case 3: bwd_nv<TX, TO, 3>(a, st); break;
    default: bwd_nv<TX, TO, 4>(a, st); break;
  }
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

}  // namespace

int layer_norm_max_channels() { return kThreads * kMaxNV * 8; }

int layer_norm_bwd_blocks(int64_t rows, int C) {
  const int64_t rpb = kThreads / ln_plan(C).lanes;
  const int64_t want = (rows + rpb - 1) / rpb;
  return static_cast<int>(want < 1024 ? (want < 1 ? 1 : want) : 1024);
}

void launch_layer_norm_fwd(LnFwdArgs a, hipStream_t st) {
  if (a.rows == 0) return;
  const LnPlan p = ln_plan(a.C);
  a.lanes = p.lanes;
  a.vec = a.C % 8 == 0 && al16(a.x) && al16(a.r) && al16(a.s) && al16(a.y);
  a.wvec = a.C % 8 == 0 && al16(a.w) && al16(a.b);
  by_types(a.x_dtype, a.y_dtype, [&](auto tx, auto to) { fwd_t<decltype(tx), decltype(to)>(a, p.nv, st); });
}

void launch_layer_norm_bwd(LnBwdArgs a, float* dw, float* db, hipStream_t st) {
  const LnPlan p = ln_plan(a.C);
  a.lanes = p.lanes;
  a.blocks = layer_norm_bwd_blocks(a.rows, a.C);
  a.vec = a.C % 8 == 0 && al16(a.x) && al16(a.dy) && al16(a.ds) && al16(a.dx) && al16(a.dr);
  a.wvec = a.C % 8 == 0 && al16(a.w);
  by_types(a.x_dtype, a.y_dtype, [&](auto tx, auto to) { bwd_t<decltype(tx), decltype(to)>(a, p.nv, st); });
  if (a.part != nullptr) ln_bwd_join_kernel<<<(2 * a.C + 15) / 16, 1024, 0, st>>>(a.part, a.blocks, a.C, dw, db);
}

}  // namespace rtseg
