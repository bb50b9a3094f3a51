// Layer norm over the last axis, backward (rtseg_ln_dev.h has the mathematics and the rows' layout).
#include "rtseg_ln_dev.h"

namespace rtseg {
namespace ln {
namespace {

// One row (or 4 .. 64 rows a block, see the layout) a turn of a grid-stride loop.  Bound by HBM: 262144 x 64 of an
// fp32 stream with a bf16 branch in 45 us, 32768 x 320 of bf16 from a checkpoint in 20 us (the loads of a turn
// issued behind its own branches and without a turn of lead: 54 and 46 us).  The grid is what the device holds at
// once, so that no block waits for another to end, and so that the partial weight gradients are few: at 1024
// blocks, a third of them alone in a second round, the join took 6.3 us, now 3.5.
// Blocks of the backward a CU, as the registers of a lane's vectors allow (unaligned rows: one less).
constexpr int bwd_blocks_cu(int nv) { return nv >= 3 ? 2 : nv == 2 ? 3 : 4; }

template <typename TX, typename TO, int NV, bool BLOCK, bool CK, bool VEC>
__global__ void __launch_bounds__(kThreads, bwd_blocks_cu(NV) - (VEC ? 0 : 1)) ln_bwd_kernel(const LnBwdArgs a) {
  __shared__ float red[2][4];
  __shared__ float col[BLOCK ? 1 : 2 * kMaxNV * 64 * 8];
  int turn = 0;
  const int G = BLOCK ? kThreads : a.lanes, rpb = kThreads / G;
  const int lane = threadIdx.x & (G - 1), rl = threadIdx.x / G;
  const float inv_c = 1.f / static_cast<float>(a.C);
  const int64_t total = a.rows * a.C;

  float w[NV][8], aw[NV][8], ab[NV][8];
  uint32_t e[NV];
  const Span<float, VEC> ws(a.w, 0, a.C);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + lane) * 8;
    e[j] = static_cast<uint32_t>(rl * a.C + c);
    Raw8<float> wr = ws.load(c, a.C - c);
    ws.settle(wr, c, a.C - c);
    unraw8<float>(wr, w[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (a.w == nullptr) w[j][i] = 1.f;
      aw[j][i] = ab[j][i] = 0.f;
    }
  }
  Raw8<TO> yr[NV];
  Raw8<TX> xr[CK ? 1 : NV], dr[NV];
  uint2 codes[CK ? NV : 1];
  uint8_t scale[CK ? NV : 1];
  float mean = 0.f, rstd = 0.f;
  // channels of the row that this lane holds in its j-th vector; aligned rows leave those past the last one to the range
  auto count = [&](int j, int64_t r0) { return VEC || rl < a.rows - r0 ? a.C - (j * G + lane) * 8 : 0; };
  auto fetch = [&](int64_t r0) {
    const Span<TO, VEC> y(a.dy, r0 * a.C, total);
    const Span<TX, VEC> x(a.x, r0 * a.C, total);
    const int64_t left = a.rows - r0;
    const auto cs = range(a.codes + r0 * a.Cp, CK ? left * a.Cp : 0);
    const auto ss = range(a.scales + r0 * (a.Cp / kBlock), CK ? left * (a.Cp / kBlock) : 0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + lane) * 8;
      yr[j] = y.load(e[j], count(j, r0));
      if constexpr (CK) {
        const uint32_t o = static_cast<uint32_t>(rl * a.Cp + c);
        codes[j] = buf8(cs, c < a.Cp ? o : kOut);
        scale[j] = buf1(ss, c < a.Cp ? o / kBlock : kOut);
      } else {
        xr[j] = x.load(e[j], count(j, r0));
      }
    }
    mean = buf_f32(range(a.mean + r0, left * 4), rl * 4);
    rstd = buf_f32(range(a.rstd + r0, left * 4), rl * 4);
  };
  auto fetch_ds = [&](int64_t r0) {
    const Span<TX, VEC> d(a.ds, r0 * a.C, total);
#pragma unroll
    for (int j = 0; j < NV; ++j) dr[j] = d.load(e[j], count(j, r0));
  };
  // every thread of a block makes the same number of turns: the row sums cross lanes.  Where there is no
  // row everything reads as 0, rstd too, and adds nothing.
  const int64_t stride = static_cast<int64_t>(gridDim.x) * rpb;
  // The next turn's loads go out as soon as this one's values have left the registers, so that few waves keep
  // the memory busy; 4 vectors a lane and unaligned rows have no registers for it.
  constexpr bool AHEAD = VEC && NV < 4;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * rpb;
  if (AHEAD && r0 < a.rows) {
    fetch(r0);
    fetch_ds(r0);
  }
  for (; r0 < a.rows; r0 += stride) {
    if constexpr (!AHEAD) {
      fetch(r0);
      fetch_ds(r0);
    }
    const Span<TO, VEC> ys(a.dy, r0 * a.C, total);
    const Span<TX, VEC> xs(a.x, r0 * a.C, total), ds(a.ds, r0 * a.C, total), dx(a.dx, r0 * a.C, total);
    const Branch<TX, VEC> drs{a.dr, a.r_dtype, r0 * a.C, total};
    float g[NV][8], h[NV][8];
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = count(j, r0);
      float v[8];
      if constexpr (CK) {
        const float s = scale_of(scale[j]);
        decode4(codes[j].x, s, v);
        decode4(codes[j].y, s, v + 4);
        hold<TX, 8>(scale[j], v);
      } else {
        xs.settle(xr[j], e[j], n);
        unraw8<TX>(xr[j], v);
      }
      ys.settle(yr[j], e[j], n);
      unraw8<TO>(yr[j], g[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // past the row g is 0 and h a number (or the row's own NaN)
        h[j][i] = (v[i] - mean) * rstd;
        aw[j][i] += g[j][i] * h[j][i];
        ab[j][i] += g[j][i];
        g[j][i] *= w[j][i];
        c1 += g[j][i];
        c2 += g[j][i] * h[j][i];
      }
    }
    const float rs = rstd;
    if (AHEAD && r0 + stride < a.rows) fetch(r0 + stride);
    c1 = row_sum<BLOCK>(c1, G, red, turn) * inv_c;
    c2 = row_sum<BLOCK>(c2, G, red, turn) * inv_c;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = count(j, r0);
      float o[8], d[8];
      ds.settle(dr[j], e[j], n);
      unraw8<TX>(dr[j], d);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = rs * (g[j][i] - c1 - h[j][i] * c2) + d[i];
      if (a.dx != nullptr) dx.store(e[j], n, raw8<TX>(o));
      if (sizeof(TX) == 4 && a.dr != nullptr) drs.store(e[j], n, o);
    }
    if (AHEAD && r0 + stride < a.rows) fetch_ds(r0 + stride);
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
    for (int o = G; o < kWave; o <<= 1)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
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

// part [nb, 2, C] -> dw, db: 16 columns x 64 row lanes a block, four rows of a lane in flight
__global__ void __launch_bounds__(1024) ln_bwd_join_kernel(const float* __restrict__ part, int nb, int C, float* dw,
                                                           float* db) {
  __shared__ float sm[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cl;
  const float* col = part + (c < 2 * C ? c : 0);
  float s = 0.f;
  for (int r = rl; r < nb; r += 256) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = col[static_cast<int64_t>(min(r + 64 * i, nb - 1)) * 2 * C];
#pragma unroll
    for (int i = 0; i < 4; ++i) s += r + 64 * i < nb ? v[i] : 0.f;
  }
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

}  // namespace
}  // namespace ln

// at most the blocks that the device holds at once, each with as many turns as the others
int layer_norm_bwd_blocks(int64_t rows, int C) {
  using namespace ln;
  const LnPlan p = ln_plan(C);
  const int64_t rpb = kThreads / p.lanes, most = 256 * bwd_blocks_cu(p.nv);
  const int64_t all = rows < 1 ? 1 : (rows + rpb - 1) / rpb, each = (all + most - 1) / most;
  return static_cast<int>((all + each - 1) / each);
}

void launch_layer_norm_bwd(LnBwdArgs a, float* dw, float* db, hipStream_t st) {
  using namespace ln;
  const LnPlan p = ln_plan(a.C);
  a.lanes = p.lanes;
  a.blocks = layer_norm_bwd_blocks(a.rows, a.C);
  const bool vec = a.C % 8 == 0 && al16(a.x) && al16(a.dy) && al16(a.ds) && al16(a.dx) && al16(a.dr) && al16(a.w);
  by_types(a.x_dtype, a.y_dtype, [&](auto tx, auto to) {
    by_plan(p, [&](auto nv, auto block) {
      by_flag(vec, [&](auto v) {
        by_flag(a.codes != nullptr, [&](auto ck) {
          constexpr auto kernel = &ln_bwd_kernel<decltype(tx), decltype(to), decltype(nv)::value, decltype(block)::value,
                                                 decltype(ck)::value, decltype(v)::value>;
          kernel<<<a.blocks, kThreads, 0, st>>>(a);
        });
      });
    });
  });
  if (a.part != nullptr) ln_bwd_join_kernel<<<(2 * a.C + 15) / 16, 1024, 0, st>>>(a.part, a.blocks, a.C, dw, db);
}

}  // namespace rtseg
