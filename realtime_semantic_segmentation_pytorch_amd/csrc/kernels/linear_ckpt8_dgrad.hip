// The checkpointing linear layer's data gradient (definitions: rtseg_linear_dev.h):
//     dx[m, k] = act'(z[m, k]) * sum_n dy[m, n] w[n, k].
//
// A block of WN x WM x WK waves owns BM = 16 TM WM rows and 64 WN columns k.  A step takes 128 bytes of n of
// each row of dy and as many rows of w as they lie ([n][k]) through registers into LDS, in two buffers, one
// barrier a step; w is read transposed (ds_read_b64_tr_b16; fp32 reads four columns at once, one for each
// tile).  w is the MFMA row operand, its columns dealt so that a lane ends with 16 consecutive columns of
// one row: one 16-byte load of codes, wide stores.
//
// What bounds it: HBM (dy is read, the codes, dx written once) and, with gelu, the 20 VALU instructions of
// act' for every element.  Where n fits one step, w stays in LDS and the block walks down the rows; few
// tiles split n over 4 groups of waves, joined in LDS in order.  Measured: 131072 x 256 to 64 channels 19 us
// (84 MB, 4.4 TB/s), 131072 x 64 to 256 with gelu's slope 33 us (118 MB, 3.6 TB/s), 32768 x 320 to 1280 with the
// slope 69 us (390 TF, 147 MB).
#include "rtseg_linear_dev.h"

namespace rtseg {
namespace lin {
namespace {

struct DgradArgs {
  const void* dy;       // [M, R]: R = the layer's outputs, the sum's range
  const void* w;        // [R, N]: N = the layer's inputs
  void* out;            // dx [M, N]
  const int8_t* codes;  // [M, Cp]
  const uint8_t* scales;
  int64_t M;
  int N, R, Cp;
  int ntiles, mtiles;   // set by the launcher
  bool vo;              // 16-byte stores to out
};

// 8-byte units of a LDS row of w, XORed with row & 3 (a 16-lane group reads 4 rows) and row bit 3 (two groups)
__device__ __forceinline__ int swz_w(int row) { return (row & 3) | ((row >> 3) & 1) << 4; }

// ONE: R fits one step: w stays, the block takes every mstep-th row tile; else a block has one tile.
// VEC: rows of dy and w are 16-byte aligned.  WAVES: waves a SIMD that the registers are cut to.
template <typename T, int ACT, int WN, int WM, int WK, int TM, bool ONE, bool VEC, int WAVES>
__global__ void __launch_bounds__(WN* WM* WK * 64, WAVES) lin_dgrad_kernel(const DgradArgs p) {
  constexpr int NT = WN * WM * WK * 64, BM = WM * TM * 16, BN = WN * 64;
  constexpr int PER = kPer16<T>, BK = 8 * PER, STEP = WK * BK;
  constexpr int ES = static_cast<int>(sizeof(T));
  constexpr int CH = BM * 8 * WK, XA = (CH + NT - 1) / NT;   // chunks of dy, and a thread's
  constexpr int RC = BN / PER, CW = STEP * RC, WB = CW / NT;  // chunks of a row of w, of the step, a thread's
  constexpr int WROWS = NT / RC;                              // rows of w a turn
  constexpr int JOIN = (WK - 1) * BM * BN * 4 / 16;           // the groups' sums
  static_assert(WK == 1 || (NT / 8 % BM == 0 && !ONE), "a staging turn covers whole groups");
  __shared__ uint4 xs[2 * CH > JOIN ? 2 * CH : JOIN];         // [2][WK][BM][8]
  constexpr int WBUF = ONE || WK > 1 ? 1 : 2;                 // (two of four groups' would leave one block a CU)
  __shared__ uint4 ws[WBUF * CW];                             // [WBUF][STEP][RC]

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wid % WN, wm = wid / WN % WM, wk = wid / (WN * WM);
  const int g = lane >> 4, r = lane & 15;
  const int lb = mdev::xcd_logical(blockIdx.x, gridDim.x);
  const int nt = lb % p.ntiles, n0 = nt * BN;
  int mt = lb / p.ntiles;

  // dy: slot = tid / 8 + i * NT / 8 is row slot % BM of group slot / BM, chunk tid % 8 of it
  const int chunk = tid & 7, srow = tid >> 3;
  const int lrow = WK == 1 ? srow : srow % BM, lk = (WK == 1 ? 0 : srow / BM * BK) + chunk * PER;
  uint32_t aoff[XA];
#pragma unroll
  for (int i = 0; i < XA; ++i)
    aoff[i] = (static_cast<uint32_t>(lrow + (WK == 1 ? NT / 8 * i : 0)) * p.R + lk + (WK == 1 ? 0 : NT / 8 * i / BM * BK)) * ES;
  uint4 ra[XA];
  // unaligned rows: a step that the tensor has in whole is read as it lies, the others chunk by chunk
  constexpr int ROWS = WK == 1 ? XA * NT / 8 : BM;
  auto whole_a = [&](int m, int k0) { return static_cast<int64_t>(m) * BM + ROWS <= p.M && k0 + STEP <= p.R; };
  auto whole_w = [&](int k0) { return n0 + BN <= p.N && k0 + STEP <= p.R; };
  auto fetch_a = [&](int m, int k0) {
    const int64_t skip = static_cast<int64_t>(m) * BM * p.R;
    const __amdgpu_buffer_rsrc_t ar = range(static_cast<const T*>(p.dy) + skip, (p.M * p.R - skip) * ES);
    if (!VEC && whole_a(m, k0)) {
#pragma unroll
      for (int i = 0; i < XA; ++i) ra[i] = here16<T>(static_cast<const T*>(p.dy) + skip + k0, aoff[i] / ES);
      return;
    }
#pragma unroll
    for (int i = 0; i < XA; ++i) {
      const int have = p.R - k0 - lk - (WK == 1 ? 0 : NT / 8 * i / BM * BK);
      if constexpr (VEC) ra[i] = buf16(ar, have > 0 ? aoff[i] : kOut, k0 * ES);
      else ra[i] = any16<T>(static_cast<const T*>(p.dy), skip + aoff[i] / ES + k0, p.M * p.R);
    }
  };
  auto stage_a = [&](int m, int k0, int buf) {
    const bool ends = !VEC && !whole_a(m, k0);
#pragma unroll
    for (int i = 0; i < XA; ++i) {
      const int slot = srow + NT / 8 * i, row = slot % BM;
      if (XA * NT > CH && slot >= WK * BM) break;
      if (ends) {
        const int64_t mm = static_cast<int64_t>(m) * BM + row;
        const int k = k0 + slot / BM * BK + chunk * PER;
        ra[i] = settle16<T>(ra[i], static_cast<const T*>(p.dy), mm * p.R + k, mm < p.M ? p.R - k : 0);
      }
      xs[buf * CH + slot * 8 + (chunk ^ swz_a(row))] = ra[i];
    }
  };
  // w: rows tid / RC + i * WROWS of the step, chunk tid % RC
  const int wrow = tid / RC, wcol = tid % RC * PER;
  const int whave = p.N - n0 - wcol;
  const T* W = static_cast<const T*>(p.w) + n0;
  const int64_t wsize = static_cast<int64_t>(p.R) * p.N - n0;
  const uint32_t woff = whave > 0 ? (static_cast<uint32_t>(wrow) * p.N + wcol) * ES : kOut;
  uint4 rw[WB];
  auto fetch_w = [&](int k0) {
    const int64_t skip = static_cast<int64_t>(k0) * p.N;
    const __amdgpu_buffer_rsrc_t wr = range(W + skip, (wsize - skip) * ES);
    if (!VEC && whole_w(k0)) {
#pragma unroll
      for (int i = 0; i < WB; ++i)
        rw[i] = here16<T>(W + skip, static_cast<uint32_t>(wrow + WROWS * i) * p.N + wcol);
      return;
    }
#pragma unroll
    for (int i = 0; i < WB; ++i) {
      const uint32_t turn = static_cast<uint32_t>(WROWS * i) * p.N;
      if constexpr (VEC) rw[i] = buf16(wr, whave > 0 ? woff + turn * ES : kOut);
      else rw[i] = any16<T>(static_cast<const T*>(p.w), n0 + skip + static_cast<int64_t>(wrow) * p.N + wcol + turn,
                            static_cast<int64_t>(p.R) * p.N);
    }
  };
  auto stage_w = [&](int k0, int buf) {
    const bool ends = !VEC && !whole_w(k0);
#pragma unroll
    for (int i = 0; i < WB; ++i) {
      const int row = wrow + WROWS * i;
      uint4 q = rw[i];
      if (ends)
        q = settle16<T>(q, static_cast<const T*>(p.w), static_cast<int64_t>(k0 + row) * p.N + n0 + wcol, k0 + row < p.R ? whave : 0);
      if constexpr (ES == 2) {
        const int x = swz_w(row);  // bit 0 of the unit: the two halves change places
        if (x & 1) q = make_uint4(q.z, q.w, q.x, q.y);
        ws[buf * CW + row * RC + (tid % RC ^ (x >> 1 & (RC - 1)))] = q;
      } else {
        ws[buf * CW + row * RC + tid % RC] = q;
      }
    }
  };

  // fragment addresses: row r of w's tile t is column 16 (r / 4) + 4 t + r % 4 of the wave's 64, for fp32 4 r + t
  int xat[2], wat[4];
#pragma unroll
  for (int s = 0; s < 2; ++s) xat[s] = (wk * BM + wm * TM * 16 + r) * 8 + ((s * 4 + g) ^ swz_a(r));
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (ES == 2) {  // 8-byte units
      const int row = g * 8 + (r >> 2);
      wat[t] = (wk * BK + row) * (BN / 4) + ((wn * 16 + (r & 3) * 4 + t) ^ (swz_w(row) & (BN / 4 - 1)));
    } else {
      wat[t] = (wk * BK + 4 * g) * BN + wn * 64 + 4 * r;
    }
  }
  const int nc = n0 + wn * 64 + 16 * g;  // this lane's 16 columns

  f32x4_t acc[TM][4];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  auto multiply = [&](int buf, int wbuf) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint4 wf[4], xf[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) xf[t] = xs[buf * CH + xat[s] + t * 128];
      if constexpr (ES == 2) {
        // k = 8 g + 0..7: two reads of 4 rows; lane 4 q + c of the group supplies row q, columns 16 c + 4 t ..
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint2* u = reinterpret_cast<const uint2*>(ws + wbuf * CW) + wat[t] + s * 32 * (BN / 4);
          const uint2 lo = tr_read(u), hi = tr_read(u + 4 * (BN / 4));
          wf[t] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      } else {
        // k = 4 g + i of this half: four columns a read, one for each tile
        float4 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          h[i] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(ws + wbuf * CW) + wat[0] + (s * 16 + i) * BN);
        wf[0] = __builtin_bit_cast(uint4, make_float4(h[0].x, h[1].x, h[2].x, h[3].x));
        wf[1] = __builtin_bit_cast(uint4, make_float4(h[0].y, h[1].y, h[2].y, h[3].y));
        wf[2] = __builtin_bit_cast(uint4, make_float4(h[0].z, h[1].z, h[2].z, h[3].z));
        wf[3] = __builtin_bit_cast(uint4, make_float4(h[0].w, h[1].w, h[2].w, h[3].w));
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mma16<T>(wf[j], xf[i], acc[i][j]);
    }
  };
  auto finish = [&](int m) {  // lane: row `row` of every tile i, columns nc .. nc + 15
    const int64_t m0 = static_cast<int64_t>(m) * BM;
    T* O = static_cast<T*>(p.out) + m0 * p.N;
    const __amdgpu_buffer_rsrc_t orr = range(O, (p.M - m0) * p.N * ES);
    uint4 cw[TM];
    uint8_t cb[TM];
    if constexpr (ACT == kCkptGelu) {
      const __amdgpu_buffer_rsrc_t cr = range(p.codes + m0 * p.Cp, (p.M - m0) * p.Cp);
      const __amdgpu_buffer_rsrc_t er = range(p.scales + m0 * (p.Cp / kBlock), (p.M - m0) * (p.Cp / kBlock));
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint32_t o = ((wm * TM + i) * 16 + r) * p.Cp + nc;  // nc is a multiple of 16, Cp of 32
        cw[i] = buf16(cr, nc < p.N ? o : kOut);
        cb[i] = buf1(er, nc < p.N ? o / kBlock : kOut);
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const uint32_t row = (wm * TM + i) * 16 + r;
      float v[16];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[ES == 4 ? 4 * e + j : 4 * j + e] = acc[i][j][e];
      if constexpr (ACT == kCkptGelu) {
        const float sc = scale_of(cb[i]);
        const uint32_t w4[4] = {cw[i].x, cw[i].y, cw[i].z, cw[i].w};
        float z[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) decode4(w4[j], sc, z + 4 * j);
        hold<T, 16>(cb[i], z);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= gelu_slope<T>(z[e]);
      }
      if (p.vo) {
#pragma unroll
        for (int e = 0; e < 16; e += PER) put16(orr, nc + e < p.N ? (row * p.N + nc + e) * ES : kOut, pack16<T>(v + e));
      } else if (m0 + row < p.M) {
        put_any<T, 16>(O + static_cast<int64_t>(row) * p.N + nc, p.N - nc, v);
      }
    }
  };

  fetch_w(0);
  fetch_a(mt, 0);
  stage_w(0, 0);
  stage_a(mt, 0, 0);
  int buf = 0;
  if constexpr (ONE) {
    const int mstep = gridDim.x / p.ntiles;  // the grid is a multiple of ntiles: a block keeps its column
    if (mt + mstep < p.mtiles) fetch_a(mt + mstep, 0);
    for (; mt < p.mtiles; mt += mstep) {
      __syncthreads();
      if (mt + mstep < p.mtiles) {
        stage_a(mt + mstep, 0, buf ^ 1);
        if (mt + 2 * mstep < p.mtiles) fetch_a(mt + 2 * mstep, 0);
      }
      clear();
      multiply(buf, 0);
      finish(mt);
      buf ^= 1;
    }
  } else {
    if (STEP < p.R) {
      fetch_w(STEP);
      fetch_a(mt, STEP);
    }
    clear();
    __syncthreads();
    for (int k0 = 0; k0 < p.R; k0 += STEP) {
      if (k0 + STEP < p.R) {  // the next step goes to the other buffers, the one after it is on its way
        if constexpr (WBUF == 2) stage_w(k0 + STEP, buf ^ 1);
        stage_a(mt, k0 + STEP, buf ^ 1);
        if (k0 + 2 * STEP < p.R) {
          if constexpr (WBUF == 2) fetch_w(k0 + 2 * STEP);
          fetch_a(mt, k0 + 2 * STEP);
        }
      }
      multiply(buf, WBUF == 2 ? buf : 0);
      __syncthreads();
      if constexpr (WBUF == 1) {
        if (k0 + STEP < p.R) {
          stage_w(k0 + STEP, 0);
          if (k0 + 2 * STEP < p.R) fetch_w(k0 + 2 * STEP);
          __syncthreads();
        }
      }
      buf ^= 1;
    }
    if constexpr (WK > 1) {
      float4* join = reinterpret_cast<float4*>(xs);
      constexpr int PER_WAVE = TM * 4, GROUP = WM * WN * PER_WAVE;
      const int place = (wm * WN + wn) * PER_WAVE;
      if (wk > 0) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            join[((wk - 1) * GROUP + place + i * 4 + j) * 64 + lane] =
                make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      }
      __syncthreads();
      if (wk > 0) return;
#pragma unroll
      for (int q = 0; q < WK - 1; ++q)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 v = join[(q * GROUP + place + i * 4 + j) * 64 + lane];
            acc[i][j][0] += v.x;
            acc[i][j][1] += v.y;
            acc[i][j][2] += v.z;
            acc[i][j][3] += v.w;
          }
    }
    finish(mt);
  }
}

template <typename T, int ACT, int WN, int WM, int WK, int TM, bool VEC, int WAVES>
void launch_cfg(DgradArgs p, hipStream_t st) {
  constexpr int BM = WM * TM * 16, BN = WN * 64;
  p.ntiles = (p.N + BN - 1) / BN;
  p.mtiles = static_cast<int>((p.M + BM - 1) / BM);
  if constexpr (WK == 1 && VEC) {
    if (p.R <= 8 * kPer16<T>) {
      constexpr int W1 = ACT == kCkptGelu && TM == 4 && WAVES > 2 ? WAVES - 1 : WAVES;  // more registers
      const auto kernel = lin_dgrad_kernel<T, ACT, WN, WM, WK, TM, true, VEC, W1>;
      static const int resident = resident_blocks(kernel, WN * WM * WK * 64);
      kernel<<<one_wave_grid(resident, p.mtiles, p.ntiles), WN * WM * WK * 64, 0, st>>>(p);
      return;
    }
  }
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(p.mtiles) * p.ntiles);
  lin_dgrad_kernel<T, ACT, WN, WM, WK, TM, false, VEC, WAVES><<<grid, WN * WM * WK * 64, 0, st>>>(p);
}

// Tiles.  A problem of fewer than 256 tiles of 64 x 256 leaves CUs idle: 64 x 128 where those are 256 (4096 x 512
// from 512 with gelu: 11.2 us against 15.8, one wave of four would work off the slopes), else 32 x 64 with the sum
// split four ways.  Of the larger ones narrow layers (N <= 64, 128) take their width and more rows, others 256
// columns x 64 rows.
template <typename T, int ACT>
void launch_dgrad(const DgradArgs& p, bool vec, hipStream_t st) {
  constexpr int F = sizeof(T) == 4 ? 1 : 0;  // fp32 holds more: fewer waves
  const int64_t tiles = (p.M + 63) / 64 * ((p.N + 255) / 256);
  const bool mid = (p.M + 63) / 64 * ((p.N + 127) / 128) >= 256;
  if (!vec) {
    if (tiles < 256 && !mid) return launch_cfg<T, ACT, 1, 1, 4, 2, false, 2>(p, st);
    return launch_cfg<T, ACT, 2, 2, 1, 2, false, 2>(p, st);
  }
  if (tiles < 256 && !mid) return launch_cfg<T, ACT, 1, 1, 4, 2, true, 3 - F>(p, st);
  if (p.N <= 64) return launch_cfg<T, ACT, 1, 4, 1, 2, true, 4 - F>(p, st);
  if (p.N <= 128 || tiles < 256) return launch_cfg<T, ACT, 2, 2, 1, 2, true, 3>(p, st);
  launch_cfg<T, ACT, 4, 1, 1, 4, true, 3 - F>(p, st);
}

}  // namespace
}  // namespace lin

void launch_lin_dgrad(const LinDgradArgs& a, hipStream_t st) {
  using namespace lin;
  if (a.M == 0) return;
  const int64_t most = kMaxBlocks / ((a.K + 63) / 64) * 16;  // rows of the smallest tiles that one launch holds
  if (a.M > most) {
    const int64_t cp = padded(a.K);
    LinDgradArgs b = a;
    b.M = most;
    launch_lin_dgrad(b, st);
    b.dy = ahead(a.dy, most * a.N * size_of(a.dtype));
    b.dx = ahead(a.dx, most * a.K * size_of(a.dtype));
    b.codes = ahead(a.codes, most * cp);
    b.scales = ahead(a.scales, most * (cp / kBlock));
    b.M = a.M - most;
    launch_lin_dgrad(b, st);
    return;
  }
  DgradArgs p{};
  p.dy = a.dy; p.w = a.w; p.out = a.dx; p.codes = a.codes; p.scales = a.scales;
  p.M = a.M; p.N = a.K; p.R = a.N; p.Cp = static_cast<int>(padded(a.K));
  const int per = 16 / size_of(a.dtype);
  p.vo = a.K % per == 0 && al16(a.dx);
  const bool vec = a.N % per == 0 && a.K % per == 0 && al16(a.dy) && al16(a.w);
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    if (a.act == kCkptGelu) launch_dgrad<T, kCkptGelu>(p, vec, st);
    else launch_dgrad<T, kCkptNone>(p, vec, st);
  });
}

}  // namespace rtseg
