// The checkpointing linear layer's forward (definitions: rtseg_linear_dev.h): y[m, n] = sum_k act(x[m, k]) w[n, k] + b[n],
// and the 8-bit checkpoint of x.
//
// A block of WN x WM x WK waves owns BM = 16 TM WM rows and 16 TN WN columns.  It stages 128 bytes of k of
// each row of x through registers into LDS -- registers because that is where the checkpoint is taken (the
// blocks of the first column write it) and the activation applied -- in two buffers, so that a step costs
// one barrier.  w goes from L2 straight into the fragments: with WM = 1 no two waves share it.  w is the
// MFMA row operand and its rows are dealt so that a lane ends with 4 TN (16) consecutive columns of one
// output row: wide stores.  Blocks have 4 or 8 waves: one of 5 loads one SIMD twice, and a second one does
// not fit beside it.
//
// What bounds it: HBM for the encoders' narrow layers (x or y is read or written once), VALU where the
// activation is evaluated -- so with gelu a tile is as wide as the layer, up to 512 columns, and each
// element is evaluated once -- and latency for small ones: few tiles split k over 4 groups of waves, whose
// sums are joined in LDS in order.  Weights whose k fits one step stay in registers while the block walks
// down the rows.  Measured: 131072 x 64 to 256 columns 27 us (93 MB, 3.4 TB/s), 131072 x 256 to
// 64 with gelu 35 us (118 MB, 3.4 TB/s), 32768 x 1280 to 320 with gelu 86 us (310 TF; waits for w, not arithmetic:
// in a run of 91 us, 88 without gelu, 92 without the products, 65 without the loads of w), 2048 x 512 to 2048
// 14.4 us (300 TF; 256 tiles, one block a CU and one wave a SIMD: nothing covers a step's wait), 32 x 256 to 256 4 us.
#include "rtseg_linear_dev.h"

namespace rtseg {
namespace lin {
namespace {

struct FwdArgs {
  const void* a;        // x [M, K]
  const void* b;        // w [N, K]
  const void* bias;     // [N] of w's type or fp32, or nullptr
  void* out;            // [M, N]
  int8_t* codes;        // [M, Cp], or nullptr
  uint8_t* scales;
  int64_t M;
  int N, K, Cp;
  int ntiles, mtiles;   // set by the launcher
  bool vo;              // 16-byte stores to out
  bool bias_f32;
};

// ONE: k fits one step: b stays in registers and the block walks down the rows, every mstep-th tile; else a
// block has one tile.  VEC: rows of a and b are 16-byte aligned.  WAVES: waves a SIMD that the registers are
// cut to.
template <typename T, int ACT, int WN, int WM, int WK, int TM, int TN, bool ONE, bool VEC, int WAVES>
__global__ void __launch_bounds__(WN* WM* WK * 64, WAVES) lin_fwd_kernel(const FwdArgs p) {
  constexpr int NT = WN * WM * WK * 64, BM = WM * TM * 16, WC = TN * 16, BN = WN * WC;
  constexpr int PER = kPer16<T>, BK = 8 * PER, STEP = WK * BK;
  constexpr int ES = static_cast<int>(sizeof(T));
  constexpr int CH = BM * 8 * WK, XA = (CH + NT - 1) / NT;  // chunks of a, and a thread's
  constexpr int JOIN = (WK - 1) * BM * BN * 4 / 16;          // the groups' sums
  static_assert(WK == 1 || (NT / 8 % BM == 0 && !ONE), "a staging turn covers whole groups");
  __shared__ uint4 xs[2 * CH > JOIN ? 2 * CH : JOIN];        // [2][WK][BM][8]
  __shared__ float bs[BN];

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wid % WN, wm = wid / WN % WM, wk = wid / (WN * WM);
  const int g = lane >> 4, r = lane & 15;
  // the column tiles of one row tile follow each other on one XCD: they share its L2's copy of a
  const int lb = mdev::xcd_logical(blockIdx.x, gridDim.x);
  const int nt = lb % p.ntiles, n0 = nt * BN;
  const bool pack = p.codes != nullptr && nt == 0;
  int mt = lb / p.ntiles;

  // a, staged: slot = tid / 8 + i * NT / 8 is row slot % BM of k group slot / BM, chunk tid % 8 of it
  const int chunk = tid & 7, srow = tid >> 3;
  const int lrow = WK == 1 ? srow : srow % BM, lk = (WK == 1 ? 0 : srow / BM * BK) + chunk * PER;
  uint32_t aoff[XA];
#pragma unroll
  for (int i = 0; i < XA; ++i)
    aoff[i] = (static_cast<uint32_t>(lrow + (WK == 1 ? NT / 8 * i : 0)) * p.K + lk + (WK == 1 ? 0 : NT / 8 * i / BM * BK)) * ES;
  uint4 ra[XA];
  // unaligned rows: a step that the tensor has in whole is read as it lies, the others chunk by chunk
  constexpr int ROWS = WK == 1 ? XA * NT / 8 : BM;
  auto whole_a = [&](int m, int k0) { return static_cast<int64_t>(m) * BM + ROWS <= p.M && k0 + STEP <= p.K; };
  auto whole_b = [&](int k0) { return n0 + BN <= p.N && k0 + STEP <= p.K; };
  auto fetch_a = [&](int m, int k0) {  // row tile m
    const int64_t skip = static_cast<int64_t>(m) * BM * p.K;
    const T* A = static_cast<const T*>(p.a) + skip;
    const __amdgpu_buffer_rsrc_t ar = range(A, (p.M * p.K - skip) * ES);
    if (!VEC && whole_a(m, k0)) {
#pragma unroll
      for (int i = 0; i < XA; ++i) ra[i] = here16<T>(A + k0, aoff[i] / ES);
      return;
    }
#pragma unroll
    for (int i = 0; i < XA; ++i) {
      const int have = p.K - k0 - lk - (WK == 1 ? 0 : NT / 8 * i / BM * BK);
      if constexpr (VEC) {
        ra[i] = buf16(ar, have > 0 ? aoff[i] : kOut, k0 * ES);
      } else {
        ra[i] = any16<T>(static_cast<const T*>(p.a), skip + aoff[i] / ES + k0, p.M * p.K);
      }
    }
  };
  // its codes: the lane's part of the address, and the scale byte's (one lane a block)
  uint32_t coff[XA], eoff[XA];
#pragma unroll
  for (int i = 0; i < XA; ++i) {
    const uint32_t row = lrow + (WK == 1 ? NT / 8 * i : 0);
    coff[i] = row * p.Cp + lk;
    eoff[i] = lk % kBlock == 0 ? row * (p.Cp / kBlock) + lk / kBlock : kOut;
  }
  auto stage_a = [&](int m, int k0, int buf) {
    const int64_t m0 = static_cast<int64_t>(m) * BM;
    const __amdgpu_buffer_rsrc_t cr = range(p.codes + m0 * p.Cp, (p.M - m0) * p.Cp);
    const __amdgpu_buffer_rsrc_t er = range(p.scales + m0 * (p.Cp / kBlock), (p.M - m0) * (p.Cp / kBlock));
    const bool ends = !VEC && !whole_a(m, k0);
#pragma unroll
    for (int i = 0; i < XA; ++i) {
      const int slot = srow + NT / 8 * i, row = slot % BM;
      if (XA * NT > CH && slot >= WK * BM) break;
      const int k = k0 + slot / BM * BK + chunk * PER;
      if (ends)
        ra[i] = settle16<T>(ra[i], static_cast<const T*>(p.a), (m0 + row) * p.K + k, m0 + row < p.M ? p.K - k : 0);
      {
        float v[PER];
        if (ACT == kCkptGelu || pack) unpack16<T>(ra[i], v);
        if (pack) {
          const uint32_t top = top_bits<T>(ra[i], v);
          const uint32_t byte = scale_byte(PER == 8 ? quad_max(top) : oct_max(top));
          const float inv = inv_scale(byte);
          // a NaN that was widened from 16 bits has a low byte of 0, and so has inf * 0: no code to clear
          uint32_t c[PER / 4];
#pragma unroll
          for (int e = 0; e < PER / 4; ++e) c[e] = code4(v + 4 * e, inv, ES == 4 && byte == 255u);
          const int kc = k0 + (WK == 1 ? 0 : NT / 8 * i / BM * BK);
          const bool in = kc + lk < p.Cp;
          if constexpr (PER == 8) {
            const u32x2_t two = {c[0], c[1]};
            __builtin_amdgcn_raw_buffer_store_b64(two, cr, static_cast<int>(in ? coff[i] : kOut), kc, 0);
          } else {
            __builtin_amdgcn_raw_buffer_store_b32(c[0], cr, static_cast<int>(in ? coff[i] : kOut), kc, 0);
          }
          __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(byte), er, static_cast<int>(in ? eoff[i] : kOut), kc / kBlock, 0);
        }
        if constexpr (ACT == kCkptGelu) {
#pragma unroll
          for (int e = 0; e < PER; ++e) v[e] = gelu<T>(v[e]);
          ra[i] = pack16<T>(v);
        }
      }
      xs[buf * CH + slot * 8 + (chunk ^ swz_a(row))] = ra[i];
    }
  };
  // fragments of b: row r of tile t is column 4 TN (r / 4) + 4 t + r % 4 of the wave's WC; half s of the step
  const int brow = wn * WC + 4 * TN * (r >> 2) + (r & 3), bk = wk * BK + g * PER;
  const T* B = static_cast<const T*>(p.b) + static_cast<int64_t>(n0) * p.K;
  const int64_t bsize = static_cast<int64_t>(p.N - n0) * p.K;
  const __amdgpu_buffer_rsrc_t br = range(B, bsize * ES);
  uint32_t boff[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) boff[t] = (static_cast<uint32_t>(brow + 4 * t) * p.K + bk) * ES;
  uint4 wf[2][TN];
  auto fetch_b = [&](int s, int k0) {
    const int kc = k0 + s * 4 * PER, have = p.K - kc - bk;
    if (!VEC && whole_b(k0)) {
#pragma unroll
      for (int t = 0; t < TN; ++t) wf[s][t] = here16<T>(B + kc, boff[t] / ES);
      return;
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      if constexpr (VEC) wf[s][t] = buf16(br, have > 0 ? boff[t] : kOut, kc * ES);
      else wf[s][t] = any16<T>(B, boff[t] / ES + kc, bsize);
    }
  };

  for (int n = tid; n < BN; n += NT)  // a barrier is in front of the first use
    bs[n] = p.bias == nullptr || n0 + n >= p.N ? 0.f
            : p.bias_f32                       ? static_cast<const float*>(p.bias)[n0 + n]
                                               : Io<T>::ld(static_cast<const T*>(p.bias) + n0 + n);
  int xat[2];  // fragment addresses of a: the XOR's bits come from the lane alone, tiles are constant offsets
#pragma unroll
  for (int s = 0; s < 2; ++s) xat[s] = (wk * BM + wm * TM * 16 + r) * 8 + ((s * 4 + g) ^ swz_a(r));
  const int nc = n0 + wn * WC + 4 * TN * g;  // this lane's 4 TN columns

  f32x4_t acc[TM][TN];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  auto multiply = [&](int s, int buf, int k0) {
    if (!VEC && !whole_b(k0)) {
      const int kc = k0 + s * 4 * PER, have = p.K - kc - bk;
#pragma unroll
      for (int t = 0; t < TN; ++t)
        wf[s][t] = settle16<T>(wf[s][t], B, boff[t] / ES + kc, n0 + brow + 4 * t < p.N ? have : 0);
    }
    uint4 xf[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) xf[t] = xs[buf * CH + xat[s] + t * 128];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mma16<T>(wf[s][j], xf[i], acc[i][j]);
  };
  auto finish = [&](int m) {  // lane: row `row` of every tile i, columns nc .. nc + 15
    const int64_t m0 = static_cast<int64_t>(m) * BM;
    T* O = static_cast<T*>(p.out) + m0 * p.N;
    const __amdgpu_buffer_rsrc_t orr = range(O, (p.M - m0) * p.N * ES);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const uint32_t row = (wm * TM + i) * 16 + r;
      float v[4 * TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] = acc[i][j][e];
#pragma unroll
      for (int e = 0; e < 4 * TN; ++e) v[e] += bs[wn * WC + 4 * TN * g + e];
      if (p.vo) {
        if constexpr (TN == 4 || ES == 4) {
#pragma unroll
          for (int e = 0; e < 4 * TN; e += PER) put16(orr, nc + e < p.N ? (row * p.N + nc + e) * ES : kOut, pack16<T>(v + e));
        } else {
#pragma unroll
          for (int e = 0; e < 4 * TN; e += 4) put8(orr, nc + e < p.N ? (row * p.N + nc + e) * ES : kOut, pack8<T>(v + e));
        }
      } else if (m0 + row < p.M) {
        put_any<T, 4 * TN>(O + static_cast<int64_t>(row) * p.N + nc, p.N - nc, v);
      }
    }
  };

  fetch_a(mt, 0);
  fetch_b(0, 0);
  fetch_b(1, 0);
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
      multiply(0, buf, 0);
      multiply(1, buf, 0);
      finish(mt);
      buf ^= 1;
    }
  } else {
    if (STEP < p.K) fetch_a(mt, STEP);
    clear();
    __syncthreads();
    for (int k0 = 0; k0 < p.K; k0 += STEP) {
      if (k0 + STEP < p.K) {  // the next step goes to the other buffer, the one after it is on its way
        stage_a(mt, k0 + STEP, buf ^ 1);
        if (k0 + 2 * STEP < p.K) fetch_a(mt, k0 + 2 * STEP);
      }
      multiply(0, buf, k0);
      if (k0 + STEP < p.K) fetch_b(0, k0 + STEP);
      multiply(1, buf, k0);
      if (k0 + STEP < p.K) fetch_b(1, k0 + STEP);
      __syncthreads();
      buf ^= 1;
    }
    if constexpr (WK > 1) {
      float4* join = reinterpret_cast<float4*>(xs);
      constexpr int PER_WAVE = TM * TN, GROUP = WM * WN * PER_WAVE;
      const int place = (wm * WN + wn) * PER_WAVE;
      if (wk > 0) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            join[((wk - 1) * GROUP + place + i * TN + j) * 64 + lane] =
                make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
      }
      __syncthreads();
      if (wk > 0) return;
#pragma unroll
      for (int q = 0; q < WK - 1; ++q)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const float4 v = join[(q * GROUP + place + i * TN + j) * 64 + lane];
            acc[i][j][0] += v.x;
            acc[i][j][1] += v.y;
            acc[i][j][2] += v.z;
            acc[i][j][3] += v.w;
          }
    }
    finish(mt);
  }
}

template <typename T, int ACT, int WN, int WM, int WK, int TM, int TN, bool VEC, int WAVES>
void launch_cfg(FwdArgs p, hipStream_t st) {
  constexpr int BM = WM * TM * 16, BN = WN * TN * 16;
  p.ntiles = (p.N + BN - 1) / BN;
  p.mtiles = static_cast<int>((p.M + BM - 1) / BM);
  if constexpr (WK == 1 && VEC && BN <= 256) {
    if (p.K <= 8 * kPer16<T>) {
      constexpr int W1 = ACT == kCkptGelu && WAVES > 2 ? WAVES - 1 : WAVES;  // more registers
      const auto kernel = lin_fwd_kernel<T, ACT, WN, WM, WK, TM, TN, true, VEC, W1>;
      static const int resident = resident_blocks(kernel, WN * WM * WK * 64);
      kernel<<<one_wave_grid(resident, p.mtiles, p.ntiles), WN * WM * WK * 64, 0, st>>>(p);
      return;
    }
  }
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(p.mtiles) * p.ntiles);
  lin_fwd_kernel<T, ACT, WN, WM, WK, TM, TN, false, VEC, WAVES><<<grid, WN * WM * WK * 64, 0, st>>>(p);
}

// Tiles.  A problem of fewer than 256 tiles of 64 x 256 leaves CUs idle: 32 x 64 (fp32: 16 x 64) with k split four
// ways.
// Else narrow layers (N <= 64, 128) take their width and more rows, others 256 columns x 64 rows, and with
// gelu all columns up to 512.
template <typename T, int ACT>
void launch_fwd(const FwdArgs& p, bool vec, hipStream_t st) {
  constexpr int F = sizeof(T) == 4 ? 1 : 0;  // fp32 holds more: fewer waves
  const int64_t tiles = (p.M + 63) / 64 * ((p.N + 255) / 256);
  if (!vec) {
    if (tiles < 256) return launch_cfg<T, ACT, 1, 1, 4, 2 - F, 4, false, 3>(p, st);
    return launch_cfg<T, ACT, 2, 2, 1, 2, 4, false, 3 - F>(p, st);
  }
  if (tiles < 256) return launch_cfg<T, ACT, 1, 1, 4, 2 - F, 4, true, 3>(p, st);
  if (p.N <= 64) return launch_cfg<T, ACT, 1, 4, 1, 2, 4, true, 3>(p, st);
  if (p.N <= 128) return launch_cfg<T, ACT, 2, 2, 1, 2, 4, true, 4 - F>(p, st);
  if constexpr (ACT == kCkptGelu) {
    if (p.N > 320) return launch_cfg<T, ACT, 8, 1, 1, 4, 4, true, 2>(p, st);
    if (p.N > 256) return launch_cfg<T, ACT, 4, 1, 1, 4, 5, true, 2>(p, st);
  }
  launch_cfg<T, ACT, 4, 1, 1, 4, 4, true, 3 - F>(p, st);
}

}  // namespace
}  // namespace lin

void launch_lin_fwd(const LinFwdArgs& a, hipStream_t st) {
  using namespace lin;
  if (a.M == 0) return;
  const int64_t most = kMaxBlocks / ((a.N + 63) / 64) * 16;  // rows of the smallest tiles that one launch holds
  if (a.M > most) {
    const int64_t cp = padded(a.K);
    LinFwdArgs b = a;
    b.M = most;
    launch_lin_fwd(b, st);
    b.x = ahead(a.x, most * a.K * size_of(a.dtype));
    b.y = ahead(a.y, most * a.N * size_of(a.dtype));
    b.codes = ahead(a.codes, most * cp);
    b.scales = ahead(a.scales, most * (cp / kBlock));
    b.M = a.M - most;
    launch_lin_fwd(b, st);
    return;
  }
  FwdArgs p{};
  p.a = a.x; p.b = a.w; p.bias = a.b; p.out = a.y; p.codes = a.codes; p.scales = a.scales;
  p.M = a.M; p.N = a.N; p.K = a.K; p.Cp = static_cast<int>(padded(a.K));
  const int per = 16 / size_of(a.dtype);
  p.vo = a.N % per == 0 && al16(a.y);
  p.bias_f32 = a.b_dtype == kF32;
  const bool vec = a.K % per == 0 && al16(a.x) && al16(a.w);
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    if (a.act == kCkptGelu) launch_fwd<T, kCkptGelu>(p, vec, st);
    else launch_fwd<T, kCkptNone>(p, vec, st);
  });
}

}  // namespace rtseg
