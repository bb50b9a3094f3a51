// The checkpointing linear layer's weight gradient (definitions: rtseg_linear_dev.h):
//     dw[n, k] = sum_m dy[m, n] act(z[m, k]),   db[n] = sum_m dy[m, n].
//
// A product over the rows: both operands are staged as they lie, [row][channel], z decoded (and activated)
// on its way into LDS, and read transposed (ds_read_b64_tr_b16; fp32 reads several columns at once, one for
// each MFMA tile).  The row range is split over blocks and the fp32 partial tiles are summed in order by a
// second kernel: no atomics, the same bits on every run.
//
// What bounds it: HBM and, with gelu, the VALU work of decoding and of the tail: some 30 instructions an element,
// 33.5 M elements of 131072 x 256 make 1.0 G lane instructions, 25 us at 256 CUs x 64 lanes x 2.4 GHz.  So with gelu a
// tile is as wide in n as the layer (up to 512), which decodes every code once, and 64 or 128 channels of k; the
// number of blocks is held near one or two a CU, because each of them writes (and the join reads) one fp32 tile.
// Measured, and the join: 131072 rows of 256 x 64 17.3 + 4.3 us (76 MB, 3.5 TB/s), of 64 x 256 with gelu 23.5 + 4.6
// us, 32768 of 320 x 1280 with gelu 59 + 8 us (400 TF).  The bias gradient alone: 131072 x 64 8.9 + 5.0 us (16.8 MB).
#include "rtseg_linear_dev.h"

namespace rtseg {
namespace lin {
namespace {

struct TnArgs {
  const void* dy;       // [M, N]
  const int8_t* codes;  // [M, Cp]
  const uint8_t* scales;
  float* ws;            // [splits][N][K], then [splits][N] of db
  void* dw;             // splits == 1: written here, of w_dtype
  void* db;
  int64_t M, rows_per_split;
  int N, K, Cp, splits, ktiles, ntiles, w_dtype;
  bool want_db;
};

__device__ __forceinline__ void put1(void* p, int dt, int64_t i, float v) {
  if (dt == kF32) static_cast<float*>(p)[i] = v;
  else if (dt == kBF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
  else static_cast<_Float16*>(p)[i] = static_cast<_Float16>(v);
}

__device__ __forceinline__ void put4(void* p, int dt, int64_t i, const float* v) {  // of any alignment
  if (dt == kF32) {
    __builtin_memcpy(static_cast<float*>(p) + i, v, 16);
  } else {
    const uint2 q = dt == kBF16 ? pack8<uint16_t>(v) : pack8<_Float16>(v);
    __builtin_memcpy(static_cast<uint16_t*>(p) + i, &q, 8);
  }
}

// WN x WK waves of 16 TN columns n and 16 TK channels k each
template <typename T, int ACT, int WN, int WK, int TK, int TN, bool VEC, int WAVES>
__global__ void __launch_bounds__(WN* WK * 64, WAVES) lin_tn_kernel(const TnArgs p) {
  constexpr int NT = WN * WK * 64, KT = WK * TK * 16, WC = 16 * TN, NB = WN * WC;
  constexpr int PER = kPer16<T>, ES = static_cast<int>(sizeof(T));
  constexpr int BS = ES == 2 ? 64 : 32;  // rows a step
  // 16-byte chunks of a LDS row, whole 256-byte bank rounds where it is longer than one: the XORs stay inside
  constexpr int ZR = KT / PER, YC = NB / PER, YR = YC > 16 ? (YC + 15) / 16 * 16 : YC;
  // dy: 8 lanes stage 128 bytes of a row; a thread has YG such groups of columns, YT rows
  constexpr int YG = YC / 8, YROWS = NT / 8, YT = (BS + YROWS - 1) / YROWS, YN = YG * YT;
  constexpr int CG = KT / 16, ZN = (BS * CG + NT - 1) / NT;  // 16-code groups a row, a thread
  __shared__ uint4 zs[BS * ZR];
  __shared__ uint4 ys[BS * YR];

  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wid % WN, wk = wid / WN;
  const int g = lane >> 4, r = lane & 15;
  const int lb = mdev::xcd_logical(blockIdx.x, gridDim.x);  // a split's tiles on one XCD: they share its rows
  const int tiles = p.ktiles * p.ntiles, split = lb / tiles, tile = lb % tiles;
  const int kt = tile % p.ktiles;
  const int k0 = kt * KT, n0 = tile / p.ktiles * NB;
  const int64_t mb = split * p.rows_per_split;
  const int64_t me = mb + p.rows_per_split < p.M ? mb + p.rows_per_split : p.M;

  constexpr int ZROWS = NT / CG;
  const int yrow = tid >> 3, ycol = (tid & 7) * PER, zrow = tid / CG, zcol = tid % CG * 16;
  const bool zin = k0 + zcol < p.Cp;
  const int ep = p.Cp / kBlock;
  const uint32_t yoff = (static_cast<uint32_t>(yrow) * p.N + ycol) * ES;
  const uint32_t zoff = static_cast<uint32_t>(zrow) * p.Cp + zcol, eoff = static_cast<uint32_t>(zrow) * ep + zcol / kBlock;

  uint4 yr[YN], zr[ZN];
  // unaligned rows: a step that the tensor has in whole is read as it lies, the others chunk by chunk
  auto whole = [&](int64_t m1) { return m1 + (YN / YG * YROWS > BS ? YN / YG * YROWS : BS) <= me && n0 + NB <= p.N; };
  uint8_t zb[ZN];
  auto fetch = [&](int64_t m1) {  // rows m1 .. m1 + BS - 1; those behind the split's last read 0
    const int64_t left = me - m1;
    const T* Y = static_cast<const T*>(p.dy) + m1 * p.N + n0;
    const __amdgpu_buffer_rsrc_t yb = range(Y, (left * p.N - n0) * ES);
    const __amdgpu_buffer_rsrc_t cb = range(p.codes + m1 * p.Cp + k0, left * p.Cp - k0);
    const __amdgpu_buffer_rsrc_t eb = range(p.scales + m1 * ep + k0 / kBlock, left * ep - k0 / kBlock);
    const bool in = !VEC && whole(m1);
#pragma unroll
    for (int i = 0; i < YN; ++i) {
      const int skip = i % YG * 8 * PER;  // columns
      const uint32_t o = yoff + static_cast<uint32_t>(i / YG * YROWS * ES) * p.N + skip * ES;
      if constexpr (VEC) yr[i] = buf16(yb, p.N - n0 - ycol - skip > 0 ? o : kOut);
      else if (in) yr[i] = here16<T>(Y, o / ES);
      else yr[i] = any16<T>(static_cast<const T*>(p.dy), m1 * p.N + n0 + o / ES, p.M * p.N);
    }
#pragma unroll
    for (int i = 0; i < ZN; ++i) {
      zr[i] = buf16(cb, zin ? zoff + static_cast<uint32_t>(ZROWS * i) * p.Cp : kOut);
      zb[i] = buf1(eb, zin ? eoff + static_cast<uint32_t>(ZROWS * i) * ep : kOut);
    }
  };
  // LDS chunk of (row, chunk): 16 bits are read transposed, a 16-lane group 4 rows x 32 bytes and the 4 groups
  // rows 8 apart, so 32-byte units are XORed with the bits that tell 8 of those 16 rows apart: with row
  // bits 0, 1, 3 where a row is 256 bytes or more, bits 1, 3 (bit 0 is the bank half) in 128-byte rows
  auto swz = [](int row, int chunks) {
    return chunks >= 16 ? (row & 3) | ((row >> 3) & 1) << 2 : ((row >> 1) & 1) | ((row >> 3) & 1) << 1;
  };
  auto at = [&](int row, int chunk, int chunks) {
    if constexpr (ES == 2) return row * chunks + ((((chunk >> 1) ^ swz(row, chunks)) << 1) | (chunk & 1));
    else return row * chunks + chunk;
  };

  // fragment addresses (8-byte units for 16 bits, floats for fp32)
  int zat[TK], yat[TN];
  if constexpr (ES == 2) {
    const int row = g * 8 + (r >> 2), half = (r >> 1) & 1, sub = r & 1;
#pragma unroll
    for (int t = 0; t < TK; ++t) zat[t] = at(row, (wk * TK + t) * 2 + half, ZR) * 2 + sub;
#pragma unroll
    for (int t = 0; t < TN; ++t) yat[t] = at(row, (wn * TN + t) * 2 + half, YR) * 2 + sub;
  } else {
    zat[0] = g * KT + wk * TK * 16 + TK * r;
    yat[0] = g * YR * PER + wn * WC + TN * r;
  }

  f32x4_t acc[TK][TN];  // [k tile][n tile]
#pragma unroll
  for (int i = 0; i < TK; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // db: one more row of the product, of ones
  f32x4_t bacc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) bacc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const bool db = p.want_db && kt == 0 && wk == 0;

  fetch(mb);
  for (int64_t m1 = mb; m1 < me; m1 += BS) {
    const bool ends = !VEC && !whole(m1);
#pragma unroll
    for (int i = 0; i < YN; ++i) {
      const int row = yrow + i / YG * YROWS, skip = i % YG * 8 * PER;
      if (YROWS > BS && row >= BS) break;
      if (ends)
        yr[i] = settle16<T>(yr[i], static_cast<const T*>(p.dy), (m1 + row) * p.N + n0 + ycol + skip,
                            m1 + row < me ? p.N - n0 - ycol - skip : 0);
      ys[at(row, (tid & 7) + i % YG * 8, YR)] = yr[i];
    }
#pragma unroll
    for (int i = 0; i < ZN; ++i) {
      const int row = zrow + ZROWS * i;
      if (ZN * NT > BS * CG && row >= BS) break;
      const float sc = scale_of(zb[i]);
      const uint32_t w4[4] = {zr[i].x, zr[i].y, zr[i].z, zr[i].w};
      float v[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) decode4(w4[q], sc, v + 4 * q);
      hold<T, 16>(zb[i], v);
      if constexpr (ACT == kCkptGelu) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = gelu<T>(v[e]);
      }
#pragma unroll
      for (int e = 0; e < 16; e += PER) zs[at(row, tid % CG * (16 / PER) + e / PER, ZR)] = pack16<T>(v + e);
    }
    __syncthreads();
    if (m1 + BS < me) fetch(m1 + BS);
    if constexpr (ES == 2) {
#pragma unroll
      for (int s = 0; s < BS / 32; ++s) {
        uint4 zf[TK], yf[TN];
        auto frag = [&](const uint4* base, int unit, int chunks) {
          const uint2* u = reinterpret_cast<const uint2*>(base) + unit + s * 32 * chunks * 2;
          const uint2 lo = tr_read(u), hi = tr_read(u + 4 * chunks * 2);
          return make_uint4(lo.x, lo.y, hi.x, hi.y);
        };
#pragma unroll
        for (int t = 0; t < TK; ++t) zf[t] = frag(zs, zat[t], ZR);
#pragma unroll
        for (int t = 0; t < TN; ++t) yf[t] = frag(ys, yat[t], YR);
#pragma unroll
        for (int i = 0; i < TK; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mma16<T>(zf[i], yf[j], acc[i][j]);
        if (db) {
          const float one[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
#pragma unroll
          for (int j = 0; j < TN; ++j) bacc[j] = mma16<T>(pack16<T>(one), yf[j], bacc[j]);
        }
      }
    } else {
      // lane r of group g reads row 4 s + g, columns TK r .. (z) and TN r .. (dy) of its wave: column TK r + t
      // is row r of tile t
#pragma unroll
      for (int s = 0; s < BS / 4; ++s) {
        float zf[TK], yf[TN];
        __builtin_memcpy(zf, __builtin_assume_aligned(reinterpret_cast<const float*>(zs) + zat[0] + 4 * s * KT, 4 * TK), 4 * TK);
        __builtin_memcpy(yf, __builtin_assume_aligned(reinterpret_cast<const float*>(ys) + yat[0] + 4 * s * YR * PER, TN == 4 ? 16 : 4), 4 * TN);
#pragma unroll
        for (int i = 0; i < TK; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(zf[i], yf[j], acc[i][j], 0, 0, 0);
        if (db) {
#pragma unroll
          for (int j = 0; j < TN; ++j) bacc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(1.f, yf[j], bacc[j], 0, 0, 0);
        }
      }
    }
    __syncthreads();
  }

  const bool direct = p.splits == 1;
  const int64_t slab = direct ? 0 : static_cast<int64_t>(split) * p.N * p.K;
  void* to = direct ? p.dw : p.ws;
  const int tt = direct ? p.w_dtype : static_cast<int>(kF32);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + wn * WC + (ES == 2 ? j * 16 + r : TN * r + j);
    if (n >= p.N) continue;
    const int64_t base = slab + static_cast<int64_t>(n) * p.K;
#pragma unroll
    for (int i = 0; i < TK; ++i) {
      const int k = k0 + wk * TK * 16 + (ES == 2 ? i * 16 + 4 * g : TK * 4 * g + 4 * i);  // 4 consecutive k from here
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = ES == 2 ? acc[i][j][e] : acc[(4 * i + e) % TK][j][(4 * i + e) / TK];
      if (k + 4 <= p.K) {
        put4(to, tt, base + k, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < p.K) put1(to, tt, base + k + e, v[e]);
      }
    }
  }
  if (db && g == 0) {  // all rows of bacc are the same
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * WC + (ES == 2 ? j * 16 + r : TN * r + j);
      if (n >= p.N) continue;
      if (direct) put1(p.db, p.w_dtype, n, bacc[j][0]);
      else p.ws[static_cast<int64_t>(p.splits) * p.N * p.K + static_cast<int64_t>(split) * p.N + n] = bacc[j][0];
    }
  }
}

// ws -> dw, db.  A block owns 256 / GR fours of elements, its GR groups of lanes every GR-th split; the groups
// are added in order: the same sum on every run, and GR times the loads in flight of one thread a four.  Planes
// that would be few blocks take 32 groups of 8 lanes: 128 x 128 from 128 splits in 3.7 us against 4.7, but 256 x 64
// from 512, which is bound by its 34 MB, in 7.7 against 6.5.  (One element a lane took 9.5 us where 512 x 512 are joined
// from 16 splits and 12.8 us for 320 x 1280 from 25: too many blocks.)
template <typename TW, int GR>
__global__ void __launch_bounds__(256) lin_wgrad_join_kernel(const float* __restrict__ ws, TW* dw, TW* db, int splits,
                                                             int64_t plane, int N) {
  constexpr int EL = 256 / GR;
  __shared__ float4 red[GR][EL];
  const int el = threadIdx.x % EL, grp = threadIdx.x / EL;
  const int64_t q = blockIdx.x * static_cast<int64_t>(EL) + el, wq = (plane + 3) / 4;
  const bool is_w = q < wq;
  const int64_t e = 4 * (is_w ? q : q - wq), left = (is_w ? plane : db != nullptr ? N : 0) - e;
  const float* src = ws + (is_w ? 0 : splits * plane) + e;
  const int64_t step = is_w ? plane : N;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& v) { s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; };
  if (left >= 4) {
#pragma unroll 8
    for (int i = grp; i < splits; i += GR) {
      float4 v;
      __builtin_memcpy(&v, src + i * step, 16);
      add(v);
    }
  } else if (left > 0) {
    for (int i = grp; i < splits; i += GR)
      add(make_float4(src[i * step], left > 1 ? src[i * step + 1] : 0.f, left > 2 ? src[i * step + 2] : 0.f, 0.f));
  }
  red[grp][el] = s;
  __syncthreads();
  if (grp != 0 || left <= 0) return;
#pragma unroll
  for (int i = 1; i < GR; ++i) add(red[i][el]);
  TW* to = (is_w ? dw : db) + e;
  const float v[4] = {s.x, s.y, s.z, s.w};
  if (left >= 4) {
    if constexpr (sizeof(TW) == 4) {
      __builtin_memcpy(to, v, 16);
    } else {
      const uint2 o = pack8<TW>(v);
      __builtin_memcpy(to, &o, 8);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) Io<TW>::st(to + i, v[i]);
  }
}

void launch_join(int dtype, const float* ws, void* dw, void* db, int splits, int64_t plane, int N, hipStream_t st) {
  const int64_t fours = (plane + 3) / 4 + (N + 3) / 4;
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, int64_t each) {
      kernel<<<static_cast<unsigned>((fours + each - 1) / each), 256, 0, st>>>(ws, static_cast<T*>(dw), static_cast<T*>(db), splits, plane, N);
    };
    if (fours <= 512 * 32 && splits > 8 && splits <= 128) go(lin_wgrad_join_kernel<T, 32>, 8);
    else go(lin_wgrad_join_kernel<T, 8>, 32);
  });
}

// column sums of dy alone (a frozen weight with a trained bias): 64 columns x 4 row lanes a block, the
// row range split over blocks, ws [splits][N] for the join above
template <typename T>
__global__ void __launch_bounds__(256) lin_colsum_kernel(const T* __restrict__ dy, float* __restrict__ ws, int64_t M, int N,
                                                         int64_t rows_per_split) {
  __shared__ float red[4][64];
  const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6;
  const int n = blockIdx.y * 64 + cl;
  const int64_t mb = blockIdx.x * rows_per_split;
  const int64_t me = mb + rows_per_split < M ? mb + rows_per_split : M;
  float s = 0.f;
  if (n < N)
    for (int64_t m = mb + rl; m < me; m += 4) s += Io<T>::ld(dy + m * N + n);
  red[rl][cl] = s;
  __syncthreads();
  if (rl == 0 && n < N)
    ws[static_cast<int64_t>(blockIdx.x) * N + n] = (red[0][cl] + red[1][cl]) + (red[2][cl] + red[3][cl]);
}

// columns (16 TN each, times 1, 2, 4, 8 waves) and channels of a block, and how many blocks share the rows
struct TnPlan { int cols, kt, splits; int64_t rows; };
TnPlan tn_plan(int64_t M, int N, int K, int act) {
  TnPlan w;
  w.cols = N <= 64 ? 64 : N <= 128 ? 128 : N <= 256 || act == kCkptNone ? 256 : N <= 320 ? 320 : 512;
  w.kt = w.cols >= 256 ? 64 : 128;
  const int64_t tiles = static_cast<int64_t>((N + w.cols - 1) / w.cols) * ((K + w.kt - 1) / w.kt);
  // one block a CU; the second one of gelu hides its arithmetic (131072 x 256 x 64: 25.7 us against 31.5), without it
  // it only doubles what is joined (131072 x 64 x 256 with its join: 21.8 us against 26.1)
  int64_t s = (act == kCkptGelu ? 512 : 256) / tiles;
  const int64_t most = (M + 127) / 128;    // of at least 128 rows each
  if (s > most) s = most;
  if (s < 1) s = 1;
  w.rows = ((M + s - 1) / s + 63) / 64 * 64;
  if (w.rows < 64) w.rows = 64;
  w.splits = static_cast<int>((M + w.rows - 1) / w.rows);
  if (w.splits < 1) w.splits = 1;
  return w;
}

template <typename T, int ACT>
void launch_tn(TnArgs p, const TnPlan& w, bool vec, hipStream_t st) {
  p.ktiles = (p.K + w.kt - 1) / w.kt;
  p.ntiles = (p.N + w.cols - 1) / w.cols;
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(p.ktiles) * p.ntiles * p.splits);
  auto go = [&](auto kernel, int threads) { kernel<<<grid, threads, 0, st>>>(p); };
  constexpr int F = sizeof(T) == 4 ? 1 : 0;  // fp32 holds more: fewer waves
  switch (w.cols) {
    case 64: vec ? go(lin_tn_kernel<T, ACT, 1, 4, 2, 4, true, 4 - F>, 256) : go(lin_tn_kernel<T, ACT, 1, 4, 2, 4, false, 2>, 256); break;
    case 128: vec ? go(lin_tn_kernel<T, ACT, 2, 2, 4, 4, true, 3>, 256) : go(lin_tn_kernel<T, ACT, 2, 2, 4, 4, false, 2>, 256); break;
    case 256: vec ? go(lin_tn_kernel<T, ACT, 4, 1, 4, 4, true, ACT == kCkptGelu ? 2 : 3 - F>, 256) : go(lin_tn_kernel<T, ACT, 4, 1, 4, 4, false, 2>, 256); break;
    default:  // behind gelu alone
      if constexpr (ACT == kCkptGelu) {
        if (w.cols == 320) vec ? go(lin_tn_kernel<T, ACT, 4, 1, 4, 5, true, 2>, 256) : go(lin_tn_kernel<T, ACT, 4, 1, 4, 5, false, 2>, 256);
        else vec ? go(lin_tn_kernel<T, ACT, 8, 1, 4, 4, true, 2>, 512) : go(lin_tn_kernel<T, ACT, 8, 1, 4, 4, false, 2>, 512);
      }
  }
}

}  // namespace
}  // namespace lin

using namespace lin;

int64_t lin_wgrad_ws_elems(int64_t M, int N, int K, int act) {
  const TnPlan w = tn_plan(M, N, K, act);
  return w.splits == 1 ? 0 : static_cast<int64_t>(w.splits) * (static_cast<int64_t>(N) * K + N);
}

void launch_lin_wgrad(const LinWgradArgs& a, hipStream_t st) {
  const TnPlan w = tn_plan(a.M, a.N, a.K, a.act);
  TnArgs p{};
  p.dy = a.dy; p.codes = a.codes; p.scales = a.scales; p.ws = a.ws; p.dw = a.dw; p.db = a.db;
  p.M = a.M; p.rows_per_split = w.rows; p.N = a.N; p.K = a.K; p.Cp = static_cast<int>(padded(a.K));
  p.splits = w.splits; p.w_dtype = a.w_dtype;
  p.want_db = a.db != nullptr;
  const bool vec = a.N % (16 / size_of(a.dtype)) == 0 && al16(a.dy);
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    if (a.act == kCkptGelu) launch_tn<T, kCkptGelu>(p, w, vec, st);
    else launch_tn<T, kCkptNone>(p, w, vec, st);
  });
  if (w.splits == 1) return;
  const int64_t plane = static_cast<int64_t>(a.N) * a.K;
  launch_join(a.w_dtype, a.ws, a.dw, a.db, w.splits, plane, a.N, st);
}

int lin_colsum_splits(int64_t M) { return static_cast<int>(M < 64 ? 1 : (M / 64 < 512 ? M / 64 : 512)); }

void launch_lin_colsum(const void* dy, int dtype, float* ws, void* db, int db_dtype, int64_t M, int N, hipStream_t st) {
  const int splits = lin_colsum_splits(M);
  const int64_t rows = (M + splits - 1) / splits;
  const dim3 grid(splits, (N + 63) / 64);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    lin_colsum_kernel<<<grid, 256, 0, st>>>(static_cast<const T*>(dy), ws, M, N, rows);
  });
  launch_join(db_dtype, ws, nullptr, db, splits, 0, N, st);
}

}  // namespace rtseg
