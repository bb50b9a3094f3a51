// The linear layer that keeps its input as an 8-bit checkpoint (rtseg_ckpt8.h), on MFMA:
//
//   forward   y = act(x) w^T + b          codes = checkpoint of x
//   dgrad     dx = (dy w) * act'(z)       z = the checkpoint's values
//   wgrad     dw = dy^T act(z), db = sum_rows dy
//
// bf16 / fp16 operands feed v_mfma_f32_16x16x32, fp32 ones v_mfma_f32_16x16x4_f32; sums are fp32.
// act = gelu is computed in fp32 and rounded to the operands' type in front of the product, which is
// what a separate activation layer hands to a linear layer.
//
// forward and dgrad are the same product, C[m, n] = sum_k A[m, k] B[n, k] with both operands k-major:
// a block stages 128 rows of A and 128 (or 64) rows of B, 128 bytes of k each, through registers into
// LDS -- registers because that is where the forward takes the checkpoint (the blocks of the first
// column write it) and applies the activation.  The weights are the MFMA row operand, so that a lane
// ends with 16 consecutive columns of one row: wide stores, and in dgrad one 16-byte load of codes.
// wgrad is a product over the rows: both operands are staged row-major and read transposed
// (ds_read_b64_tr_b16; fp32 reads four columns at once, which feed four MFMA tiles), the row range is
// split over blocks and the fp32 partial tiles are summed by a second kernel: no atomics.
#include "rtseg_ckpt8.h"
#include "rtseg_launch.h"
#include "rtseg_mfma_dev.h"

namespace rtseg {
namespace {

using namespace ckpt8;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

// Phi(-|x|), the normal tail, by Abramowitz and Stegun 7.1.26 (erfc(z) = t (a1 + ... + a5 t^4) exp(-z^2),
// t = 1 / (1 + p z), error below 1.5e-7) with z = |x| / sqrt(2) folded into the constants; e = exp(-x^2 / 2)
__device__ __forceinline__ float normal_tail(float ax, float e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(ax, 0.3275911f * 0.70710678118654752f, 1.f));
  float q = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = __builtin_fmaf(t, q, 0.5f * 1.421413741f);
  q = __builtin_fmaf(t, q, 0.5f * -0.284496736f);
  q = __builtin_fmaf(t, q, 0.5f * 0.254829592f);
  return q * t * e;
}
__device__ __forceinline__ float exp_half_square(float x) {  // exp(-x^2 / 2)
  return __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);
}
// gelu(x) = x Phi(x) = max(x, 0) - |x| Phi(-|x|), gelu'(x) = Phi(x) + x phi(x).  16-bit operands take the tail
// above (14 full-rate and 2 quarter-rate instructions, 0.75e-7 |x| off, far below their rounding: a fifth of
// erff's cost, which bound all three products); fp32 ones erff.
template <typename T>
__device__ __forceinline__ float gelu(float x) {
  if constexpr (sizeof(T) == 4) return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
  const float ax = fabsf(x);  // the factor is cut off where the tail is 0: inf - inf * 0 is inf
  return __builtin_fmaf(-fminf(ax, 64.f), normal_tail(ax, exp_half_square(x)), fmaxf(x, 0.f));
}
template <typename T>
__device__ __forceinline__ float gelu_slope(float x) {
  if constexpr (sizeof(T) == 4)
    return 0.5f * (1.f + erff(x * 0.70710678118654752f)) + x * 0.39894228040143268f * __expf(-0.5f * x * x);
  const float e = exp_half_square(x), tail = normal_tail(fabsf(x), e);
  return __builtin_fmaf(x * 0.39894228040143268f, e, x >= 0.f ? 1.f - tail : tail);
}

// 16 bytes of operand: 8 (bf16 / fp16) or 4 (fp32) consecutive k
template <typename T> constexpr int kPer16 = 16 / static_cast<int>(sizeof(T));

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

// A range of a tensor as a buffer: accesses past `bytes` read 0, so a tile's missing rows cost no branch.
// kOut as an offset is past every range.
constexpr uint32_t kOut = 0xfffffff0u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t range(const void* p, int64_t bytes) {
  const uint32_t n = bytes < 0 ? 0u : bytes > 0xffffff00ll ? 0xffffff00u : static_cast<uint32_t>(bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(n), 0x00020000);
}
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 buf16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(uint4, static_cast<u32x4_t>(__builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(off), 0, 0)));
}
// 16 bytes of T at byte offset off, of which the first n elements exist (n <= 0: none); VEC: off is
// 16-byte aligned and n is <= 0 or whole
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off, int n) {
  if constexpr (VEC) return buf16(r, n > 0 ? off : kOut);
  T t[kPer16<T>];
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i) {
    const int o = static_cast<int>(i < n ? off + i * sizeof(T) : kOut);
    if constexpr (sizeof(T) == 4) t[i] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0));
    else t[i] = __builtin_bit_cast(T, static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0)));
  }
  uint4 q;
  __builtin_memcpy(&q, t, 16);
  return q;
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

// ------------------------------------------------------------------------------- forward, dgrad
struct NtArgs {
  const void* a;        // [M, K]: x, or dy
  const void* w;        // forward [N, K]; dgrad [K, N]
  const void* bias;     // [N] of w's type, or nullptr
  void* out;            // [M, N]
  int8_t* codes;        // forward: written, of a; dgrad with gelu: read, of out
  uint8_t* scales;
  int64_t M;
  int N, K, Cp;         // Cp: columns of codes
  int ntiles;           // column tiles
  bool w_f32;           // w (and bias) are fp32 beside 16-bit operands
  bool vo;              // 16-byte stores to out
};

__device__ __forceinline__ uint2 tr_read(const void* p) {
  auto q = (__attribute__((address_space(3))) mdev::i16x4_t*)((__attribute__((address_space(3))) void*)const_cast<void*>(p));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(q));
}

// A lane of a fragment ends with columns 16 g .. 16 g + 15 of its wave's 64 (g = lane / 16): row r of the
// row operand's tile t is column 16 (r / 4) + 4 t + r % 4, for fp32 in dgrad 4 r + t.
//
// LDS.  a: rows of 8 chunks of 16 bytes, chunk ^ (row & 7).  Forward w, the same, with the XOR taken from
// the row bits that one fragment read runs over.  dgrad w: BK rows of BN columns as in memory, read
// transposed: 8-byte units, XORed with row & 3 (a 16-lane group reads 4 rows) and row bit 3 (two groups).
__device__ __forceinline__ int swz_a(int row) { return row & 7; }
__device__ __forceinline__ int swz_w(int row) { return (row & 3) | ((row >> 4) & 1) << 2; }
__device__ __forceinline__ int swz_t8(int row) { return (row & 3) | ((row >> 3) & 1) << 4; }

// FWD: the a operand passes act and leaves its checkpoint, bias is added.  Else (dgrad): out is
// multiplied by act'.  VEC: rows of a and w are 16-byte aligned.
template <typename T, bool FWD, int ACT, int BN, bool VEC>
__global__ void __launch_bounds__(BN >= 256 ? 512 : 256) lin_nt_kernel(const NtArgs p) {
  constexpr int NT = BN >= 256 ? 512 : 256;
  constexpr int BM = 128, PER = kPer16<T>, BK = 8 * PER;
  constexpr int WN = BN / 64, WM = NT / 64 / WN, TM = BM / WM / 16;  // a wave: TM * 16 rows x 64 columns
  constexpr int XA = BM * 8 / NT, WB = BN * 8 / NT;
  constexpr int RC = BN / PER;  // dgrad: chunks of a LDS row of w
  __shared__ uint4 xs[BM * 8];
  __shared__ uint4 ws[BN * 8];

  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int wn = wid % WN, wm = wid / WN;
  const int g = lane >> 4, r = lane & 15;
  // the column tiles of one row tile follow each other on one XCD: they share its L2's copy of a
  const int lb = mdev::xcd_logical(blockIdx.x, gridDim.x);
  const int nt = lb % p.ntiles;
  const int n0 = nt * BN;
  const int64_t m0 = static_cast<int64_t>(lb / p.ntiles) * BM;
  const int chunk = tid & 7, srow = tid >> 3;  // staging of rows of 128 bytes
  const bool wide = sizeof(T) == 2 && p.w_f32;

  const __amdgpu_buffer_rsrc_t ar = range(static_cast<const T*>(p.a) + m0 * p.K,
                                          (p.M - m0) * p.K * static_cast<int64_t>(sizeof(T)));
  const int ew = wide ? 4 : static_cast<int>(sizeof(T));
  const int64_t wskip = FWD ? static_cast<int64_t>(n0) * p.K : n0;
  const __amdgpu_buffer_rsrc_t wr = range(static_cast<const char*>(p.w) + wskip * ew,
                                          (static_cast<int64_t>(p.N) * p.K - wskip) * ew);

  uint4 ra[XA], rw[WB], rw2[WB];
  auto fetch = [&](int k0) {
    const int k = k0 + chunk * PER;
#pragma unroll
    for (int i = 0; i < XA; ++i) {
      const uint32_t row = srow + NT / 8 * i;
      ra[i] = load16<T, VEC>(ar, (row * p.K + k) * static_cast<uint32_t>(sizeof(T)), p.K - k);
    }
#pragma unroll
    for (int i = 0; i < WB; ++i) {
      uint32_t off;
      int have;
      if constexpr (FWD) {
        off = static_cast<uint32_t>(srow + NT / 8 * i) * p.K + k;
        have = p.K - k;
      } else {
        const int id = tid + NT * i, row = id / RC, c = id % RC * PER;
        off = static_cast<uint32_t>(k0 + row) * p.N + c;
        have = k0 + row < p.K ? p.N - n0 - c : 0;
      }
      if (wide) {
        rw[i] = load16<float, VEC>(wr, off * 4, have);
        rw2[i] = load16<float, VEC>(wr, off * 4 + 16, have - 4);
      } else {
        rw[i] = load16<T, VEC>(wr, off * static_cast<uint32_t>(sizeof(T)), have);
      }
    }
  };

  f32x4_t acc[TM][4];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  fetch(0);
  for (int k0 = 0; k0 < p.K; k0 += BK) {
    if (k0 > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < XA; ++i) {
      const int row = srow + NT / 8 * i;
      if constexpr (FWD) {
        float v[PER];
        if (ACT == kCkptGelu || (p.codes != nullptr && nt == 0)) unpack16<T>(ra[i], v);
        if (p.codes != nullptr && nt == 0) {
          uint32_t m = 0;
#pragma unroll
          for (int e = 0; e < PER; ++e) m = max(m, abs_bits(v[e]));
          const uint32_t byte = scale_byte(PER == 8 ? quad_max(m) : oct_max(m));
          const float inv = inv_scale(byte);
          const int64_t mm = m0 + row;
          const int k = k0 + chunk * PER;
          if (mm < p.M && k < p.Cp) {
            const int64_t o = mm * p.Cp + k;
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.codes + o);
#pragma unroll
            for (int e = 0; e < PER / 4; ++e) dst[e] = code4(v + 4 * e, inv, byte == 255u);
            if (k % kBlock == 0) p.scales[o / kBlock] = static_cast<uint8_t>(byte);
          }
        }
        if constexpr (ACT == kCkptGelu) {
#pragma unroll
          for (int e = 0; e < PER; ++e) v[e] = gelu<T>(v[e]);
          ra[i] = pack16<T>(v);
        }
      }
      xs[row * 8 + (chunk ^ swz_a(row))] = ra[i];
    }
#pragma unroll
    for (int i = 0; i < WB; ++i) {
      if (wide) {
        float v[8];
        __builtin_memcpy(v, &rw[i], 16);
        __builtin_memcpy(v + 4, &rw2[i], 16);
        rw[i] = pack16<T>(v);
      }
      if constexpr (FWD) {
        const int row = srow + NT / 8 * i;
        ws[row * 8 + (chunk ^ swz_w(row))] = rw[i];
      } else {
        const int id = tid + NT * i, row = id / RC, c = id % RC;
        if constexpr (sizeof(T) == 2) {
          const int x = swz_t8(row);  // bit 0 of the unit: the two halves change places
          const uint4 q = (x & 1) ? make_uint4(rw[i].z, rw[i].w, rw[i].x, rw[i].y) : rw[i];
          ws[row * RC + (c ^ (x >> 1 & (RC - 1)))] = q;
        } else {
          ws[row * RC + c] = rw[i];
        }
      }
    }
    __syncthreads();
    if (k0 + BK < p.K) fetch(k0 + BK);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint4 wf[4], xf[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        const int row = (wm * TM + t) * 16 + r;
        xf[t] = xs[row * 8 + ((s * 4 + g) ^ swz_a(row))];
      }
      if constexpr (FWD) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int row = wn * 64 + 16 * (r >> 2) + 4 * t + (r & 3);
          wf[t] = ws[row * 8 + ((s * 4 + g) ^ swz_w(row))];
        }
      } else if constexpr (sizeof(T) == 2) {
        // k = 8 g + 0..7: two reads of 4 rows; lane 4 q + c of the group supplies row q, columns 16 c + 4 t ..
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint2 h[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = s * 32 + g * 8 + 4 * e + (r >> 2);
            const int unit = wn * 16 + (r & 3) * 4 + t;
            h[e] = tr_read(reinterpret_cast<const uint2*>(ws) + row * (BN / 4) + (unit ^ (swz_t8(row) & (BN / 4 - 1))));
          }
          wf[t] = make_uint4(h[0].x, h[0].y, h[1].x, h[1].y);
        }
      } else {
        // k = 4 g + i of this half: four columns a read, one for each tile
        const float* base = reinterpret_cast<const float*>(ws) + wn * 64 + 4 * r;
        float4 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const float4*>(base + (s * 16 + 4 * g + i) * BN);
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
  }

  // lane: row m of every tile i, columns nc .. nc + 15
  const int nc = n0 + wn * 64 + 16 * g;
  float bias[16];
  if constexpr (FWD) {
#pragma unroll
    for (int e = 0; e < 16; ++e) bias[e] = 0.f;
    if (p.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (nc + e < p.N)
          bias[e] = wide ? static_cast<const float*>(p.bias)[nc + e] : Io<T>::ld(static_cast<const T*>(p.bias) + nc + e);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + (wm * TM + i) * 16 + r;
    if (m >= p.M || nc >= p.N) continue;
    float v[16];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[!FWD && sizeof(T) == 4 ? 4 * e + j : 4 * j + e] = acc[i][j][e];
    if constexpr (FWD) {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] += bias[e];
    } else if constexpr (ACT == kCkptGelu) {
      const int64_t o = m * p.Cp + nc;  // nc is a multiple of 16, Cp of 32
      const uint4 cw = *reinterpret_cast<const uint4*>(p.codes + o);
      const float sc = scale_of(p.scales[o / kBlock]);
      const uint32_t w4[4] = {cw.x, cw.y, cw.z, cw.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float z[4];
        decode4(w4[j], sc, z);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * j + e] *= gelu_slope<T>(z[e]);
      }
    }
    T* out = static_cast<T*>(p.out) + m * p.N + nc;
    if (p.vo) {
#pragma unroll
      for (int e = 0; e < 16; e += PER)
        if (nc + e < p.N) *reinterpret_cast<uint4*>(out + e) = pack16<T>(v + e);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (nc + e < p.N) Io<T>::st(out + e, v[e]);
    }
  }
}

// ------------------------------------------------------------------------------- wgrad
struct TnArgs {
  const void* dy;       // [M, N]
  const int8_t* codes;  // [M, Cp]
  const uint8_t* scales;
  float* ws;            // [splits][N][K], then [splits][N] of db
  int64_t M, rows_per_split;
  int N, K, Cp, splits, ktiles, ntiles;
  bool want_db;
};

// LDS rows of 128 (or 64) columns.  16 bits: the transposed reads of a 16-lane group take 4 rows x 32
// bytes, the 4 groups rows 8 apart, so 32-byte units are XORed with (row & 3, row bit 3).
__device__ __forceinline__ int swz_t(int row) { return (row & 3) | ((row >> 3) & 1) << 2; }

template <typename T, int ACT, int BT, bool VEC>  // BT x BT output tile, 2 x 2 waves
__global__ void __launch_bounds__(kThreads) lin_tn_kernel(const TnArgs p) {
  constexpr int PER = kPer16<T>;
  constexpr int BS = sizeof(T) == 2 ? 64 : 32;       // rows a step
  constexpr int RC = BT / PER;                       // 16-byte chunks a LDS row
  constexpr int TT = BT / 2 / 16;                    // tiles a wave, each way
  constexpr int YC = BS * RC / kThreads;             // dy chunks a thread
  constexpr int CG = BT / 16;                        // 16-code groups a row
  constexpr int ZC = (BS * CG + kThreads - 1) / kThreads;
  constexpr int UM = BT / 16 - 1;                    // 32-byte units a 16-bit row - 1
  __shared__ uint4 zs[BS * RC];
  __shared__ uint4 ys[BS * RC];

  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int wk = wid & 1, wn = wid >> 1;
  const int g = lane >> 4, r = lane & 15;
  const int lb = mdev::xcd_logical(blockIdx.x, gridDim.x);  // a split's tiles on one XCD: they share its rows
  const int tiles = p.ktiles * p.ntiles, split = lb / tiles, tile = lb % tiles;
  const int kt = tile % p.ktiles;
  const int k0 = kt * BT, n0 = tile / p.ktiles * BT;
  const int64_t mb = split * p.rows_per_split;
  const int64_t me = mb + p.rows_per_split < p.M ? mb + p.rows_per_split : p.M;
  const bool db = p.want_db && kt == 0;

  const int64_t rows = me - mb;  // buffers over this split's rows: what lies behind reads 0
  const __amdgpu_buffer_rsrc_t yb = range(static_cast<const T*>(p.dy) + mb * p.N, rows * p.N * static_cast<int64_t>(sizeof(T)));
  const __amdgpu_buffer_rsrc_t cb = range(p.codes + mb * p.Cp, rows * p.Cp);
  const __amdgpu_buffer_rsrc_t eb = range(p.scales + mb * (p.Cp / kBlock), rows * (p.Cp / kBlock));

  uint4 yr[YC], zr[ZC];
  uint8_t zb[ZC];
  auto fetch = [&](int64_t m1) {
    const uint32_t mr = static_cast<uint32_t>(m1 - mb);
#pragma unroll
    for (int i = 0; i < YC; ++i) {
      const int id = tid + i * kThreads;
      const int n = n0 + (id % RC) * PER;
      yr[i] = load16<T, VEC>(yb, ((mr + id / RC) * p.N + n) * static_cast<uint32_t>(sizeof(T)), p.N - n);
    }
#pragma unroll
    for (int i = 0; i < ZC; ++i) {
      const int id = tid + i * kThreads;
      const int k = k0 + (id % CG) * 16;
      const bool in = id < BS * CG && k < p.Cp;
      const uint32_t o = (mr + id / CG) * p.Cp + k;
      zr[i] = buf16(cb, in ? o : kOut);
      zb[i] = static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(eb, static_cast<int>(in ? o / kBlock : kOut), 0, 0));
    }
  };
  auto at = [](int row, int chunk) {  // 16-byte slot of (row, chunk)
    if constexpr (sizeof(T) == 2) return row * RC + ((((chunk >> 1) ^ (swz_t(row) & UM)) << 1) | (chunk & 1));
    else return row * RC + chunk;
  };

  f32x4_t acc[TT][TT];  // [k tile][n tile]
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float sb[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) sb[e] = 0.f;

  if (mb < me) fetch(mb);
  for (int64_t m1 = mb; m1 < me; m1 += BS) {
    if (m1 > mb) __syncthreads();
#pragma unroll
    for (int i = 0; i < YC; ++i) {
      const int id = tid + i * kThreads;
      if (db) {  // a thread's chunks are all of the same columns
        float v[PER];
        unpack16<T>(yr[i], v);
#pragma unroll
        for (int e = 0; e < PER; ++e) sb[e] += v[e];
      }
      ys[at(id / RC, id % RC)] = yr[i];
    }
#pragma unroll
    for (int i = 0; i < ZC; ++i) {
      const int id = tid + i * kThreads;
      if (id < BS * CG) {
        const float sc = scale_of(zb[i]);
        const uint32_t w4[4] = {zr[i].x, zr[i].y, zr[i].z, zr[i].w};
        float v[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) decode4(w4[q], sc, v + 4 * q);
        if constexpr (ACT == kCkptGelu) {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = gelu<T>(v[e]);
        }
#pragma unroll
        for (int e = 0; e < 16; e += PER) zs[at(id / CG, (id % CG) * (16 / PER) + e / PER)] = pack16<T>(v + e);
      }
    }
    __syncthreads();
    if (m1 + BS < me) fetch(m1 + BS);
    if constexpr (sizeof(T) == 2) {
      const int q = r >> 2, c4 = (r & 3) * 4;
#pragma unroll
      for (int s = 0; s < BS / 32; ++s) {
        uint4 zf[TT], yf[TT];
        auto frag = [&](const uint4* base, int col) {
          const int cc = col + c4;
          uint2 h[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = s * 32 + g * 8 + 4 * e + q;
            h[e] = tr_read(reinterpret_cast<const char*>(base + at(row, cc >> 3)) + ((cc >> 2) & 1) * 8);
          }
          return make_uint4(h[0].x, h[0].y, h[1].x, h[1].y);
        };
#pragma unroll
        for (int t = 0; t < TT; ++t) zf[t] = frag(zs, (wk * TT + t) * 16);
#pragma unroll
        for (int t = 0; t < TT; ++t) yf[t] = frag(ys, (wn * TT + t) * 16);
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int j = 0; j < TT; ++j) acc[i][j] = mma16<T>(zf[i], yf[j], acc[i][j]);
      }
    } else {
      // lane r of group g reads row 4 s + g, columns TT * r .. + TT - 1 of its wave: column TT * r + t is
      // row r of tile t
#pragma unroll
      for (int s = 0; s < BS / 4; ++s) {
        float zf[TT], yf[TT];
        const float* zp = reinterpret_cast<const float*>(zs) + (4 * s + g) * BT + wk * (BT / 2) + TT * r;
        const float* yp = reinterpret_cast<const float*>(ys) + (4 * s + g) * BT + wn * (BT / 2) + TT * r;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
          zf[t] = zp[t];
          yf[t] = yp[t];
        }
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int j = 0; j < TT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(zf[i], yf[j], acc[i][j], 0, 0, 0);
      }
    }
  }

  float* slab = p.ws + static_cast<int64_t>(split) * p.N * p.K;
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dk = sizeof(T) == 2 ? i * 16 + 4 * g + e : TT * (4 * g + e) + i;
        const int dn = sizeof(T) == 2 ? j * 16 + r : TT * r + j;
        const int k = k0 + wk * (BT / 2) + dk, n = n0 + wn * (BT / 2) + dn;
        if (k < p.K && n < p.N) slab[static_cast<int64_t>(n) * p.K + k] = acc[i][j][e];
      }
  if (db) {
    __syncthreads();
    float* red = reinterpret_cast<float*>(ys);  // [kThreads / RC][BT]
#pragma unroll
    for (int e = 0; e < PER; ++e) red[(tid / RC) * BT + (tid % RC) * PER + e] = sb[e];
    __syncthreads();
    if (tid < BT && n0 + tid < p.N) {
      float s = 0.f;
      for (int q = 0; q < kThreads / RC; ++q) s += red[q * BT + tid];
      p.ws[static_cast<int64_t>(p.splits) * p.N * p.K + static_cast<int64_t>(split) * p.N + n0 + tid] = s;
    }
  }
}

// ws -> dw, db: one thread an element, the splits in order
template <typename TW>
__global__ void __launch_bounds__(256) lin_wgrad_join_kernel(const float* __restrict__ ws, TW* dw, TW* db, int splits,
                                                             int64_t plane, int N) {
  const int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  if (e < plane) {
    if (dw == nullptr) return;
    float s = 0.f;
#pragma unroll 8
    for (int i = 0; i < splits; ++i) s += ws[i * plane + e];
    Io<TW>::st(dw + e, s);
  } else if (e < plane + N && db != nullptr) {
    const float* w = ws + splits * plane + (e - plane);
    float s = 0.f;
#pragma unroll 8
    for (int i = 0; i < splits; ++i) s += w[static_cast<int64_t>(i) * N];
    Io<TW>::st(db + (e - plane), s);
  }
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

bool al16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <class F>
void by_type(int dt, F f) {
  if (dt == kF32) f(float{});
  else if (dt == kBF16) f(uint16_t{});
  else f(_Float16{});
}
int elem(int dt) { return dt == kF32 ? 4 : 2; }

struct WgradPlan { int tile, splits; int64_t rows; };
WgradPlan wgrad_plan(int64_t M, int N, int K) {
  WgradPlan w;
  w.tile = N <= 64 || K <= 64 ? 64 : 128;
  const int64_t tiles = static_cast<int64_t>((N + w.tile - 1) / w.tile) * ((K + w.tile - 1) / w.tile);
  int64_t s = 512 / tiles;                 // two blocks a CU
  const int64_t most = (M + 255) / 256;    // of at least 256 rows each
  if (s > most) s = most;
  if (s < 1) s = 1;
  w.rows = ((M + s - 1) / s + 63) / 64 * 64;
  if (w.rows < 64) w.rows = 64;
  w.splits = static_cast<int>((M + w.rows - 1) / w.rows);
  if (w.splits < 1) w.splits = 1;
  return w;
}

template <typename T, bool FWD, int ACT, int BN>
void launch_nt_bn(NtArgs p, bool vec, hipStream_t st) {
  p.ntiles = (p.N + BN - 1) / BN;
  const unsigned grid = static_cast<unsigned>((p.M + 127) / 128 * p.ntiles);
  constexpr int threads = BN >= 256 ? 512 : 256;
  if (vec) lin_nt_kernel<T, FWD, ACT, BN, true><<<grid, threads, 0, st>>>(p);
  else lin_nt_kernel<T, FWD, ACT, BN, false><<<grid, threads, 0, st>>>(p);
}
template <typename T, bool FWD, int ACT>
void launch_nt(const NtArgs& p, bool vec, hipStream_t st) {
  if (p.N <= 64) launch_nt_bn<T, FWD, ACT, 64>(p, vec, st);
  else if (p.N <= 128) launch_nt_bn<T, FWD, ACT, 128>(p, vec, st);
  else launch_nt_bn<T, FWD, ACT, 256>(p, vec, st);
}

}  // namespace

void launch_lin_fwd(const LinFwdArgs& a, hipStream_t st) {
  if (a.M == 0) return;
  NtArgs p{};
  p.a = a.x; p.w = a.w; p.bias = a.b; p.out = a.y; p.codes = a.codes; p.scales = a.scales;
  p.M = a.M; p.N = a.N; p.K = a.K; p.Cp = static_cast<int>(padded(a.K));
  const int per = 16 / elem(a.dtype);
  p.w_f32 = a.w_dtype == kF32;
  p.vo = a.N % per == 0 && al16(a.y);
  const bool vec = a.K % per == 0 && al16(a.x) && al16(a.w);
  by_type(a.dtype, [&](auto t) {
    if (a.act == kCkptGelu) launch_nt<decltype(t), true, kCkptGelu>(p, vec, st);
    else launch_nt<decltype(t), true, kCkptNone>(p, vec, st);
  });
}

void launch_lin_dgrad(const LinDgradArgs& a, hipStream_t st) {
  if (a.M == 0) return;
  NtArgs p{};
  p.a = a.dy; p.w = a.w; p.out = a.dx;
  p.codes = const_cast<int8_t*>(a.codes); p.scales = const_cast<uint8_t*>(a.scales);
  p.M = a.M; p.N = a.K; p.K = a.N; p.Cp = static_cast<int>(padded(a.K));
  const int per = 16 / elem(a.dtype);
  p.w_f32 = a.w_dtype == kF32;
  p.vo = a.K % per == 0 && al16(a.dx);
  const bool vec = a.N % per == 0 && a.K % per == 0 && al16(a.dy) && al16(a.w);
  by_type(a.dtype, [&](auto t) {
    if (a.act == kCkptGelu) launch_nt<decltype(t), false, kCkptGelu>(p, vec, st);
    else launch_nt<decltype(t), false, kCkptNone>(p, vec, st);
  });
}

int64_t lin_wgrad_ws_elems(int64_t M, int N, int K) {
  const WgradPlan w = wgrad_plan(M, N, K);
  return static_cast<int64_t>(w.splits) * (static_cast<int64_t>(N) * K + N);
}

void launch_lin_wgrad(const LinWgradArgs& a, hipStream_t st) {
  const WgradPlan w = wgrad_plan(a.M, a.N, a.K);
  TnArgs p{};
  p.dy = a.dy; p.codes = a.codes; p.scales = a.scales; p.ws = a.ws;
  p.M = a.M; p.rows_per_split = w.rows; p.N = a.N; p.K = a.K; p.Cp = static_cast<int>(padded(a.K));
  p.splits = w.splits;
  const bool vec = a.N % (16 / elem(a.dtype)) == 0 && al16(a.dy);
  p.want_db = a.db != nullptr;
  p.ktiles = (a.K + w.tile - 1) / w.tile;
  p.ntiles = (a.N + w.tile - 1) / w.tile;
  const unsigned grid = static_cast<unsigned>(p.ktiles * p.ntiles * w.splits);
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, st>>>(p); };
    const bool gelu = a.act == kCkptGelu;
    if (w.tile == 64) {
      if (vec) go(gelu ? lin_tn_kernel<T, kCkptGelu, 64, true> : lin_tn_kernel<T, kCkptNone, 64, true>);
      else go(gelu ? lin_tn_kernel<T, kCkptGelu, 64, false> : lin_tn_kernel<T, kCkptNone, 64, false>);
    } else {
      if (vec) go(gelu ? lin_tn_kernel<T, kCkptGelu, 128, true> : lin_tn_kernel<T, kCkptNone, 128, true>);
      else go(gelu ? lin_tn_kernel<T, kCkptGelu, 128, false> : lin_tn_kernel<T, kCkptNone, 128, false>);
    }
  });
  const int64_t plane = static_cast<int64_t>(a.N) * a.K;
  const unsigned jg = static_cast<unsigned>((plane + a.N + 255) / 256);
  by_type(a.w_dtype, [&](auto t) {
    using T = decltype(t);
    lin_wgrad_join_kernel<T><<<jg, 256, 0, st>>>(a.ws, static_cast<T*>(a.dw), static_cast<T*>(a.db), w.splits, plane, a.N);
  });
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
  by_type(db_dtype, [&](auto t) {
    using T = decltype(t);
    lin_wgrad_join_kernel<T><<<(N + 255) / 256, 256, 0, st>>>(ws, static_cast<T*>(nullptr), static_cast<T*>(db), splits, 0, N);
  });
}

}  // namespace rtseg
