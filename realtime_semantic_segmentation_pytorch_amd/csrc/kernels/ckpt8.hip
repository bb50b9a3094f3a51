// 8-bit activation checkpoints: pack and unpack (format: rtseg_ckpt8.h).
//
// Both are one pass over the data and bound by HBM: 8 channels a lane (16 or 32 bytes), the block
// maximum of 32 channels across 4 lanes by two DPP moves, no LDS.  The loads in flight come from the
// grid's many waves; nothing is reused, so there is nothing to tile.  131072 x 256 of bf16: pack 18 us, unpack 16 us
// (102 MB each, 5.6 and 6.2 TB/s with what the caches still hold).
#include <type_traits>

#include "rtseg_ckpt8.h"
#include "rtseg_launch.h"
#include "rtseg_rows_dev.h"

namespace rtseg {
namespace {

using namespace ckpt8;
using namespace rows;

// item = 8 channels of the padded row: items_row = Cp / 8 per row, 4 consecutive items = one block
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) ckpt8_pack_kernel(const T* __restrict__ x, uint2* __restrict__ codes,
                                                         uint8_t* __restrict__ scales, int64_t items, int64_t rows, int C,
                                                         int items_row) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t it = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; it < items; it += step) {
    const int64_t row = it / items_row;
    const int c = static_cast<int>(it - row * items_row) * 8;
    const int n = C - c;
    Raw8<T> r;
    float v[8];
    if constexpr (VEC) {  // a lane behind the last channel reads its row's first ones and drops them
      const uint4* p = reinterpret_cast<const uint4*>(x + row * C + (n > 0 ? c : 0));
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
        r.q[i] = p[i];
        if (n <= 0) r.q[i] = make_uint4(0u, 0u, 0u, 0u);
      }
    } else {
      const Span<T, false> s(x, row * C, rows * C);
      r = s.load(c, n);
      s.settle(r, c, n);
    }
    unraw8<T>(r, v);
    uint32_t byte;
    codes[it] = encode8(v, byte);  // items is a multiple of 4: a block's lanes leave the loop together
    if ((it & 3) == 0) scales[it >> 2] = static_cast<uint8_t>(byte);
  }
}

// H: the type of the tensor that was packed
template <typename T, typename H, bool VEC>
__global__ void __launch_bounds__(256) ckpt8_unpack_kernel(const uint2* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, T* __restrict__ x,
                                                           int64_t items, int64_t rows, int C, int items_row) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t it = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; it < items; it += step) {
    const int64_t row = it / items_row;
    const int c = static_cast<int>(it - row * items_row) * 8;
    const uint2 w = codes[it];
    const uint32_t byte = scales[it >> 2];
    const float s = scale_of(byte);
    float v[8];
    decode4(w.x, s, v);
    decode4(w.y, s, v + 4);
    hold<H, 8>(byte, v);
    const Raw8<T> r = raw8<T>(v);
    if constexpr (VEC) {
      if (c < C) {
        uint4* p = reinterpret_cast<uint4*>(x + row * C + c);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) p[i] = r.q[i];
      }
    } else {
      Span<T, false>(x, row * C, rows * C).store(c, C - c, r);
    }
  }
}

// f(T{}, are the rows 16-byte aligned?)
template <class F>
void by_rows(int dtype, const void* p, int C, F f) {
  auto with = [&](auto t) {
    if (C % 8 == 0 && al16(p)) f(t, std::true_type{});
    else f(t, std::false_type{});
  };
  if (dtype == kF32) with(float{});
  else if (dtype == kBF16) with(uint16_t{});
  else with(_Float16{});
}

}  // namespace

void launch_ckpt8_pack(const void* x, int dtype, int8_t* codes, uint8_t* scales, int64_t rows, int C, hipStream_t st) {
  const int per = static_cast<int>(padded(C) / 8);
  const int64_t items = rows * per;
  if (items == 0) return;
  const int grid = stream_grid(items, 256);
  by_rows(dtype, x, C, [&](auto t, auto vec) {
    using T = decltype(t);
    constexpr auto kernel = &ckpt8_pack_kernel<T, decltype(vec)::value>;
    kernel<<<grid, 256, 0, st>>>(static_cast<const T*>(x), reinterpret_cast<uint2*>(codes), scales, items, rows, C, per);
  });
}

void launch_ckpt8_unpack(const int8_t* codes, const uint8_t* scales, void* x, int dtype, int held, int64_t rows, int C,
                         hipStream_t st) {
  const int per = static_cast<int>(padded(C) / 8);
  const int64_t items = rows * per;
  if (items == 0) return;
  const int grid = stream_grid(items, 256);
  by_rows(dtype, x, C, [&](auto t, auto vec) {
    using T = decltype(t);
    auto go = [&](auto kernel) {
      kernel<<<grid, 256, 0, st>>>(reinterpret_cast<const uint2*>(codes), scales, static_cast<T*>(x), items, rows, C, per);
    };
    if (held == kF32) go(&ckpt8_unpack_kernel<T, float, decltype(vec)::value>);
    else if (held == kBF16) go(&ckpt8_unpack_kernel<T, uint16_t, decltype(vec)::value>);
    else go(&ckpt8_unpack_kernel<T, _Float16, decltype(vec)::value>);
  });
}

}  // namespace rtseg
