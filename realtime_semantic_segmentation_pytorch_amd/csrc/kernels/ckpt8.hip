// 8-bit activation checkpoints: pack and unpack (format: rtseg_ckpt8.h).
//
// Both are one pass over the data and bound by HBM: 8 channels a lane (16 or 32 bytes), the block
// maximum of 32 channels across 4 lanes by two DPP moves, no LDS.  A lane keeps two rows' worth of
// loads in flight through the grid's many waves; nothing is reused, so there is nothing to tile.
#include "rtseg_ckpt8.h"
#include "rtseg_launch.h"

namespace rtseg {
namespace {

using namespace ckpt8;

// item = 8 channels of the padded row: items_row = Cp / 8 per row, 4 consecutive items = one block
template <typename T>
__global__ void __launch_bounds__(256) ckpt8_pack_kernel(const T* __restrict__ x, uint2* __restrict__ codes,
                                                         uint8_t* __restrict__ scales, int64_t items, int C,
                                                         int items_row, bool vec) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t it = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; it < items; it += step) {
    const int64_t row = it / items_row;
    const int c = static_cast<int>(it - row * items_row) * 8;
    float v[8];
    unraw8<T>(load8<T>(x + row * C + c, C - c, vec), v);
    uint32_t byte;
    codes[it] = encode8(v, byte);  // items is a multiple of 4: a block's lanes leave the loop together
    if ((it & 3) == 0) scales[it >> 2] = static_cast<uint8_t>(byte);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ckpt8_unpack_kernel(const uint2* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, T* __restrict__ x,
                                                           int64_t items, int C, int items_row, bool vec) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t it = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; it < items; it += step) {
    const int64_t row = it / items_row;
    const int c = static_cast<int>(it - row * items_row) * 8;
    const uint2 w = codes[it];
    const float s = scale_of(scales[it >> 2]);
    float v[8];
    decode4(w.x, s, v);
    decode4(w.y, s, v + 4);
    store8<T>(x + row * C + c, raw8<T>(v), C - c, vec);
  }
}

bool vec_ok(const void* p, int C) { return C % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

void launch_ckpt8_pack(const void* x, int dtype, int8_t* codes, uint8_t* scales, int64_t rows, int C, hipStream_t st) {
  const int per = static_cast<int>(padded(C) / 8);
  const int64_t items = rows * per;
  if (items == 0) return;
  const int grid = stream_grid(items, 256);
  const bool vec = vec_ok(x, C);
  auto* cd = reinterpret_cast<uint2*>(codes);
  switch (dtype) {
    case kF32: ckpt8_pack_kernel<<<grid, 256, 0, st>>>(static_cast<const float*>(x), cd, scales, items, C, per, vec); break;
    case kBF16: ckpt8_pack_kernel<<<grid, 256, 0, st>>>(static_cast<const uint16_t*>(x), cd, scales, items, C, per, vec); break;
    default: ckpt8_pack_kernel<<<grid, 256, 0, st>>>(static_cast<const _Float16*>(x), cd, scales, items, C, per, vec); break;
  }
}

void launch_ckpt8_unpack(const int8_t* codes, const uint8_t* scales, void* x, int dtype, int64_t rows, int C,
                         hipStream_t st) {
  const int per = static_cast<int>(padded(C) / 8);
  const int64_t items = rows * per;
  if (items == 0) return;
  const int grid = stream_grid(items, 256);
  const bool vec = vec_ok(x, C);
  const auto* cd = reinterpret_cast<const uint2*>(codes);
  switch (dtype) {
    case kF32: ckpt8_unpack_kernel<<<grid, 256, 0, st>>>(cd, scales, static_cast<float*>(x), items, C, per, vec); break;
    case kBF16: ckpt8_unpack_kernel<<<grid, 256, 0, st>>>(cd, scales, static_cast<uint16_t*>(x), items, C, per, vec); break;
    default: ckpt8_unpack_kernel<<<grid, 256, 0, st>>>(cd, scales, static_cast<_Float16*>(x), items, C, per, vec); break;
  }
}

}  // namespace rtseg
