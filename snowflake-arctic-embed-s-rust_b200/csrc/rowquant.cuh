// Per-token int8 quantization from the bits of a row's largest |y|.
#pragma once
#include <cstdint>

#include "rowmath.cuh"

namespace ae {

// Smallest row maximum that quantizes to anything but zeros: below it 127 / top would not be finite.
constexpr float kTinyTop = 0x1p-119f;

// The bits of |y| order as |y| does, and a NaN's are above every number's.
struct RowScale {
  float inv, scale;
  bool any;
  __device__ __forceinline__ explicit RowScale(uint32_t top_bits) {
    // a row that holds an infinity or a NaN has no scale: its scale is NaN, and so is its row of the product
    const bool finite = top_bits < 0x7f800000u;
    const float top = __uint_as_float(top_bits);
    any = finite && top >= kTinyTop;
    inv = any ? 127.0f / top : 0.0f;
    scale = any ? top / 127.0f : (finite ? 0.0f : __uint_as_float(0x7fc00000u));
  }
  // Four values as int8 bytes, the first in the lowest.
  __device__ __forceinline__ uint32_t four(const float* y) const {
    return any ? pack_i8x4(quant_bits_scaled(y[0] * inv), quant_bits_scaled(y[1] * inv), quant_bits_scaled(y[2] * inv),
                           quant_bits_scaled(y[3] * inv))
               : 0u;
  }
};

}  // namespace ae
