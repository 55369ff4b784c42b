// Rows of 4-bit pages. A head's row of `head_dim` values, head_dim a multiple
// of 32, is head_dim / 2 bytes of codes (dim 2i in the low half of byte i),
// then for each group of 32 dims two bf16, its step and its offset; a value is
// offset + step * code. 5 bits a value: 80 bytes for 128 dims.
//
// A group's offset is its lowest value, rounded down to bf16; its step a 15th
// of highest - offset, rounded to float32 and then up to bf16 (0 where that is
// below float32's normal range), so that offset .. offset + 15 step holds the
// whole group and no value is further than step / 2 from what is held. The
// code is the nearest whole number, ties to even, to (value - offset) * (1 /
// step rounded to float32). A group with a value that is not finite, or with
// an offset outside bf16's range, has NaN for both and is NaN when read.
//
// The arithmetic is in 64 bits: 16-bit values divided by a step of 8 bits lie
// on the borders between codes often (1 in 2^8), and in 64 bits the products
// are exact, so the codes do not depend on the order of the operations.
#pragma once

#include "cbk_common.hpp"

namespace cbk {

constexpr int kInt4Group = 32;                   // dims that share a step and an offset
constexpr int kInt4GroupBytes = kInt4Group / 2 + 4;  // codes, step and offset

__host__ __device__ inline int64_t int4_row_bytes(int64_t head_dim) { return head_dim / kInt4Group * kInt4GroupBytes; }

struct Int4Scale {
  float step, offset;  // bf16 values
  double inverse;      // of the step, a float32 value; 0 where the step is 0 or NaN
};

// From a group's extremes; `finite`: all of its values are.
__device__ __forceinline__ Int4Scale int4_scale(double low, double high, bool finite) {
  Int4Scale r;
  float f = float(low);
  if (double(f) > low) f = __uint_as_float(f > 0.f ? __float_as_uint(f) - 1u : f == 0.f ? 0x80000001u : __float_as_uint(f) + 1u);
  uint32_t bits = __float_as_uint(f);
  if (f < 0.f) bits += 0xffffu;  // away from zero is down
  r.offset = __uint_as_float(bits & 0xffff0000u);
  const float step = float((high - double(r.offset)) / 15.0);
  r.step = __uint_as_float((__float_as_uint(step) + 0xffffu) & 0xffff0000u);
  if (r.step < 0x1p-126f) r.step = 0.f;
  r.inverse = r.step > 0.f ? double(1.f / r.step) : 0.0;
  if (!finite || !(fabsf(r.offset) < __builtin_inff())) {
    r.step = r.offset = __uint_as_float(0x7fc00000u);
    r.inverse = 0.0;
  }
  return r;
}

// 0 .. 15; 0 for a group without an inverse
__device__ __forceinline__ uint32_t int4_code(double x, const Int4Scale& s) {
  if (s.inverse == 0.0) return 0u;
  return uint32_t(int32_t(fmin(fmax(__builtin_rint((x - double(s.offset)) * s.inverse), 0.0), 15.0)));
}

__device__ __forceinline__ uint32_t int4_scale_word(const Int4Scale& s) {
  return (__float_as_uint(s.step) >> 16) | (__float_as_uint(s.offset) & 0xffff0000u);
}

// The value of a code (the product of 8 and 4 bits is exact: one rounding).
__device__ __forceinline__ float int4_value(uint32_t code, uint32_t scale_word) {
  return fmaf(__uint_as_float(scale_word << 16), float(code), __uint_as_float(scale_word & 0xffff0000u));
}

}  // namespace cbk
