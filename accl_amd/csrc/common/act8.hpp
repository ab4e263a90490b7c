// Activations kept in 8 bits: the element formulas, shared host/device.
//
// A group of GROUP values along a row shares a power of two 2^e, and a value
// x is held as code = round(x / 2^e), ties to even, within -127..127:
//   e = max(floor(log2(max |x|)) - 6, -126).
// x / 2^e then lies below 128, so that only values above 127.5 units are cut
// to 127. A power of two makes the division exact and leaves code * 2^e with
// seven significant bits: it is exact in bfloat16 and float32, and in float16
// for values that came from float16. The matrix product of a backward pass
// thus reads exactly what is held.
//
// A group with an infinity or a NaN has the exponent byte -128 and codes of
// zero, and stands for NaN: an overflow stays visible in the gradients.
#pragma once
#include "types.hpp"

namespace accl {
namespace act8 {

constexpr u32 GROUP = 32;
constexpr int LOST = -128;  // exponent byte of a group that holds no numbers

ACCL_HD inline u32 float_bits(float f) {
  u32 b;
  __builtin_memcpy(&b, &f, 4);
  return b;
}
ACCL_HD inline float bits_float(u32 b) {
  float f;
  __builtin_memcpy(&f, &b, 4);
  return f;
}

// |x| as bits: ordered as the magnitudes are, infinities above all numbers
// and NaN above those
ACCL_HD inline u32 magnitude(float x) { return float_bits(x) & 0x7FFFFFFFu; }

ACCL_HD inline int exponent_of(u32 largest) {
  int field = int(largest >> 23);
  if (field == 255) return LOST;
  int e = field - 133;
  return e < -126 ? -126 : e;
}

// The exponent by which float16 products take a group. Values that came from
// float16 have at most 9 and are exact in it; a group beyond that is taken as
// lost, since what it holds would overflow.
constexpr int F16_MOST = 9;
ACCL_HD inline int exponent_in_f16(int e) { return e > F16_MOST ? LOST : e; }

// 1 / 2^e, and 0 where the group is lost (-126 <= e <= 121 otherwise)
ACCL_HD inline float step_inverse(int e) {
  return e == LOST ? 0.0f : bits_float(u32(127 - e) << 23);
}

// 2^e. The byte of a lost group gives minus infinity, which its codes of zero
// turn into NaN.
ACCL_HD inline float step(int e) { return bits_float(u32(e + 127) << 23); }

ACCL_HD inline int code_of(float x, float inverse) {
  float v = __builtin_rintf(x * inverse);
  v = v > 127.0f ? 127.0f : v;
  v = v < -127.0f ? -127.0f : v;
  return int(v);
}

ACCL_HD inline u64 groups_of(u64 width) { return (width + GROUP - 1) / GROUP; }

}  // namespace act8
}  // namespace accl
