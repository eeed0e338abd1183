// Rows in 8 bits: blocks of 32 columns share a power of two 2^E, E = e - 127, and a
// value is q 2^E with q = round(x 2^-E) in [-127, 127].
//
// A power of two keeps everything exact but the one rounding: x 2^-E, q 2^E and the
// choice of E (from the exponent field of the block's largest magnitude) have no
// error, so every part of the library and of a test finds the same bits.  A scale of
// largest / 127 would leave 0.7 of the error on average, at a division a block and
// results that turn on its rounding.
//
// In a block that reaches to the top of its type's range the largest value is 64 steps,
// and 64 of them may be the power of two behind the type's largest (fp16: 65280 on, held
// as 64 * 1024).  What was finite is read back finite: cut to the type's largest value,
// which is nearer to what was packed than the 64 steps are.
#pragma once

#include "rp_rows.h"

namespace rp {

constexpr int kPackBlock = 32;

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kCtrl, 0xf, 0xf, true);
}

// Eight values of a lane to 8 bits, four adjacent lanes (a quad) holding a block:
// e, and the two words of q.  Lanes past the row hold zeros.
__device__ __forceinline__ uint32_t pack_block(const float (&v)[8], uint32_t (&q)[2]) {
  // the largest magnitude by its bits, which order NaN above infinity above all else
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  uint32_t o = dpp_u<0xb1>(top);  // quad_perm [1, 0, 3, 2]
  top = o > top ? o : top;
  o = dpp_u<0x4e>(top);  // quad_perm [2, 3, 0, 1]
  top = o > top ? o : top;
  // 1.m 2^(field - 127): times 2^(133 - field) it is in [64, 128), and rounds to 128
  // from 127.5 on
  int e = (int)(top >> 23) - 6 + ((top & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
  e = e < 1 ? 1 : e;
  const bool fine = top < 0x7f800000u;
  const float down = fine ? __uint_as_float((uint32_t)(254 - e) << 23) : 0.f;
  q[0] = q[1] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = fine ? (int)rintf(v[i] * down) : 0;
    q[i / 4] |= ((uint32_t)k & 0xffu) << (8 * (i & 3));
  }
  return fine ? (uint32_t)e : 255u;
}

// What they hold of values of a type (255: infinity times q = 0, a NaN).
__device__ __forceinline__ void unpack_block(const uint32_t (&q)[2], uint32_t e, int dtype,
                                             float (&v)[8]) {
  const float up = __uint_as_float(e << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)(int8_t)(q[i / 4] >> (8 * (i & 3))) * up;
  // (the least step of which 127 pass the type's largest value)
  if (e >= (dtype == RP_F16 ? 137u : 249u)) {
    const float top = dtype == RP_F16 ? 65504.f : __uint_as_float(dtype == RP_BF16 ? 0x7f7f0000u : 0x7f7fffffu);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] > top ? top : v[i] < -top ? -top : v[i];  // (a NaN stays)
  }
}

// The bytes at `col` .. col + 7 of a row of d (zeros at and past d).
__device__ __forceinline__ void load_q8(const int8_t* row, int64_t col, int64_t d, uint32_t (&q)[2]) {
  q[0] = q[1] = 0;
  if (col + 8 <= d) {
    const u32x2_any v = *reinterpret_cast<const u32x2_any*>(row + col);
    q[0] = v[0];
    q[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i) {
      if (col + i >= d) break;
      q[i / 4] |= (uint32_t)(uint8_t)row[col + i] << (8 * (i & 3));
    }
  }
}

__device__ __forceinline__ void store_q8(int8_t* row, int64_t col, int64_t d, const uint32_t (&q)[2]) {
  if (col + 8 <= d) {
    u32x2_any v;
    v[0] = q[0];
    v[1] = q[1];
    *reinterpret_cast<u32x2_any*>(row + col) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i) {
      if (col + i >= d) break;
      row[col + i] = (int8_t)(q[i / 4] >> (8 * (i & 3)));
    }
  }
}

}  // namespace rp
