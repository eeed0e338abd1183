// Row access and activations of the head operators (layer norm, dropout): rows
// are taken in blocks of eight columns, the columns that share one counter of
// the dropout generator, so that a lane holds whole blocks whatever the row's
// length, stride or alignment.
#pragma once

#include "rp_device.h"
#include "rp_philox.h"

namespace rp {

// Four words at an address of any alignment: global memory takes 16-byte
// accesses at any byte address, and a row of odd length puts every other row's
// start off a vector boundary.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// Eight elements as stored: 8 words of fp32, or 4 words of two 16-bit values.
template <int ES>
struct Raw8 {
  uint32_t w[2 * ES];
};

// The eight elements at `col` of a row that has them all.
template <int ES>
__device__ __forceinline__ Raw8<ES> load_full8(const char* row, int64_t col) {
  Raw8<ES> r;
#pragma unroll
  for (int q = 0; q < ES / 2; ++q) {
    const u32x4_any v = *reinterpret_cast<const u32x4_any*>(row + col * ES + 16 * q);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[4 * q + i] = v[i];
  }
  return r;
}

// The eight elements at `col` of a row of d (those at or past d as zero bits;
// nothing past the row's end is read).
template <int ES>
__device__ __forceinline__ Raw8<ES> load_raw8(const char* row, int64_t col, int64_t d) {
  Raw8<ES> r;
  if (col + 8 <= d) {
    r = load_full8<ES>(row, col);
  } else {
#pragma unroll
    for (int i = 0; i < 2 * ES; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (col + i >= d) break;
      if constexpr (ES == 4)
        r.w[i] = reinterpret_cast<const uint32_t*>(row)[col + i];
      else
        r.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[col + i] << (16 * (i & 1));
    }
  }
  return r;
}

template <int ES>
__device__ __forceinline__ void to_floats(const Raw8<ES>& r, int dtype, float (&v)[8]) {
  if constexpr (ES == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
  } else if (dtype == RP_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r.w[i] << 16);
      v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = static_cast<float>(
          __builtin_bit_cast(_Float16, static_cast<uint16_t>(r.w[i / 2] >> (16 * (i & 1)))));
  }
}

// Eight elements at `col`, in fp32 (zeros at and past d).
__device__ __forceinline__ void load8(const void* row, int64_t col, int64_t d, int dtype,
                                      float (&v)[8]) {
  if (dtype == RP_F32)
    to_floats(load_raw8<4>(static_cast<const char*>(row), col, d), dtype, v);
  else
    to_floats(load_raw8<2>(static_cast<const char*>(row), col, d), dtype, v);
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dtype) {
  if (dtype == RP_BF16) {  // one instruction: to nearest even, a NaN stays one
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
  }
  const auto h = [](float f) {
    return (uint32_t)__builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  };
  return h(lo) | (h(hi) << 16);
}

// Eight elements at `col` of a row that has them all, rounded to nearest even.
__device__ __forceinline__ void store_full8(char* row, int64_t col, int dtype, const float (&v)[8]) {
  u32x4_any w;
  if (dtype == RP_F32) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[4 * q + i]);
      *reinterpret_cast<u32x4_any*>(row + col * 4 + 16 * q) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack16(v[2 * i], v[2 * i + 1], dtype);
    *reinterpret_cast<u32x4_any*>(row + col * 2) = w;
  }
}

// The same; those at and past d are not stored.
__device__ __forceinline__ void store8(void* row, int64_t col, int64_t d, int dtype,
                                       const float (&v)[8]) {
  if (col + 8 <= d) {
    store_full8(static_cast<char*>(row), col, dtype, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (col + i >= d) break;
    if (dtype == RP_F32)
      static_cast<float*>(row)[col + i] = v[i];
    else
      static_cast<uint16_t*>(row)[col + i] = (uint16_t)pack16(v[i], 0.f, dtype);
  }
}

// GELU(x) = x Phi(x), Phi the normal distribution.  With a = |x|,
//     Phi(-a) = exp(-a^2 / 2) P(t),  t = 1 / (1 + a / 4),
// P of degree 6 fitted by linear programming to the least largest error of
// Phi(-a) max(1, a): 2.0e-8, a third of a rounding of Phi near 1.  In fp32 the
// root mean square error of x Phi(x) over normal x is 2.8e-8 of its size.  An
// erfc of full relative accuracy would cost about twice the instructions, for
// the far tail's own digits, which no sum over the row keeps.
struct Gelu {
  float half;  // Phi(|x|) - 1/2
  float e;     // exp(-x^2 / 2)
};
__device__ __forceinline__ Gelu gelu_parts(float x) {
  const float a = fabsf(x);
  const float e = exp2_hw((x * x) * -0.72134752044448170f);
  const float t = __builtin_amdgcn_rcpf(ffma(a, 0.25f, 1.f));
  float q = -0.17316568477026575f;
  q = ffma(q, t, 0.9649922472688132f);
  q = ffma(q, t, -1.3460685369763286f);
  q = ffma(q, t, 1.3055142384554645f);
  q = ffma(q, t, -0.4882596902776471f);
  q = ffma(q, t, 0.25405431713520465f);
  q = ffma(q, t, -0.017066889858532747f);
  return {ffma(-e, q, 0.5f), e};
}
// x Phi(x) = x / 2 + |x| (Phi(|x|) - 1/2) (NaN for an infinite x, which leaves a
// row without a mean either way)
__device__ __forceinline__ float gelu_of(float x, const Gelu& g) {
  return ffma(fabsf(x), g.half, 0.5f * x);
}
// The same and GELU'(x) = Phi(x) + x phi(x), which share Phi(x).
__device__ __forceinline__ void gelu_both(const float x, float& value, float& slope) {
  const Gelu g = gelu_parts(x);
  const float cdf = 0.5f + copysignf(g.half, x);
  value = x * cdf;
  slope = ffma(x, g.e * 0.3989422804014327f, cdf);
}

}  // namespace rp
