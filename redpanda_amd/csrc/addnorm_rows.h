// RMS norm kernels that hold their rows in registers: one read of each row a pass.
// (The mathematics is in addnorm.hip, the way rows are shared by groups of lanes in
// layernorm_rows.h.)
//
// HBM bounds both ways: a row is read once, the next one while the present one is worked
// on, with the element sizes compiled in (chosen at run time, both forms of each load
// stayed in registers, and fewer waves fitted).  Forward and backward of the norm with
// add, against their bytes at the rate of a large copy:
//   16384 x 768, fp32 + bf16 -> bf16        31 + 42 us  (29 + 39)
//   131072 x 1024 bf16                     188 + 202    (209 + 261)
//   the same, kept in 8 bits               219 + 191    (236 + 236)
//   6000 x 9000, fp32 + bf16 -> bf16       114 + 173    (126 + 168)
#pragma once

#include "layernorm_rows.h"
#include "rp_pack8.h"
#include "rp_train.h"

namespace rp {

// A lane's blocks of a row of any type: fp32 or 16-bit elements as stored, or 8 bits
// with their exponent.
template <int ES>
struct AnyRow {
  Raw8<ES> r;
  __device__ __forceinline__ void floats(int dtype, float (&v)[8]) const { to_floats(r, dtype, v); }
};
template <>
struct AnyRow<1> {
  uint32_t q[2], e;
  __device__ __forceinline__ void floats(int dtype, float (&v)[8]) const {
    unpack_block(q, e, dtype, v);
  }
};

template <int ES, int G, int NB>
__device__ __forceinline__ void load_any(const NormCols<G, NB>& c, const char* row,
                                         AnyRow<ES> (&r)[NB]) {
  Raw8<ES> raw[NB];
  c.template load<ES>(row, raw);
#pragma unroll
  for (int j = 0; j < NB; ++j) r[j].r = raw[j];
}
// q, e: the row's bytes and exponents
template <int G, int NB>
__device__ __forceinline__ void load_kept(const NormCols<G, NB>& c, const int8_t* q, const uint8_t* e,
                                          AnyRow<1> (&r)[NB]) {
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    r[j].q[0] = r[j].q[1] = 0;
    r[j].e = 1;
    if (j + 1 < NB || c.any) {
      load_q8(q, c.col[j], c.d, r[j].q);
      r[j].e = e[c.col[j] / kPackBlock];
    }
  }
}

// v rounded to a type and back.
__device__ __forceinline__ void round_to(int dtype, float (&v)[8]) {
  if (dtype == RP_F32) return;
  Raw8<2> h;
#pragma unroll
  for (int i = 0; i < 4; ++i) h.w[i] = pack16(v[2 * i], v[2 * i + 1], dtype);
  to_floats(h, dtype, v);
}

// ES: bytes of an element of x (1: the rows are held in 8 bits), EA: of add.
template <int ES, int EA, int G, int NB>
__global__ __launch_bounds__(norm_threads(G)) void addnorm_fwd_rows_kernel(AddNormParams p) {
  constexpr int kW = G > kWave ? G / kWave : 1;
  __shared__ float buf[2][kW][1];
  NormRows<G> at;
  if (at.row >= p.rows) return;  // (whole workgroups where they share a row)
  const NormCols<G, NB> cols(at.g, p.d);
  const float invd = 1.f / (float)cols.d;
  const int64_t ne = (p.d + kPackBlock - 1) / kPackBlock;
  float w[NB][8];
  cols.load_weight(p.w, 1.f, 1.f, w);
  AnyRow<ES> rx[NB];
  Raw8<EA> ra[NB];
  auto load = [&](int64_t row) {
    if constexpr (ES == 1)
      load_kept(cols, p.q8 + row * p.d, p.e8 + row * ne, rx);
    else
      load_any<ES>(cols, static_cast<const char*>(p.x) + row * p.xsr * ES, rx);
    if (ES != 1 && p.add != nullptr)
      cols.template load<EA>(static_cast<const char*>(p.add) + row * p.asr * EA, ra);
  };
  load(at.row);
  for (int it = 0; at.row < p.rows; at.row += at.step, it ^= 1) {
    float v[NB][8];
#pragma unroll
    for (int j = 0; j < NB; ++j) rx[j].floats(ES == 1 ? p.dt_sum : p.dt_x, v[j]);
    if constexpr (ES != 1) {
      if (p.add != nullptr) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          float a[8];
          to_floats(ra[j], p.dt_add, a);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] += a[i];
          round_to(p.dt_sum, v[j]);
        }
      }
    }
    if (at.row + at.step < p.rows) load(at.row + at.step);
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] = ffma(v[j][i], v[j][i], s[0]);  // (0 past the row)
    if constexpr (ES != 1) {
      if (p.sum != nullptr)
        cols.store(static_cast<char*>(p.sum) + at.row * p.d * p.es_sum, p.dt_sum, v);
      if (p.q8 != nullptr) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          uint32_t q[2];
          const uint32_t e = pack_block(v[j], q);
          if (j + 1 < NB || cols.any) {
            store_q8(p.q8 + at.row * p.d, cols.col[j], p.d, q);
            if (cols.col[j] % kPackBlock == 0)
              p.e8[at.row * ne + cols.col[j] / kPackBlock] = (uint8_t)e;
          }
        }
      }
    }
    if (p.out == nullptr) continue;
    group_sum<G>(s, buf[it]);
    const float r = rsqrtf(ffma(s[0], invd, p.eps));
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = (v[j][i] * r) * w[j][i];
    cols.store(static_cast<char*>(p.out) + at.row * p.d * p.es_out, p.dt_out, v);
  }
}

// ds to dx and dadd, and the workgroup's sums of g xh over its rows to
// part[workgroup].  ES: bytes of an element of the rows s (1: in 8 bits), EO: of dout,
// ED: of dsum (ES, but for rows in 8 bits).
template <int ES, int EO, int ED, int G, int NB>
__global__ __launch_bounds__(norm_threads(G)) void addnorm_bwd_rows_kernel(AddNormParams p,
                                                                           AddNormGrad g) {
  constexpr int kW = G > kWave ? G / kWave : 1;
  constexpr int kGroups = norm_threads(G) / G;
  __shared__ float buf[2][kW][2];
  NormRows<G> at;
  const NormCols<G, NB> cols(at.g, p.d);
  const float invd = 1.f / (float)cols.d;
  const int64_t ne = (p.d + kPackBlock - 1) / kPackBlock;
  // 1024 threads have 128 registers each: there the weights are read for each row, no
  // row is read ahead, and the columns' sums are in LDS
  constexpr bool kAhead = G < 1024;
  __shared__ float dw_lds[kAhead ? 1 : 8 * NB][kAhead ? 1 : G];
  float w[NB][8], dw[NB][8] = {};
  if constexpr (kAhead) {
    cols.load_weight(p.w, 1.f, 1.f, w);
  } else {
#pragma unroll
    for (int i = 0; i < 8 * NB; ++i) dw_lds[i][at.g] = 0.f;
  }
  AnyRow<ES> rx[NB];
  Raw8<EO> rg[NB];
  Raw8<ED> rd[NB];
  auto load = [&](int64_t row) {
    if constexpr (ES == 1)
      load_kept(cols, p.q8 + row * p.d, p.e8 + row * ne, rx);
    else
      load_any<ES>(cols, static_cast<const char*>(p.x) + row * p.xsr * ES, rx);
    cols.template load<EO>(static_cast<const char*>(g.dout) + row * g.dosr * EO, rg);
    if (g.dsum != nullptr)
      cols.template load<ED>(static_cast<const char*>(g.dsum) + row * g.dssr * ED, rd);
  };
  if (kAhead && at.row < p.rows) load(at.row);
  for (int it = 0; at.row < p.rows; at.row += at.step, it ^= 1) {
    if constexpr (!kAhead) {
      load(at.row);
      const float* pw = p.w;
      asm volatile("" : "+s"(pw));  // (or the weights would be read once, and kept)
      cols.load_weight(pw, 1.f, 1.f, w);
    }
    float v[NB][8], q[NB][8], d[NB][8];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      rx[j].floats(p.dt_sum, v[j]);
      to_floats(rg[j], p.dt_out, q[j]);
      if (g.dsum != nullptr) {
        to_floats(rd[j], p.dt_sum, d[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[j][i] = 0.f;
      }
    }
    if (kAhead && at.row + at.step < p.rows) load(at.row + at.step);
    // mean(q xh) = r sum(q s) / d, so that one look at the row gives r and it
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[0] = ffma(v[j][i], v[j][i], s[0]);
        s[1] = ffma(q[j][i] * w[j][i], v[j][i], s[1]);
      }
    group_sum<G>(s, buf[it]);
    const float r = rsqrtf(ffma(s[0], invd, p.eps));
    const float m = r * s[1] * invd;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xh = v[j][i] * r;
        if constexpr (kAhead)
          dw[j][i] = ffma(q[j][i], xh, dw[j][i]);
        else
          dw_lds[j * 8 + i][at.g] = ffma(q[j][i], xh, dw_lds[j * 8 + i][at.g]);
        d[j][i] = ffma(ffma(-xh, m, q[j][i] * w[j][i]), r, d[j][i]);
      }
    if (g.dx != nullptr)
      cols.store(static_cast<char*>(g.dx) + at.row * p.d * p.es_x, p.dt_x, d);
    if (g.dadd != nullptr)
      cols.store(static_cast<char*>(g.dadd) + at.row * p.d * p.es_add, p.dt_add, d);
  }
  if (g.dw == nullptr) return;
  if constexpr (!kAhead) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[j][i] = dw_lds[j * 8 + i][at.g];
  }
  // the groups' sums: over a wave's groups by lane exchanges, then wave by wave
  // through LDS in order
  float* part = g.part + (int64_t)blockIdx.x * p.d;
  __shared__ float cols_sum[kGroups > 1 ? 8 * NB : 1][kWave];
  if constexpr (kGroups > 1) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int m = G; m < kWave; m <<= 1) dw[j][i] += __shfl_xor(dw[j][i], m);
    for (int t = 0; t < kWaves; ++t) {
      if (wave == t) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float* a = &cols_sum[j * 8 + i][lane];
            if (t > 0) dw[j][i] += *a;
            if (t + 1 < kWaves) *a = dw[j][i];
          }
      }
      __syncthreads();
    }
    if (wave + 1 < kWaves || lane >= G) return;
  }
  cols.store(reinterpret_cast<char*>(part), RP_F32, dw);
}

// The shapes (G, NB), by the blocks they hold.  (At least four lanes share a block of
// 32 columns: G is a multiple of four.)
#define RP_FOR_EACH_ADDNORM_SHAPE(X) \
  X(16, 1) X(32, 1) X(64, 1) X(32, 3) X(64, 2) X(64, 3) X(256, 1) X(256, 2) X(512, 2) X(1024, 2)

// Lanes a row of d columns is taken by; 0 for rows longer than the largest shape.
inline int addnorm_group(int64_t d) {
#define RP_CASE(G, NB) \
  if (d <= G * NB * 8) return G;
  RP_FOR_EACH_ADDNORM_SHAPE(RP_CASE)
#undef RP_CASE
  return 0;
}

// Workgroups that a launch fills the card with: as many as its registers let be
// resident.
inline int addnorm_workgroups_fwd(int64_t d) {
  const int G = addnorm_group(d);
  if (G > 256) return G == 1024 ? 256 : 512;
  const int nb = (int)((d + 8 * G - 1) / (8 * G));
  return 256 * (nb == 1 ? 7 : nb == 2 ? 5 : G < kWave ? 3 : 4);
}
inline int addnorm_workgroups_bwd(int64_t d) {
  const int G = addnorm_group(d);
  if (G > 256) return 256;
  const int nb = (int)((d + 8 * G - 1) / (8 * G));
  return 256 * (nb == 1 ? 5 : nb == 2 ? 3 : 2);
}

template <int ES, int EA>
hipError_t launch_addnorm_fwd_rows(const AddNormParams& p, unsigned wg, hipStream_t st) {
#define RP_CASE(G, NB)                                                                          \
  if (p.d <= G * NB * 8) {                                                                      \
    hipLaunchKernelGGL((addnorm_fwd_rows_kernel<ES, EA, G, NB>), dim3(wg), dim3(norm_threads(G)), 0, \
                       st, p);                                                                  \
    return hipGetLastError();                                                                   \
  }
  RP_FOR_EACH_ADDNORM_SHAPE(RP_CASE)
#undef RP_CASE
  return hipErrorInvalidValue;
}

template <int ES, int EO, int ED>
hipError_t launch_addnorm_bwd_rows(const AddNormParams& p, const AddNormGrad& g, unsigned wg,
                                   hipStream_t st) {
#define RP_CASE(G, NB)                                                                    \
  if (p.d <= G * NB * 8) {                                                                \
    hipLaunchKernelGGL((addnorm_bwd_rows_kernel<ES, EO, ED, G, NB>), dim3(wg),                \
                       dim3(norm_threads(G)), 0, st, p, g);                               \
    return hipGetLastError();                                                             \
  }
  RP_FOR_EACH_ADDNORM_SHAPE(RP_CASE)
#undef RP_CASE
  return hipErrorInvalidValue;
}

// The instantiations, one file each: element sizes of the rows and of add; of the rows,
// of dout and of dsum.
#define RP_ADDNORM_FWD(ES, EA) \
  hipError_t launch_addnorm_fwd##ES##EA(const AddNormParams& p, unsigned wg, hipStream_t st)
#define RP_ADDNORM_BWD(ES, EO, ED)                                                                 \
  hipError_t launch_addnorm_bwd##ES##EO##ED(const AddNormParams& p, const AddNormGrad& g, unsigned wg, \
                                            hipStream_t st)
RP_ADDNORM_FWD(4, 4);
RP_ADDNORM_FWD(4, 2);
RP_ADDNORM_FWD(2, 4);
RP_ADDNORM_FWD(2, 2);
RP_ADDNORM_FWD(1, 2);
RP_ADDNORM_BWD(4, 4, 4);
RP_ADDNORM_BWD(4, 2, 4);
RP_ADDNORM_BWD(2, 4, 2);
RP_ADDNORM_BWD(2, 2, 2);
RP_ADDNORM_BWD(1, 4, 4);
RP_ADDNORM_BWD(1, 4, 2);
RP_ADDNORM_BWD(1, 2, 4);
RP_ADDNORM_BWD(1, 2, 2);

}  // namespace rp
