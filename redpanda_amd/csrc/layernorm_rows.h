// Layer norm kernels that hold their rows in registers: one read of each row a
// pass.  (The mathematics is in layernorm.hip.)
//
// A row is taken by a group of G lanes, each holding NB blocks of eight columns
// (block g + G j for lane g), so G NB blocks are the most a row may have; the
// launcher takes the shape with the fewest spare ones.  G is a part of a wave (8,
// 16, 32, or all 64 lanes: narrow rows share a wave, and sums over a group are a
// few lane exchanges without LDS), or several waves of one workgroup.  Only the
// last of a lane's blocks can be past the row or cut by its end.
//
// A group walks rows a grid apart, the next row's loads issued before the
// present one is worked on; its columns stay, so the weights are read once, the
// backward keeps the columns' sums in registers over all its rows, and the
// generator's first products, which depend on the column alone, leave the loop.
//
// 131072 x 1024 in bf16: without GELU and dropout 93 us forward (5.8 TB/s) and 150
// backward (5.4), which HBM bounds; with both 151 and 217, which vector
// instructions bound (31 and 41 an element: GELU 16 forward and 21 backward, the
// generator 5).  16384 x 768, bf16 in and fp32 out, no GELU: 18 and 22 us; fp32 both
// 18 and 29.  A few rows are a launch's latency: one row of 384 3.9 us, 512 x 768
// fp32 with both 5.6 and 8.3, and 3.4 for the partial sums.  Rows of 8193 to 16384
// fall behind: their 1024 lanes have 128 registers each, the backward spills 46 to
// 88 of what it keeps (8192 x 9000 with both: fp32 189 and 335 us, bf16 139 and 447).
#pragma once

#include "rp_heads.h"
#include "rp_rows.h"

namespace rp {

constexpr int norm_threads(int G) { return G > kThreads ? G : kThreads; }

template <int kCtrl>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xf, 0xf, true));
}

// Sum over groups of G adjacent lanes (8 .. 64) of a wave, each lane the same.
template <int G>
__device__ __forceinline__ float lane_sum(float v) {
  v += dpp_f<0xb1>(v);   // quad_perm [1, 0, 3, 2]
  v += dpp_f<0x4e>(v);   // quad_perm [2, 3, 0, 1]
  v += dpp_f<0x141>(v);  // row_half_mirror: the other four of eight
  if constexpr (G >= 16) v += dpp_f<0x140>(v);  // row_mirror: the other eight
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// Sums of N values over a group; beyond a wave through LDS, `buf` being free
// again after the next barrier.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*buf)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum<(G < kWave ? G : kWave)>(v[i]);
  if constexpr (G > kWave) {
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = buf[0][i];
#pragma unroll
      for (int w = 1; w < G / kWave; ++w) v[i] += buf[w][i];
    }
  }
}

// A lane's blocks of the columns.
template <int G, int NB>
struct NormCols {
  int col[NB];
  int d;
  bool any;   // the last block holds columns of the row
  bool cut;   // the row's length is no multiple of eight (the same in every lane)

  __device__ __forceinline__ NormCols(int g, int64_t dd) {
    d = (int)dd;
#pragma unroll
    for (int j = 0; j < NB; ++j) col[j] = (g + G * j) * 8;
    any = col[NB - 1] < d;
    cut = d % 8 != 0;
  }
  template <int ES>
  __device__ __forceinline__ void load(const char* row, Raw8<ES> (&r)[NB]) const {
#pragma unroll
    for (int j = 0; j + 1 < NB; ++j) r[j] = load_full8<ES>(row, col[j]);
    if (cut) {
      r[NB - 1] = load_raw8<ES>(row, col[NB - 1], d);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * ES; ++i) r[NB - 1].w[i] = 0;
      if (any) r[NB - 1] = load_full8<ES>(row, col[NB - 1]);
    }
  }
  __device__ __forceinline__ void load_weight(const float* w, float dflt, float mul,
                                              float (&v)[NB][8]) const {
    Raw8<4> r[NB];
    if (w != nullptr) load<4>(reinterpret_cast<const char*>(w), r);
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = (w != nullptr ? __uint_as_float(r[j].w[i]) : dflt) * mul;
  }
  __device__ __forceinline__ void store(char* row, int dtype, const float (&v)[NB][8]) const {
#pragma unroll
    for (int j = 0; j + 1 < NB; ++j) store_full8(row, col[j], dtype, v[j]);
    if (cut)
      store8(row, col[NB - 1], d, dtype, v[NB - 1]);
    else if (any)
      store_full8(row, col[NB - 1], dtype, v[NB - 1]);
  }
};

// The seed and thresholds, in scalar registers.
struct DropState {
  uint64_t seed;
  uint32_t stream, lo, hi;
  __device__ __forceinline__ DropState(const DropParams& d) {
    seed = drop_seed(d);
    stream = d.stream;
    lo = d.t - 1;
    hi = (d.t << 16) - 1;
  }
  // v[i] = kept ? v[i] : 0 for a block
  __device__ __forceinline__ void apply(uint32_t block, uint64_t row, float (&v)[8]) const {
    const DropWords m = drop_words(block, row, stream, seed);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = (uint16_t)m.w[i] > (uint16_t)lo ? v[2 * i] : 0.f;
      v[2 * i + 1] = m.w[i] > hi ? v[2 * i + 1] : 0.f;
    }
  }
};

template <int G>
struct NormRows {
  int64_t row, step;
  int g;
  __device__ __forceinline__ NormRows() {
    constexpr int kGroups = norm_threads(G) / G;
    g = threadIdx.x % G;
    int group = threadIdx.x / G;
    if constexpr (G >= kWave) group = __builtin_amdgcn_readfirstlane(group);
    row = (int64_t)blockIdx.x * kGroups + group;
    step = (int64_t)gridDim.x * kGroups;
  }
};

template <int ES, int G, int NB>
__global__ __launch_bounds__(norm_threads(G)) void layernorm_fwd_rows_kernel(LayerNormParams p) {
  constexpr int kW = G > kWave ? G / kWave : 1;
  __shared__ float buf[2][kW][1];
  NormRows<G> at;
  if (at.row >= p.rows) return;  // (whole workgroups where they share a row)
  const NormCols<G, NB> cols(at.g, p.d);
  const DropState drop(p.drop);
  const float scale = p.drop.t != 0 ? p.drop.scale : 1.f;
  const float invd = 1.f / (float)cols.d;
  float w[NB][8], b[NB][8];
  cols.load_weight(p.w, 1.f, scale, w);
  cols.load_weight(p.b, 0.f, scale, b);
  const char* x = static_cast<const char*>(p.x);
  Raw8<ES> raw[NB];
  cols.template load<ES>(x + at.row * p.xsr * ES, raw);
  for (; at.row < p.rows; at.row += at.step) {
    float h[NB][8];
#pragma unroll
    for (int j = 0; j < NB; ++j) to_floats(raw[j], p.dt_x, h[j]);
    if (at.row + at.step < p.rows) cols.template load<ES>(x + (at.row + at.step) * p.xsr * ES, raw);
    if (p.gelu) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] = gelu_of(h[j][i], gelu_parts(h[j][i]));
    }
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] += h[j][i];  // (0 past the row)
    group_sum<G>(s, buf[0]);
    const float mu = s[0] * invd;
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] -= mu;
      if (j + 1 < NB || cols.any) {
        if (j + 1 == NB && cols.cut) {
#pragma unroll
          for (int i = 0; i < 8; ++i) h[j][i] = cols.col[j] + i < cols.d ? h[j][i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] = ffma(h[j][i], h[j][i], s[0]);
      }
    }
    group_sum<G>(s, buf[1]);
    const float r = rsqrtf(ffma(s[0], invd, p.eps));
    if (p.stats != nullptr && at.g == 0) {
      p.stats[2 * at.row] = mu;
      p.stats[2 * at.row + 1] = r;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = ffma(h[j][i] * r, w[j][i], b[j][i]);
      if (p.drop.t != 0) drop.apply((uint32_t)(at.g + G * j), (uint64_t)at.row, h[j]);
    }
    cols.store(static_cast<char*>(p.out) + at.row * p.d * p.es_out, p.dt_out, h);
  }
}

// dx, and the workgroup's sums of g xh and g over its rows to part[workgroup].
template <int ES, int EO, int G, int NB>
__global__ __launch_bounds__(norm_threads(G)) void layernorm_bwd_rows_kernel(LayerNormParams p,
                                                                             LayerNormGrad g) {
  constexpr int kW = G > kWave ? G / kWave : 1;
  constexpr int kGroups = norm_threads(G) / G;
  __shared__ float buf[2][kW][2];
  NormRows<G> at;
  const NormCols<G, NB> cols(at.g, p.d);
  const DropState drop(p.drop);
  const float scale = p.drop.t != 0 ? p.drop.scale : 1.f;
  const float invd = 1.f / (float)cols.d;
  // 1024 threads have 128 registers each: there the weights are read for each
  // row, and no row ahead
  constexpr bool kAhead = G < 1024;
  float w[NB][8], dw[NB][8] = {}, db[NB][8] = {};
  if constexpr (kAhead) cols.load_weight(p.w, 1.f, 1.f, w);
  const char* x = static_cast<const char*>(p.x);
  const char* go = static_cast<const char*>(g.dout);
  Raw8<ES> rx[NB];
  Raw8<EO> rg[NB];
  float mu = 0.f, r = 0.f;
  auto load = [&](int64_t row) {
    cols.template load<ES>(x + row * p.xsr * ES, rx);
    cols.template load<EO>(go + row * g.dosr * EO, rg);
    mu = p.stats[2 * row];
    r = p.stats[2 * row + 1];
  };
  if (kAhead && at.row < p.rows) load(at.row);
  for (int it = 0; at.row < p.rows; at.row += at.step, it ^= 1) {
    if constexpr (!kAhead) load(at.row);
    float xh[NB][8], q[NB][8], slope[NB][8];
    const float r0 = r, shift = -mu * r, rs = r * scale;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      to_floats(rx[j], p.dt_x, xh[j]);
      to_floats(rg[j], p.dt_out, q[j]);
    }
    if (kAhead && at.row + at.step < p.rows) load(at.row + at.step);
    if (p.drop.t != 0) {
#pragma unroll
      for (int j = 0; j < NB; ++j) drop.apply((uint32_t)(at.g + G * j), (uint64_t)at.row, q[j]);
    }
    if (p.gelu) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          gelu_both(xh[j][i], xh[j][i], slope[j][i]);
          slope[j][i] *= rs;
        }
    } else {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) slope[j][i] = rs;
    }
    if constexpr (!kAhead) {
      const float* pw = p.w;
      asm volatile("" : "+s"(pw));
      cols.load_weight(pw, 1.f, 1.f, w);
    }
    // (the dropout's scale is in rs, and at the end in dw and db)
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xh[j][i] = ffma(xh[j][i], r0, shift);
        // past the row the gradient is 0 and adds nothing
        dw[j][i] = ffma(q[j][i], xh[j][i], dw[j][i]);
        db[j][i] += q[j][i];
        q[j][i] *= w[j][i];
        s[0] += q[j][i];
        s[1] = ffma(q[j][i], xh[j][i], s[1]);
      }
    group_sum<G>(s, buf[it]);
    const float m1 = s[0] * invd, m2 = s[1] * invd;
    if (g.dx != nullptr) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[j][i] = ffma(-xh[j][i], m2, q[j][i] - m1) * slope[j][i];
      cols.store(static_cast<char*>(g.dx) + at.row * p.d * p.es_x, p.dt_x, q);
    }
  }
  if (g.dw == nullptr) return;
  // the groups' sums: over a wave's groups by lane exchanges, then wave by wave
  // through LDS in order
  float* part = g.part + (int64_t)blockIdx.x * 2 * p.d;
  __shared__ float cols_sum[kGroups > 1 ? 16 * NB : 1][kWave];
  if constexpr (kGroups > 1) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int m = G; m < kWave; m <<= 1) {
          dw[j][i] += __shfl_xor(dw[j][i], m);
          db[j][i] += __shfl_xor(db[j][i], m);
        }
      }
    for (int t = 0; t < kWaves; ++t) {
      if (wave == t) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float* a = &cols_sum[(2 * j) * 8 + i][lane];
            float* c = &cols_sum[(2 * j + 1) * 8 + i][lane];
            if (t > 0) {
              dw[j][i] += *a;
              db[j][i] += *c;
            }
            if (t + 1 < kWaves) {
              *a = dw[j][i];
              *c = db[j][i];
            }
          }
      }
      __syncthreads();
    }
    if (wave + 1 < kWaves || lane >= G) return;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[j][i] *= scale;
      db[j][i] *= scale;
    }
  cols.store(reinterpret_cast<char*>(part), RP_F32, dw);
  cols.store(reinterpret_cast<char*>(part + p.d), RP_F32, db);
}

// The shapes (G, NB), by the blocks they hold.
#define RP_FOR_EACH_NORM_SHAPE(X) \
  X(8, 1) X(16, 1) X(8, 3) X(32, 1) X(16, 3) X(64, 1) X(32, 3) X(64, 2) X(64, 3) X(256, 1) \
  X(256, 2) X(512, 2) X(1024, 2)

// Lanes a row of d columns is taken by, and its groups in a workgroup; 0 for
// rows longer than the largest shape.
inline int norm_group(int64_t d) {
#define RP_CASE(G, NB) \
  if (d <= G * NB * 8) return G;
  RP_FOR_EACH_NORM_SHAPE(RP_CASE)
#undef RP_CASE
  return 0;
}

// Workgroups that a launch of G lanes a row fills the card with: as many as its
// registers let be resident, since a second round of a part of them would cost
// as much as a whole one (131072 x 1024 backward: 1024 workgroups where 768 fit
// took a quarter longer).  The backward's registers go by the bytes of an element
// of x and of a gradient: with fp32 on both sides fewer fit (two blocks a lane
// 173 of them, three 262 or 252; backward of 131072 x 1024 309 us by 768
// workgroups, 278 by the 512 that fit; 16384 x 768 33 and 29).
inline int norm_workgroups_fwd(int64_t d) {
  const int G = norm_group(d);
  if (G > 256) return G == 1024 ? 256 : 512;
  const int nb = (int)((d + 8 * G - 1) / (8 * G));
  return 256 * (nb == 1 ? 7 : nb == 2 ? 5 : 3);
}
inline int norm_workgroups_bwd(int64_t d, int es_x, int es_out) {
  const int G = norm_group(d);
  if (G > 256) return 256;
  const int nb = (int)((d + 8 * G - 1) / (8 * G));
  const bool wide = es_x + es_out == 8 || (G == 256 && es_out == 4);
  return 256 * (nb == 1 ? 4 : nb == 2 ? (wide ? 2 : 3) : es_x + es_out == 8 && G < kWave ? 1 : 2);
}

template <int ES>
hipError_t launch_norm_fwd_rows(const LayerNormParams& p, unsigned wg, hipStream_t st) {
#define RP_CASE(G, NB)                                                                            \
  if (p.d <= G * NB * 8) {                                                                        \
    hipLaunchKernelGGL((layernorm_fwd_rows_kernel<ES, G, NB>), dim3(wg), dim3(norm_threads(G)), 0, \
                       st, p);                                                                    \
    return hipGetLastError();                                                                     \
  }
  RP_FOR_EACH_NORM_SHAPE(RP_CASE)
#undef RP_CASE
  return hipErrorInvalidValue;
}

template <int ES, int EO>
hipError_t launch_norm_bwd_rows(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg,
                                hipStream_t st) {
#define RP_CASE(G, NB)                                                                       \
  if (p.d <= G * NB * 8) {                                                                   \
    hipLaunchKernelGGL((layernorm_bwd_rows_kernel<ES, EO, G, NB>), dim3(wg),                 \
                       dim3(norm_threads(G)), 0, st, p, g);                                  \
    return hipGetLastError();                                                                \
  }
  RP_FOR_EACH_NORM_SHAPE(RP_CASE)
#undef RP_CASE
  return hipErrorInvalidValue;
}

// The instantiations, one file each (element sizes of x and of the gradient).
hipError_t launch_norm_fwd4(const LayerNormParams& p, unsigned wg, hipStream_t st);
hipError_t launch_norm_fwd2(const LayerNormParams& p, unsigned wg, hipStream_t st);
hipError_t launch_norm_bwd44(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg, hipStream_t st);
hipError_t launch_norm_bwd42(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg, hipStream_t st);
hipError_t launch_norm_bwd24(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg, hipStream_t st);
hipError_t launch_norm_bwd22(const LayerNormParams& p, const LayerNormGrad& g, unsigned wg, hipStream_t st);

}  // namespace rp
