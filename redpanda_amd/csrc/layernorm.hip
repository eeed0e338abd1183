// Layer norm over the last dimension, with GELU on the way in and dropout on
// the way out folded in (the middle of a head: Linear -> GELU -> LayerNorm ->
// dropout -> Linear), and its backward pass.  With h = x or GELU(x), per row:
//     mu = mean(h),  r = 1 / sqrt(mean((h - mu)^2) + eps),  xh = (h - mu) r
//     out = k s (xh w + b)                 k the dropout's mask, s its scale
// and for the output's gradient go:
//     g = k s go,  q = g w,  db = sum g,  dw = sum g xh        (over the rows)
//     dx = r (q - mean(q) - xh mean(q xh)) [GELU'(x)]
// The mask is drawn again and h, xh are formed again from x and the row's (mu,
// r), so nothing of the rows' size is kept between the passes.  All sums in
// fp32 or wider; the variance from the centred values (a second look at the
// row), since a mean of squares would cancel for rows far from zero.

#include "layernorm_rows.h"

namespace rp {

namespace {

// Sum over the workgroup; every thread gets it.  `buf` holds a float a wave and
// is free again for the next call after it.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = wave_sum(v);
  __syncthreads();
  if (threadIdx.x % kWave == 0) buf[threadIdx.x / kWave] = v;
  __syncthreads();
  float s = buf[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) s += buf[i];
  return s;
}

__device__ __forceinline__ void load_weights(const float* w, int64_t col, int64_t d, float dflt,
                                             float (&v)[8]) {
  if (w != nullptr) {
    load8(w, col, d, RP_F32, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = dflt;
  }
}

}  // namespace

// One workgroup per row, any length (for rows beyond the shapes of
// layernorm_rows.h).
__global__ __launch_bounds__(kThreads) void layernorm_fwd_kernel(LayerNormParams p) {
  __shared__ float buf[kWaves];
  const uint64_t seed = drop_seed(p.drop);
  const float invd = 1.f / (float)p.d;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const char* x = static_cast<const char*>(p.x) + row * p.xsr * p.es_x;
    auto load_h = [&](int64_t col, float (&h)[8]) {
      load8(x, col, p.d, p.dt_x, h);
      if (p.gelu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = gelu_of(h[i], gelu_parts(h[i]));
      }
    };
    float s = 0.f;
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float h[8];
      load_h(col, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += h[i];
    }
    const float mu = block_sum(s, buf) * invd;
    s = 0.f;
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float h[8];
      load_h(col, h);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < p.d) s = ffma(h[i] - mu, h[i] - mu, s);
    }
    const float r = rsqrtf(block_sum(s, buf) * invd + p.eps);
    if (threadIdx.x == 0 && p.stats != nullptr) {
      p.stats[2 * row] = mu;
      p.stats[2 * row + 1] = r;
    }
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float h[8], w[8], b[8];
      load_h(col, h);
      load_weights(p.w, col, p.d, 1.f, w);
      load_weights(p.b, col, p.d, 0.f, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = ffma((h[i] - mu) * r, w[i], b[i]);
      if (p.drop.t != 0) {
        const DropWords m = drop_words((uint32_t)(col / 8), (uint64_t)row, p.drop.stream, seed);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = drop_keep(m, i, p.drop.t) ? h[i] * p.drop.scale : 0.f;
      }
      store8(static_cast<char*>(p.out) + row * p.d * p.es_out, col, p.d, p.dt_out, h);
    }
  }
}

namespace {

// g (after the mask) and x of eight columns of a row, and from them xh and
// GELU'(x) (1 without GELU).
__device__ __forceinline__ void load_grad(const LayerNormParams& p, const LayerNormGrad& g,
                                          uint64_t seed, int64_t row, int64_t col, float mu, float r,
                                          float (&go)[8], float (&xh)[8], float (&slope)[8]) {
  load8(static_cast<const char*>(g.dout) + row * g.dosr * p.es_out, col, p.d, p.dt_out, go);
  load8(static_cast<const char*>(p.x) + row * p.xsr * p.es_x, col, p.d, p.dt_x, xh);
  if (p.drop.t != 0) {
    const DropWords m = drop_words((uint32_t)(col / 8), (uint64_t)row, p.drop.stream, seed);
#pragma unroll
    for (int i = 0; i < 8; ++i) go[i] = drop_keep(m, i, p.drop.t) ? go[i] * p.drop.scale : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    slope[i] = 1.f;
    if (p.gelu) gelu_both(xh[i], xh[i], slope[i]);
    xh[i] = (xh[i] - mu) * r;
  }
}

}  // namespace

__global__ __launch_bounds__(kThreads) void layernorm_dx_kernel(LayerNormParams p, LayerNormGrad g) {
  __shared__ float buf[kWaves];
  const uint64_t seed = drop_seed(p.drop);
  const float invd = 1.f / (float)p.d;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mu = p.stats[2 * row], r = p.stats[2 * row + 1];
    float s = 0.f, sx = 0.f;
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float go[8], xh[8], sl[8], w[8];
      load_grad(p, g, seed, row, col, mu, r, go, xh, sl);
      load_weights(p.w, col, p.d, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (col + i >= p.d) break;
        const float q = go[i] * w[i];
        s += q;
        sx = ffma(q, xh[i], sx);
      }
    }
    s = block_sum(s, buf) * invd;
    sx = block_sum(sx, buf) * invd;
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float go[8], xh[8], sl[8], w[8];
      load_grad(p, g, seed, row, col, mu, r, go, xh, sl);
      load_weights(p.w, col, p.d, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) go[i] = (r * (ffma(go[i], w[i], -s) - xh[i] * sx)) * sl[i];
      store8(static_cast<char*>(g.dx) + row * p.d * p.es_x, col, p.d, p.dt_x, go);
    }
  }
}

// Column sums of g xh and g: workgroup (x, y) takes the columns of 64 blocks
// and every gridDim.y-th group of 4 rows, a wave one row at a time; the partial
// sums go to part[y][0: dw, 1: db][d].
__global__ __launch_bounds__(kThreads) void layernorm_dw_kernel(LayerNormParams p, LayerNormGrad g) {
  __shared__ float buf[kWaves][kWave * 16];
  const uint64_t seed = drop_seed(p.drop);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t col = ((int64_t)blockIdx.x * kWave + lane) * 8;
  float dw[8] = {}, db[8] = {};
  if (col < p.d) {
    for (int64_t row = (int64_t)blockIdx.y * kWaves + wave; row < p.rows;
         row += (int64_t)gridDim.y * kWaves) {
      float go[8], xh[8], sl[8];
      load_grad(p, g, seed, row, col, p.stats[2 * row], p.stats[2 * row + 1], go, xh, sl);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[i] = ffma(go[i], xh[i], dw[i]);
        db[i] += go[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    buf[wave][i * kWave + lane] = dw[i];
    buf[wave][(8 + i) * kWave + lane] = db[i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kWave * 16; e += kThreads) {
    const int64_t c = ((int64_t)blockIdx.x * kWave + e % kWave) * 8 + e / kWave % 8;
    if (c >= p.d) continue;
    g.part[((int64_t)blockIdx.y * 2 + e / (8 * kWave)) * p.d + c] =
        (buf[0][e] + buf[1][e]) + (buf[2][e] + buf[3][e]);
  }
}

// dw, db: the n partial sums of each column, in fp64 and in a fixed order: 16
// waves take every 16th of them for 64 columns, then one adds the waves'.
__global__ __launch_bounds__(16 * kWave) void layernorm_sum_kernel(const float* part, int n, int64_t d,
                                                                   float* dw, float* db) {
  __shared__ double buf[16][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t c = (int64_t)blockIdx.x * kWave + lane;
  double s = 0.0;
  if (c < 2 * d) {
    const float* at = part + c;
    int i = wave;
    for (; i + 7 * 16 < n; i += 8 * 16) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = at[(int64_t)(i + 16 * k) * 2 * d];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; i < n; i += 16) s += at[(int64_t)i * 2 * d];
  }
  buf[wave][lane] = s;
  __syncthreads();
  if (wave > 0 || c >= 2 * d) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += buf[w][lane];
  (c < d ? dw : db)[c < d ? c : c - d] = (float)s;
}

namespace {

unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

// Workgroups of a launch whose groups of G lanes walk rows.
unsigned walk_grid(int64_t rows, int G, int most) {
  const int groups = norm_threads(G) / G;
  const int64_t n = (rows + groups - 1) / groups;
  return (unsigned)(n < most ? n : most);
}

}  // namespace

int layernorm_parts(int64_t rows, int64_t d, int es_x, int es_out) {
  const int G = norm_group(d);
  if (G != 0) return (int)walk_grid(rows, G, norm_workgroups_bwd(d, es_x, es_out));
  const int64_t tiles = (d + 8 * kWave - 1) / (8 * kWave);
  const int64_t n = (rows + 4 * kWaves - 1) / (4 * kWaves);
  const int64_t most = (2048 + tiles - 1) / tiles;
  return (int)(n < most ? n : most);
}

hipError_t launch_layernorm_fwd(const LayerNormParams& p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  const int G = norm_group(p.d);
  if (G != 0) {
    const unsigned wg = walk_grid(p.rows, G, norm_workgroups_fwd(p.d));
    return p.es_x == 4 ? launch_norm_fwd4(p, wg, st) : launch_norm_fwd2(p, wg, st);
  }
  hipLaunchKernelGGL(layernorm_fwd_kernel, dim3(row_grid(p.rows)), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_layernorm_bwd(const LayerNormParams& p, const LayerNormGrad& g, hipStream_t st) {
  const int n = layernorm_parts(p.rows, p.d, p.es_x, p.es_out);
  if (p.rows > 0 && norm_group(p.d) != 0) {
    auto* launch = p.es_x == 4 ? (p.es_out == 4 ? launch_norm_bwd44 : launch_norm_bwd42)
                               : (p.es_out == 4 ? launch_norm_bwd24 : launch_norm_bwd22);
    const hipError_t e = launch(p, g, (unsigned)n, st);
    if (e != hipSuccess) return e;
  } else if (p.rows > 0) {
    if (g.dx != nullptr)
      hipLaunchKernelGGL(layernorm_dx_kernel, dim3(row_grid(p.rows)), dim3(kThreads), 0, st, p, g);
    if (g.dw != nullptr)
      hipLaunchKernelGGL(layernorm_dw_kernel, dim3((unsigned)((p.d + 8 * kWave - 1) / (8 * kWave)), n),
                         dim3(kThreads), 0, st, p, g);
  }
  if (g.dw != nullptr)
    hipLaunchKernelGGL(layernorm_sum_kernel, dim3((unsigned)((2 * p.d + kWave - 1) / kWave)),
                       dim3(16 * kWave), 0, st, g.part, n, p.d, g.dw, g.db);
  return hipGetLastError();
}

}  // namespace rp
