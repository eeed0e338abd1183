// RMS norm with the residual's addition, for training: with s = x [+ add] (rounded to
// its own type first, as the stream is kept), per row
//     r = 1 / sqrt(mean(s^2) + eps),  xh = s r,  out = xh w
// and for the gradients go of out and gs of s:
//     q = go w,  ds = gs + r (q - xh mean(q xh)),  dw = sum over the rows of go xh
// r is formed again in the backward, from the same look at the row that the mean of
// q xh takes, so the stream s is all that is kept between the passes; or s in 8 bits
// (rp_pack8.h), which the forward writes beside the rest and the backward takes in
// its place: the gradient is then exact for the values that were kept.  All sums in
// fp32 or wider.
//
// Rows of up to 16384 columns are held in registers (addnorm_rows.h); longer ones are
// read again for each use, here.

#include "addnorm_rows.h"

namespace rp {

namespace {

// Sum over the workgroup; every thread gets it.  `buf` holds a float a wave.
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

__device__ __forceinline__ void load_w(const float* w, int64_t col, int64_t d, float (&v)[8]) {
  if (w != nullptr) {
    load8(w, col, d, RP_F32, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 1.f;
  }
}

// Eight columns of the rows s that a backward reads.
__device__ __forceinline__ void load_s(const AddNormParams& p, int64_t row, int64_t col,
                                       float (&v)[8]) {
  if (p.x != nullptr) {
    load8(static_cast<const char*>(p.x) + row * p.xsr * p.es_sum, col, p.d, p.dt_sum, v);
  } else {
    uint32_t q[2];
    load_q8(p.q8 + row * p.d, col, p.d, q);
    unpack_block(q, p.e8[row * ((p.d + kPackBlock - 1) / kPackBlock) + col / kPackBlock], p.dt_sum, v);
  }
}

}  // namespace

// One workgroup per row, any length (for rows beyond the shapes of addnorm_rows.h).
__global__ __launch_bounds__(kThreads) void addnorm_fwd_kernel(AddNormParams p) {
  __shared__ float buf[kWaves];
  const float invd = 1.f / (float)p.d;
  const int64_t ne = (p.d + kPackBlock - 1) / kPackBlock;
  const int64_t lanes = ne * 4;  // whole quads
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    auto load = [&](int64_t col, float (&v)[8]) {
      if (p.x == nullptr) {
        load_s(p, row, col, v);
        return;
      }
      load8(static_cast<const char*>(p.x) + row * p.xsr * p.es_x, col, p.d, p.dt_x, v);
      if (p.add != nullptr) {
        float a[8];
        load8(static_cast<const char*>(p.add) + row * p.asr * p.es_add, col, p.d, p.dt_add, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += a[i];
        round_to(p.dt_sum, v);
      }
    };
    float s = 0.f;
    for (int64_t at = threadIdx.x; at < lanes; at += kThreads) {
      const int64_t col = at * 8;
      float v[8] = {};
      if (col < p.d) load(col, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = ffma(v[i], v[i], s);
      if (p.x == nullptr) continue;
      if (p.sum != nullptr && col < p.d)
        store8(static_cast<char*>(p.sum) + row * p.d * p.es_sum, col, p.d, p.dt_sum, v);
      if (p.q8 != nullptr) {
        uint32_t q[2];
        const uint32_t e = pack_block(v, q);
        if (col < p.d) store_q8(p.q8 + row * p.d, col, p.d, q);
        if (at % 4 == 0) p.e8[row * ne + at / 4] = (uint8_t)e;
      }
    }
    if (p.out == nullptr) continue;
    const float r = rsqrtf(ffma(block_sum(s, buf), invd, p.eps));
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float v[8], w[8];
      load(col, v);
      load_w(p.w, col, p.d, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (v[i] * r) * w[i];
      store8(static_cast<char*>(p.out) + row * p.d * p.es_out, col, p.d, p.dt_out, v);
    }
  }
}

// The same for the backward; each row's r goes to rstd, for the sums over the rows.
__global__ __launch_bounds__(kThreads) void addnorm_ds_kernel(AddNormParams p, AddNormGrad g,
                                                              float* rstd) {
  __shared__ float buf[kWaves];
  const float invd = 1.f / (float)p.d;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const char* go = static_cast<const char*>(g.dout) + row * g.dosr * p.es_out;
    float ss = 0.f, sq = 0.f;
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float v[8], q[8], w[8];
      load_s(p, row, col, v);
      load8(go, col, p.d, p.dt_out, q);
      load_w(p.w, col, p.d, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss = ffma(v[i], v[i], ss);
        sq = ffma(q[i] * w[i], v[i], sq);
      }
    }
    const float r = rsqrtf(ffma(block_sum(ss, buf), invd, p.eps));
    const float m = r * block_sum(sq, buf) * invd;
    if (threadIdx.x == 0) rstd[row] = r;
    if (g.dx == nullptr && g.dadd == nullptr) continue;
    for (int64_t col = threadIdx.x * 8; col < p.d; col += kThreads * 8) {
      float v[8], q[8], w[8], d[8] = {};
      load_s(p, row, col, v);
      load8(go, col, p.d, p.dt_out, q);
      load_w(p.w, col, p.d, w);
      if (g.dsum != nullptr)
        load8(static_cast<const char*>(g.dsum) + row * g.dssr * p.es_sum, col, p.d, p.dt_sum, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = ffma(ffma(-(v[i] * r), m, q[i] * w[i]), r, d[i]);
      if (g.dx != nullptr)
        store8(static_cast<char*>(g.dx) + row * p.d * p.es_x, col, p.d, p.dt_x, d);
      if (g.dadd != nullptr)
        store8(static_cast<char*>(g.dadd) + row * p.d * p.es_add, col, p.d, p.dt_add, d);
    }
  }
}

// Column sums of go xh: workgroup (x, y) takes the columns of 64 blocks of eight and
// every gridDim.y-th group of 4 rows, a wave one row at a time.
__global__ __launch_bounds__(kThreads) void addnorm_dw_kernel(AddNormParams p, AddNormGrad g,
                                                              const float* rstd) {
  __shared__ float buf[kWaves][kWave * 8];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t col = ((int64_t)blockIdx.x * kWave + lane) * 8;
  float dw[8] = {};
  if (col < p.d) {
    for (int64_t row = (int64_t)blockIdx.y * kWaves + wave; row < p.rows;
         row += (int64_t)gridDim.y * kWaves) {
      float v[8], q[8];
      load_s(p, row, col, v);
      load8(static_cast<const char*>(g.dout) + row * g.dosr * p.es_out, col, p.d, p.dt_out, q);
      const float r = rstd[row];
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[i] = ffma(q[i], v[i] * r, dw[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) buf[wave][i * kWave + lane] = dw[i];
  __syncthreads();
  for (int e = threadIdx.x; e < kWave * 8; e += kThreads) {
    const int64_t c = ((int64_t)blockIdx.x * kWave + e % kWave) * 8 + e / kWave;
    if (c < p.d)
      g.part[(int64_t)blockIdx.y * p.d + c] = (buf[0][e] + buf[1][e]) + (buf[2][e] + buf[3][e]);
  }
}

// dw: the n partial sums of each column, in fp64 and in a fixed order: 16 waves take
// every 16th of them for 64 columns, then one adds the waves'.
__global__ __launch_bounds__(16 * kWave) void addnorm_sum_kernel(const float* part, int n, int64_t d,
                                                                 float* dw) {
  __shared__ double buf[16][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t c = (int64_t)blockIdx.x * kWave + lane;
  double s = 0.0;
  if (c < d) {
    const float* at = part + c;
    int i = wave;
    for (; i + 7 * 16 < n; i += 8 * 16) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = at[(int64_t)(i + 16 * k) * d];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; i < n; i += 16) s += at[(int64_t)i * d];
  }
  buf[wave][lane] = s;
  __syncthreads();
  if (wave > 0 || c >= d) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += buf[w][lane];
  dw[c] = (float)s;
}

namespace {

unsigned row_grid(int64_t rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

// Workgroups of a launch whose groups of G lanes walk rows: as few as walk as many rows
// each as `most` would.
unsigned walk_grid(int64_t rows, int G, int most) {
  const int groups = norm_threads(G) / G;
  const int64_t n = (rows + groups - 1) / groups, turns = (n + most - 1) / most;
  return (unsigned)(turns > 0 ? (n + turns - 1) / turns : 0);
}

}  // namespace

static int addnorm_parts(int64_t rows, int64_t d) {
  const int G = addnorm_group(d);
  if (G != 0) return (int)walk_grid(rows, G, addnorm_workgroups_bwd(d));
  const int64_t tiles = (d + 8 * kWave - 1) / (8 * kWave);
  const int64_t n = (rows + 4 * kWaves - 1) / (4 * kWaves);
  const int64_t most = (2048 + tiles - 1) / tiles;
  return (int)(n < most ? n : most);
}

int64_t addnorm_work_floats(int64_t rows, int64_t d) {
  return (int64_t)addnorm_parts(rows, d) * d + (addnorm_group(d) == 0 ? rows : 0);
}

hipError_t launch_addnorm_fwd(const AddNormParams& p, hipStream_t st) {
  if (p.rows == 0) return hipSuccess;
  const int G = addnorm_group(p.d);
  if (G != 0) {
    const unsigned wg = walk_grid(p.rows, G, addnorm_workgroups_fwd(p.d));
    if (p.x == nullptr) return launch_addnorm_fwd12(p, wg, st);
    auto* launch = p.es_x == 4 ? (p.es_add == 4 ? launch_addnorm_fwd44 : launch_addnorm_fwd42)
                               : (p.es_add == 4 ? launch_addnorm_fwd24 : launch_addnorm_fwd22);
    return launch(p, wg, st);
  }
  hipLaunchKernelGGL(addnorm_fwd_kernel, dim3(row_grid(p.rows)), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_addnorm_bwd(const AddNormParams& p, const AddNormGrad& g, hipStream_t st) {
  const int es_s = p.x == nullptr ? 1 : p.es_sum;
  const int n = addnorm_parts(p.rows, p.d);
  if (p.rows > 0 && addnorm_group(p.d) != 0) {
    auto* launch = es_s == 4   ? (p.es_out == 4 ? launch_addnorm_bwd444 : launch_addnorm_bwd424)
                   : es_s == 2 ? (p.es_out == 4 ? launch_addnorm_bwd242 : launch_addnorm_bwd222)
                   : p.es_sum == 4 ? (p.es_out == 4 ? launch_addnorm_bwd144 : launch_addnorm_bwd124)
                                   : (p.es_out == 4 ? launch_addnorm_bwd142 : launch_addnorm_bwd122);
    const hipError_t e = launch(p, g, (unsigned)n, st);
    if (e != hipSuccess) return e;
  } else if (p.rows > 0) {
    float* rstd = g.part + (int64_t)n * p.d;
    hipLaunchKernelGGL(addnorm_ds_kernel, dim3(row_grid(p.rows)), dim3(kThreads), 0, st, p, g, rstd);
    if (g.dw != nullptr)
      hipLaunchKernelGGL(addnorm_dw_kernel, dim3((unsigned)((p.d + 8 * kWave - 1) / (8 * kWave)), n),
                         dim3(kThreads), 0, st, p, g, rstd);
  }
  if (g.dw != nullptr)
    hipLaunchKernelGGL(addnorm_sum_kernel, dim3((unsigned)((p.d + kWave - 1) / kWave)),
                       dim3(16 * kWave), 0, st, g.part, n, p.d, g.dw);
  return hipGetLastError();
}

}  // namespace rp
