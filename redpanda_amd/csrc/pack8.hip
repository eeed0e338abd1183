// Rows to 8 bits and back (the format is described in rp_pack8.h): one thread per
// eight columns, four adjacent threads a block of 32.  HBM bounds both (131072 x 1024
// bf16: 88 us there and 83 back, 79 each at the rate of a large copy; 16384 x 768 fp32 11
// and 13).

#include "rp_pack8.h"
#include "rp_train.h"

namespace rp {

namespace {

// Threads of a row: whole quads, so that a block's lanes are adjacent.
__host__ __device__ __forceinline__ int64_t quad_lanes(int64_t d) { return (d + 31) / 32 * 4; }

__device__ __forceinline__ int64_t row_of(int64_t e, int64_t n, int64_t lanes) {
  return n <= 0xffffffffll ? (int64_t)((uint32_t)e / (uint32_t)lanes) : e / lanes;
}

}  // namespace

__global__ __launch_bounds__(kThreads) void pack8_kernel(Pack8Params p) {
  const int64_t lanes = quad_lanes(p.d), n = p.rows * lanes;
  // (n and the step are multiples of four: a quad stays together)
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * kThreads) {
    const int64_t row = row_of(e, n, lanes), at = e - row * lanes, col = at * 8;
    float v[8] = {};
    if (col < p.d) load8(static_cast<const char*>(p.x) + row * p.xsr * p.es, col, p.d, p.dt, v);
    uint32_t q[2];
    const uint32_t b = pack_block(v, q);
    if (col < p.d) store_q8(p.q8 + row * p.d, col, p.d, q);
    if (at % 4 == 0) p.e8[(row * lanes + at) / 4] = (uint8_t)b;
  }
}

__global__ __launch_bounds__(kThreads) void unpack8_kernel(Pack8Params p) {
  const int64_t lanes = quad_lanes(p.d), n = p.rows * lanes;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * kThreads) {
    const int64_t row = row_of(e, n, lanes), at = e - row * lanes, col = at * 8;
    if (col >= p.d) continue;
    uint32_t q[2];
    float v[8];
    load_q8(p.q8 + row * p.d, col, p.d, q);
    unpack_block(q, p.e8[(row * lanes + at) / 4], p.dt_held, v);
    store8(static_cast<char*>(p.x) + row * p.xsr * p.es, col, p.d, p.dt, v);
  }
}

namespace {
dim3 pack_grid(const Pack8Params& p) {
  const int64_t wg = (p.rows * quad_lanes(p.d) + kThreads - 1) / kThreads;
  return dim3((unsigned)(wg < (1 << 20) ? wg : (1 << 20)));
}
}  // namespace

hipError_t launch_pack8(const Pack8Params& p, hipStream_t st) {
  if (p.rows * p.d == 0) return hipSuccess;
  hipLaunchKernelGGL(pack8_kernel, pack_grid(p), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_unpack8(const Pack8Params& p, hipStream_t st) {
  if (p.rows * p.d == 0) return hipSuccess;
  hipLaunchKernelGGL(unpack8_kernel, pack_grid(p), dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace rp
