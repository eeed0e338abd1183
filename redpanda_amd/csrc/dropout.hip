// Dropout with an optional residual: out = [res +] keep * s * x per element,
// keep from the counter-based generator of rp_philox.h, so the backward pass is
// the same call on the output's gradient (without the residual).
//
// One thread per block of eight columns: one generator call, one or two wide
// loads a tensor, wide stores whatever the rows' alignment.  HBM bounds it: the
// generator's 20 products a block hide behind the memory traffic.  16384 x 768, a
// bf16 branch on an fp32 stream: forward and backward together 40 us for 201 MB
// (5.0 TB/s, what a large copy reaches).

#include "rp_heads.h"
#include "rp_rows.h"

namespace rp {

__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutParams p) {
  const int64_t nb = (p.d + kDropBlock - 1) / kDropBlock;
  const int64_t n = p.rows * nb;
  const uint64_t seed = drop_seed(p.drop);
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * kThreads) {
    const int64_t row = e / nb, b = e % nb, col = b * kDropBlock;
    float v[8], res[8];
    load8(static_cast<const char*>(p.x) + row * p.xsr * p.es_x, col, p.d, p.dt_x, v);
    if (p.res != nullptr)
      load8(static_cast<const char*>(p.res) + row * p.rsr * p.es_res, col, p.d, p.dt_res, res);
    const DropWords m = drop_words((uint32_t)b, (uint64_t)row, p.drop.stream, seed);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = drop_keep(m, i, p.drop.t) ? v[i] * p.drop.scale : 0.f;
      if (p.res != nullptr) v[i] += res[i];
    }
    store8(static_cast<char*>(p.out) + row * p.d * p.es_out, col, p.d, p.dt_out, v);
  }
}

hipError_t launch_dropout(const DropoutParams& p, hipStream_t st) {
  const int64_t n = p.rows * ((p.d + kDropBlock - 1) / kDropBlock);
  if (n == 0) return hipSuccess;
  const int64_t wg = (n + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(dropout_kernel, dim3((unsigned)(wg < (1 << 20) ? wg : (1 << 20))),
                     dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

}  // namespace rp
