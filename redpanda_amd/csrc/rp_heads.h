// Parameter blocks and host-side launchers of the head operators: dropout, layer
// norm and sampling (internal to the library).
#pragma once

#include "rp_launch.h"

namespace rp {

// Dropout with an optional residual (dropout.hip).  The generator's part is
// described in rp_philox.h.
struct DropParams {
  uint32_t t;       // threshold, 0 .. 65536; 0: off
  uint32_t stream;
  float scale;      // 65536 / (65536 - t); 0 when nothing is kept
  uint64_t seed;
  const uint64_t* seed_ptr;  // the seed in device memory, or null
};

struct DropoutParams {
  int64_t rows, d;
  int dt_x, dt_res, dt_out;
  int es_x, es_res, es_out;  // element sizes
  DropParams drop;
  const void* x;    // (rows, d), row stride xsr
  int64_t xsr;
  const void* res;  // (rows, d) or null, row stride rsr
  int64_t rsr;
  void* out;        // (rows, d) contiguous
};

hipError_t launch_dropout(const DropoutParams& p, hipStream_t st);

// Layer norm with GELU and dropout (layernorm.hip).
struct LayerNormParams {
  int64_t rows, d;
  int dt_x, dt_out;
  int es_x, es_out;
  int gelu;
  float eps;
  DropParams drop;
  const void* x;   // (rows, d), row stride xsr
  int64_t xsr;
  const float* w;  // (d,) or null
  const float* b;
  void* out;       // (rows, d) contiguous
  float* stats;    // (rows, 2): mean, 1 / standard deviation
};

struct LayerNormGrad {
  const void* dout;  // (rows, d) in dt_out, row stride dosr
  int64_t dosr;
  void* dx;          // (rows, d) contiguous in dt_x, or null
  float* dw;         // (d,), or both null
  float* db;
  float* part;       // (layernorm_parts, 2, d) workspace
};

// Partial sums of the weights' gradients that a backward writes (es: bytes of an
// element).
int layernorm_parts(int64_t rows, int64_t d, int es_x, int es_out);
hipError_t launch_layernorm_fwd(const LayerNormParams& p, hipStream_t st);
hipError_t launch_layernorm_bwd(const LayerNormParams& p, const LayerNormGrad& g, hipStream_t st);

// Sampling (sample.hip).
struct SampleParams {
  int64_t R;
  int V;
  int n;      // elements of a row: V, or the length of the id lists
  int dt;
  int shift;  // weights are held as round(w 2^shift)
  const void* logits;
  int64_t lsr;
  const float* u;
  const int32_t* tokens;  // (R, n), row stride tsr, or null
  int64_t tsr;
  double T, tp, mp;
  int64_t k;
  const float* T_row;  // (R,) settings of each row, or null
  const float* tp_row;
  const float* mp_row;
  const int32_t* k_row;
  int64_t* ids;  // (R,)
  float* logp;   // (R,) or null
  void* work;    // sample_wide_bytes, or null
};

hipError_t launch_sample(const SampleParams& p, hipStream_t st);

// Few long rows, which several workgroups share (sample_wide.hip): whether a call
// is of that kind, its workspace, and its launches.
constexpr int kSampleWideRows = 128;
bool sample_is_wide(int64_t R, int64_t n, bool lists);
int64_t sample_wide_bytes(int64_t R);
hipError_t launch_sample_wide(const SampleParams& p, hipStream_t st);

}  // namespace rp
