// Parameter blocks and host-side launchers of the training operators: embedding,
// RMS norm with the residual's addition, checkpoints in 8 bits, and the gated
// recurrence (internal to the library).
#pragma once

#include "rp_launch.h"

namespace rp {

// e / n for 0 <= e < 2^31 by one product: m = ceil(2^(31 + s) / n) with 2^s >= n
// fits 32 bits and is off by less than n <= 2^s, which e < 2^31 does not let reach the
// quotient.
struct FastDiv {
  uint32_t m, s, n;
  FastDiv() : m(0), s(0), n(1) {}
  explicit FastDiv(uint32_t d) : s(0), n(d) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t e) const {
    return (uint32_t)(((uint64_t)e * m) >> (31 + s));
  }
};

// Embedding (embedding.hip).
struct EmbedParams {
  int64_t N, V, d;
  int dt_w, dt_out, es_w, es_out;
  int ids64;        // ids are int64, else int32
  int64_t pad;      // an id whose row gets no gradient, or -1
  float scale;
  const void* ids;  // (N,)
  const void* w;    // (V, d), row stride wsr
  int64_t wsr;
  void* out;        // (N, d) contiguous
};

// How a backward is laid out.
struct EmbedPlan {
  int lg;         // ids are sorted in 2^lg buckets by their low bits
  int range;      // ids of a bucket, and the bits of their numbers in it
  int bits;
  int share;      // sorted places of a wave of the sums
  int64_t slots;  // 2^lg range
  int64_t shares;
  int64_t parts;  // of the split before the sort, or 0
  int64_t unit;   // parts of a wave of the count, and the number of such units
  int64_t units;
};
constexpr int64_t kSplitPart = 2048;  // places of a part
constexpr int kSplitSegs = 257;       // where each value of the low eight bits begins, and the end
EmbedPlan embed_plan(int64_t N, int64_t V, int64_t d, int es_out);

// A place and its id, as the split leaves them.
struct EmbedPair {
  int32_t id, at;
};

struct EmbedGrad {
  const void* dout;  // (N, d) in dt_out, row stride dosr
  int64_t dosr;
  void* dw;          // (V, d) contiguous in dt_w
  int32_t* start;    // (slots + 1,) workspace: where each id's places begin in `place`
  int32_t* place;    // (N,) workspace: the places 0 .. N - 1 with equal ids together
  int32_t* sorted;   // (N,) workspace: their ids
  float* part;       // (shares, 2, d) workspace
  EmbedPair* divided;  // (shares,) workspace: the id that begins in a share and goes on
                       //   behind it, and the number of its pieces (or 0)
  EmbedPair* pairs;  // (parts, 2048) workspace
  int32_t* segs;     // (parts, kSplitSegs) workspace
  int32_t* counts;   // (units, slots) workspace
  int32_t* totals;   // (units, buckets) workspace, where buckets are of more than eight bits
  EmbedPlan plan;
};

hipError_t launch_embed_fwd(const EmbedParams& p, hipStream_t st);
hipError_t launch_embed_bwd(const EmbedParams& p, const EmbedGrad& g, hipStream_t st);

// RMS norm with the residual's addition (addnorm.hip).
struct AddNormParams {
  int64_t rows, d;
  int dt_x, dt_add, dt_sum, dt_out;
  int es_x, es_add, es_sum, es_out;
  float eps;
  const void* x;    // (rows, d), row stride xsr; null: the rows are held in q8, e8
  int64_t xsr;
  const void* add;  // (rows, d) or null, row stride asr
  int64_t asr;
  const float* w;   // (d,) or null
  void* sum;        // (rows, d) contiguous in dt_sum, or null
  void* out;        // (rows, d) contiguous, or null
  int8_t* q8;       // (rows, d) and (rows, ceil(d / 32)): the sum in 8 bits
  uint8_t* e8;      //   (written where x is given, read where it is not), or null
};

struct AddNormGrad {
  const void* dout;  // (rows, d) in dt_out, row stride dosr
  int64_t dosr;
  const void* dsum;  // (rows, d) in dt_sum or null, row stride dssr
  int64_t dssr;
  void* dx;          // (rows, d) contiguous in dt_x, or null
  void* dadd;        // (rows, d) contiguous in dt_add, or null
  float* dw;         // (d,), or null
  float* part;       // addnorm_work_floats of workspace
};

// Floats of workspace that a backward needs.
int64_t addnorm_work_floats(int64_t rows, int64_t d);
hipError_t launch_addnorm_fwd(const AddNormParams& p, hipStream_t st);
// The backward's rows are p.x (row stride p.xsr, in dt_sum), or p.q8 and p.e8.
hipError_t launch_addnorm_bwd(const AddNormParams& p, const AddNormGrad& g, hipStream_t st);

// Rows in 8 bits (pack8.hip).
struct Pack8Params {
  int64_t rows, d;
  int dt, es;
  int dt_held;   // (unpack) the type that was packed
  void* x;       // (rows, d), row stride xsr; read by the pack, written by the unpack
  int64_t xsr;
  int8_t* q8;    // (rows, d) contiguous
  uint8_t* e8;   // (rows, ceil(d / 32))
};
hipError_t launch_pack8(const Pack8Params& p, hipStream_t st);
hipError_t launch_unpack8(const Pack8Params& p, hipStream_t st);

// Gated linear recurrence (gated_fwd.hip, gated_bwd.hip).
constexpr int kGatedK = 16;  // steps between the states that the backward starts from
struct GatedParams {
  int64_t B, L, D;
  int dt, es;
  const void* x;     // (B, L, D), strides xsb, xsl
  int64_t xsb, xsl;
  const void* g;     // the gates, likewise
  int64_t gsb, gsl;
  const float* h0;   // (B, D) or null
  const uint8_t* starts;  // (B, L), batch stride ssb, or null
  int64_t ssb;
  void* y;           // (B, L, D) contiguous
  float* h_last;     // (B, D) or null
  float* ckpt;       // (B, ceil(L / kGatedK), D) or null: the state before every 16th step
  float* agg;        // workspace of gated_work_floats
  int v;             // channels of a lane
  int nw;            // waves of a workgroup
  int nchunk;        // time chunks, each of `chunk` steps (a multiple of 16 nw)
  int64_t chunk;
};
struct GatedGrad {
  const void* dy;    // (B, L, D) or null, strides dysb, dysl
  int64_t dysb, dysl;
  const float* dh;   // (B, D) or null: the gradient of the last state
  void* dx;          // (B, L, D) contiguous each
  void* dg;
  float* dh0;        // (B, D) or null
};
// Sets p.v, p.nw, p.nchunk and p.chunk; the floats of workspace that p.agg needs.
int64_t gated_plan(GatedParams* p);
hipError_t launch_gated_fwd(const GatedParams& p, hipStream_t st);
hipError_t launch_gated_bwd(const GatedParams& p, const GatedGrad& g, hipStream_t st);

}  // namespace rp
