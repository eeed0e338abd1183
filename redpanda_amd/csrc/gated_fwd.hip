// Gated linear recurrence: per channel, with a_t = 1 / (1 + exp(-z_t)),
//     h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t
// and h_{t-1} taken as 0 where a sequence begins.  The state is fp32 in a register.
//
// The steps are a chain of one multiply-add each, so time goes by what is in flight:
// each wave loads the next eight steps' inputs while it works on the present ones.
// Where sequences times channels are too few waves for the card, the time axis is
// split: a first launch takes each chunk's (product of gates, end state from 0), a
// second joins them to the state that enters each chunk, and the main one starts from
// those.  The inputs are read twice then.

#include "gated.h"

namespace rp {

namespace {
constexpr int kAhead = 8;
}

// kWhole: writes y (and the checkpoints); else only the chunks' (product, end).
template <int ES, int V, bool kWhole>
__global__ __launch_bounds__(kWave) void gated_fwd_kernel(GatedParams p) {
  const GatedAt<V> at(p);
  if (!kWhole && at.c + 1 == p.nchunk) return;  // (nothing comes behind the last)
  float h[V], prod[V];
  float* slot = p.agg + ((at.b * p.nchunk + at.c) * 2) * p.D + at.ch;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h[i] = 0.f;
    prod[i] = 1.f;
    if (kWhole && p.nchunk > 1) h[i] = slot[i];
    if (kWhole && p.nchunk == 1 && p.h0 != nullptr) h[i] = p.h0[at.b * p.D + at.ch + i];
  }
  const char* x = static_cast<const char*>(p.x) + (at.b * p.xsb + at.ch) * ES;
  const char* g = static_cast<const char*>(p.g) + (at.b * p.gsb + at.ch) * ES;
  char* y = static_cast<char*>(p.y) + (at.b * p.L * p.D + at.ch) * ES;
  GatedRaw<ES, V> rx[kAhead], rg[kAhead];
  uint32_t bits = 0;
  auto load = [&](int64_t t) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      // (past the chunk the last step again)
      const int64_t s = t + u < at.t1 ? t + u : at.t1 - 1;
      rx[u] = gated_load<ES, V>(x + s * p.xsl * ES);
      rg[u] = gated_load<ES, V>(g + s * p.gsl * ES);
    }
    bits = start_bits(p, at.b, t, (int)(at.t1 - t < kAhead ? at.t1 - t : kAhead));
  };
  load(at.t0);
  for (int64_t t = at.t0; t < at.t1; t += kAhead) {
    GatedRaw<ES, V> cx[kAhead], cg[kAhead];
    const uint32_t now = bits;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      cx[u] = rx[u];
      cg[u] = rg[u];
    }
    if (t + kAhead < at.t1) load(t + kAhead);
    if (kWhole && p.ckpt != nullptr && t % kGatedK == 0) {
      float* to = p.ckpt + (at.b * ((p.L + kGatedK - 1) / kGatedK) + t / kGatedK) * p.D + at.ch;
      gated_store<4, V>(reinterpret_cast<char*>(to), h, RP_F32);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (t + u >= at.t1) break;
      const bool begin = now >> u & 1;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a, na;
        gate_of(gated_value(cg[u], i, p.dt), a, na);
        const float prev = begin ? 0.f : h[i];
        h[i] = ffma(a, prev, na * gated_value(cx[u], i, p.dt));
        if (!kWhole) prod[i] = begin ? -0.f : prod[i] * a;
      }
      if (kWhole) gated_store<ES, V>(y + (t + u) * p.D * ES, h, p.dt);
    }
  }
  if (!kWhole) {
    gated_store<4, V>(reinterpret_cast<char*>(slot), prod, RP_F32);
    gated_store<4, V>(reinterpret_cast<char*>(slot + p.D), h, RP_F32);
  } else if (p.h_last != nullptr && at.c + 1 == p.nchunk) {
    gated_store<4, V>(reinterpret_cast<char*>(p.h_last + at.b * p.D + at.ch), h, RP_F32);
  }
}

// What enters each chunk, over its product: forwards from `in` (h0), or backwards from
// the gradient of the last state.  One thread a channel.
__global__ __launch_bounds__(kWave) void gated_fold_kernel(GatedParams p, const float* in,
                                                           bool backward) {
  const uint32_t tiles = (uint32_t)((p.D + kWave - 1) / kWave);
  const int64_t b = blockIdx.x / tiles;
  const int64_t ch = (int64_t)(blockIdx.x % tiles) * kWave + threadIdx.x;
  if (ch >= p.D) return;
  float h = in != nullptr ? in[b * p.D + ch] : 0.f;
  float* base = p.agg + b * p.nchunk * 2 * p.D + ch;
  constexpr int kN = 8;
  for (int k0 = 0; k0 < p.nchunk; k0 += kN) {
    float a[kN], e[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      // (the last one's own product is never formed; nothing comes behind it)
      const int64_t i = k0 + k < p.nchunk - 1 ? k0 + k : p.nchunk - 2;
      const float* s = base + (backward ? p.nchunk - 1 - i : i) * 2 * p.D;
      a[k] = s[0];
      e[k] = s[p.D];
    }
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int i = k0 + k;
      if (i >= p.nchunk) break;
      base[(int64_t)(backward ? p.nchunk - 1 - i : i) * 2 * p.D] = h;
      h = gated_join(a[k], e[k], h);
    }
  }
}

hipError_t launch_gated_fold(const GatedParams& p, const float* in, bool backward, hipStream_t st) {
  hipLaunchKernelGGL(gated_fold_kernel, dim3((unsigned)(p.B * ((p.D + kWave - 1) / kWave))),
                     dim3(kWave), 0, st, p, in, backward);
  return hipGetLastError();
}

int64_t gated_plan(GatedParams* p, bool backward) {
  const int V = gated_lane_channels(p->B, p->D, backward);
  const int64_t waves = p->B * ((p->D + kWave * V - 1) / (kWave * V));
  p->nchunk = 1;
  p->chunk = (p->L + kGatedK - 1) / kGatedK * kGatedK;
  if (waves < 1024 && waves > 0 && p->L >= 128) {
    int64_t n = (2048 + waves - 1) / waves;
    if (n > (p->L + 63) / 64) n = (p->L + 63) / 64;
    const int64_t each = (p->L + n - 1) / n;
    p->chunk = (each + kGatedK - 1) / kGatedK * kGatedK;
    p->nchunk = (int)((p->L + p->chunk - 1) / p->chunk);
  }
  return p->nchunk > 1 ? p->B * p->nchunk * 2 * p->D : 0;
}

namespace {

template <int ES, int V>
hipError_t run(const GatedParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.nchunk * ((p.D + kWave * V - 1) / (kWave * V))));
  if (p.nchunk > 1) {
    hipLaunchKernelGGL((gated_fwd_kernel<ES, V, false>), grid, dim3(kWave), 0, st, p);
    const hipError_t e = launch_gated_fold(p, p.h0, false, st);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((gated_fwd_kernel<ES, V, true>), grid, dim3(kWave), 0, st, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_gated_fwd(const GatedParams& p, hipStream_t st) {
  const int V = gated_lane_channels(p.B, p.D, false);
  if (p.es == 4) return V == 4 ? run<4, 4>(p, st) : V == 2 ? run<4, 2>(p, st) : run<4, 1>(p, st);
  return V == 4 ? run<2, 4>(p, st) : V == 2 ? run<2, 2>(p, st) : run<2, 1>(p, st);
}

}  // namespace rp
