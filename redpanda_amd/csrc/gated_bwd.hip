// Backward of the gated recurrence.  With l_t = dy_t + a_{t+1} l_{t+1} (nothing from
// a step that begins a sequence; the last state's gradient at the end), from
// h_t = a_t h_{t-1} + (1 - a_t) x_t:
//     dx_t = (1 - a_t) l_t,   dz_t = (h_{t-1} - x_t) a_t (1 - a_t) l_t
// The states are computed again, 16 steps at a time from the forward's checkpoints (a
// sixteenth of the states, in fp32), so that only x, z and dy are read; the gates and
// states of 16 steps stay in registers between the way there and the way back.  The
// time axis is split as in the forward.

#include "gated.h"

namespace rp {

template <int ES, int V, bool kWhole>
__global__ __launch_bounds__(kWave) void gated_bwd_kernel(GatedParams p, GatedGrad d) {
  constexpr int K = kGatedK;
  const GatedAt<V> at(p);
  if (!kWhole && at.c == 0) return;  // (nothing comes before the first)
  float l[V], prod[V];
  float* slot = p.agg + ((at.b * p.nchunk + at.c) * 2) * p.D + at.ch;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    l[i] = 0.f;
    prod[i] = 1.f;
    if (kWhole && p.nchunk > 1) l[i] = slot[i];
    if (kWhole && p.nchunk == 1 && d.dh != nullptr) l[i] = d.dh[at.b * p.D + at.ch + i];
  }
  const char* x = static_cast<const char*>(p.x) + (at.b * p.xsb + at.ch) * ES;
  const char* g = static_cast<const char*>(p.g) + (at.b * p.gsb + at.ch) * ES;
  const char* dy = static_cast<const char*>(d.dy) + (d.dy != nullptr ? (at.b * d.dysb + at.ch) * ES : 0);
  char* dx = static_cast<char*>(d.dx) + (at.b * p.L * p.D + at.ch) * ES;
  char* dg = static_cast<char*>(d.dg) + (at.b * p.L * p.D + at.ch) * ES;
  const float* ck = p.ckpt + at.b * ((p.L + K - 1) / K) * p.D + at.ch;
  GatedRaw<ES, V> rx[K], rg[K], rd[K];
  GatedRaw<4, V> rh;
  uint32_t bits = 0;
  auto load = [&](int64_t t) {
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int64_t s = t + u < at.t1 ? t + u : at.t1 - 1;
      if (kWhole) rx[u] = gated_load<ES, V>(x + s * p.xsl * ES);
      rg[u] = gated_load<ES, V>(g + s * p.gsl * ES);
      if (d.dy != nullptr) rd[u] = gated_load<ES, V>(dy + s * d.dysl * ES);
    }
    if (kWhole) rh = gated_load<4, V>(reinterpret_cast<const char*>(ck + t / K * p.D));
    bits = start_bits(p, at.b, t, (int)(at.t1 - t < K ? at.t1 - t : K));
  };
  int64_t t = (at.t1 - 1) / K * K;  // (chunks begin at multiples of K)
  load(t);
  for (; t >= at.t0; t -= K) {
    // the way there: a, 1 - a and (h_{t-1} - x) a (1 - a)
    float a[K][V], na[K][V], c[K][V], gy[K][V], h[V];
    const uint32_t now = bits;
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = kWhole ? __uint_as_float(rh.w[i]) : 0.f;
#pragma unroll
    for (int u = 0; u < K; ++u) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        gate_of(gated_value(rg[u], i, p.dt), a[u][i], na[u][i]);
        gy[u][i] = d.dy != nullptr ? gated_value(rd[u], i, p.dt) : 0.f;
        if (kWhole) {
          const float xv = gated_value(rx[u], i, p.dt);
          const float prev = now >> u & 1 ? 0.f : h[i];
          c[u][i] = (prev - xv) * (a[u][i] * na[u][i]);
          h[i] = ffma(a[u][i], prev, na[u][i] * xv);
        }
      }
    }
    if (t - K >= at.t0) load(t - K);
    // the way back
#pragma unroll
    for (int u = K - 1; u >= 0; --u) {
      if (t + u >= at.t1) continue;
      const bool begin = now >> u & 1;
      float ox[V], og[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float s = gy[u][i] + l[i];
        ox[i] = s * na[u][i];
        og[i] = s * c[u][i];
        l[i] = begin ? 0.f : a[u][i] * s;
        if (!kWhole) prod[i] = begin ? -0.f : prod[i] * a[u][i];
      }
      if (kWhole) {
        gated_store<ES, V>(dx + (t + u) * p.D * ES, ox, p.dt);
        gated_store<ES, V>(dg + (t + u) * p.D * ES, og, p.dt);
      }
    }
  }
  if (!kWhole) {
    gated_store<4, V>(reinterpret_cast<char*>(slot), prod, RP_F32);
    gated_store<4, V>(reinterpret_cast<char*>(slot + p.D), l, RP_F32);
  } else if (d.dh0 != nullptr && at.c == 0) {
    gated_store<4, V>(reinterpret_cast<char*>(d.dh0 + at.b * p.D + at.ch), l, RP_F32);
  }
}

namespace {

template <int ES, int V>
hipError_t run(const GatedParams& p, const GatedGrad& g, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.nchunk * ((p.D + kWave * V - 1) / (kWave * V))));
  if (p.nchunk > 1) {
    hipLaunchKernelGGL((gated_bwd_kernel<ES, V, false>), grid, dim3(kWave), 0, st, p, g);
    const hipError_t e = launch_gated_fold(p, g.dh, true, st);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((gated_bwd_kernel<ES, V, true>), grid, dim3(kWave), 0, st, p, g);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_gated_bwd(const GatedParams& p, const GatedGrad& g, hipStream_t st) {
  const int V = gated_lane_channels(p.B, p.D, true);
  if (p.es == 4) return V == 2 ? run<4, 2>(p, g, st) : run<4, 1>(p, g, st);
  return V == 2 ? run<2, 2>(p, g, st) : run<2, 1>(p, g, st);
}

}  // namespace rp
