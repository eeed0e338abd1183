// Backward of the gated recurrence.  With l_t = dy_t + a_{t+1} l_{t+1} (nothing from
// a step that begins a sequence; the last state's gradient at the end), from
// h_t = a_t h_{t-1} + (1 - a_t) x_t:
//     dx_t = (1 - a_t) l_t,   dz_t = (h_{t-1} - x_t) a_t (1 - a_t) l_t
// The states are computed again, 16 steps at a time from the forward's checkpoints (a
// sixteenth of the states, in fp32), so that only x, z and dy are read.  As in the
// forward the waves of a workgroup stand one behind the other in time, and the time
// axis is split among workgroups where there are few.
//
// Registers bound it: 16 steps of gates, complements and factors are a wave's; two channels
// a lane take 168 and three waves a SIMD, one channel 120 and four.  The rows' scalar
// addresses, of 16 steps and up to five arrays in two unrolled bodies, do not fit the scalar
// registers: 360 to 440 of them are kept in lanes of vector registers, and with two channels
// 12 bytes a lane are in scratch, 232 in the kernel of up to 16 steps.  (256 x 64 x 1536
// bf16: 64 us, 50 at the rate of a large copy; 64 x 2048 x 1024 300 for 267; 1 x 131072 x
// 1024: sums 144, join 9, main 293 for 261; 4096 x 1 x 1024 93 for 18, 4096 x 12 x 1024 251
// for 108.)

#include "gated.h"

namespace rp {

template <int T, int V, int NW>
__global__ __launch_bounds__(kWave* NW)
__attribute__((amdgpu_waves_per_eu(3))) void gated_bwd_kernel(GatedParams p, GatedGrad d) {
  constexpr int K = kGatedK, ES = gated_es(T);
  __shared__ GatedShare<V, NW> share;
  const GatedAt<V> at(p);
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  float l[V];  // what enters the waves' steps from behind
  const float* slot = p.agg + ((at.b * p.nchunk + at.c) * 2) * p.D;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    l[i] = 0.f;
    if (p.nchunk > 1) l[i] = slot[at.ch + i];
    if (p.nchunk == 1 && d.dh != nullptr) l[i] = d.dh[at.b * p.D + at.ch + i];
  }
  const char* x = static_cast<const char*>(p.x) + at.b * p.xsb * ES;
  const char* g = static_cast<const char*>(p.g) + at.b * p.gsb * ES;
  const char* dy = static_cast<const char*>(d.dy) + (d.dy != nullptr ? at.b * d.dysb * ES : 0);
  char* dx = static_cast<char*>(d.dx) + at.b * p.L * p.D * ES;
  char* dg = static_cast<char*>(d.dg) + at.b * p.L * p.D * ES;
  const float* ck = p.ckpt + at.b * ((p.L + K - 1) / K) * p.D;
  int turn = 0;
  for (int64_t t0 = at.t0 + (at.t1 - at.t0 - 1) / (K * NW) * (K * NW); t0 >= at.t0;
       t0 -= K * NW, turn ^= 1) {
    const int64_t t = t0 + wave * K;
    const int n = at.t1 - t < K ? (int)(at.t1 - t) : K;  // (0 or less: no steps left)
    const uint32_t bits = n > 0 ? start_bits(p, at.b, t, n) : 0;
    // 16 steps of one sequence, as nearly all are, go without a branch or a choice
    const bool full = n == K && bits == 0 && d.dy != nullptr;
    // the gates, and what turns a step's l_t into dz_t
    GatedRaw<ES, V> rd[K];
    float a[K][V], na[K][V], c[K][V], prod[V], end[V], from[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      prod[i] = 1.f;
      end[i] = 0.f;
    }
    auto there = [&](auto whole) {
      GatedRaw<ES, V> rx[K], rg[K];
      float h[V] = {};
      if (whole() || n > 0) {
        const GatedRaw<4, V> r = gated_load<4, V>(reinterpret_cast<const char*>(ck + t / K * p.D), at.ch * 4);
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = __uint_as_float(r.w[i]);
      }
#pragma unroll
      for (int u = 0; u < K; ++u) {
        if (!whole()) {
#pragma unroll
          for (int i = 0; i < GatedRaw<ES, V>::kWords; ++i) rd[u].w[i] = 0;
        }
        if (whole() || u < n) {
          rx[u] = gated_load<ES, V>(x + (t + u) * p.xsl * ES, at.ch * ES);
          rg[u] = gated_load<ES, V>(g + (t + u) * p.gsl * ES, at.ch * ES);
          if (whole() || d.dy != nullptr) rd[u] = gated_load<ES, V>(dy + (t + u) * d.dysl * ES, at.ch * ES);
        }
      }
#pragma unroll
      for (int u = 0; u < K; ++u) {
        if (whole() || u < n) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            gate_of(gated_value<T>(rg[u], i), a[u][i], na[u][i]);
            const float xv = gated_value<T>(rx[u], i);
            const float prev = !whole() && bits >> u & 1 ? 0.f : h[i];
            c[u][i] = (prev - xv) * (a[u][i] * na[u][i]);
            h[i] = ffma(a[u][i], prev, na[u][i] * xv);
          }
          // (a scheduler free to work on all steps at once takes half as many registers
          // again for it)
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // the way back from 0, for what the wave passes on
      if constexpr (NW > 1) {
#pragma unroll
        for (int u = K - 1; u >= 0; --u) {
          if (whole() || u < n) {
            const bool begin = !whole() && bits >> u & 1;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float s = gated_value<T>(rd[u], i) + end[i];
              end[i] = begin ? 0.f : a[u][i] * s;
              prod[i] = begin ? -0.f : prod[i] * a[u][i];
            }
          }
        }
      }
    };
    if (full)
      there(std::true_type{});
    else
      there(std::false_type{});
    if constexpr (NW > 1) {
      gated_above_0<K>(prod, n, [&](int u, int i) { return a[u][i]; });
      gated_store<RP_F32, V>(reinterpret_cast<char*>(&share.prod[turn][wave]), lane * V * 4, prod);
      gated_store<RP_F32, V>(reinterpret_cast<char*>(&share.end[turn][wave]), lane * V * 4, end);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) from[i] = l[i];
#pragma unroll
      for (int w = NW - 1; w >= 0; --w) {
        if (w == wave) {
#pragma unroll
          for (int i = 0; i < V; ++i) from[i] = l[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          l[i] = gated_join(share.prod[turn][w][lane * V + i], share.end[turn][w][lane * V + i], l[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) from[i] = l[i];
    }
    auto again = [&](auto whole) {
#pragma unroll
      for (int u = K - 1; u >= 0; --u) {
        if (whole() || u < n) {
          const bool begin = !whole() && bits >> u & 1;
          float ox[V], og[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float s = gated_value<T>(rd[u], i) + from[i];
            ox[i] = s * na[u][i];
            og[i] = s * c[u][i];
            from[i] = begin ? 0.f : a[u][i] * s;
          }
          gated_store<T, V>(dx + (t + u) * p.D * ES, at.ch * ES, ox);
          gated_store<T, V>(dg + (t + u) * p.D * ES, at.ch * ES, og);
        }
      }
    };
    if (full)
      again(std::true_type{});
    else
      again(std::false_type{});
    if constexpr (NW == 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) l[i] = from[i];
    }
    if (d.dh0 != nullptr && t == 0)
      gated_store<RP_F32, V>(reinterpret_cast<char*>(d.dh0 + at.b * p.D), at.ch * 4, from);
  }
}

// A chunk's (product, what it passes on) from behind: each wave walks its share of the
// steps backwards.
template <int T, int V, int NW>
__global__ __launch_bounds__(kWave* NW) void gated_bwd_sum_kernel(GatedParams p, GatedGrad d) {
  constexpr int K = kGatedK, ES = gated_es(T);
  __shared__ GatedShare<V, NW> share;
  const GatedAt<V> at(p);
  if (at.c == 0) return;  // (nothing comes before the first)
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const char* g = static_cast<const char*>(p.g) + at.b * p.gsb * ES;
  const char* dy = static_cast<const char*>(d.dy) + (d.dy != nullptr ? at.b * d.dysb * ES : 0);
  const int64_t first = at.t0 + wave * (p.chunk / NW);
  int64_t last = first + p.chunk / NW;
  if (last > at.t1) last = at.t1;  // (the last chunk's shares are cut, or empty)
  float prod[V], end[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    prod[i] = 1.f;
    end[i] = 0.f;
  }
  GatedRaw<ES, V> rg[K], rd[K];
  uint32_t bits = 0;
  int n = 0;
  auto load = [&](int64_t t) {
    n = last - t < K ? (int)(last - t) : K;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      const int64_t s = u < n ? t + u : t;  // (past the end the first step again)
      rg[u] = gated_load<ES, V>(g + s * p.gsl * ES, at.ch * ES);
#pragma unroll
      for (int i = 0; i < GatedRaw<ES, V>::kWords; ++i) rd[u].w[i] = 0;
      if (d.dy != nullptr) rd[u] = gated_load<ES, V>(dy + s * d.dysl * ES, at.ch * ES);
    }
    bits = start_bits(p, at.b, t, n);
  };
  int64_t t = first + (last - first - 1) / K * K;
  if (first < last) load(t);
  for (; first < last && t >= first; t -= K) {
    GatedRaw<ES, V> cg[K], cd[K];
    const uint32_t now = bits;
    const int m = n;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      cg[u] = rg[u];
      cd[u] = rd[u];
    }
    if (t - K >= first) load(t - K);
    float part[V];
#pragma unroll
    for (int i = 0; i < V; ++i) part[i] = 1.f;
    auto walk = [&](auto whole) {
#pragma unroll
      for (int u = K - 1; u >= 0; --u) {
        if (whole() || u < m) {
          const bool begin = !whole() && now >> u & 1;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float a, na;
            gate_of(gated_value<T>(cg[u], i), a, na);
            const float s = gated_value<T>(cd[u], i) + end[i];
            end[i] = begin ? 0.f : a * s;
            part[i] = begin ? -0.f : part[i] * a;
          }
        }
      }
    };
    if (now == 0 && m == K)
      walk(std::true_type{});
    else
      walk(std::false_type{});
    gated_above_0<K>(part, m, [&](int u, int i) {
      float a, na;
      gate_of(gated_value<T>(cg[u], i), a, na);
      return a;
    });
#pragma unroll
    for (int i = 0; i < V; ++i) prod[i] = gated_product(prod[i], part[i]);
  }
  gated_leave<V, NW>(p, at.b, at.c, at.ch, lane, wave, true, prod, end, share);
}

namespace {

template <int T, int V, int NW>
hipError_t run(const GatedParams& p, const GatedGrad& g, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.nchunk * ((p.D + kWave * V - 1) / (kWave * V))));
  if (p.nchunk > 1) {
    if constexpr (NW == kSplitWaves) {
      hipLaunchKernelGGL((gated_bwd_sum_kernel<T, V, NW>), grid, dim3(kWave * NW), 0, st, p, g);
      const hipError_t e = launch_gated_fold(p, g.dh, true, st);
      if (e != hipSuccess) return e;
    } else {
      return hipErrorInvalidValue;
    }
  }
  hipLaunchKernelGGL((gated_bwd_kernel<T, V, NW>), grid, dim3(kWave * NW), 0, st, p, g);
  return hipGetLastError();
}

template <int T, int V>
hipError_t run_waves(const GatedParams& p, const GatedGrad& g, hipStream_t st) {
#define RP_CASE(NW) if (p.nw == NW) return run<T, V, NW>(p, g, st);
  RP_CASE(1) RP_CASE(2) RP_CASE(4)
  if constexpr (V == 1) {
    RP_CASE(8) RP_CASE(16)
  }
#undef RP_CASE
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_gated_bwd(const GatedParams& p, const GatedGrad& g, hipStream_t st) {
  if (p.dt == RP_F32) return run_waves<RP_F32, 1>(p, g, st);
  if (p.v == 2)
    return p.dt == RP_BF16 ? run_waves<RP_BF16, 2>(p, g, st) : run_waves<RP_F16, 2>(p, g, st);
  return p.dt == RP_BF16 ? run_waves<RP_BF16, 1>(p, g, st) : run_waves<RP_F16, 1>(p, g, st);
}

}  // namespace rp
