// Gated linear recurrence: per channel, with a_t = 1 / (1 + exp(-z_t)),
//     h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t
// and h_{t-1} taken as 0 where a sequence begins.  The state is fp32 in a register.
//
// Walked step by step a sequence goes by the latency of its loads.  So the waves of a
// workgroup stand one behind the other in time: each loads 16 steps at once, forms the
// product of their gates and the end state that they reach from 0, and leaves both in
// LDS; the states that enter the waves follow from those (one multiply-add a wave),
// and each wave goes over its 16 steps again, from registers.  The inputs are read
// once.  Where sequences times channels are too few workgroups for the card, the time
// axis is split among workgroups too: a launch takes each chunk's (product, end), a
// second joins them, and the main one starts from there; the inputs are read twice
// then.
//
// HBM bounds it where the card is full (256 x 64 x 1536 bf16: 33 us, 31 at the rate of a
// large copy; 64 x 2048 x 1024 174 for 163; 1 x 131072 x 1024: sums 129, join 9, main 160
// for 157).  A wave that walked its whole stretch with eight steps loaded ahead took 45
// us for the first and 422 for the last.

#include "gated.h"

namespace rp {

template <int T, int V, int NW>
__global__ __launch_bounds__(kWave* NW) void gated_fwd_kernel(GatedParams p) {
  constexpr int K = kGatedK, ES = gated_es(T);
  __shared__ GatedShare<V, NW> share;
  const GatedAt<V> at(p);
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  float h[V];  // the state that enters the waves' steps
  const float* slot = p.agg + ((at.b * p.nchunk + at.c) * 2) * p.D;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h[i] = 0.f;
    if (p.nchunk > 1) h[i] = slot[at.ch + i];
    if (p.nchunk == 1 && p.h0 != nullptr) h[i] = p.h0[at.b * p.D + at.ch + i];
  }
  const char* x = static_cast<const char*>(p.x) + at.b * p.xsb * ES;
  const char* g = static_cast<const char*>(p.g) + at.b * p.gsb * ES;
  char* y = static_cast<char*>(p.y) + at.b * p.L * p.D * ES;
  int turn = 0;
  for (int64_t t0 = at.t0; t0 < at.t1; t0 += K * NW, turn ^= 1) {
    const int64_t t = t0 + wave * K;
    const int n = at.t1 - t < K ? (int)(at.t1 - t) : K;  // (0 or less: no steps left)
    const uint32_t bits = n > 0 ? start_bits(p, at.b, t, n) : 0;
    // 16 steps of one sequence, as nearly all are, go without a branch or a choice
    const bool full = n == K && bits == 0;
    float a[K][V], in[K][V], prod[V], end[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      prod[i] = 1.f;
      end[i] = 0.f;
    }
    auto there = [&](auto whole) {
      GatedRaw<ES, V> rx[K], rg[K];
#pragma unroll
      for (int u = 0; u < K; ++u) {
        if (whole() || u < n) {
          rx[u] = gated_load<ES, V>(x + (t + u) * p.xsl * ES, at.ch * ES);
          rg[u] = gated_load<ES, V>(g + (t + u) * p.gsl * ES, at.ch * ES);
        }
      }
#pragma unroll
      for (int u = 0; u < K; ++u) {
        if (whole() || u < n) {
          const bool begin = !whole() && bits >> u & 1;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float na;
            gate_of(gated_value<T>(rg[u], i), a[u][i], na);
            in[u][i] = na * gated_value<T>(rx[u], i);
            prod[i] = begin ? -0.f : prod[i] * a[u][i];
            end[i] = ffma(a[u][i], begin ? 0.f : end[i], in[u][i]);
          }
        }
      }
    };
    if (full)
      there(std::true_type{});
    else
      there(std::false_type{});
    float from[V];
    if constexpr (NW > 1) {
      gated_above_0<K>(prod, n, [&](int u, int i) { return a[u][i]; });
      gated_store<RP_F32, V>(reinterpret_cast<char*>(&share.prod[turn][wave]), lane * V * 4, prod);
      gated_store<RP_F32, V>(reinterpret_cast<char*>(&share.end[turn][wave]), lane * V * 4, end);
      // (the next turn's stores go to the other half, and the one behind that waits for
      // this turn's reads at the next turn's barrier)
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) from[i] = h[i];
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w == wave) {
#pragma unroll
          for (int i = 0; i < V; ++i) from[i] = h[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[i] = gated_join(share.prod[turn][w][lane * V + i], share.end[turn][w][lane * V + i], h[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) from[i] = h[i];
    }
    if (n > 0 && p.ckpt != nullptr) {
      float* to = p.ckpt + (at.b * ((p.L + K - 1) / K) + t / K) * p.D;
      gated_store<RP_F32, V>(reinterpret_cast<char*>(to), at.ch * 4, from);
    }
    auto again = [&](auto whole) {
#pragma unroll
      for (int u = 0; u < K; ++u) {
        if (whole() || u < n) {
          const bool begin = !whole() && bits >> u & 1;
#pragma unroll
          for (int i = 0; i < V; ++i) from[i] = ffma(a[u][i], begin ? 0.f : from[i], in[u][i]);
          gated_store<T, V>(y + (t + u) * p.D * ES, at.ch * ES, from);
        }
      }
    };
    if (full)
      again(std::true_type{});
    else
      again(std::false_type{});
    if constexpr (NW == 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = from[i];
    }
    // the wave with the last step has the last state, as its own steps give it
    if (p.h_last != nullptr && t < p.L && t + n == p.L)
      gated_store<RP_F32, V>(reinterpret_cast<char*>(p.h_last + at.b * p.D), at.ch * 4, from);
  }
}

// A chunk's (product, end): each wave walks its share of the steps, the next 16 loaded
// while it works on the present ones.
template <int T, int V, int NW>
__global__ __launch_bounds__(kWave* NW) void gated_fwd_sum_kernel(GatedParams p) {
  constexpr int K = kGatedK, ES = gated_es(T);
  __shared__ GatedShare<V, NW> share;
  const GatedAt<V> at(p);
  if (at.c + 1 == p.nchunk) return;  // (nothing comes behind the last)
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const char* x = static_cast<const char*>(p.x) + at.b * p.xsb * ES;
  const char* g = static_cast<const char*>(p.g) + at.b * p.gsb * ES;
  // (every chunk but the last is whole: its shares are multiples of 16 steps)
  const int64_t first = at.t0 + wave * (p.chunk / NW), last = first + p.chunk / NW;
  float prod[V], end[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    prod[i] = 1.f;
    end[i] = 0.f;
  }
  GatedRaw<ES, V> rx[K], rg[K];
  uint32_t bits = 0;
  auto load = [&](int64_t t) {
#pragma unroll
    for (int u = 0; u < K; ++u) {
      rx[u] = gated_load<ES, V>(x + (t + u) * p.xsl * ES, at.ch * ES);
      rg[u] = gated_load<ES, V>(g + (t + u) * p.gsl * ES, at.ch * ES);
    }
    bits = start_bits(p, at.b, t, K);
  };
  load(first);
  for (int64_t t = first; t < last; t += K) {
    GatedRaw<ES, V> cx[K], cg[K];
    const uint32_t now = bits;
#pragma unroll
    for (int u = 0; u < K; ++u) {
      cx[u] = rx[u];
      cg[u] = rg[u];
    }
    if (t + K < last) load(t + K);
    float part[V];
#pragma unroll
    for (int i = 0; i < V; ++i) part[i] = 1.f;
    auto walk = [&](auto whole) {
#pragma unroll
      for (int u = 0; u < K; ++u) {
        const bool begin = !whole() && now >> u & 1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float a, na;
          gate_of(gated_value<T>(cg[u], i), a, na);
          part[i] = begin ? -0.f : part[i] * a;
          end[i] = ffma(a, begin ? 0.f : end[i], na * gated_value<T>(cx[u], i));
        }
      }
    };
    if (now == 0)
      walk(std::true_type{});
    else
      walk(std::false_type{});
    gated_above_0<K>(part, K, [&](int u, int i) {
      float a, na;
      gate_of(gated_value<T>(cg[u], i), a, na);
      return a;
    });
#pragma unroll
    for (int i = 0; i < V; ++i) prod[i] = gated_product(prod[i], part[i]);
  }
  gated_leave<V, NW>(p, at.b, at.c, at.ch, lane, wave, false, prod, end, share);
}

// Few steps (a rollout's single token): no stretch to share, one thread for 16 bytes of
// a row.
template <int T, int V>
__global__ __launch_bounds__(kWave) void gated_few_kernel(GatedParams p) {
  constexpr int ES = gated_es(T);
  const GatedAt<V> at(p);
  float h[V];
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = 0.f;
  if (p.h0 != nullptr) {
    const GatedRaw<4, V> r =
        gated_load<4, V>(reinterpret_cast<const char*>(p.h0 + at.b * p.D), at.ch * 4);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = __uint_as_float(r.w[i]);
  }
  const char* x = static_cast<const char*>(p.x) + at.b * p.xsb * ES;
  const char* g = static_cast<const char*>(p.g) + at.b * p.gsb * ES;
  char* y = static_cast<char*>(p.y) + at.b * p.L * p.D * ES;
  if (p.ckpt != nullptr)
    gated_store<RP_F32, V>(reinterpret_cast<char*>(p.ckpt + at.b * p.D), at.ch * 4, h);
  for (int64_t t = 0; t < p.L; ++t) {
    const GatedRaw<ES, V> rx = gated_load<ES, V>(x + t * p.xsl * ES, at.ch * ES);
    const GatedRaw<ES, V> rg = gated_load<ES, V>(g + t * p.gsl * ES, at.ch * ES);
    const bool begin = start_bits(p, at.b, t, 1) != 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a, na;
      gate_of(gated_value<T>(rg, i), a, na);
      h[i] = ffma(a, begin ? 0.f : h[i], na * gated_value<T>(rx, i));
    }
    gated_store<T, V>(y + t * p.D * ES, at.ch * ES, h);
  }
  if (p.h_last != nullptr)
    gated_store<RP_F32, V>(reinterpret_cast<char*>(p.h_last + at.b * p.D), at.ch * 4, h);
}

// What enters each chunk, over its product: forwards from `in` (h0), or backwards from
// the gradient of the last state.  16 waves take a sixteenth of the chunks of 64
// channels each, as the waves above take steps.
constexpr int kFoldWaves = 16;
__global__ __launch_bounds__(kFoldWaves* kWave) void gated_fold_kernel(GatedParams p, const float* in,
                                                                       bool backward) {
  __shared__ float prods[kFoldWaves][kWave], ends[kFoldWaves][kWave];
  const uint32_t tiles = (uint32_t)((p.D + kWave - 1) / kWave);
  const int64_t b = blockIdx.x / tiles;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int64_t ch = (int64_t)(blockIdx.x % tiles) * kWave + lane;
  if (ch > p.D - 1) ch = p.D - 1;
  float* base = p.agg + b * p.nchunk * 2 * p.D + ch;
  auto slot = [&](int i) { return base + (int64_t)(backward ? p.nchunk - 1 - i : i) * 2 * p.D; };
  // (the last chunk's own product is never formed; nothing comes behind it)
  const int n = p.nchunk - 1, each = (n + kFoldWaves - 1) / kFoldWaves;
  const int first = wave * each < n ? wave * each : n, last = first + each < n ? first + each : n;
  float prod = 1.f, end = 0.f;
  // (16 chunks at a time: all of their loads before the first use, and before the stores)
  constexpr int kN = 16;
  auto walk = [&](auto f) {
    for (int i0 = first; i0 < last; i0 += kN) {
      float a[kN], e[kN];
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const float* s = slot(i0 + k < last ? i0 + k : last - 1);
        a[k] = s[0];
        e[k] = s[p.D];
      }
#pragma unroll
      for (int k = 0; k < kN; ++k)
        if (i0 + k < last) f(i0 + k, a[k], e[k]);
    }
  };
  walk([&](int, float a, float e) {
    end = gated_join(a, e, end);
    prod = gated_product(prod, a);
  });
  prods[wave][lane] = prod;
  ends[wave][lane] = end;
  __syncthreads();
  float h = in != nullptr ? in[b * p.D + ch] : 0.f;
  for (int w = 0; w < wave; ++w) h = gated_join(prods[w][lane], ends[w][lane], h);
  walk([&](int i, float a, float e) {
    *slot(i) = h;
    h = gated_join(a, e, h);
  });
  // (the waves behind the last chunk have folded all of it)
  if (wave == kFoldWaves - 1) *slot(n) = h;
}

hipError_t launch_gated_fold(const GatedParams& p, const float* in, bool backward, hipStream_t st) {
  hipLaunchKernelGGL(gated_fold_kernel, dim3((unsigned)(p.B * ((p.D + kWave - 1) / kWave))),
                     dim3(kFoldWaves * kWave), 0, st, p, in, backward);
  return hipGetLastError();
}

// Three shapes, by the workgroups that sequences and channels alone give (bf16, both ways,
// kernels):
//   256 or more: four waves each, the whole sequence (32 x 2048 x 1024, 256 workgroups: 330
//     us, split 371; 64 x 2048 x 1024 with eight waves, of which one workgroup is resident a
//     CU, 519 for 496)
//   fewer, up to 256 steps: a lane a channel and all steps at once
//   fewer, more steps: split among about 2048 workgroups (16 x 2048 x 1024, 128 workgroups:
//     196 us, whole 230; 1 x 131072 x 1024, 8 workgroups: 735)
int64_t gated_plan(GatedParams* p) {
  const int V = p->v = p->es == 2 && p->D >= 2 ? 2 : 1;
  const int64_t tiles = p->B * ((p->D + kWave * V - 1) / (kWave * V));
  int64_t n = 1;
  int most = kSplitWaves;
  if (tiles < 256 && p->L <= 16 * kGatedK) {
    p->v = 1;
    most = 16;
  } else if (tiles < 256) {
    n = (2048 + tiles - 1) / tiles;
    const int64_t few = (p->L + kGatedK * kSplitWaves - 1) / (kGatedK * kSplitWaves);
    if (n > few) n = few;
  }
  p->nw = 1;
  while (p->nw < most && p->nw * kGatedK < p->L) p->nw *= 2;
  const int64_t step = kGatedK * p->nw, each = (p->L + n - 1) / n;
  p->chunk = (each + step - 1) / step * step;
  p->nchunk = (int)((p->L + p->chunk - 1) / p->chunk);
  return p->nchunk > 1 ? p->B * p->nchunk * 2 * p->D : 0;
}

namespace {

template <int T, int V, int NW>
hipError_t run(const GatedParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.nchunk * ((p.D + kWave * V - 1) / (kWave * V))));
  if (p.nchunk > 1) {
    if constexpr (NW == kSplitWaves) {
      hipLaunchKernelGGL((gated_fwd_sum_kernel<T, V, NW>), grid, dim3(kWave * NW), 0, st, p);
      const hipError_t e = launch_gated_fold(p, p.h0, false, st);
      if (e != hipSuccess) return e;
    } else {
      return hipErrorInvalidValue;
    }
  }
  hipLaunchKernelGGL((gated_fwd_kernel<T, V, NW>), grid, dim3(kWave * NW), 0, st, p);
  return hipGetLastError();
}

template <int T, int V>
hipError_t run_few(const GatedParams& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * ((p.D + kWave * V - 1) / (kWave * V))));
  hipLaunchKernelGGL((gated_few_kernel<T, V>), grid, dim3(kWave), 0, st, p);
  return hipGetLastError();
}

template <int T, int V>
hipError_t run_waves(const GatedParams& p, hipStream_t st) {
#define RP_CASE(NW) if (p.nw == NW) return run<T, V, NW>(p, st);
  RP_CASE(1) RP_CASE(2) RP_CASE(4)
  if constexpr (V == 1) {
    RP_CASE(8) RP_CASE(16)
  }
#undef RP_CASE
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_gated_fwd(const GatedParams& p, hipStream_t st) {
  if (p.L <= 4 && p.D >= 4) {
    return p.dt == RP_F32    ? run_few<RP_F32, 4>(p, st)
           : p.dt == RP_BF16 ? run_few<RP_BF16, 4>(p, st)
                             : run_few<RP_F16, 4>(p, st);
  }
  if (p.dt == RP_F32) return run_waves<RP_F32, 1>(p, st);
  if (p.v == 2)
    return p.dt == RP_BF16 ? run_waves<RP_BF16, 2>(p, st) : run_waves<RP_F16, 2>(p, st);
  return p.dt == RP_BF16 ? run_waves<RP_BF16, 1>(p, st) : run_waves<RP_F16, 1>(p, st);
}

}  // namespace rp
