// What the gated recurrence's passes share (the mathematics is in gated_fwd.hip).
//
// A workgroup takes 64 V adjacent channels of one sequence, V a lane, and a chunk of its
// steps, NW waves times 16 steps at a time, each wave the 16 behind those of the wave
// before it.  A row's last lanes take channels that end with the row, so that every
// access is a whole vector (channels in two lanes get the same values twice).
#pragma once

#include "rp_rows.h"
#include "rp_train.h"

namespace rp {

// The storage types are known when the kernels are compiled (T, an RP_* code): choosing
// between the two of 16 bits for each value kept both forms in registers.
constexpr int gated_es(int T) { return T == RP_F32 ? 4 : 2; }

// V adjacent elements as stored.
template <int ES, int V>
struct GatedRaw {
  static constexpr int kWords = ES * V >= 4 ? ES * V / 4 : 1;
  uint32_t w[kWords];
};

// (a row, the same in every lane, and the lane's bytes into it: one scalar address for
// all lanes and no vector registers for the rows')
template <int ES, int V>
__device__ __forceinline__ GatedRaw<ES, V> gated_load(const char* row, uint32_t at) {
  const char* p = row + at;
  GatedRaw<ES, V> r;
  if constexpr (ES * V == 2) {
    r.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (ES * V == 4) {
    typedef uint32_t u32_any __attribute__((aligned(1)));
    r.w[0] = *reinterpret_cast<const u32_any*>(p);
  } else if constexpr (ES * V == 8) {
    const u32x2_any v = *reinterpret_cast<const u32x2_any*>(p);
    r.w[0] = v[0];
    r.w[1] = v[1];
  } else {
    const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = v[i];
  }
  return r;
}

template <int T, int ES, int V>
__device__ __forceinline__ float gated_value(const GatedRaw<ES, V>& r, int i) {
  if constexpr (T == RP_F32) {
    return __uint_as_float(r.w[i]);
  } else if constexpr (T == RP_BF16) {
    return __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
  } else {
    return static_cast<float>(
        __builtin_bit_cast(_Float16, static_cast<uint16_t>(r.w[i / 2] >> (16 * (i & 1)))));
  }
}

template <int T, int V>
__device__ __forceinline__ void gated_store(char* row, uint32_t at, const float (&v)[V]) {
  constexpr int ES = T == RP_F32 ? 4 : 2;
  char* p = row + at;
  if constexpr (ES == 4) {
    if constexpr (V == 4) {
      u32x4_any w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
      *reinterpret_cast<u32x4_any*>(p) = w;
    } else if constexpr (V == 2) {
      u32x2_any w;
      w[0] = __float_as_uint(v[0]);
      w[1] = __float_as_uint(v[1]);
      *reinterpret_cast<u32x2_any*>(p) = w;
    } else {
      *reinterpret_cast<float*>(p) = v[0];
    }
  } else if constexpr (V == 4) {
    u32x2_any w;
    w[0] = pack16(v[0], v[1], T);
    w[1] = pack16(v[2], v[3], T);
    *reinterpret_cast<u32x2_any*>(p) = w;
  } else if constexpr (V == 2) {
    typedef uint32_t u32_any __attribute__((aligned(1)));
    *reinterpret_cast<u32_any*>(p) = pack16(v[0], v[1], T);
  } else {
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)pack16(v[0], 0.f, T);
  }
}

// a = 1 / (1 + exp(-z)) and 1 - a, neither from the other by a subtraction: of exp(-|z|) /
// (1 + exp(-|z|)) and 1 / (1 + exp(-|z|)) each is the one or the other.  The exponent |z|
// log2 e is rounded, so each is off by up to (2 |z| + 6) 2^-24 of itself; the smaller is 0
// beyond |z| = 87.3, where fp32's normal numbers end.
__device__ __forceinline__ void gate_of(float z, float& a, float& na) {
  const float e = exp2_hw(fabsf(z) * -kLog2e);
  const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
  a = z >= 0.f ? big : small;
  na = z >= 0.f ? small : big;
}

// Which of the `n` steps (up to 16) from t on begin a sequence, a bit each, the same in
// every lane.
__device__ __forceinline__ uint32_t start_bits(const GatedParams& p, int64_t b, int64_t t, int n) {
  if (p.starts == nullptr) return 0;
  const int lane = threadIdx.x % kWave;
  return (uint32_t)__ballot(lane < n && p.starts[b * p.ssb + t + (lane < n ? lane : 0)] != 0);
}

// A workgroup's place: its sequence, its time chunk and its lanes' first channels.
template <int V>
struct GatedAt {
  int64_t b, c, t0, t1;
  uint32_t ch;
  __device__ __forceinline__ GatedAt(const GatedParams& p) {
    const uint32_t tiles = (uint32_t)((p.D + kWave * V - 1) / (kWave * V));
    const uint32_t rest = blockIdx.x / tiles, tile = blockIdx.x - rest * tiles;
    b = rest / (uint32_t)p.nchunk;
    c = rest - (uint32_t)b * (uint32_t)p.nchunk;
    ch = (tile * kWave + threadIdx.x % kWave) * V;
    if (ch > (uint32_t)p.D - V) ch = (uint32_t)p.D - V;
    t0 = c * p.chunk;
    t1 = t0 + p.chunk < p.L ? t0 + p.chunk : p.L;
  }
};

// The (product of the gates, end from 0) of a stretch, applied to what enters it.  A
// stretch in which a sequence begins has the product -0 and passes nothing on, not even
// an infinity.  Else the product is 0 where a gate is, and only there: one that underflows
// is held at kGatedLeast, so that an infinity goes through any number of gates above 0 as
// it does step by step, where 0 times it would be NaN.  (Of a finite state 2^-149 of it
// comes through then, 5e-7 at most.)
constexpr float kGatedLeast = 0x1p-149f;
__device__ __forceinline__ float gated_join(float prod, float end, float in) {
  return __float_as_uint(prod) == 0x80000000u ? end : ffma(prod, in, end);
}
// And of two stretches, one behind the other.
__device__ __forceinline__ float gated_product(float first, float second) {
  float p = first * second;
  if (p == 0.f && first != 0.f && second != 0.f) p = kGatedLeast;
  return __float_as_uint(first) == 0x80000000u || __float_as_uint(second) == 0x80000000u ? -0.f : p;
}
// The products of n steps' gates (up to K) that have come out as 0: held above it unless
// one of the gates, gate(step, channel), is 0 itself.
template <int K, int V, typename F>
__device__ __forceinline__ void gated_above_0(float (&prod)[V], int n, F gate) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (__float_as_uint(prod[i]) != 0u) continue;
    float low = 1.f;
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (u < n) low = fminf(low, gate(u, i));
    prod[i] = low > 0.f ? kGatedLeast : 0.f;
  }
}

// What the waves of a workgroup know of their stretches.
template <int V, int NW>
struct GatedShare {
  float prod[2][NW][kWave * V];
  float end[2][NW][kWave * V];
};

// The waves' (product, end) of a chunk, joined in order (from behind: the last wave's
// first), to the chunk's slot.
template <int V, int NW>
__device__ __forceinline__ void gated_leave(const GatedParams& p, int64_t b, int64_t c, uint32_t ch,
                                            int lane, int wave, bool behind, float (&prod)[V],
                                            float (&end)[V], GatedShare<V, NW>& share) {
  gated_store<RP_F32, V>(reinterpret_cast<char*>(&share.prod[0][wave]), lane * V * 4, prod);
  gated_store<RP_F32, V>(reinterpret_cast<char*>(&share.end[0][wave]), lane * V * 4, end);
  __syncthreads();
  if (wave > 0) return;
  float total[V], out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    total[i] = 1.f;
    out[i] = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const int w = behind ? NW - 1 - k : k;
      const float pw = share.prod[0][w][lane * V + i];
      out[i] = gated_join(pw, share.end[0][w][lane * V + i], out[i]);
      total[i] = gated_product(total[i], pw);
    }
  }
  float* slot = p.agg + (b * p.nchunk + c) * 2 * p.D;
  gated_store<RP_F32, V>(reinterpret_cast<char*>(slot), ch * 4, total);
  gated_store<RP_F32, V>(reinterpret_cast<char*>(slot + p.D), ch * 4, out);
}

hipError_t launch_gated_fold(const GatedParams& p, const float* in, bool backward, hipStream_t st);

// Waves of a workgroup, at most where there are many, and always where the time axis is
// split among workgroups.
constexpr int kSplitWaves = 4;

}  // namespace rp
