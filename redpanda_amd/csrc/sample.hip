// Sampling of one token a row from logits, with temperature, top-k, top-p and
// min-p, from given uniform numbers; over the whole vocabulary or over a list
// of ids a row (a rollout's legal moves).
//
// The candidates of a row are its logits above -inf (NaN and ids outside the
// vocabulary are none).  Ordered by value, then by place in the row, with the
// weights w = exp((l - max) / T), a prefix of that order is kept:
//   top-k   the first k,
//   top-p   those whose weight before them is below top_p times that of the k,
//   min-p   those with w >= min_p;
// the first is always kept.  The token is the first kept one, in order of its
// place, at which the running sum of the kept weights exceeds u times their
// total.  T = 0 takes the first of the order.
//
// Weights are held as whole numbers, round(w 2^s) in 64 bits with 2^s up to
// 2^51 (less for rows above 2^11, so that no sum can pass 2^62): their sums are
// the same in any order, so a row's result does not depend on which thread or
// atomic came first, and every cut is an exact comparison of sums.  w comes
// from a 2^f polynomial in fp64, whose multiply-adds cost what fp32's do here:
// a border that falls between two tokens is then missed by about 1e-13 of the
// total, where fp32's 1e-7 would pick another token every few thousand rows.
//
// A cut is found without sorting: a histogram (counts or weights) over 1024
// steps of max - l, the step in which the running sum passes the threshold, and
// the order among that step's few elements by comparing each with all others.
// A step with more of them (equal logits, or an outlier that stretches the
// range) is split again by the elements' order keys, 10 bits at a time.

#include <type_traits>

#include "rp_device.h"
#include "rp_heads.h"

namespace rp {

namespace {

constexpr int kBins = 1024;
constexpr int kList = 256;

// A value's place in the order: larger is earlier.  The upper half orders the
// values (-0 as +0), the lower half the places, the first one largest.
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  uint32_t b = __float_as_uint(v);
  if (b == 0x80000000u) b = 0u;
  b ^= (b & 0x80000000u) ? 0xffffffffu : 0x80000000u;
  return ((uint64_t)b << 32) | ~(uint32_t)i;
}

struct RowWeights {
  float top;    // the largest logit
  float xmax;   // top - l beyond which a weight rounds to nothing
  float scale;  // histogram steps per unit of top - l
  double c;     // log2(e) / T
  double magic; // 2^(52 - s)

  __device__ __forceinline__ bool some(float v) const { return v == top || top - v <= xmax; }
  // exp((v - top) / T); `some(v)` holds
  __device__ __forceinline__ double weight(float v) const {
    const double y = v == top ? 0.0 : ((double)v - (double)top) * c;
    constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double t = y + kShift;
    const double f = y - (t - kShift);
    // (2^f - 1) / f on [-1/2, 1/2], interpolated at Chebyshev's nodes: the
    // power is right to 3.7e-14
    double q = 1.0203121063382838e-07;
    q = __builtin_fma(q, f, 1.3255224878668817e-06);
    q = __builtin_fma(q, f, 1.5252686846267769e-05);
    q = __builtin_fma(q, f, 0.00015403455852453838);
    q = __builtin_fma(q, f, 0.0013333558179043112);
    q = __builtin_fma(q, f, 0.009618129159402558);
    q = __builtin_fma(q, f, 0.055504108664760424);
    q = __builtin_fma(q, f, 0.2402265069581299);
    q = __builtin_fma(q, f, 0.6931471805599453);
    q = __builtin_fma(q, f, 1.0);
    const int k = (int)(uint32_t)__double_as_longlong(t);
    return __longlong_as_double(__double_as_longlong(q) + ((int64_t)k << 52));
  }
  // The whole number it is held as: the sum with 2^(52 - s) has w's bits down
  // to 2^-s, rounded, in its mantissa.
  __device__ __forceinline__ uint64_t fixed(double w) const {
    return (uint64_t)(__double_as_longlong(w + magic) - __double_as_longlong(magic));
  }
  __device__ __forceinline__ int bin(float v) const {
    const float x = v == top ? 0.f : top - v;
    return (int)fminf(x * scale, (float)(kBins - 1));
  }
};

template <int WAVES>
struct Scratch {
  uint64_t hist[kBins];
  uint64_t key[kList], mass[kList];
  uint64_t red[WAVES];
  uint64_t base;
  int bin, count;
};

template <int WAVES, class F>
__device__ __forceinline__ uint64_t block_reduce(uint64_t v, Scratch<WAVES>& s, F f) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) v = f(v, (uint64_t)__shfl_xor((unsigned long long)v, m));
  __syncthreads();
  if (threadIdx.x % kWave == 0) s.red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = s.red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) v = f(v, s.red[i]);
  return v;
}

struct Add {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a + b; }
};
struct Max {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
struct Min {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a < b ? a : b; }
};

// floor(u total), below total.  u 2^64 is a whole number for u from 2^-40 on, so
// that the product's upper half is exact: u on a border between two tokens takes
// the second, as the comparison of real numbers does.
__device__ __forceinline__ uint64_t draw_at(float u, uint64_t total) {
  const double v = fmin(fmax((double)u, 0.0), 1.0);
  return v < 1.0 ? __umul64hi((uint64_t)(v * 18446744073709551616.0), total) : total - 1;
}

// Running sum over the wave's lanes, each its own included.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, int lane) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const uint64_t o = __shfl_up((unsigned long long)v, m);
    if (lane >= m) v += o;
  }
  return v;
}

// The step of the histogram in which the running sum reaches thr: true, with
// the step in s.bin and the sum before it in s.base, or false when the whole
// sum is below thr.
template <int WAVES>
__device__ __forceinline__ bool find_step(Scratch<WAVES>& s, uint64_t thr) {
  constexpr int kPer = kBins / (WAVES * kWave);
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  uint64_t h[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    h[j] = s.hist[tid * kPer + j];
    sum += h[j];
  }
  const uint64_t incl = wave_scan(sum, lane);
  if (tid == 0) s.bin = -1;
  if (lane == kWave - 1) s.red[wave] = incl;
  __syncthreads();
  uint64_t before = incl - sum;
  for (int i = 0; i < wave; ++i) before += s.red[i];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (before < thr && before + h[j] >= thr) {
      s.bin = tid * kPer + j;
      s.base = before;
    }
    before += h[j];
  }
  __syncthreads();
  return s.bin >= 0;
}

// The key of the last element that is kept when those are kept whose counts
// (kMass: weights) before them are below thr, among the elements with keys from
// `floor` on; `floor` itself where nothing is cut.  `each(f)` calls f(value,
// place) for the thread's elements of the row.
template <bool kMass, int WAVES, class Each>
__device__ uint64_t cut(Scratch<WAVES>& s, const RowWeights& rw, uint64_t thr, uint64_t floor,
                        Each each) {
  const int tid = threadIdx.x;
  constexpr int kT = WAVES * kWave;
  auto unit = [&](float v) -> uint64_t { return kMass ? rw.fixed(rw.weight(v)) : 1; };
  __syncthreads();
  for (int i = tid; i < kBins; i += kT) s.hist[i] = 0;
  __syncthreads();
  each([&](float v, int i) {
    if (rw.some(v) && rank_key(v, i) >= floor)
      atomicAdd((unsigned long long*)&s.hist[rw.bin(v)], (unsigned long long)unit(v));
  });
  __syncthreads();
  if (!find_step(s, thr)) return floor;
  const int step = s.bin;
  uint64_t base = s.base, lo = floor, hi = ~0ull;
  int n;
  for (;;) {
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
    each([&](float v, int i) {
      if (!rw.some(v) || rw.bin(v) != step) return;
      const uint64_t key = rank_key(v, i);
      if (key < lo || key > hi) return;
      const int at = atomicAdd(&s.count, 1);
      if (at < kList) {
        s.key[at] = key;
        s.mass[at] = unit(v);
      }
    });
    __syncthreads();
    n = s.count;
    if (n <= kList) break;
    // too many: split their range of keys
    uint64_t kmax = 0, kmin = ~0ull;
    for (int i = tid; i < kBins; i += kT) s.hist[i] = 0;
    each([&](float v, int i) {
      if (!rw.some(v) || rw.bin(v) != step) return;
      const uint64_t key = rank_key(v, i);
      if (key < lo || key > hi) return;
      kmax = Max()(kmax, key);
      kmin = Min()(kmin, key);
    });
    kmax = block_reduce(kmax, s, Max());
    kmin = block_reduce(kmin, s, Min());
    const int bits = 64 - __clzll((long long)(kmax - kmin));
    const int shift = bits > 10 ? bits - 10 : 0;
    each([&](float v, int i) {
      if (!rw.some(v) || rw.bin(v) != step) return;
      const uint64_t key = rank_key(v, i);
      if (key < kmin || key > kmax) return;
      atomicAdd((unsigned long long*)&s.hist[(kmax - key) >> shift], (unsigned long long)unit(v));
    });
    __syncthreads();
    find_step(s, thr - base);  // it is reached: these elements' sum passes thr
    base += s.base;
    hi = kmax - ((uint64_t)s.bin << shift);
    lo = Max()(kmin, hi - (((uint64_t)1 << shift) - 1));
  }
  // each element's sum before it, from all the others
  uint64_t last = ~0ull;
  if (tid < n) {
    const uint64_t mine = s.key[tid];
    uint64_t before = base;
    for (int j = 0; j < n; ++j) before += s.key[j] > mine ? (kMass ? s.mass[j] : 1) : 0;
    if (before < thr) last = mine;
  }
  return block_reduce(last, s, Min());
}

}  // namespace

template <int WAVES, int DT>
__global__ __launch_bounds__(WAVES* kWave) void sample_kernel(SampleParams p) {
  __shared__ Scratch<WAVES> s;
  constexpr int kT = WAVES * kWave;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int n = p.n;
  for (int64_t row = blockIdx.x; row < p.R; row += gridDim.x) {
    const int64_t lbase = row * p.lsr, tbase = row * p.tsr;
    // the element at place i (-inf: no candidate)
    auto at = [&](int i) -> float {
      int64_t c = i;
      if (p.tokens != nullptr) {
        c = p.tokens[tbase + i];
        if (c < 0 || c >= p.V) return -__builtin_inff();
      }
      float v;
      if constexpr (DT == RP_F32)
        v = static_cast<const float*>(p.logits)[lbase + c];
      else if constexpr (DT == RP_BF16)
        v = __uint_as_float((uint32_t)static_cast<const uint16_t*>(p.logits)[lbase + c] << 16);
      else
        v = static_cast<float>(static_cast<const _Float16*>(p.logits)[lbase + c]);
      return v > -__builtin_inff() ? v : -__builtin_inff();
    };
    auto each = [&](auto f) {
      for (int i = tid; i < n; i += kT) {
        const float v = at(i);
        if (v > -__builtin_inff()) f(v, i);
      }
    };
    uint64_t first = 0, low = ~0ull;
    each([&](float v, int i) {
      const uint64_t key = rank_key(v, i);
      first = Max()(first, key);
      low = Min()(low, key);
    });
    first = block_reduce(first, s, Max());
    low = block_reduce(low, s, Min());
    const double T = p.T_row != nullptr ? (double)p.T_row[row] : p.T;
    const double tp = p.tp_row != nullptr ? (double)p.tp_row[row] : p.tp;
    const double mp = p.mp_row != nullptr ? (double)p.mp_row[row] : p.mp;
    const int64_t k = p.k_row != nullptr ? (int64_t)p.k_row[row] : p.k;
    const auto give = [&](int i, float logp) {
      p.ids[row] = i < 0 ? -1 : p.tokens != nullptr ? p.tokens[tbase + i] : i;
      if (p.logp != nullptr) p.logp[row] = logp;
    };
    const int best = (int)~(uint32_t)first;
    // no candidate; or the first of the order is the only one kept
    if (first == 0 || !(T > 0.0) || k == 1 || !(mp <= 1.0) || !(tp > 0.0)) {
      if (tid == 0) give(first == 0 ? -1 : best, first == 0 ? -__builtin_inff() : 0.f);
      continue;
    }
    RowWeights rw;
    rw.top = at(best);
    const float range = rw.top - at((int)~(uint32_t)low);
    rw.c = 1.4426950408889634 / T;
    rw.xmax = fminf((float)(36.1 * T), 3.4e38f);  // w < 2^-52
    rw.scale = (float)kBins / fminf(range, rw.xmax);
    rw.magic = __longlong_as_double((int64_t)(1023 + 52 - p.shift) << 52);
    uint64_t floor = 0;
    if (k > 0 && k < n) floor = cut<false>(s, rw, (uint64_t)k, floor, each);
    if (tp < 1.0) {
      uint64_t sum = 0;
      each([&](float v, int i) {
        if (rw.some(v) && rank_key(v, i) >= floor) sum += rw.fixed(rw.weight(v));
      });
      sum = block_reduce(sum, s, Add());
      floor = cut<true>(s, rw, (uint64_t)ceil(tp * (double)sum), floor, each);
    }
    // the draw: each wave sums a stretch of the row, and the one that u falls
    // into walks it again
    const auto kept = [&](int i, int end) -> uint64_t {
      if (i >= end) return 0;
      const float v = at(i);
      if (!(v > -__builtin_inff()) || !rw.some(v) || rank_key(v, i) < floor) return 0;
      const double w = rw.weight(v);
      return w >= mp ? rw.fixed(w) : 0;
    };
    const int stretch = ((n + WAVES - 1) / WAVES + kWave - 1) / kWave * kWave;
    const int from = wave * stretch < n ? wave * stretch : n;
    const int to = from + stretch < n ? from + stretch : n;
    uint64_t mine = 0;
    for (int i = from; i < to; i += kWave) mine += kept(i + lane, to);
    const uint64_t incl = wave_scan(mine, lane);
    __syncthreads();
    if (lane == kWave - 1) s.red[wave] = incl;
    __syncthreads();
    uint64_t before = 0, total = 0;
    for (int i = 0; i < WAVES; ++i) {
      if (i < wave) before += s.red[i];
      total += s.red[i];
    }
    const uint64_t stop = before + s.red[wave];
    const uint64_t want = draw_at(p.u[row], total);
    if (before <= want && want < stop) {
      for (int i = from; i < to; i += kWave) {
        const uint64_t run = before + wave_scan(kept(i + lane, to), lane);
        const uint64_t hit = __ballot(run > want);
        if (hit != 0) {
          const int l = __ffsll((unsigned long long)hit) - 1;
          if (lane == l) {
            const float v = at(i + l);
            const double x = v == rw.top ? 0.0 : ((double)v - (double)rw.top) / T;
            give(i + l, (float)(x - log((double)total * ldexp(1.0, -p.shift))));
          }
          break;
        }
        before = __shfl((unsigned long long)run, kWave - 1);
      }
    }
    __syncthreads();
  }
}

hipError_t launch_sample(const SampleParams& p, hipStream_t st) {
  if (p.R == 0) return hipSuccess;
  const dim3 grid((unsigned)(p.R < (1 << 20) ? p.R : (1 << 20)));
  auto go = [&](auto dt_tag) {
    constexpr int DT = decltype(dt_tag)::value;
    // many threads a row where the rows alone do not fill the card
    if (p.R < 512 && p.n > 2048)
      hipLaunchKernelGGL((sample_kernel<16, DT>), grid, dim3(16 * kWave), 0, st, p);
    else
      hipLaunchKernelGGL((sample_kernel<4, DT>), grid, dim3(4 * kWave), 0, st, p);
  };
  if (p.dt == RP_F32)
    go(std::integral_constant<int, RP_F32>{});
  else if (p.dt == RP_BF16)
    go(std::integral_constant<int, RP_BF16>{});
  else
    go(std::integral_constant<int, RP_F16>{});
  return hipGetLastError();
}

}  // namespace rp
