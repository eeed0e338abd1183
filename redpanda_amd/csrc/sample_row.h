// Device code of the sampling kernels (sample.hip has what they compute and why;
// sample_wide.hip the rows that several workgroups share).
#pragma once

#include "rp_heads.h"
#include "rp_rows.h"

namespace rp {

namespace {

constexpr int kGroups = 256;  // groups whose largest values bound the k-th
constexpr int kSegments = 8;  // of a wave's stretch, for the draw
// A workgroup's LDS.  A wave that has a row for itself takes half of what
// several take together: 8 KB, so that LDS holds as many rows on a CU as the
// registers do (16; with 16 KB it held 9).
constexpr int list_of(int waves) { return waves == 1 ? 256 : waves == 4 ? 1024 : 2048; }
// the largest top-k that is listed: as many as bound a list that mostly fits it
constexpr int listed_of(int waves) {
  return 2 * waves * kWave < list_of(waves) ? 2 * waves * kWave : list_of(waves) - 1;
}
// bits of an exact histogram's steps
constexpr int bits_of(int waves) { return waves == 1 ? 9 : waves == 4 ? 10 : 11; }
constexpr int bins_of(int waves) { return 1 << bits_of(waves); }
constexpr int fine_of(int waves) { return 2 * bins_of(waves); }   // the fp32 one, in the same words

// A value's place in the order: larger is earlier.  The upper half orders the
// values (-0 as +0), the lower half the places, the first one largest.
__device__ __forceinline__ uint32_t value_key(float v) {
  uint32_t b = __float_as_uint(v);
  if (b == 0x80000000u) b = 0u;
  return b ^ ((b & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t rank_key(float v, int i) {
  return ((uint64_t)value_key(v) << 32) | ~(uint32_t)i;
}
__device__ __forceinline__ int key_place(uint64_t k) { return (int)~(uint32_t)k; }

struct RowWeights {
  float top;     // the largest logit
  float xmax;    // top - l beyond which a weight rounds to nothing
  float scale;   // exact histograms' steps per unit of top - l
  float fscale;  // the fp32 one's
  float c32;     // log2(e) / T
  double topd, c;
  double magic;  // 2^(52 - s)

  __device__ __forceinline__ RowWeights(const SampleParams& p, float t, double T)
      : top(t), topd((double)t), c(1.4426950408889634 / T) {
    c32 = (float)c;
    xmax = (float)(36.1 * T);  // w < 2^-52 (infinite where the type's lowest value has a weight)
    magic = __longlong_as_double((int64_t)(1023 + 52 - p.shift) << 52);
  }
  // log(w / total)
  __device__ __forceinline__ float log_share(float v, uint64_t total, double T, int shift) const {
    return (float)(((double)v - topd) / T - log((double)total * ldexp(1.0, -shift)));
  }

  __device__ __forceinline__ bool some(float v) const { return top - v <= xmax; }
  // exp((v - top) / T); 2^-100 at most for what lies further down than that
  __device__ __forceinline__ double weight(float v) const {
    const double y = fmax(((double)v - topd) * c, -100.0);
    constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double t = y + kShift;
    const double f = y - (t - kShift);
    // (2^f - 1) / f on [-1/2, 1/2], interpolated at Chebyshev's nodes: the
    // power is right to 2.2e-12
    double q = 1.325080551750225e-06;
    q = __builtin_fma(q, f, 1.5303700711365693e-05);
    q = __builtin_fma(q, f, 0.00015403475186530786);
    q = __builtin_fma(q, f, 0.0013333478473685416);
    q = __builtin_fma(q, f, 0.00961812913523614);
    q = __builtin_fma(q, f, 0.055504109063258665);
    q = __builtin_fma(q, f, 0.24022650695888503);
    q = __builtin_fma(q, f, 0.6931471805568324);
    q = __builtin_fma(q, f, 1.0);
    const uint64_t k = (uint64_t)__double_as_longlong(t) << 52;
    return __longlong_as_double(__double_as_longlong(q) + (int64_t)k);
  }
  // The whole number w is held as: the sum with 2^(52 - s) has w's bits down to
  // 2^-s, rounded, in its mantissa.  `raw` leaves 2^(52 - s)'s own bits in.
  __device__ __forceinline__ uint64_t raw(double w) const {
    return (uint64_t)__double_as_longlong(w + magic);
  }
  __device__ __forceinline__ uint64_t base() const { return (uint64_t)__double_as_longlong(magic); }
  __device__ __forceinline__ uint64_t fixed(double w) const { return raw(w) - base(); }
  template <int BINS>
  __device__ __forceinline__ int bin(float v) const {
    return (int)fminf((top - v) * scale, (float)(BINS - 1));
  }
};

template <int WAVES>
struct Scratch {
  static constexpr int kBins = bins_of(WAVES), kFineBins = fine_of(WAVES), kList = list_of(WAVES);
  union {
    uint64_t hist[kBins];
    uint32_t fine[kFineBins];
    uint32_t groups[kGroups];
    uint64_t okey[kList];  // a list in order
  };
  uint64_t key[kList], mass[kList];
  uint64_t seg[WAVES * kSegments];  // kept weights by segment
  uint64_t red[2 * WAVES];
  uint64_t base;
  int bin, hi, count;
};

struct Add {
  template <class V>
  __device__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  template <class V>
  __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct Min {
  template <class V>
  __device__ V operator()(V a, V b) const { return a < b ? a : b; }
};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int l) { return __shfl((unsigned long long)v, l); }

// A value moved between lanes, word by word.
template <class V, class M>
__device__ __forceinline__ V by_words(V v, M move) {
  if constexpr (sizeof(V) == 8) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(V, (uint64_t)move((uint32_t)(b >> 32)) << 32 | move((uint32_t)b));
  } else {
    return __builtin_bit_cast(V, move(__builtin_bit_cast(uint32_t, v)));
  }
}
template <int kCtrl, class V>
__device__ __forceinline__ V dpp(V v) {
  return by_words(v, [](uint32_t w) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)w, kCtrl, 0xf, 0xf, true);
  });
}

// f over the wave's lanes, the same in each: exchanges within rows of 16 lanes,
// then of whole rows and halves, without LDS.
template <class V, class F>
__device__ __forceinline__ V wave_all(V v, F f) {
  v = f(v, dpp<0xb1>(v));   // quad_perm [1, 0, 3, 2]
  v = f(v, dpp<0x4e>(v));   // quad_perm [2, 3, 0, 1]
  v = f(v, dpp<0x141>(v));  // row_half_mirror
  v = f(v, dpp<0x140>(v));  // row_mirror
  const auto first16 = [](uint32_t w) { return __builtin_amdgcn_permlane16_swap(w, w, false, false)[0]; };
  const auto second16 = [](uint32_t w) { return __builtin_amdgcn_permlane16_swap(w, w, false, false)[1]; };
  v = f(by_words(v, first16), by_words(v, second16));
  const auto first32 = [](uint32_t w) { return __builtin_amdgcn_permlane32_swap(w, w, false, false)[0]; };
  const auto second32 = [](uint32_t w) { return __builtin_amdgcn_permlane32_swap(w, w, false, false)[1]; };
  return f(by_words(v, first32), by_words(v, second32));
}

template <int WAVES, class V, class F>
__device__ __forceinline__ V block_reduce(V v, Scratch<WAVES>& s, F f) {
  v = wave_all(v, f);
  if constexpr (WAVES == 1) return v;
  V* red = reinterpret_cast<V*>(s.red);
  __syncthreads();
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) v = f(v, red[i]);
  return v;
}

// Sums of two values over the workgroup.
template <int WAVES>
__device__ __forceinline__ void block_sums(uint64_t& a, uint64_t& b, Scratch<WAVES>& s) {
  a = wave_all(a, Add());
  b = wave_all(b, Add());
  if constexpr (WAVES > 1) {
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
      s.red[2 * (threadIdx.x / kWave)] = a;
      s.red[2 * (threadIdx.x / kWave) + 1] = b;
    }
    __syncthreads();
    a = s.red[0];
    b = s.red[1];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
      a += s.red[2 * i];
      b += s.red[2 * i + 1];
    }
  }
}

// floor(u total), below total.  u 2^64 is a whole number for u from 2^-40 on, so
// that the product's upper half is exact: u on a border between two tokens takes
// the second, as the comparison of real numbers does.
__device__ __forceinline__ uint64_t draw_at(float u, uint64_t total) {
  const double v = fmin(fmax((double)u, 0.0), 1.0);
  return v < 1.0 ? __umul64hi((uint64_t)(v * 18446744073709551616.0), total) : total - 1;
}

// Running sum over the wave's lanes, each its own included.
template <class V>
__device__ __forceinline__ V wave_scan(V v, int lane) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    V o;
    if constexpr (sizeof(V) == 8)
      o = __shfl_up((unsigned long long)v, m);
    else
      o = __shfl_up(v, m);
    if (lane >= m) v += o;
  }
  return v;
}

// The step of a histogram in which the running sum reaches thr_of(total): true,
// with the step in s.bin and the sum before it in s.base, or false when the whole
// sum is below it.  With `grains`, a histogram of rounded weights: the first and
// the last step that the sums so many grains and 2^-18 of the total below and
// above the threshold fall into, in s.bin and s.hi.
template <int BINS, int WAVES, class H, class F>
__device__ __forceinline__ bool find_step(Scratch<WAVES>& s, const H* hist, F thr_of,
                                          uint64_t grains = 0) {
  constexpr int kPer = BINS / (WAVES * kWave);
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  H h[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    h[j] = hist[tid * kPer + j];
    sum += h[j];
  }
  const H incl = wave_scan(sum, lane);
  if (tid == 0) {
    s.bin = -1;
    s.hi = BINS - 1;
  }
  if (lane == kWave - 1) s.red[wave] = incl;
  __syncthreads();
  uint64_t before = incl - sum, total = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i < wave) before += s.red[i];
    total += s.red[i];
  }
  const uint64_t thr = thr_of(total), margin = grains != 0 ? grains + (total >> 18) : 0;
  const uint64_t low = thr > margin ? thr - margin : 1, high = thr + margin;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (before < low && before + h[j] >= low) {
      s.bin = tid * kPer + j;
      s.base = before;
    }
    if (margin != 0 && before < high && before + h[j] >= high) s.hi = tid * kPer + j;
    before += h[j];
  }
  __syncthreads();
  return s.bin >= 0;
}

// The elements of a row that a thread holds or reads: `blocks` blocks of eight,
// a wave's stretch being blocks * 512 elements in segments of `per` blocks.
// NBLK of them in registers, or (NBLK = 0) as many as the row's length asks for,
// read anew at each look.  NaN are left as they are: every look compares in a
// way that passes them by.  Places past the row read as -inf.
// WAVES is the number of waves that share the row: a workgroup's, or for the rows
// of sample_wide.hip those of several.
template <int WAVES, int NBLK, int ES>
struct Row {
  static constexpr int kWaves = WAVES;
  static constexpr int kSegs = NBLK > 0 ? NBLK : WAVES > 16 ? 2 : kSegments;
  const SampleParams& p;
  int64_t lbase, tbase;
  int n, blocks, per;
  int first;      // the place of the thread's first element
  bool only_inf;  // +inf is there: what is not, is no candidate
  float v[NBLK > 0 ? NBLK : 1][8];

  __device__ __forceinline__ Row(const SampleParams& pp, int64_t row, bool inf = false)
      : Row(pp, row, inf, __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave)) {}
  __device__ __forceinline__ Row(const SampleParams& pp, int64_t row, bool inf, int wave)
      : p(pp), only_inf(inf) {
    lbase = row * p.lsr;
    tbase = row * p.tsr;
    n = p.n;
    blocks = NBLK > 0 ? NBLK : (n + WAVES * kWave * 8 - 1) / (WAVES * kWave * 8);
    per = NBLK > 0 ? 1 : (blocks + 2 * kSegs - 1) / (2 * kSegs) * 2;  // (walked in pairs)
    at_wave(wave);
    if constexpr (NBLK > 0) {
#pragma unroll
      for (int j = 0; j < NBLK; ++j) read(j, v[j]);
    }
  }
  __device__ __forceinline__ void at_wave(int w) {
    first = w * blocks * (kWave * 8) + (int)(threadIdx.x % kWave) * 8;
  }
  __device__ __forceinline__ int place(int j) const { return first + j * (kWave * 8); }
  // The segment (of the workgroup's) that a place is in.
  __device__ __forceinline__ int segment(int at) const {
    const int b = at / (kWave * 8), wave = b / blocks;
    return wave * kSegs + (b - wave * blocks) / per;
  }
  __device__ __forceinline__ void read(int j, float (&x)[8]) const {
    const int at = place(j);
    constexpr float kNone = -__builtin_inff();
    if (p.tokens != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = kNone;
        if (at + i >= n) continue;
        const int c = p.tokens[tbase + at + i];
        if (c >= 0 && c < p.V) x[i] = load_in(p.logits, lbase + c, p.dt);
      }
    } else {
      to_floats(load_raw8<ES>(static_cast<const char*>(p.logits) + lbase * ES, at, n), p.dt, x);
      if (at + 8 > n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = at + i < n ? x[i] : kNone;
      }
    }
  }
  // f(values, place of the first) for the thread's blocks, end(segment) after
  // each segment.  The empty asm and the scheduling barrier keep the compiler
  // from holding what one look computes of a value (weights, steps) in registers
  // for the next, and from working on all blocks at once: that takes more
  // registers than there are.
  template <class F, class E>
  __device__ __forceinline__ void walk(F f, E end) {
    if constexpr (NBLK > 0) {
#pragma unroll
      for (int j = 0; j < NBLK; ++j) {
        asm volatile("" : "+v"(v[j][0]), "+v"(v[j][1]), "+v"(v[j][2]), "+v"(v[j][3]), "+v"(v[j][4]),
                     "+v"(v[j][5]), "+v"(v[j][6]), "+v"(v[j][7]));
        asm volatile("" : "+v"(first));
        f(v[j], place(j));
        end(j);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // two buffers: one block's loads are in flight while the other is looked at
      float x[8], y[8];
      read(0, x);
      int j = 0;
      for (int g = 0; g < kSegs; ++g) {
        for (int b = 0; b < per && j < blocks; b += 2, j += 2) {
          if (j + 1 < blocks) read(j + 1, y);
          keep_inf(x);
          f(x, place(j));
          if (j + 2 < blocks) read(j + 2, x);
          if (j + 1 < blocks) {
            keep_inf(y);
            f(y, place(j + 1));
          }
        }
        end(g);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void blocks_of(F f) {
    walk(f, [](int) {});
  }
  // f(values, place) for the blocks of one segment of the wave, until it returns
  // true
  template <class F>
  __device__ __forceinline__ void segment_of(int g, F f) {
    if constexpr (NBLK > 0) {
#pragma unroll
      for (int j = 0; j < NBLK; ++j)
        if (j == g) f(v[j], place(j));
    } else {
      for (int j = g * per; j < (g + 1) * per && j < blocks; ++j) {
        float x[8];
        read(j, x);
        keep_inf(x);
        if (f(x, place(j))) return;
      }
    }
  }
  // f(value, place) for the thread's candidates
  template <class F>
  __device__ __forceinline__ void each(F f) {
    blocks_of([&](const float (&x)[8], int at) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (x[i] > -__builtin_inff()) f(x[i], at + i);
    });
  }
  __device__ __forceinline__ void keep_inf(float (&x)[8]) const {
    if (only_inf) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] == __builtin_inff() ? 0.f : -__builtin_inff();
    }
  }
  // From here on only the +inf are candidates, as zeros.
  __device__ __forceinline__ void take_inf() {
    only_inf = true;
    if constexpr (NBLK > 0) {
#pragma unroll
      for (int j = 0; j < NBLK; ++j) keep_inf(v[j]);
    }
  }
};

// The last kept element of a prefix: elements stand before it, or are it.
struct Floor {
  float value;
  int at;
  __device__ __forceinline__ explicit Floor(uint64_t key)
      : value(key_value((uint32_t)(key >> 32))), at(key_place(key)) {}
  __device__ __forceinline__ bool keeps(float v, int i) const {
    return v > value || (v == value && i <= at);
  }
};

// The key of the last element that is kept when those are kept whose counts
// (kMass: weights) before them are below thr, among the elements with keys from
// `floor` on; `floor` itself where nothing is cut.  Exact for every row.
template <bool kMass, int WAVES, class R>
__device__ __forceinline__ uint64_t cut(Scratch<WAVES>& s, const RowWeights& rw, R& row, uint64_t thr,
                                     uint64_t floor) {
  const int tid = threadIdx.x;
  constexpr int kT = WAVES * kWave, kBins = bins_of(WAVES), kBits = bits_of(WAVES), kList = list_of(WAVES);
  auto unit = [&](float v) -> uint64_t { return kMass ? rw.fixed(rw.weight(v)) : 1; };
  __syncthreads();
  for (int i = tid; i < kBins; i += kT) s.hist[i] = 0;
  __syncthreads();
  row.each([&](float v, int i) {
    if (rw.some(v) && rank_key(v, i) >= floor)
      atomicAdd((unsigned long long*)&s.hist[rw.template bin<kBins>(v)], (unsigned long long)unit(v));
  });
  __syncthreads();
  if (!find_step<kBins>(s, s.hist, [&](uint64_t) { return thr; })) return floor;
  const int step = s.bin;
  uint64_t base = s.base, lo = floor, hi = ~0ull;
  int n;
  for (;;) {
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
    row.each([&](float v, int i) {
      if (!rw.some(v) || rw.template bin<kBins>(v) != step) return;
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
    row.each([&](float v, int i) {
      if (!rw.some(v) || rw.template bin<kBins>(v) != step) return;
      const uint64_t key = rank_key(v, i);
      if (key < lo || key > hi) return;
      kmax = Max()(kmax, key);
      kmin = Min()(kmin, key);
    });
    kmax = block_reduce(kmax, s, Max());
    kmin = block_reduce(kmin, s, Min());
    const int bits = 64 - __clzll((long long)(kmax - kmin));
    const int shift = bits > kBits ? bits - kBits : 0;
    __syncthreads();
    row.each([&](float v, int i) {
      if (!rw.some(v) || rw.template bin<kBins>(v) != step) return;
      const uint64_t key = rank_key(v, i);
      if (key < kmin || key > kmax) return;
      atomicAdd((unsigned long long*)&s.hist[(kmax - key) >> shift], (unsigned long long)unit(v));
    });
    __syncthreads();
    find_step<kBins>(s, s.hist, [&](uint64_t) { return thr - base; });  // it is reached: these elements' sum passes thr
    base += s.base;
    hi = kmax - ((uint64_t)s.bin << shift);
    lo = Max()(kmin, hi - (((uint64_t)1 << shift) - 1));
  }
  // each element's sum before it, from all the others
  uint64_t last = ~0ull;
  for (int e = tid; e < n; e += kT) {
    const uint64_t mine = s.key[e];
    uint64_t before = base;
    for (int j = 0; j < n; ++j) before += s.key[j] > mine ? (kMass ? s.mass[j] : 1) : 0;
    if (before < thr) last = Min()(last, mine);
  }
  return block_reduce(last, s, Min());
}

// Lists the elements from `bound` on: false where they are too many.
template <int WAVES, class R>
__device__ __forceinline__ bool gather(Scratch<WAVES>& s, R& row, float bound) {
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  row.blocks_of([&](const float (&x)[8], int at) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (x[i] >= bound && x[i] > -__builtin_inff()) {
        const int e = atomicAdd(&s.count, 1);
        if (e < s.kList) s.key[e] = rank_key(x[i], at + i);
      }
    }
  });
  __syncthreads();
  return s.count <= s.kList;
}

// s.okey: the listed keys in order, by how many are ahead of each, or for a long
// list by a bitonic network in LDS.  Comparing takes n steps without a barrier
// (16 cycles each, 1 us for 190 elements); the network 28 to 66, with a barrier
// of all the waves in each (200 cycles for one wave, 400 for sixteen).
template <int WAVES>
__device__ __forceinline__ void order_list(Scratch<WAVES>& s) {
  constexpr int kT = WAVES * kWave;
  const int tid = threadIdx.x, n = s.count;
  if (n > (WAVES == 1 ? 2 : 8) * kWave) {
    int len = 2 * kWave;
    while (len < n) len <<= 1;
    for (int i = tid; i < len; i += kT) s.okey[i] = i < n ? s.key[i] : 0;
    for (int kk = 2; kk <= len; kk <<= 1) {
      for (int j = kk >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int t = tid; t < len / 2; t += kT) {
          const int i = 2 * t - (t & (j - 1));
          const uint64_t a = s.okey[i], b = s.okey[i + j];
          const bool swap = (a < b) == ((i & kk) == 0);  // larger ones first
          s.okey[i] = swap ? b : a;
          s.okey[i + j] = swap ? a : b;
        }
      }
    }
  } else {
    for (int i = tid; i < n; i += kT) {
      const uint64_t mine = s.key[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += s.key[j] > mine ? 1 : 0;
      s.okey[rank] = mine;
    }
  }
  __syncthreads();
}

// The key of the last kept element of the list's first m, `ahead` of weight
// standing before them: kept are those with w >= mp and a weight before them
// below thr_of(the whole sum, theirs included).  Their weights are added to
// s.seg.  0 where the threshold is not reached in the list (*reached false).
template <int WAVES, class R, class F>
__device__ __forceinline__ uint64_t cut_list(Scratch<WAVES>& s, const RowWeights& rw, R& row, int m,
                                             uint64_t ahead, double mp, F thr_of, bool* reached) {
  constexpr int kT = WAVES * kWave;
  constexpr int kPer = (list_of(WAVES) + kT - 1) / kT;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  order_list(s);
  // weights in order, and their running sum: thread t takes kPer in a row
  uint64_t q[kPer], sum = 0;
  uint32_t kept = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int i = tid * kPer + e;
    q[e] = 0;
    if (i < m) {
      const double w = rw.weight(key_value((uint32_t)(s.okey[i] >> 32)));
      q[e] = rw.fixed(w);
      kept |= w >= mp ? 1u << e : 0u;
    }
    sum += q[e];
  }
  const uint64_t incl = wave_scan(sum, lane);
  if (lane == kWave - 1) s.red[wave] = incl;
  __syncthreads();
  uint64_t before = ahead + incl - sum, all = ahead;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += s.red[w];
    all += s.red[w];
  }
  const uint64_t thr = thr_of(all);
  *reached = ahead < thr && thr <= all;
  uint64_t last = ~0ull;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if ((kept >> e & 1) && before < thr) {
      last = s.okey[tid * kPer + e];
      atomicAdd((unsigned long long*)&s.seg[row.segment(key_place(last))], (unsigned long long)q[e]);
    }
    before += q[e];
  }
  return block_reduce(last, s, Min());
}

// The same from a list that holds all that can be kept.
template <int WAVES, class R>
__device__ __forceinline__ uint64_t cut_all(Scratch<WAVES>& s, const RowWeights& rw, R& row, int64_t k,
                                            double tp, double mp) {
  for (int i = threadIdx.x; i < R::kWaves * R::kSegs; i += WAVES * kWave) s.seg[i] = 0;
  const int n = s.count;
  bool reached;
  return cut_list(
      s, rw, row, k > 0 && k < n ? (int)k : n, 0, mp,
      [&](uint64_t all) { return tp < 1.0 ? (uint64_t)ceil(tp * (double)all) : all; }, &reached);
}

// The fp32 weights of a thread's elements, in grains, into the histogram in s.fine.
template <int WAVES, class R>
__device__ __forceinline__ void fine_weights(Scratch<WAVES>& s, const RowWeights& rw, R& row, float grain) {
  constexpr int kT = WAVES * kWave, kFineBins = fine_of(WAVES);
  const int tid = threadIdx.x, lane = tid % kWave;
  __syncthreads();
  for (int i = tid; i < kFineBins; i += kT) s.fine[i] = 0;
  __syncthreads();
  // rounded up or down by a lane's own share, so that weights below a grain are
  // not lost on the whole
  const float dither = ((float)(lane * 39 % kWave) + 0.5f) * (1.f / kWave);
  row.blocks_of([&](const float (&x)[8], int) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (the maximum and the minimum turn a NaN into nothing, in the last step)
      const float l = rw.top - x[i];
      const uint32_t q = (uint32_t)fmaxf(ffma(exp2_hw(l * -rw.c32), grain, dither), 0.f);
      if (q != 0) atomicAdd(&s.fine[(int)fminf(l * rw.fscale, (float)(kFineBins - 1))], q);
    }
  });
  __syncthreads();
}

// A grain that lets the histogram's sums reach a part of 2^32, by the total as a
// sample gives it (n, the most there can be, where it does not).
__device__ __forceinline__ float grain_of(float sampled, int n) {
  const float most = sampled >= 0.f && 32.f * sampled < (float)n ? 32.f * (sampled + 1.f) : (float)n;
  return 3e9f / fmaxf(most, 2.f);
}

// The steps [lo, hi) of that histogram that the cut falls into, as (top - l)
// fscale (the last step holds what lies beyond, too); false without one.
// The histogram's sums are off by the roundings to grains (up to sqrt(n) / 2 of
// them on the whole) and by fp32's.  Equal values lie in lumps with empty steps
// between, so the steps follow from the sums, not the other way.
template <int WAVES>
__device__ __forceinline__ bool cut_steps(Scratch<WAVES>& s, int n, double tp, float* lo, float* hi) {
  constexpr int kFineBins = fine_of(WAVES);
  const uint64_t grains = (uint64_t)(3.f * sqrtf((float)n)) + 16;
  if (!find_step<kFineBins>(
          s, s.fine, [&](uint64_t all) { return (uint64_t)ceil(tp * (double)all); }, grains))
    return false;
  *lo = (float)s.bin;
  *hi = s.hi < kFineBins - 1 ? (float)(s.hi + 1) : __builtin_inff();
  return true;
}

// Exact weights of a thread's elements: all of them (*sum), those before the
// steps (*ahead, and by segment in `seg`, the wave's), and a list of those in
// them.  kMin: those that min-p leaves, too, by segment in min_seg.
template <bool kMin, int WAVES, class R>
__device__ __forceinline__ void exact_weights(Scratch<WAVES>& s, const RowWeights& rw, R& row, float lo,
                                              float hi, uint64_t* seg, uint64_t* sum, uint64_t* ahead,
                                              double mp, uint64_t* min_seg) {
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  uint64_t all = 0, before = 0, part = 0, min_part = 0;
  const uint64_t base = rw.base();
  row.walk(
      [&](const float (&x)[8], int at) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = (rw.top - x[i]) * rw.fscale;
          const double weight = rw.weight(x[i]);
          const uint64_t q = rw.raw(weight);
          all += q;
          part += y[i] < lo ? q : base;
          if constexpr (kMin) min_part += weight >= mp ? q : base;
        }
        all -= 8 * base;
        part -= 8 * base;
        if constexpr (kMin) min_part -= 8 * base;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!(y[i] < lo) && y[i] < hi && x[i] > -__builtin_inff()) {
            const int e = atomicAdd(&s.count, 1);
            if (e < s.kList) s.key[e] = rank_key(x[i], at + i);
          }
        }
      },
      [&](int g) {
        before += part;
        part = wave_all(part, Add());
        if (threadIdx.x % kWave == 0) seg[g] = part;
        part = 0;
        if constexpr (kMin) {
          min_part = wave_all(min_part, Add());
          if (threadIdx.x % kWave == 0) min_seg[g] = min_part;
          min_part = 0;
        }
      });
  *sum = all;
  *ahead = before;
}

// The key of the nucleus' last element, or 0 where the list does not tell; what
// of the list it keeps is added to s.seg.
template <int WAVES, class R>
__device__ __forceinline__ uint64_t nucleus_cut(Scratch<WAVES>& s, const RowWeights& rw, R& row, double tp,
                                                uint64_t sum, uint64_t ahead) {
  const int n = s.count;
  if (n > s.kList) return 0;
  bool reached;
  const uint64_t last = cut_list(
      s, rw, row, n, ahead, 0.0, [&](uint64_t) { return (uint64_t)ceil(tp * (double)sum); }, &reached);
  return reached ? last : 0;
}

// A nucleus of the whole row: the key of its last element, or 0 where this does
// not tell.  Leaves its weights' sums in s.seg.
template <int WAVES, class R>
__device__ __forceinline__ uint64_t nucleus(Scratch<WAVES>& s, const RowWeights& rw, R& row, double tp,
                                            float grain) {
  float lo, hi;
  uint64_t sum, ahead;
  fine_weights(s, rw, row, grain);
  if (!cut_steps(s, row.n, tp, &lo, &hi)) return 0;
  exact_weights<false>(s, rw, row, lo, hi, &s.seg[threadIdx.x / kWave * R::kSegs], &sum, &ahead, 0.0,
                       nullptr);
  block_sums(sum, ahead, s);
  __syncthreads();
  return nucleus_cut(s, rw, row, tp, sum, ahead);
}

// The kept weights' sums by segment, of the elements from `floor` on (0: all)
// that min-p leaves.  `bound`: a value below which nothing is kept, where few
// elements are: their weights alone are taken.
// `seg`: the wave's.
template <class R>
__device__ __forceinline__ void segment_weights(const RowWeights& rw, R& row, uint64_t floor, double mp,
                                                float bound, uint64_t* seg) {
  const Floor fl(floor);
  uint64_t sum = 0;
  const auto end = [&](int g) {
    sum = wave_all(sum, Add());
    if (threadIdx.x % kWave == 0) seg[g] = sum;
    sum = 0;
  };
  __syncthreads();
  if (floor == 0 && !(mp > 0.0)) {
    row.walk(
        [&](const float (&x)[8], int) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += rw.raw(rw.weight(x[i]));
          sum -= 8 * rw.base();
        },
        end);
  } else {
    row.walk(
        [&](const float (&x)[8], int at) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (!(x[i] >= bound)) continue;
            const double w = rw.weight(x[i]);
            sum += (floor == 0 || fl.keeps(x[i], at + i)) && w >= mp ? rw.fixed(w) : 0;
          }
        },
        end);
  }
}

// The token, from the segments' sums: the wave whose segment u falls into looks
// at that again.
template <int WAVES, class R, class G>
__device__ __forceinline__ void draw(Scratch<WAVES>& s, const RowWeights& rw, R& row, uint64_t floor,
                                     double mp, float u, G give) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const Floor fl(floor);
  __syncthreads();
  // (two segments a lane: sixteen waves' eight are the most)
  constexpr int kAll = R::kWaves * R::kSegs;
  const uint64_t a = 2 * lane < kAll ? s.seg[2 * lane] : 0;
  const uint64_t b = 2 * lane + 1 < kAll ? s.seg[2 * lane + 1] : 0;
  const uint64_t incl = wave_scan(a + b, lane);
  const uint64_t total = shfl64(incl, kWave - 1);
  const uint64_t want = draw_at(u, total);
  const uint64_t past = __ballot(incl > want);
  if (past == 0) {
    // The largest value is kept and weighs 2^shift, so that some segment holds u
    // unless the logits are written while they are looked at.
    if (threadIdx.x == 0) give(-1, -__builtin_inff(), 1);
    return;
  }
  const int l = __ffsll((unsigned long long)past) - 1;
  uint64_t before = shfl64(incl - a - b, l);
  const uint64_t head = shfl64(a, l);
  int g = 2 * l;
  if (before + head <= want) {
    before += head;
    ++g;
  }
  if (g / R::kSegs % WAVES != wave) return;
  if constexpr (R::kWaves != WAVES) row.at_wave(g / R::kSegs);
  row.segment_of(g % R::kSegs, [&](const float (&x)[8], int at) {
    uint64_t q[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double w = rw.weight(x[i]);
      q[i] = (floor == 0 || fl.keeps(x[i], at + i)) && w >= mp ? rw.fixed(w) : 0;
      sum += q[i];
    }
    const uint64_t run = before + wave_scan(sum, lane);
    const uint64_t hit = __ballot(run > want);
    before = shfl64(run, kWave - 1);
    if (hit == 0) return false;
    if (lane == __ffsll((unsigned long long)hit) - 1) {
      uint64_t from = run - sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (from <= want && want < from + q[i]) give(at + i, x[i], total);
        from += q[i];
      }
    }
    return true;
  });
}

// The k-th largest of the groups' keys, or a little below it (the lower 12 bits
// zero): found bit by bit from how many reach it.  One wave, four keys a lane.
__device__ __forceinline__ uint32_t kth_of_groups(const uint32_t (&g)[4], int k) {
  uint32_t bound = 0;
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t t = bound | (1u << bit);
    int reach = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) reach += __popcll(__ballot(g[i] >= t));
    if (reach >= k) bound = t;
  }
  return bound;
}

// The same over every thread's four groups.
template <int WAVES>
__device__ __forceinline__ uint32_t kth_of_all(Scratch<WAVES>& s, const uint32_t (&g)[4], int k) {
  uint32_t bound = 0;
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t t = bound | (1u << bit);
    int reach = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) reach += __popcll(__ballot(g[i] >= t));
    uint32_t* count = reinterpret_cast<uint32_t*>(s.red) + (bit & 1) * WAVES;
    if (threadIdx.x % kWave == 0) count[threadIdx.x / kWave] = reach;
    __syncthreads();
    reach = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) reach += count[w];
    if (reach >= k) bound = t;
  }
  __syncthreads();
  return bound;
}

struct Settings {
  double T, tp, mp;
  int64_t k;
  float u;
  __device__ __forceinline__ Settings(const SampleParams& p, int64_t r) {
    T = p.T_row != nullptr ? (double)p.T_row[r] : p.T;
    // (infinity times the logarithm of a min-p of 1 would be a NaN; all weights are 1
    // from far below this on)
    if (T > 1e300) T = 1e300;
    tp = p.tp_row != nullptr ? (double)p.tp_row[r] : p.tp;
    mp = p.mp_row != nullptr ? (double)p.mp_row[r] : p.mp;
    k = p.k_row != nullptr ? (int64_t)p.k_row[r] : p.k;
    u = p.u[r];
  }
  // The first of the order is the only one kept.
  __device__ __forceinline__ bool first_only() const {
    return !(T > 0.0) || k == 1 || !(mp <= 1.0) || !(tp > 0.0);
  }
};

__device__ __forceinline__ void put_token(const SampleParams& p, int64_t r, int i, float logp) {
  p.ids[r] = i < 0 ? -1 : p.tokens != nullptr ? p.tokens[r * p.tsr + i] : i;
  if (p.logp != nullptr) p.logp[r] = logp;
}

// A value below which nothing is kept: min-p's bound (a little below it), or the
// last kept one's.
__device__ __forceinline__ float keep_bound(const RowWeights& rw, double T, double mp, uint64_t floor) {
  const double b = rw.topd + T * log(mp);
  const float least = mp > 0.0 ? (float)(b - 1e-6 * (fabs(b) + T)) : -__builtin_inff();
  return floor != 0 ? fmaxf(least, Floor(floor).value) : least;
}

// The first look at a thread's elements: the largest value by four groups, the
// least, and of every fourth element the weights against the first largest at
// hand.
struct RowLook {
  float most[4], least, ref, some, c32;

  template <class R>
  __device__ __forceinline__ void take(R& row, double T) {
    constexpr float kInf = __builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i) most[i] = -kInf;
    least = kInf;
    ref = -kInf;
    some = 0.f;
    c32 = (float)(1.4426950408889634 / T);
    row.blocks_of([&](const float (&x)[8], int) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        most[i % 4] = x[i] > most[i % 4] ? x[i] : most[i % 4];
        // (of a quarter of them: it only scales the histograms' steps)
        if (i % 4 == 0) least = x[i] > -kInf && x[i] < least ? x[i] : least;
      }
      if (ref == -kInf) ref = wave_all(largest(), Max());
      if (ref > -kInf) some += exp2_hw((x[0] - ref) * c32) + exp2_hw((x[4] - ref) * c32);
    });
  }
  __device__ __forceinline__ float largest() const {
    return Max()(Max()(most[0], most[1]), Max()(most[2], most[3]));
  }
  // The thread's part of the total, as the sample gives it.
  __device__ __forceinline__ float sampled(float top) const {
    return some != 0.f ? 4.f * some * exp2_hw((ref - top) * c32) : 0.f;
  }
};

// A row by a workgroup of its own.
template <int WAVES, int NBLK, int ES>
__device__ __forceinline__ void sample_row(const SampleParams& p, int64_t r, Scratch<WAVES>& s) {
  constexpr int kT = WAVES * kWave;
  constexpr float kInf = __builtin_inff();
  const int tid = threadIdx.x;
  const Settings set(p, r);
  const double T = set.T, tp = set.tp, mp = set.mp;
  const int64_t k = set.k;
  const float u = set.u;
  Row<WAVES, NBLK, ES> row(p, r);
  RowLook look;
  look.take(row, T);
  float top = block_reduce(look.largest(), s, Max());
  if (top == -kInf) {
    if (tid == 0) put_token(p, r, -1, -kInf);
    return;
  }
  if (set.first_only()) {
    uint32_t at = 0xffffffffu;
    row.each([&](float v, int i) {
      if (v == top) at = Min()(at, (uint32_t)i);
    });
    at = block_reduce(at, s, Min());
    if (tid == 0) put_token(p, r, (int)at, 0.f);
    return;
  }
  if (top == kInf) {
    row.take_inf();
    top = look.least = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) look.most[i] = look.most[i] == kInf ? 0.f : -kInf;
  }
  RowWeights rw(p, top, T);
  const auto give = [&](int i, float v, uint64_t total) { put_token(p, r, i, rw.log_share(v, total, T, p.shift)); };
  const bool cut_k = k > 0 && k < p.n, cut_p = tp < 1.0;
  // a list of all that can be kept
  bool listed = false;
  if (cut_k && k <= listed_of(WAVES)) {
    uint32_t g[4], bound;
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = value_key(look.most[i]);
    if (WAVES > 1 && k < kGroups * 3 / 4) {
      // so many threads' groups together that there are 256
      uint32_t own = Max()(Max()(g[0], g[1]), Max()(g[2], g[3]));
      constexpr int kPart = WAVES > 1 ? kT / kGroups : 1;
      if constexpr (kPart > 1) {
        own = Max()(own, dpp<0xb1>(own));
        own = Max()(own, dpp<0x4e>(own));
      }
      __syncthreads();
      if (tid % kPart == 0) s.groups[tid / kPart] = own;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = s.groups[tid % kWave * 4 + i];
      bound = kth_of_groups(g, (int)k);
    } else if (WAVES > 1) {
      bound = kth_of_all(s, g, (int)k);
    } else {
      bound = kth_of_groups(g, (int)k);
    }
    // (no bound where fewer groups hold a candidate: then all are listed)
    listed = gather(s, row, key_value(Max()(bound, value_key(-kInf))));
  } else if (p.n <= s.kList && (cut_k || cut_p)) {
    listed = gather(s, row, -kInf);
  }
  if (listed) {
    const uint64_t last = cut_all(s, rw, row, k, tp, mp);
    draw(s, rw, row, last, mp, u, give);
    return;
  }
  uint64_t floor = 0;
  if (cut_k || cut_p) {
    // the range that the histograms' steps divide
    const float range = fminf(top - block_reduce(look.least, s, Min()), rw.xmax);
    rw.scale = (float)s.kBins / range;
    rw.fscale = (float)s.kFineBins / range;
    if (!cut_k) {
      const float sampled = block_reduce(look.sampled(top), s, Add());
      floor = nucleus(s, rw, row, tp, grain_of(sampled, p.n));
      // (min-p keeps all of the nucleus when it keeps the last of it)
      if (floor != 0 && rw.weight(Floor(floor).value) >= mp) {
        draw(s, rw, row, floor, mp, u, give);
        return;
      }
    }
    if (floor == 0) {
      Row<WAVES, 0, ES> slow(p, r, row.only_inf);
      if (cut_k) floor = cut<false>(s, rw, slow, (uint64_t)k, 0);
      if (cut_p) {
        uint64_t sum = 0;
        slow.each([&](float v, int i) { sum += rank_key(v, i) >= floor ? rw.fixed(rw.weight(v)) : 0; });
        sum = block_reduce(sum, s, Add());
        floor = cut<true>(s, rw, slow, (uint64_t)ceil(tp * (double)sum), floor);
      }
    }
  }
  __syncthreads();
  segment_weights(rw, row, floor, mp, keep_bound(rw, T, mp, floor), &s.seg[tid / kWave * row.kSegs]);
  draw(s, rw, row, floor, mp, u, give);
}

}  // namespace

}  // namespace rp
