// Embedding: out[i] = scale w[ids[i]], and the table's gradient
//     dw[v] = scale sum of dout[i] over the places i with ids[i] = v.
//
// Forward: a wave takes eight places and 16 bytes a lane of their rows, all loads before
// the stores (short rows: eight columns of four places a thread); the places' rows are
// written once and the table's come from L2 where ids repeat.
//
// Backward.  Tokens are far from uniform (a board's empty square is a quarter of
// them), so the places are sorted by id first and the sums run over equal shares of
// the sorted places, whatever the ids are; no float is added by an atomic, and the
// sums' order is fixed:
//   sort   ids of the same low bits are a bucket (so that frequent ids next to each other
//          fall to different ones).  Up to 4096 places: a workgroup a bucket looks at all
//          ids; how many belong to buckets below is where its places begin, its own are
//          counted and written together, id by id.  More: each 2048 places are put in
//          order of their ids' low eight bits (split), several workgroups a bucket count
//          what that put together for it (count), and write it (place).  No workgroup
//          waits for another.
//   sum    a wave takes a share of the sorted places and 16 bytes a lane of their rows,
//          and adds while the id stays the same.  An id whose places end inside is
//          written to dw, what may go on in the next share, or began in one before, to
//          `part`.  Ids that do not occur get zeros.
//   join   the share in which a divided id begins adds its pieces in order.
// HBM bounds the rows and the sums, the sums by reads in the order of the ids.  131072
// places of 8192 x 1024 bf16: rows 57 us, sort 35, sums 87 (at 3.1 TB/s), join 16; adding
// in the order of the places would read at 4.3, by atomics.  16384 of 8192 x 768 fp32: 15,
// 17, 15, 5.

#include "rp_rows.h"
#include "rp_train.h"

namespace rp {

namespace {

constexpr int kSortWaves = 16;
constexpr int kSortRange = 256;  // most ids of a bucket
constexpr int kZeroRows = 32;    // ids that a wave looks at for absent ones

template <typename Id>
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i) {
  return static_cast<const Id*>(ids)[i];
}

// Buckets are the ids' low lg bits (8 or more), ordered by the lowest eight first.
__device__ __forceinline__ int32_t bucket_of(const EmbedPlan& plan, int32_t id) {
  return (id & 255) << (plan.lg - 8) | (id >> 8 & ((1 << (plan.lg - 8)) - 1));
}
__device__ __forceinline__ int64_t slot_of(const EmbedPlan& plan, int32_t id) {
  return (int64_t)bucket_of(plan, id) * plan.range + (id >> plan.lg);
}

}  // namespace

template <typename Id, int ES>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(EmbedParams p, FastDiv blocks) {
  constexpr int kRows = 4;
  const int64_t n = p.N * (int64_t)blocks.n, step = (int64_t)gridDim.x * kRows * kThreads;
  for (int64_t e0 = (int64_t)blockIdx.x * kRows * kThreads + threadIdx.x; e0 < n; e0 += step) {
    int64_t at[kRows], id[kRows];
    uint32_t col[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int64_t e = e0 + k * kThreads;
      at[k] = -1;
      if (e < n) {
        at[k] = n <= 0x7fffffff ? (int64_t)blocks.div((uint32_t)e) : e / blocks.n;
        col[k] = (uint32_t)(e - at[k] * blocks.n) * 8;
        id[k] = id_at<Id>(p.ids, at[k]);
      }
    }
    Raw8<ES> r[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
#pragma unroll
      for (int i = 0; i < 2 * ES; ++i) r[k].w[i] = 0;
      if (at[k] >= 0 && id[k] >= 0 && id[k] < p.V)
        r[k] = load_raw8<ES>(static_cast<const char*>(p.w) + id[k] * p.wsr * ES, col[k], p.d);
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (at[k] < 0) continue;
      float v[8];
      to_floats(r[k], p.dt_w, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= p.scale;
      store8(static_cast<char*>(p.out) + at[k] * p.d * p.es_out, col[k], p.d, p.dt_out, v);
    }
  }
}

namespace {

// 16 bytes of a row as stored, C columns, from `col` on (zeros at and past d).
template <int ES>
struct Row16 {
  static constexpr int kCols = 16 / ES;
  uint32_t w[4];
  __device__ __forceinline__ void load(const char* row, int64_t col, int64_t d) {
    if (col + kCols <= d) {
      const u32x4_any v = *reinterpret_cast<const u32x4_any*>(row + col * ES);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = 0;
#pragma unroll
      for (int i = 0; i < kCols - 1; ++i) {
        if (col + i >= d) break;
        if constexpr (ES == 4)
          w[i] = reinterpret_cast<const uint32_t*>(row)[col + i];
        else
          w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[col + i] << (16 * (i & 1));
      }
    }
  }
  template <int T>
  __device__ __forceinline__ void floats(float (&v)[kCols]) const {
    if constexpr (ES == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
      Raw8<2> r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = w[i];
      to_floats(r, T, v);
    }
  }
  template <int T>
  __device__ __forceinline__ void add_to(float (&v)[kCols]) const {
    float f[kCols];
    floats<T>(f);
#pragma unroll
    for (int i = 0; i < kCols; ++i) v[i] += f[i];
  }
};

__device__ __forceinline__ void store_cols(void* row, int64_t col, int64_t d, int dtype,
                                           const float (&v)[8]) {
  store8(row, col, d, dtype, v);
}
__device__ __forceinline__ void store_cols(void* row, int64_t col, int64_t d, int dtype,
                                           const float (&v)[4]) {
  if (col + 4 <= d) {
    if (dtype == RP_F32) {
      u32x4_any w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
      *reinterpret_cast<u32x4_any*>(static_cast<char*>(row) + col * 4) = w;
    } else {
      u32x2_any w;
      w[0] = pack16(v[0], v[1], dtype);
      w[1] = pack16(v[2], v[3], dtype);
      *reinterpret_cast<u32x2_any*>(static_cast<char*>(row) + col * 2) = w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (col + i >= d) break;
    if (dtype == RP_F32)
      static_cast<float*>(row)[col + i] = v[i];
    else
      static_cast<uint16_t*>(row)[col + i] = (uint16_t)pack16(v[i], 0.f, dtype);
  }
}

}  // namespace

// Rows of half a kilobyte on: their addresses and ids are the wave's.
template <typename Id, int T>
__global__ __launch_bounds__(kThreads) void embed_rows_kernel(EmbedParams p) {
  constexpr int ES = T == RP_F32 ? 4 : 2, C = Row16<ES>::kCols, kRows = 8;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t col = ((int64_t)blockIdx.y * kWave + lane) * C;
  const int64_t row0 = ((int64_t)blockIdx.x * kWaves + wave) * kRows;
  if (col >= p.d) return;
  Row16<ES> r[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[k].w[i] = 0;
    const int64_t id = row0 + k < p.N ? id_at<Id>(p.ids, row0 + k) : -1;
    if (id >= 0 && id < p.V) r[k].load(static_cast<const char*>(p.w) + id * p.wsr * ES, col, p.d);
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (row0 + k >= p.N) break;
    float v[C];
    r[k].template floats<T>(v);
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] *= p.scale;
    store_cols(static_cast<char*>(p.out) + (row0 + k) * p.d * p.es_out, col, p.d, p.dt_out, v);
  }
}

// Workgroup: 2048 places to pairs[2048 workgroup ..], ordered by the ids' low eight bits;
// where each of the 256 begins (and the last ends) to segs[workgroup].
template <typename Id>
__global__ __launch_bounds__(kThreads) void embed_split_kernel(EmbedParams p, EmbedGrad g) {
  static_assert(kThreads == 256, "a thread for each value of the low bits");
  constexpr int kGroups = kSplitPart / kThreads;
  __shared__ int32_t cnt[kWaves][256];
  __shared__ int32_t scan[kWaves];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t part0 = (int64_t)blockIdx.x * kSplitPart, first = part0 + wave * (kSplitPart / kWaves);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) cnt[w][threadIdx.x] = 0;
  int32_t id[kGroups];
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    const int64_t i = first + u * kWave + lane;
    const int64_t v = i < p.N ? id_at<Id>(p.ids, i) : -1;
    id[u] = v >= 0 && v < p.V && v != p.pad ? (int32_t)v : -1;
  }
  __syncthreads();
  // the lanes of the same low bits (none for a lane without an id)
  uint64_t same[kGroups];
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    uint64_t m = __ballot(id[u] >= 0);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t set = __ballot(id[u] >> b & 1);
      m &= id[u] >> b & 1 ? set : ~set;
    }
    same[u] = id[u] >= 0 ? m : 0;
    if (same[u] != 0 && __builtin_ctzll(same[u]) == lane)
      atomicAdd(&cnt[wave][id[u] & 255], (int32_t)__popcll(same[u]));
  }
  __syncthreads();
  // a thread each: an inclusive scan over the low bits, then wave by wave
  int32_t c[kWaves], mine = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) mine += c[w] = cnt[w][threadIdx.x];
  int32_t inc = mine;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const int32_t o = __shfl_up(inc, m);
    if (lane >= m) inc += o;
  }
  if (lane == kWave - 1) scan[wave] = inc;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    if (w < wave) inc += scan[w];
  int32_t* segs = g.segs + (int64_t)blockIdx.x * kSplitSegs;
  segs[threadIdx.x] = inc - mine;
  if (threadIdx.x == kThreads - 1) segs[kSplitSegs - 1] = inc;
  int32_t at = inc - mine;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    cnt[w][threadIdx.x] = at;
    at += c[w];
  }
  __syncthreads();
  EmbedPair* out = g.pairs + part0;
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    if (same[u] != 0)
      out[cnt[wave][id[u] & 255] + __popcll(same[u] & ((1ull << lane) - 1))] = {
          id[u], (int32_t)(first + u * kWave + lane)};
    // (read by all of its lanes before the first of them moves it on)
    __builtin_amdgcn_wave_barrier();
    if (same[u] != 0 && __builtin_ctzll(same[u]) == lane)
      atomicAdd(&cnt[wave][id[u] & 255], (int32_t)__popcll(same[u]));
    __builtin_amdgcn_wave_barrier();
  }
}

namespace {

// The lanes of a mask below this one.
__device__ __forceinline__ int rank_in(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// The lanes of `left` whose key (of `bits` bits) is the lane's: most often all of them,
// else by a ballot for each bit.
__device__ __forceinline__ uint64_t same_key(int key, uint64_t left, int bits) {
  const int k0 = __builtin_amdgcn_readlane(key, __builtin_ctzll(left));
  uint64_t m = left;
  if ((__ballot(key == k0) & left) == left) return m;
  for (int b = 0; b < bits; ++b) {
    const bool one = key >> b & 1;
    const uint64_t set = __ballot(one);
    m &= one ? set : ~set;
  }
  return m;
}

// 64 lanes' keys (where `in`) counted in cnt.
__device__ __forceinline__ void count_keys(int32_t* cnt, int key, bool in, int bits) {
  const uint64_t left = __ballot(in);
  if (left == 0) return;
  const uint64_t same = same_key(key, left, bits);
  if (in && rank_in(same) == 0) atomicAdd(&cnt[key], (int32_t)__popcll(same));
}

// 64 lanes' places, written where cnt says that their keys' next ones go.
__device__ __forceinline__ void put_places(const EmbedGrad& g, int32_t* cnt, int32_t at, int32_t id,
                                           bool in) {
  const uint64_t left = __ballot(in);
  if (left == 0) return;
  const int key = id >> g.plan.lg;
  const uint64_t same = same_key(key, left, g.plan.bits);
  const int rank = rank_in(same);
  if (in) {
    const int32_t pos = cnt[key] + rank;
    g.place[pos] = at;
    g.sorted[pos] = id;
  }
  // (read by all of its lanes before the first of them moves it on)
  __builtin_amdgcn_wave_barrier();
  if (in && rank == 0) atomicAdd(&cnt[key], (int32_t)__popcll(same));
  __builtin_amdgcn_wave_barrier();
}

// f(the lane's id or -1, its place) for the places that the split put together for a
// bucket, in the parts of a unit, 64 at a time.
template <typename F>
__device__ __forceinline__ void look_at_parts(const EmbedGrad& g, int32_t bucket, int64_t unit, F f) {
  constexpr int kGroups = 4;
  const int lane = threadIdx.x % kWave;
  const int32_t low8 = bucket >> (g.plan.lg - 8);
  const int64_t first = unit * g.plan.unit;
  const int64_t last = first + g.plan.unit < g.plan.parts ? first + g.plan.unit : g.plan.parts;
  for (int64_t q = first; q < last; ++q) {
    const int from = __builtin_amdgcn_readfirstlane(g.segs[q * kSplitSegs + low8]);
    const int n = __builtin_amdgcn_readfirstlane(g.segs[q * kSplitSegs + low8 + 1]) - from;
    const EmbedPair* pairs = g.pairs + q * kSplitPart + from;
    for (int j0 = 0; j0 < n; j0 += kGroups * kWave) {
      EmbedPair e[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        const int j = j0 + u * kWave + lane;
        e[u] = {-1, 0};
        if (j < n) e[u] = pairs[j];
      }
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        if (j0 + u * kWave >= n) break;
        // (a bucket of more than eight bits shares the low eight with others)
        if (g.plan.lg > 8 && bucket_of(g.plan, e[u].id) != bucket) e[u].id = -1;
        f(e[u].id, e[u].at);
      }
    }
  }
}

}  // namespace

// Workgroup (bucket, y): its four waves are units 4 y .. 4 y + 3, whose places they count
// id by id.
__global__ __launch_bounds__(kThreads) void embed_count_kernel(EmbedGrad g) {
  __shared__ int32_t cnt[kWaves][kSortRange];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t unit = (int64_t)blockIdx.y * kWaves + wave;
  const int range = g.plan.range;
  for (int i = lane; i < range; i += kWave) cnt[wave][i] = 0;
  __syncthreads();
  look_at_parts(g, (int32_t)blockIdx.x, unit, [&](int32_t id, int32_t) {
    count_keys(cnt[wave], id >> g.plan.lg, id >= 0, g.plan.bits);
  });
  __syncthreads();
  if (unit >= g.plan.units) return;
  int32_t* out = g.counts + unit * g.plan.slots + (int64_t)blockIdx.x * range;
  int32_t total = 0;
  for (int i = lane; i < range; i += kWave) total += out[i] = cnt[wave][i];
  if (g.plan.lg == 8) return;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) total += __shfl_xor(total, m);
  if (lane == 0) g.totals[(unit << g.plan.lg) + blockIdx.x] = total;
}

// The same workgroups write their places: behind those of the buckets below, the bucket's
// lower ids, and the units below.
__global__ __launch_bounds__(kThreads) void embed_place_kernel(EmbedGrad g) {
  __shared__ int32_t cnt[kWaves][kSortRange], alls[kWaves][kSortRange], lowers[kWaves][kSortRange];
  __shared__ int32_t scan[kWaves];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int range = g.plan.range, lg = g.plan.lg;
  const int32_t bucket = (int32_t)blockIdx.x, low8 = bucket >> (lg - 8);
  const int64_t unit0 = (int64_t)blockIdx.y * kWaves;
  // the places of lower low bits, and of the buckets below that share the low eight
  int32_t under = 0;
  for (int64_t q = threadIdx.x; q < g.plan.parts; q += kThreads) under += g.segs[q * kSplitSegs + low8];
  const int64_t slot0 = (int64_t)bucket * range;
  if (lg > 8)
    for (int64_t u = 0; u < g.plan.units; ++u)
      for (int32_t b = (low8 << (lg - 8)) + (int32_t)threadIdx.x; b < bucket; b += kThreads)
        under += g.totals[(u << lg) + b];
  auto sum_before = [&](int32_t v, int32_t& total) {
    // exclusive over the workgroup's threads
    int32_t inc = v;
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
      const int32_t o = __shfl_up(inc, m);
      if (lane >= m) inc += o;
    }
    __syncthreads();
    if (lane == kWave - 1) scan[wave] = inc;
    __syncthreads();
    int32_t before = inc - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += scan[w];
      total += scan[w];
    }
    return before;
  };
  // each wave adds a quarter of the units' counts, all of them and those below unit0, and
  // looks up its own
  const int64_t quarter = (g.plan.units + kWaves - 1) / kWaves, u0 = wave * quarter;
  const int64_t u1 = u0 + quarter < g.plan.units ? u0 + quarter : g.plan.units;
  const int32_t* counts = g.counts + slot0;
  for (int i = lane; i < range; i += kWave) {
    int32_t all = 0, lower = 0;
#pragma unroll 8
    for (int64_t u = u0; u < u1; ++u) {
      const int32_t c = counts[u * g.plan.slots + i];
      all += c;
      lower += u < unit0 ? c : 0;
    }
    alls[wave][i] = all;
    lowers[wave][i] = lower;
    cnt[wave][i] = unit0 + wave < g.plan.units ? counts[(unit0 + wave) * g.plan.slots + i] : 0;
  }
  int32_t base;
  sum_before(under, base);  // (and a barrier)
  for (int i0 = 0; i0 < range; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    int32_t all = 0, lower = 0;
    if (i < range) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        all += alls[w][i];
        lower += lowers[w][i];
      }
    }
    int32_t total;
    const int32_t at = base + sum_before(all, total);
    if (i < range) {
      if (blockIdx.y == 0) {
        g.start[slot0 + i] = at;
        if (slot0 + i == g.plan.slots - 1) g.start[slot0 + i + 1] = at + all;
      }
      int32_t next = at + lower;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int32_t c = cnt[w][i];
        cnt[w][i] = next;
        next += c;
      }
    }
    base += total;
  }
  __syncthreads();
  look_at_parts(g, bucket, unit0 + wave,
                [&](int32_t id, int32_t at) { put_places(g, cnt[wave], at, id, id >= 0); });
}

// Few places: one launch, whose workgroups each look at all of them, for one bucket.
template <typename Id>
__global__ __launch_bounds__(kSortWaves* kWave) void embed_sort_kernel(EmbedParams p, EmbedGrad g) {
  __shared__ int32_t cnt[kSortWaves][kSortRange];
  __shared__ int32_t below[kSortWaves], scan[kSortWaves];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int range = g.plan.range, lg = g.plan.lg;
  const int32_t bucket = (int32_t)blockIdx.x;
  for (int i = lane; i < range; i += kWave) cnt[wave][i] = 0;
  // f(each lane's id or -1, its place) for the wave's stretch of the places, 64 at a time
  auto look = [&](auto f) {
    constexpr int kGroups = 4;
    const int64_t stretch = ((p.N + kSortWaves * kWave - 1) / (kSortWaves * kWave)) * kWave;
    const int64_t first = wave * stretch;
    const int64_t last = first + stretch < p.N ? first + stretch : p.N;
    for (int64_t i0 = first; i0 < last; i0 += kGroups * kWave) {
      int32_t id[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; ++u) {
        const int64_t i = i0 + u * kWave + lane;
        const int64_t v = i < last ? id_at<Id>(p.ids, i) : -1;
        id[u] = v >= 0 && v < p.V && v != p.pad ? (int32_t)v : -1;
      }
#pragma unroll
      for (int u = 0; u < kGroups; ++u) f(id[u], (int32_t)(i0 + u * kWave) + lane);
    }
  };
  int32_t under = 0;
  look([&](int32_t id, int32_t) {
    const int32_t b = bucket_of(g.plan, id);
    under += id >= 0 && b < bucket;
    count_keys(cnt[wave], id >> lg, id >= 0 && b == bucket, g.plan.bits);
  });
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) under += __shfl_xor(under, m);
  if (lane == 0) below[wave] = under;
  __syncthreads();
  // where each id's places begin: behind the buckets below, then id by id (an inclusive
  // scan over them, a thread each)
  int32_t count = 0;
  if ((int)threadIdx.x < range)
    for (int w = 0; w < kSortWaves; ++w) count += cnt[w][threadIdx.x];
  int32_t inc = count;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const int32_t o = __shfl_up(inc, m);
    if (lane >= m) inc += o;
  }
  if (lane == kWave - 1) scan[wave] = inc;
  __syncthreads();
  int32_t base = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    base += below[w];
    if (w < wave) base += scan[w];
  }
  if ((int)threadIdx.x < range) {
    int32_t at = base + inc - count;
    const int64_t slot = (int64_t)bucket * range + threadIdx.x;
    g.start[slot] = at;
    if (slot == g.plan.slots - 1) g.start[slot + 1] = at + count;
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t c = cnt[w][threadIdx.x];
      cnt[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
  look([&](int32_t id, int32_t at) {
    put_places(g, cnt[wave], at, id, id >= 0 && bucket_of(g.plan, id) == bucket);
  });
}

// Workgroups of one wave: blockIdx.x below `shares` are shares of the sorted places, the
// ones behind them ids that may be absent; blockIdx.y takes a wave's columns.
// T: the type of dout.
template <int T>
__global__ __launch_bounds__(kWave) void embed_sum_kernel(EmbedParams p, EmbedGrad g) {
  constexpr int EO = T == RP_F32 ? 4 : 2, C = Row16<EO>::kCols;
  const int lane = threadIdx.x;
  const int64_t col = ((int64_t)blockIdx.y * kWave + lane) * C;
  const bool mine = col < p.d;
  float acc[C] = {};
  if ((int64_t)blockIdx.x >= g.plan.shares) {
    const int64_t v0 = ((int64_t)blockIdx.x - g.plan.shares) * kZeroRows;
    const int64_t v = v0 + lane, slot = slot_of(g.plan, (int32_t)v);
    const bool none = lane < kZeroRows && v < p.V && g.start[slot] == g.start[slot + 1];
    for (uint64_t m = __ballot(none); m != 0; m &= m - 1) {
      const int64_t row = v0 + __builtin_ctzll(m);
      if (mine) store_cols(static_cast<char*>(g.dw) + row * p.d * p.es_w, col, p.d, p.dt_w, acc);
    }
    return;
  }
  // the first 64 places, and the ids next to the share, are asked for before it is known
  // whether there are so many (those behind the last are never used)
  const int64_t pos0 = (int64_t)blockIdx.x * g.plan.share, back = p.N - 1;
  const int64_t ahead = pos0 + lane < back ? pos0 + lane : back;
  const int64_t next0 = pos0 + g.plan.share < back ? pos0 + g.plan.share : back;
  int32_t place = g.place[ahead], id = g.sorted[ahead];
  const int32_t before = g.sorted[pos0 > 0 ? pos0 - 1 : 0], behind = g.sorted[next0];
  const int32_t total = g.start[g.plan.slots];
  if (pos0 >= total) {
    if (blockIdx.y == 0 && threadIdx.x == 0) g.divided[blockIdx.x] = {0, 0};
    return;
  }
  const int64_t pos1 = pos0 + g.plan.share < total ? pos0 + g.plan.share : total;
  // whether the share's first id began before it
  int32_t cur = __builtin_amdgcn_readfirstlane(id);
  bool head = pos0 > 0 && before == cur;
  float* part = g.part + (int64_t)blockIdx.x * 2 * p.d;
  const char* rows = static_cast<const char*>(g.dout);
  auto flush = [&](bool last) {
    if (mine) {
      // (at the end: whether the last id goes on behind)
      if (head || (last && pos1 < total && behind == cur)) {
        // unscaled, in fp32
        store_cols(part + (head ? 0 : p.d), col, p.d, RP_F32, acc);
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) acc[i] *= p.scale;
        store_cols(static_cast<char*>(g.dw) + (int64_t)cur * p.d * p.es_w, col, p.d, p.dt_w, acc);
      }
    }
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    head = false;
  };
  // the next eight rows are loaded while the present ones are added
  constexpr int kAhead = 8;
  for (int64_t pos = pos0; pos < pos1; pos += kWave) {
    const int n = (int)(pos1 - pos < kWave ? pos1 - pos : kWave);
    if (pos > pos0 && lane < n) {
      place = g.place[pos + lane];
      id = g.sorted[pos + lane];
    }
    Row16<EO> r[kAhead];
    auto load = [&](int j0) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        // (past the end the last row again)
        const int64_t row = __builtin_amdgcn_readlane(place, j0 + j < n ? j0 + j : n - 1);
        if (mine) r[j].load(rows + row * g.dosr * EO, col, p.d);
      }
    };
    load(0);
    for (int j0 = 0; j0 < n; j0 += kAhead) {
      Row16<EO> now[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) now[j] = r[j];
      if (j0 + kAhead < n) load(j0 + kAhead);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (j0 + j >= n) break;
        const int32_t next = __builtin_amdgcn_readlane(id, j0 + j);
        if (next != cur) {
          flush(false);
          cur = next;
        }
        if (mine) now[j].template add_to<T>(acc);
      }
    }
  }
  flush(true);
  // the pieces of an id that begins here and goes on, for the join
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    int32_t pieces = 0;
    if (pos1 < total && behind == cur) {
      const int64_t slot = slot_of(g.plan, cur);
      if (g.start[slot] >= pos0)
        pieces = (g.start[slot + 1] - 1) / g.plan.share - (int32_t)blockIdx.x + 1;
    }
    g.divided[blockIdx.x] = {cur, pieces};
  }
}

// A workgroup takes 16 shares and 256 columns: for each share in which an id begins that
// goes on behind it, the id's pieces, a wave for those of up to eight, and all waves (a
// sixteenth each) for those of more, of which there are two at most.
__global__ __launch_bounds__(kSortWaves* kWave) void embed_join_kernel(EmbedParams p, EmbedGrad g) {
  constexpr int kFew = 8;
  __shared__ float buf[kSortWaves][4][kWave];
  const int64_t c0 = (int64_t)blockIdx.x * kSortWaves;
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t col = ((int64_t)blockIdx.y * kWave + lane) * 4;
  auto piece = [&](int64_t c, int64_t k) {
    Row16<4> r;
    r.load(reinterpret_cast<const char*>(g.part + ((c + k) * 2 + (k == 0)) * p.d), col, p.d);
    return r;
  };
  auto finish = [&](int32_t id, float (&acc)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= p.scale;
    store_cols(static_cast<char*>(g.dw) + (int64_t)id * p.d * p.es_w, col, p.d, p.dt_w, acc);
  };
  // lane l of every wave knows share c0 + l's
  EmbedPair divided = {0, 0};
  if (lane < kSortWaves && c0 + lane < g.plan.shares) divided = g.divided[c0 + lane];
  const int32_t pieces = __builtin_amdgcn_readlane(divided.at, wave);
  if (pieces > 0 && pieces <= kFew && col < p.d) {
    Row16<4> r[kFew];
#pragma unroll
    for (int k = 0; k < kFew; ++k)
      if (k < pieces) r[k] = piece(c0 + wave, k);
    float acc[4] = {};
#pragma unroll
    for (int k = 0; k < kFew; ++k)
      if (k < pieces) r[k].add_to<RP_F32>(acc);
    finish(__builtin_amdgcn_readlane(divided.id, wave), acc);
  }
  for (uint64_t many = __ballot(divided.at > kFew); many != 0; many &= many - 1) {
    const int s = __builtin_ctzll(many);
    const int32_t n = __builtin_amdgcn_readlane(divided.at, s);
    const int32_t each = (n + kSortWaves - 1) / kSortWaves;
    const int32_t last = (wave + 1) * each < n ? (wave + 1) * each : n;
    float acc[4] = {};
    if (col < p.d) {
#pragma unroll 8
      for (int64_t k = wave * each; k < last; ++k) piece(c0 + s, k).add_to<RP_F32>(acc);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) buf[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave > 0 || col >= p.d) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 1; w < kSortWaves; ++w) acc[i] += buf[w][i][lane];
    finish(__builtin_amdgcn_readlane(divided.id, s), acc);
  }
}

EmbedPlan embed_plan(int64_t N, int64_t V, int64_t d, int es_out) {
  EmbedPlan plan;
  plan.lg = 8;  // a workgroup a CU
  while (((V + (1ll << plan.lg) - 1) >> plan.lg) > kSortRange) ++plan.lg;
  plan.range = (int)((V + (1ll << plan.lg) - 1) >> plan.lg);
  plan.slots = (int64_t)plan.range << plan.lg;
  plan.bits = 0;
  while ((1 << plan.bits) < plan.range) ++plan.bits;
  // shares as long as leave 4096 waves: each writes up to two rows of `part`
  const int64_t tiles = (d * es_out + 16 * kWave - 1) / (16 * kWave);
  plan.share = 32;
  while (plan.share < 128 && N * tiles >= 4096 * 2 * plan.share) plan.share *= 2;
  plan.shares = (N + plan.share - 1) / plan.share;
  // (every workgroup looking at all ids takes 5 us for 600 of them, 16 for 16384, 88 for
  // 131072)
  plan.parts = N > 4096 ? (N + kSplitPart - 1) / kSplitPart : 0;
  // units: no more than let all workgroups of 256 buckets be resident, or leave more
  // counters of a bucket than 2048 (131072 places: 64 units 9 us to count and
  // 23 to place, 32 units 13 and 17)
  int64_t units = plan.range < 64 ? 32 : 2048 / plan.range;
  if (units > plan.parts) units = plan.parts;
  plan.unit = units > 0 ? (plan.parts + units - 1) / units : 1;
  plan.units = (plan.parts + plan.unit - 1) / plan.unit;
  return plan;
}

namespace {

template <int T>
void launch_embed_rows(const EmbedParams& p, hipStream_t st) {
  const int64_t wide = 16 * kWave;  // bytes of a wave's columns
  const dim3 grid((unsigned)((p.N + 8 * kWaves - 1) / (8 * kWaves)),
                  (unsigned)((p.d * p.es_w + wide - 1) / wide));
  if (p.ids64)
    hipLaunchKernelGGL((embed_rows_kernel<int64_t, T>), grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL((embed_rows_kernel<int32_t, T>), grid, dim3(kThreads), 0, st, p);
}

}  // namespace

hipError_t launch_embed_fwd(const EmbedParams& p, hipStream_t st) {
  const int64_t nb = (p.d + 7) / 8, n = p.N * nb;
  if (n == 0) return hipSuccess;
  if (p.d * p.es_w >= 512) {
    p.dt_w == RP_F32 ? launch_embed_rows<RP_F32>(p, st)
    : p.dt_w == RP_BF16 ? launch_embed_rows<RP_BF16>(p, st)
                        : launch_embed_rows<RP_F16>(p, st);
    return hipGetLastError();
  }
  const int64_t wg = (n + 4 * kThreads - 1) / (4 * kThreads);
  const dim3 grid((unsigned)(wg < (1 << 20) ? wg : (1 << 20)));
  const FastDiv blocks((uint32_t)nb);
  auto* launch = p.ids64 ? (p.es_w == 4 ? embed_fwd_kernel<int64_t, 4> : embed_fwd_kernel<int64_t, 2>)
                         : (p.es_w == 4 ? embed_fwd_kernel<int32_t, 4> : embed_fwd_kernel<int32_t, 2>);
  hipLaunchKernelGGL(launch, grid, dim3(kThreads), 0, st, p, blocks);
  return hipGetLastError();
}

hipError_t launch_embed_bwd(const EmbedParams& p, const EmbedGrad& g, hipStream_t st) {
  if (p.V * p.d == 0) return hipSuccess;
  const unsigned buckets = 1u << g.plan.lg;
  if (g.plan.parts > 0) {
    const dim3 grid(buckets, (unsigned)((g.plan.units + kWaves - 1) / kWaves));
    hipLaunchKernelGGL((p.ids64 ? embed_split_kernel<int64_t> : embed_split_kernel<int32_t>),
                       dim3((unsigned)g.plan.parts), dim3(kThreads), 0, st, p, g);
    hipLaunchKernelGGL(embed_count_kernel, grid, dim3(kThreads), 0, st, g);
    hipLaunchKernelGGL(embed_place_kernel, grid, dim3(kThreads), 0, st, g);
  } else {
    hipLaunchKernelGGL((p.ids64 ? embed_sort_kernel<int64_t> : embed_sort_kernel<int32_t>),
                       dim3(buckets), dim3(kSortWaves * kWave), 0, st, p, g);
  }
  const int es = p.es_out;
  const int64_t wide = 16 * kWave;  // bytes of a wave's columns
  const dim3 sums((unsigned)(g.plan.shares + (p.V + kZeroRows - 1) / kZeroRows),
                  (unsigned)((p.d * es + wide - 1) / wide));
  auto* sum = p.dt_out == RP_F32    ? embed_sum_kernel<RP_F32>
              : p.dt_out == RP_BF16 ? embed_sum_kernel<RP_BF16>
                                    : embed_sum_kernel<RP_F16>;
  hipLaunchKernelGGL(sum, sums, dim3(kWave), 0, st, p, g);
  if (g.plan.shares > 1)
    hipLaunchKernelGGL(embed_join_kernel,
                       dim3((unsigned)((g.plan.shares + kSortWaves - 1) / kSortWaves),
                            (unsigned)((p.d + 4 * kWave - 1) / (4 * kWave))),
                       dim3(kSortWaves * kWave), 0, st, p, g);
  return hipGetLastError();
}

}  // namespace rp
