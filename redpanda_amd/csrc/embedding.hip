// Embedding: out[i] = scale w[ids[i]], and the table's gradient
//     dw[v] = scale sum of dout[i] over the places i with ids[i] = v.
//
// Forward: one thread per eight columns of a place; the places' rows are written
// once and the table's come from L2 where ids repeat.
//
// Backward.  Tokens are far from uniform (a board's empty square is a quarter of
// them), so the places are sorted by id first and the sums run over equal shares of
// the sorted places, whatever the ids are; nothing is added by atomics, and the sums'
// order is fixed:
//   sort   workgroup g owns a range of ids and looks at all of them: how many lie
//          below its range is where its places begin, its own are counted by id and
//          written in order of id, then of place.  No workgroup waits for another.
//   sum    a wave takes 32 sorted places and 256 columns, and adds rows while the
//          id stays the same.  An id whose places end inside is written to dw, what
//          may go on in the next share, or began in one before, to `part`.  Ids that
//          do not occur get zeros.
//   join   the share in which a divided id begins adds its pieces in order.

#include "rp_rows.h"
#include "rp_train.h"

namespace rp {

namespace {

constexpr int kSortWaves = 16;
constexpr int kSortRange = 512;   // most ids of a workgroup's range
constexpr int kChunk = 32;        // sorted places of a wave's share
constexpr int kCols = 4 * kWave;  // columns of a wave's share

template <typename Id>
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i) {
  return static_cast<const Id*>(ids)[i];
}

}  // namespace

template <typename Id>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(EmbedParams p) {
  const int64_t nb = (p.d + 7) / 8, n = p.N * nb;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * kThreads) {
    // (32-bit division where it fits: a 64-bit one costs more than the row)
    const int64_t i = n <= 0xffffffffll ? (int64_t)((uint32_t)e / (uint32_t)nb) : e / nb;
    const int64_t col = (e - i * nb) * 8;
    const int64_t id = id_at<Id>(p.ids, i);
    float v[8] = {};
    if (id >= 0 && id < p.V)
      load8(static_cast<const char*>(p.w) + id * p.wsr * p.es_w, col, p.d, p.dt_w, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= p.scale;
    store8(static_cast<char*>(p.out) + i * p.d * p.es_out, col, p.d, p.dt_out, v);
  }
}

template <typename Id>
__global__ __launch_bounds__(kSortWaves* kWave) void embed_sort_kernel(EmbedParams p, EmbedGrad g,
                                                                       int range) {
  __shared__ int32_t cnt[kSortWaves][kSortRange];
  __shared__ int32_t below[kSortWaves];
  __shared__ int32_t scan[kSortWaves];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t lo = (int64_t)blockIdx.x * range;
  const int64_t hi = lo + range < p.V ? lo + range : p.V;
  // each wave looks at its own stretch of places, in order
  const int64_t stretch = ((p.N + kSortWaves * kWave - 1) / (kSortWaves * kWave)) * kWave;
  const int64_t first = wave * stretch;
  const int64_t last = first + stretch < p.N ? first + stretch : p.N;
  for (int i = lane; i < range; i += kWave) cnt[wave][i] = 0;
  int32_t under = 0;
#pragma unroll 4
  for (int64_t i = first + lane; i < last; i += kWave) {
    const int64_t id = id_at<Id>(p.ids, i);
    if (id >= lo && id < hi && id != p.pad) atomicAdd(&cnt[wave][id - lo], 1);
    under += id >= 0 && id < lo && id != p.pad;
  }
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) under += __shfl_xor(under, m);
  if (lane == 0) below[wave] = under;
  __syncthreads();
  // where each id's places begin: the places below the range, then the ids of the
  // range in order (an inclusive scan over them, a thread each)
  int32_t mine = 0;
  if ((int)threadIdx.x < range)
    for (int w = 0; w < kSortWaves; ++w) mine += cnt[w][threadIdx.x];
  int32_t inc = mine;
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
  int32_t at = base + inc - mine;
  if ((int)threadIdx.x < range) {
    if (lo + threadIdx.x < hi) g.start[lo + threadIdx.x] = at;
    if (lo + threadIdx.x == p.V - 1) g.start[p.V] = at + mine;
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t c = cnt[w][threadIdx.x];
      cnt[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = first; i0 < last; i0 += kWave) {
    const int64_t i = i0 + lane;
    const int64_t id = i < last ? id_at<Id>(p.ids, i) : -1;
    const bool in = id >= lo && id < hi && id != p.pad;
    uint64_t left = __ballot(in);
    while (left != 0) {  // one turn for each id of the range among the 64
      const int lead = __builtin_ctzll(left);
      const int key = __builtin_amdgcn_readlane((int)(id - lo), lead);
      const bool same = in && (int)(id - lo) == key;
      const uint64_t those = __ballot(same);
      const int32_t to = cnt[wave][key];
      if (same) {
        const int32_t pos = to + __popcll(those & ((1ull << lane) - 1));
        g.place[pos] = (int32_t)i;
        g.sorted[pos] = (int32_t)id;
      }
      if (lane == lead) cnt[wave][key] = to + __popcll(those);
      left &= ~those;
    }
  }
}

namespace {

// Four elements at `col` of a row of d (zeros at and past d), as stored.
template <int ES>
struct Raw4 {
  uint32_t w[ES];
};

template <int ES>
__device__ __forceinline__ Raw4<ES> load4(const char* row, int64_t col, int64_t d) {
  Raw4<ES> r;
  if (col + 4 <= d) {
    if constexpr (ES == 4) {
      const u32x4_any v = *reinterpret_cast<const u32x4_any*>(row + col * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = v[i];
    } else {
      const u32x2_any v = *reinterpret_cast<const u32x2_any*>(row + col * 2);
      r.w[0] = v[0];
      r.w[1] = v[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < ES; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (col + i >= d) break;
      if constexpr (ES == 4)
        r.w[i] = reinterpret_cast<const uint32_t*>(row)[col + i];
      else
        r.w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[col + i] << (16 * (i & 1));
    }
  }
  return r;
}

template <int ES>
__device__ __forceinline__ void add4(const Raw4<ES>& r, int dtype, float (&v)[4]) {
  if constexpr (ES == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] += cvt_raw(r.w[i / 2] >> (16 * (i & 1)) & 0xffff, dtype);
  }
}

__device__ __forceinline__ void store4(char* row, int64_t col, int64_t d, int dtype,
                                       const float (&v)[4]) {
  if (col + 4 <= d) {
    if (dtype == RP_F32) {
      u32x4_any w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
      *reinterpret_cast<u32x4_any*>(row + col * 4) = w;
    } else {
      u32x2_any w;
      w[0] = pack16(v[0], v[1], dtype);
      w[1] = pack16(v[2], v[3], dtype);
      *reinterpret_cast<u32x2_any*>(row + col * 2) = w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (col + i >= d) break;
    if (dtype == RP_F32)
      reinterpret_cast<float*>(row)[col + i] = v[i];
    else
      reinterpret_cast<uint16_t*>(row)[col + i] = (uint16_t)pack16(v[i], 0.f, dtype);
  }
}

}  // namespace

// Workgroups of four waves: blockIdx.x below `chunks` are shares of the sorted
// places, the ones behind them ids that may be absent, 32 each; blockIdx.y takes four
// waves' columns.
template <int EO>
__global__ __launch_bounds__(kThreads) void embed_sum_kernel(EmbedParams p, EmbedGrad g,
                                                             int64_t chunks) {
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t col = ((int64_t)blockIdx.y * kWaves + wave) * kCols + 4 * lane;
  const bool mine = col < p.d;
  float acc[4] = {};
  if ((int64_t)blockIdx.x >= chunks) {
    const int64_t v0 = ((int64_t)blockIdx.x - chunks) * kChunk;
    const int64_t v = v0 + lane;
    const bool none = lane < kChunk && v < p.V && g.start[v] == g.start[v + 1];
    for (uint64_t m = __ballot(none); m != 0; m &= m - 1) {
      const int64_t row = v0 + __builtin_ctzll(m);
      if (mine) store4(static_cast<char*>(g.dw) + row * p.d * p.es_w, col, p.d, p.dt_w, acc);
    }
    return;
  }
  const int32_t total = g.start[p.V];
  const int64_t pos0 = (int64_t)blockIdx.x * kChunk;
  if (pos0 >= total) return;
  const int n = (int)(total - pos0 < kChunk ? total - pos0 : kChunk);
  int32_t place = 0, id = -1;
  if (lane < n) {
    place = g.place[pos0 + lane];
    id = g.sorted[pos0 + lane];
  }
  // the ids next to the share: whether its first and last id go on there
  int32_t cur = __builtin_amdgcn_readlane(id, 0);
  bool head = pos0 > 0 && g.sorted[pos0 - 1] == cur;
  const bool tail = pos0 + n < total && g.sorted[pos0 + n] == __builtin_amdgcn_readlane(id, n - 1);
  float* part = g.part + (int64_t)blockIdx.x * 2 * p.d;
  const char* rows = static_cast<const char*>(g.dout);
  auto flush = [&](bool last) {
    if (mine) {
      if (head || (last && tail)) {
        // unscaled, in fp32
        store4(reinterpret_cast<char*>(part + (head ? 0 : p.d)), col, p.d, RP_F32, acc);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= p.scale;
        store4(static_cast<char*>(g.dw) + (int64_t)cur * p.d * p.es_w, col, p.d, p.dt_w, acc);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.f;
    head = false;
  };
  constexpr int kAhead = 8;
  for (int j0 = 0; j0 < n; j0 += kAhead) {
    Raw4<EO> r[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      // (a share's end reads its last row again)
      const int64_t row = __builtin_amdgcn_readlane(place, j0 + j < n ? j0 + j : n - 1);
      if (mine) r[j] = load4<EO>(rows + row * g.dosr * EO, col, p.d);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (j0 + j >= n) break;
      const int32_t next = __builtin_amdgcn_readlane(id, j0 + j);
      if (next != cur) {
        flush(false);
        cur = next;
      }
      if (mine) add4(r[j], p.dt_out, acc);
    }
  }
  flush(true);
}

// One workgroup for each share: if an id begins in it and goes on behind it, its
// pieces, which 16 waves add a sixteenth each.
__global__ __launch_bounds__(kSortWaves* kWave) void embed_join_kernel(EmbedParams p, EmbedGrad g) {
  __shared__ float buf[kSortWaves][4][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int32_t total = g.start[p.V];
  const int64_t c = blockIdx.x, end = (c + 1) * kChunk;
  if (end >= total) return;
  const int32_t id = g.sorted[end];
  const int64_t first = g.start[id];
  // (one that ends with the share, or began before it, is another's or none)
  if (first >= end || first < c * kChunk) return;
  const int64_t pieces = ((int64_t)g.start[id + 1] - 1) / kChunk - c + 1;
  const int64_t each = (pieces + kSortWaves - 1) / kSortWaves;
  const int64_t col = (int64_t)blockIdx.y * kCols + 4 * lane;
  const int64_t k1 = (wave + 1) * each < pieces ? (wave + 1) * each : pieces;
  float acc[4] = {};
  if (col < p.d) {
#pragma unroll 8
    for (int64_t k = wave * each; k < k1; ++k)
      add4(load4<4>(reinterpret_cast<const char*>(g.part + ((c + k) * 2 + (k == 0)) * p.d), col, p.d),
           RP_F32, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) buf[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave > 0 || col >= p.d) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int w = 1; w < kSortWaves; ++w) acc[i] += buf[w][i][lane];
    acc[i] *= p.scale;
  }
  store4(static_cast<char*>(g.dw) + (int64_t)id * p.d * p.es_w, col, p.d, p.dt_w, acc);
}

int64_t embed_chunks(int64_t N) { return (N + kChunk - 1) / kChunk; }

hipError_t launch_embed_fwd(const EmbedParams& p, hipStream_t st) {
  const int64_t n = p.N * ((p.d + 7) / 8);
  if (n == 0) return hipSuccess;
  const int64_t wg = (n + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(wg < (1 << 20) ? wg : (1 << 20)));
  if (p.ids64)
    hipLaunchKernelGGL(embed_fwd_kernel<int64_t>, grid, dim3(kThreads), 0, st, p);
  else
    hipLaunchKernelGGL(embed_fwd_kernel<int32_t>, grid, dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_embed_bwd(const EmbedParams& p, const EmbedGrad& g, hipStream_t st) {
  if (p.V * p.d == 0) return hipSuccess;
  // about one workgroup a CU, more where the ids would not fit their counters
  int64_t range = (p.V + 255) / 256;
  if (range > kSortRange) range = kSortRange;
  const dim3 grid((unsigned)((p.V + range - 1) / range));
  if (p.ids64)
    hipLaunchKernelGGL(embed_sort_kernel<int64_t>, grid, dim3(kSortWaves * kWave), 0, st, p, g, (int)range);
  else
    hipLaunchKernelGGL(embed_sort_kernel<int32_t>, grid, dim3(kSortWaves * kWave), 0, st, p, g, (int)range);
  const int64_t chunks = embed_chunks(p.N);
  const dim3 sums((unsigned)(chunks + (p.V + kChunk - 1) / kChunk),
                  (unsigned)((p.d + kCols * kWaves - 1) / (kCols * kWaves)));
  if (p.es_out == 4)
    hipLaunchKernelGGL(embed_sum_kernel<4>, sums, dim3(kThreads), 0, st, p, g, chunks);
  else
    hipLaunchKernelGGL(embed_sum_kernel<2>, sums, dim3(kThreads), 0, st, p, g, chunks);
  if (chunks > 1)
    hipLaunchKernelGGL(embed_join_kernel, dim3((unsigned)(chunks - 1), (unsigned)((p.d + kCols - 1) / kCols)),
                       dim3(kSortWaves * kWave), 0, st, p, g);
  return hipGetLastError();
}

}  // namespace rp
