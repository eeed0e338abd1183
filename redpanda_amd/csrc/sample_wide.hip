// Sampling from long rows where there are few of them: a row is shared by 16
// workgroups of four waves, since one CU reads a row of 100,000 logits at a
// twentieth of what the card's memory gives.  Four launches, each a look at the
// row: its largest value; what the cut needs first (the list that top-k leaves,
// the fp32 histogram of a nucleus); the exact weights; and one workgroup a row
// that makes the cut and draws.  What they share of a row is in the workspace.
// Sums are of whole numbers and lists are put in order, so the order in which
// workgroups add to them does not matter.  Rows that this does not hold (a long
// list, a large top-k, +inf, min-p above 1) the last launch does by itself, as
// sample_kernel does.
//
// 64 rows of 100003 fp32 logits: top-50 29 us (31 by a workgroup a row), a nucleus
// 52 (67), no cut 27 (38); one row of 131072 bf16: top-50 22 (32), a nucleus 35
// (78).  A launch is 4 us of it whatever it does; the first look reads the 26 MB
// in 8.

#include "sample_row.h"

namespace rp {

namespace {

constexpr int kSlices = 16;                  // workgroups a row
constexpr int kSliceWaves = 4;
constexpr int kShare = kSlices * kSliceWaves;  // waves a row
constexpr int kLastWaves = 16;               // of the last launch's workgroups
constexpr int kWideFine = fine_of(kSliceWaves);
constexpr int kWideList = list_of(kLastWaves);
constexpr int kWideSegs = 2 * kShare;
constexpr int kSliceGroups = kGroups / kSlices;
constexpr int kTooMany = 1 << 24;

template <int ES>
using WideRowOf = Row<kShare, 0, ES>;

struct WideRow {
  unsigned long long sum, ahead;
  uint32_t count, first;  // listed; the first place of the largest value
  float top[kSlices], least[kSlices], some[kSlices];
  uint32_t groups[kGroups];
  uint32_t fine[kWideFine];
  uint64_t seg[kWideSegs];
  uint64_t min_seg[kWideSegs];  // of what min-p leaves (a nucleus' rows)
  uint64_t key[kWideList];
};

enum Plan { kNone, kFirst, kListed, kNucleus, kAll, kAlone };

__device__ __forceinline__ Plan plan_of(const SampleParams& p, const Settings& set, float top) {
  if (top == -__builtin_inff()) return kNone;
  if (set.first_only()) return kFirst;
  if (top == __builtin_inff()) return kAlone;
  if (set.k > 0 && set.k < p.n) return set.k < kGroups * 3 / 4 ? kListed : kAlone;
  return set.tp < 1.0 ? kNucleus : kAll;
}

// The slices' values together.
__device__ __forceinline__ float wide_top(const WideRow& w) {
  float t = w.top[0];
#pragma unroll
  for (int i = 1; i < kSlices; ++i) t = Max()(t, w.top[i]);
  return t;
}
__device__ __forceinline__ void wide_scale(const WideRow& w, RowWeights& rw) {
  float least = w.least[0];
#pragma unroll
  for (int i = 1; i < kSlices; ++i) least = Min()(least, w.least[i]);
  rw.fscale = (float)kWideFine / fminf(rw.top - least, rw.xmax);
}

// The workgroup's list to the row's.
__device__ __forceinline__ void add_list(Scratch<kSliceWaves>& s, WideRow& w) {
  __syncthreads();
  const int n = s.count;
  if (n == 0) return;
  if (threadIdx.x == 0) s.bin = (int)atomicAdd(&w.count, n <= s.kList ? (uint32_t)n : (uint32_t)kTooMany);
  __syncthreads();
  if (n > s.kList) return;
  for (int i = threadIdx.x; i < n; i += kSliceWaves * kWave) {
    const uint32_t at = (uint32_t)s.bin + i;
    if (at < kWideList) w.key[at] = s.key[i];
  }
}

}  // namespace

#define RP_WIDE_ROW                                                  \
  __shared__ Scratch<kSliceWaves> s;                                 \
  const int64_t r = blockIdx.y;                                      \
  const int slice = blockIdx.x;                                      \
  const int share = slice * kSliceWaves +                            \
                    __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave); \
  WideRow& w = static_cast<WideRow*>(p.work)[r];                     \
  const Settings set(p, r);                                          \
  WideRowOf<ES> row(p, r, false, share)

// The largest values; the row's sums and histogram cleared.
template <int ES>
__global__ __launch_bounds__(kSliceWaves* kWave) void sample_wide_top_kernel(SampleParams p) {
  RP_WIDE_ROW;
  RowLook look;
  look.take(row, set.T);
  const float mine = look.largest();
  uint32_t g = value_key(mine);
  g = Max()(g, dpp<0xb1>(g));
  g = Max()(g, dpp<0x4e>(g));
  g = Max()(g, dpp<0x141>(g));
  g = Max()(g, dpp<0x140>(g));
  if (threadIdx.x % 16 == 0) w.groups[slice * kSliceGroups + threadIdx.x / 16] = g;
  const float top = block_reduce(mine, s, Max());
  const float least = block_reduce(look.least, s, Min());
  const float some = block_reduce(look.sampled(top), s, Add());
  constexpr int kPart = kWideFine / kSlices;
  for (int i = threadIdx.x; i < kPart; i += kSliceWaves * kWave) w.fine[slice * kPart + i] = 0;
  if (threadIdx.x == 0) {
    w.top[slice] = top;
    w.least[slice] = least;
    w.some[slice] = top > -__builtin_inff() ? some : 0.f;
    if (slice == 0) {
      w.sum = w.ahead = 0;
      w.count = 0;
      w.first = 0xffffffffu;
    }
  }
}

// The list of top-k, the histogram of a nucleus, or the place of the largest.
template <int ES>
__global__ __launch_bounds__(kSliceWaves* kWave) void sample_wide_look_kernel(SampleParams p) {
  RP_WIDE_ROW;
  const float top = wide_top(w);
  const Plan plan = plan_of(p, set, top);
  if (plan == kFirst) {
    if (w.top[slice] < top) return;
    uint32_t at = 0xffffffffu;
    row.each([&](float v, int i) {
      if (v == top) at = Min()(at, (uint32_t)i);
    });
    at = block_reduce(at, s, Min());
    if (threadIdx.x == 0) atomicMin(&w.first, at);
  } else if (plan == kListed) {
    uint32_t g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = w.groups[threadIdx.x % kWave * 4 + i];
    gather(s, row, key_value(Max()(kth_of_groups(g, (int)set.k), value_key(-__builtin_inff()))));
    add_list(s, w);
  } else if (plan == kNucleus) {
    RowWeights rw(p, top, set.T);
    wide_scale(w, rw);
    float some = 0.f;
#pragma unroll
    for (int i = 0; i < kSlices; ++i) some += w.some[i] * exp2_hw((w.top[i] - top) * rw.c32);
    fine_weights(s, rw, row, grain_of(some, p.n));
    for (int i = threadIdx.x; i < kWideFine; i += kSliceWaves * kWave)
      if (s.fine[i] != 0) atomicAdd(&w.fine[i], s.fine[i]);
  }
}

// Exact weights by segment.
template <int ES>
__global__ __launch_bounds__(kSliceWaves* kWave) void sample_wide_weights_kernel(SampleParams p) {
  RP_WIDE_ROW;
  const float top = wide_top(w);
  const Plan plan = plan_of(p, set, top);
  if (plan != kNucleus && plan != kAll) return;
  RowWeights rw(p, top, set.T);
  uint64_t* seg = &w.seg[share * row.kSegs];
  if (plan == kAll) {
    segment_weights(rw, row, 0, set.mp, keep_bound(rw, set.T, set.mp, 0), seg);
    return;
  }
  wide_scale(w, rw);
  for (int i = threadIdx.x; i < kWideFine; i += kSliceWaves * kWave) s.fine[i] = w.fine[i];
  __syncthreads();
  float lo, hi;
  if (!cut_steps(s, p.n, set.tp, &lo, &hi)) {
    if (threadIdx.x == 0) atomicAdd(&w.count, (uint32_t)kTooMany);
    return;
  }
  uint64_t sum, ahead;
  if (set.mp > 0.0)
    exact_weights<true>(s, rw, row, lo, hi, seg, &sum, &ahead, set.mp, &w.min_seg[share * row.kSegs]);
  else
    exact_weights<false>(s, rw, row, lo, hi, seg, &sum, &ahead, 0.0, nullptr);
  block_sums(sum, ahead, s);
  if (threadIdx.x == 0) {
    atomicAdd(&w.sum, (unsigned long long)sum);
    atomicAdd(&w.ahead, (unsigned long long)ahead);
  }
  add_list(s, w);
}

// The cut and the draw.
template <int ES>
__global__ __launch_bounds__(kLastWaves* kWave) void sample_wide_draw_kernel(SampleParams p) {
  __shared__ Scratch<kLastWaves> s;
  constexpr int kT = kLastWaves * kWave;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const WideRow& w = static_cast<const WideRow*>(p.work)[r];
  const Settings set(p, r);
  const float top = wide_top(w);
  Plan plan = plan_of(p, set, top);
  // no look has found the first place: min-p above 1 is a row's own setting, which
  // the host does not see, and too rare for a launch in every call that has min-p a row
  if (plan == kFirst && w.first == 0xffffffffu) plan = kAlone;
  if (plan == kNone || plan == kFirst) {
    if (tid == 0) {
      if (plan == kNone)
        put_token(p, r, -1, -__builtin_inff());
      else
        put_token(p, r, (int)w.first, 0.f);
    }
    return;
  }
  if (plan != kAlone && w.count <= kWideList) {
    WideRowOf<ES> row(p, r, false, 0);
    const RowWeights rw(p, top, set.T);
    const auto give = [&](int i, float v, uint64_t total) {
      put_token(p, r, i, rw.log_share(v, total, set.T, p.shift));
    };
    if (tid == 0) s.count = (int)w.count;
    for (int i = tid; i < (int)w.count; i += kT) s.key[i] = w.key[i];
    if (plan == kListed) {
      __syncthreads();
      const uint64_t last = cut_all(s, rw, row, set.k, set.tp, set.mp);
      draw(s, rw, row, last, set.mp, set.u, give);
      return;
    }
    for (int i = tid; i < kWideSegs; i += kT) s.seg[i] = w.seg[i];
    __syncthreads();
    if (plan == kAll) {
      draw(s, rw, row, 0, set.mp, set.u, give);
      return;
    }
    const uint64_t floor = nucleus_cut(s, rw, row, set.tp, w.sum, w.ahead);
    if (floor != 0) {
      // (min-p keeps all of the nucleus when it keeps the last of it; else all
      // that it leaves is in the nucleus)
      if (rw.weight(Floor(floor).value) >= set.mp) {
        draw(s, rw, row, floor, set.mp, set.u, give);
      } else {
        for (int i = tid; i < kWideSegs; i += kT) s.seg[i] = w.min_seg[i];
        draw(s, rw, row, 0, set.mp, set.u, give);
      }
      return;
    }
  }
  __syncthreads();
  sample_row<kLastWaves, 0, ES>(p, r, s);
}

#undef RP_WIDE_ROW

// Rows beyond 16384 elements, as long as they are fewer than fill the card with a
// workgroup each.
bool sample_is_wide(int64_t R, int64_t n, bool lists) {
  return !lists && n > 16384 && R <= kSampleWideRows;
}

int64_t sample_wide_bytes(int64_t R) { return R * (int64_t)sizeof(WideRow); }

hipError_t launch_sample_wide(const SampleParams& p, hipStream_t st) {
  const dim3 grid(kSlices, (unsigned)p.R);
  const dim3 block(kSliceWaves * kWave);
  // looks that no row's settings ask for are left out, where the host has them
  const bool first = p.T_row == nullptr && !(p.T > 0.0);
  const bool cut_k = p.k_row == nullptr && p.k > 0 && p.k < p.n;
  const bool whole = p.k_row == nullptr && !cut_k;
  const bool all = whole && p.tp_row == nullptr && p.tp >= 1.0;
  const bool look = !all || p.T_row != nullptr || first;
  const bool weights = !first && !cut_k;
  auto go = [&](auto es) {
    constexpr int ES = decltype(es)::value;
    hipLaunchKernelGGL(sample_wide_top_kernel<ES>, grid, block, 0, st, p);
    if (look) hipLaunchKernelGGL(sample_wide_look_kernel<ES>, grid, block, 0, st, p);
    if (weights) hipLaunchKernelGGL(sample_wide_weights_kernel<ES>, grid, block, 0, st, p);
    hipLaunchKernelGGL(sample_wide_draw_kernel<ES>, dim3((unsigned)p.R), dim3(kLastWaves * kWave), 0, st, p);
  };
  if (p.dt == RP_F32)
    go(std::integral_constant<int, 4>{});
  else
    go(std::integral_constant<int, 2>{});
  return hipGetLastError();
}

}  // namespace rp
