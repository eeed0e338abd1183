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
// a border that falls between two tokens is then missed by about 1e-12 of the
// total, where fp32's 1e-7 would pick another token every few thousand rows.
//
// A workgroup takes a row, each wave a stretch of it, eight elements a lane and
// step: one wave a row where the rows are many (no barriers, and sixteen rows in
// flight on a CU), up to sixteen where they are few.  Rows are read again for
// each look (from L2), or held in registers where a wave's stretch is short.
// After the largest value:
//   - top-k: the k-th largest of 256 groups' largest values (for large k, of four
//     a thread) bounds the row's k-th from below, and few elements reach it.  They
//     are listed in LDS and ordered, and weights are taken of the list alone.
//   - top-p over the whole row: a histogram of fp32 weights in 32 bits over 2048
//     steps of max - l says in which one or two steps the cut falls; then one
//     look takes the exact weights, summing those before the steps and listing
//     those within.  The list's own sums tell the cut, and that it fell there.
//   - anything these do not hold (long lists, equal logits, a step too full):
//     the cut is found from exact histograms, splitting a step that is too full
//     by its elements' order keys, 9 or 10 bits at a time.
// The draw has the kept weights' sums by segments of the row, and looks at the
// one that u falls into again.
//
// What bounds it: vector instructions.  A nucleus of 4096 rows of 8192 bf16
// logits takes 83-93 us, of which 63 are issue: some 72 instructions an element,
// 16 of them in the first look, 15 for the histogram and 32 for the exact weights
// (its 67 MB would take 13 us).  Without cuts 63 us (fp32, 134 MB), top-40 58,
// top-200 and top-1000 (bf16, the lists' order and the exact histograms) 159 and
// 196; one row of 8192 12.6, 777 lists of up to 218 ids 10.

#include "sample_row.h"

namespace rp {

template <int WAVES, int NBLK, int ES>
__global__ __launch_bounds__(WAVES* kWave) void sample_kernel(SampleParams p) {
  __shared__ Scratch<WAVES> s;
  const int64_t r = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (r < p.R) sample_row<WAVES, NBLK, ES>(p, r, s);
}

namespace {

template <int ES>
void go(const SampleParams& p, hipStream_t st) {
  const int64_t x = p.R < (1 << 20) ? p.R : (1 << 20);
  const dim3 grid((unsigned)x, (unsigned)((p.R + x - 1) / x));
#define RP_GO(WAVES, NBLK)                                                                       \
  hipLaunchKernelGGL((sample_kernel<WAVES, NBLK, ES>), grid, dim3(WAVES* kWave), 0, st, p)
  // A wave a row where that fills the card (nuclei of 8192: 1000 rows 54 us by
  // one wave each, 41 by four; 2000 rows of 1000: 24 and 79).  Four waves a row
  // else, in registers up to 8192 elements; sixteen for the rows that are too few
  // and too long for that (300 rows of 16000: 37 us by four, 54 by sixteen, of
  // which a CU holds two workgroups; 130 of 131072: 165 and 84).
  // A top-k beyond what a shape lists is cut by histograms, from several more looks
  // at the row.  One wave does that sooner than four list it while the row is short
  // (4096 rows of 8192, top-129: 93 and 134 us; the rows' own k are taken so, too),
  // not beyond (1300 of 16000: 130 and 55; 4000 of 12000: 127 and 108, though at
  // top-191 135 and 152); and sixteen waves list what four do later once there are
  // more rows than the card holds at a time (1000 of 30000, top-192: 108 by sixteen,
  // 49 by four; 330 of 100000: 77 and 96).
  const int64_t k = p.k_row != nullptr ? 0 : p.k;
  const bool few = k < 192;
  if (p.n <= 512 && p.R >= 512)
    RP_GO(1, 1);
  else if (p.R >= (p.n <= 2048 ? 512 : 1280) && (p.n <= 8192 ? few : k <= listed_of(1)))
    RP_GO(1, 0);
  else if (p.n <= 2048)
    RP_GO(4, 1);
  else if (p.n <= 4096)
    RP_GO(4, 2);
  else if (p.n <= 8192)
    RP_GO(4, 4);
  else if ((p.R > (p.n <= 16384 ? 64 : 320) && few) || (p.R > 512 && k <= listed_of(4)))
    RP_GO(4, 0);
  else
    RP_GO(16, 0);
#undef RP_GO
}

}  // namespace

hipError_t launch_sample(const SampleParams& p, hipStream_t st) {
  if (p.R == 0) return hipSuccess;
  if (p.dt == RP_F32)
    go<4>(p, st);
  else
    go<2>(p, st);
  return hipGetLastError();
}

}  // namespace rp
