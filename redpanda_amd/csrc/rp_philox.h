// Counter-based random bits for dropout: Philox4x32-10 (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).  A mask is
// never stored: forward and backward draw the same bits from the seed and the
// element's place.
//
// Key: the 64-bit seed.  Counter of the eight columns 8 b .. 8 b + 7 of a row:
// (b, low word of the row, stream, high word of the row).  Column 8 b + 2 j + i
// takes half i (0: low) of output word j, and is kept where that half is at
// least the threshold t = round(65536 p); kept values are scaled by
// 65536 / (65536 - t), the inverse of the share that is kept.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rp_heads.h"

namespace rp {

constexpr int kDropBlock = 8;  // columns that share one counter

struct DropWords {
  uint32_t w[4];
};

// One instruction; the compiler makes two of it.
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

__device__ __forceinline__ DropWords drop_words(uint32_t block, uint64_t row, uint32_t stream,
                                                uint64_t seed) {
  uint32_t c0 = block, c1 = (uint32_t)row, c2 = stream, c3 = (uint32_t)(row >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Whether the block's column i (0 .. 7) is kept.
__device__ __forceinline__ bool drop_keep(const DropWords& m, int i, uint32_t t) {
  const uint32_t h = (i & 1) ? m.w[i / 2] >> 16 : m.w[i / 2] & 0xffffu;
  return h >= t;
}

// The seed's value, or the one in device memory (which a captured graph reads
// anew on each replay).
__device__ __forceinline__ uint64_t drop_seed(const DropParams& d) {
  return d.seed_ptr != nullptr ? *d.seed_ptr : d.seed;
}

}  // namespace rp
