// Random bits from a counter: Philox4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011). The same key and counter give the same bits on every device and in
// every launch shape, so a mask is made again wherever it is needed and stored nowhere.
#pragma once

#include "ksd_common.h"

namespace ksd {

__device__ __forceinline__ uint4 philox(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u, b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1, (uint32_t)a);
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return c;
}

// A dropout mask over a matrix: 16 bits for each value, a value is dropped where they are below `drop` (65536
// times the probability, rounded). Columns 8 b .. 8 b + 7 of a row take the 8 halves of one counter
// (b, row, row >> 32, stream), so the mask depends on neither the row pitch nor the type. 16 bits: a
// probability is met to 2^-17, and the 1 / (1 - p) of the kept values is that of the rounded one; 32 bits
// a value would double the generator's work, which at 8 values a counter is the smaller half of a pass.
struct Mask {
  const uint64_t *from;  // the seed on the device, or NULL
  uint64_t seed;
  uint32_t stream, drop;
  float scale;
};

struct MaskKey {
  uint32_t k0, k1;
};
__device__ __forceinline__ MaskKey mask_key(const Mask &m) {
  const uint64_t s = m.from ? *m.from : m.seed;
  return MaskKey{(uint32_t)s, (uint32_t)(s >> 32)};
}
__device__ __forceinline__ uint4 mask_bits(const Mask &m, MaskKey k, int64_t row, uint32_t block) {
  return philox(make_uint4(block, (uint32_t)row, (uint32_t)(row >> 32), m.stream), k.k0, k.k1);
}
// v[j] scaled or 0 for the 8 values of a counter's bits.
__device__ __forceinline__ void apply_mask(const Mask &m, uint4 bits, float *v) {
  const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
    v[j] = u >= m.drop ? v[j] * m.scale : 0.0f;
  }
}

inline bool make_mask(Mask &m, int64_t drop, uint64_t seed, const void *seed_from, int64_t stream) {
  if (drop < 0 || drop > 65536 || stream < 0 || stream > 0xffffffffLL || (uintptr_t)seed_from % 8) return false;
  m = Mask{(const uint64_t *)seed_from, seed, (uint32_t)stream, (uint32_t)drop,
           drop == 65536 ? 0.0f : (float)(65536.0 / (double)(65536 - drop))};
  return true;
}

}  // namespace ksd
