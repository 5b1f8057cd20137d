// Dropout with the mask made from a counter: out = x * keep / (1 - p) (+ residual), rounded once. The same
// call on the gradient is its backward pass; no mask is stored.
#include "ksd_random.h"

#include <algorithm>

namespace ksd {
namespace drop {

// One thread per counter (8 values of a row). chunk / nb by the product with ceil(2^64 / nb), exact for
// chunks and nb below 2^32. Memory bounds it, with the generator's 20 wide products a counter behind the loads: bf16 8192 x
// 1536 with a residual 16.0 us (4.7 TB/s), without 12.3 (4.1), where a large copy reaches 5.1. A thread needs nothing of
// another one, so small tensors take one launch's time (17 rows 3.0 us).
template <int DT, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const void *__restrict__ x, int64_t stride, const void *__restrict__ res,
                                                      int64_t res_stride, void *__restrict__ out, int64_t row0, uint32_t chunks,
                                                      uint32_t nb, uint64_t inv, int64_t d, const Mask m) {
  using T = typename Elem<DT>::T;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= chunks) return;
  const uint32_t r = nb == 1 ? i : (uint32_t)__umul64hi((uint64_t)i, inv), b = i - r * nb;
  const int64_t row = row0 + r, c = (int64_t)b * 8;
  const int n = (int)min((int64_t)8, d - c);
  float v[8], add[8];
  load_any<DT>((const T *)x + row * stride + c, n, v);
  if constexpr (RES) load_any<DT>((const T *)res + row * res_stride + c, n, add);
  apply_mask(m, mask_bits(m, mask_key(m), row, b), v);
  if constexpr (RES) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += add[j];
  }
  store_any<DT>((T *)out + row * d + c, n, v);
}

}  // namespace drop
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_dropout(const void *x, int dtype, int64_t rows, int64_t d, int64_t stride, int64_t drop, uint64_t seed,
                           const void *seed_from, int64_t stream_id, const void *residual, int64_t residual_stride, void *out,
                           void *stream) {
  if (rows < 0 || d < 0 || stride < d || (residual && residual_stride < d)) return fail(KSD_EINVAL, "dropout: bad shape");
  if (dtype != KSD_F32 && dtype != KSD_BF16 && dtype != KSD_F16) return fail(KSD_ETYPE, "dropout: unsupported element type");
  Mask m;
  if (!make_mask(m, drop, seed, seed_from, stream_id)) return fail(KSD_EINVAL, "dropout: bad probability, seed or stream");
  if (rows == 0 || d == 0) return KSD_OK;
  if (!x || !out) return fail(KSD_EINVAL, "dropout: null pointer");
  const int64_t nb = cdiv(d, 8);
  if (nb > 0x7fffffff) return fail(KSD_EINVAL, "dropout: rows too long");
  hipStream_t st = (hipStream_t)stream;
  const uint64_t inv = nb == 1 ? 0 : ~0ull / (uint64_t)nb + 1;
  const int64_t most = 0x80000000LL / nb;  // rows of a launch: its chunks stay below 2^32 threads
  for (int64_t row0 = 0; row0 < rows; row0 += most) {
    const uint32_t chunks = (uint32_t)(std::min<int64_t>(rows - row0, most) * nb);
    const unsigned g = (unsigned)cdiv(chunks, 256);
#define KSD_DROP(DT)                                                                                                    \
  if (residual) drop::dropout_kernel<DT, true><<<g, 256, 0, st>>>(x, stride, residual, residual_stride, out, row0,      \
                                                                  chunks, (uint32_t)nb, inv, d, m);                     \
  else drop::dropout_kernel<DT, false><<<g, 256, 0, st>>>(x, stride, nullptr, 0, out, row0, chunks, (uint32_t)nb, inv, d, m);
    if (dtype == KSD_F32) { KSD_DROP(KSD_F32) }
    else if (dtype == KSD_BF16) { KSD_DROP(KSD_BF16) }
    else { KSD_DROP(KSD_F16) }
#undef KSD_DROP
  }
  return check_launch("dropout");
}
