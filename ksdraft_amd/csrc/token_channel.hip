// W8A8 product with one fp32 scale per row of each operand (per token and per output channel):
//
//   y[m,n] = ((sum_k a[m,k] w[n,k]) * sa[m]) * sw[n]  (+ bias[n])  (+ residual[m,n]),  rounded once
//
// The scales stand outside the sum, so the whole reduction stays in the int8 matrix unit with exact
// int32 sums; the group-128 product of gemm.hip rescales every 128 steps on the VALU instead.
//
// What bounds it (us, bf16 output, one product over and over): long products the power that the matrix unit
// draws, 8192^3 410 to 480 by card (2290 TOPS and more) on random codes and 334 on zeros; at K = 1536 a launch's
// start and a tile's end as well, 8192 x 1536 x 1536 22 to 25 (1580 TOPS and more), with a residual 27 to 29, 4096 x
// 150144 x 1536 920 to 955 (2.0 POPS; 1016 to 1062 between the other passes of a training call).
//
// Row quantization (ksd_tc_quantize_rows): a = max |x[r,:]|; where a < 2^-100 the row's scale and
// codes are 0, else scale = a / 127, code = rint(x * (127 / a)), each operation rounded to fp32.
// |x * (127 / a)| <= 127 (1 + 2^-23), so no clamp is needed. A row that holds NaN or inf has scale
// NaN and codes 0.
//
// Gradients: the codes of W and X are used as they are, their scales move into dY before it is
// quantized, so nothing is requantized or transposed in memory:
//   dX = diag(e) Q W_q,    (Q, e) = row quantization of dY * sw[n]
//   dW = diag(f) C^T X_q,  (C, f) = column quantization of dY * sx[m]
// Both contract over the row index of a row-major operand; such an operand ("T") is staged as it
// lies in memory and transposed by the LDS reads (ds_read_b64_tr_b8).
#include "ksd_common.h"

#include <algorithm>
#include <type_traits>

namespace ksd {
namespace tc {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

constexpr float kTiny = 0x1p-100f;

// scale and reciprocal of a row from its largest magnitude (NaN sorts above inf in abs-bit order)
__device__ __forceinline__ void row_scale(uint32_t bits, float &scale, float &inv) {
  const float a = __builtin_bit_cast(float, bits);
  if (bits >= 0x7f800000u) {
    scale = __builtin_nanf("");
    inv = 0.0f;
  } else if (a < kTiny) {
    scale = inv = 0.0f;
  } else {
    scale = a / 127.0f;
    inv = 127.0f / a;
  }
}

// Codes of four products p with |p| <= 127 (1 + 2^-22): p + 1.5 * 2^23 rounds p to the nearest
// integer, ties to even, and leaves it in the low byte. NaN and inf products (a row with inv 0 and
// non-finite values) must have been masked by the caller.
__device__ __forceinline__ uint32_t pack4(float p0, float p1, float p2, float p3) {
  constexpr float kMagic = 12582912.0f;
  const uint32_t b0 = __builtin_bit_cast(uint32_t, p0 + kMagic), b1 = __builtin_bit_cast(uint32_t, p1 + kMagic);
  const uint32_t b2 = __builtin_bit_cast(uint32_t, p2 + kMagic), b3 = __builtin_bit_cast(uint32_t, p3 + kMagic);
  return __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u) | __builtin_amdgcn_perm(b3, b2, 0x04000c0cu);
}

// 8 consecutive elements at any element alignment (global loads need none beyond the element's).
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T *p, float *v) {
  struct __attribute__((packed, aligned(DT == KSD_F32 ? 4 : 2))) Any { uint4 q; };
  Raw8<DT> r;
  r.a = ((const Any *)p)->q;
  if constexpr (DT == KSD_F32) r.b = ((const Any *)(p + 4))->q;
  cvt_raw8<DT>(r, true, v);
}
// elements [k, k + 8) of a row of K, zeros past its end
template <int DT>
__device__ __forceinline__ void load8_tail(const typename Elem<DT>::T *row, int64_t k, int64_t K, float *v) {
  if (k + 8 <= K) {
    load8<DT>(row + k, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? Elem<DT>::load(row + k + j) : 0.0f;
  }
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = group_max_u32<16>(v);
  v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return max(v, (uint32_t)__shfl_xor((int)v, 32));
}

// ------------------------------------------------------------------------------------ rows
struct Rows {
  const void *x;
  int64_t M, K, stride, ld;
  int8_t *codes;
  float *scales;
};

// LANES threads per row (64: four rows per workgroup; 256: one), the first NCH * LANES * 8 elements
// kept in registers between the maximum and the codes, the rest read again (from cache).
template <int DT, int LANES, int NCH>
__device__ __forceinline__ void quant_rows(const Rows &p, int64_t block) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x % LANES;
  const int64_t m = block * (256 / LANES) + threadIdx.x / LANES, K = p.K, ld = p.ld;
  if (LANES == 64 && m >= p.M) return;
  const T *row = (const T *)p.x + m * p.stride;
  float v[NCH][8];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t k = ((int64_t)c * LANES + lane) * 8;
    if (k < K) {
      load8_tail<DT>(row, k, K, v[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) top = max(top, __builtin_bit_cast(uint32_t, abs_max<8>(v[c])));
  for (int64_t k = ((int64_t)NCH * LANES + lane) * 8; k < K; k += LANES * 8) {
    float t[8];
    load8_tail<DT>(row, k, K, t);
    top = max(top, __builtin_bit_cast(uint32_t, abs_max<8>(t)));
  }
  top = wave_max(top);
  if constexpr (LANES == 256) {
    __shared__ uint32_t part[4];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
  }
  float scale, inv;
  row_scale(top, scale, inv);
  const bool bad = top >= 0x7f800000u;
  if (lane == 0) p.scales[m] = scale;
  int8_t *out = p.codes + m * ld;
  auto put = [&](int64_t k, const float *t) {
    uint2 w;
    w.x = bad ? 0 : pack4(t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv);
    w.y = bad ? 0 : pack4(t[4] * inv, t[5] * inv, t[6] * inv, t[7] * inv);
    *(uint2 *)(out + k) = w;
  };
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t k = ((int64_t)c * LANES + lane) * 8;
    if (k < ld) put(k, v[c]);
  }
  for (int64_t k = ((int64_t)NCH * LANES + lane) * 8; k < ld; k += LANES * 8) {
    float t[8];
    load8_tail<DT>(row, k, K, t);
    put(k, t);
  }
}

// Workgroups below `blocks0` take the first matrix, the others the second (of type DT1; a layer's weights
// and its tokens have one row length, so one launch covers both).
template <int DT0, int DT1, int LANES, int NCH>
__global__ __launch_bounds__(256) void quant_rows_kernel(const Rows a, const Rows b, unsigned blocks0) {
  if (blockIdx.x < blocks0) quant_rows<DT0, LANES, NCH>(a, blockIdx.x);
  else quant_rows<DT1, LANES, NCH>(b, blockIdx.x - blocks0);
}

template <int DT0, int DT1>
static void launch_rows(const Rows &a, const Rows &b, hipStream_t st) {
  const int64_t per = a.K <= 1536 ? 4 : 1, n0 = cdiv(a.M, per), n = n0 + cdiv(b.M, per);
  if (a.K <= 512) quant_rows_kernel<DT0, DT1, 64, 1><<<(unsigned)n, 256, 0, st>>>(a, b, (unsigned)n0);
  else if (a.K <= 1536) quant_rows_kernel<DT0, DT1, 64, 3><<<(unsigned)n, 256, 0, st>>>(a, b, (unsigned)n0);
  else quant_rows_kernel<DT0, DT1, 256, 4><<<(unsigned)n, 256, 0, st>>>(a, b, (unsigned)n0);
}
static void launch_rows(const Rows &a, int t, hipStream_t st) {
  const Rows none{nullptr, 0, a.K, 0, 0, nullptr, nullptr};
  if (t == KSD_F32) launch_rows<KSD_F32, KSD_F32>(a, none, st);
  else if (t == KSD_BF16) launch_rows<KSD_BF16, KSD_BF16>(a, none, st);
  else launch_rows<KSD_F16, KSD_F16>(a, none, st);
}

// ------------------------------------------------------------------------------- gradient's codes
// Two reads of dY, bound by memory: the first leaves per row block the column maxima of |dY * sx| and
// the column sums, per column block the row maxima of |dY * sw|; a fold in a fixed order makes scales of
// them; the second writes both codes. (bf16, us: 8192 x 1536 9, 7.6 and 14.4; 4096 x 150144 294, 16 and 459, 4.2
// and 5.4 TB/s.)
// A wave takes `rows` (a multiple of 16) x 64 V columns: lane l holds columns V l .. V l + V - 1, 16 rows'
// loads in flight. A row's maximum crosses the lanes through LDS, 16 rows at once.
// Row blocks run along y, and along z past the 65535 that y holds.
__device__ __forceinline__ int64_t row_block() { return (int64_t)blockIdx.z * gridDim.y + blockIdx.y; }
static dim3 row_grid(int64_t x, int64_t rows) {
  const int64_t z = cdiv(rows, 65535);
  return dim3((unsigned)x, (unsigned)cdiv(rows, z), (unsigned)z);
}
template <int DT, int V>
__device__ __forceinline__ void load_vec(const typename Elem<DT>::T *p, float *v) {
  if constexpr (V == 8) {
    load8<DT>(p, v);
  } else if constexpr (DT == KSD_F32) {
    struct __attribute__((packed, aligned(4))) Any { float w[4]; };
    const Any q = *(const Any *)p;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = q.w[j];
  } else {
    struct __attribute__((packed, aligned(2))) Any { uint32_t w[2]; };
    const Any q = *(const Any *)p;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t h = (uint16_t)(q.w[j / 2] >> (j % 2 * 16));
      v[j] = Elem<DT>::load(&h);
    }
  }
}

template <int DT, int V>
__global__ __launch_bounds__(256) void grad_stats_kernel(const void *__restrict__ g, int64_t M, int64_t N, int64_t stride, int rows,
                                                         const float *__restrict__ sx, const float *__restrict__ sw,
                                                         uint32_t *__restrict__ row_part, uint32_t *__restrict__ col_part,
                                                         float *__restrict__ sum_part) {
  using T = typename Elem<DT>::T;
  __shared__ uint32_t rmax_all[4][16][65];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t(*const rmax)[65] = rmax_all[wave];
  const int64_t cb = (int64_t)blockIdx.x * 4 + wave, rb = row_block(), c = (cb * 64 + lane) * V;
  const int64_t m0 = rb * rows, m1 = min(M, m0 + rows);
  if (cb * 64 * V >= N || m0 >= M) return;
  const bool cols = (cb + 1) * 64 * V <= N;
  float w[V], sum[V];
  uint32_t cm[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    w[j] = c + j < N ? sw[c + j] : 0.0f;
    sum[j] = 0.0f;
    cm[j] = 0;
  }
  for (int64_t mb = m0; mb < m1; mb += 16) {
    float v[16][V], s[16];
    if (cols && mb + 16 <= m1) {
#pragma unroll
      for (int r = 0; r < 16; ++r) load_vec<DT, V>((const T *)g + (mb + r) * stride + c, v[r]);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = sx[mb + r];
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = mb + r < m1 ? sx[mb + r] : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[r][j] = c + j < N && mb + r < m1 ? Elem<DT>::load((const T *)g + (mb + r) * stride + c + j) : 0.0f;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float t[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        t[j] = v[r][j] * w[j];
        sum[j] += v[r][j];
        cm[j] = max(cm[j], __builtin_bit_cast(uint32_t, fabsf(v[r][j] * s[r])));
      }
      rmax[r][lane] = __builtin_bit_cast(uint32_t, abs_max<V>(t));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) top = max(top, rmax[lane >> 2][(lane & 3) * 16 + k]);
    top = group_max_u32<4>(top);
    if ((lane & 3) == 0 && mb + (lane >> 2) < m1) row_part[cb * M + mb + (lane >> 2)] = top;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (c + j < N) {
      col_part[rb * N + c + j] = cm[j];
      if (sum_part) sum_part[rb * N + c + j] = sum[j];
    }
}

// Scales, reciprocals and column sums from the partial results: workgroup b < ceil(M / 64) folds 64 rows, the
// others 64 columns each; wave w takes every 16th part, the waves' results meet in wave order.
__global__ __launch_bounds__(1024) void grad_fold_kernel(const uint32_t *__restrict__ row_part, const uint32_t *__restrict__ col_part,
                                                         const float *__restrict__ sum_part, int64_t M, int64_t N, int ncb, int nrb,
                                                         float *__restrict__ e, float *__restrict__ einv, float *__restrict__ f,
                                                         float *__restrict__ finv, float *__restrict__ db) {
  __shared__ uint32_t tops[16][64];
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rblocks = (M + 63) / 64;
  const bool is_row = blockIdx.x < rblocks;
  const int64_t i = (is_row ? (int64_t)blockIdx.x : (int64_t)blockIdx.x - rblocks) * 64 + lane, L = is_row ? M : N;
  const uint32_t *part = is_row ? row_part : col_part;
  const int n = is_row ? ncb : nrb;
  const bool add = !is_row && db;
  uint32_t top = 0;
  float sum = 0.0f;
  if (i < L) {
#pragma unroll 8
    for (int b = wave; b < n; b += 16) {
      top = max(top, part[(int64_t)b * L + i]);
      if (add) sum += sum_part[(int64_t)b * L + i];
    }
  }
  tops[wave][lane] = top;
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && i < L) {
    for (int k = 1; k < 16; ++k) {
      top = max(top, tops[k][lane]);
      sum += sums[k][lane];
    }
    float s, inv;
    row_scale(top, s, inv);
    (is_row ? e : f)[i] = s;
    (is_row ? einv : finv)[i] = inv;
    if (add) db[i] = sum;
  }
}

// Both codes of dY, in its own layout: q (rows, for dX) and c (columns, for dW), rows of ld bytes with zeros
// past N. A thread holds 8 columns over 8 H rows, 8 of them in flight. A row or column whose scale is NaN
// has codes of no meaning: its products are NaN through the scale.
template <int DT, int H>
__global__ __launch_bounds__(256) void grad_codes_kernel(const void *__restrict__ g, int64_t M, int64_t N, int64_t stride,
                                                         const float *__restrict__ sx, const float *__restrict__ sw,
                                                         const float *__restrict__ einv, const float *__restrict__ finv,
                                                         int8_t *__restrict__ q, int8_t *__restrict__ cq, int64_t ld) {
  using T = typename Elem<DT>::T;
  const int64_t c = ((int64_t)blockIdx.x * 64 + (threadIdx.x & 63)) * 8;
  const int64_t m0 = row_block() * (32 * H) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * (8 * H);
  if (c >= ld) return;
  const bool cols = (int64_t)(blockIdx.x + 1) * 512 <= N;
  float w[8], fi[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = c + j < N ? sw[c + j] : 0.0f;
    fi[j] = c + j < N ? finv[c + j] : 0.0f;
  }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    float v[8][8];
    if (cols && m0 + h * 8 + 8 <= M) {
#pragma unroll
      for (int r = 0; r < 8; ++r) load8<DT>((const T *)g + (m0 + h * 8 + r) * stride + c, v[r]);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[r][j] = m0 + h * 8 + r < M && c + j < N ? Elem<DT>::load((const T *)g + (m0 + h * 8 + r) * stride + c + j) : 0.0f;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t m = m0 + h * 8 + r;
      if (m >= M) break;
      if (q) {
        const float inv = einv[m];
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = (v[r][j] * w[j]) * inv;
        *(uint2 *)(q + m * ld + c) = make_uint2(pack4(t[0], t[1], t[2], t[3]), pack4(t[4], t[5], t[6], t[7]));
      }
      if (cq) {
        const float s = sx[m];
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = (v[r][j] * s) * fi[j];
        *(uint2 *)(cq + m * ld + c) = make_uint2(pack4(t[0], t[1], t[2], t[3]), pack4(t[4], t[5], t[6], t[7]));
      }
    }
  }
}

// A large dY is read in pieces of 16 bytes, 64 rows to a wave, which halves the partial results; a small one in
// pieces of 4 elements, 32 rows to a wave (and 8, not 16, in the second read), for more waves.
static bool large_grad(int64_t M, int64_t N) { return M * N >= (int64_t)1 << 25; }
static int stats_rows(int64_t M, int64_t N) { return large_grad(M, N) ? 64 : 32; }

// ------------------------------------------------------------------------------------ product
// One operand of the product. Plain ("N"): (rows, K) with the reduction contiguous; "T": (K, rows)
// with the output index contiguous. ld is the row pitch in bytes, a multiple of 16, and the bytes
// of a row up to ceil16 of its length are readable. Bytes past K of an N operand must be zero in A.
struct Prob {
  const int8_t *A, *W;
  const float *sa, *sw, *bias;
  const void *R;
  void *Y;
  int32_t *parts;  // splits > 1: (splits, M, N) int32 sums
  int64_t lda, ldw;
  int M, N, K, splits, ksteps;  // ksteps: steps of 128 of one split
  int nt;                       // non-temporal stores
};

constexpr int BK = 128;

typedef __attribute__((address_space(3))) const v4i lds_v4i;
typedef __attribute__((address_space(3))) v2i lds_v2i;
__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)(p);
}

// Position of 16-byte chunk c of LDS row r, in bytes. N tiles have rows of 128 bytes (the reduction),
// T tiles rows of B bytes (the output index), row = reduction step. The chunk index is XORed so that
// the 16 lanes that read one fragment chunk (16 rows of an N tile; 8 rows of a T tile, two such row
// sets per 32 lanes) hit 16 different 16-byte bank groups.
template <bool T, int B>
__device__ __forceinline__ constexpr int lds_swz(int r) {
  if constexpr (!T) return (r >> 1) & 7;
  else if constexpr (B == 256) return (r & 7) | ((r >> 1) & 8);
  else if constexpr (B == 192 || B == 64) return ((r >> 2) & 1) | ((r >> 3) & 2);
  else return ((r >> 1) & 3) | ((r >> 2) & 4);
}
template <bool T, int B>
__device__ __forceinline__ constexpr int lds_pos(int r, int c) {
  return r * (T ? B : BK) + ((c ^ lds_swz<T, B>(r)) << 4);
}

// The DMA of one operand's B x 128 tile into LDS: 1 KB instructions, lane l of instruction i fills
// chunk 64 i + l of the tile. PERM > 0: the output index of LDS row p within each block of 16 PERM rows
// is permuted so that one lane's results are PERM consecutive columns (see the store). What lies
// outside the operand reads as zero (offsets past the buffer's range).
template <bool T, int B, int NW, int PERM>
struct Stage {
  static constexpr int INSTR = B * BK / 1024, D = INSTR / NW;
  static_assert(INSTR % NW == 0, "whole instructions per wave");
  uint32_t off[D];
  const int8_t *base;
  int64_t ld;
  int k0, K, valid, cb;

  __device__ __forceinline__ void start(const int8_t *P, int64_t pitch, int rows, int Kn, int row0, int kfirst, int wave, int lane) {
    ld = pitch, k0 = kfirst, K = Kn;
    if constexpr (!T) {
      valid = min(B, rows - row0);
      base = P + (int64_t)row0 * ld + kfirst;
#pragma unroll
      for (int i = 0; i < D; ++i) {
        const int p = (wave * D + i) * 8 + (lane >> 3), c = (lane & 7) ^ lds_swz<false, B>(p);
        int row = p;
        if constexpr (PERM > 0) {
          const int b = p / (16 * PERM), o = p % (16 * PERM), j = o >> 4, ii = o & 15;
          row = b * (16 * PERM) + ii * PERM + j;
        }
        off[i] = row < valid ? (uint32_t)(row * (int)ld + c * 16) : kOob;
      }
    } else {
      cb = (rows + 15) & ~15;
      base = P + (int64_t)kfirst * ld + row0;
#pragma unroll
      for (int i = 0; i < D; ++i) {
        const int L = (wave * D + i) * 64 + lane, r = L / (B / 16), c = (L % (B / 16)) ^ lds_swz<true, B>(r);
        off[i] = row0 + c * 16 < cb ? (uint32_t)(r * (int)ld + c * 16) : kOob;
      }
    }
  }
  typedef uint32_t rsrc4 __attribute__((ext_vector_type(4)));
  rsrc4 rs;
  bool tail;
  // before the issues of a step; not live: every load reads as zero
  __device__ __forceinline__ void open(bool live) {
    const uint64_t a = (uint64_t)base;
    const int rows_k = min(BK, K - k0);
    uint32_t bytes;
    if constexpr (!T) bytes = (uint32_t)(valid - 1) * (uint32_t)ld + BK;
    else bytes = (uint32_t)rows_k * (uint32_t)ld;
    if (!live) bytes = 0;
    tail = !T && rows_k < BK;
    rs = (rsrc4){(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), (uint32_t)kBufFlags};
  }
  __device__ __forceinline__ void issue(int i, uint32_t lds, int wave, int lane) {
    uint32_t o = off[i];
    if constexpr (!T) {
      if (__builtin_expect(tail, 0)) {
        const int p = (wave * D + i) * 8 + (lane >> 3), c = (lane & 7) ^ lds_swz<false, B>(p);
        if (k0 + c * 16 >= ((K + 15) & ~15)) o = kOob;
      }
    }
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(o), "s"(rs), "s"(lds + (uint32_t)(wave * D + i) * 1024) : "memory", "m0");
  }
  __device__ __forceinline__ void next() {
    k0 += BK;
    base += T ? (int64_t)BK * ld : BK;
  }
};

// Reads of 16 output rows x 64 reduction steps as an MFMA operand: lane l holds row l % 16, steps
// 16 (l / 16) .. + 15 of half kk. The swizzle of an N tile does not depend on the block of 16 rows i and
// that of a T tile not on kk, so few lane addresses serve all reads and the rest is an immediate.
template <bool T, int B, int NB>
struct Reader {
  uint32_t pos[T ? NB : 2];
  __device__ __forceinline__ void start(uint32_t lds, int row0, int lane) {
    if constexpr (!T) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) pos[kk] = lds + row0 * BK + lds_pos<false, B>(lane & 15, kk * 4 + (lane >> 4));
    } else {
      // lanes 2r, 2r + 1 of each 16 address the two halves of step r's 16 bytes; the read leaves lane
      // c the 8 steps of column c
      const int kr = (lane >> 4) * 16 + ((lane & 15) >> 1);
#pragma unroll
      for (int i = 0; i < NB; ++i) pos[i] = lds + lds_pos<true, B>(kr, row0 / 16 + i) + (lane & 1) * 8;
    }
  }
  __device__ __forceinline__ void shift(uint32_t by) {
#pragma unroll
    for (int i = 0; i < (T ? NB : 2); ++i) pos[i] += by;
  }
  __device__ __forceinline__ v4i read(int i, int kk) const {
    if constexpr (!T) {
      return *(lds_v4i *)(uintptr_t)(pos[kk] + i * 16 * BK);
    } else {
      const v2i lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(uintptr_t)(pos[i] + kk * 64 * B));
      const v2i hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i *)(uintptr_t)(pos[i] + kk * 64 * B + 8 * B));
      return (v4i){lo.x, lo.y, hi.x, hi.y};
    }
  }
};

template <int OUT>
__device__ __forceinline__ float load_out(const void *p, int64_t i) {
  return Elem<OUT>::load((const typename Elem<OUT>::T *)p + i);
}
// W (even) consecutive elements at any element alignment
template <int OUT, int W>
__device__ __forceinline__ void loadv(const void *p, int64_t i, float *v) {
  if constexpr (OUT == KSD_F32) {
    struct __attribute__((packed, aligned(4))) Any { float w[W]; };
    const Any a = *(const Any *)((const float *)p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = a.w[j];
  } else {
    struct __attribute__((packed, aligned(2))) Any { uint32_t w[W / 2]; };
    const Any a = *(const Any *)((const uint16_t *)p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint16_t h = (uint16_t)(a.w[j / 2] >> (j % 2 * 16));
      v[j] = Elem<OUT>::load(&h);
    }
  }
}
// nt: non-temporal, so that a streamed output does not push the operands' panels out of L2.
template <int OUT, int W, bool nt>
__device__ __forceinline__ void storev(void *p, int64_t i, const float *v) {
  if constexpr (OUT == KSD_F32) {
    typedef float vec __attribute__((ext_vector_type(W), aligned(4)));
    vec a;
#pragma unroll
    for (int j = 0; j < W; ++j) a[j] = v[j];
    vec *const q = (vec *)((float *)p + i);
    if constexpr (nt) __builtin_nontemporal_store(a, q);
    else *q = a;
  } else {
    typedef uint32_t vec __attribute__((ext_vector_type(W / 2), aligned(2)));
    vec a;
#pragma unroll
    for (int j = 0; j < W / 2; ++j) {
      if constexpr (OUT == KSD_BF16) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        a[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){v[2 * j], v[2 * j + 1]}, bf16x2));
      } else {
        a[j] = f16_bits(v[2 * j]) | (uint32_t)f16_bits(v[2 * j + 1]) << 16;
      }
    }
    vec *const q = (vec *)((uint16_t *)p + i);
    if constexpr (nt) __builtin_nontemporal_store(a, q);
    else *q = a;
  }
}

__device__ __forceinline__ void wg_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// BM x BN tiles, WM x WN waves; TA, TW: the operand is a T one. Persistent: a workgroup walks its
// units (tile, part of the reduction) through a ring of S LDS slots of 128 reduction steps each, filled by DMA
// up to S steps ahead, across unit ends. Per step each wave multiplies the first half (64) of the step while it
// reads the fragments of the second, then one barrier, then the second half while it reads the next step's first.
template <int BM, int BN, int WM, int WN, int S, bool TA, bool TW, int OUT>
__global__ __launch_bounds__(WM *WN * 64, WM *WN == 8 ? 1 : 2) void gemm_kernel(const Prob p) {
  constexpr int NW = WM * WN, NI = BM / WM / 16, NJ = BN / WN / 16;
  constexpr int PERM = TW ? 0 : NJ;
  constexpr uint32_t SA = BM * BK, SLOT = (BM + BN) * BK;
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];  // S slots of an A and a W tile
  const uint32_t lds0 = lds_addr(smem);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN, units = tm * tn * p.splits;
  const int kt = (p.K + BK - 1) / BK;

  // units of this workgroup: those of one XCD (blockIdx % 8) are consecutive, its workgroups
  // take them in turn
  int u, u_end, u_step;
  {
    const int G = gridDim.x, x = blockIdx.x % 8;
    const int nx = (G - x + 7) / 8, before = (G / 8) * x + min(x, G % 8);
    const int lo = (int)((int64_t)units * before / G);
    u_end = (int)((int64_t)units * (before + nx) / G);
    u = lo + blockIdx.x / 8;
    u_step = nx;
  }
  if (u >= u_end) return;
  // unit -> tile: groups of 8 tile rows, column by column
  auto tile_of = [&](int v, int &m0, int &n0, int &part) __attribute__((always_inline)) {
    part = v % p.splits;
    const int t = v / p.splits, per = 8 * tn, g = t / per, gm = min(8, tm - g * 8), r = t - g * per;
    m0 = (g * 8 + r % gm) * BM;
    n0 = r / gm * BN;
  };

  Stage<TA, BM, NW, 0> a;
  Stage<TW, BN, NW, PERM> w;
  int is_u = u, is_left = 0;  // issue cursor: unit and its steps left
  auto is_start = [&]() __attribute__((always_inline)) {
    int m0, n0, part;
    tile_of(is_u, m0, n0, part);
    const int q0 = part * p.ksteps;
    is_left = min(kt, q0 + p.ksteps) - q0;
    a.start(p.A, p.lda, p.M, p.K, m0, q0 * BK, wave, lane);
    w.start(p.W, p.ldw, p.N, p.K, n0, q0 * BK, wave, lane);
  };
  auto is_next = [&]() __attribute__((always_inline)) {
    a.next();
    w.next();
    if (__builtin_expect(--is_left == 0, 0)) {
      is_u += u_step;
      if (is_u < u_end) is_start();
      else is_left = 0x7fffffff;
    }
  };
  is_start();
  constexpr int DA = Stage<TA, BM, NW, 0>::D, DT = DA + Stage<TW, BN, NW, PERM>::D;
  auto open = [&]() __attribute__((always_inline)) {
    a.open(is_u < u_end);
    w.open(is_u < u_end);
  };
  auto issue = [&](int d, uint32_t slot) __attribute__((always_inline)) {
    if (d < DA) a.issue(d, slot, wave, lane);
    else w.issue(d - DA, slot + SA, wave, lane);
  };

  // With a permuted W, lane (g, c) = (lane / 16, lane % 16) holds rows 4 g .. 4 g + 3 of each 16 and NJ
  // consecutive columns from c NJ on: 16 lanes store one contiguous piece of a row. A T operand's columns
  // cannot be permuted: its product is formed transposed, so that a lane holds row c and columns 4 g .. 4 g + 3
  // of each 16.
  auto store = [&](const v4i (&acc)[NI][NJ], int v) __attribute__((always_inline)) {
    int m0, n0, part;
    tile_of(v, m0, n0, part);
    const int c = lane & 15, g = lane >> 4;
    constexpr int RR = PERM ? 4 : 1;       // rows of a lane per i
    constexpr int CW = PERM ? NJ : 4;      // columns of one store
    constexpr int CN = PERM ? 1 : NJ;      // stores of a row
    const int nb = n0 + wn * (BN / WN) + (PERM ? c * NJ : g * 4);
    const int mb = m0 + wm * (BM / WM) + (PERM ? g * 4 : c);
    const bool full = m0 + BM <= p.M && n0 + BN <= p.N;
    auto at = [&](int i, int r, int q, int j) __attribute__((always_inline)) {
      return PERM ? acc[i][j][r] : acc[i][q][j];
    };
    // This wave's loads have arrived, the DMA of the next step with them: its wait, which would also
    // wait for the stores below, is left out (`ahead` in the main loop).
    if (p.splits > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      int32_t *const o = p.parts + ((int64_t)part * p.M + mb) * p.N + nb;
      typedef int vec __attribute__((ext_vector_type(CW), aligned(4)));
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          if (full || mb + i * 16 + r < p.M) {
#pragma unroll
            for (int q = 0; q < CN; ++q) {
              int32_t *const z = o + (int64_t)(i * 16 + r) * p.N + q * 16;
              if (full || nb + q * 16 + CW <= p.N) {
                vec t;
#pragma unroll
                for (int j = 0; j < CW; ++j) t[j] = at(i, r, q, j);
                *(vec *)z = t;
              } else {
#pragma unroll
                for (int j = 0; j < CW; ++j)
                  if (nb + q * 16 + j < p.N) z[j] = at(i, r, q, j);
              }
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      return;
    }
    float sw[CN][CW], bs[CN][CW];
#pragma unroll
    for (int q = 0; q < CN; ++q)
#pragma unroll
      for (int j = 0; j < CW; ++j) {
        const int n = min(nb + q * 16 + j, p.N - 1);
        sw[q][j] = p.sw ? p.sw[n] : 1.0f;
        bs[q][j] = p.bias ? p.bias[n] : 0.0f;
      }
    float sa[NI][RR];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int r = 0; r < RR; ++r) sa[i][r] = p.sa ? p.sa[min(mb + i * 16 + r, p.M - 1)] : 1.0f;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    auto rows = [&](auto full_c, auto nt_c) __attribute__((always_inline)) {
      constexpr bool whole = decltype(full_c)::value, nt = decltype(nt_c)::value;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          if (whole || mb + i * 16 + r < p.M) {
#pragma unroll
            for (int q = 0; q < CN; ++q) {
              const int64_t to = (int64_t)(mb + i * 16 + r) * p.N + nb + q * 16;
              float y[CW];
#pragma unroll
              for (int j = 0; j < CW; ++j) {
                y[j] = (float)at(i, r, q, j) * sa[i][r];
                if (!TW || p.sw) y[j] *= sw[q][j];
                if (p.bias) y[j] += bs[q][j];
              }
              if (whole || nb + q * 16 + CW <= p.N) {
                if (p.R) {
                  float t[CW];
                  loadv<OUT, CW>(p.R, to, t);
#pragma unroll
                  for (int j = 0; j < CW; ++j) y[j] += t[j];
                }
                storev<OUT, CW, nt>(p.Y, to, y);
              } else {
#pragma unroll
                for (int j = 0; j < CW; ++j)
                  if (nb + q * 16 + j < p.N) {
                    if (p.R) y[j] += load_out<OUT>(p.R, to + j);
                    store_out<OUT>(p.Y, to + j, y[j]);
                  }
              }
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (!full) rows(std::false_type(), std::false_type());
    else if (p.nt) rows(std::true_type(), std::true_type());
    else rows(std::true_type(), std::false_type());
  };

  Reader<TA, BM, NI> ra;
  Reader<TW, BN, NJ> rw;
  ra.start(lds0, wm * (BM / WM), lane);
  rw.start(lds0 + SA, wn * (BN / WN), lane);
  // half b's products, spread between them the reads of the other half and, with DMA, the loads of a
  // later step into `slot`
  auto half = [&](v4i (&acc)[NI][NJ], v4i (&fa)[2][NI], v4i (&fw)[2][NJ], auto b_c, uint32_t slot) __attribute__((always_inline)) {
    constexpr int b = decltype(b_c)::value;
    constexpr bool dma = b == 1;
#pragma unroll
    for (int j = 0; j < NJ; ++j) fw[b ^ 1][j] = rw.read(j, b ^ 1);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      fa[b ^ 1][i] = ra.read(i, b ^ 1);
      if constexpr (dma) {
#pragma unroll
        for (int d = i * DT / NI; d < (i + 1) * DT / NI; ++d) issue(d, slot);
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        acc[i][j] = PERM ? __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[b][i], fw[b][j], acc[i][j], 0, 0, 0)
                         : __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[b][j], fa[b][i], acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int q = 0; q < S; ++q) {
    open();
#pragma unroll
    for (int d = 0; d < DT; ++d) issue(d, lds0 + q * SLOT);
    is_next();
  }
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"((S - 1) * DT) : "memory");
  wg_barrier();
  uint32_t slot = 0;  // byte offset of the slot that is multiplied
  int ahead = 0;      // steps whose data is known to have arrived
  for (; u < u_end; u += u_step) {
    v4i acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = (v4i){0, 0, 0, 0};
    v4i fa[2][NI], fw[2][NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) fw[0][j] = rw.read(j, 0);
#pragma unroll
    for (int i = 0; i < NI; ++i) fa[0][i] = ra.read(i, 0);
    const int q0 = (u % p.splits) * p.ksteps;
    for (int left = min(kt, q0 + p.ksteps) - q0; left > 0; --left) {
      half(acc, fa, fw, std::integral_constant<int, 0>(), 0);
      // the next step's data has arrived (the DMA of S - 2 later steps may be under way), and every wave
      // holds this step's second half
      if (ahead > 0) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"((S - 2) * DT) : "memory");
      --ahead;
      wg_barrier();
      const uint32_t by = slot == (S - 1) * SLOT ? 0u - (S - 1) * SLOT : SLOT;
      ra.shift(by);
      rw.shift(by);
      open();
      half(acc, fa, fw, std::integral_constant<int, 1>(), lds0 + slot);
      is_next();
      slot += by;
    }
    store(acc, u);
    ahead = S - 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA into LDS outlives the workgroup
}

// Joins the parts of a split reduction, V columns per thread. Their sum may pass 32 bits (K > 133144):
// 64-bit integers. (The 4096 x 1536 bf16 outputs of 150144 terms: 14 us of the product's 920.)
template <int OUT, int V>
__global__ __launch_bounds__(256) void combine_kernel(const Prob p) {
  const int per = p.N / V;
  const int64_t total = (int64_t)p.M * p.N, n = (int64_t)p.M * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / per;
    const int c = (int)(i - m * per) * V;
    const int64_t at = m * p.N + c;
    typedef int vec __attribute__((ext_vector_type(V)));
    int64_t s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = 0;
#pragma unroll 4
    for (int k = 0; k < p.splits; ++k) {
      const vec q = *(const vec *)(p.parts + k * total + at);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] += q[j];
    }
    const float sa = p.sa ? p.sa[m] : 1.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float y = (float)s[j] * sa;
      if (p.sw) y = y * p.sw[c + j];
      if (p.bias) y = y + p.bias[c + j];
      if (p.R) y = y + load_out<OUT>(p.R, at + j);
      store_out<OUT>(p.Y, at + j, y);
    }
  }
}
template <int OUT>
static void launch_combine(const Prob &p, hipStream_t st) {
  const unsigned g = (unsigned)std::min<int64_t>(cdiv((int64_t)p.M * p.N, p.N % 4 == 0 ? 1024 : 256), 16384);
  if (p.N % 4 == 0) combine_kernel<OUT, 4><<<g, 256, 0, st>>>(p);
  else combine_kernel<OUT, 1><<<g, 256, 0, st>>>(p);
}

// int32 sums of |a w| <= 127^2 hold 133144 terms
constexpr int kMaxSteps = 1024;

// Tile, parts of the reduction, and steps of a part: the least time by a model of a launch (us), 5 + rounds of
// units over the CUs * (steps * step + unit), and for parts their traffic at 4.5 TB/s and the combine's launch.
// `step` and `unit` are fitted to measured products (us, best form and its neighbours): 8192^3 256 x 256 480,
// 256 x 192 547, 128 x 128 614; 8192 x 1536 x 1536 256 x 192 24.7, 256 x 256 26, 128 x 128 30.3; 2047 x 1792
// x 6869 128 x 128 alone on a CU 38.5, 64 x 128 40.5, two per CU with 2 parts 45.8; 2047 x 1792 x 1792 64 x
// 128 15.9, 128 x 128 alone 18.1, 64 x 64 19.6; 1021 x 1792 x 597 64 x 64 8.5, 64 x 128 8.7, 128 x 128 11.1;
// 300 x 333 x 500 64 x 64 5.4, 128 x 128 8.8.
struct Form {
  int bm, bn, per_cu;
  float step, unit;
};
constexpr Form kForms[] = {{256, 256, 1, 1.82f, 3.5f}, {256, 192, 1, 1.4f, 2.6f}, {128, 128, 2, 1.0f, 2.2f},
                           {128, 128, 1, 0.53f, 4.5f}, {64, 128, 2, 0.62f, 2.2f}, {64, 64, 2, 0.42f, 1.4f}};
constexpr int kNumForms = sizeof(kForms) / sizeof(kForms[0]);

struct Plan {
  int form, splits, ksteps;
};
static Plan plan(int64_t M, int64_t N, int64_t K) {
  const int64_t kt = cdiv(K, BK), s_min = cdiv(kt, kMaxSteps);
  Plan best{0, 1, (int)kt};
  double best_t = 1e30;
  for (int f = 0; f < kNumForms; ++f) {
    const Form &c = kForms[f];
    const int64_t tiles = cdiv(M, c.bm) * cdiv(N, c.bn), slots = 256 * c.per_cu;
    const int64_t s_max = std::max(s_min, std::min<int64_t>({cdiv(kt, 4), std::max<int64_t>(1, 2 * slots / tiles), 64}));
    for (int64_t s = s_min; s <= s_max; ++s) {
      const int64_t ks = cdiv(kt, s), sp = cdiv(kt, ks), units = tiles * sp;
      // one workgroup of two on a CU runs its steps faster
      const double step = c.per_cu == 2 && units <= 256 ? 0.65 * c.step : c.step;
      double t = 5.0 + (double)cdiv(units, slots) * ((double)ks * step + c.unit);
      if (sp > 1) t += 5.0 + (double)(M * N) * (5.2 * (double)sp + 4.0) / 4.5e6;
      if (t < best_t) best_t = t, best = Plan{f, (int)sp, (int)ks};
    }
  }
  return best;
}

template <int BM, int BN, int WM, int WN, int S, bool TA, bool TW, int OUT>
static void launch_tile(const Prob &p, int per_cu, hipStream_t st) {
  constexpr int lds = S * (BM + BN) * BK;
  static const hipError_t set = hipFuncSetAttribute((const void *)gemm_kernel<BM, BN, WM, WN, S, TA, TW, OUT>,
                                                    hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  (void)set;
  const int64_t units = cdiv(p.M, BM) * cdiv(p.N, BN) * p.splits;
  gemm_kernel<BM, BN, WM, WN, S, TA, TW, OUT>
      <<<(unsigned)std::min<int64_t>(units, (int64_t)cu_count() * per_cu), WM * WN * 64, lds, st>>>(p);
}

template <bool TA, bool TW, int OUT>
static void launch_form(int form, const Prob &p, hipStream_t st) {
  const int n = kForms[form].per_cu;
  switch (form) {
    case 0: launch_tile<256, 256, 2, 4, 2, TA, TW, OUT>(p, n, st); break;
    case 1: launch_tile<256, 192, 4, 2, 2, TA, TW, OUT>(p, n, st); break;
    case 2: launch_tile<128, 128, 2, 2, 2, TA, TW, OUT>(p, n, st); break;
    case 3: launch_tile<128, 128, 2, 2, 4, TA, TW, OUT>(p, n, st); break;
    case 4: launch_tile<64, 128, 2, 2, 3, TA, TW, OUT>(p, n, st); break;
    default: launch_tile<64, 64, 2, 2, 4, TA, TW, OUT>(p, n, st);
  }
}

template <int OUT>
static void launch(int form, const Prob &p, bool ta, bool tw, hipStream_t st) {
  if (ta) {  // a weight gradient
    if constexpr (OUT == KSD_F32) launch_form<true, true, OUT>(form, p, st);
  } else if (tw) {
    launch_form<false, true, OUT>(form, p, st);
  } else {
    launch_form<false, false, OUT>(form, p, st);
  }
  if (p.splits > 1) launch_combine<OUT>(p, st);
}


// -------------------------------------------------------------------------------------- few rows
// y for few tokens in one launch: what bounds it is one read of the codes of W (or the launch itself).
// Every workgroup quantizes the M tokens into LDS (their first W chunks are already on the way) and walks
// tiles of 16 columns; its 4 waves take every fourth 64 steps of the reduction, W straight into MFMA registers
// (each byte is used once), and meet in LDS. (bf16, us: 1 x 1536 -> 512 4.5, quantizing and a 128 x 128 product
// 13; 4 x 1536 -> 150144 38, 6.1 TB/s, against 52.)
struct Few {
  const void *x;
  const int8_t *W;
  const float *sw, *bias;
  const void *R;
  void *Y;
  int64_t stride, ldw;
  int M, N, K, pitch;  // pitch: bytes of an LDS row of codes, = 16 mod 256 (16 rows on 16 bank groups)
};

template <int DT, int OUT>
__global__ __launch_bounds__(256) void few_rows_kernel(const Few p) {
  using T = typename Elem<DT>::T;
  constexpr int U = 6;  // W chunks in flight per wave
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];  // codes, then 2 x 4 x 256 int32 and M scales
  int32_t *const part = (int32_t *)(smem + (int64_t)p.M * p.pitch);
  float *const sx = (float *)(part + 2 * 4 * 256);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int nk = (p.K + 63) / 64, kb = (p.K + 15) & ~15, tiles = (p.N + 15) / 16;
  v4i w[U];
  auto load = [&](int t, int k0) __attribute__((always_inline)) {
    const int8_t *row = p.W + (int64_t)min(t * 16 + c16, p.N - 1) * p.ldw;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = (k0 + i * 4) * 64 + g * 16;
      w[i] = *(const v4i *)(row + (k < kb ? k : 0));  // steps past K meet zero codes of x
    }
  };
  int t = blockIdx.x;
  load(t, wave);
  for (int m = wave; m < p.M; m += 4) {
    const T *row = (const T *)p.x + m * p.stride;
    constexpr int NC = 4;
    float v[NC][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = (c * 64 + lane) * 8;
      if (k < p.K) {
        load8_tail<DT>(row, k, p.K, v[c]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) top = max(top, __builtin_bit_cast(uint32_t, abs_max<8>(v[c])));
    for (int k = (NC * 64 + lane) * 8; k < p.K; k += 512) {
      float q[8];
      load8_tail<DT>(row, k, p.K, q);
      top = max(top, __builtin_bit_cast(uint32_t, abs_max<8>(q)));
    }
    top = wave_max(top);
    float scale, inv;
    row_scale(top, scale, inv);
    const bool bad = top >= 0x7f800000u;
    if (lane == 0) sx[m] = scale;
    int8_t *out = smem + m * p.pitch;
    auto put = [&](int k, const float *q) __attribute__((always_inline)) {
      const uint2 o = make_uint2(bad ? 0 : pack4(q[0] * inv, q[1] * inv, q[2] * inv, q[3] * inv),
                                 bad ? 0 : pack4(q[4] * inv, q[5] * inv, q[6] * inv, q[7] * inv));
      *(uint2 *)(out + k) = o;
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = (c * 64 + lane) * 8;
      if (k < nk * 64) put(k, v[c]);
    }
    for (int k = (NC * 64 + lane) * 8; k < nk * 64; k += 512) {
      float q[8];
      if (k < p.K) {
        load8_tail<DT>(row, k, p.K, q);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = 0.0f;
      }
      put(k, q);
    }
  }
  __syncthreads();
  const int8_t *const arow = smem + (int64_t)min(c16, p.M - 1) * p.pitch + g * 16;
  int par = 0;
  for (; t < tiles; t += gridDim.x, par ^= 1) {
    v4i acc = (v4i){0, 0, 0, 0};
    for (int k0 = wave; k0 < nk; k0 += 4 * U) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int k = k0 + i * 4;
        if (k < nk) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const v4i *)(arow + k * 64), w[i], acc, 0, 0, 0);
      }
      if (k0 + 4 * U < nk) load(t, k0 + 4 * U);
      else if (t + (int)gridDim.x < tiles) load(t + gridDim.x, wave);
    }
    if (wave >= nk && t + (int)gridDim.x < tiles) load(t + gridDim.x, wave);
    int32_t *const q = part + (par * 4 + wave) * 256;
#pragma unroll
    for (int r = 0; r < 4; ++r) q[(g * 4 + r) * 16 + c16] = acc[r];
    __syncthreads();
    const int m = tid >> 4, n = t * 16 + (tid & 15);
    if (m < p.M && n < p.N) {
      const int32_t *z = part + par * 4 * 256 + tid;
      const int32_t sum = z[0] + z[256] + z[2 * 256] + z[3 * 256];
      float y = ((float)sum * sx[m]) * p.sw[n];
      const int64_t at = (int64_t)m * p.N + n;
      if (p.bias) y += p.bias[n];
      if (p.R) y += load_out<OUT>(p.R, at);
      store_out<OUT>(p.Y, at, y);
    }
  }
}

// Every workgroup quantizes all tokens, a wave a quarter of them one after the other: up to 8192 values of a
// wave. (us, against quantizing and the product, in a graph: 1536 -> 512 2 tokens 3.6 and 9.2, 16 tokens 7.2 and
// 9.8; 1536 -> 150144 2 tokens 37 and 39, 8 tokens 37 and 41, 16 tokens 41.7 and 40.7; outside one 24 x 1536 -> 512
// 10.6 and 11.4, 4 x 6869 -> 1792 12.6 and 13.3, 8 tokens 19.9 and 13.4, 1 x 16384 -> 1024 22 and 16. The rule does not
// look at N: short rows onto many columns are quantized in more workgroups than pays, 512 -> 32003 8 tokens 8.6 and
// 8.3, 16 tokens 10.6 and 8.4.)
static bool few_rows(int64_t M, int64_t K) { return M <= 16 && cdiv(M, 4) * K <= 8192; }

template <int DT, int OUT>
static void launch_few(const Few &p, hipStream_t st) {
  const int lds = p.M * p.pitch + 2 * 4 * 1024 + 4 * p.M;  // at most 42 KB
  // 4 workgroups on a CU: more quantize more often (16 x 512 -> 32003, us: 4 11.8, 8 15.7), fewer read W more
  // slowly (4 x 1536 -> 150144: 4 38, 1 50).
  const int per_cu = std::min(4, 160 * 1024 / lds);
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(p.N, 16), (int64_t)cu_count() * per_cu);
  few_rows_kernel<DT, OUT><<<grid, 256, lds, st>>>(p);
}
template <int DT>
static void launch_few(int out, const Few &p, hipStream_t st) {
  if (out == KSD_F32) launch_few<DT, KSD_F32>(p, st);
  else if (out == KSD_BF16) launch_few<DT, KSD_BF16>(p, st);
  else launch_few<DT, KSD_F16>(p, st);
}

static bool float_type(int t) { return t == KSD_F32 || t == KSD_BF16 || t == KSD_F16; }
static int64_t pad256(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t pitch16(int64_t n) { return (n + 15) / 16 * 16; }

}  // namespace tc
}  // namespace ksd

using namespace ksd;

// Checks what every entry asks of a float matrix and its codes.
static int check_rows(const char *who, const void *x, int t, int64_t M, int64_t K, const int8_t *codes, int64_t ld, const float *scales) {
  if (M < 0 || K < 1) return fail(KSD_EINVAL, "%s: bad shape (%lld, %lld)", who, (long long)M, (long long)K);
  if (!tc::float_type(t)) return fail(KSD_ETYPE, "%s: unsupported element type %d", who, t);
  if (ld != tc::pitch16(K)) return fail(KSD_EINVAL, "%s: pitch %lld must be K rounded up to 16", who, (long long)ld);
  if (M == 0) return KSD_OK;
  if (!x || !codes || !scales) return fail(KSD_EINVAL, "%s: null pointer", who);
  if (((uintptr_t)codes) % 16) return fail(KSD_EINVAL, "%s: codes must be 16-byte aligned", who);
  if (!grid_fits(M, 256)) return fail(KSD_EINVAL, "%s: too many rows", who);
  return KSD_OK;
}

extern "C" int ksd_tc_quantize_rows(const void *x, int x_dtype, int64_t M, int64_t K, int64_t stride, int8_t *codes,
                                    int64_t ld, float *scales, void *stream) {
  const int rc = check_rows("tc_quantize_rows", x, x_dtype, M, K, codes, ld, scales);
  if (rc || M == 0) return rc;
  tc::launch_rows(tc::Rows{x, M, K, stride, ld, codes, scales}, x_dtype, (hipStream_t)stream);
  return check_launch("tc_quantize_rows");
}

extern "C" int ksd_tc_gemm_workspace(int64_t M, int64_t N, int64_t K, int64_t *bytes) {
  if (M < 0 || N < 0 || K < 1 || !bytes) return fail(KSD_EINVAL, "tc_gemm_workspace: bad arguments");
  const int splits = M > 0 && N > 0 ? tc::plan(M, N, K).splits : 1;
  *bytes = splits > 1 ? (int64_t)splits * M * N * 4 : 0;
  return KSD_OK;
}

extern "C" int ksd_tc_gemm_form(int64_t M, int64_t N, int64_t K, int *tile_m, int *tile_n, int *per_cu, int *splits) {
  if (M < 1 || N < 1 || K < 1 || !tile_m || !tile_n || !per_cu || !splits) return fail(KSD_EINVAL, "tc_gemm_form: bad arguments");
  const tc::Plan pl = tc::plan(M, N, K);
  *tile_m = tc::kForms[pl.form].bm, *tile_n = tc::kForms[pl.form].bn, *per_cu = tc::kForms[pl.form].per_cu;
  *splits = pl.splits;
  return KSD_OK;
}

extern "C" int ksd_tc_gemm(const int8_t *a, int64_t lda, int a_t, const float *sa, const int8_t *w, int64_t ldw, int w_t,
                           const float *sw, int64_t M, int64_t N, int64_t K, const float *bias, const void *residual,
                           void *y, int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  if (M < 0 || N < 0 || K < 1)
    return fail(KSD_EINVAL, "tc_gemm: bad shape (%lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
  if (out_dtype != KSD_F32 && out_dtype != KSD_BF16 && out_dtype != KSD_F16)
    return fail(KSD_ETYPE, "tc_gemm: unsupported output type %d", out_dtype);
  if (a_t && (!w_t || out_dtype != KSD_F32))
    return fail(KSD_EINVAL, "tc_gemm: a transposed A needs a transposed W and an fp32 output");
  const int64_t ra = a_t ? K : M, ca = a_t ? M : K, rw = w_t ? K : N, cw = w_t ? N : K;
  if (lda % 16 || ldw % 16 || lda < cdiv(ca, 16) * 16 || ldw < cdiv(cw, 16) * 16)
    return fail(KSD_EINVAL, "tc_gemm: row pitches must be multiples of 16 that cover the rows");
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff || lda > 0x3fffff || ldw > 0x3fffff || ra < 0 || rw < 0)
    return fail(KSD_EINVAL, "tc_gemm: shape too large");
  if (M == 0 || N == 0) return KSD_OK;
  if (!a || !w || !y) return fail(KSD_EINVAL, "tc_gemm: null pointer");
  if (((uintptr_t)a) % 16 || ((uintptr_t)w) % 16) return fail(KSD_EINVAL, "tc_gemm: codes must be 16-byte aligned");
  tc::Prob p{a, w, sa, sw, bias, residual, y, (int32_t *)workspace, lda, ldw, (int)M, (int)N, (int)K, 1, 0, 0};
  const tc::Plan pl = tc::plan(M, N, K);
  p.splits = pl.splits, p.ksteps = pl.ksteps;
  // Where 16 lanes store whole 64-byte pieces (4096 x 150144 x 1536 over and over: 1090 -> 925 us); pieces that
  // other stores complete are put together in L2 (8192 x 1536 from a T operand: 28 us, non-temporal 40).
  p.nt = !w_t && ((uintptr_t)y) % 64 == 0 && N * (out_dtype == KSD_F32 ? 4 : 2) % 64 == 0;
  const int64_t need = p.splits > 1 ? (int64_t)p.splits * M * N * 4 : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(KSD_EINVAL, "tc_gemm: workspace of %lld bytes needed", (long long)need);
  if (!grid_fits(cdiv(M, 64) * cdiv(N, 64), 256)) return fail(KSD_EINVAL, "tc_gemm: shape too large");
  hipStream_t st = (hipStream_t)stream;
  switch (out_dtype) {
    case KSD_F32: tc::launch<KSD_F32>(pl.form, p, a_t, w_t, st); break;
    case KSD_BF16: tc::launch<KSD_BF16>(pl.form, p, a_t, w_t, st); break;
    default: tc::launch<KSD_F16>(pl.form, p, a_t, w_t, st);
  }
  return check_launch("tc_gemm");
}

extern "C" int ksd_tc_grad_workspace(int64_t M, int64_t N, int64_t *bytes) {
  if (M < 0 || N < 0 || !bytes) return fail(KSD_EINVAL, "tc_grad_workspace: bad arguments");
  const int64_t ncb = cdiv(N, 256), nrb = cdiv(M, tc::stats_rows(M, N));
  *bytes = 4 * (ncb * M + 2 * nrb * N + M + N);
  return KSD_OK;
}

extern "C" int ksd_tc_quantize_grad(const void *g, int g_dtype, int64_t M, int64_t N, int64_t stride, const float *sx,
                                    const float *sw, int8_t *q, float *e, int8_t *c, float *f, int64_t ld, float *db,
                                    void *workspace, int64_t workspace_bytes, void *stream) {
  if (M < 0 || N < 0) return fail(KSD_EINVAL, "tc_quantize_grad: bad shape");
  if (g_dtype != KSD_F32 && g_dtype != KSD_BF16 && g_dtype != KSD_F16)
    return fail(KSD_ETYPE, "tc_quantize_grad: unsupported element type %d", g_dtype);
  if (ld < N || ld % 16 != 0) return fail(KSD_EINVAL, "tc_quantize_grad: pitch must be N rounded up to 16");
  if (M == 0 || N == 0) return KSD_OK;
  int64_t need = 0;
  ksd_tc_grad_workspace(M, N, &need);
  if (!g || !sx || !sw || !e || !f || !workspace || workspace_bytes < need)
    return fail(KSD_EINVAL, "tc_quantize_grad: null pointer or short workspace");
  const int rows = tc::stats_rows(M, N);
  const bool large = tc::large_grad(M, N);
  const int64_t ncb = cdiv(N, large && g_dtype != KSD_F32 ? 512 : 256), nrb = cdiv(M, rows);
  if (!grid_fits(cdiv(M, 64) + cdiv(N, 64), 1024)) return fail(KSD_EINVAL, "tc_quantize_grad: too many rows or columns");
  uint32_t *row_part = (uint32_t *)workspace, *col_part = row_part + ncb * M;
  float *sum_part = (float *)(col_part + nrb * N), *einv = sum_part + nrb * N, *finv = einv + M;
  float *sums = db ? sum_part : nullptr;
  hipStream_t st = (hipStream_t)stream;
  const dim3 gs = tc::row_grid(cdiv(ncb, 4), nrb), gq = tc::row_grid(cdiv(ld, 512), cdiv(M, large ? 64 : 32));
  const unsigned folds = (unsigned)(cdiv(M, 64) + cdiv(N, 64));
#define KSD_TC(DT, V)                                                                                                  \
  if (large) tc::grad_stats_kernel<DT, V><<<gs, 256, 0, st>>>(g, M, N, stride, rows, sx, sw, row_part, col_part, sums); \
  else tc::grad_stats_kernel<DT, 4><<<gs, 256, 0, st>>>(g, M, N, stride, rows, sx, sw, row_part, col_part, sums);       \
  tc::grad_fold_kernel<<<folds, 1024, 0, st>>>(row_part, col_part, sum_part, M, N, (int)ncb, (int)nrb, e, einv, f, finv, db); \
  if ((q || c) && large) tc::grad_codes_kernel<DT, 2><<<gq, 256, 0, st>>>(g, M, N, stride, sx, sw, einv, finv, q, c, ld); \
  else if (q || c) tc::grad_codes_kernel<DT, 1><<<gq, 256, 0, st>>>(g, M, N, stride, sx, sw, einv, finv, q, c, ld);
  switch (g_dtype) {
    case KSD_F32: KSD_TC(KSD_F32, 4) break;
    case KSD_BF16: KSD_TC(KSD_BF16, 8) break;
    default: KSD_TC(KSD_F16, 8)
  }
#undef KSD_TC
  return check_launch("tc_quantize_grad");
}

extern "C" int ksd_tc_linear_workspace(int64_t M, int64_t N, int64_t K, int64_t *bytes) {
  if (M < 0 || N < 0 || K < 1 || !bytes) return fail(KSD_EINVAL, "tc_linear_workspace: bad arguments");
  if (tc::few_rows(M, K)) {
    *bytes = 0;
    return KSD_OK;
  }
  const int rc = ksd_tc_gemm_workspace(M, N, K, bytes);
  *bytes += tc::pad256(M * tc::pitch16(K)) + tc::pad256(4 * M);
  return rc;
}

extern "C" int ksd_tc_linear(const void *x, int x_dtype, int64_t M, int64_t K, int64_t stride, const int8_t *w, int64_t ldw,
                             const float *sw, int64_t N, const float *bias, const void *residual, void *y, int out_dtype,
                             void *workspace, int64_t workspace_bytes, void *stream) {
  int64_t need = 0;
  const int rc = ksd_tc_linear_workspace(M, N, K, &need);
  if (rc) return rc;
  if (!tc::float_type(x_dtype) || !tc::float_type(out_dtype)) return fail(KSD_ETYPE, "tc_linear: unsupported element type");
  if (M == 0 || N == 0) return KSD_OK;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(KSD_EINVAL, "tc_linear: workspace of %lld bytes needed", (long long)need);
  hipStream_t st = (hipStream_t)stream;
  if (tc::few_rows(M, K)) {
    if (!x || !w || !sw || !y) return fail(KSD_EINVAL, "tc_linear: null pointer");
    if (ldw % 16 || ldw < tc::pitch16(K) || ((uintptr_t)w) % 16)
      return fail(KSD_EINVAL, "tc_linear: the codes' rows must be 16-byte aligned and cover K rounded up to 16");
    if (N > 0x7fffffff / 2) return fail(KSD_EINVAL, "tc_linear: shape too large");
    const tc::Few p{x, w, sw, bias, residual, y, stride, ldw, (int)M, (int)N, (int)K, (int)(cdiv(K, 256) * 256 + 16)};
    if (x_dtype == KSD_F32) tc::launch_few<KSD_F32>(out_dtype, p, st);
    else if (x_dtype == KSD_BF16) tc::launch_few<KSD_BF16>(out_dtype, p, st);
    else tc::launch_few<KSD_F16>(out_dtype, p, st);
    return check_launch("tc_linear");
  }
  int8_t *codes = (int8_t *)workspace;
  const int64_t ld = tc::pitch16(K), cb = tc::pad256(M * ld), sb = tc::pad256(4 * M);
  float *scales = (float *)(codes + cb);
  const int rq = ksd_tc_quantize_rows(x, x_dtype, M, K, stride, codes, ld, scales, stream);
  if (rq) return rq;
  return ksd_tc_gemm(codes, ld, 0, scales, w, ldw, 0, sw, M, N, K, bias, residual, y, out_dtype, codes + cb + sb,
                     workspace_bytes - cb - sb, stream);
}

extern "C" int ksd_tc_linear_train(const void *x, int x_dtype, int64_t M, int64_t K, int64_t stride, const void *w, int w_dtype,
                                   int64_t N, int64_t w_stride, const float *bias, const void *residual, int8_t *x_codes,
                                   float *x_scales, int8_t *w_codes, float *w_scales, void *y, int out_dtype, void *workspace,
                                   int64_t workspace_bytes, void *stream) {
  const int64_t ld = tc::pitch16(K);
  int rc = check_rows("tc_linear_train", x, x_dtype, M, K, x_codes, ld, x_scales);
  if (!rc) rc = check_rows("tc_linear_train", w, w_dtype, N, K, w_codes, ld, w_scales);
  if (rc) return rc;
  if (!grid_fits(M + N, 256)) return fail(KSD_EINVAL, "tc_linear_train: too many rows");
  const tc::Rows a{w, N, K, w_stride, ld, w_codes, w_scales}, b{x, M, K, stride, ld, x_codes, x_scales};
  hipStream_t st = (hipStream_t)stream;
  if (M + N > 0) {
    if (w_dtype != KSD_F32) {
      if (N > 0) tc::launch_rows(a, w_dtype, st);
      if (M > 0) tc::launch_rows(b, x_dtype, st);
    } else if (x_dtype == KSD_F32) {
      tc::launch_rows<KSD_F32, KSD_F32>(a, b, st);
    } else if (x_dtype == KSD_BF16) {
      tc::launch_rows<KSD_F32, KSD_BF16>(a, b, st);
    } else {
      tc::launch_rows<KSD_F32, KSD_F16>(a, b, st);
    }
  }
  return ksd_tc_gemm(x_codes, ld, 0, x_scales, w_codes, ld, 0, w_scales, M, N, K, bias, residual, y, out_dtype, workspace,
                     workspace_bytes, stream);
}

namespace {
// the backward's scratch: q, c, scales, then one region that the gradient's statistics and the two
// products' parts use in turn
struct BackwardScratch {
  int64_t q, c, ef, rest, bytes;
};
BackwardScratch backward_scratch(int64_t M, int64_t N, int64_t K, bool dx, bool dw) {
  BackwardScratch s;
  const int64_t codes = tc::pad256(M * tc::pitch16(N));
  s.q = 0;
  s.c = s.q + (dx ? codes : 0);
  s.ef = s.c + (dw ? codes : 0);
  s.rest = s.ef + tc::pad256(4 * (M + N));
  int64_t a = 0, b = 0, c = 0;
  ksd_tc_grad_workspace(M, N, &a);
  if (dx) ksd_tc_gemm_workspace(M, K, N, &b);
  if (dw) ksd_tc_gemm_workspace(N, K, M, &c);
  s.bytes = s.rest + std::max(a, std::max(b, c));
  return s;
}
}  // namespace

extern "C" int ksd_tc_linear_backward_workspace(int64_t M, int64_t N, int64_t K, int need_dx, int need_dw, int64_t *bytes) {
  if (M < 1 || N < 1 || K < 1 || !bytes) return fail(KSD_EINVAL, "tc_linear_backward_workspace: bad arguments");
  *bytes = backward_scratch(M, N, K, need_dx, need_dw).bytes;
  return KSD_OK;
}

extern "C" int ksd_tc_linear_backward(const void *g, int g_dtype, int64_t M, int64_t N, int64_t stride, int64_t K,
                                      const int8_t *x_codes, const float *x_scales, const int8_t *w_codes, const float *w_scales,
                                      void *dx, int dx_dtype, float *dw, float *db, void *workspace, int64_t workspace_bytes,
                                      void *stream) {
  if (M < 1 || N < 1 || K < 1) return fail(KSD_EINVAL, "tc_linear_backward: bad shape");
  const BackwardScratch s = backward_scratch(M, N, K, dx, dw);
  if (!workspace || workspace_bytes < s.bytes) return fail(KSD_EINVAL, "tc_linear_backward: workspace of %lld bytes needed", (long long)s.bytes);
  char *ws = (char *)workspace;
  int8_t *q = dx ? (int8_t *)(ws + s.q) : nullptr, *c = dw ? (int8_t *)(ws + s.c) : nullptr;
  float *e = (float *)(ws + s.ef), *f = e + M;
  const int64_t ld = tc::pitch16(N), ldk = tc::pitch16(K), rest = workspace_bytes - s.rest;
  int rc = ksd_tc_quantize_grad(g, g_dtype, M, N, stride, x_scales, w_scales, q, e, c, f, ld, db, ws + s.rest, rest, stream);
  if (!rc && dx)
    rc = ksd_tc_gemm(q, ld, 0, e, w_codes, ldk, 1, nullptr, M, K, N, nullptr, nullptr, dx, dx_dtype, ws + s.rest, rest, stream);
  if (!rc && dw)
    rc = ksd_tc_gemm(c, ld, 1, f, x_codes, ldk, 1, nullptr, N, K, M, nullptr, nullptr, dw, KSD_F32, ws + s.rest, rest, stream);
  return rc;
}
