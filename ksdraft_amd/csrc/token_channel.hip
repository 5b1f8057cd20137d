// W8A8 product with one fp32 scale per row of each operand (per token and per output channel):
//
//   y[m,n] = ((sum_k a[m,k] w[n,k]) * sa[m]) * sw[n]  (+ bias[n])  (+ residual[m,n]),  rounded once
//
// The scales stand outside the sum, so the whole reduction stays in the int8 matrix unit with exact
// int32 sums; the group-128 product of gemm.hip rescales every 128 steps on the VALU instead.
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

namespace ksd {
namespace tc {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

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
// LANES threads per row (64: four rows per workgroup; 256: one), the first NCH * LANES * 8 elements
// kept in registers between the maximum and the codes, the rest read again (from cache).
template <int DT, int LANES, int NCH>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void *__restrict__ x, int64_t M, int64_t K,
                                                         int64_t stride, int8_t *__restrict__ codes, int64_t ld,
                                                         float *__restrict__ scales) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x % LANES;
  const int64_t m = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (LANES == 64 && m >= M) return;
  const T *row = (const T *)x + m * stride;
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
  if (lane == 0) scales[m] = scale;
  int8_t *out = codes + m * ld;
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

template <int DT>
static void launch_rows(const void *x, int64_t M, int64_t K, int64_t stride, int8_t *codes, int64_t ld,
                        float *scales, hipStream_t st) {
  if (K <= 512) quant_rows_kernel<DT, 64, 1><<<(unsigned)cdiv(M, 4), 256, 0, st>>>(x, M, K, stride, codes, ld, scales);
  else if (K <= 1536) quant_rows_kernel<DT, 64, 3><<<(unsigned)cdiv(M, 4), 256, 0, st>>>(x, M, K, stride, codes, ld, scales);
  else quant_rows_kernel<DT, 256, 4><<<(unsigned)M, 256, 0, st>>>(x, M, K, stride, codes, ld, scales);
}

// ------------------------------------------------------------------------------- gradient's codes
// Workgroup (row block, column block) of 64 x 1024 elements of dY: thread t holds columns 4t .. 4t+3
// over all rows (column maxima of |dY * sx| and column sums), each row's maximum of |dY * sw| goes
// through the workgroup. Partial results per block, folded by grad_fold_kernel in a fixed order.
constexpr int GR = 64, GC = 1024;

template <int DT>
__device__ __forceinline__ void load4_tail(const typename Elem<DT>::T *row, int64_t c, int64_t N, float *v) {
  using T = typename Elem<DT>::T;
  if (c + 4 <= N) {
    if constexpr (DT == KSD_F32) {
      struct __attribute__((packed, aligned(4))) Any { uint4 q; };
      const uint4 q = ((const Any *)(row + c))->q;
      v[0] = __builtin_bit_cast(float, q.x), v[1] = __builtin_bit_cast(float, q.y);
      v[2] = __builtin_bit_cast(float, q.z), v[3] = __builtin_bit_cast(float, q.w);
    } else {
      struct __attribute__((packed, aligned(2))) Any { uint2 q; };
      const uint2 q = ((const Any *)(row + c))->q;
      const T h[4] = {(T)(q.x & 0xffff), (T)(q.x >> 16), (T)(q.y & 0xffff), (T)(q.y >> 16)};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = Elem<DT>::load(&h[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < N ? Elem<DT>::load(row + c + j) : 0.0f;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void grad_stats_kernel(const void *__restrict__ g, int64_t M, int64_t N, int64_t stride,
                                                         const float *__restrict__ sx, const float *__restrict__ sw,
                                                         uint32_t *__restrict__ row_part, uint32_t *__restrict__ col_part,
                                                         float *__restrict__ sum_part) {
  using T = typename Elem<DT>::T;
  __shared__ uint32_t rmax[GR][4];
  const int tid = threadIdx.x;
  const int64_t cb = blockIdx.x, rb = blockIdx.y, c = cb * GC + tid * 4, m0 = rb * GR;
  float w[4], sum[4] = {0, 0, 0, 0};
  uint32_t cm[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = c + j < N ? sw[c + j] : 0.0f;
  const int rows = (int)min((int64_t)GR, M - m0);
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    float v[4] = {0, 0, 0, 0};
    if (c < N) load4_tail<DT>((const T *)g + (m0 + r) * stride, c, N, v);
    const float s = sx[m0 + r];
    float t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      t[j] = c + j < N ? v[j] * w[j] : 0.0f;
      sum[j] += v[j];
      cm[j] = max(cm[j], __builtin_bit_cast(uint32_t, fabsf(v[j] * s)));
    }
    const uint32_t top = wave_max(__builtin_bit_cast(uint32_t, abs_max<4>(t)));
    if ((tid & 63) == 0) rmax[r][tid >> 6] = top;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < N) {
      col_part[rb * N + c + j] = cm[j];
      if (sum_part) sum_part[rb * N + c + j] = sum[j];
    }
  __syncthreads();
  if (tid < rows)
    row_part[cb * M + m0 + tid] = max(max(rmax[tid][0], rmax[tid][1]), max(rmax[tid][2], rmax[tid][3]));
}

// scales, reciprocals and column sums from the partial results; thread i < M is row i, the next N
// threads are the columns
__global__ __launch_bounds__(256) void grad_fold_kernel(const uint32_t *__restrict__ row_part, const uint32_t *__restrict__ col_part,
                                                        const float *__restrict__ sum_part, int64_t M, int64_t N, int ncb, int nrb,
                                                        float *__restrict__ e, float *__restrict__ einv, float *__restrict__ f,
                                                        float *__restrict__ finv, float *__restrict__ db) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < M) {
    uint32_t top = 0;
    for (int b = 0; b < ncb; ++b) top = max(top, row_part[(int64_t)b * M + i]);
    float s, inv;
    row_scale(top, s, inv);
    e[i] = s, einv[i] = inv;
  } else if (i < M + N) {
    const int64_t n = i - M;
    uint32_t top = 0;
    float sum = 0.0f;
    for (int b = 0; b < nrb; ++b) {
      top = max(top, col_part[(int64_t)b * N + n]);
      if (sum_part) sum += sum_part[(int64_t)b * N + n];
    }
    float s, inv;
    row_scale(top, s, inv);
    f[n] = s, finv[n] = inv;
    if (db) db[n] = sum;
  }
}

// Both codes of dY, in its own layout: q (rows, for dX) and c (columns, for dW), rows of ld bytes
// with zeros past N. A thread holds 8 columns over 8 rows.
template <int DT>
__global__ __launch_bounds__(256) void grad_codes_kernel(const void *__restrict__ g, int64_t M, int64_t N, int64_t stride,
                                                         const float *__restrict__ sx, const float *__restrict__ sw,
                                                         const float *__restrict__ einv, const float *__restrict__ finv,
                                                         const float *__restrict__ e, const float *__restrict__ f,
                                                         int8_t *__restrict__ q, int8_t *__restrict__ cq, int64_t ld) {
  using T = typename Elem<DT>::T;
  const int64_t c = ((int64_t)blockIdx.x * 64 + (threadIdx.x & 63)) * 8;
  const int64_t m0 = (int64_t)blockIdx.y * 32 + (threadIdx.x >> 6) * 8;
  if (c >= ld) return;
  float w[8], fi[8];
  bool cbad[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = c + j < N ? sw[c + j] : 0.0f;
    fi[j] = c + j < N ? finv[c + j] : 0.0f;
    cbad[j] = c + j < N && f[c + j] != f[c + j];
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t m = m0 + r;
    if (m >= M) break;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c < N) load8_tail<DT>((const T *)g + m * stride, c, N, v);
    if (q) {
      const float inv = einv[m];
      const bool bad = e[m] != e[m];
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = bad || c + j >= N ? 0.0f : (v[j] * w[j]) * inv;
      *(uint2 *)(q + m * ld + c) = make_uint2(pack4(t[0], t[1], t[2], t[3]), pack4(t[4], t[5], t[6], t[7]));
    }
    if (cq) {
      const float s = sx[m];
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = cbad[j] || c + j >= N ? 0.0f : (v[j] * s) * fi[j];
      *(uint2 *)(cq + m * ld + c) = make_uint2(pack4(t[0], t[1], t[2], t[3]), pack4(t[4], t[5], t[6], t[7]));
    }
  }
}

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
};

constexpr int BK = 128;

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)(p);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t off, int8_t *lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16, off, 0, 0, 0);
}

// Position of 16-byte chunk c of LDS row r, in bytes. N tiles have rows of 128 bytes (the reduction),
// T tiles rows of B bytes (the output index), row = reduction step. The chunk index is XORed so that
// the 16 lanes that read one fragment chunk (16 rows of an N tile; 8 rows of a T tile, two such row
// sets per 32 lanes) hit 16 different 16-byte bank groups.
template <bool T, int B>
__device__ __forceinline__ int lds_pos(int r, int c) {
  if constexpr (!T) return r * BK + ((c ^ ((r >> 1) & 7)) << 4);
  else if constexpr (B == 256) return r * 256 + ((c ^ ((r & 7) | ((r >> 1) & 8))) << 4);
  else return r * 128 + ((c ^ (((r >> 1) & 3) | ((r >> 2) & 4))) << 4);
}

// Fills a B x 128 tile: rows [row0, row0 + B) (output index), reduction steps [k0, k0 + 128) of an
// operand with `rows` output rows and K reduction steps. NW waves; what lies outside reads as zero.
// PERM: the output index of LDS row p within each block of 16 NJ rows is permuted so that one lane's
// results are 4 NJ consecutive columns (see the store).
template <bool T, int B, int NW, int NJ>
__device__ __forceinline__ void fill(const int8_t *P, int64_t ld, int rows, int K, int row0, int k0, int8_t *lds,
                                     int wave, int lane) {
  constexpr int INSTR = B * BK / 1024;  // 1 KB each
  if constexpr (!T) {
    const int valid = min(B, rows - row0), kb = (K + 15) & ~15;
    const __amdgpu_buffer_rsrc_t r = rsrc(P + (int64_t)row0 * ld, (int64_t)valid * ld);
#pragma unroll
    for (int i = wave; i < INSTR; i += NW) {
      const int p = i * 8 + (lane >> 3), c = (lane & 7) ^ ((p >> 1) & 7);
      int row = p;
      if constexpr (NJ > 0) {
        const int b = p / (16 * NJ), o = p % (16 * NJ), j = o >> 4, ii = o & 15;
        row = b * (16 * NJ) + (ii >> 2) * (4 * NJ) + j * 4 + (ii & 3);
      }
      const int k = k0 + c * 16;
      const uint32_t off = row < valid && k < kb ? (uint32_t)(row * ld + k) : kOob;
      dma16(r, off, lds + i * 1024);
    }
  } else {
    const int valid = min(BK, K - k0), cb = (rows + 15) & ~15;
    const __amdgpu_buffer_rsrc_t r = rsrc(P + (int64_t)k0 * ld, (int64_t)max(valid, 0) * ld);
#pragma unroll
    for (int i = wave; i < INSTR; i += NW) {
      constexpr int CPR = B / 16;
      const int kr = i * (64 / CPR) + lane / CPR, slot = lane % CPR;
      const int c = slot ^ ((lds_pos<true, B>(kr, 0) >> 4) & (CPR - 1));
      const int col = row0 + c * 16;
      const uint32_t off = kr < valid && col < cb ? (uint32_t)(kr * ld + col) : kOob;
      dma16(r, off, lds + i * 1024);
    }
  }
}

// 16 output rows x 64 reduction steps as an MFMA operand: lane l holds row l % 16, steps
// 16 (l / 16) .. + 15 of half kk.
template <bool T, int B>
__device__ __forceinline__ v4i frag(const int8_t *lds, int row0, int kk, int lane) {
  if constexpr (!T) {
    return *(const v4i *)(lds + lds_pos<false, B>(row0 + (lane & 15), kk * 4 + (lane >> 4)));
  } else {
    // lanes 2r, 2r + 1 of each 16 address the two halves of step r's 16 bytes; the read leaves lane
    // c the 8 steps of column c
    typedef __attribute__((address_space(3))) v2i lds_v2i;
    const int kr = kk * 64 + (lane >> 4) * 16 + ((lane & 15) >> 1);
    const v2i lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_v2i *)(lds + lds_pos<true, B>(kr, row0 >> 4) + (lane & 1) * 8));
    const v2i hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_v2i *)(lds + lds_pos<true, B>(kr + 8, row0 >> 4) + (lane & 1) * 8));
    return (v4i){lo.x, lo.y, hi.x, hi.y};
  }
}

template <int OUT>
__device__ __forceinline__ float load_out(const void *p, int64_t i) {
  return Elem<OUT>::load((const typename Elem<OUT>::T *)p + i);
}

// BM x BN tiles, WM x WN waves; TA, TW: the operand is a T one.
template <int BM, int BN, int WM, int WN, bool TA, bool TW, int OUT>
__global__ __launch_bounds__(WM *WN * 64) void gemm_kernel(const Prob p) {
  constexpr int NW = WM * WN, NI = BM / WM / 16, NJ = BN / WN / 16;
  constexpr int PERM = TW ? 0 : NJ;
  __shared__ __attribute__((aligned(16))) int8_t sA[2][BM * BK];
  __shared__ __attribute__((aligned(16))) int8_t sW[2][BN * BK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tn = (p.N + BN - 1) / BN;
  const int t = blockIdx.x / p.splits, part = blockIdx.x % p.splits;
  const int m0 = t / tn * BM, n0 = t % tn * BN;
  const int kt = (p.K + BK - 1) / BK, q0 = part * p.ksteps, q1 = min(kt, q0 + p.ksteps);
  auto stage = [&](int q) {
    fill<TA, BM, NW, 0>(p.A, p.lda, p.M, p.K, m0, q * BK, sA[q & 1], wave, lane);
    fill<TW, BN, NW, PERM>(p.W, p.ldw, p.N, p.K, n0, q * BK, sW[q & 1], wave, lane);
  };
  v4i acc[NI][NJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = (v4i){0, 0, 0, 0};
  if (q0 < q1) stage(q0);
  for (int q = q0; q < q1; ++q) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (q + 1 < q1) stage(q + 1);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      v4i a[NI], w[NJ];
#pragma unroll
      for (int i = 0; i < NI; ++i) a[i] = frag<TA, BM>(sA[q & 1], wm * (BM / WM) + i * 16, kk, lane);
#pragma unroll
      for (int j = 0; j < NJ; ++j) w[j] = frag<TW, BN>(sW[q & 1], wn * (BN / WN) + j * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], a[i], acc[i][j], 0, 0, 0);
    }
  }
  // lane l of tile (i, j) holds row l % 16 and 4 consecutive columns
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int m = m0 + wm * (BM / WM) + i * 16 + (lane & 15);
    if (m >= p.M) continue;
    const float sa = p.sa ? p.sa[m] : 1.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + wn * (BN / WN) + (PERM ? (lane >> 4) * 4 * NJ + j * 4 : j * 16 + (lane >> 4) * 4) + r;
        if (n >= p.N) continue;
        const int64_t at = (int64_t)m * p.N + n;
        if (p.splits > 1) {
          p.parts[(int64_t)part * p.M * p.N + at] = acc[i][j][r];
          continue;
        }
        float y = (float)acc[i][j][r] * sa;
        if (p.sw) y = y * p.sw[n];
        if (p.bias) y = y + p.bias[n];
        if (p.R) y = y + load_out<OUT>(p.R, at);
        store_out<OUT>(p.Y, at, y);
      }
  }
}

// Joins the parts of a split reduction. Their sum may pass 32 bits (K > 133144): 64-bit integers.
template <int OUT>
__global__ __launch_bounds__(256) void combine_kernel(const Prob p) {
  const int64_t total = (int64_t)p.M * p.N;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
    int64_t s = 0;
    for (int k = 0; k < p.splits; ++k) s += p.parts[k * total + at];
    const int64_t m = at / p.N, n = at - m * p.N;
    float y = (float)s * (p.sa ? p.sa[m] : 1.0f);
    if (p.sw) y = y * p.sw[n];
    if (p.bias) y = y + p.bias[n];
    if (p.R) y = y + load_out<OUT>(p.R, at);
    store_out<OUT>(p.Y, at, y);
  }
}

constexpr int TM = 128, TN = 128;
// int32 sums of |a w| <= 127^2 hold 133144 terms
constexpr int kMaxSteps = 1024;

static void plan(int64_t M, int64_t N, int64_t K, int &splits, int &ksteps) {
  const int64_t tiles = cdiv(M, TM) * cdiv(N, TN), kt = cdiv(K, BK);
  int64_t s = 1;
  if (tiles < 256) s = std::max<int64_t>(1, std::min<int64_t>(512 / tiles, kt / 4));
  s = std::max(s, cdiv(kt, kMaxSteps));
  ksteps = (int)cdiv(kt, s);
  splits = (int)cdiv(kt, ksteps);
}

template <int OUT>
static void launch(const Prob &p, bool ta, bool tw, hipStream_t st) {
  const unsigned g = (unsigned)(cdiv(p.M, TM) * cdiv(p.N, TN) * p.splits);
  if (ta && tw) gemm_kernel<TM, TN, 2, 2, true, true, OUT><<<g, 256, 0, st>>>(p);
  else if (tw) gemm_kernel<TM, TN, 2, 2, false, true, OUT><<<g, 256, 0, st>>>(p);
  else gemm_kernel<TM, TN, 2, 2, false, false, OUT><<<g, 256, 0, st>>>(p);
  if (p.splits > 1) combine_kernel<OUT><<<(unsigned)std::min<int64_t>(cdiv((int64_t)p.M * p.N, 256), 8192), 256, 0, st>>>(p);
}

}  // namespace tc
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_tc_quantize_rows(const void *x, int x_dtype, int64_t M, int64_t K, int64_t stride, int8_t *codes,
                                    int64_t ld, float *scales, void *stream) {
  if (M < 0 || K < 1) return fail(KSD_EINVAL, "tc_quantize_rows: bad shape (%lld, %lld)", (long long)M, (long long)K);
  if (x_dtype != KSD_F32 && x_dtype != KSD_BF16 && x_dtype != KSD_F16)
    return fail(KSD_ETYPE, "tc_quantize_rows: unsupported element type %d", x_dtype);
  if (ld < K || ld % 16 != 0 || ld >= K + 16)
    return fail(KSD_EINVAL, "tc_quantize_rows: pitch %lld must be K rounded up to 16", (long long)ld);
  if (M == 0) return KSD_OK;
  if (!x || !codes || !scales) return fail(KSD_EINVAL, "tc_quantize_rows: null pointer");
  if (((uintptr_t)codes) % 16) return fail(KSD_EINVAL, "tc_quantize_rows: codes must be 16-byte aligned");
  if (!grid_fits(M, 256)) return fail(KSD_EINVAL, "tc_quantize_rows: too many rows");
  hipStream_t st = (hipStream_t)stream;
  switch (x_dtype) {
    case KSD_F32: tc::launch_rows<KSD_F32>(x, M, K, stride, codes, ld, scales, st); break;
    case KSD_BF16: tc::launch_rows<KSD_BF16>(x, M, K, stride, codes, ld, scales, st); break;
    default: tc::launch_rows<KSD_F16>(x, M, K, stride, codes, ld, scales, st);
  }
  return check_launch("tc_quantize_rows");
}

extern "C" int ksd_tc_gemm_workspace(int64_t M, int64_t N, int64_t K, int64_t *bytes) {
  if (M < 0 || N < 0 || K < 1 || !bytes) return fail(KSD_EINVAL, "tc_gemm_workspace: bad arguments");
  int splits = 1, ksteps = 0;
  if (M > 0 && N > 0) tc::plan(M, N, K, splits, ksteps);
  *bytes = splits > 1 ? (int64_t)splits * M * N * 4 : 0;
  return KSD_OK;
}

extern "C" int ksd_tc_gemm(const int8_t *a, int64_t lda, int a_t, const float *sa, const int8_t *w, int64_t ldw, int w_t,
                           const float *sw, int64_t M, int64_t N, int64_t K, const float *bias, const void *residual,
                           void *y, int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  if (M < 0 || N < 0 || K < 1)
    return fail(KSD_EINVAL, "tc_gemm: bad shape (%lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
  if (out_dtype != KSD_F32 && out_dtype != KSD_BF16 && out_dtype != KSD_F16)
    return fail(KSD_ETYPE, "tc_gemm: unsupported output type %d", out_dtype);
  if (a_t && !w_t) return fail(KSD_EINVAL, "tc_gemm: a transposed A needs a transposed W");
  const int64_t ra = a_t ? K : M, ca = a_t ? M : K, rw = w_t ? K : N, cw = w_t ? N : K;
  if (lda % 16 || ldw % 16 || lda < cdiv(ca, 16) * 16 || ldw < cdiv(cw, 16) * 16)
    return fail(KSD_EINVAL, "tc_gemm: row pitches must be multiples of 16 that cover the rows");
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff || lda > 0x3fffff || ldw > 0x3fffff || ra < 0 || rw < 0)
    return fail(KSD_EINVAL, "tc_gemm: shape too large");
  if (M == 0 || N == 0) return KSD_OK;
  if (!a || !w || !y) return fail(KSD_EINVAL, "tc_gemm: null pointer");
  if (((uintptr_t)a) % 16 || ((uintptr_t)w) % 16) return fail(KSD_EINVAL, "tc_gemm: codes must be 16-byte aligned");
  tc::Prob p{a, w, sa, sw, bias, residual, y, (int32_t *)workspace, lda, ldw, (int)M, (int)N, (int)K, 1, 0};
  tc::plan(M, N, K, p.splits, p.ksteps);
  const int64_t need = p.splits > 1 ? (int64_t)p.splits * M * N * 4 : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(KSD_EINVAL, "tc_gemm: workspace of %lld bytes needed", (long long)need);
  if (!grid_fits(cdiv(M, tc::TM) * cdiv(N, tc::TN) * p.splits, 256)) return fail(KSD_EINVAL, "tc_gemm: shape too large");
  hipStream_t st = (hipStream_t)stream;
  switch (out_dtype) {
    case KSD_F32: tc::launch<KSD_F32>(p, a_t, w_t, st); break;
    case KSD_BF16: tc::launch<KSD_BF16>(p, a_t, w_t, st); break;
    default: tc::launch<KSD_F16>(p, a_t, w_t, st);
  }
  return check_launch("tc_gemm");
}

extern "C" int ksd_tc_grad_workspace(int64_t M, int64_t N, int64_t *bytes) {
  if (M < 0 || N < 0 || !bytes) return fail(KSD_EINVAL, "tc_grad_workspace: bad arguments");
  const int64_t ncb = cdiv(N, tc::GC), nrb = cdiv(M, tc::GR);
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
  const int64_t ncb = cdiv(N, tc::GC), nrb = cdiv(M, tc::GR);
  if (nrb > 65535 || cdiv(M, 32) > 65535) return fail(KSD_EINVAL, "tc_quantize_grad: too many rows");
  uint32_t *row_part = (uint32_t *)workspace, *col_part = row_part + ncb * M;
  float *sum_part = (float *)(col_part + nrb * N), *einv = sum_part + nrb * N, *finv = einv + M;
  hipStream_t st = (hipStream_t)stream;
  const dim3 gs((unsigned)ncb, (unsigned)nrb), gq((unsigned)cdiv(ld, 512), (unsigned)cdiv(M, 32));
#define KSD_TC(DT)                                                                                                  \
  tc::grad_stats_kernel<DT><<<gs, 256, 0, st>>>(g, M, N, stride, sx, sw, row_part, col_part, db ? sum_part : nullptr); \
  tc::grad_fold_kernel<<<(unsigned)cdiv(M + N, 256), 256, 0, st>>>(row_part, col_part, db ? sum_part : nullptr, M, N, \
                                                                   (int)ncb, (int)nrb, e, einv, f, finv, db);       \
  if (q || c) tc::grad_codes_kernel<DT><<<gq, 256, 0, st>>>(g, M, N, stride, sx, sw, einv, finv, e, f, q, c, ld);
  switch (g_dtype) {
    case KSD_F32: KSD_TC(KSD_F32) break;
    case KSD_BF16: KSD_TC(KSD_BF16) break;
    default: KSD_TC(KSD_F16)
  }
#undef KSD_TC
  return check_launch("tc_quantize_grad");
}
