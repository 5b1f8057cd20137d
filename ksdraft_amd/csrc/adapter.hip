// Low-rank adapters of many requests beside a shared projection, forward and backward.
//
//   h[m] = s_i x~[m] A_i^T,   y[m] = base[m] + h[m] B_i^T           i = index[m]
//   g[m] = s_i dY[m] B_i,     dX[m] = dXbase[m] + mask(g[m] A_i)
//   dA_i = sum of g[m]^T x~[m],   dB_i = sum of dY[m]^T h[m]         over the tokens m of adapter i
//
// with x~ = dropout(x) where a mask is given (made from its counter, stored nowhere). A token without an adapter
// keeps base. Adapters of other tokens never touch a token's row, whatever they hold.
//
// Both passes of a token's row are one launch of pair_kernel: a workgroup of 8 waves holds up to 32 rows; the
// waves split the contraction of the narrow product, their sums join in LDS, and the same waves then split the
// columns of the wide one. h is never rounded on its way: it is fp32 in LDS and enters the 16-bit matrix
// instructions as a rounded value and the rounding's rest, side by side along the contraction, which a rank of 16
// leaves half empty anyway. What bounds it is memory: x and base read once, y written once.
#include "ksd_random.h"

#include <algorithm>

namespace ksd {
namespace adp {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8;

// 8 elements of one row as an operand holds them: raw 16-bit values, or floats.
template <int DT> struct Oct { using V = s16x8; };
template <> struct Oct<KSD_F32> { using V = f32x8; };

// Elements c .. c + 7 of a row of n, zeros from n on, at any alignment of the type.
template <int DT>
__device__ __forceinline__ typename Oct<DT>::V load_oct(const typename Elem<DT>::T *row, int64_t c, int64_t n) {
  using T = typename Elem<DT>::T;
  using V = typename Oct<DT>::V;
  struct __attribute__((packed, aligned(sizeof(T)))) Any { V v; };
  if (c + 8 <= n) return ((const Any *)(row + c))->v;
  V v;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    T e = 0;
    if (c + j < n) e = row[c + j];
    if constexpr (DT == KSD_F32) v[j] = e;
    else v[j] = (short)e;
  }
  return v;
}
__device__ __forceinline__ f32x4 load_four(const float *row, int c, int n) {
  struct __attribute__((packed, aligned(4))) Any { f32x4 v; };
  if (c + 4 <= n) return ((const Any *)(row + c))->v;
  f32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = c + j < n ? row[c + j] : 0.0f;
  return v;
}
template <int DT>
__device__ __forceinline__ void to_floats(const typename Oct<DT>::V &v, float *f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (DT == KSD_F32) f[j] = v[j];
    else if constexpr (DT == KSD_BF16) f[j] = bf16_to_f32((uint16_t)v[j]);
    else f[j] = f16_to_f32((uint16_t)v[j]);
  }
}
template <int DT>
__device__ __forceinline__ typename Oct<DT>::V from_floats(const float *f) {
  typename Oct<DT>::V v;
  if constexpr (DT == KSD_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f[j];
  } else if constexpr (DT == KSD_BF16) {
    f32x8 w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = f[j];
    v = __builtin_bit_cast(s16x8, __builtin_convertvector(w, bf16x8));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (short)f16_bits(f[j]);
  }
  return v;
}
template <int DT>
__device__ __forceinline__ void store_oct(typename Elem<DT>::T *row, int64_t c, int64_t n, const float *f) {
  using T = typename Elem<DT>::T;
  using V = typename Oct<DT>::V;
  struct __attribute__((packed, aligned(sizeof(T)))) Any { V v; };
  const V v = from_floats<DT>(f);
  if (c + 8 <= n) {
    ((Any *)(row + c))->v = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c + j < n) {
      if constexpr (DT == KSD_F32) row[c + j] = v[j];
      else row[c + j] = (T)v[j];
    }
}

// One step of a contraction over 32 columns (8 per lane group of 16): 16-bit types one matrix instruction, fp32
// eight of 4 columns, the j-th of which takes the lanes' j-th values.
template <int DT>
__device__ __forceinline__ f32x4 product(const typename Oct<DT>::V &a, const typename Oct<DT>::V &b, f32x4 c) {
  if constexpr (DT == KSD_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == KSD_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
}

struct PairArgs {
  const void *x;           // (M, K), row stride
  int64_t x_stride, M, K, N;
  const void *a;           // (n, r, K)
  const void *b;           // (n, N, r)
  const void *index;       // one for `per` rows
  int wide;                // int64
  int64_t per;
  const float *scales;     // (n,) or NULL
  const void *base;        // (M, N) or NULL
  int64_t base_stride;
  void *y;                 // (M, N) dense
  float *hidden;           // (M, r) or NULL
  int n, r, rows, cols;    // rows and columns (a multiple of 64) of a workgroup
  Mask mask;
  int mask_x, mask_y;
};

__device__ __forceinline__ int adapter_of(const void *index, int wide, int64_t per, int64_t m, int n) {
  const int64_t at = per == 1 ? m : m / per;
  const int64_t i = wide ? ((const int64_t *)index)[at] : (int64_t)((const int32_t *)index)[at];
  return i >= 0 && i < n ? (int)i : -1;
}

// R16: blocks of 16 ranks; RT: blocks of 16 rows.
template <int DT, int R16, int RT, bool MASK>
__global__ __launch_bounds__(64 * kWaves) void pair_kernel(const PairArgs p) {
  using T = typename Elem<DT>::T;
  using V = typename Oct<DT>::V;
  constexpr int R = 16 * R16, U = DT == KSD_F32 ? (R16 <= 2 ? 2 : 1) : (R16 <= 2 ? 4 : 2);
  constexpr int pitch = R + 4;  // floats: a row's four lanes of 16 bytes start 4 banks further than the last row's
  extern __shared__ float lds[];  // (kWaves, 16 RT, pitch): sums of a wave's columns; the first holds h
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * p.rows;
  const int rows = (int)min((int64_t)p.rows, p.M - row0);
  // lane l < 16 RT: the adapter of row l
  const int mine = lane < rows ? adapter_of(p.index, p.wide, p.per, row0 + lane, p.n) : -1;
  int of[RT];  // of the rows that this lane's columns of the products are
#pragma unroll
  for (int t = 0; t < RT; ++t) of[t] = __shfl(mine, t * 16 + col);
  const uint64_t with = __ballot(mine >= 0);
  MaskKey key{};
  if constexpr (MASK) key = mask_key(p.mask);

  if (with) {
    // ---- h: D[rank][token] = A x^T over this wave's columns
    const int64_t steps = (p.K + 31) / 32, share = ((steps + kWaves - 1) / kWaves + 1) & ~1ll;
    const int64_t from = wave * share, to = min(steps, from + share);
    for (uint64_t left = with; left;) {
      const int i = __shfl(mine, __builtin_ctzll(left));
      left &= ~__ballot(mine == i);
      const T *const a = (const T *)p.a + (int64_t)i * p.r * p.K;
      f32x4 acc[RT][R16] = {};
      for (int64_t s = from; s < to; s += U) {
        V xv[U][RT], av[U][R16];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t k = (s + u) * 32 + grp * 8;
          const bool in = s + u < to;
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            xv[u][t] = V{};
            if (in && of[t] == i) xv[u][t] = load_oct<DT>((const T *)p.x + (row0 + t * 16 + col) * p.x_stride, k, p.K);
          }
#pragma unroll
          for (int q = 0; q < R16; ++q) {
            av[u][q] = V{};
            if (in && q * 16 + col < p.r) av[u][q] = load_oct<DT>(a + (int64_t)(q * 16 + col) * p.K, k, p.K);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if constexpr (MASK) {
            if (p.mask_x) {
#pragma unroll
              for (int t = 0; t < RT; ++t) {
                float f[8];
                to_floats<DT>(xv[u][t], f);
                apply_mask(p.mask, mask_bits(p.mask, key, row0 + t * 16 + col, (uint32_t)((s + u) * 4 + grp)), f);
                // 16-bit: the scaled value would be rounded; the scale goes to h instead
                if constexpr (DT != KSD_F32) {
#pragma unroll
                  for (int j = 0; j < 8; ++j) xv[u][t][j] = f[j] == 0.0f ? (short)0 : xv[u][t][j];
                } else {
                  xv[u][t] = from_floats<DT>(f);
                }
              }
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int q = 0; q < R16; ++q) acc[t][q] = product<DT>(av[u][q], xv[u][t], acc[t][q]);
        }
      }
      float s = p.scales ? p.scales[i] : 1.0f;
      if constexpr (MASK && DT != KSD_F32) s *= p.mask_x ? p.mask.scale : 1.0f;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (of[t] == i) {
          float *const o = lds + ((int64_t)wave * 16 * RT + t * 16 + col) * pitch + grp * 4;
#pragma unroll
          for (int q = 0; q < R16; ++q) *(f32x4 *)(o + q * 16) = acc[t][q] * s;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * RT * R; e += 64 * kWaves) {
      const int t = e / R, q = e % R;
      if (t < rows && (with >> t & 1)) {
        float v = lds[t * pitch + q];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += lds[(w * 16 * RT + t) * pitch + q];
        lds[t * pitch + q] = v;
        if (p.hidden && blockIdx.y == 0 && q < p.r) p.hidden[(row0 + t) * p.r + q] = v;
      }
    }
    __syncthreads();
  }
  if (p.hidden && blockIdx.y == 0) {  // rows without an adapter
    for (int e = threadIdx.x; e < rows * p.r; e += 64 * kWaves)
      if (!(with >> (e / p.r) & 1)) p.hidden[row0 * p.r + e] = 0.0f;
  }

  // ---- y: D[column][token] = B h^T. Row i of product t is column (i / 4) 16 + 4 t + i % 4 of a block of 64, so a
  // lane ends with 16 consecutive columns of its token.
  using H = typename Oct<DT>::V;
  H hv[RT][R16];
  float back[RT];
  if (with) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float *const h = lds + (t * 16 + col) * pitch;
      back[t] = 1.0f;
      if constexpr (DT == KSD_F32) {  // ranks 4 grp .. + 3 of a block of 16 (the upper 4 stay unused)
#pragma unroll
        for (int q = 0; q < R16; ++q) {
          const f32x4 v = *(const f32x4 *)(h + q * 16 + grp * 4);
          hv[t][q] = H{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
        }
      } else {  // ranks 8 (grp % 2) .. + 7: rounded in the lower two groups, the rest in the upper two
        float up = 1.0f;
        if constexpr (DT == KSD_F16) {  // brought to [1, 2) by a power of two: fp16's range is short
          float top = 0.0f;
#pragma unroll
          for (int q = 0; q < R16; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(h[q * 16 + (grp & 1) * 8 + j]));
          top = fmaxf(top, __shfl_xor(top, 16));
          const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
          if (e > 0 && e < 254) {
            up = __builtin_bit_cast(float, (uint32_t)(254 - e) << 23);
            back[t] = __builtin_bit_cast(float, (uint32_t)e << 23);
          }
        }
#pragma unroll
        for (int q = 0; q < R16; ++q) {
          float f[8], g[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = h[q * 16 + (grp & 1) * 8 + j] * up;
          hv[t][q] = from_floats<DT>(f);
          if (grp >= 2) {
            to_floats<DT>(hv[t][q], g);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = fabsf(g[j]) <= 3.0e38f ? f[j] - g[j] : 0.0f;
            hv[t][q] = from_floats<DT>(f);
          }
        }
      }
    }
  }
  if (!p.y) return;
  const int64_t n0 = (int64_t)blockIdx.y * p.cols, n1 = min(p.N, n0 + p.cols);
  for (int64_t c = n0 + wave * 64; c < n1; c += 64 * kWaves) {
    const int64_t at = c + grp * 16;
    V bv[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        bv[t][v] = V{};
        if (p.base && t * 16 + col < rows && at + v * 8 < p.N)
          bv[t][v] = load_oct<DT>((const T *)p.base + (row0 + t * 16 + col) * p.base_stride, at + v * 8, p.N);
      }
    f32x4 acc[RT][4] = {};
    for (uint64_t left = with; left;) {
      const int i = __shfl(mine, __builtin_ctzll(left));
      left &= ~__ballot(mine == i);
      f32x4 d[RT][4] = {};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t n = min(c + (col >> 2) * 16 + t * 4 + (col & 3), p.N - 1);
        const T *const b = (const T *)p.b + ((int64_t)i * p.N + n) * p.r;
#pragma unroll
        for (int q = 0; q < R16; ++q) {
          if constexpr (DT == KSD_F32) {
            const f32x4 w = load_four(b, q * 16 + grp * 4, p.r);
#pragma unroll
            for (int u = 0; u < RT; ++u)
#pragma unroll
              for (int j = 0; j < 4; ++j) d[u][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[j], hv[u][q][j], d[u][t], 0, 0, 0);
          } else {
            const V w = load_oct<DT>(b, q * 16 + (grp & 1) * 8, p.r);
#pragma unroll
            for (int u = 0; u < RT; ++u) d[u][t] = product<DT>(w, hv[u][q], d[u][t]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[u][t] = of[u] == i ? d[u][t] * back[u] : acc[u][t];
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      if (u * 16 + col >= rows) continue;
      const int64_t m = row0 + u * 16 + col;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (at + v * 8 >= p.N) continue;
        float f[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = acc[u][v * 2 + j / 4][j & 3];
        if constexpr (MASK) {
          if (p.mask_y) apply_mask(p.mask, mask_bits(p.mask, key, m, (uint32_t)((at >> 3) + v)), f);
        }
        to_floats<DT>(bv[u][v], g);
        if (p.base) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = of[u] >= 0 ? f[j] + g[j] : g[j];
        }
        store_oct<DT>((T *)p.y + m * p.N, at + v * 8, p.N, f);
      }
    }
  }
}

template <int DT, int R16, int RT>
static void launch_pair(const PairArgs &p, bool mask, hipStream_t st) {
  const dim3 g((unsigned)cdiv(p.M, p.rows), (unsigned)cdiv(p.N, p.cols));
  constexpr int lds = kWaves * 16 * RT * (16 * R16 + 4) * 4;
  if constexpr (lds > 65536) {  // past HIP's default
    static const hipError_t set[2] = {
        hipFuncSetAttribute((const void *)pair_kernel<DT, R16, RT, false>, hipFuncAttributeMaxDynamicSharedMemorySize, lds),
        hipFuncSetAttribute((const void *)pair_kernel<DT, R16, RT, true>, hipFuncAttributeMaxDynamicSharedMemorySize, lds)};
    (void)set;
  }
  if (mask) pair_kernel<DT, R16, RT, true><<<g, 64 * kWaves, lds, st>>>(p);
  else pair_kernel<DT, R16, RT, false><<<g, 64 * kWaves, lds, st>>>(p);
}
template <int DT>
static void launch_pair(const PairArgs &p, bool mask, hipStream_t st) {
  const bool one = p.rows <= 16;
  if (p.r <= 16) one ? launch_pair<DT, 1, 1>(p, mask, st) : launch_pair<DT, 1, 2>(p, mask, st);
  else if (p.r <= 32) one ? launch_pair<DT, 2, 1>(p, mask, st) : launch_pair<DT, 2, 2>(p, mask, st);
  else if (p.r <= 64) one ? launch_pair<DT, 4, 1>(p, mask, st) : launch_pair<DT, 4, 2>(p, mask, st);
  else launch_pair<DT, 8, 1>(p, mask, st);
}

// Rows and columns of a workgroup.
static void shape(PairArgs &p) {
  const int most = p.r <= 64 ? 32 : 16;
  p.rows = (int)std::max<int64_t>(1, std::min<int64_t>(most, cdiv(p.M, 256)));
  if (p.rows > 16 && p.rows < 32) p.rows = 16;
  const int64_t tiles = cdiv(p.M, p.rows), blocks = cdiv(p.N, 64);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(cdiv(blocks, kWaves), cdiv(512, tiles)));
  p.cols = (int)(cdiv(blocks, parts) * 64);
}

// ------------------------------------------------------------------------------- the adapters' gradients
// Tokens are listed by adapter (stable), each adapter's list in pieces of kPiece. Piece j of adapter i is slot
// start_i / kPiece + i + j: slots of different adapters never meet, and a slot knows its adapter without a sum over the
// earlier ones' pieces.
constexpr int kPiece = 256;

struct Slot {
  int adapter, from, to, pad;  // -1: empty
};

struct GroupArgs {
  const void *index;
  int wide, n;
  int64_t per, M;
  int32_t *order;   // (M,)
  Slot *slots;      // (M / kPiece + n,)
  int2 *spans;      // (n,): first slot, slots
};

// Workgroup i lists adapter i's tokens.
__global__ __launch_bounds__(256) void group_kernel(const GroupArgs a) {
  const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ int sums[2][4], counts[4];
  int less = 0, mine = 0;
  for (int64_t m = tid; m < a.M; m += 256) {
    const int v = adapter_of(a.index, a.wide, a.per, m, a.n);
    less += v >= 0 && v < i, mine += v == i;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) less += __shfl_xor(less, o), mine += __shfl_xor(mine, o);
  if (lane == 0) sums[0][wave] = less, sums[1][wave] = mine;
  __syncthreads();
  const int start = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3], len = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  const int slot = start / kPiece + i, next = (start + len) / kPiece + i + 1, pieces = (len + kPiece - 1) / kPiece;
  // the last adapter's workgroup empties the slots behind it too: tokens without an adapter take none
  const int upto = i == a.n - 1 ? (int)(a.M / kPiece) + a.n : next;
  for (int s = slot + tid; s < upto; s += 256) {
    const int at = start + (s - slot) * kPiece;
    a.slots[s] = s - slot < pieces ? Slot{i, at, min(at + kPiece, start + len), 0} : Slot{-1, 0, 0, 0};
  }
  if (tid == 0) a.spans[i] = make_int2(slot, pieces);
  if (len == 0) return;
  int done = start;
  for (int64_t base = 0; base < a.M; base += 256) {
    const int64_t m = base + tid;
    const bool in = m < a.M && adapter_of(a.index, a.wide, a.per, m, a.n) == i;
    const uint64_t b = __ballot(in);
    __syncthreads();
    if (lane == 0) counts[wave] = __popcll(b);
    __syncthreads();
    int at = done;
    for (int w = 0; w < wave; ++w) at += counts[w];
    if (in) a.order[at + __popcll(b & ((1ull << lane) - 1))] = (int32_t)m;
    done += counts[0] + counts[1] + counts[2] + counts[3];
  }
}

// out[i][c][r] = in[i][r][c] of 16- or 32-bit values, tiles of 32 x 32.
template <typename T>
__global__ __launch_bounds__(256) void turn_kernel(const T *__restrict__ in, T *__restrict__ out, int64_t rows, int64_t cols) {
  __shared__ T tile[32][33];
  const int64_t tr = (rows + 31) / 32, tc = (cols + 31) / 32;
  const int64_t t = blockIdx.x % (tr * tc), i = blockIdx.x / (tr * tc), r0 = t / tc * 32, c0 = t % tc * 32;
  in += i * rows * cols, out += i * rows * cols;
  for (int e = threadIdx.x; e < 1024; e += 256) {
    const int64_t r = r0 + e / 32, c = c0 + e % 32;
    if (r < rows && c < cols) tile[e / 32][e % 32] = in[r * cols + c];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 1024; e += 256) {
    const int64_t c = c0 + e / 32, r = r0 + e % 32;
    if (r < rows && c < cols) out[c * rows + r] = tile[e % 32][e / 32];
  }
}

struct GradArgs {
  const void *x, *g;        // (M, K), (M, N)
  int64_t x_stride, g_stride, K, N;
  const float *gh, *h;      // (M, r): the gradient's narrow product, the forward's
  const int32_t *order;
  const Slot *slots;
  float *parts;             // (slots, r K + N r)
  int r, a_blocks, masked;
  Mask mask;
};

// A slot's sums over its tokens for 128 columns of dA or dB and 64 ranks: D[rank][column] = p^T z in fp32 matrix
// instructions of 4 tokens, which read both operands as they lie in memory.
template <int DT>
__global__ __launch_bounds__(256) void grad_kernel(const GradArgs p) {
  using T = typename Elem<DT>::T;
  const Slot s = p.slots[blockIdx.y];
  if (s.adapter < 0) return;
  const bool of_a = (int)blockIdx.x < p.a_blocks;
  const int64_t width = of_a ? p.K : p.N, stride = of_a ? p.x_stride : p.g_stride;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  const int64_t c = (int64_t)(of_a ? blockIdx.x : blockIdx.x - p.a_blocks) * 128 + col * 8;
  const T *const z = (const T *)(of_a ? p.x : p.g);
  const float *const q = of_a ? p.gh : p.h;
  const int r0 = blockIdx.z * 64;
  const MaskKey key = p.masked ? mask_key(p.mask) : MaskKey{};
  f32x4 acc[4][8] = {};
  for (int m0 = s.from + wave * 4; m0 < s.to; m0 += 16) {
    const bool in = m0 + grp < s.to;
    const int64_t m = in ? p.order[m0 + grp] : 0;
    float f[8] = {};
    if (in && c < width) {
      to_floats<DT>(load_oct<DT>(z + m * stride, c, width), f);
      if (of_a && p.masked) apply_mask(p.mask, mask_bits(p.mask, key, m, (uint32_t)(c >> 3)), f);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (r0 + b * 16 >= p.r) break;
      const int rank = r0 + b * 16 + col;
      const float v = in && rank < p.r ? q[m * p.r + rank] : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, f[j], acc[b][j], 0, 0, 0);
    }
  }
  __shared__ f32x4 sum[4][8][64];
  float *const out = p.parts + (int64_t)blockIdx.y * p.r * (p.K + p.N);
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    if (r0 + b * 16 >= p.r) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[wave][j][lane] = acc[b][j];
    __syncthreads();
    // thread: 2 of the 8 products of its lane
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = wave * 2 + u;
      const f32x4 v = sum[0][j][lane] + sum[1][j][lane] + sum[2][j][lane] + sum[3][j][lane];
      const int64_t at = c + j;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int rank = r0 + b * 16 + grp * 4 + e;
        if (at < width && rank < p.r) {
          if (of_a) out[rank * p.K + at] = v[e];
          else out[p.r * p.K + at * p.r + rank] = v[e];
        }
      }
    }
  }
}

// da, db: an adapter's slots added in order.
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ parts, const int2 *__restrict__ spans, int64_t na,
                                                   int64_t nb, float *__restrict__ da, float *__restrict__ db) {
  const int i = blockIdx.y;
  const int2 s = spans[i];
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= na + nb) return;
  float v = 0.0f;
  for (int j = 0; j < s.y; ++j) v += parts[(s.x + j) * (na + nb) + e];
  if (e < na) {
    if (da) da[i * na + e] = v;
  } else if (db) {
    db[i * nb + e - na] = v;
  }
}

static bool float_type(int t) { return t == KSD_F32 || t == KSD_BF16 || t == KSD_F16; }
static int64_t size_of(int t) { return t == KSD_F32 ? 4 : 2; }

struct Layout {
  int64_t order, slots, spans, at, bt, gh, parts, bytes;
};
static Layout layout(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int dtype) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t b) {
    const int64_t v = at;
    at += (b + 255) / 256 * 256;
    return v;
  };
  l.order = take(M * 4);
  l.slots = take((M / kPiece + n) * (int64_t)sizeof(Slot));
  l.spans = take(n * 8);
  l.at = take(n * r * K * size_of(dtype));
  l.bt = take(n * r * N * size_of(dtype));
  l.gh = take(M * r * 4);
  l.parts = take((M / kPiece + n) * r * (K + N) * 4);
  l.bytes = at;
  return l;
}

// Sizes for which every index fits its type.
static bool fits(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n) {
  return M >= 0 && K >= 1 && N >= 1 && r >= 1 && r <= 128 && n >= 1 && n <= 65535 && M <= 0x7fffffff - 65536 &&
         K <= 0x7fffffff - 65536 && N <= 0x7fffffff - 65536;
}

static int run_pair(const PairArgs &args, int dtype, bool mask, hipStream_t st) {
  PairArgs p = args;
  shape(p);
  if (!grid_fits(cdiv(p.M, p.rows), 64 * kWaves) || cdiv(p.N, p.cols) > 65535)
    return fail(KSD_EINVAL, "adapter_linear: too many rows or columns");
  if (dtype == KSD_F32) launch_pair<KSD_F32>(p, mask, st);
  else if (dtype == KSD_BF16) launch_pair<KSD_BF16>(p, mask, st);
  else launch_pair<KSD_F16>(p, mask, st);
  return check_launch("adapter_linear");
}

template <typename T>
static void turn(const void *in, void *out, int64_t n, int64_t rows, int64_t cols, hipStream_t st) {
  turn_kernel<T><<<(unsigned)(n * cdiv(rows, 32) * cdiv(cols, 32)), 256, 0, st>>>((const T *)in, (T *)out, rows, cols);
}

}  // namespace adp
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_adapter_linear(const void *x, int dtype, int64_t M, int64_t K, int64_t x_stride, const void *a, const void *b,
                                  int64_t n, int64_t r, int64_t N, const void *index, int index_wide, int64_t rows_per_index,
                                  const float *scales, const void *base, int64_t base_stride, int64_t drop, uint64_t seed,
                                  const void *seed_from, int64_t stream_id, void *y, float *hidden, void *stream) {
  if (!adp::fits(M, K, N, r, n) || rows_per_index < 1 || (M > 1 && (x_stride < K || (base && base_stride < N))))
    return fail(KSD_EINVAL, "adapter_linear: bad shape");
  if (!adp::float_type(dtype)) return fail(KSD_ETYPE, "adapter_linear: unsupported element type");
  Mask m;
  if (!make_mask(m, drop, seed, seed_from, stream_id)) return fail(KSD_EINVAL, "adapter_linear: bad probability, seed or stream");
  if (M == 0) return KSD_OK;
  if (!x || !a || !b || !index || !y) return fail(KSD_EINVAL, "adapter_linear: null pointer");
  adp::PairArgs p{x, x_stride, M, K, N, a, b, index, index_wide, rows_per_index, scales, base, base_stride, y, hidden,
                  (int)n, (int)r, 0, 0, m, 1, 0};
  return adp::run_pair(p, dtype, drop > 0, (hipStream_t)stream);
}

extern "C" int ksd_adapter_linear_backward_workspace(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int dtype,
                                                     int64_t *bytes) {
  if (!bytes || !adp::fits(M, K, N, r, n) || !adp::float_type(dtype))
    return fail(KSD_EINVAL, "adapter_linear_backward_workspace: bad arguments");
  *bytes = adp::layout(M, K, N, r, n, dtype).bytes;
  return KSD_OK;
}

extern "C" int ksd_adapter_linear_backward(const void *g, int dtype, int64_t M, int64_t N, int64_t g_stride, const void *x,
                                           int64_t K, int64_t x_stride, const float *hidden, const void *a, const void *b,
                                           int64_t n, int64_t r, const void *index, int index_wide, int64_t rows_per_index,
                                           const float *scales, const void *base, int64_t base_stride, int64_t drop,
                                           uint64_t seed, const void *seed_from, int64_t stream_id, void *dx, float *da,
                                           float *db, void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace adp;
  if (!fits(M, K, N, r, n) || rows_per_index < 1 ||
      (M > 1 && (x_stride < K || g_stride < N || (base && base_stride < K))))
    return fail(KSD_EINVAL, "adapter_linear_backward: bad shape");
  if (!float_type(dtype)) return fail(KSD_ETYPE, "adapter_linear_backward: unsupported element type");
  Mask m;
  if (!make_mask(m, drop, seed, seed_from, stream_id))
    return fail(KSD_EINVAL, "adapter_linear_backward: bad probability, seed or stream");
  if (M > 0 && (!g || !x || !hidden || !a || !b || !index)) return fail(KSD_EINVAL, "adapter_linear_backward: null pointer");
  const Layout l = layout(M, K, N, r, n, dtype);
  if (!workspace || workspace_bytes < l.bytes || (uintptr_t)workspace % 16)
    return fail(KSD_EINVAL, "adapter_linear_backward: short or misaligned workspace");
  const int64_t slots = M / kPiece + n, blocks_a = cdiv(K, 128), blocks_b = cdiv(N, 128), each = r * (K + N);
  if (slots > 65535 || !grid_fits(blocks_a + blocks_b, 256) || !grid_fits(cdiv(each, 256), 256) ||
      !grid_fits(n * cdiv(r, 32) * std::max(cdiv(K, 32), cdiv(N, 32)), 256))
    return fail(KSD_EINVAL, "adapter_linear_backward: too many tokens, columns or adapters");
  hipStream_t st = (hipStream_t)stream;
  char *const w = (char *)workspace;
  // the narrow product contracts dY's columns, the wide one the ranks: both banks the other way round
  if (dtype == KSD_F32) {
    turn<uint32_t>(a, w + l.at, n, r, K, st);
    turn<uint32_t>(b, w + l.bt, n, N, r, st);
  } else {
    turn<uint16_t>(a, w + l.at, n, r, K, st);
    turn<uint16_t>(b, w + l.bt, n, N, r, st);
  }
  float *const gh = (float *)(w + l.gh);
  if (M > 0) {
    PairArgs p{g, g_stride, M, N, K, w + l.bt, w + l.at, index, index_wide, rows_per_index, scales, base, base_stride, dx, gh,
               (int)n, (int)r, 0, 0, m, 0, 1};
    const int rc = run_pair(p, dtype, drop > 0, st);
    if (rc) return rc;
  }
  if (!da && !db) return KSD_OK;
  GroupArgs ga{index, index_wide, (int)n, rows_per_index, M, (int32_t *)(w + l.order), (Slot *)(w + l.slots), (int2 *)(w + l.spans)};
  group_kernel<<<(unsigned)n, 256, 0, st>>>(ga);
  float *const parts = (float *)(w + l.parts);
  if (M > 0) {
    GradArgs q{x, g, x_stride, g_stride, K, N, gh, hidden, ga.order, ga.slots, parts, (int)r, (int)blocks_a, drop > 0, m};
    const dim3 grid((unsigned)(blocks_a + blocks_b), (unsigned)slots, (unsigned)cdiv(r, 64));
    if (dtype == KSD_F32) grad_kernel<KSD_F32><<<grid, 256, 0, st>>>(q);
    else if (dtype == KSD_BF16) grad_kernel<KSD_BF16><<<grid, 256, 0, st>>>(q);
    else grad_kernel<KSD_F16><<<grid, 256, 0, st>>>(q);
  }
  join_kernel<<<dim3((unsigned)cdiv(each, 256), (unsigned)n), 256, 0, st>>>(parts, ga.spans, r * K, r * N, da, db);
  return check_launch("adapter_linear_backward");
}
