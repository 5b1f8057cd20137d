// Low-rank adapters of many requests beside a shared projection, forward and backward.
//
//   h[m] = s_i x~[m] A_i^T,   y[m] = base[m] + h[m] B_i^T           i = index[m]
//   g[m] = s_i dY[m] B_i,     dX[m] = dXbase[m] + mask(g[m] A_i)
//   dA_i = sum of g[m]^T x~[m],   dB_i = sum of dY[m]^T h[m]         over the tokens m of adapter i
//
// with x~ = dropout(x) where a mask is given (made from its counter, stored nowhere). A token without an adapter
// keeps base. Adapters of other tokens never touch a token's row, whatever they hold.
//
// Both passes of a token's row are one launch of pair_kernel: a workgroup of 8 waves holds up to 32 rows; the waves
// split the contraction of the narrow product, their sums join in LDS, and the same waves then split the columns of
// the wide one. h keeps its 24 bits on its way: it is fp32 in LDS and enters the 16-bit matrix instructions as a
// rounded value and the rounding's rest, side by side along the contraction, which a rank of 16 leaves half empty
// anyway (fp16: 11 bits each), and bf16, of 8 bits a part, as the rest's rest in another instruction. What bounds it
// is memory: x and base read once, y written once. 8192 tokens of 1536 to 1536, rank 16: bf16 20 us for 76 MB (3.8
// TB/s), fp32 43 us for 151 MB (3.5; the narrow product alone 17, the wide one 24). Few tokens take a launch's
// latency: one token 5.4 us, 64 of as many adapters 6.7.
#include "ksd_random.h"

#include <algorithm>
#include <atomic>

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

// Tokens are listed by adapter (stable; those without one last, as adapter n), each list in pieces. Piece j of adapter
// i is slot start_i / piece + i + j: slots of different adapters never meet, and a slot knows its adapter without a sum
// over the earlier ones' pieces.
constexpr int kTile = 32, kLeast = 64;  // of the products by rows; the smallest of the gradients' sums

struct Slot {
  int adapter, from, to, pad;  // -1: empty
};

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
  int odd_x, odd_y;        // 16-bit rows of x or a, of base or y, may begin on an odd half word
  const int32_t *order;    // tokens listed by adapter, and the pieces of the lists (NULL: rows as they lie)
  const Slot *slots;
  int tiles;               // workgroups of a piece
  int splits;              // > 0: the narrow product's columns in so many parts, in a launch of its own
  int phase;               // 0: both products; 1: the narrow one's part blockIdx.y into sums; 2: the wide one from sums
  float *sums;             // (splits, M, r)
};

__device__ __forceinline__ int adapter_of(const void *index, int wide, int64_t per, int64_t m, int n) {
  const int64_t at = per == 1 ? m : (uint32_t)m / (uint32_t)per;
  const int64_t i = wide ? ((const int64_t *)index)[at] : (int64_t)((const int32_t *)index)[at];
  return i >= 0 && i < n ? (int)i : -1;
}

// 8 elements from c on that lie inside a row.
template <int DT>
__device__ __forceinline__ typename Oct<DT>::V whole_oct(const typename Elem<DT>::T *row, int64_t c) {
  struct __attribute__((packed, aligned(sizeof(typename Elem<DT>::T)))) Any { typename Oct<DT>::V v; };
  return ((const Any *)(row + c))->v;
}

// 8 values of 16 bits of a row that may begin on an odd half word: 16 bytes from the word that holds the first one, and
// the word behind them, moved together once they are used. (A 16-byte load on an odd half word takes several times
// as long: 2047 rows of 6869 columns 31.8 us in such loads and stores, of 6870 21.5.)
template <int DT> struct Held {
  typename Oct<DT>::V v;
  uint32_t e;
};
template <int DT, bool ODD>
__device__ __forceinline__ void hold(Held<DT> &h, const typename Elem<DT>::T *row, int64_t c) {
  if constexpr (ODD && DT != KSD_F32) {
    const uintptr_t at = (uintptr_t)(row + c), word = at & ~(uintptr_t)3;
    struct __attribute__((packed, aligned(4))) Word { typename Oct<DT>::V v; };
    h.v = ((const Word *)word)->v;
    h.e = *(const uint32_t *)(word + (at & 2 ? 16 : 12));
  } else {
    h.v = whole_oct<DT>(row, c);
  }
}
template <int DT, bool ODD>
__device__ __forceinline__ typename Oct<DT>::V held(const Held<DT> &h, const typename Elem<DT>::T *row, int64_t c) {
  if constexpr (ODD && DT != KSD_F32) {
    const uint32_t by = ((uintptr_t)(row + c) & 2) * 8;
    const u32x4 w = __builtin_bit_cast(u32x4, h.v);
    return __builtin_bit_cast(typename Oct<DT>::V, u32x4{__builtin_amdgcn_alignbit(w.y, w.x, by), __builtin_amdgcn_alignbit(w.z, w.y, by),
                                                         __builtin_amdgcn_alignbit(w.w, w.z, by), __builtin_amdgcn_alignbit(h.e, w.w, by)});
  } else {
    return h.v;
  }
}
template <int DT>
__device__ __forceinline__ void put_oct(typename Elem<DT>::T *row, int64_t c, const typename Oct<DT>::V &v, bool odd) {
  struct __attribute__((packed, aligned(sizeof(typename Elem<DT>::T)))) Any { typename Oct<DT>::V v; };
  if constexpr (DT != KSD_F32) {
    if (odd && ((uintptr_t)(row + c) & 2)) {
      typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
      struct __attribute__((packed, aligned(4))) Three { u32x3 v; };
      const u32x4 w = __builtin_bit_cast(u32x4, v);
      row[c] = (uint16_t)w.x;
      ((Three *)(row + c + 1))->v = u32x3{__builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16),
                                          __builtin_amdgcn_alignbit(w.w, w.z, 16)};
      row[c + 7] = (uint16_t)(w.w >> 16);
      return;
    }
  }
  ((Any *)(row + c))->v = v;
}

// The dropped ones of 8 values become 0; the kept ones stay as they are (fp32: are scaled). 16-bit values would be
// rounded by the scale, which their sums take instead.
template <int DT>
__device__ __forceinline__ void drop_oct(const Mask &m, uint4 bits, typename Oct<DT>::V &v) {
  const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
    if constexpr (DT == KSD_F32) v[j] = u >= m.drop ? v[j] * m.scale : 0.0f;
    else v[j] = u >= m.drop ? v[j] : (short)0;
  }
}

// U steps of 32 columns of the narrow product. Rows of other adapters and ranks from r on are read from a
// row that exists: their results are not used. `whole`: no step passes the row's end.
template <int DT, int R16, int RT, int U, bool MASK, bool ODD>
__device__ __forceinline__ void narrow(const PairArgs &p, const typename Elem<DT>::T *const (&xr)[RT],
                                       const typename Elem<DT>::T *const (&ar)[R16], int64_t s, bool whole, MaskKey key,
                                       const int64_t (&row)[RT], int grp, f32x4 (&acc)[RT][R16]) {
  using V = typename Oct<DT>::V;
  V xv[U][RT], av[U][R16];
  if (whole) {
    Held<DT> xh[U][RT], ah[U][R16];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (s + u) * 32 + grp * 8;
#pragma unroll
      for (int t = 0; t < RT; ++t) hold<DT, ODD>(xh[u][t], xr[t], k);
#pragma unroll
      for (int q = 0; q < R16; ++q) hold<DT, ODD>(ah[u][q], ar[q], k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (s + u) * 32 + grp * 8;
#pragma unroll
      for (int t = 0; t < RT; ++t) xv[u][t] = held<DT, ODD>(xh[u][t], xr[t], k);
#pragma unroll
      for (int q = 0; q < R16; ++q) av[u][q] = held<DT, ODD>(ah[u][q], ar[q], k);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = (s + u) * 32 + grp * 8;
#pragma unroll
      for (int t = 0; t < RT; ++t) xv[u][t] = load_oct<DT>(xr[t], k, p.K);
#pragma unroll
      for (int q = 0; q < R16; ++q) av[u][q] = load_oct<DT>(ar[q], k, p.K);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if constexpr (MASK) {
      if (p.mask_x) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
          drop_oct<DT>(p.mask, mask_bits(p.mask, key, row[t], (uint32_t)((s + u) * 4 + grp)), xv[u][t]);
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int q = 0; q < R16; ++q) acc[t][q] = product<DT>(av[u][q], xv[u][t], acc[t][q]);
  }
}

// What a lane takes of a bank row of r ranks in a block of 16: fp32 ranks 4 grp .. + 3, 16-bit types ranks 8 (grp % 2) ..
// + 7; zeros from r on. ALIGNED: r is a multiple of that, else value by value (r = 23: 8 loads for one).
template <int DT, bool ALIGNED>
__device__ __forceinline__ typename Oct<DT>::V bank_oct(const typename Elem<DT>::T *row, int q, int grp, int r) {
  using V = typename Oct<DT>::V;
  constexpr int W = DT == KSD_F32 ? 4 : 8;
  const int c = q * 16 + (DT == KSD_F32 ? grp : grp & 1) * W;
  V w{};
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const auto e = row[min(c + j, r - 1)];
      w[j] = c + j < r ? e : 0;
    }
  } else if constexpr (DT == KSD_F32) {
    struct __attribute__((packed, aligned(4))) Any { f32x4 v; };
    const f32x4 v = ((const Any *)(row + (c < r ? c : 0)))->v;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = c < r ? v[j] : 0.0f;
  } else {
    w = whole_oct<DT>(row, c < r ? c : 0);
    w = c < r ? w : V{};
  }
  return w;
}

// R16: blocks of 16 ranks; RT: blocks of 16 rows. KIND: kPlain; kOdd: 16-bit rows may begin on an odd half word; kAnyRank:
// that, and a rank that is no multiple of a lane's. Each in registers of its own: with odd rows' code 8192 plain rows of 1536
// take 21.6 us for 19.3.
constexpr int kPlain = 0, kOdd = 1, kAnyRank = 2;
// Masked 16-bit rows of rank up to 16 are held to the registers of two workgroups a CU (4000 tokens of 1536 with dropout: 24.2
// us, in the registers of one 29.1). Unmasked ones whose rank is a lane's multiple are that small by themselves (up to 128); the
// other forms run one.
template <int DT, int R16, int RT, bool MASK>
constexpr bool kTwo = MASK && DT != KSD_F32 && RT == 1 && R16 == 1;
// Forms of rank up to 16 that stay within two workgroups' registers only if the bank's rows are loaded where they are used, 32
// columns at a time (fp16, rank 7, 4000 tokens of 1536, a training call with dropout: 72.7 us, with rows ahead 80.9; bf16, rank
// 16: 57 us and 59.5, in the spills that h's third part then makes).
template <int DT, int R16, int RT, bool MASK, int KIND>
constexpr bool kLean = kTwo<DT, R16, RT, MASK> || (DT == KSD_BF16 && RT == 1 && R16 == 1 && KIND == kOdd);
// bf16 values of a row of h's third parts: 16 ranks, 16 zeros for the upper two groups, and so on; 16 bytes more spread rows
// over the banks. (Two blocks' parts side by side in one instruction need the bank's rows side by side too: 8192 tokens of
// 1536 to 1536, rank 64, 47 us for 34.)
template <int R16>
constexpr int kThirdPitch = 32 * R16 + 8;
template <int DT, int R16, int RT, bool MASK, int KIND>
__global__ __launch_bounds__(64 * kWaves, (kTwo<DT, R16, RT, MASK> ? 4 : 2)) void pair_kernel(const PairArgs p) {
  using T = typename Elem<DT>::T;
  using V = typename Oct<DT>::V;
  constexpr int R = 16 * R16, U = DT == KSD_F32 ? (R16 <= 1 ? 4 : R16 <= 2 ? 2 : 1) : (kTwo<DT, R16, RT, MASK> ? 3 : R16 <= 1 ? 6 : R16 <= 2 ? 4 : 2);
  constexpr int TB = kLean<DT, R16, RT, MASK, KIND> ? 2 : R16 <= 2 ? 4 : R16 == 4 ? 2 : 1;  // products whose bank rows are loaded together
  constexpr bool kMayBeOdd = DT != KSD_F32 && KIND != kPlain;
  constexpr bool kAhead = R16 == 1 && !kLean<DT, R16, RT, MASK, KIND>;  // the next bank rows are loaded during a block's products: more ranks, no registers for it
  constexpr int pitch = R + 4;  // floats: a row's four lanes of 16 bytes start 4 banks further than the last row's
  constexpr bool kThird = DT == KSD_BF16;
  extern __shared__ float lds[];  // (kWaves, 16 RT, pitch): sums of a wave's columns; the first holds h
  int16_t *const thirds = (int16_t *)(lds + kWaves * 16 * RT * pitch);  // (16 RT, kThirdPitch)
  const auto put_third = [&](int t, int q, float v) {
    float f[8] = {v}, g[8];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      to_floats<DT>(from_floats<DT>(f), g);
      f[0] = fabsf(g[0]) <= 3.0e38f ? f[0] - g[0] : 0.0f;
    }
    int16_t *const to = thirds + t * kThirdPitch<R16> + (q >> 4) * 32 + (q & 15);
    to[0] = from_floats<DT>(f)[0];
    to[16] = 0;  // the upper two groups' ranks
  };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  // lane l < rows: its token and the token's adapter
  int rows, mine = -1, token = 0;
  if (p.slots) {
    const Slot s = p.slots[blockIdx.x / p.tiles];
    const int from = s.from + (int)(blockIdx.x % p.tiles) * p.rows;
    rows = s.adapter < 0 ? 0 : min(p.rows, s.to - from);
    if (rows <= 0) return;
    if (lane < rows) token = p.order[from + lane], mine = s.adapter < p.n ? s.adapter : -1;
  } else {
    const int64_t row0 = (int64_t)blockIdx.x * p.rows;
    rows = (int)min((int64_t)p.rows, p.M - row0);
    if (lane < rows) token = (int)row0 + lane, mine = adapter_of(p.index, p.wide, p.per, token, p.n);
  }
  int of[RT];  // of the rows that this lane's columns of the products are
  int64_t at_row[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    of[t] = __shfl(mine, t * 16 + col);
    at_row[t] = __shfl(token, t * 16 + col < rows ? t * 16 + col : 0);
  }
  const uint64_t with = __ballot(mine >= 0);
  MaskKey key{};
  if constexpr (MASK) key = mask_key(p.mask);

  const int64_t n0 = (int64_t)blockIdx.y * p.cols, n1 = min(p.N, n0 + p.cols);
  // base of a block of 64 columns: 16 of them per lane
  const auto load_base = [&](int64_t c, Held<DT> (&v)[RT][2]) {
    const bool whole = c + 64 <= p.N;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const T *const row = (const T *)p.base + at_row[t] * p.base_stride;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t at = c + e * 32 + grp * 8;
        if (!whole) v[t][e].v = load_oct<DT>(row, at, p.N);
        else if (kMayBeOdd && p.odd_y) hold<DT, true>(v[t][e], row, at);
        else hold<DT, false>(v[t][e], row, at);
      }
    }
  };
  Held<DT> bv[RT][2] = {};
  int64_t c = n0 + wave * 64;
  const bool wide = p.y && p.phase != 1, based = p.base && wide;
  if (based && c < n1) load_base(c, bv);
  // An adapter's bank rows for tiles t0 .. of a block. Which of its columns row i of product t is: such that a lane ends
  // with two runs of 8 columns of its token, and four lanes' runs lie side by side.
  const auto load_bank = [&](int64_t c, int i, int t0, V (&w)[TB][R16]) {
    const T *const b = (const T *)p.b + (int64_t)i * p.N * p.r;
    const bool whole = c + 64 <= p.N;
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      const int64_t n = c + (t0 + t) / 2 * 32 + (col >> 2) * 8 + (t0 + t) % 2 * 4 + (col & 3);
#pragma unroll
      for (int q = 0; q < R16; ++q) w[t][q] = bank_oct<DT, KIND != kAnyRank>(b + (whole ? n : min(n, p.N - 1)) * p.r, q, grp, p.r);
    }
  };
  const auto lowest = [&](uint64_t rows) { return __shfl(mine, __builtin_ctzll(rows)); };
  V w[TB][R16] = {};
  if (kAhead && with && wide && c < n1) load_bank(c, lowest(with), 0, w);

  if (with && p.phase == 2) {
    __shared__ int tokens[16 * RT];
    if (wave == 0 && lane < 16 * RT) tokens[lane] = token;
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * RT * R; e += 64 * kWaves) {
      const int t = e / R, q = e % R;
      float v = 0.0f;
      if (t < rows && (with >> t & 1) && q < p.r) {
        const float *const from = p.sums + (int64_t)tokens[t] * p.r + q;
        for (int k = 0; k < p.splits; ++k) v += from[k * p.M * p.r];
      }
      lds[t * pitch + q] = v;
      if constexpr (kThird) put_third(t, q, v);
    }
    __syncthreads();
  } else if (with) {
    // ---- h: D[rank][token] = A x^T over this wave's columns
    const T *xr[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) xr[t] = (const T *)p.x + at_row[t] * p.x_stride;
    const int64_t steps = (p.K + 31) / 32, full = p.K / 32;
    const int waves = p.phase ? kWaves * p.splits : kWaves, mark = p.phase ? blockIdx.y * kWaves + wave : wave;
    const int64_t share = (steps + waves - 1) / waves;
    const int64_t from = mark * share, to = min(steps, from + share), upto = min(to, full);
    for (uint64_t left = with; left;) {
      const int i = __shfl(mine, __builtin_ctzll(left));
      left &= ~__ballot(mine == i);
      const T *const a = (const T *)p.a + (int64_t)i * p.r * p.K;
      const T *ar[R16];
#pragma unroll
      for (int q = 0; q < R16; ++q) ar[q] = a + (int64_t)min(q * 16 + col, p.r - 1) * p.K;
      f32x4 acc[RT][R16] = {};
      int64_t s = from;
      if (kMayBeOdd && p.odd_x) {
        constexpr int O = R16 == 2 ? 3 : (U + 1) / 2;  // a step's loads take one more register per operand
        for (; s + O <= upto; s += O) narrow<DT, R16, RT, O, MASK, true>(p, xr, ar, s, true, key, at_row, grp, acc);
      } else {
        for (; s + U <= upto; s += U) narrow<DT, R16, RT, U, MASK, false>(p, xr, ar, s, true, key, at_row, grp, acc);
        if constexpr (U > 2) {
          for (; s + 2 <= upto; s += 2) narrow<DT, R16, RT, 2, MASK, false>(p, xr, ar, s, true, key, at_row, grp, acc);
        }
      }
      for (; s < to; ++s) narrow<DT, R16, RT, 1, MASK, false>(p, xr, ar, s, s < full, key, at_row, grp, acc);
      float scale = p.scales ? p.scales[i] : 1.0f;
      if constexpr (MASK && DT != KSD_F32) scale *= p.mask_x ? p.mask.scale : 1.0f;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (of[t] == i) {
          float *const o = lds + ((int64_t)wave * 16 * RT + t * 16 + col) * pitch + grp * 4;
#pragma unroll
          for (int q = 0; q < R16; ++q) *(f32x4 *)(o + q * 16) = acc[t][q] * scale;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * RT * R; e += 64 * kWaves) {
      const int t = e / R, q = e % R;
      if (t < rows && (with >> t & 1)) {
        float v = lds[t * pitch + q];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += lds[(w * 16 * RT + t) * pitch + q];
        v = q < p.r ? v : 0.0f;
        lds[t * pitch + q] = v;
        if constexpr (kThird) put_third(t, q, v);
      }
    }
    __syncthreads();
  }
  if (p.phase == 1) {
    for (int t = wave; t < rows; t += kWaves) {
      float *const to = p.sums + ((int64_t)blockIdx.y * p.M + __shfl(token, t)) * p.r;
      if (with >> t & 1)
        for (int q = lane; q < p.r; q += 64) to[q] = lds[t * pitch + q];
    }
    return;
  }
  if (p.hidden && blockIdx.y == 0) {
    for (int t = wave; t < rows; t += kWaves) {
      const int64_t m = __shfl(token, t);
      for (int q = lane; q < p.r; q += 64) p.hidden[m * p.r + q] = with >> t & 1 ? lds[t * pitch + q] : 0.0f;
    }
  }
  if (!wide) return;

  // ---- y: D[column][token] = B h^T
  V hv[RT][R16];
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
          hv[t][q] = V{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
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
  for (; c < n1; c += 64 * kWaves) {
    const bool whole = c + 64 <= p.N;
    Held<DT> next[RT][2] = {};
    if (based && c + 64 * kWaves < n1) load_base(c + 64 * kWaves, next);
    f32x4 acc[RT][4] = {};
    for (uint64_t left = with; left;) {
      const int i = lowest(left);
      left &= ~__ballot(mine == i);
      f32x4 d[RT][4] = {};
#pragma unroll
      for (int t0 = 0; t0 < 4; t0 += TB) {
        V ahead[TB][R16] = {};
        if constexpr (kAhead) {  // the next adapter's or the next block's rows are on the way during these products
          const int64_t then = left ? c : c + 64 * kWaves;
          if (then < n1) load_bank(then, lowest(left ? left : with), 0, ahead);
        } else {
          load_bank(c, i, t0, w);
        }
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
          for (int q = 0; q < R16; ++q)
#pragma unroll
            for (int u = 0; u < RT; ++u) {
              f32x4 &o = d[u][t0 + t];
              if constexpr (DT == KSD_F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o = __builtin_amdgcn_mfma_f32_16x16x4f32(w[t][q][j], hv[u][q][j], o, 0, 0, 0);
              } else {
                o = product<DT>(w[t][q], hv[u][q], o);
                if constexpr (kThird) {
                  o = product<DT>(w[t][q], *(const V *)(thirds + (u * 16 + col) * kThirdPitch<R16> + q * 32 + grp * 8), o);
                }
              }
            }
        if constexpr (kAhead) {
#pragma unroll
          for (int t = 0; t < TB; ++t)
#pragma unroll
            for (int q = 0; q < R16; ++q) w[t][q] = ahead[t][q];
        }
      }
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[u][t] = of[u] == i ? d[u][t] * back[u] : acc[u][t];
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const int64_t m = at_row[u];
      T *const out = (T *)p.y + m * p.N;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int64_t at = c + v * 32 + grp * 8;
        float f[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = acc[u][v * 2 + j / 4][j & 3];
        if constexpr (MASK) {
          if (p.mask_y) apply_mask(p.mask, mask_bits(p.mask, key, m, (uint32_t)(at >> 3)), f);
        }
        if (based) {
          const T *const row = (const T *)p.base + at_row[u] * p.base_stride;
          to_floats<DT>(kMayBeOdd && p.odd_y && whole ? held<DT, true>(bv[u][v], row, at) : bv[u][v].v, g);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = of[u] >= 0 ? f[j] + g[j] : g[j];
        }
        if (u * 16 + col < rows) {
          if (whole) put_oct<DT>(out, at, from_floats<DT>(f), kMayBeOdd && p.odd_y);
          else store_oct<DT>(out, at, p.N, f);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) bv[t][0] = next[t][0], bv[t][1] = next[t][1];
  }
}

// Bytes of LDS: the waves' sums, and bf16's third parts of h.
template <int DT, int R16, int RT>
constexpr int kLds = kWaves * 16 * RT * (16 * R16 + 4) * 4 + (DT == KSD_BF16 ? 16 * RT * kThirdPitch<R16> * 2 : 0);

static bool aligned_rank(int64_t r, int dtype) { return r % (dtype == KSD_F32 ? 4 : 8) == 0; }

template <int DT, int R16, int RT, bool MASK, int KIND>
static void launch_pair(const PairArgs &p, unsigned tiles, hipStream_t st) {
  const dim3 g(tiles, (unsigned)(p.phase == 1 ? p.splits : cdiv(p.N, p.cols)));
  constexpr int lds = kLds<DT, R16, RT>;
  if constexpr (lds > 65536) {  // past HIP's default, once on each device
    static std::atomic<uint64_t> known{0};
    int dev = 0;
    (void)hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (!(known.load(std::memory_order_relaxed) & bit)) {
      (void)hipFuncSetAttribute((const void *)pair_kernel<DT, R16, RT, MASK, KIND>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      known.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  pair_kernel<DT, R16, RT, MASK, KIND><<<g, 64 * kWaves, lds, st>>>(p);
}
template <int DT, int R16, int RT>
static void launch_pair(const PairArgs &p, bool mask, unsigned tiles, hipStream_t st) {
  if constexpr (RT == 1) {
    if (!aligned_rank(p.r, DT)) {
      if (mask) launch_pair<DT, R16, RT, true, kAnyRank>(p, tiles, st);
      else launch_pair<DT, R16, RT, false, kAnyRank>(p, tiles, st);
      return;
    }
    if constexpr (DT != KSD_F32) {
      if (p.odd_x || p.odd_y) {
        if (mask) launch_pair<DT, R16, RT, true, kOdd>(p, tiles, st);
        else launch_pair<DT, R16, RT, false, kOdd>(p, tiles, st);
        return;
      }
    }
  }
  if (mask) launch_pair<DT, R16, RT, true, kPlain>(p, tiles, st);
  else launch_pair<DT, R16, RT, false, kPlain>(p, tiles, st);
}
template <int DT>
static void launch_pair(const PairArgs &p, bool mask, unsigned tiles, hipStream_t st) {
  const bool one = p.rows <= 16;
  if (p.r <= 16) one ? launch_pair<DT, 1, 1>(p, mask, tiles, st) : launch_pair<DT, 1, 2>(p, mask, tiles, st);
  else if (p.r <= 32) one ? launch_pair<DT, 2, 1>(p, mask, tiles, st) : launch_pair<DT, 2, 2>(p, mask, tiles, st);
  else if (p.r <= 64) one ? launch_pair<DT, 4, 1>(p, mask, tiles, st) : launch_pair<DT, 4, 2>(p, mask, tiles, st);
  else launch_pair<DT, 8, 1>(p, mask, tiles, st);
}

// Rows and columns of a workgroup. Rows that may have several adapters and do not go by lists: one at a time (64 tokens of
// as many adapters, 1536 x 1536, rank 16: 8.8 us, two 10.4). Else up to 16, whose products fill the instructions
// (1021 tokens, 1536 x 1536: 9.9 us with 16 rows and 11.0 with 4; 256 tokens: 9.4 and 8.7), and 32 where 256
// workgroups are left (8192 tokens: 18.6 us, with 16 rows 19.2; rank 64: 33 and 45). Columns are shared out where
// fewer workgroups than CUs would run, each part forming h again: not where that is the longer product (2047 tokens,
// 6869 to 1792: 43 us, in two parts 69; 1792 to 6869: 54 us, in 4 parts 47).
// Every workgroup reads its adapter's banks: ranks past 16 take more rows (400 tokens, 1536 to 4096, fp32, rank 64: 24.6 us,
// in fewer rows 40.5), and large banks 32 rows from 4096 tokens on (6110 tokens, 5974 to 6862, rank 32: 122 us and 168;
// 6000 tokens, 4096 to 4096, rank 16: 57.5 and 48.5).
static void shape(PairArgs &p, bool lists, bool plain) {
  const int64_t few = p.M * cdiv(p.r, 16);
  const bool tall = p.M >= 8192 || (p.M >= 4096 && p.r * (p.K + p.N) >= 1 << 18);
  if (!lists && p.n > 1 && p.per < 16) p.rows = (int)std::max<int64_t>(1, std::min<int64_t>(16, cdiv(p.M, 1024)));
  else p.rows = few <= 64 ? 1 : few <= 256 ? 4 : few <= 512 ? 8 : tall && p.r <= 64 && plain ? 32 : 16;
  if (lists)
    while (kTile % p.rows) --p.rows;
  const int64_t tiles = std::max<int64_t>(1, cdiv(p.M, p.rows)), blocks = cdiv(p.N, 64);
  // (the workspace is sized by the splits of a plain call, which are those of others or more)
  // a long narrow product of few rows goes to several workgroups first (2047 tokens, 6869 to 1792: 44 us, so 34; one
  // token 24 and 13), whose sums the wide product's add
  p.splits = p.K >= 4096 && tiles < 256 ? 4 : 0;
  // more parts where a row is long (a train call with dropout of 2047 tokens of 1792 to 6869: 88.8 us with 256 workgroups,
  // 86.6 with 512, which are resident together there: rank 8 in 16 bits, two a CU; measured in that form alone). The tiles that
  // lists add at each adapter's end are not counted.
  const int64_t want = blocks < 64 ? 256 : 512;
  const int64_t parts = std::min({blocks / 6, cdiv(want, tiles), p.splits ? blocks : 4 * p.N / p.K});
  p.cols = (int)(cdiv(blocks, std::max<int64_t>(1, parts)) * 64);
}

// ------------------------------------------------------------------------------- lists by adapter
struct GroupArgs {
  const void *index;
  int wide, n;
  int64_t per, M;
  int32_t *order;        // (M,)
  Slot *tiles, *pieces;  // (M / kTile + n + 1,), (M / piece + n + 1,)
  int2 *spans;           // (n + 1,): an adapter's first of `pieces`, and how many
  int piece;             // tokens of one of `pieces`
};

// Workgroup i lists adapter i's tokens, workgroup n those without one: 8192 tokens at a time, whose indices are
// loaded together. Each counts all indices instead of waiting for another one's sum. (1021 tokens of 5 adapters 5.8 us, 8192
// of one 8.3 with the turned banks: two passes of latency.)
__device__ __forceinline__ void list_tokens(const GroupArgs &a, int i) {
  constexpr int U = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ int sums[2][16], counts[2][U][16];
  int v[U];
  const auto load = [&](int64_t base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t m = base + u * 1024 + tid;
      v[u] = a.n + 1;  // in no list
      if (m < a.M) {
        v[u] = adapter_of(a.index, a.wide, a.per, m, a.n);
        v[u] = v[u] < 0 ? a.n : v[u];
      }
    }
  };
  int less = 0, mine = 0;
  for (int64_t base = 0; base < a.M; base += U * 1024) {
    load(base);
#pragma unroll
    for (int u = 0; u < U; ++u) less += v[u] < i, mine += v[u] == i;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) less += __shfl_xor(less, o), mine += __shfl_xor(mine, o);
  if (lane == 0) sums[0][wave] = less, sums[1][wave] = mine;
  __syncthreads();
  int start = 0, len = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) start += sums[0][w], len += sums[1][w];
  const auto cut = [&](Slot *slots, int piece) {
    // every slot is written: all tokens are in one of the n + 1 lists, so the last one ends at M / piece + n + 1
    const int slot = start / piece + i, next = (start + len) / piece + i + 1, pieces = (len + piece - 1) / piece;
    for (int s = slot + tid; s < next; s += 1024) {
      const int at = start + (s - slot) * piece;
      slots[s] = s - slot < pieces ? Slot{i, at, min(at + piece, start + len), 0} : Slot{-1, 0, 0, 0};
    }
    return make_int2(slot, pieces);
  };
  cut(a.tiles, kTile);
  const int2 span = cut(a.pieces, a.piece);
  if (tid == 0) a.spans[i] = span;
  int done = start, turn = 0;
  for (int64_t base = 0; base < a.M && done < start + len; base += U * 1024, turn ^= 1) {
    if (a.M > U * 1024) load(base);
    uint64_t b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      b[u] = __ballot(v[u] == i);
      if (lane == 0) counts[turn][u][wave] = __popcll(b[u]);
    }
    __syncthreads();  // the other half of counts is read until the next round's
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * 1024 >= a.M) break;
      int at = done;
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const int n = counts[turn][u][w];
        at += w < wave ? n : 0;
        done += n;
      }
      if (v[u] == i) a.order[at + __popcll(b[u] & ((1ull << lane) - 1))] = (int32_t)(base + u * 1024 + tid);
    }
  }
}

__global__ __launch_bounds__(1024) void group_kernel(const GroupArgs a) { list_tokens(a, blockIdx.x); }

// ------------------------------------------------------------------------------- the adapters' gradients
// A bank the other way round: (r, width) to (width, r) or back, `cols` columns of all ranks at a time, whose (cols, r) side
// is one run of memory. (48 adapters of rank 8, 1752 to 5504, fp32: 48 us in tiles of 32 x 32, three quarters of them empty.)
// Smaller tiles where few of the largest would run: 3 adapters of rank 8, 1792 to 6869, 5.9 us in 27 workgroups, 4.0 in 204.
constexpr int kTurn = 8192;  // the most values of a tile
static int turn_cols(int64_t n, int64_t r, int64_t K, int64_t N) {
  const int64_t values = std::min<int64_t>(kTurn, std::max<int64_t>(1024, n * r * (K + N) / 256));
  return (int)std::max<int64_t>(64, std::min<int64_t>(4096, values / r / 64 * 64));
}
template <typename T>
__device__ __forceinline__ void turn(const T *__restrict__ in, T *__restrict__ out, int r, int64_t width, int cols, bool to_run,
                                     unsigned block) {
  __shared__ T tile[kTurn + 128];
  const unsigned each = (unsigned)((width + cols - 1) / cols);
  const int64_t i = block / each, c0 = (int64_t)(block % each) * cols;
  const int n = (int)min((int64_t)cols, width - c0), pitch = cols + 1;
  in += i * r * width, out += i * r * width;
  for (int e = threadIdx.x; e < n * r; e += 1024) {
    const int q = to_run ? e / n : e % r, c = to_run ? e % n : e / r;
    tile[q * pitch + c] = in[to_run ? q * width + c0 + c : c0 * r + e];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * r; e += 1024) {
    const int q = to_run ? e % r : e / n, c = to_run ? e / r : e % n;
    out[to_run ? c0 * r + e : q * width + c0 + c] = tile[q * pitch + c];
  }
}
// What the backward pass starts with: both banks the other way round, and the lists where the forward made none.
template <typename T>
__global__ __launch_bounds__(1024) void prepare_kernel(const T *__restrict__ a, T *__restrict__ at, const T *__restrict__ b,
                                                       T *__restrict__ bt, int r, int64_t K, int64_t N, int cols,
                                                       unsigned a_blocks, unsigned lists, const GroupArgs g) {
  if (blockIdx.x < lists) list_tokens(g, blockIdx.x);
  else if (blockIdx.x - lists < a_blocks) turn<T>(a, at, r, K, cols, true, blockIdx.x - lists);
  else turn<T>(b, bt, r, N, cols, false, blockIdx.x - lists - a_blocks);
}

struct GradArgs {
  const void *x, *g;        // (M, K), (M, N)
  int64_t x_stride, g_stride, K, N;
  const float *gh, *h;      // (M, r): the gradient's narrow product, the forward's
  const int32_t *order;
  const Slot *slots;
  float *parts;             // (slots, r K + N r)
  int r, n, a_blocks, masked;
  Mask mask;
};

// A slot's sums over its tokens for 128 columns of dA or dB and 16 RB ranks: D[rank][column] = p^T z in fp32 matrix
// instructions of 4 tokens, which read both operands as they lie in memory. A wave takes 16 tokens at a time and has
// the next 16 on the way. Memory bounds it where adapters have many tokens (fp32, 8192 of 1536 and 1536, rank 16: 28 us for
// 101 MB, 3.6 TB/s); in short pieces it is the two steps' latency (bf16, 2047 of 1792 and 6869, rank 8, masked: 18 us for 35).
template <int DT, int RB>
__global__ __launch_bounds__(256) void grad_kernel(const GradArgs p) {
  using T = typename Elem<DT>::T;
  using V = typename Oct<DT>::V;
  const Slot s = p.slots[blockIdx.y];
  if (s.adapter < 0 || s.adapter >= p.n) return;
  const bool of_a = (int)blockIdx.x < p.a_blocks;
  const int64_t width = of_a ? p.K : p.N, stride = of_a ? p.x_stride : p.g_stride;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
  const int64_t c = (int64_t)(of_a ? blockIdx.x : blockIdx.x - p.a_blocks) * 128 + col * 8;
  const bool whole = c + 8 <= width;
  const T *const z = (const T *)(of_a ? p.x : p.g);
  const float *const q = of_a ? p.gh : p.h;
  const int r0 = blockIdx.z * 64;
  const bool masked = of_a && p.masked, odd = DT != KSD_F32 && ((uintptr_t)z & 3 || stride & 1);
  const MaskKey key = p.masked ? mask_key(p.mask) : MaskKey{};
  struct Step {
    Held<DT> z[4];
    float p[4][RB];
    int m[4];
  };
  const auto load = [&](int m0, Step &o) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = m0 + u * 4 + grp < s.to;
      const int64_t m = p.order[in ? m0 + u * 4 + grp : s.from];
      o.m[u] = (int)m;
      o.z[u] = Held<DT>{};
      if (in) {
        if (!whole) o.z[u].v = load_oct<DT>(z + m * stride, c, width);
        else if (odd) hold<DT, true>(o.z[u], z + m * stride, c);
        else hold<DT, false>(o.z[u], z + m * stride, c);
      }
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const int rank = r0 + b * 16 + col;
        o.p[u][b] = in && rank < p.r ? q[m * p.r + rank] : 0.0f;
      }
    }
  };
  f32x4 acc[RB][8] = {};
  Step now, next;
  int m0 = s.from + wave * 16;
  if (m0 < s.to) load(m0, now);
  for (; m0 < s.to; m0 += 64) {
    if (m0 + 64 < s.to) load(m0 + 64, next);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float f[8];
      to_floats<DT>(odd && whole ? held<DT, true>(now.z[u], z + now.m[u] * stride, c) : now.z[u].v, f);
      if (masked) apply_mask(p.mask, mask_bits(p.mask, key, now.m[u], (uint32_t)(c >> 3)), f);
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(now.p[u][b], f[j], acc[b][j], 0, 0, 0);
    }
    now = next;
  }
  __shared__ f32x4 sum[4][8][64];
  float *const out = p.parts + (int64_t)blockIdx.y * p.r * (p.K + p.N);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
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

// da, db: an adapter's slots added by four waves, every fourth slot each, and the four sums in order.
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ parts, const int2 *__restrict__ spans, int64_t na,
                                                   int64_t nb, float *__restrict__ da, float *__restrict__ db) {
  __shared__ float sums[4][64];
  const int i = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int2 s = spans[i];
  const int64_t e = (int64_t)blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (e < na + nb) {
#pragma unroll 4
    for (int j = wave; j < s.y; j += 4) v += parts[(s.x + j) * (na + nb) + e];
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave || e >= na + nb) return;
  v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
  if (e < na) da[i * na + e] = v;
  else db[i * nb + e - na] = v;
}

// The same where an adapter has few slots: 1024 values a workgroup, slot after slot (48 adapters of 50 slots: 14 us in
// the other form).
__global__ __launch_bounds__(256) void join_few_kernel(const float *__restrict__ parts, const int2 *__restrict__ spans, int64_t na,
                                                       int64_t nb, float *__restrict__ da, float *__restrict__ db) {
  const int i = blockIdx.y;
  const int2 s = spans[i];
  const int64_t e0 = (int64_t)blockIdx.x * 1024 + threadIdx.x;
  float v[4] = {};
  for (int j = 0; j < s.y; ++j)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (e0 + u * 256 < na + nb) v[u] += parts[(s.x + j) * (na + nb) + e0 + u * 256];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t e = e0 + u * 256;
    if (e < na) da[i * na + e] = v[u];
    else if (e < na + nb) db[i * nb + e - na] = v[u];
  }
}

static bool float_type(int t) { return t == KSD_F32 || t == KSD_BF16 || t == KSD_F16; }
static int64_t size_of(int t) { return t == KSD_F32 ? 4 : 2; }

struct Take {
  int64_t at = 0;
  int64_t operator()(int64_t bytes) {
    const int64_t v = at;
    at += (bytes + 255) / 256 * 256;
    return v;
  }
};
// Tokens of a piece of the gradients' sums: such that the columns and pieces give the device enough workgroups (train
// calls, 8192 tokens of 1536 to 1536: 256 tokens 123 us, 128 tokens 128, 512 tokens 134; 2047 of 1792 to 6869: 119, 113, 134).
static int piece_of(int64_t M, int64_t K, int64_t N) {
  int piece = 256;
  while (piece > kLeast && cdiv(M, piece) * (cdiv(K, 128) + cdiv(N, 128)) < 768) piece /= 2;
  return piece;
}
struct Groups {
  int64_t order, tiles, pieces, spans, bytes;
};
static Groups groups(int64_t M, int64_t n) {
  Take take;
  Groups l;
  l.order = take(M * 4);
  l.tiles = take((M / kTile + n + 1) * (int64_t)sizeof(Slot));
  l.pieces = take((M / kLeast + n + 1) * (int64_t)sizeof(Slot));
  l.spans = take((n + 1) * 8);
  l.bytes = take.at;
  return l;
}
// Whether the products go by the lists: tokens in any order whose adapters, read for each token by itself, would be
// more than 32 MB (the list's launch costs as much as that, about 5 us).
static bool by_lists(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int64_t per, int dtype) {
  return n > 1 && per < 16 && M > 64 && M * r * (K + N) * size_of(dtype) > (32 << 20);
}

// The workspace of a forward pass: lists, then the narrow product's parts.
struct Forward {
  bool lists;
  int64_t sums, bytes;
};
static Forward forward(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int64_t per, int dtype) {
  Forward l;
  l.lists = by_lists(M, K, N, r, n, per, dtype);
  PairArgs p{};
  p.M = M, p.K = K, p.N = N, p.r = (int)r, p.n = (int)n, p.per = per;
  shape(p, l.lists, aligned_rank(r, dtype));
  l.sums = l.lists ? groups(M, n).bytes : 0;
  l.bytes = l.sums + p.splits * M * r * 4;
  return l;
}
struct Layout {
  int64_t at, bt, gh, parts, groups, sums, bytes;
};
static Layout layout(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int64_t per, int dtype) {
  Take take;
  Layout l;
  l.at = take(n * r * K * size_of(dtype));
  l.bt = take(n * r * N * size_of(dtype));
  l.gh = take(M * r * 4);
  l.parts = take((M / piece_of(M, K, N) + n + 1) * r * (K + N) * 4);
  const Forward f = forward(M, N, K, r, n, per, dtype);
  l.groups = take(groups(M, n).bytes);
  l.sums = take(f.bytes - f.sums);
  l.bytes = take.at;
  return l;
}

// Sizes for which every index fits its type.
static bool fits(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n) {
  return M >= 0 && K >= 1 && N >= 1 && r >= 1 && r <= 128 && n >= 1 && n <= 65535 && M <= 0x7fffffff - 65536 &&
         K <= 0x7fffffff - 65536 && N <= 0x7fffffff - 65536;
}

// adapter_of divides by it in 32 bits.
static bool per_fits(int64_t per) { return per >= 1 && per <= 0x7fffffff; }

static int run_pair(const PairArgs &args, int dtype, bool mask, hipStream_t st) {
  PairArgs p = args;
  if (dtype != KSD_F32) {
    p.odd_x = (((uintptr_t)p.x | (uintptr_t)p.a) & 3) != 0 || ((p.x_stride | p.K) & 1);
    p.odd_y = (((uintptr_t)p.base | (uintptr_t)p.y) & 3) != 0 || ((p.base_stride | p.N) & 1);
  }
  shape(p, p.slots != nullptr, aligned_rank(p.r, dtype) && !p.odd_x && !p.odd_y);
  int64_t tiles = cdiv(p.M, p.rows);
  if (p.slots) {
    p.tiles = kTile / p.rows;
    tiles = (p.M / kTile + p.n + 1) * p.tiles;
  }
  if (!grid_fits(tiles, 64 * kWaves) || cdiv(p.N, p.cols) > 65535)
    return fail(KSD_EINVAL, "adapter_linear: too many rows or columns");
  for (p.phase = p.splits ? 1 : 0; p.phase < 3; p.phase += p.splits ? 1 : 3) {
    if (dtype == KSD_F32) launch_pair<KSD_F32>(p, mask, (unsigned)tiles, st);
    else if (dtype == KSD_BF16) launch_pair<KSD_BF16>(p, mask, (unsigned)tiles, st);
    else launch_pair<KSD_F16>(p, mask, (unsigned)tiles, st);
  }
  return check_launch("adapter_linear");
}

static GroupArgs group_args(const void *index, int wide, int64_t per, int64_t M, int64_t K, int64_t N, int64_t n, char *w) {
  const Groups l = groups(M, n);
  return GroupArgs{index, wide, (int)n, per, M, (int32_t *)(w + l.order), (Slot *)(w + l.tiles), (Slot *)(w + l.pieces),
                   (int2 *)(w + l.spans), piece_of(M, K, N)};
}

template <int DT>
static void launch_grad(const GradArgs &q, dim3 grid, hipStream_t st) {
  if (q.r <= 16) grad_kernel<DT, 1><<<grid, 256, 0, st>>>(q);
  else if (q.r <= 32) grad_kernel<DT, 2><<<grid, 256, 0, st>>>(q);
  else grad_kernel<DT, 4><<<grid, 256, 0, st>>>(q);
}
template <typename T>
static void launch_prepare(const void *a, void *at, const void *b, void *bt, int64_t n, int64_t r, int64_t K, int64_t N, bool lists,
                           const GroupArgs &g, hipStream_t st) {
  const int cols = turn_cols(n, r, K, N);
  const unsigned blocks = (unsigned)(n * cdiv(K, cols)), lists_n = lists ? (unsigned)n + 1 : 0;
  prepare_kernel<T><<<lists_n + blocks + (unsigned)(n * cdiv(N, cols)), 1024, 0, st>>>(
      (const T *)a, (T *)at, (const T *)b, (T *)bt, (int)r, K, N, cols, blocks, lists_n, g);
}
static void launch_join(const float *parts, const int2 *spans, int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, float *da,
                        float *db, hipStream_t st) {
  const int64_t each = r * (K + N);
  if (M / piece_of(M, K, N) <= 4 * n)
    join_few_kernel<<<dim3((unsigned)cdiv(each, 1024), (unsigned)n), 256, 0, st>>>(parts, spans, r * K, r * N, da, db);
  else
    join_kernel<<<dim3((unsigned)cdiv(each, 64), (unsigned)n), 256, 0, st>>>(parts, spans, r * K, r * N, da, db);
}

}  // namespace adp
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_adapter_linear_workspace(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int64_t rows_per_index, int dtype,
                                            int64_t *bytes) {
  if (!bytes || !adp::fits(M, K, N, r, n) || !adp::float_type(dtype) || !adp::per_fits(rows_per_index))
    return fail(KSD_EINVAL, "adapter_linear_workspace: bad arguments");
  *bytes = adp::forward(M, K, N, r, n, rows_per_index, dtype).bytes;
  return KSD_OK;
}

extern "C" int ksd_adapter_linear(const void *x, int dtype, int64_t M, int64_t K, int64_t x_stride, const void *a, const void *b,
                                  int64_t n, int64_t r, int64_t N, const void *index, int index_wide, int64_t rows_per_index,
                                  const float *scales, const void *base, int64_t base_stride, int64_t drop, uint64_t seed,
                                  const void *seed_from, int64_t stream_id, void *y, float *hidden, void *workspace,
                                  int64_t workspace_bytes, void *stream) {
  using namespace adp;
  if (!fits(M, K, N, r, n) || !per_fits(rows_per_index) || (M > 1 && (x_stride < K || (base && base_stride < N))))
    return fail(KSD_EINVAL, "adapter_linear: bad shape");
  if (!float_type(dtype)) return fail(KSD_ETYPE, "adapter_linear: unsupported element type");
  Mask m;
  if (!make_mask(m, drop, seed, seed_from, stream_id)) return fail(KSD_EINVAL, "adapter_linear: bad probability, seed or stream");
  if (M == 0) return KSD_OK;
  const Forward l = forward(M, K, N, r, n, rows_per_index, dtype);
  if (l.bytes && (!workspace || workspace_bytes < l.bytes || (uintptr_t)workspace % 16))
    return fail(KSD_EINVAL, "adapter_linear: short or misaligned workspace");
  if (!x || !a || !b || !index || !y) return fail(KSD_EINVAL, "adapter_linear: null pointer");
  hipStream_t st = (hipStream_t)stream;
  char *const w = (char *)workspace;
  PairArgs p{x, x_stride, M, K, N, a, b, index, index_wide, rows_per_index, scales, base, base_stride, y, hidden,
             (int)n, (int)r, 0, 0, m, 1, 0, 0, 0, nullptr, nullptr, 1, 0, 0, (float *)(w + l.sums)};
  if (l.lists) {
    const GroupArgs g = group_args(index, index_wide, rows_per_index, M, K, N, n, w);
    group_kernel<<<(unsigned)(n + 1), 1024, 0, st>>>(g);
    p.order = g.order, p.slots = g.tiles;
  }
  return run_pair(p, dtype, drop > 0, st);
}

extern "C" int ksd_adapter_linear_backward_workspace(int64_t M, int64_t K, int64_t N, int64_t r, int64_t n, int64_t rows_per_index,
                                                     int dtype, int64_t *bytes) {
  if (!bytes || !adp::fits(M, K, N, r, n) || !adp::float_type(dtype) || !adp::per_fits(rows_per_index))
    return fail(KSD_EINVAL, "adapter_linear_backward_workspace: bad arguments");
  *bytes = adp::layout(M, K, N, r, n, rows_per_index, dtype).bytes;
  return KSD_OK;
}

extern "C" int ksd_adapter_linear_backward(const void *g, int dtype, int64_t M, int64_t N, int64_t g_stride, const void *x,
                                           int64_t K, int64_t x_stride, const float *hidden, const void *forward_workspace,
                                           int64_t forward_bytes, const void *a, const void *b, int64_t n, int64_t r,
                                           const void *index, int index_wide, int64_t rows_per_index, const float *scales,
                                           const void *base, int64_t base_stride, int64_t drop, uint64_t seed,
                                           const void *seed_from, int64_t stream_id, void *dx, float *da, float *db,
                                           void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace adp;
  if (!fits(M, K, N, r, n) || !per_fits(rows_per_index) ||
      (M > 1 && (x_stride < K || g_stride < N || (base && base_stride < K))))
    return fail(KSD_EINVAL, "adapter_linear_backward: bad shape");
  if (!float_type(dtype)) return fail(KSD_ETYPE, "adapter_linear_backward: unsupported element type");
  Mask m;
  if (!make_mask(m, drop, seed, seed_from, stream_id))
    return fail(KSD_EINVAL, "adapter_linear_backward: bad probability, seed or stream");
  if ((M > 0 && (!g || !x || !hidden || !a || !b || !index)) || !da != !db)
    return fail(KSD_EINVAL, "adapter_linear_backward: null pointer");
  const Layout l = layout(M, K, N, r, n, rows_per_index, dtype);
  const Forward f = forward(M, K, N, r, n, rows_per_index, dtype);
  if (!workspace || workspace_bytes < l.bytes || (uintptr_t)workspace % 16 ||
      (M > 0 && f.lists && (!forward_workspace || forward_bytes < f.sums || (uintptr_t)forward_workspace % 16)))
    return fail(KSD_EINVAL, "adapter_linear_backward: short or misaligned workspace");
  const int64_t slots = M / piece_of(M, K, N) + n + 1, blocks_a = cdiv(K, 128), blocks_b = cdiv(N, 128), each = r * (K + N);
  const int64_t cols = turn_cols(n, r, K, N);
  if (slots > 65535 || !grid_fits(blocks_a + blocks_b, 256) || !grid_fits(cdiv(each, 64), 256) ||
      !grid_fits(n * (cdiv(K, cols) + cdiv(N, cols)) + n + 1, 1024))
    return fail(KSD_EINVAL, "adapter_linear_backward: too many tokens, columns or adapters");
  hipStream_t st = (hipStream_t)stream;
  char *const w = (char *)workspace;
  if (M == 0) {  // no slot has a token: zeros
    if (!da) return KSD_OK;
    group_kernel<<<(unsigned)(n + 1), 1024, 0, st>>>(group_args(index, index_wide, rows_per_index, M, K, N, n, w + l.groups));
    launch_join(nullptr, (const int2 *)(w + l.groups + groups(M, n).spans), M, K, N, r, n, da, db, st);
    return check_launch("adapter_linear_backward");
  }
  const bool lists = f.lists;
  const GroupArgs ga = group_args(index, index_wide, rows_per_index, M, K, N, n, lists ? (char *)forward_workspace : w + l.groups);
  float *const gh = (float *)(w + l.gh);
  // the narrow product contracts dY's columns, the wide one the ranks: both banks the other way round
  if (dtype == KSD_F32) launch_prepare<uint32_t>(a, w + l.at, b, w + l.bt, n, r, K, N, !lists && da, ga, st);
  else launch_prepare<uint16_t>(a, w + l.at, b, w + l.bt, n, r, K, N, !lists && da, ga, st);
  PairArgs p{g, g_stride, M, N, K, w + l.bt, w + l.at, index, index_wide, rows_per_index, scales, base, base_stride, dx, gh,
             (int)n, (int)r, 0, 0, m, 0, 1, 0, 0, nullptr, nullptr, 1, 0, 0, (float *)(w + l.sums)};
  if (lists) p.order = ga.order, p.slots = ga.tiles;
  const int rc = run_pair(p, dtype, drop > 0, st);
  if (rc || !da) return rc;
  float *const parts = (float *)(w + l.parts);
  GradArgs q{x, g, x_stride, g_stride, K, N, gh, hidden, ga.order, ga.pieces, parts, (int)r, (int)n, (int)blocks_a, drop > 0, m};
  const dim3 grid((unsigned)(blocks_a + blocks_b), (unsigned)slots, (unsigned)cdiv(r, 64));
  if (dtype == KSD_F32) launch_grad<KSD_F32>(q, grid, st);
  else if (dtype == KSD_BF16) launch_grad<KSD_BF16>(q, grid, st);
  else launch_grad<KSD_F16>(q, grid, st);
  launch_join(parts, ga.spans, M, K, N, r, n, da, db, st);
  return check_launch("adapter_linear_backward");
}
