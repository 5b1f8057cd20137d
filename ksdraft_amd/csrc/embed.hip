// Embedding lookup with a scale, and the table's gradient by sorted tokens.
//
//   y[i]  = round(scale * W[id_i])
//   dW[v] = scale * sum of g[i] over the positions i with id_i = v, in fp32
//
// The positions are sorted by token (stable radix sort), so every token's rows are one run of the
// sorted list and no float atomics are needed. Runs are cut at multiples of 16 or 32 sorted positions, so a
// token that fills the batch is spread over the device like any other. Rows are added in the order of
// their positions within a piece, the pieces of a cut run in order, a long run's in 16 shares whose sums are
// added in order (few tokens: a token's positions in up to 4 such shares). That is not the sum of the rows one
// after the other, but it depends on the ids and sizes alone: repeated calls give the same bits.
#include "ksd_common.h"

#include <algorithm>

namespace ksd {
namespace emb {

__device__ __forceinline__ int64_t load_id(const void *ids, int wide, int64_t i) {
  return wide ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
}

template <int DT>
__device__ __forceinline__ void load_any(const typename Elem<DT>::T *p, int n, float *v) {
  if (n >= 8) {
    struct __attribute__((packed, aligned(DT == KSD_F32 ? 4 : 2))) Any { uint4 q; };
    Raw8<DT> r;
    r.a = ((const Any *)p)->q;
    if constexpr (DT == KSD_F32) r.b = ((const Any *)(p + 4))->q;
    cvt_raw8<DT>(r, true, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? Elem<DT>::load(p + j) : 0.0f;
  }
}
template <int DT>
__device__ __forceinline__ void store_any(typename Elem<DT>::T *p, int n, const float *v) {
  struct __attribute__((packed, aligned(DT == KSD_F32 ? 4 : 2))) Any { uint4 q; };
  if (n >= 8) {
    if constexpr (DT == KSD_F32) {
      uint4 a, b;
      a.x = __builtin_bit_cast(uint32_t, v[0]), a.y = __builtin_bit_cast(uint32_t, v[1]);
      a.z = __builtin_bit_cast(uint32_t, v[2]), a.w = __builtin_bit_cast(uint32_t, v[3]);
      b.x = __builtin_bit_cast(uint32_t, v[4]), b.y = __builtin_bit_cast(uint32_t, v[5]);
      b.z = __builtin_bit_cast(uint32_t, v[6]), b.w = __builtin_bit_cast(uint32_t, v[7]);
      ((Any *)p)->q = a;
      ((Any *)(p + 4))->q = b;
    } else {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint16_t lo, hi;
        store_out<DT>(&lo, 0, v[2 * k]);
        store_out<DT>(&hi, 0, v[2 * k + 1]);
        w[k] = lo | (uint32_t)hi << 16;
      }
      ((Any *)p)->q = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) store_out<DT>(p, j, v[j]);
  }
}

// One wave per row. (65521 tokens of a table 32003 x 1792, bf16 to bf16: 72 us, 6.5 TB/s; a few tokens: the launch.)
template <int DT, int OUT>
__global__ __launch_bounds__(256) void lookup_kernel(const void *__restrict__ table, const void *__restrict__ ids, int wide,
                                                     int64_t n, int64_t V, int64_t d, int64_t stride, float scale,
                                                     void *__restrict__ out) {
  using T = typename Elem<DT>::T;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= n) return;
  const int64_t id = load_id(ids, wide, i);
  const bool ok = id >= 0 && id < V;
  const T *row = (const T *)table + (ok ? id : 0) * stride;
  typename Elem<OUT>::T *o = (typename Elem<OUT>::T *)out + i * d;
  for (int64_t c = (threadIdx.x & 63) * 8; c < d; c += 512) {
    float v[8];
    const int m = (int)min((int64_t)8, d - c);
    load_any<DT>(row + c, m, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ok ? v[j] * scale : 0.0f;
    store_any<OUT>(o + c, m, v);
  }
}

// ------------------------------------------------------------------------------------ sort
// Stable, least significant digit first, at most 9 bits a pass. Ids that take no part (the padding
// token, ids out of range) become the key V, which sorts last. Keys of one digit keep their order:
// rank = earlier tiles' + earlier waves' + earlier rounds of 64 + lower lanes with that digit, the last
// from ballots over the digit's bits.
constexpr int kDigits = 512;
constexpr int kOne = 8192;  // keys that are placed by counting

__device__ __forceinline__ uint32_t key_of(const void *ids, int wide, int64_t i, int64_t V, int64_t pad) {
  const int64_t id = load_id(ids, wide, i);
  return (uint32_t)(id < 0 || id >= V || id == pad ? V : id);
}

// Zeros for n bytes at p, 16-byte aligned: workgroup `block` of 256 threads writes one piece of 4 KB, so that
// the stores walk through memory in launch order. (922 MB: 6.3 to 6.6 TB/s; loops over a smaller grid 4.7 to
// 6.1, larger pieces 4.2 to 5.6. Non-temporal: 8192 rows' sums after it take 15 us, after ordinary stores,
// whose dirty lines have to leave first, 28.)
struct Fill {
  char *p;
  int64_t n;
};
static int64_t fill_blocks(const Fill &f) { return cdiv(f.n, 4096); }
__device__ __forceinline__ void fill(const Fill &f, int64_t block) {
  typedef uint32_t vec __attribute__((ext_vector_type(4)));
  const int64_t at = (block * 256 + threadIdx.x) * 16;
  if (at + 16 <= f.n) __builtin_nontemporal_store((vec){0, 0, 0, 0}, (vec *)(f.p + at));
  else
    for (int64_t i = at; i < f.n; ++i) f.p[i] = 0;
}

struct SortArgs {
  const void *ids;  // first pass: the ids (positions are the index); later passes: NULL
  const uint32_t *keys;
  const int32_t *pos;
  uint32_t *out_keys;
  int32_t *out_pos;
  uint32_t *counts;  // (tiles, kDigits)
  int64_t V, pad;
  int n, tiles, shift, bits, wide;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, int i) {
  return a.ids ? key_of(a.ids, a.wide, i, a.V, a.pad) : a.keys[i];
}

// Lanes of the wave that hold digit d too (`in`: lanes that hold a key).
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool in) {
  uint64_t m = __ballot(in);
  for (int b = 0; b < bits; ++b) {
    const uint64_t bal = __ballot((d >> b) & 1);
    m &= (d >> b) & 1 ? bal : ~bal;
  }
  return m;
}

// Exclusive sum over one value per thread of a workgroup of NT threads (scratch: NT / 64 words).
template <int NT>
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t v, uint32_t *scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)s, o);
    if (lane >= o) s += u;
  }
  if (lane == 63) scratch[wave] = s;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += scratch[w];
  __syncthreads();
  return before + s - v;
}

// Tiles of 256 R keys, four waves of R rounds. Digit counts of the tiles; workgroups past them clear `out`.
// (65521 ids, per pass: 4.7 us, the scatter 8.9, both short launches at latency.)
template <int R>
__global__ __launch_bounds__(256) void sort_count_kernel(const SortArgs a, const Fill f) {
  __shared__ uint32_t h[kDigits];
  if ((int)blockIdx.x >= a.tiles) {
    fill(f, (int64_t)blockIdx.x - a.tiles);
    return;
  }
  const int tid = threadIdx.x, t0 = blockIdx.x * (256 * R);
  h[tid] = h[tid + 256] = 0;
  __syncthreads();
  const uint32_t mask = (1u << a.bits) - 1;
#pragma unroll 4
  for (int r = 0; r < R; ++r) {
    const int i = t0 + r * 256 + tid;
    if (i < a.n) atomicAdd(&h[(sort_key(a, i) >> a.shift) & mask], 1u);
  }
  __syncthreads();
  uint32_t *const c = a.counts + (int64_t)blockIdx.x * kDigits;
  c[tid] = h[tid];
  c[tid + 256] = h[tid + 256];
}

template <int R>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const SortArgs a) {
  __shared__ uint32_t h[4][kDigits];
  __shared__ uint32_t scratch[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int base = blockIdx.x * (256 * R) + wave * (64 * R);
  const uint32_t mask = (1u << a.bits) - 1;
  const uint64_t below = (1ull << lane) - 1;
  uint32_t key[R];
  int32_t pos[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = base + r * 64 + lane;
    key[r] = i < a.n ? sort_key(a, i) : 0;
    pos[r] = a.ids || i >= a.n ? i : a.pos[i];
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) h[w][tid] = h[w][tid + 256] = 0;
  // digits 2 tid, 2 tid + 1: keys of earlier tiles, and of all tiles for the digits' starts
  uint2 earlier = make_uint2(0, 0), all = make_uint2(0, 0);
#pragma unroll 8
  for (int t = 0; t < a.tiles; ++t) {
    const uint2 c = *(const uint2 *)(a.counts + (int64_t)t * kDigits + 2 * tid);
    all.x += c.x, all.y += c.y;
    if (t < (int)blockIdx.x) earlier.x += c.x, earlier.y += c.y;
  }
  const uint32_t start = exclusive_sum<256>(all.x + all.y, scratch);
  uint64_t same[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = base + r * 64 + lane < a.n;
    const uint32_t d = (key[r] >> a.shift) & mask;
    same[r] = same_digit(d, a.bits, in);
    if (in && (same[r] & below) == 0) h[wave][d] += (uint32_t)__popcll(same[r]);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t at = start + (e ? all.x + earlier.y : earlier.x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t c = h[w][2 * tid + e];
      h[w][2 * tid + e] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = base + r * 64 + lane < a.n;
    const uint32_t d = (key[r] >> a.shift) & mask;
    uint32_t first = 0;
    if (in) {
      first = h[wave][d];
      const uint32_t to = first + (uint32_t)__popcll(same[r] & below);
      a.out_keys[to] = key[r];
      a.out_pos[to] = pos[r];
    }
    __builtin_amdgcn_wave_barrier();
    if (in && (same[r] & below) == 0) h[wave][d] = first + (uint32_t)__popcll(same[r]);
    __builtin_amdgcn_wave_barrier();
  }
}

// Up to kOne keys below 2^19: each key's place is the number of smaller (key, position) pairs, one word each,
// counted by all CUs at 256 keys and kOthers others a workgroup. (8192 tokens of 942 by 93: the gradient takes
// 22 us, with a radix sort's four launches 27.) Workgroups past the counting ones clear `out` meanwhile.
constexpr int kOthers = 512;
__device__ __forceinline__ uint32_t pair_of(const SortArgs &a, int i) {
  return i < a.n ? key_of(a.ids, a.wide, i, a.V, a.pad) * (uint32_t)kOne + (uint32_t)i : 0xffffffffu;
}
__global__ __launch_bounds__(256) void rank_count_kernel(const SortArgs a, unsigned counting, const Fill f) {
  __shared__ __attribute__((aligned(16))) uint32_t others[kOthers];
  if (blockIdx.x >= counting) {
    fill(f, blockIdx.x - counting);
    return;
  }
  const int mine = (a.n + 255) / 256, slice = blockIdx.x / mine, i = (blockIdx.x % mine) * 256 + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kOthers / 256; ++k) others[k * 256 + threadIdx.x] = pair_of(a, slice * kOthers + k * 256 + threadIdx.x);
  const uint32_t c = pair_of(a, i);
  __syncthreads();
  uint32_t less = 0;
#pragma unroll 8
  for (int j = 0; j < kOthers; j += 4) {
    const uint4 q = *(const uint4 *)(others + j);
    less += (q.x < c) + (q.y < c) + (q.z < c) + (q.w < c);
  }
  if (i < a.n) a.counts[(int64_t)slice * a.n + i] = less;
}
__global__ __launch_bounds__(256) void rank_scatter_kernel(const SortArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x, slices = (a.n + kOthers - 1) / kOthers;
  if (i >= a.n) return;
  uint32_t to = 0;
  for (int s = 0; s < slices; ++s) to += a.counts[(int64_t)s * a.n + i];
  a.out_keys[to] = key_of(a.ids, a.wide, i, a.V, a.pad);
  a.out_pos[to] = i;
}
// Up to kPlace keys: 64 a workgroup, counted against a quarter of all by each wave and placed at once. (1024 tokens
// of 942 by 93: the gradient takes 20 us, by the two launches above 24.)
constexpr int kPlace = 2048;
__global__ __launch_bounds__(256) void rank_place_kernel(const SortArgs a, unsigned counting, const Fill f) {
  __shared__ __attribute__((aligned(16))) uint32_t others[kPlace];
  __shared__ uint32_t part[4][64];
  if (blockIdx.x >= counting) {
    fill(f, blockIdx.x - counting);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
#pragma unroll
  for (int k = 0; k < kPlace / 256; ++k) others[k * 256 + threadIdx.x] = pair_of(a, k * 256 + threadIdx.x);
  const uint32_t c = pair_of(a, i);
  __syncthreads();
  uint32_t less = 0;
#pragma unroll 8
  for (int j = wave * (kPlace / 4); j < (wave + 1) * (kPlace / 4); j += 4) {
    const uint4 q = *(const uint4 *)(others + j);
    less += (q.x < c) + (q.y < c) + (q.z < c) + (q.w < c);
  }
  part[wave][lane] = less;
  __syncthreads();
  if (wave > 0 || i >= a.n) return;
  const uint32_t to = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
  a.out_keys[to] = c / kOne;
  a.out_pos[to] = i;
}

// ------------------------------------------------------------------------------------ sums
struct SumArgs {
  const uint32_t *keys;
  const int32_t *pos;
  const void *g;
  void *out;
  float *parts;  // (2, chunks, d): the piece of the run that a chunk begins in, and the one it ends in
  int64_t d, stride, V;
  int64_t rows;                     // rows of out that this launch writes where no token occurs
  int n, chunks, run, slices, add;  // run: sorted positions of a chunk; slices of 64 lanes' columns
  unsigned sums;                    // workgroups that sum
  float scale;
};

// A lane's NV columns (16 bytes) from c on as raw bits, loaded at c0 = min(c, d - NV) so that rows need no
// branches.
template <int DT, int NV>
struct RawCols {
  using T = typename Elem<DT>::T;
  uint32_t w[NV * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T *row, int64_t c0, int64_t d) {
    constexpr int W = NV * sizeof(T) / 4;
    if (d >= NV) {
      struct __attribute__((packed, aligned(sizeof(T)))) Any { uint32_t w[W]; };
      const Any q = *(const Any *)(row + c0);
#pragma unroll
      for (int j = 0; j < W; ++j) w[j] = q.w[j];
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if constexpr (DT == KSD_F32) w[j] = j < d ? __builtin_bit_cast(uint32_t, row[j]) : 0;
        else w[j] = (2 * j < d ? row[2 * j] : 0) | (uint32_t)(2 * j + 1 < d ? row[2 * j + 1] : 0) << 16;
      }
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (DT == KSD_F32) {
      return __builtin_bit_cast(float, w[j]);
    } else {
      const uint16_t h = (uint16_t)(w[j / 2] >> (j % 2 * 16));
      return Elem<DT>::load(&h);
    }
  }
};
template <int DT, int NV>
__device__ __forceinline__ void load_cols(const typename Elem<DT>::T *row, int64_t c0, int64_t d, float *v) {
  RawCols<DT, NV> q;
  q.load(row, c0, d);
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = q.at(j);
}

template <int OUT, int NV>
__device__ __forceinline__ void put_row(const SumArgs &a, uint32_t key, int64_t c, int64_t c0, const float *acc) {
  typename Elem<OUT>::T *o = (typename Elem<OUT>::T *)a.out + (int64_t)key * a.d;
  if (c + NV <= a.d) {
    float v[NV], was[NV];
    if (a.add) load_cols<OUT, NV>(o, c, a.d, was);
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = a.add ? was[j] + acc[j] * a.scale : acc[j] * a.scale;
    if constexpr (OUT == KSD_F32) {
      struct __attribute__((packed, aligned(4))) Any { float w[NV]; } q;
#pragma unroll
      for (int j = 0; j < NV; ++j) q.w[j] = v[j];
      *(Any *)(o + c) = q;
    } else {
      struct __attribute__((packed, aligned(2))) Any { uint16_t w[NV]; } q;
#pragma unroll
      for (int j = 0; j < NV; ++j) store_out<OUT>(&q.w[j], 0, v[j]);
      *(Any *)(o + c) = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {  // columns c0 + j, those from c on
      const int64_t i = c0 + j;
      if (i >= c && i < a.d) store_out<OUT>(o, i, a.add ? Elem<OUT>::load(o + i) + acc[j] * a.scale : acc[j] * a.scale);
    }
  }
}

template <int NV>
__device__ __forceinline__ void put_part(float *o, int64_t c, int64_t c0, int64_t d, const float *acc) {
  if (c + NV <= d) {
    struct __attribute__((packed, aligned(4))) Any { float w[NV]; } q;
#pragma unroll
    for (int j = 0; j < NV; ++j) q.w[j] = acc[j];
    *(Any *)(o + c) = q;
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (c0 + j >= c && c0 + j < d) o[c0 + j] = acc[j];
  }
}

// Clears the rows [v0, v0 + kGap) of `out` below `rows` whose token does not occur: lane i looks row v0 + i up
// in the sorted keys.
constexpr int kGap = 16;
template <int OUT>
__device__ __forceinline__ void fill_gaps(const SumArgs &a, int64_t v0) {
  using T = typename Elem<OUT>::T;
  const int lane = threadIdx.x & 63;
  const int64_t v = v0 + (lane & (kGap - 1));
  int lo = 0, hi = a.n;  // first key >= v
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if ((int64_t)a.keys[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  const uint64_t there = __ballot(lo < a.n && a.keys[min(lo, a.n - 1)] == (uint32_t)v);
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
  constexpr int NV = 16 / sizeof(T);
  for (int r = threadIdx.x >> 6; r < kGap && v0 + r < a.rows; r += 4) {  // a row per wave
    if (there >> r & 1) continue;
    T *o = (T *)a.out + (v0 + r) * a.d;
#pragma unroll 4
    for (int64_t c = lane * NV; c < a.d; c += 64 * NV) {
      if (c + NV <= a.d) {
        __builtin_nontemporal_store((vec){0, 0, 0, 0}, (vec *)(o + c));
      } else {
        for (int64_t j = c; j < a.d; ++j) o[j] = (T)0;
      }
    }
  }
}

// One wave per chunk and slice of 64 NV columns: sums the chunk's runs in order, 8 rows in flight. A run
// that lies in the chunk is finished; the pieces of runs that reach past it go to parts. Workgroups past
// `sums` clear the rows without a token meanwhile, so every row of `out` is written once. (8192 x 1536 fp32 sums
// alone 15 us; 65521 x 1792 bf16 into 32003 fp32 rows 105, 4.4 TB/s: rows gathered in 3.5 KB pieces.)
template <int DT, int OUT>
__global__ __launch_bounds__(256) void sum_kernel(const SumArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int NV = DT == KSD_F32 ? 4 : 8;
  if (blockIdx.x >= a.sums) {
    fill_gaps<OUT>(a, (int64_t)(blockIdx.x - a.sums) * kGap);
    return;
  }
  const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = (int)(id / a.slices), slice = (int)(id % a.slices);
  if (b >= a.chunks) return;
  const int64_t c = ((int64_t)slice * 64 + (threadIdx.x & 63)) * NV, c0 = max((int64_t)0, min(c, a.d - NV));
  const int s0 = b * a.run, s1 = min(a.n, s0 + a.run);
  const T *g = (const T *)a.g;
  uint32_t key = a.keys[s0];
  bool whole = b == 0 || a.keys[s0 - 1] != key;  // the run begins in this chunk
  float acc[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) acc[j] = 0.0f;
  for (int sb = s0; sb < s1; sb += 8) {
    uint32_t k[8];
    RawCols<DT, NV> v[8];
    const T *row[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int i = min(sb + r, s1 - 1);
      k[r] = a.keys[i];
      row[r] = g + (int64_t)a.pos[i] * a.stride;
    }
    if (k[0] >= a.V) break;  // ids that take no part sort last
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r].load(row[r], c0, a.d);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (sb + r >= s1 || k[r] >= a.V) continue;
      if (k[r] != key) {
        if (whole) put_row<OUT, NV>(a, key, c, c0, acc);
        else put_part<NV>(a.parts + (int64_t)b * a.d, c, c0, a.d, acc);
#pragma unroll
        for (int j = 0; j < NV; ++j) acc[j] = 0.0f;
        key = k[r];
        whole = true;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) acc[j] += v[r].at(j);
    }
  }
  if (key >= a.V) return;
  if (!whole) put_part<NV>(a.parts + (int64_t)b * a.d, c, c0, a.d, acc);
  else if (s1 < a.n && a.keys[s1] == key) put_part<NV>(a.parts + ((int64_t)a.chunks + b) * a.d, c, c0, a.d, acc);
  else put_row<OUT, NV>(a, key, c, c0, acc);
}

// Joins the pieces of runs that reach past the chunk they begin in, 256 columns each: a wave looks at one chunk,
// its lanes find the run's last chunk, 64 points of the range at a time. It adds a short run's pieces itself, in
// order; a longer run's are shared out over the workgroup's waves, whose sums are added in order. (The
// gradient for 131072 tokens, us: 942 x 93, all equal, shared by 4 waves 316, by 16 121; 32003 x 1792, a natural
// text's frequencies, all runs shared by 4 waves 238, this way 218.)
constexpr int kJoin = 16;   // waves of a workgroup
constexpr int kAlone = 16;  // pieces of a short run
__device__ __forceinline__ void add_pieces(const SumArgs &a, int b, int lo, int hi, int64_t c0, float *acc) {
#pragma unroll 8
  for (int q = lo; q < hi; ++q) {
    float v[4];
    load_cols<KSD_F32, 4>(a.parts + (q == 0 ? (int64_t)a.chunks + b : (int64_t)b + q) * a.d, c0, a.d, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += v[j];
  }
}
template <int OUT>
__global__ __launch_bounds__(64 * kJoin) void join_kernel(const SumArgs a) {
  __shared__ float part[kJoin][64][4];
  __shared__ int pieces[kJoin];
  __shared__ uint32_t keys[kJoin];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t c = ((int64_t)blockIdx.y * 64 + lane) * 4, c0 = max((int64_t)0, min(c, a.d - 4));
  const int first = (int)blockIdx.x * kJoin;
  const int mine = first + wave, s0 = min(mine, a.chunks - 1) * a.run, s1 = min(s0 + a.run, a.n - 1);
  const uint32_t key = a.keys[s1 - 1 > s0 ? s1 - 1 : s0];
  const bool begins = mine < a.chunks && s0 + a.run < a.n && key < a.V && a.keys[s1] == key &&
                      !(a.keys[s0] == key && mine > 0 && a.keys[s0 - 1] == key);
  int m = 0;  // pieces: the one that the chunk ends in, then the beginnings of the next m - 1
  if (begins) {
    int last = mine + 2, end = a.chunks;  // chunks mine + 1 .. last - 1 begin with the key, chunk `end` does not
    for (int step = 1; last < end; step = (end - last + 63) / 64) {
      const int64_t q = last + (int64_t)lane * step;
      const uint64_t hit = __ballot(q < end && a.keys[min(q, (int64_t)a.chunks - 1) * a.run] == key);
      const int more = hit == ~0ull ? 64 : __builtin_ctzll(~hit);  // points with the key: all before the others
      if (more < 64) end = (int)min((int64_t)end, last + (int64_t)more * step);
      if (more > 0) last += (more - 1) * step + 1;
    }
    m = last - mine;
    if (m <= kAlone) {
      float acc[4] = {0, 0, 0, 0};
      add_pieces(a, mine, 0, m, c0, acc);
      put_row<OUT, 4>(a, key, c, c0, acc);
      m = 0;
    }
  }
  if (lane == 0) pieces[wave] = m, keys[wave] = key;
  __syncthreads();
  for (int i = 0; i < kJoin; ++i) {
    const int64_t n = pieces[i];
    if (n == 0) continue;
    float acc[4] = {0, 0, 0, 0};
    add_pieces(a, first + i, (int)(n * wave / kJoin), (int)(n * (wave + 1) / kJoin), c0, acc);
    __syncthreads();  // the last run's sums are read
#pragma unroll
    for (int j = 0; j < 4; ++j) part[wave][lane][j] = acc[j];
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kJoin; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += part[w][lane][j];
      put_row<OUT, 4>(a, keys[i], c, c0, acc);
    }
  }
}

// Up to kFew tokens in one launch without a sort: workgroup b owns the rows b, b + grid, b + 2 grid, .. (so that
// neighbouring frequent tokens meet different workgroups), lists the tokens of its rows in order, and sums or
// clears its rows. (The sorted form's time hardly depends on the tokens, this one's grows with the most frequent
// one's: 942 x 93, us: 512 tokens 7, all equal 52, sorted 16 to 20; 2048 tokens 22, 186, 19 to 21.)
// Tables past kLarge are cleared by a launch of their own before (us: one token of 150144 x 1536, 922 MB, 143 and
// here 167; 512 tokens of 32003 x 1792, 229 MB, 47 and 46).
constexpr int64_t kLarge = (int64_t)256 << 20;
constexpr int kFew = 512;
template <int DT, int OUT>
__global__ __launch_bounds__(256) void few_tokens_kernel(const SumArgs a, const void *__restrict__ ids, int wide, int64_t pad) {
  using T = typename Elem<DT>::T;
  using TO = typename Elem<OUT>::T;
  constexpr int NV = DT == KSD_F32 ? 4 : 8;
  __shared__ uint32_t keys[kFew];
  __shared__ uint16_t pos[kFew];
  __shared__ uint8_t first[kFew];
  __shared__ uint16_t list[4][kFew];
  __shared__ float part[4][64][NV];
  __shared__ uint32_t counts[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t grid = gridDim.x, me = blockIdx.x;
  // the tokens of this workgroup's rows in order: thread t looks at positions P t .. P t + P - 1
  constexpr int P = kFew / 256;
  uint32_t k[P];
  bool hit[P];
  int mine = 0;
#pragma unroll
  for (int r = 0; r < P; ++r) {
    const int i = tid * P + r;
    k[r] = i < a.n ? key_of(ids, wide, i, a.V, pad) : (uint32_t)a.V;
    hit[r] = k[r] < a.V && k[r] % grid == me;
    mine += hit[r];
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 63) counts[wave] = incl;
  __syncthreads();
  int at = incl - mine, m = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < wave) at += counts[w];
    m += counts[w];
  }
#pragma unroll
  for (int r = 0; r < P; ++r)
    if (hit[r]) {
      keys[at] = k[r];
      pos[at++] = (uint16_t)(tid * P + r);
    }
  __syncthreads();
  for (int e = tid; e < m; e += 256) {
    bool f = true;
    for (int j = 0; j < e && f; ++j) f = keys[j] != keys[e];
    first[e] = f;
  }
  __syncthreads();
  // this workgroup's columns; its waves stand side by side over them, or share out a token's positions where
  // few columns are left
  const int64_t width = (int64_t)((a.slices + gridDim.y - 1) / gridDim.y) * 64 * NV;
  const int64_t c_lo = blockIdx.y * width, c_hi = min(a.d, c_lo + width);
  const int across = width > 2 * 64 * NV ? 4 : width > 64 * NV ? 2 : 1, shares = 4 / across;
  const int wc = wave % across, ws = wave / across;
  for (int e = 0; e < m; ++e) {
    if (!first[e]) continue;
    const uint32_t key = keys[e];
    int n = 0;  // its positions in order, each wave for itself
    for (int b = e; b < m; b += 64) {
      const bool same = b + lane < m && keys[min(b + lane, m - 1)] == key;
      const uint64_t all = __ballot(same);
      if (same) list[wave][n + __popcll(all & ((1ull << lane) - 1))] = pos[b + lane];
      n += __popcll(all);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int lo = n * ws / shares, hi = n * (ws + 1) / shares;
    for (int64_t cc = c_lo; cc < c_hi; cc += (int64_t)across * 64 * NV) {
      const int64_t c = cc + (wc * 64 + lane) * NV, c0 = max((int64_t)0, min(c, a.d - NV));
      float acc[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) acc[j] = 0.0f;
      for (int b = lo; b < hi; b += 8) {  // 8 rows in flight
        RawCols<DT, NV> v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          v[r].load((const T *)a.g + (int64_t)__builtin_amdgcn_readfirstlane(list[wave][min(b + r, hi - 1)]) * a.stride, c0, a.d);
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (b + r < hi) {
#pragma unroll
            for (int j = 0; j < NV; ++j) acc[j] += v[r].at(j);
          }
      }
      if (shares > 1) {  // added in the order of the shares
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NV; ++j) part[wave][lane][j] = acc[j];
        __syncthreads();
        for (int w = 1; w < shares; ++w)
#pragma unroll
          for (int j = 0; j < NV; ++j) acc[j] += part[w * across + wc][lane][j];
      }
      if (ws == 0 && c < c_hi) put_row<OUT, NV>(a, key, c, c0, acc);
    }
  }
  typedef uint32_t vec __attribute__((ext_vector_type(4), aligned(2)));
  constexpr int NZ = 16 / sizeof(TO);
  for (int64_t v = me + (int64_t)wave * grid; v < a.rows; v += (int64_t)4 * grid) {  // a row per wave
    bool there = false;
    for (int b = 0; b < m && !there; b += 64) there = __ballot(b + lane < m && keys[min(b + lane, m - 1)] == (uint32_t)v) != 0;
    if (there) continue;
    TO *o = (TO *)a.out + v * a.d;
#pragma unroll 4
    for (int64_t c = c_lo + lane * NZ; c < c_hi; c += 64 * NZ) {
      if (c + NZ <= c_hi) {
        __builtin_nontemporal_store((vec){0, 0, 0, 0}, (vec *)(o + c));
      } else {
        for (int64_t j = c; j < c_hi; ++j) o[j] = (TO)0;
      }
    }
  }
}

__global__ __launch_bounds__(256) void fill_kernel(const Fill f) { fill(f, blockIdx.x); }

// Rounds of a tile: short tiles spread few keys over the CUs, long ones keep the tiles few whose counts every
// workgroup adds up. (942 x 93, us, 4 and 16 rounds: 131072 tokens 51 and 62, 262144 80 and 80, 524288 136 and
// 114, 2^20 407 and 209.)
static int rounds_of(int64_t n) { return n <= 262144 ? 4 : 16; }

static void digits(int64_t V, int &passes, int &bits) {  // keys are 0 .. V
  int all = 1;
  while (all < 32 && (V >> all)) ++all;
  passes = (all + 8) / 9;
  bits = (all + passes - 1) / passes;
}
// Short chunks where few rows would leave CUs idle. (942 x 93, us, 16 and 32: 3000 tokens 22 and 25, 8192 23
// and 25.5; 32003 x 1792, 16384 tokens, a fifth of them equal: 87 and 74.)
static int run_of(int64_t n) { return n <= 8192 ? 16 : 32; }

struct Layout {
  int64_t keys[2], pos[2], counts, parts, bytes;
};
static Layout layout(int64_t n, int64_t d) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t b) {
    const int64_t r = at;
    at += (b + 255) / 256 * 256;
    return r;
  };
  for (int i = 0; i < 2; ++i) l.keys[i] = take(n * 4), l.pos[i] = take(n * 4);
  l.counts = take(std::max(cdiv(n, 256 * rounds_of(n)) * kDigits, n <= kOne ? cdiv(n, kOthers) * n : 0) * 4);
  l.parts = take(2 * cdiv(n, run_of(n)) * d * 4);
  l.bytes = at;
  return l;
}

template <int DT>
static void launch_lookup(int out, unsigned g, const void *t, const void *ids, int wide, int64_t n, int64_t V, int64_t d,
                          int64_t stride, float scale, void *y, hipStream_t st) {
  if (out == KSD_F32) lookup_kernel<DT, KSD_F32><<<g, 256, 0, st>>>(t, ids, wide, n, V, d, stride, scale, y);
  else if (out == KSD_BF16) lookup_kernel<DT, KSD_BF16><<<g, 256, 0, st>>>(t, ids, wide, n, V, d, stride, scale, y);
  else lookup_kernel<DT, KSD_F16><<<g, 256, 0, st>>>(t, ids, wide, n, V, d, stride, scale, y);
}
template <int DT, int OUT>
static void launch_few(const SumArgs &a, const SortArgs &s, hipStream_t st) {
  // at most 16 rows of a workgroup where all are written, at least one
  const int64_t some = std::min<int64_t>(a.V, 1024), all = std::max<int64_t>(some, cdiv(a.V, 16));
  const int64_t x = a.rows == 0 ? some : all;
  // columns apart where that gives more workgroups: a frequent token's rows are one workgroup's
  const dim3 g((unsigned)x, (unsigned)std::max<int64_t>(1, std::min<int64_t>(a.slices, 2048 / x)));
  few_tokens_kernel<DT, OUT><<<g, 256, 0, st>>>(a, s.ids, s.wide, s.pad);
}
template <int DT>
static void launch_few(int out, const SumArgs &a, const SortArgs &s, hipStream_t st) {
  if (out == KSD_F32) launch_few<DT, KSD_F32>(a, s, st);
  else if (out == KSD_BF16) launch_few<DT, KSD_BF16>(a, s, st);
  else launch_few<DT, KSD_F16>(a, s, st);
}
template <int DT, int OUT>
static void launch_sums(SumArgs a, hipStream_t st) {
  a.sums = (unsigned)cdiv((int64_t)a.chunks * a.slices, 4);
  sum_kernel<DT, OUT><<<a.sums + (unsigned)cdiv(a.rows, kGap), 256, 0, st>>>(a);
  if (a.chunks > 1)
    join_kernel<OUT><<<dim3((unsigned)cdiv(a.chunks, kJoin), (unsigned)cdiv(a.d, 256)), 64 * kJoin, 0, st>>>(a);
}

static bool float_type(int t) { return t == KSD_F32 || t == KSD_BF16 || t == KSD_F16; }

}  // namespace emb
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_embedding_lookup(const void *table, int table_dtype, int64_t V, int64_t d, int64_t stride, const void *ids,
                                    int ids_wide, int64_t n, float scale, void *out, int out_dtype, void *stream) {
  if (n < 0 || V < 0 || d < 0 || stride < d) return fail(KSD_EINVAL, "embedding_lookup: bad shape");
  if (!emb::float_type(table_dtype) || !emb::float_type(out_dtype))
    return fail(KSD_ETYPE, "embedding_lookup: unsupported element type");
  if (n == 0 || d == 0) return KSD_OK;
  if (V == 0) return fail(KSD_EINVAL, "embedding_lookup: ids into an empty table");
  if (!table || !ids || !out) return fail(KSD_EINVAL, "embedding_lookup: null pointer");
  if (!grid_fits(cdiv(n, 4), 256)) return fail(KSD_EINVAL, "embedding_lookup: too many ids");
  const unsigned g = (unsigned)cdiv(n, 4);
  hipStream_t st = (hipStream_t)stream;
  switch (table_dtype) {
    case KSD_F32: emb::launch_lookup<KSD_F32>(out_dtype, g, table, ids, ids_wide, n, V, d, stride, scale, out, st); break;
    case KSD_BF16: emb::launch_lookup<KSD_BF16>(out_dtype, g, table, ids, ids_wide, n, V, d, stride, scale, out, st); break;
    default: emb::launch_lookup<KSD_F16>(out_dtype, g, table, ids, ids_wide, n, V, d, stride, scale, out, st);
  }
  return check_launch("embedding_lookup");
}

extern "C" int ksd_embedding_gradient_workspace(int64_t n, int64_t d, int64_t *bytes) {
  if (n < 0 || d < 0 || !bytes) return fail(KSD_EINVAL, "embedding_gradient_workspace: bad arguments");
  *bytes = emb::layout(n, d).bytes;
  return KSD_OK;
}

extern "C" int ksd_embedding_gradient(const void *g, int g_dtype, int64_t n, int64_t d, int64_t stride, const void *ids,
                                      int ids_wide, int64_t V, int64_t padding, float scale, int accumulate, void *out,
                                      int out_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  if (n < 0 || V < 0 || d < 0 || (n > 0 && stride < d)) return fail(KSD_EINVAL, "embedding_gradient: bad shape");
  if (!emb::float_type(g_dtype) || !emb::float_type(out_dtype))
    return fail(KSD_ETYPE, "embedding_gradient: unsupported element type");
  if (n > 0x7fffffff - 65536 || V > 0x7ffffffe) return fail(KSD_EINVAL, "embedding_gradient: more than 2^31 ids or rows");
  if (V == 0 || d == 0) return KSD_OK;
  if (!out) return fail(KSD_EINVAL, "embedding_gradient: null pointer");
  if (((uintptr_t)out) % 16) return fail(KSD_EINVAL, "embedding_gradient: out must be 16-byte aligned");
  if (cdiv(d, 256) > 65535) return fail(KSD_EINVAL, "embedding_gradient: rows too long");
  const emb::Layout l = emb::layout(n, d);
  if (n > 0 && (!g || !ids || !workspace || workspace_bytes < l.bytes))
    return fail(KSD_EINVAL, "embedding_gradient: null pointer or short workspace");
  const int run = emb::run_of(n), vec = g_dtype == KSD_F32 ? 4 : 8, es = out_dtype == KSD_F32 ? 4 : 2;
  const int64_t chunks = cdiv(n, run), slices = cdiv(d, 64 * vec);
  if (!grid_fits(cdiv(chunks * slices, 4) + cdiv(V, emb::kGap), 256)) return fail(KSD_EINVAL, "embedding_gradient: too many ids");
  hipStream_t st = (hipStream_t)stream;
  const emb::Fill f{(char *)out, V * d * es};
  if (n == 0) {
    if (accumulate) return KSD_OK;
    if (!grid_fits(emb::fill_blocks(f), 256)) return fail(KSD_EINVAL, "embedding_gradient: table too large");
    emb::fill_kernel<<<(unsigned)emb::fill_blocks(f), 256, 0, st>>>(f);
    return check_launch("embedding_gradient");
  }
  char *w = (char *)workspace;
  emb::SortArgs s{};
  s.ids = ids, s.V = V, s.pad = padding, s.n = (int)n, s.wide = ids_wide;
  s.counts = (uint32_t *)(w + l.counts);
  emb::SumArgs a{nullptr, nullptr, g, out, (float *)(w + l.parts), d, stride, V, accumulate ? 0 : V,
                 (int)n, (int)chunks, run, (int)slices, accumulate, 0, scale};
  if (n <= emb::kFew) {
    if (!accumulate && V * d * es > emb::kLarge && grid_fits(emb::fill_blocks(f), 256)) {
      emb::fill_kernel<<<(unsigned)emb::fill_blocks(f), 256, 0, st>>>(f);
      a.rows = 0;
    }
    if (g_dtype == KSD_F32) emb::launch_few<KSD_F32>(out_dtype, a, s, st);
    else if (g_dtype == KSD_BF16) emb::launch_few<KSD_BF16>(out_dtype, a, s, st);
    else emb::launch_few<KSD_F16>(out_dtype, a, s, st);
    return check_launch("embedding_gradient");
  }
  int at = 0;
  if (n <= emb::kOne && V < (1 << 19)) {
    s.out_keys = (uint32_t *)(w + l.keys[0]), s.out_pos = (int32_t *)(w + l.pos[0]);
    const unsigned counting = (unsigned)(n <= emb::kPlace ? cdiv(n, 64) : cdiv(n, 256) * cdiv(n, emb::kOthers));
    const bool blind = !accumulate && grid_fits(emb::fill_blocks(f) + counting, 256);
    if (blind) a.rows = 0;
    const unsigned clear = blind ? (unsigned)emb::fill_blocks(f) : 0;
    if (n <= emb::kPlace) {
      emb::rank_place_kernel<<<counting + clear, 256, 0, st>>>(s, counting, f);
    } else {
      emb::rank_count_kernel<<<counting + clear, 256, 0, st>>>(s, counting, f);
      emb::rank_scatter_kernel<<<(unsigned)cdiv(n, 256), 256, 0, st>>>(s);
    }
  } else {
    const int rounds = emb::rounds_of(n);
    int passes;
    emb::digits(V, passes, s.bits);
    s.tiles = (int)cdiv(n, 256 * rounds);
    // Where few rows have a token, clearing beside the sort costs less than in the sums' launch (us, uniform
    // tokens: 150144 x 1536, 12000 tokens 185 and 198; 32003 x 1792, 12000 tokens 80 and 66).
    const bool blind = !accumulate && n <= V / 4 && grid_fits(emb::fill_blocks(f) + s.tiles, 256);
    if (blind) a.rows = 0;
    for (int p = 0; p < passes; ++p, at ^= 1) {
      if (p > 0) s.ids = nullptr;
      s.keys = (uint32_t *)(w + l.keys[at ^ 1]), s.pos = (int32_t *)(w + l.pos[at ^ 1]);
      s.out_keys = (uint32_t *)(w + l.keys[at]), s.out_pos = (int32_t *)(w + l.pos[at]);
      s.shift = p * s.bits;
      const int64_t clear = blind && p == 0 ? emb::fill_blocks(f) : 0;
      if (rounds == 4) {
        emb::sort_count_kernel<4><<<(unsigned)(s.tiles + clear), 256, 0, st>>>(s, f);
        emb::sort_scatter_kernel<4><<<s.tiles, 256, 0, st>>>(s);
      } else {
        emb::sort_count_kernel<16><<<(unsigned)(s.tiles + clear), 256, 0, st>>>(s, f);
        emb::sort_scatter_kernel<16><<<s.tiles, 256, 0, st>>>(s);
      }
    }
    at ^= 1;  // the last pass's output
  }
  a.keys = (uint32_t *)(w + l.keys[at]), a.pos = (int32_t *)(w + l.pos[at]);
#define KSD_SUMS(DT)                                                        \
  if (out_dtype == KSD_F32) emb::launch_sums<DT, KSD_F32>(a, st);           \
  else if (out_dtype == KSD_BF16) emb::launch_sums<DT, KSD_BF16>(a, st);    \
  else emb::launch_sums<DT, KSD_F16>(a, st);
  switch (g_dtype) {
    case KSD_F32: KSD_SUMS(KSD_F32) break;
    case KSD_BF16: KSD_SUMS(KSD_BF16) break;
    default: KSD_SUMS(KSD_F16)
  }
#undef KSD_SUMS
  return check_launch("embedding_gradient");
}
