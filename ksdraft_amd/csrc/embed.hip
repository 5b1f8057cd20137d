// Embedding lookup with a scale, and the table's gradient by sorted tokens.
//
//   y[i]  = round(scale * W[id_i])
//   dW[v] = scale * sum of g[i] over the positions i with id_i = v, in the order of i, in fp32
//
// The positions are sorted by token (stable radix sort), so every token's rows are one run of the
// sorted list and no float atomics are needed: the sums have a fixed order and repeated calls give
// the same bits. Runs are cut at multiples of 32 sorted positions, so a token that fills the batch
// is spread over the device like any other; the pieces of a cut run are joined in order.
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

// One wave per row.
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
// Least significant digit first, 8 bits a pass, tiles of 2048 keys. Ids that take no part (the
// padding token, ids out of range) become the key V, which sorts last.
constexpr int kTile = 2048;

__device__ __forceinline__ uint32_t key_of(const void *ids, int wide, int64_t i, int64_t V, int64_t pad) {
  const int64_t id = load_id(ids, wide, i);
  return (uint32_t)(id < 0 || id >= V || id == pad ? V : id);
}

struct SortArgs {
  const void *ids;  // first pass: the ids (positions are the index); later passes: NULL
  const uint32_t *keys;
  const int32_t *pos;
  uint32_t *out_keys;
  int32_t *out_pos;
  uint32_t *counts;  // (256, tiles)
  int64_t V, pad;
  int n, tiles, shift, wide;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, int i) {
  return a.ids ? key_of(a.ids, a.wide, i, a.V, a.pad) : a.keys[i];
}

__global__ __launch_bounds__(256) void sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t h[256];
  const int tid = threadIdx.x, t0 = blockIdx.x * kTile;
  h[tid] = 0;
  __syncthreads();
  for (int i = t0 + tid; i < min(a.n, t0 + kTile); i += 256) atomicAdd(&h[(sort_key(a, i) >> a.shift) & 255], 1u);
  __syncthreads();
  a.counts[tid * a.tiles + blockIdx.x] = h[tid];
}

// exclusive sum over `len` counts, one workgroup
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t *counts, int len) {
  __shared__ uint32_t part[16];
  __shared__ uint32_t carry;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int b = 0; b < len; b += 1024) {
    const uint32_t v = b + tid < len ? counts[b + tid] : 0;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = (uint32_t)__shfl_up((int)s, o);
      if (lane >= o) s += u;
    }
    if (lane == 63) part[tid >> 6] = s;
    __syncthreads();
    uint32_t before = carry;
    for (int w = 0; w < tid >> 6; ++w) before += part[w];
    if (b + tid < len) counts[b + tid] = before + s - v;
    __syncthreads();
    if (tid == 1023) carry = before + s;
    __syncthreads();
  }
}

// Wave w of a tile takes its keys [512 w, 512 w + 512) in 8 rounds of 64, so keys of one digit keep
// their order: rank = earlier tiles' (counts) + earlier waves' + earlier rounds' + lower lanes'.
__global__ __launch_bounds__(256) void sort_scatter_kernel(const SortArgs a) {
  __shared__ uint32_t h[4][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int base = blockIdx.x * kTile + wave * 512;
  for (int w = 0; w < 4; ++w) h[w][tid] = 0;
  __syncthreads();
  uint32_t key[8];
  uint64_t same[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int i = base + r * 64 + lane;
    const bool in = i < a.n;
    key[r] = in ? sort_key(a, i) : 0xffffffffu;
    const uint32_t d = (key[r] >> a.shift) & 255;
    uint64_t m = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t bal = __ballot((d >> b) & 1);
      m &= (d >> b) & 1 ? bal : ~bal;
    }
    same[r] = m;
    if (in && (m & ((1ull << lane) - 1)) == 0) h[wave][d] += (uint32_t)__popcll(m);
  }
  __syncthreads();
  {
    uint32_t at = a.counts[tid * a.tiles + blockIdx.x];
    for (int w = 0; w < 4; ++w) {
      const uint32_t c = h[w][tid];
      h[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int i = base + r * 64 + lane;
    const uint32_t d = (key[r] >> a.shift) & 255;
    uint32_t first = 0;
    if (i < a.n) {
      first = h[wave][d];
      const uint32_t to = first + (uint32_t)__popcll(same[r] & ((1ull << lane) - 1));
      a.out_keys[to] = key[r];
      a.out_pos[to] = a.ids ? i : a.pos[i];
    }
    __builtin_amdgcn_wave_barrier();
    if (i < a.n && (same[r] & ((1ull << lane) - 1)) == 0) h[wave][d] = first + (uint32_t)__popcll(same[r]);
    __builtin_amdgcn_wave_barrier();
  }
}

// ------------------------------------------------------------------------------------ sums
constexpr int kRun = 32;  // sorted positions of a chunk

struct SumArgs {
  const uint32_t *keys;
  const int32_t *pos;
  const void *g;
  void *out;
  float *parts;  // (2, chunks, d): the piece of the run that a chunk begins in, and the one it ends in
  int64_t d, stride, V;
  int n, chunks, add;
  float scale;
};

template <int OUT>
__device__ __forceinline__ void put_row(const SumArgs &a, uint32_t key, int64_t c, int m, const float *acc) {
  typename Elem<OUT>::T *o = (typename Elem<OUT>::T *)a.out + (int64_t)key * a.d + c;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = acc[j] * a.scale;
  if (a.add) {
    float was[8];
    load_any<OUT>(o, m, was);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = was[j] + v[j];
  }
  store_any<OUT>(o, m, v);
}

// Chunk blockIdx.x, columns blockIdx.y * 2048 + 8 tid ..: sums its runs in order. A run that lies in
// the chunk is finished; the pieces of runs that reach past it go to parts.
template <int DT, int OUT>
__global__ __launch_bounds__(256) void sum_kernel(const SumArgs a) {
  using T = typename Elem<DT>::T;
  const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  if (c >= a.d) return;
  const int m = (int)min((int64_t)8, a.d - c);
  const int b = blockIdx.x, s0 = b * kRun, s1 = min(a.n, s0 + kRun);
  const T *g = (const T *)a.g + c;
  uint32_t key = a.keys[s0];
  bool whole = b == 0 || a.keys[s0 - 1] != key;  // the run begins in this chunk
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  auto part = [&](int which) {
    float *o = a.parts + ((int64_t)which * a.chunks + b) * a.d + c;
    store_any<KSD_F32>(o, m, acc);
  };
  for (int s = s0; s < s1; ++s) {
    const uint32_t k = a.keys[s];
    if (k != key) {
      if (whole) put_row<OUT>(a, key, c, m, acc);
      else part(0);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
      key = k;
      whole = true;
    }
    if (k >= a.V) return;  // ids that take no part sort last
    float v[8];
    load_any<DT>(g + (int64_t)a.pos[s] * a.stride, m, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
  if (!whole) part(0);
  else if (s1 < a.n && a.keys[s1] == key) part(1);
  else put_row<OUT>(a, key, c, m, acc);
}

// Joins the pieces of the run that begins in chunk blockIdx.x and reaches past it.
template <int OUT>
__global__ __launch_bounds__(256) void join_kernel(const SumArgs a) {
  const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  const int b = blockIdx.x, s0 = b * kRun, s1 = s0 + kRun;
  if (c >= a.d || s1 >= a.n) return;
  const uint32_t key = a.keys[s1 - 1];
  if (key >= a.V || a.keys[s1] != key) return;
  if (a.keys[s0] == key && b > 0 && a.keys[s0 - 1] == key) return;  // it began earlier
  const int m = (int)min((int64_t)8, a.d - c);
  float acc[8], v[8];
  load_any<KSD_F32>(a.parts + ((int64_t)a.chunks + b) * a.d + c, m, acc);
  for (int q = b + 1; q < a.chunks && a.keys[q * kRun] == key; ++q) {
    load_any<KSD_F32>(a.parts + (int64_t)q * a.d + c, m, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] += v[j];
  }
  put_row<OUT>(a, key, c, m, acc);
}

__global__ __launch_bounds__(256) void fill_kernel(uint4 *p, int64_t n16, char *tail, int ntail) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256)
    p[i] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x == 0 && (int)threadIdx.x < ntail) tail[threadIdx.x] = 0;
}

static int passes(int64_t V) {
  int bits = 1;
  while (bits < 32 && (V >> bits)) ++bits;
  return (bits + 7) / 8;
}

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
  l.counts = take(cdiv(n, kTile) * 256 * 4);
  l.parts = take(2 * cdiv(n, kRun) * d * 4);
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
static void launch_sums(const SumArgs &a, hipStream_t st) {
  const dim3 g((unsigned)a.chunks, (unsigned)cdiv(a.d, 2048));
  sum_kernel<DT, OUT><<<g, 256, 0, st>>>(a);
  if (a.chunks > 1) join_kernel<OUT><<<g, 256, 0, st>>>(a);
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
  if (n > 0x7fffffff - emb::kTile || V > 0x7ffffffe) return fail(KSD_EINVAL, "embedding_gradient: more than 2^31 ids or rows");
  if (V == 0 || d == 0) return KSD_OK;
  if (!out) return fail(KSD_EINVAL, "embedding_gradient: null pointer");
  if (((uintptr_t)out) % 16) return fail(KSD_EINVAL, "embedding_gradient: out must be 16-byte aligned");
  if (cdiv(d, 2048) > 65535) return fail(KSD_EINVAL, "embedding_gradient: rows too long");
  const emb::Layout l = emb::layout(n, d);
  if (n > 0 && (!g || !ids || !workspace || workspace_bytes < l.bytes))
    return fail(KSD_EINVAL, "embedding_gradient: null pointer or short workspace");
  hipStream_t st = (hipStream_t)stream;
  if (!accumulate) {
    const int64_t bytes = V * d * (out_dtype == KSD_F32 ? 4 : 2), n16 = bytes / 16;
    emb::fill_kernel<<<(unsigned)std::max<int64_t>(1, std::min<int64_t>(cdiv(n16, 256 * 8), 1 << 20)), 256, 0, st>>>(
        (uint4 *)out, n16, (char *)out + n16 * 16, (int)(bytes % 16));
  }
  if (n == 0) return check_launch("embedding_gradient");
  char *w = (char *)workspace;
  emb::SortArgs s{};
  s.counts = (uint32_t *)(w + l.counts);
  s.V = V, s.pad = padding, s.n = (int)n, s.tiles = (int)cdiv(n, emb::kTile), s.wide = ids_wide;
  int at = 0;
  for (int p = 0; p < emb::passes(V); ++p, at ^= 1) {
    s.ids = p == 0 ? ids : nullptr;
    s.keys = (uint32_t *)(w + l.keys[at ^ 1]), s.pos = (int32_t *)(w + l.pos[at ^ 1]);
    s.out_keys = (uint32_t *)(w + l.keys[at]), s.out_pos = (int32_t *)(w + l.pos[at]);
    s.shift = p * 8;
    emb::sort_count_kernel<<<s.tiles, 256, 0, st>>>(s);
    emb::sort_scan_kernel<<<1, 1024, 0, st>>>(s.counts, s.tiles * 256);
    emb::sort_scatter_kernel<<<s.tiles, 256, 0, st>>>(s);
  }
  at ^= 1;  // the last pass's output
  emb::SumArgs a{(uint32_t *)(w + l.keys[at]), (int32_t *)(w + l.pos[at]), g, out, (float *)(w + l.parts), d, stride, V,
                 (int)n, (int)cdiv(n, emb::kRun), accumulate, scale};
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
