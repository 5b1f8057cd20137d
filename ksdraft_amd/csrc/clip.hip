// Global norm of many gradient tensors, and their clipping:
//
//   norm = sqrt(sum of all g^2) / loss_scale   (or max |g| / loss_scale)
//   factor = min(1, max_norm / (norm + 1e-6)) / loss_scale,   g' = g * factor
//
// Squares and their sums are fp64: an fp32 gradient's square neither overflows nor underflows there,
// and at one fma per element the fp64 pipe keeps up with memory. The partial sums of a fixed
// assignment of chunks to workgroups are added in a fixed order: repeated calls give the same bits.
#include "ksd_common.h"

#include <stdlib.h>

#include <algorithm>

namespace ksd {
namespace clip {

constexpr int kBatch = 96;     // tensors of a launch (their descriptors are its arguments)
constexpr int kChunk = 16384;  // elements of a chunk
constexpr int kGrid = 1024;    // workgroups of a launch, at most

struct Tensor {
  const void *g;
  void *out;
  int64_t n;
  int32_t first, type;  // first chunk; element type
};
struct Batch {
  Tensor t[kBatch];
  int n, chunks;
};

__device__ __forceinline__ const Tensor &tensor_of(const Batch &b, int chunk) {
  int lo = 0, hi = b.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (b.t[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return b.t[lo];
}

template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T *p, float *v) {
  struct __attribute__((packed, aligned(DT == KSD_F32 ? 4 : 2))) Any { uint4 q; };
  Raw8<DT> r;
  r.a = ((const Any *)p)->q;
  if constexpr (DT == KSD_F32) r.b = ((const Any *)(p + 4))->q;
  cvt_raw8<DT>(r, true, v);
}

template <int DT, bool MAX>
__device__ __forceinline__ void chunk_norm(const Tensor &t, int64_t e0, double &sum, uint32_t &top) {
  using T = typename Elem<DT>::T;
  const T *g = (const T *)t.g;
  const int64_t e1 = min(t.n, e0 + kChunk);
  for (int64_t e = e0 + threadIdx.x * 8; e < e1; e += 2048) {
    float v[8];
    if (e + 8 <= e1) {
      load8<DT>(g + e, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = e + j < e1 ? Elem<DT>::load(g + e + j) : 0.0f;
    }
    if constexpr (MAX) {
      top = max(top, __builtin_bit_cast(uint32_t, abs_max<8>(v)));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma((double)v[j], (double)v[j], sum);
    }
  }
}

// Bound by one read of the gradients. (509 fp32 tensors, 2.97 GB: 532 us, 5.6 TB/s.)
template <bool MAX>
__global__ __launch_bounds__(256) void norm_kernel(const Batch b, double *__restrict__ parts) {
  double sum = 0.0;
  uint32_t top = 0;
  for (int c = blockIdx.x; c < b.chunks; c += gridDim.x) {
    const Tensor &t = tensor_of(b, c);
    const int64_t e0 = (int64_t)(c - t.first) * kChunk;
    if (t.type == KSD_F32) chunk_norm<KSD_F32, MAX>(t, e0, sum, top);
    else if (t.type == KSD_BF16) chunk_norm<KSD_BF16, MAX>(t, e0, sum, top);
    else chunk_norm<KSD_F16, MAX>(t, e0, sum, top);
  }
  if constexpr (MAX) sum = (double)__builtin_bit_cast(float, top);
  __shared__ double s[256];
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) {
      const double x = s[threadIdx.x], y = s[threadIdx.x + o];
      s[threadIdx.x] = MAX ? (x != x || x > y ? x : y) : x + y;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) parts[blockIdx.x] = s[0];
}

template <bool MAX>
__global__ __launch_bounds__(1024) void fold_kernel(const double *__restrict__ parts, int n, float max_norm, float loss_scale,
                                                    float *__restrict__ norm, float *__restrict__ factor) {
  __shared__ double s[1024];
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const double y = parts[i];
    sum = MAX ? (sum != sum || sum > y ? sum : y) : sum + y;
  }
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) {
      const double x = s[threadIdx.x], y = s[threadIdx.x + o];
      s[threadIdx.x] = MAX ? (x != x || x > y ? x : y) : x + y;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float total = (float)((MAX ? s[0] : sqrt(s[0])) / (double)loss_scale);
    norm[0] = total;
    if (factor) {
      float c = max_norm / (total + 1e-6f);
      c = c > 1.0f ? 1.0f : c;  // a NaN norm stays
      factor[0] = c / loss_scale;
    }
  }
}

template <int DT>
__device__ __forceinline__ void chunk_scale(const Tensor &t, int64_t e0, float f) {
  using T = typename Elem<DT>::T;
  const T *g = (const T *)t.g;
  T *o = (T *)t.out;
  const int64_t e1 = min(t.n, e0 + kChunk);
  for (int64_t e = e0 + threadIdx.x * 8; e < e1; e += 2048) {
    float v[8];
    if (e + 8 <= e1) {
      load8<DT>(g + e, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
      struct __attribute__((packed, aligned(DT == KSD_F32 ? 4 : 2))) Any { uint32_t w[4]; };
      Any *q = (Any *)(o + e);
      if constexpr (DT == KSD_F32) {
        Any a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) a.w[j] = __builtin_bit_cast(uint32_t, v[j]), b.w[j] = __builtin_bit_cast(uint32_t, v[4 + j]);
        q[0] = a, q[1] = b;
      } else {
        Any a;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint16_t lo, hi;
          store_out<DT>(&lo, 0, v[2 * k]);
          store_out<DT>(&hi, 0, v[2 * k + 1]);
          a.w[k] = lo | (uint32_t)hi << 16;
        }
        q[0] = a;
      }
    } else {
      for (int j = 0; j < 8 && e + j < e1; ++j) store_out<DT>(o, e + j, Elem<DT>::load(g + e + j) * f);
    }
  }
}

// Bound by a read and a write of the gradients. (The same tensors: 1190 us, 5.0 TB/s; a large copy 4.9.)
__global__ __launch_bounds__(256) void scale_kernel(const Batch b, const float *__restrict__ factor) {
  const float f = factor[0];
  for (int c = blockIdx.x; c < b.chunks; c += gridDim.x) {
    const Tensor &t = tensor_of(b, c);
    if (f == 1.0f && t.g == t.out) continue;  // in place, nothing to change
    const int64_t e0 = (int64_t)(c - t.first) * kChunk;
    if (t.type == KSD_F32) chunk_scale<KSD_F32>(t, e0, f);
    else if (t.type == KSD_BF16) chunk_scale<KSD_BF16>(t, e0, f);
    else chunk_scale<KSD_F16>(t, e0, f);
  }
}

// Calls launch(batch, grid) for batches of the tensors, from the last to the first with `back`.
struct List {
  const void *const *grads;
  void *const *outs;
  const int64_t *sizes;
  const int32_t *types;
  int n;
};
template <class F>
static void batches(const List &l, bool back, F launch) {
  Batch b;
  b.n = b.chunks = 0;
  for (int k = 0; k < l.n; ++k) {
    const int i = back ? l.n - 1 - k : k;
    if (l.sizes[i] == 0) continue;
    const int64_t chunks = cdiv(l.sizes[i], kChunk);
    if (b.n == kBatch || b.chunks + chunks > 0x7fffffff) {
      launch(b, std::min(b.chunks, kGrid));
      b.n = b.chunks = 0;
    }
    b.t[b.n++] = Tensor{l.grads[i], l.outs ? l.outs[i] : nullptr, l.sizes[i], b.chunks, l.types[i]};
    b.chunks += (int)chunks;
  }
  if (b.n) launch(b, std::min(b.chunks, kGrid));
}

static int check(const List &l, const char *who, bool out) {
  if (l.n < 0 || (l.n > 0 && (!l.grads || !l.sizes || !l.types || (out && !l.outs))))
    return fail(KSD_EINVAL, "%s: bad tensor list", who);
  for (int i = 0; i < l.n; ++i) {
    if (l.sizes[i] < 0 || l.sizes[i] > (int64_t)kChunk * 0x7fffffff) return fail(KSD_EINVAL, "%s: tensor %d: bad size", who, i);
    if (l.types[i] != KSD_F32 && l.types[i] != KSD_BF16 && l.types[i] != KSD_F16)
      return fail(KSD_ETYPE, "%s: tensor %d: unsupported element type %d", who, i, l.types[i]);
    if (l.sizes[i] > 0 && (!l.grads[i] || (out && !l.outs[i]))) return fail(KSD_EINVAL, "%s: tensor %d: null pointer", who, i);
  }
  return KSD_OK;
}

// Two workgroups must not write one element, nor one read what another writes: an output's memory may meet
// its own gradient's only where both are the same, and no other tensor's. (392 tensors in any order: 6 us of host in
// place, 14 into other tensors, while the norm runs.)
struct Span {
  uintptr_t lo, hi;
  int i;
};
static int64_t width_of(int type) { return type == KSD_F32 ? 4 : 2; }
static int apart(const List &l, const char *who) {
  Span *const s = (Span *)malloc(sizeof(Span) * (size_t)std::max(l.n, 1));
  if (!s) return fail(KSD_EHIP, "%s: out of host memory", who);
  int n = 0, rc = KSD_OK;
  bool in_place = true;
  for (int i = 0; i < l.n; ++i) {
    if (l.sizes[i] == 0) continue;
    const uintptr_t lo = (uintptr_t)l.outs[i];
    s[n++] = Span{lo, lo + (uintptr_t)(l.sizes[i] * width_of(l.types[i])), i};
    in_place &= l.outs[i] == l.grads[i];
  }
  std::sort(s, s + n, [](const Span &a, const Span &b) { return a.lo < b.lo; });
  for (int k = 1; k < n && !rc; ++k)
    if (s[k].lo < s[k - 1].hi) rc = fail(KSD_EINVAL, "%s: tensors %d and %d are written to the same memory", who, s[k - 1].i, s[k].i);
  for (int i = 0; i < l.n && !rc && !in_place; ++i) {
    if (l.sizes[i] == 0) continue;
    const uintptr_t lo = (uintptr_t)l.grads[i], hi = lo + (uintptr_t)(l.sizes[i] * width_of(l.types[i]));
    const Span *const f = std::upper_bound(s, s + n, lo, [](uintptr_t v, const Span &a) { return v < a.hi; });  // first to end past lo
    if (f < s + n && f->lo < hi && !(f->i == i && f->lo == lo))
      rc = fail(KSD_EINVAL, "%s: output %d lies in the memory of gradient %d", who, f->i, i);
  }
  free(s);
  return rc;
}

}  // namespace clip
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_grad_norm_workspace(const int64_t *sizes, int n, int64_t *bytes) {
  if (!bytes || n < 0 || (n > 0 && !sizes)) return fail(KSD_EINVAL, "grad_norm_workspace: bad arguments");
  // at most kGrid results per launch and one per chunk
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    if (sizes[i] < 0) return fail(KSD_EINVAL, "grad_norm_workspace: tensor %d: bad size", i);
    chunks += cdiv(sizes[i], clip::kChunk);
  }
  const int64_t launches = cdiv(n, clip::kBatch) + chunks / 0x7fffffff + 1;
  *bytes = 8 * std::max<int64_t>(1, std::min(chunks, launches * clip::kGrid));
  return KSD_OK;
}

extern "C" int ksd_grad_norm(const void *const *grads, const int64_t *sizes, const int32_t *types, int n, int max_kind,
                             float max_norm, float loss_scale, float *norm, float *factor, void *workspace,
                             int64_t workspace_bytes, void *stream) {
  const clip::List l{grads, nullptr, sizes, types, n};
  int rc = clip::check(l, "grad_norm", false);
  if (rc) return rc;
  int64_t need = 0;
  rc = ksd_grad_norm_workspace(sizes, n, &need);
  if (rc) return rc;
  if (!norm || !workspace || workspace_bytes < need) return fail(KSD_EINVAL, "grad_norm: null pointer or short workspace");
  hipStream_t st = (hipStream_t)stream;
  double *parts = (double *)workspace;
  int at = 0;
  clip::batches(l, false, [&](const clip::Batch &b, int grid) {
    if (max_kind) clip::norm_kernel<true><<<grid, 256, 0, st>>>(b, parts + at);
    else clip::norm_kernel<false><<<grid, 256, 0, st>>>(b, parts + at);
    at += grid;
  });
  if (max_kind) clip::fold_kernel<true><<<1, 1024, 0, st>>>(parts, at, max_norm, loss_scale, norm, factor);
  else clip::fold_kernel<false><<<1, 1024, 0, st>>>(parts, at, max_norm, loss_scale, norm, factor);
  return check_launch("grad_norm");
}

extern "C" int ksd_grad_scale(const void *const *grads, void *const *outs, const int64_t *sizes, const int32_t *types, int n,
                              const float *factor, void *stream) {
  const clip::List l{grads, outs, sizes, types, n};
  int rc = clip::check(l, "grad_scale", true);
  if (!rc) rc = clip::apart(l, "grad_scale");
  if (rc) return rc;
  if (!factor) return fail(KSD_EINVAL, "grad_scale: null pointer");
  hipStream_t st = (hipStream_t)stream;
  // backwards: the tensors that the norm has read last are still in the last-level cache
  clip::batches(l, true, [&](const clip::Batch &b, int grid) { clip::scale_kernel<<<grid, 256, 0, st>>>(b, factor); });
  return check_launch("grad_scale");
}
