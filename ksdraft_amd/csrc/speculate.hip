// Verification of drafted tokens against the target's logits, and drawing a token from logits, from given
// random numbers. With p = softmax(z / T) of a target row and q that of the draft's:
//
//   position t is accepted while u[t] q(token) < p(token)       (no draft logits: q(token) = 1)
//   the first refused one, or the one behind the last, draws the first token whose running sum of
//   weights passes u[L] times their sum: weights max(p - q, 0), or p where nothing was refused
//   T = 0: accepted while the token is the row's largest logit (the lowest index of equal ones), which is drawn too
//
// One read of the rows gives each row's largest logit and sum of powers in 32 bits (stats_kernel): the tests
// need p and q of one token a row. A power's exponent y is rounded three times and the power once, and a sum of 150144 is
// about 40 roundings deep: with |y| 17 on average at most (log2 of the vocabulary) a sum is off by less than 100 * 2^-24 =
// 6e-6 of itself, by 1e-7 or so where the roundings are as random as they look. That moves one test in a hundred
// thousand at the worst, whose u lies so near its border. The drawn token is
// another matter: with 150144 tokens a running sum has as many borders, and sums in 32 bits would move about one draw in
// a hundred across one. The one row of a stream that is drawn from is therefore read again with powers and sums in 64
// bits (total_kernel, weight_kernel, draw_kernel). Logits of -inf have probability 0. A row with NaN or +inf has no
// distribution (greedy: with NaN, +inf is a largest logit like any other), a target's without a finite logit neither: a
// target's refuses its token and draws -1, a draft's refuses the token and draws from p. A draft's row of nothing but
// -inf is q = 0: its token is accepted wherever p > 0.
#include "ksd_common.h"

#include <float.h>

#include <algorithm>

namespace ksd {
namespace spec {

struct Part {  // of a row's piece: largest logit, sum of 2^((z - m) c); greedy: largest logit (NaN where there is one), its place
  float m;
  int at;
  double s;
};

struct Args {
  const void *target, *draft;  // (B, L + 1, V), (B, L, V) or NULL
  int64_t tb, tt, db, dt;      // strides in elements
  const int64_t *tokens;       // (B, L)
  const void *uniforms;        // (B, L + 1)
  int wide;                    // uniforms are fp64
  const float *temps;          // (B,) or NULL (`temp`)
  float temp;
  const int64_t *lengths;      // (B,) or NULL (L)
  int64_t *out, *accepted;
  Part *parts;                 // (B, 2 L + 1, splits): target rows, then draft rows
  double *totals, *weights;    // (B, pieces, 2) each
  struct Draw *draws;          // (B,)
  int *refused;                // (kRanges, B): the first refused position, as far as the ranges before one tell
  int B, L, V, splits, chunk, pieces, piece;
  int range, t0, t1, before;   // positions of this launch of stats_kernel, and where its predecessor's began
  int exact;                   // stats_kernel's sums are 64-bit already
};
constexpr int kRanges = 6, kNone = 0x7fffffff, kHeld = 4;
// Logits from which positions go in several launches, and of the first of them
constexpr int64_t kSeveral = 64 << 20, kFirst = 40 << 20, kFew = 12 << 20;

__device__ __forceinline__ float temperature(const Args &a, int b) { return a.temps ? a.temps[b] : a.temp; }
__device__ __forceinline__ float clamped(float t) { return fminf(fmaxf(t, 1e-37f), 1e37f); }
__device__ __forceinline__ int length(const Args &a, int b) {
  return a.lengths ? (int)min(max(a.lengths[b], (int64_t)0), (int64_t)a.L) : a.L;
}
__device__ __forceinline__ double uniform(const Args &a, int b, int t) {
  const int64_t i = (int64_t)b * (a.L + 1) + t;
  return a.wide ? ((const double *)a.uniforms)[i] : (double)((const float *)a.uniforms)[i];
}
template <int DT>
__device__ __forceinline__ const typename Elem<DT>::T *target_row(const Args &a, int b, int t) {
  return (const typename Elem<DT>::T *)a.target + b * a.tb + t * a.tt;
}
template <int DT>
__device__ __forceinline__ const typename Elem<DT>::T *draft_row(const Args &a, int b, int t) {
  return (const typename Elem<DT>::T *)a.draft + b * a.db + t * a.dt;
}
__device__ __forceinline__ const Part *parts_of(const Args &a, int b, int row) {
  return a.parts + ((int64_t)b * (2 * a.L + 1) + row) * a.splits;
}

// 8 logits of a row from column c on, -inf from column n on.
template <int DT>
__device__ __forceinline__ void load_logits(const typename Elem<DT>::T *row, int c, int n, float *v) {
  load_any<DT>(row + c, min(n - c, 8), v);
  if (c + 8 > n) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < n ? v[j] : -INFINITY;
  }
}

// ------------------------------------------------------------------------------- powers
// 2^y in 64 bits for y <= 0: 2^k times the Taylor polynomial of e^(r ln 2), |r| <= 1/2, to the 11th power, whose rest
// is below 9e-15 of it, roundings included. NaN stays NaN; below 2^-1100 it is 0. (About 20 instructions for each of the two rows' logits,
// twice; with the library's exp the two launches took 24 and 30 us for 64 streams of 150144 tokens.)
__device__ __forceinline__ double power2(double y) {
  y = y < -1100.0 ? -1100.0 : y;
  const double k = __builtin_rint(y), r = y - k;
  constexpr double l = 0.693147180559945309417232121458;
  constexpr double c1 = l, c2 = c1 * l / 2, c3 = c2 * l / 3, c4 = c3 * l / 4, c5 = c4 * l / 5, c6 = c5 * l / 6, c7 = c6 * l / 7,
                   c8 = c7 * l / 8, c9 = c8 * l / 9, c10 = c9 * l / 10, c11 = c10 * l / 11;
  double p = fma(c11, r, c10);
  p = fma(p, r, c9);
  p = fma(p, r, c8);
  p = fma(p, r, c7);
  p = fma(p, r, c6);
  p = fma(p, r, c5);
  p = fma(p, r, c4);
  p = fma(p, r, c3);
  p = fma(p, r, c2);
  p = fma(p, r, c1);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)k);
}
constexpr double kLog2e = 1.44269504088896340735992468100189214;
// e^((z - m) / T) = power2((z - m) c), c = log2(e) / T; the difference first, which is 0 at the largest logit at any T
struct Exponent {
  double c, m;
};
__device__ __forceinline__ Exponent exponent(float T, float m) { return Exponent{kLog2e / (double)clamped(T), (double)m}; }
__device__ __forceinline__ double power(double z, Exponent e) { return power2((z - e.m) * e.c); }

// ------------------------------------------------------------------------------- reductions
struct Best {
  float m;
  int at;
};
__device__ __forceinline__ Best better(Best x, Best y) {
  return y.m > x.m || (y.m == x.m && y.at < x.at) ? y : x;
}
__device__ __forceinline__ double block_sum(double v, double *scratch) {  // 256 threads
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}
__device__ __forceinline__ float block_max(float v, float *scratch) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3]));
}

// The largest logit of a piece of a row (greedy streams).
template <int DT>
__device__ __forceinline__ void best_part(const typename Elem<DT>::T *row, int from, int to, Part *out) {
  __shared__ Best found[4];
  Best best{-INFINITY, kNone};
  bool bad = false;
  for (int k = from + threadIdx.x * 8; k < to; k += 2048) {
    float v[8];
    load_logits<DT>(row, k, to, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad |= v[j] != v[j];
      if (v[j] > best.m) best = Best{v[j], k + j};
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) best = better(best, Best{__shfl_xor(best.m, o), __shfl_xor(best.at, o)});
  if (__ballot(bad)) best.m = NAN;
  if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) best = best.m != best.m || found[w].m != found[w].m ? Best{NAN, 0} : better(best, found[w]);
    *out = Part{best.m, best.at, 0.0};
  }
}

// ------------------------------------------------------------------------------- acceptance
// What 16 lanes make of a row's pieces (at most 32): every lane gets the result.
struct Stat {
  float m;
  double s;
};
__device__ __forceinline__ Stat row_stat(const Args &a, const Part *p, float T) {
  const int i = threadIdx.x & 15;
  Part x{-FLT_MAX, 0, 0.0}, y = x;
  if (i < a.splits) x = p[i];
  if (i + 16 < a.splits) y = p[i + 16];
  float m = fmaxf(x.m, y.m);
#pragma unroll
  for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  double s;
  if (a.exact) {
    const Exponent e = exponent(T, m);
    s = x.s * power((double)x.m, e) + y.s * power((double)y.m, e);
  } else {
    const float c = 1.4426950408889634f / clamped(T);
    s = x.s * (double)__builtin_amdgcn_exp2f((x.m - m) * c) + y.s * (double)__builtin_amdgcn_exp2f((y.m - m) * c);
  }
#pragma unroll
  for (int o = 8; o; o >>= 1) s += __shfl_xor(s, o);
  return Stat{m, s};
}
// The place of a greedy row's largest logit; -1 where it has none.
__device__ __forceinline__ int row_best(const Args &a, const Part *p, int splits) {
  Best best{-INFINITY, kNone};
  int bad = 0;
  for (int i = threadIdx.x & 15; i < splits; i += 16) {
    const Part x = p[i];
    best = better(best, Best{x.m, x.at}), bad |= x.m != x.m;
  }
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    best = better(best, Best{__shfl_xor(best.m, o), __shfl_xor(best.at, o)});
    bad |= __shfl_xor(bad, o);
  }
  return bad || best.m == -INFINITY ? -1 : best.at;
}

template <int DT>
__device__ __forceinline__ bool accepts(const Args &a, int b, int t, float T) {  // 16 lanes
  const int64_t token = a.tokens[(int64_t)b * a.L + t];
  if (!(T > 0)) return row_best(a, parts_of(a, b, t), a.splits) == token && token >= 0;
  const bool in = token >= 0 && token < a.V;
  const float zp = in ? Elem<DT>::load(target_row<DT>(a, b, t) + token) : 0.0f;
  const float zq = in && a.draft ? Elem<DT>::load(draft_row<DT>(a, b, t) + token) : 0.0f;
  const double u = uniform(a, b, t);
  const Stat p = row_stat(a, parts_of(a, b, t), T);
  const double pt = power((double)zp, exponent(T, p.m)) / p.s;
  double qt = 1.0;
  if (a.draft) {
    const Stat q = row_stat(a, parts_of(a, b, a.L + 1 + t), T);
    qt = q.s == 0 ? 0.0 : power((double)zq, exponent(T, q.m)) / q.s;
  }
  return in && u * qt < pt;
}

// The first refused position in [from, to), else kNone: a workgroup, 16 threads a position.
template <int DT>
__device__ __forceinline__ int refused_in(const Args &a, int b, int from, int to, float T) {
  __shared__ int first;
  if (threadIdx.x == 0) first = kNone;
  __syncthreads();
  for (int base = from; base < to; base += blockDim.x >> 4) {
    const int t = base + (threadIdx.x >> 4);
    if (t < to && !accepts<DT>(a, b, t, T) && (threadIdx.x & 15) == 0) atomicMin(&first, t);
    __syncthreads();
    const int r = first;
    __syncthreads();  // before the next positions' refusals
    if (r != kNone) return r;
  }
  return kNone;
}

// ------------------------------------------------------------------------------- row statistics
// The rows of the positions [t0, t1). A long batch goes through its positions in several launches: a stream's rows
// behind a refused token need not be read, and a launch knows what its predecessors' rows refuse (64 streams, 48 of them
// drawn, 16 drafted tokens of 150144 with their logits, 93% of them accepted: a whole call 185 us with one launch, 147 with
// three, by 6 pieces a row). What bounds it is memory and a workgroup's start and end: the three launches take 97 us at 4
// pieces a row, the first one's 101 MB 28.5 us, 3.5 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void stats_kernel(const Args a) {
  // blocks: split fastest, then target and draft, then requests, then positions
  const int split = blockIdx.x % a.splits;
  int i = blockIdx.x / a.splits;
  const int sides = a.draft ? 2 : 1;
  const bool drafted = i % sides;
  i /= sides;
  const int b = i % a.B, t = a.t0 + i / a.B;
  const int len = length(a, b);
  const float T = temperature(a, b);
  const bool greedy = !(T > 0);
  const bool note = a.range > 0 && t == a.t0 && split == 0 && !drafted;  // whose workgroup writes down what was refused
  const bool idle = t > len || (drafted && (t == len || greedy));
  if (idle && !note) return;
  if (a.range > 0) {
    int r = a.range > 1 ? a.refused[(int64_t)(a.range - 1) * a.B + b] : kNone;
    if (r == kNone) r = refused_in<DT>(a, b, a.before, min(a.t0, len), T);
    if (note && threadIdx.x == 0) a.refused[(int64_t)a.range * a.B + b] = r;
    if (r != kNone || idle) return;
  }
  const typename Elem<DT>::T *const row = drafted ? draft_row<DT>(a, b, t) : target_row<DT>(a, b, t);
  const int from = split * a.chunk, to = min(a.V, from + a.chunk);
  Part *const out = const_cast<Part *>(parts_of(a, b, drafted ? a.L + 1 + t : t)) + split;
  if (greedy) {
    best_part<DT>(row, from, to, out);
    return;
  }
  if (a.exact) {  // few rows: their pieces fit the registers
    __shared__ float tops[4];
    __shared__ double scratch[4];
    float v[kHeld][8], m = -FLT_MAX;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int k = from + (u * 256 + threadIdx.x) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = -INFINITY;
      if (k < to) load_logits<DT>(row, k, to, v[u]);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, v[u][j]);
    }
    m = block_max(m, tops);
    const Exponent e = exponent(T, m);
    double s = 0;
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (u * 2048 < a.chunk) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s += power((double)v[u][j], e);
      }
    s = block_sum(s, scratch);
    if (threadIdx.x == 0) *out = Part{m, 0, s};
    return;
  }
  const float c = 1.4426950408889634f / clamped(T);
  __shared__ float sm[4], ss[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int U = 4;
  float m = -FLT_MAX, s = 0.0f;  // not -inf: a piece of nothing but -inf then has differences of -inf and sum 0
  for (int k = from + threadIdx.x * 8; k < to; k += 2048 * U) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u * 2048 < to) {
        load_logits<DT>(row, k + u * 2048, to, v[u]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u][j] = -INFINITY;
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, v[u][j]);
    float sum[U] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[u] += __builtin_amdgcn_exp2f((v[u][j] - top) * c);
    s = s * __builtin_amdgcn_exp2f((m - top) * c) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
    m = top;
  }
  const auto join = [&](float m2, float s2) {
    const float top = fmaxf(m, m2);
    s = s * __builtin_amdgcn_exp2f((m - top) * c) + s2 * __builtin_amdgcn_exp2f((m2 - top) * c);
    m = top;
  };
#pragma unroll
  for (int o = 32; o; o >>= 1) join(__shfl_xor(m, o), __shfl_xor(s, o));
  if (lane == 0) sm[wave] = m, ss[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) join(sm[w], ss[w]);
    *out = Part{m, 0, (double)s};
  }
}

// ------------------------------------------------------------------------------- the drawn token
// What the draw of a stream works on.
struct Draw {
  int at, rest;        // position; whether a refused token's draft row is subtracted
  Exponent p, q;
  double rp, rq;       // reciprocals of the sums of powers, where stats_kernel's sums are 64-bit
  int64_t without;     // the token that is left out (refused, and no draft logits), or -1
};
__device__ __forceinline__ double reciprocal(double s) { return s > 0 ? 1.0 / s : s; }  // an empty draft row: q = 0; NaN stays
// A workgroup tests its stream's tokens; d is in LDS.
template <int DT>
__device__ __forceinline__ void find_draw(const Args &a, int b, float T, Draw &d) {
  const int len = length(a, b);
  int r = a.range > 0 ? a.refused[(int64_t)a.range * a.B + b] : kNone;
  if (r == kNone) r = refused_in<DT>(a, b, a.range > 0 ? a.t0 : 0, len, T);
  const int at = min(r, len);
  if (!(T > 0)) {
    if (threadIdx.x == 0) d.at = at;
  } else if (threadIdx.x < 16) {
    const bool refused = at < len, rest = refused && a.draft;
    const Stat p = row_stat(a, parts_of(a, b, at), T);
    const Stat q = rest ? row_stat(a, parts_of(a, b, a.L + 1 + at), T) : Stat{0.0f, 0.0};
    if (threadIdx.x == 0)
      d = Draw{at, rest, exponent(T, p.m), exponent(T, q.m), 1.0 / p.s, reciprocal(q.s),
               refused && !a.draft ? a.tokens[(int64_t)b * a.L + at] : -1};
  }
  __syncthreads();
}

// Without a draft there is nothing to test: a piece's largest logit and sum of powers in 64 bits at once (150144 fp32
// logits: 3.9 us, the latency of a launch that reads once).
template <int DT>
__global__ __launch_bounds__(256) void sample_kernel(const Args a) {
  const int b = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const float T = temperature(a, b);
  const typename Elem<DT>::T *const row = target_row<DT>(a, b, 0);
  const int from = piece * a.piece, to = min(a.V, from + a.piece);
  if (!(T > 0)) {
    best_part<DT>(row, from, to, a.parts + (int64_t)b * a.pieces + piece);
    return;
  }
  __shared__ float tops[4];
  __shared__ double scratch[4];
  float m = -FLT_MAX, v[8];
  for (int k = from + threadIdx.x * 8; k < to; k += 2048) {
    load_logits<DT>(row, k, to, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, v[j]);
  }
  m = block_max(m, tops);
  const Exponent e = exponent(T, m);
  double s = 0;
  for (int k = from + threadIdx.x * 8; k < to; k += 2048) {
    if (a.piece > 2048) load_logits<DT>(row, k, to, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += power((double)v[j], e);
  }
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) {
    double *const o = a.totals + ((int64_t)b * a.pieces + piece) * 2;
    o[0] = s, o[1] = (double)m;
  }
}

// Sums of e^((z - m) / T) in 64 bits of a piece of the row that is drawn from, target and draft. Each workgroup finds the
// row for itself, a read of its stream's few statistics. (64 streams of 150144 tokens: 24 us, by count about a third of them
// 64-bit arithmetic.)
template <int DT>
__global__ __launch_bounds__(256) void total_kernel(const Args a) {
  const int b = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const float T = temperature(a, b);
  if (!(T > 0) && piece) return;
  __shared__ Draw d;
  __shared__ double scratch[4];
  find_draw<DT>(a, b, T, d);
  if (piece == 0 && threadIdx.x == 0) a.draws[b] = d;
  if (!(T > 0)) return;
  const int from = piece * a.piece, to = min(a.V, from + a.piece);
  double s0 = 0, s1 = 0;
  for (int k = from + threadIdx.x * 8; k < to; k += 2048) {
    float v[8], w[8];
    load_logits<DT>(target_row<DT>(a, b, d.at), k, to, v);
    if (d.rest) load_logits<DT>(draft_row<DT>(a, b, d.at), k, to, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double e = power((double)v[j], d.p);
      if (k + j == d.without) s1 += e;
      else s0 += e;
    }
    if (d.rest) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s1 += power((double)w[j], d.q);
    }
  }
  s0 = block_sum(s0, scratch);
  s1 = block_sum(s1, scratch);
  if (threadIdx.x == 0) {
    double *const o = a.totals + ((int64_t)b * a.pieces + piece) * 2;
    o[0] = s0, o[1] = s1;
  }
}

// The pieces' values of one of two sides, i and i + 64 of them in lane i (at most 128 pieces).
__device__ __forceinline__ double piece_value(const double *v, int i, int n, int side) {
  return i < n ? v[2 * i + side] : 0.0;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Reciprocals of the sums of the drawn row's powers and of its draft's (1 and 0 where p need not be normalised).
struct Norms {
  double rp, rq;
};
__device__ __forceinline__ Norms norms_of(const Args &a, int b, int lane) {
  const double *const t = a.totals + (int64_t)b * a.pieces * 2;
  const double sp = wave_sum(piece_value(t, lane, a.pieces, 0) + piece_value(t, lane + 64, a.pieces, 0));
  const double sq = wave_sum(piece_value(t, lane, a.pieces, 1) + piece_value(t, lane + 64, a.pieces, 1));
  return Norms{1.0 / sp, reciprocal(sq)};
}

// The weights of 8 tokens from column k on: rest[j] = what is drawn from, chance[j] = p (or a multiple of it).
template <int DT>
__device__ __forceinline__ void weights_of(const Args &a, int b, const Draw &d, Norms n, int k, int to, double *rest,
                                           double *chance) {
  float v[8], w[8];
  load_logits<DT>(target_row<DT>(a, b, d.at), k, to, v);
  if (d.rest) load_logits<DT>(draft_row<DT>(a, b, d.at), k, to, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    chance[j] = power((double)v[j], d.p) * n.rp;
    rest[j] = k + j == d.without ? 0.0 : chance[j];
  }
  if (d.rest) {
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = fmax(rest[j] - power((double)w[j], d.q) * n.rq, 0.0);
  }
}

// Sums of the weights of a piece, where a draft row is subtracted (elsewhere total_kernel's sums are the weights). 64
// streams of 150144 tokens: 21 us, the arithmetic of total_kernel again; powers kept in memory would be 16 bytes a token.
template <int DT>
__global__ __launch_bounds__(256) void weight_kernel(const Args a) {
  const int b = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces, lane = threadIdx.x & 63;
  const float T = temperature(a, b);
  __shared__ Draw d;
  __shared__ double scratch[4];
  if (!(T > 0) && (piece || !a.exact)) return;
  if (a.exact) {
    find_draw<DT>(a, b, T, d);
    if (piece == 0 && threadIdx.x == 0) a.draws[b] = d;
    if (!(T > 0)) return;
  } else {
    if (threadIdx.x == 0) d = a.draws[b];
    __syncthreads();
  }
  if (!d.rest) return;
  const Norms n = a.exact ? Norms{d.rp, d.rq} : norms_of(a, b, lane);
  double rest[8], chance[8], sr = 0, sc = 0;
  const int from = piece * a.piece, to = min(a.V, from + a.piece);
  for (int k = from + threadIdx.x * 8; k < to; k += 2048) {
    weights_of<DT>(a, b, d, n, k, to, rest, chance);
#pragma unroll
    for (int j = 0; j < 8; ++j) sr += rest[j], sc += chance[j];
  }
  sr = block_sum(sr, scratch);
  sc = block_sum(sc, scratch);
  if (threadIdx.x == 0) {
    double *const o = a.weights + ((int64_t)b * a.pieces + piece) * 2;
    o[0] = sr, o[1] = sc;
  }
}

// A workgroup finds a stream's drawn token and writes its row of the result. The running sum goes by piece (each wave
// for itself), then by 8192 tokens of the piece, by thread and by token. In a launch of its own: a stream's last
// workgroup of weight_kernel could do it, but the fence that every workgroup then needs writes its XCD's L2 back
// (64 streams of 150144 tokens: 97 us, as two launches 27). Alone it takes 11 us for 64 streams and 7 for one, the latency
// of its steps.
template <int DT>
__global__ __launch_bounds__(1024) void draw_kernel(const Args a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ double scratch[16];
  __shared__ int2 hits[16];
  __shared__ Draw d;
  const float T = temperature(a, b);
  const double *const totals = a.totals + (int64_t)b * a.pieces * 2;
  int found = -1, pieces = a.pieces, piece = a.piece;
  if (a.L && a.exact && !a.draft) {
    find_draw<DT>(a, b, T, d);
  } else if (a.L) {
    if (tid == 0) d = a.draws[b];
  } else if (T > 0) {
    float m = fmaxf(lane < pieces ? (float)totals[2 * lane + 1] : -FLT_MAX,
                    lane + 64 < pieces ? (float)totals[2 * (lane + 64) + 1] : -FLT_MAX);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (tid == 0) d = Draw{0, 0, exponent(T, m), Exponent{0, 0}, 1.0, 0.0, -1};
  } else if (tid == 0) {
    d.at = 0;
  }
  __syncthreads();
  if (!(T > 0)) {
    found = row_best(a, a.L ? parts_of(a, b, d.at) : a.parts + (int64_t)b * a.pieces, a.L ? a.splits : a.pieces);
  } else {
    // weights of the pieces lane and lane + 64; of the second choice, p itself
    double lo, hi = 0, lo1, hi1 = 0;
    Norms n{1.0, 0.0};
    if (a.L && a.exact && !d.rest) {  // stats_kernel's pieces, with largest logits of their own
      pieces = a.splits, piece = a.chunk;
      const Part p = lane < pieces ? parts_of(a, b, d.at)[lane] : Part{-FLT_MAX, 0, 0.0};
      lo = lo1 = p.s * power((double)p.m, d.p);
      if (d.without >= 0 && d.without < a.V) {  // its piece again without it: a difference could leave what is not there
        const int own = (int)(d.without / piece), to = min(a.V, (own + 1) * piece);
        double s = 0;
        for (int k = own * piece + tid * 8; k < to; k += 8192) {
          float v[8];
          load_logits<DT>(target_row<DT>(a, b, d.at), k, to, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) s += k + j == d.without ? 0.0 : power((double)v[j], d.p);
        }
        s = wave_sum(s);
        if (lane == 0) scratch[wave] = s;
        __syncthreads();
        s = 0;
        for (int v = 0; v < 16; ++v) s += scratch[v];
        if (lane == own) lo = s;
      }
    } else if (d.rest) {
      n = a.exact ? Norms{d.rp, d.rq} : norms_of(a, b, lane);
      const double *const w = a.weights + (int64_t)b * pieces * 2;
      lo = piece_value(w, lane, pieces, 0), hi = piece_value(w, lane + 64, pieces, 0);
      lo1 = piece_value(w, lane, pieces, 1), hi1 = piece_value(w, lane + 64, pieces, 1);
    } else {
      lo = piece_value(totals, lane, pieces, 0), hi = piece_value(totals, lane + 64, pieces, 0);
      lo1 = piece_value(totals, lane, pieces, 1), hi1 = piece_value(totals, lane + 64, pieces, 1);
      if (a.L) {
        lo1 += lo, hi1 += hi;
      } else {  // pieces with largest logits of their own; a lane without one has none, and 0 may lie far above the row's
        lo *= power(lane < pieces ? lo1 : -FLT_MAX, d.p), hi *= power(lane + 64 < pieces ? hi1 : -FLT_MAX, d.p);
        lo1 = lo, hi1 = hi;
      }
    }
    const bool side = !(wave_sum(lo + hi) > 0);
    if (side) lo = lo1, hi = hi1;
    const auto scan = [&](double v) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o);
        if (lane >= o) v += u;
      }
      return v;
    };
    const double run_lo = scan(lo), half = __shfl(run_lo, 63), run_hi = half + scan(hi), whole = __shfl(run_hi, 63);
    if (whole > 0 && whole <= DBL_MAX) {
      const double goal = uniform(a, b, a.L) * whole;
      const uint64_t in_lo = __ballot(lo > 0 && run_lo > goal), in_hi = __ballot(hi > 0 && run_hi > goal);
      int at;
      if (in_lo) at = __builtin_ctzll(in_lo);
      else if (in_hi) at = 64 + __builtin_ctzll(in_hi);
      else {  // a number of 1 or more, or none: the last token with a weight
        const uint64_t some_lo = __ballot(lo > 0), some_hi = __ballot(hi > 0);
        at = some_hi ? 127 - __builtin_clzll(some_hi) : 63 - __builtin_clzll(some_lo);
      }
      // what runs before the piece: the sums of the pieces before it, so that no difference is taken
      double run = at & 63 ? __shfl(at < 64 ? run_lo : run_hi, (at & 63) - 1) : (at < 64 ? 0.0 : half);
      const int from = at * piece, to = min(a.V, from + piece);
      int some = -1;
      for (int base = from; base < to && found < 0; base += 8192) {
        const int k = base + tid * 8;
        double rest[8], chance[8], mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] = 0;
        if (k < to) {
          weights_of<DT>(a, b, d, n, k, to, rest, chance);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            rest[j] = side ? chance[j] : rest[j];
            mine += rest[j];
          }
        }
        const double s = scan(mine);
        __syncthreads();  // the last 8192 tokens' sums and hits have been read
        if (lane == 63) scratch[wave] = s;
        __syncthreads();
        double before = run;
        for (int v = 0; v < wave; ++v) before += scratch[v];
        for (int v = 0; v < 16; ++v) run += scratch[v];
        before += s - mine;
        int first = kNone, final = -1;  // the first token past the goal, and the last one with a weight
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          before += rest[j];
          if (rest[j] > 0) {
            final = k + j;
            if (before > goal && first == kNone) first = k + j;
          }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) first = min(first, __shfl_xor(first, o)), final = max(final, __shfl_xor(final, o));
        if (lane == 0) hits[wave] = make_int2(first, final);
        __syncthreads();
        for (int v = 0; v < 16; ++v) first = min(first, hits[v].x), final = max(final, hits[v].y);
        some = max(some, final);
        if (first != kNone) found = first;
      }
      if (found < 0) found = some;
    }
  }
  for (int t = tid; t <= a.L; t += 1024)
    a.out[(int64_t)b * (a.L + 1) + t] = t < d.at ? a.tokens[(int64_t)b * a.L + t] : t == d.at ? found : -1;
  if (tid == 0 && a.accepted) a.accepted[b] = d.at;
}

struct Layout {
  int splits, chunk, pieces, piece, ranges, exact;
  int64_t parts, totals, weights, draws, refused, bytes;
};
// Pieces of whole 2048 tokens (256 threads, 16 or 32 bytes each), about so many workgroups of them. The statistics' hold 7
// a CU: 6 leave a launch without a second turn (64 streams, 16 drafted tokens of 150144 with their logits: 143 us at 4
// pieces a row, 150 at 5, 154 at 6, 148 at 3, 166 at 2; 158 at 11).
constexpr int64_t kStats = 6 * 256, kDraws = 8 * 256;
static void cut(int64_t V, int64_t rows, int64_t groups, int64_t most, int &n, int &size) {
  const int64_t want = std::min<int64_t>(cdiv(V, 2048), std::max<int64_t>(1, std::min<int64_t>(most, cdiv(groups, rows))));
  size = (int)(cdiv(cdiv(V, want), 2048) * 2048);
  n = (int)cdiv(V, size);
}
// Positions of the launches of stats_kernel: the last of them ends with L + 1.
static int ranges_of(int64_t B, int64_t L, int64_t V, int draft, int *ends) {
  int n = 0;
  const int64_t logits = B * V * (draft ? 2 : 1);  // of a position
  if (logits * (L + 1) < kSeveral) {
    ends[n++] = (int)L + 1;
    return n;
  }
  int64_t at = 0, step = std::max<int64_t>(1, cdiv(kFirst, logits));
  while (n < kRanges - 1 && at + 2 * step < L + 1) {
    at += step;
    ends[n++] = (int)at;
    step += (step + 1) / 2;
  }
  ends[n++] = (int)L + 1;
  return n;
}
static Layout layout(int64_t B, int64_t L, int64_t V, int draft) {
  Layout l;
  int ends[kRanges];
  l.ranges = ranges_of(B, L, V, draft, ends);
  cut(V, B * ends[0] * (L && draft ? 2 : 1), kStats, 32, l.splits, l.chunk);
  cut(V, B, kDraws, 128, l.pieces, l.piece);
  // Few logits: 64-bit sums of all rows cost less than another launch (one stream's 16 tokens of 150144: 26 us, with
  // total_kernel 30)
  l.exact = L > 0 && l.ranges == 1 && B * (L + 1 + (draft ? L : 0)) * V <= kFew && l.chunk <= kHeld * 2048;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  l.parts = take(L ? B * (2 * L + 1) * l.splits * (int64_t)sizeof(Part) : B * l.pieces * (int64_t)sizeof(Part));
  l.totals = take(B * l.pieces * 16);
  l.weights = take(B * l.pieces * 16);
  l.draws = take(B * (int64_t)sizeof(Draw));
  l.refused = take(kRanges * B * 4);
  l.bytes = at;
  return l;
}

template <int DT>
static void launch(Args a, hipStream_t st) {
  const unsigned all = (unsigned)((int64_t)a.B * a.pieces);
  if (a.L) {
    int ends[kRanges];
    const int n = ranges_of(a.B, a.L, a.V, a.draft != nullptr, ends);
    for (a.range = 0; a.range < n; ++a.range) {
      a.before = a.range > 1 ? ends[a.range - 2] : 0;
      a.t0 = a.range ? ends[a.range - 1] : 0, a.t1 = ends[a.range];
      stats_kernel<DT><<<(unsigned)((int64_t)a.splits * (a.draft ? 2 : 1) * a.B * (a.t1 - a.t0)), 256, 0, st>>>(a);
    }
    --a.range;
    if (!a.exact) total_kernel<DT><<<all, 256, 0, st>>>(a);
  } else {
    sample_kernel<DT><<<all, 256, 0, st>>>(a);
  }
  if (a.draft) weight_kernel<DT><<<all, 256, 0, st>>>(a);
  draw_kernel<DT><<<(unsigned)a.B, 1024, 0, st>>>(a);
}

static bool fits(int64_t B, int64_t L, int64_t V) {
  return B >= 0 && L >= 0 && V >= 1 && B <= (1 << 20) && L <= (1 << 16) && V <= 0x7fffffff - 65536 &&
         B * (2 * L + 1) <= (1 << 22);
}

}  // namespace spec
}  // namespace ksd

using namespace ksd;

extern "C" int ksd_verify_draft_workspace(int64_t B, int64_t L, int64_t V, int draft, int64_t *bytes) {
  if (!bytes || !spec::fits(B, L, V)) return fail(KSD_EINVAL, "verify_draft_workspace: bad arguments");
  *bytes = spec::layout(B, L, V, draft).bytes;
  return KSD_OK;
}

extern "C" int ksd_verify_draft(const void *target, const void *draft, int dtype, int64_t B, int64_t L, int64_t V,
                                int64_t target_b, int64_t target_t, int64_t draft_b, int64_t draft_t, const int64_t *tokens,
                                const void *uniforms, int uniforms_wide, const float *temperatures, float temperature,
                                const int64_t *lengths, int64_t *out, int64_t *accepted, void *workspace, int64_t workspace_bytes, void *stream) {
  if (!spec::fits(B, L, V)) return fail(KSD_EINVAL, "verify_draft: bad shape");
  if (dtype != KSD_F32 && dtype != KSD_BF16 && dtype != KSD_F16) return fail(KSD_ETYPE, "verify_draft: unsupported element type");
  if (B == 0) return KSD_OK;
  if (!target || (!uniforms && (temperatures || temperature > 0)) || !out || (L > 0 && !accepted) || !workspace || (L > 0 && !tokens))
    return fail(KSD_EINVAL, "verify_draft: null pointer");
  if (target_b < 0 || target_t < 0 || draft_b < 0 || draft_t < 0) return fail(KSD_EINVAL, "verify_draft: negative stride");
  const spec::Layout l = spec::layout(B, L, V, draft != nullptr);
  if (workspace_bytes < l.bytes) return fail(KSD_EINVAL, "verify_draft: short workspace");
  char *w = (char *)workspace;
  spec::Args a{target, L ? draft : nullptr, target_b, target_t, draft_b, draft_t, tokens, uniforms, uniforms_wide, temperatures,
               temperature, lengths, out, accepted, (spec::Part *)(w + l.parts), (double *)(w + l.totals), (double *)(w + l.weights),
               (spec::Draw *)(w + l.draws), (int *)(w + l.refused), (int)B, (int)L, (int)V, l.splits,
               l.chunk, l.pieces, l.piece, 0, 0, 0, 0, l.exact};
  hipStream_t st = (hipStream_t)stream;
  if (!grid_fits((int64_t)l.splits * 2 * B * (L + 1), 256) || !grid_fits(B * l.pieces, 256))
    return fail(KSD_EINVAL, "verify_draft: too many rows");
  switch (dtype) {
    case KSD_F32: spec::launch<KSD_F32>(a, st); break;
    case KSD_BF16: spec::launch<KSD_BF16>(a, st); break;
    default: spec::launch<KSD_F16>(a, st);
  }
  return check_launch("verify_draft");
}
