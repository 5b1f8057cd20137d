// Verification of drafted tokens against the target's logits, and drawing a token from logits, from given
// random numbers. With p = softmax(z / T) of a target row and q that of the draft's:
//
//   position t is accepted while u[t] q(token) < p(token)       (no draft logits: q(token) = 1)
//   the first refused one, or the one behind the last, draws the first token whose running sum of
//   weights passes u[L] times their sum: weights max(p - q, 0), or p where nothing was refused
//   T = 0: accepted while the token is the row's largest logit (the lowest index of equal ones), which is drawn too
//
// One read of the rows gives each row's largest logit and sum of powers in 32 bits (stats_kernel): the tests
// need p and q of one token a row, and an error of 2^-24 there moves one test in ten million. The drawn token is
// another matter: with 150144 tokens a running sum has as many borders, and sums in 32 bits would move about one draw in
// a hundred across one. The one row of a stream that is drawn from is therefore read again with powers and sums in 64
// bits (total_kernel, draw_kernel). Logits of -inf have probability 0; a row without a finite logit, or with NaN or
// +inf, has no distribution: a target's is refused and draws -1, a draft's refuses the token and draws from p.
#include "ksd_common.h"

#include <float.h>

#include <algorithm>

namespace ksd {
namespace spec {

struct Part {  // of a row's piece: largest logit, sum of 2^((z - m) c); greedy: largest logit, -, its place
  float m, s;
  int at, bad;
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
  int *arrived;                // (B,)
  int B, L, V, splits, chunk, pieces, piece;
};

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

// ------------------------------------------------------------------------------- row statistics
struct Best {
  float m;
  int at;
};
__device__ __forceinline__ Best better(Best x, Best y) {
  return y.m > x.m || (y.m == x.m && y.at < x.at) ? y : x;
}

template <int DT>
__global__ __launch_bounds__(256) void stats_kernel(const Args a, int t0, int nt) {
  // blocks: split fastest, then target and draft, then requests, then positions
  const int split = blockIdx.x % a.splits;
  int i = blockIdx.x / a.splits;
  const int sides = a.draft ? 2 : 1;
  const bool drafted = i % sides;
  i /= sides;
  const int b = i % a.B, t = t0 + i / a.B;
  const int len = length(a, b);
  const float T = temperature(a, b);
  const bool greedy = !(T > 0);
  if (t > len || (drafted && (t == len || greedy))) return;
  const typename Elem<DT>::T *const row = drafted ? draft_row<DT>(a, b, t) : target_row<DT>(a, b, t);
  const int from = split * a.chunk, to = min(a.V, from + a.chunk);
  const float c = 1.4426950408889634f / clamped(T);
  __shared__ float sm[4], ss[4];
  __shared__ int si[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int U = 4;
  Part *const out = const_cast<Part *>(parts_of(a, b, drafted ? a.L + 1 + t : t)) + split;
  if (greedy) {
    Best best{-INFINITY, 0x7fffffff};
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
    const int any = __ballot(bad) != 0;
    if (lane == 0) sm[wave] = best.m, si[wave] = best.at, ss[wave] = any ? 1.0f : 0.0f;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 4; ++w) best = better(best, Best{sm[w], si[w]});
      *out = Part{best.m, 0.0f, best.at, ss[0] + ss[1] + ss[2] + ss[3] > 0};
    }
    return;
  }
  float m = -FLT_MAX, s = 0.0f;  // not -inf: a piece of nothing but -inf then has differences of -inf and sum 0
  for (int k = from + threadIdx.x * 8; k < to; k += 2048 * U) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u * 2048 < to) load_logits<DT>(row, k + u * 2048, to, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u * 2048 >= to) break;
      float top = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, v[u][j]);
      s *= __builtin_amdgcn_exp2f((m - top) * c);
      m = top;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += __builtin_amdgcn_exp2f((v[u][j] - m) * c);
    }
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
    *out = Part{m, s, 0, 0};
  }
}

// ------------------------------------------------------------------------------- acceptance
struct Stat {
  float m;
  double s;
};
__device__ __forceinline__ Stat row_stat(const Args &a, const Part *p, float c) {
  Stat r{-FLT_MAX, 0.0};
  for (int i = 0; i < a.splits; ++i) r.m = fmaxf(r.m, p[i].m);
  for (int i = 0; i < a.splits; ++i) r.s += (double)(p[i].s * __builtin_amdgcn_exp2f((p[i].m - r.m) * c));
  return r;
}
// The place of a greedy row's largest logit; -1 where it has none.
__device__ __forceinline__ int row_best(const Args &a, const Part *p) {
  Best best{-INFINITY, 0x7fffffff};
  int bad = 0;
  for (int i = 0; i < a.splits; ++i) best = better(best, Best{p[i].m, p[i].at}), bad |= p[i].bad;
  return bad || best.m == -INFINITY ? -1 : best.at;
}
__device__ __forceinline__ double power(float z, float m, double inv) {  // e^((z - m) / T)
  return exp(((double)z - (double)m) * inv);
}

template <int DT>
__device__ __forceinline__ bool accepts(const Args &a, int b, int t, float T) {
  const int64_t token = a.tokens[(int64_t)b * a.L + t];
  if (!(T > 0)) return row_best(a, parts_of(a, b, t)) == token && token >= 0;
  if (token < 0 || token >= a.V) return false;
  const float c = 1.4426950408889634f / clamped(T);
  const double inv = 1.0 / (double)clamped(T);
  const Stat p = row_stat(a, parts_of(a, b, t), c);
  const double pt = power(Elem<DT>::load(target_row<DT>(a, b, t) + token), p.m, inv) / p.s;
  double qt = 1.0;
  if (a.draft) {
    const Stat q = row_stat(a, parts_of(a, b, a.L + 1 + t), c);
    qt = q.s == 0 ? 0.0 : power(Elem<DT>::load(draft_row<DT>(a, b, t) + token), q.m, inv) / q.s;
  }
  return uniform(a, b, t) * qt < pt;
}

// Accepted positions among the first `most` (a whole wave; every lane gets the result).
template <int DT>
__device__ __forceinline__ int accepted_of(const Args &a, int b, int most, float T) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < most; base += 64) {
    const int t = base + lane;
    const bool refused = t < most && !accepts<DT>(a, b, t, T);
    const uint64_t m = __ballot(refused);
    if (m) return base + __builtin_ctzll(m);
  }
  return most;
}

// ------------------------------------------------------------------------------- the drawn token
template <int NT>
__device__ __forceinline__ double block_sum(double v, double *scratch) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) r += scratch[w];
  return r;
}

// What the draw of a stream works on.
struct Draw {
  int at, refused;     // position, and whether its token was refused
  float mp, mq;        // largest logits
  double inv;
  int64_t token;       // the refused token
};

template <int DT>
__device__ __forceinline__ void draw_of(const Args &a, int b, Draw &d) {  // wave 0 writes d (in LDS)
  const float T = temperature(a, b);
  const int len = length(a, b);
  const int at = accepted_of<DT>(a, b, len, T);
  if ((threadIdx.x & 63) == 0) {
    d.at = at, d.refused = at < len;
    d.inv = 1.0 / (double)clamped(T);
    d.token = at < len ? a.tokens[(int64_t)b * a.L + at] : -1;
    float m = -FLT_MAX;
    const Part *p = parts_of(a, b, at);
    for (int i = 0; i < a.splits; ++i) m = fmaxf(m, p[i].m);
    d.mp = m;
    m = -FLT_MAX;
    if (d.refused && a.draft) {
      p = parts_of(a, b, a.L + 1 + at);
      for (int i = 0; i < a.splits; ++i) m = fmaxf(m, p[i].m);
    }
    d.mq = m;
  }
}

// Sums of e^((z - m) / T) in 64 bits of a piece of the row that is drawn from, target and draft.
template <int DT>
__global__ __launch_bounds__(256) void total_kernel(const Args a) {
  const int b = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  if (!(temperature(a, b) > 0)) {
    if (piece == 0 && threadIdx.x == 0) a.arrived[b] = 0;
    return;
  }
  __shared__ Draw d;
  __shared__ double scratch[4];
  if (threadIdx.x < 64) draw_of<DT>(a, b, d);
  __syncthreads();
  const int from = piece * a.piece, to = min(a.V, from + a.piece);
  const bool both = d.refused && a.draft;
  double sp = 0, sq = 0;
  for (int k = from + threadIdx.x * 8; k < to; k += 2048) {
    float v[8];
    load_logits<DT>(target_row<DT>(a, b, d.at), k, to, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) sp += power(v[j], d.mp, d.inv);
    if (both) {
      load_logits<DT>(draft_row<DT>(a, b, d.at), k, to, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sq += power(v[j], d.mq, d.inv);
    }
  }
  sp = block_sum<256>(sp, scratch);
  sq = block_sum<256>(sq, scratch);
  if (threadIdx.x == 0) {
    double *const o = a.totals + ((int64_t)b * a.pieces + piece) * 2;
    o[0] = sp, o[1] = sq;
    if (piece == 0) a.arrived[b] = 0;
  }
}

// The weights of 8 tokens from column k on: rest[j] = what is drawn from, chance[j] = p.
template <int DT>
__device__ __forceinline__ void weights_of(const Args &a, int b, const Draw &d, double rp, double rq, int k, int to,
                                           double *rest, double *chance) {
  float v[8];
  load_logits<DT>(target_row<DT>(a, b, d.at), k, to, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = chance[j] = power(v[j], d.mp, d.inv) * rp;
  if (!d.refused) return;
  if (a.draft) {
    load_logits<DT>(draft_row<DT>(a, b, d.at), k, to, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = fmax(rest[j] - power(v[j], d.mq, d.inv) * rq, 0.0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j == d.token) rest[j] = 0.0;
  }
}

// Sums of the weights of a piece; the stream's last workgroup finds the drawn token. Only the order in which
// workgroups end decides which one that is: sums are added by piece.
template <int DT>
__global__ __launch_bounds__(256) void draw_kernel(const Args a) {
  const int b = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ Draw d;
  __shared__ double scratch[4];
  __shared__ int last, found;
  const float T = temperature(a, b);
  const bool greedy = !(T > 0);
  if (greedy && piece) return;
  if (tid < 64) {
    if (greedy) {
      const int at = accepted_of<DT>(a, b, length(a, b), T);
      if (lane == 0) d.at = at, found = row_best(a, parts_of(a, b, at));
    } else {
      draw_of<DT>(a, b, d);
    }
  }
  __syncthreads();
  if (!greedy) {
    double sp = 0, sq = 0;
    for (int i = 0; i < a.pieces; ++i) {
      const double *const o = a.totals + ((int64_t)b * a.pieces + i) * 2;
      sp += o[0], sq += o[1];
    }
    const double rp = 1.0 / sp, rq = sq > 0 ? 1.0 / sq : sq;  // an empty draft row: q = 0; NaN stays
    double rest[8], chance[8], sr = 0, sc = 0;
    {
      const int from = piece * a.piece, to = min(a.V, from + a.piece);
      for (int k = from + tid * 8; k < to; k += 2048) {
        weights_of<DT>(a, b, d, rp, rq, k, to, rest, chance);
#pragma unroll
        for (int j = 0; j < 8; ++j) sr += rest[j], sc += chance[j];
      }
      sr = block_sum<256>(sr, scratch);
      sc = block_sum<256>(sc, scratch);
    }
    if (tid == 0) {
      double *const o = a.weights + ((int64_t)b * a.pieces + piece) * 2;
      o[0] = sr, o[1] = sc;
      __threadfence();
      last = atomicAdd(&a.arrived[b], 1) == a.pieces - 1;
      __threadfence();
    }
    __syncthreads();
    if (!last) return;
    // the running sum by piece, then by 2048 tokens of the piece, then by thread and token
    const double *const w = a.weights + (int64_t)b * a.pieces * 2;
    double whole = 0, all = 0;
    for (int i = 0; i < a.pieces; ++i) whole += __builtin_nontemporal_load(w + 2 * i), all += __builtin_nontemporal_load(w + 2 * i + 1);
    const int side = whole > 0 ? 0 : 1;
    if (side) whole = all;
    if (tid == 0) found = -1;
    if (whole > 0 && whole <= DBL_MAX) {
      const double goal = uniform(a, b, a.L) * whole;
      double run = 0;
      int at = -1, some = -1;
      for (int i = 0; i < a.pieces; ++i) {
        const double s = __builtin_nontemporal_load(w + 2 * i + side);
        if (s > 0) some = i;
        if (s > 0 && run + s > goal) {
          at = i;
          break;
        }
        run += s;
      }
      if (at < 0) {  // a number of 1 or more, or none: the last token with a weight
        at = some;
        for (run = 0, some = 0; some < at; ++some) run += __builtin_nontemporal_load(w + 2 * some + side);
      }
      const int from = at * a.piece, to = min(a.V, from + a.piece);
      __shared__ int first, final;
      if (tid == 0) first = 0x7fffffff, final = -1;
      __syncthreads();
      for (int base = from; base < to; base += 2048) {
        const int k = base + tid * 8;
        double mine = 0;
        if (k < to) {
          weights_of<DT>(a, b, d, rp, rq, k, to, rest, chance);
          if (side) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rest[j] = chance[j];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) mine += rest[j];
        }
        double s = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const double u = __shfl_up(s, o);
          if (lane >= o) s += u;
        }
        if (lane == 63) scratch[wave] = s;
        __syncthreads();
        double before = run;
        for (int v = 0; v < wave; ++v) before += scratch[v];
        double end = run;
        for (int v = 0; v < 4; ++v) end += scratch[v];
        before += s - mine;
        if (k < to) {
          for (int j = 0; j < 8; ++j) {
            if (rest[j] > 0) {
              before += rest[j];
              atomicMax(&final, k + j);
              if (before > goal) {
                atomicMin(&first, k + j);
                break;
              }
            }
          }
        }
        __syncthreads();
        run = end;
        if (first != 0x7fffffff) break;
      }
      if (tid == 0) found = first != 0x7fffffff ? first : final;
    }
    __syncthreads();
  }
  for (int t = tid; t <= a.L; t += 256)
    a.out[(int64_t)b * (a.L + 1) + t] = t < d.at ? a.tokens[(int64_t)b * a.L + t] : t == d.at ? found : -1;
  if (tid == 0) a.accepted[b] = d.at;
}

struct Layout {
  int splits, chunk, pieces, piece;
  int64_t parts, totals, weights, arrived, bytes;
};
// Pieces of whole 2048 tokens (256 threads, 16 or 32 bytes each), enough of them to occupy the device a few times over.
static void cut(int64_t V, int64_t rows, int64_t most, int &n, int &size) {
  const int64_t want = std::min<int64_t>(cdiv(V, 2048), std::max<int64_t>(1, std::min<int64_t>(most, cdiv(2048, rows))));
  size = (int)(cdiv(cdiv(V, want), 2048) * 2048);
  n = (int)cdiv(V, size);
}
static Layout layout(int64_t B, int64_t L, int64_t V, int draft) {
  Layout l;
  cut(V, B * (L + 1 + (draft ? L : 0)), 32, l.splits, l.chunk);
  cut(V, B, 128, l.pieces, l.piece);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  l.parts = take(B * (2 * L + 1) * l.splits * (int64_t)sizeof(Part));
  l.totals = take(B * l.pieces * 16);
  l.weights = take(B * l.pieces * 16);
  l.arrived = take(B * 4);
  l.bytes = at;
  return l;
}

template <int DT>
static void launch(const Args &a, hipStream_t st) {
  const int sides = a.draft ? 2 : 1;
  stats_kernel<DT><<<(unsigned)((int64_t)a.splits * sides * a.B * (a.L + 1)), 256, 0, st>>>(a, 0, a.L + 1);
  total_kernel<DT><<<(unsigned)((int64_t)a.B * a.pieces), 256, 0, st>>>(a);
  draw_kernel<DT><<<(unsigned)((int64_t)a.B * a.pieces), 256, 0, st>>>(a);
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
  if (!target || (!uniforms && (temperatures || temperature > 0)) || !out || !accepted || !workspace || (L > 0 && !tokens))
    return fail(KSD_EINVAL, "verify_draft: null pointer");
  if (target_b < 0 || target_t < 0 || draft_b < 0 || draft_t < 0) return fail(KSD_EINVAL, "verify_draft: negative stride");
  const spec::Layout l = spec::layout(B, L, V, draft != nullptr);
  if (workspace_bytes < l.bytes) return fail(KSD_EINVAL, "verify_draft: short workspace");
  char *w = (char *)workspace;
  spec::Args a{target, L ? draft : nullptr, target_b, target_t, draft_b, draft_t, tokens, uniforms, uniforms_wide, temperatures,
               temperature, lengths, out, accepted, (spec::Part *)(w + l.parts), (double *)(w + l.totals), (double *)(w + l.weights),
               (int *)(w + l.arrived), (int)B, (int)L, (int)V, l.splits, l.chunk, l.pieces, l.piece};
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
