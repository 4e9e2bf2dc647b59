// Log probabilities of given tokens under rows of logits, with entropy and the best alternatives.
//   m = max x,  s = sum exp(x - m),  log p_v = (x_v - m) - log s
//   H = -sum p log p = log s - (sum e d) / s  with d = x - m, e = exp(d)
// m and log s stay apart (stats): in a row of the type's lowest value m + log s would be m.
// Any m near the largest logit serves, for the sums are floating point: stats holds a running
// reference that is up to kSlack below it.
// -inf is a masked token: probability 0 and nothing to the entropy.  A row of nothing else has
// logp -inf for every token, entropy 0 and no gradient.  A row with NaN or +inf gives NaN.
// The alternatives are ordered by logit, NaN above all, the lowest id first among equals.
// A token below 0 is a position that is not scored: logp 0, no gradient through it.  One at or
// beyond V gives NaN and raises bit 1 of the sticky device word.
// Gradient, with S = dlogp + sum of dtop:
//   dx_v = dlogp [v = token] + sum_j dtop_j [v = id_j] - p_v (S + dH (log p_v + H)).
#include <algorithm>

#include "lm.h"

namespace hsl {
namespace {

constexpr int kMaxTop = 32;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxParts = 64;        // of a row
constexpr int kFineParts = 16;       // up to which a part has groups of 16 lanes, not of 64
constexpr int kBwdVecs = 2;          // vectors of a thread in the backward
constexpr int kShortRow = 2048;      // logits of a row that one wave takes
constexpr long long kLaunchRows = 1 << 23;  // workgroups of a launch: their threads stay below 2^32
constexpr int kRowLanes = 4;         // of a group in a row of one workgroup
constexpr int kCandidates = 2048;    // elements that may be ranked among a row's alternatives
constexpr float kLog2e = 1.44269502162933349609375f;
constexpr float kLowest = -3.402823466e38f;
// A running sum keeps its reference until a logit exceeds it by this much: e^8 is far from
// overflow, and the terms of sd stay within 8 + their distance from the largest logit.
constexpr float kSlack = 8.0f;

// The order of the alternatives as whole numbers: the value's order above (-0 as 0, NaN the
// largest), the smallest index the largest below.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xFFFFFFFEu;  // (no key is all ones)
  const unsigned u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) {
  if (o == 0xFFFFFFFEu) return __builtin_nanf("");
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ unsigned long long key_of(float x, int v) {
  return (unsigned long long)order_of(x) << 32 | (0xFFFFFFFFu - (unsigned)v);
}

__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
  for (int d = 32; d; d >>= 1) {
    const unsigned long long o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}

// 16 bytes of a row at any element's alignment (global memory takes unaligned accesses).
// NT: non-temporal, for rows that no cache holds until their next use.
template <int F>
struct Vec {
  static constexpr int N = 16 / sizeof(typename Elem<F>::T);
  typename Elem<F>::T v[N];
};
template <int F>
__device__ __forceinline__ Vec<F> load_vec(const typename Elem<F>::T* p) {
  Vec<F> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <int F, bool NT>
__device__ __forceinline__ void store_vec(typename Elem<F>::T* p, const Vec<F>& x) {
  if constexpr (NT)
    store16_nt(p, x);
  else
    __builtin_memcpy(p, &x, sizeof(x));
}
// Vector i of a row of V elements, the part beyond the row masked.
template <int F>
__device__ __forceinline__ Vec<F> load_edge(const typename Elem<F>::T* row, int i, int V) {
  Vec<F> r;
  const int first = i * Vec<F>::N;
  if (first + Vec<F>::N <= V) return load_vec<F>(row + first);
#pragma unroll
  for (int e = 0; e < Vec<F>::N; ++e)
    r.v[e] = first + e < V ? row[first + e] : Elem<F>::down(-__builtin_inff());
  return r;
}

// s = sum e^(x - r), sd = sum e^(x - r) (x - r) over some elements; r is one of them or kLowest.
struct Sums {
  float r, s, sd;
  // the same with another reference, no smaller
  __device__ __forceinline__ void rebase(float to) {
    const float gap = r - to, c = __builtin_amdgcn_exp2f(gap * kLog2e);
    sd = c == 0.f ? 0.f : c * __builtin_fmaf(gap, s, sd);  // (gap may be -inf)
    s *= c;
    r = to;
  }
};

// The running sums and, with TOP, the largest element's value and vector of one thread.
template <int F, bool TOP>
struct Running {
  Sums q{kLowest, 0.f, 0.f};
  float best = -__builtin_inff();
  int at = 0x7FFFFFFF;
  __device__ __forceinline__ void take(const Vec<F>& x, int i) {
    constexpr int N = Vec<F>::N;
    float f[N], m = Elem<F>::up(x.v[0]);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = Elem<F>::up(x.v[e]);
#pragma unroll
    for (int e = 1; e < N; ++e) m = fmaxf(m, f[e]);
    if (TOP && (m > best || at == 0x7FFFFFFF)) {  // the first vector too, if it holds -inf alone
      best = m;
      at = i;
    }
    if (__any(m > q.r + kSlack)) {
      if (m > q.r) q.rebase(m);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      // exp2 of the rounded product is within 1.3 |d| 2^-24 of e^d, little where e^d counts
      const float d = f[e] - q.r, p = __builtin_amdgcn_exp2f(d * kLog2e);
      q.s += p;
      q.sd = __builtin_fmaf(p, fmaxf(d, -1e30f), q.sd);  // p = 0 for d = -inf
    }
  }
};

// One workgroup's elements: the vectors first .. last-1 of a row.  Four loads are in flight.
template <int F, bool TOP, int W>
__device__ __forceinline__ void scan_part(const typename Elem<F>::T* __restrict__ row, int first, int last, int V,
                                          Running<F, TOP>& a) {
  constexpr int N = Vec<F>::N, kAhead = 4, kN = W * 64;
  const int whole = min(last, V / N);
  int i = first + threadIdx.x;
  for (; i + (kAhead - 1) * kN < whole; i += kAhead * kN) {
    Vec<F> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) x[k] = load_vec<F>(row + (size_t)(i + k * kN) * N);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) a.take(x[k], i + k * kN);
  }
  for (; i < last; i += kN) a.take(load_edge<F>(row, i, V), i);
}

// The sums of the whole workgroup, in every thread: the largest reference first, to which each
// lane's sums are brought once.
template <int W>
__device__ __forceinline__ Sums join_block(Sums q, Sums (&lds)[W]) {
  float to = q.r;
#pragma unroll
  for (int d = 32; d; d >>= 1) to = fmaxf(to, __shfl_xor(to, d));
  if (q.r != to) q.rebase(to);
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    q.s += __shfl_xor(q.s, d);
    q.sd += __shfl_xor(q.sd, d);
  }
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = q;
    __syncthreads();
    to = lds[0].r;
#pragma unroll
    for (int w = 1; w < W; ++w) to = fmaxf(to, lds[w].r);
    Sums sum{to, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      Sums o = lds[w];
      if (o.r != to) o.rebase(to);
      sum.s += o.s;
      sum.sd += o.sd;
    }
    q = sum;
  }
  return q;
}

struct Out {
  float *logp, *entropy, *stats, *top_logp;
  long long* top_ids;
};

// The row's token and its logit, read before anything else.
struct Token {
  long long id;  // -1: none
  float x;
};
template <int F>
__device__ __forceinline__ Token load_token(const void* tokens, int tok64, size_t n, const typename Elem<F>::T* row,
                                            int V) {
  Token t{-1, 0.f};
  if (tokens) t.id = load_id(tokens, tok64, n);
  if (t.id >= 0 && t.id < V) t.x = Elem<F>::up(row[t.id]);
  return t;
}

// Row n's results from its sums; returns whether nothing in it is above -inf.
__device__ __forceinline__ bool finish_row(size_t n, const Sums& q, float ls, const Token& t, int V, const Out& o,
                                           unsigned* err) {
  const bool none = q.s == 0.f;  // (not of a row with NaN)
  if (threadIdx.x == 0) {
    o.stats[2 * n] = none ? -__builtin_inff() : q.r;
    o.stats[2 * n + 1] = ls;
    o.entropy[n] = none ? 0.f : ls - q.sd / q.s;
    if (o.logp) {
      float r = 0.f;
      if (t.id >= V) {
        atomicOr(err, kErrId);
        r = __builtin_nanf("");
      } else if (t.id >= 0) {
        r = none ? -__builtin_inff() : t.x - q.r - ls;
      }
      o.logp[n] = r;
    }
  }
  return none;
}

// The alternatives of a row.  The vectors are in groups, of each of which the largest element is
// known by its value and its vector (key: 0 if the group is empty).  The k groups with the largest
// keys hold the k largest elements: any other group's elements are all below those k.  So only these
// groups are read again, for the elements at or above the k-th group's key, and those are ranked by
// counting.  Groups are GL lanes wide: group g has vectors (g / (n / GL)) * part + n i +
// (g mod (n / GL)) * GL + 0 .. GL-1, n the threads.  A row of one workgroup has 64 groups, which one
// wave ranks; with 256 of one lane the ranking took 2 us of the workgroup's time instead of 0.1.
// There each lane's own key (LANES) then says whether its part of a group has to be read: with 20
// alternatives that is 9% of the row, not 31%.
struct alignas(16) TopShared {
  unsigned long long key[kThreads];  // one for each group
  unsigned long long cand[kCandidates];
  int unit[kThreads];  // what is read again: groups, or lanes
  unsigned long long least;
  int count[kWaves];
  int ncand, nunit;
};
template <int F, int W, int GL, int KEYS, bool LANES>
__device__ void choose_top(const typename Elem<F>::T* __restrict__ row, int V, int top, int part, int nvec,
                           unsigned long long key, unsigned long long lane_key, float r, float ls, bool nan_row,
                           bool none, size_t n, const Out& o, TopShared& sh) {
  constexpr int N = Vec<F>::N, kN = W * 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (threadIdx.x < KEYS) sh.key[threadIdx.x] = key;
  if (threadIdx.x == 0) sh.ncand = sh.nunit = 0;
  const int groups = min(__syncthreads_count(threadIdx.x < KEYS && key != 0), top);
  if (threadIdx.x < KEYS) {
    int rank = 0;
#pragma unroll 8
    for (int u = 0; u < KEYS; u += 2) {
      const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(&sh.key[u]);
      rank += (k.x > key) + (k.y > key);
    }
    if (!LANES && rank < groups) sh.unit[rank] = threadIdx.x;
    if (rank == groups - 1) {
      // the smallest key that an element of that group's vector with that value can have; with fewer
      // groups than asked for, every element is a candidate
      const unsigned long long back = (0xFFFFFFFFull - (key & 0xFFFFFFFFull)) * N + N - 1;
      sh.least = groups < top ? 0 : (key | 0xFFFFFFFFull) - back;
    }
  }
  __syncthreads();
  const unsigned long long least = sh.least;
  if constexpr (LANES) {
    // the largest key that an element of the lane's vectors can have
    const unsigned long long most = (lane_key | 0xFFFFFFFFull) - (0xFFFFFFFFull - (lane_key & 0xFFFFFFFFull)) * N;
    if (lane_key && most >= least) sh.unit[atomicAdd(&sh.nunit, 1)] = threadIdx.x;
    __syncthreads();
  }
  constexpr int kUnit = LANES ? 1 : GL, kUnits = kN / kUnit;  // lanes of a unit, units of a round
  const int units = LANES ? sh.nunit : groups;
  const int each = (part + kN - 1) / kN * kUnit;  // vectors of a unit
  const float tau = least ? value_of((unsigned)(least >> 32)) : -__builtin_inff();
  // the units' elements at or above `from`, or above tau alone
  auto collect = [&](unsigned long long from, bool above_tau) {
    constexpr int kAhead = 4;  // loads in flight
    for (int i0 = threadIdx.x; i0 < units * each; i0 += kAhead * kN) {
      Vec<F> x[kAhead];
      int vec[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * kN;
        vec[a] = nvec;
        if (i < units * each) {
          const int g = sh.unit[i / each], j = i % each;
          const int at = (j / kUnit) * kN + (g % kUnits) * kUnit + j % kUnit;
          if (at < part) vec[a] = min((g / kUnits) * part + at, nvec);
        }
        if (vec[a] < nvec) x[a] = load_edge<F>(row, vec[a], V);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (vec[a] >= nvec) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float f = Elem<F>::up(x[a].v[e]);
          if (f < tau || (above_tau && f == tau)) continue;  // most
          const unsigned long long k = key_of(f, vec[a] * N + e);
          if (k >= from && vec[a] * N + e < V) {
            const int c = atomicAdd(&sh.ncand, 1);
            if (c < kCandidates) sh.cand[c] = k;
          }
        }
      }
    }
  };
  if (!nan_row) collect(least, false);
  __syncthreads();
  int ncand = sh.ncand;
  if (!nan_row && ncand > kCandidates) {
    // Many equal elements, as in a row of masks: those above tau, and of those equal to it the
    // first in the row.
    __syncthreads();
    if (threadIdx.x == 0) sh.ncand = 0;
    __syncthreads();
    collect(0, true);
    __syncthreads();
    ncand = sh.ncand;
    if (ncand <= kCandidates - kMaxTop) {
      for (int i0 = 0; i0 < nvec && ncand < top; i0 += kN) {
        const int i = i0 + threadIdx.x;
        Vec<F> x;
        int equal = 0;
        if (i < nvec) {
          x = load_edge<F>(row, i, V);
#pragma unroll
          for (int e = 0; e < N; ++e) equal += i * N + e < V && Elem<F>::up(x.v[e]) == tau;
        }
        int upto = equal;  // of the wave's lanes up to this one, then of the workgroup's
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const int v = __shfl_up(upto, d);
          if (lane >= d) upto += v;
        }
        if (lane == 63) sh.count[w] = upto;
        __syncthreads();
        int at = ncand + upto - equal;
        for (int u = 0; u < W; ++u) {
          if (u < w) at += sh.count[u];
          ncand += sh.count[u];
        }
        if (equal) {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (i * N + e < V && Elem<F>::up(x.v[e]) == tau) {
              if (at < top) sh.cand[at] = key_of(tau, i * N + e);
              ++at;
            }
        }
        __syncthreads();
      }
      ncand = min(ncand, max(top, sh.ncand));
    }
  }
  if (!nan_row && ncand <= kCandidates) {
    for (int c = threadIdx.x; c < ncand; c += kN) {
      const unsigned long long k = sh.cand[c];
      int above = 0;
#pragma unroll 8
      for (int u = 0; u < ncand; ++u) above += sh.cand[u] > k;
      if (above < top) {
        o.top_ids[n * top + above] = 0xFFFFFFFFu - (unsigned)k;
        o.top_logp[n * top + above] = none ? -__builtin_inff() : value_of((unsigned)(k >> 32)) - r - ls;
      }
    }
    return;
  }
  // a row with NaN, or one whose large elements crowd in a few groups: one round over the row each
  unsigned long long last = ~0ull;
  for (int j = 0; j < top; ++j) {
    unsigned long long best = 0;
    for (int v = threadIdx.x; v < V; v += kN) {
      const unsigned long long c = key_of(Elem<F>::up(row[v]), v);
      if (c < last && c > best) best = c;
    }
    best = wave_max(best);
    __syncthreads();
    if (lane == 0) sh.key[w] = best;
    __syncthreads();
    for (int u = 0; u < W; ++u) best = sh.key[u] > best ? sh.key[u] : best;
    last = best;
    if (threadIdx.x == 0) {
      o.top_ids[n * top + j] = 0xFFFFFFFFu - (unsigned)best;
      o.top_logp[n * top + j] = nan_row ? __builtin_nanf("") : none ? -__builtin_inff()
                                                                    : value_of((unsigned)(best >> 32)) - r - ls;
    }
  }
}

// A group's key: the value's order above, the smallest vector the largest below; 0 without one.
__device__ __forceinline__ unsigned long long group_key(float best, int at) {
  return at == 0x7FFFFFFF ? 0 : key_of(best, at);
}

// One workgroup per row, one pass: the running sums and each group's largest element.  Bound by HBM:
// N8192 V32768 bf16 95 us for 537 MB (5.7 TB/s; 105 on average in training passes on inputs in turn),
// with 20 alternatives 122.  A row of up to kShortRow logits takes one wave, which needs no barriers.  us
// without and with 4 alternatives, one wave / four:
//   bf16 N8192 V512: 5.7, 21 / 11, 27;  V2048: 8.9, 25 / 14, 29;  V4096: 16, 31 / 19, 33
//   fp32 N8192 V512: 5.9, 20 / 11, 25;  V2048: 14, 26 / 16, 30;  V4096: 23, 35 / 22, 32
// With 64 rows the two are within 0.5 up to V2048.
template <int F, bool TOP, int W>
__global__ __launch_bounds__(W * 64) void logprob_row_kernel(const typename Elem<F>::T* __restrict__ logits,
                                                               long long ld, const void* __restrict__ tokens,
                                                               int tok64, Out o, int V, int top, unsigned* err) {
  __shared__ Sums lds[W];
  const size_t n = blockIdx.x;
  const auto* const row = logits + (long long)n * ld;
  const int nvec = (int)(((long long)V + Vec<F>::N - 1) / Vec<F>::N);
  const Token token = load_token<F>(tokens, tok64, n, row, V);
  Running<F, TOP> a;
  scan_part<F, TOP, W>(row, 0, nvec, V, a);
  const Sums q = join_block(a.q, lds);
  const float ls = logf(q.s);
  const bool none = finish_row(n, q, ls, token, V, o, err);
  if constexpr (TOP) {
    constexpr int GL = W > 1 ? kRowLanes : 1;  // 64 groups
    __shared__ TopShared sh;
    __shared__ unsigned long long keys[W * 64 / GL];
    const unsigned long long lane_key = group_key(a.best, a.at);
    unsigned long long key = lane_key;
#pragma unroll
    for (int d = 1; d < GL; d *= 2) {
      const unsigned long long other = __shfl_xor(key, d);
      key = other > key ? other : key;
    }
    key = __shfl(key, (threadIdx.x * GL) & 63);  // of thread t: group 16 (t / 64) + t mod 16
    if ((threadIdx.x & 63) < 64 / GL) keys[threadIdx.x / 64 * (64 / GL) + (threadIdx.x & 63)] = key;
    __syncthreads();
    key = threadIdx.x < W * 64 / GL ? keys[threadIdx.x] : 0;
    choose_top<F, W, GL, W * 64 / GL, (GL > 1)>(row, V, top, nvec, nvec, key, lane_key, q.r, ls, q.s != q.s, none, n, o,
                                                sh);
  }
}

// Fewer than 512 rows leave CUs idle: each is cut into parts of `part` vectors, whose sums and groups'
// keys go to ws, and a workgroup per row joins them (4 rows of 131072 bf16 with 20 alternatives: 4 and
// 10 us, latency).  GL: lanes of a group, as many as give at most kThreads groups.
template <int F, bool TOP, int GL>
__global__ __launch_bounds__(kThreads) void logprob_part_kernel(const typename Elem<F>::T* __restrict__ logits,
                                                                long long ld, Sums* __restrict__ sums,
                                                                unsigned long long* __restrict__ keys, int V,
                                                                int part) {
  __shared__ Sums lds[kWaves];
  const size_t n = blockIdx.y;
  const int nvec = (int)(((long long)V + Vec<F>::N - 1) / Vec<F>::N), p = blockIdx.x;
  Running<F, TOP> a;
  scan_part<F, TOP, kWaves>(logits + (long long)n * ld, p * part, min(nvec, (p + 1) * part), V, a);
  const Sums q = join_block(a.q, lds);
  if (threadIdx.x == 0) sums[n * gridDim.x + p] = q;
  if constexpr (TOP) {
    unsigned long long key = group_key(a.best, a.at);
#pragma unroll
    for (int d = GL / 2; d; d >>= 1) {
      const unsigned long long other = __shfl_xor(key, d);
      key = other > key ? other : key;
    }
    if (threadIdx.x % GL == 0) keys[(n * gridDim.x + p) * (kThreads / GL) + threadIdx.x / GL] = key;
  }
}

template <int F, bool TOP, int GL>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(const typename Elem<F>::T* __restrict__ logits,
                                                                long long ld, const Sums* __restrict__ sums,
                                                                const unsigned long long* __restrict__ keys,
                                                                const void* __restrict__ tokens, int tok64, Out o,
                                                                int V, int part, int parts, int top, unsigned* err) {
  __shared__ Sums lds[kWaves];
  const size_t n = blockIdx.x;
  const auto* const row = logits + (long long)n * ld;
  const int nvec = (int)(((long long)V + Vec<F>::N - 1) / Vec<F>::N);
  const Token token = load_token<F>(tokens, tok64, n, row, V);
  Sums q{kLowest, 0.f, 0.f};
  if ((int)threadIdx.x < parts) q = sums[n * parts + threadIdx.x];
  unsigned long long key = 0;
  constexpr int kPer = kThreads / GL;
  if (TOP && (int)threadIdx.x < parts * kPer) key = keys[n * parts * kPer + threadIdx.x];
  q = join_block<kWaves>(q, lds);
  const float ls = logf(q.s);
  const bool none = finish_row(n, q, ls, token, V, o, err);
  if constexpr (TOP) {
    __shared__ TopShared sh;
    choose_top<F, kWaves, GL, kThreads, false>(row, V, top, part, nvec, key, 0, q.r, ls, q.s != q.s, none, n, o, sh);
  }
}

// Bound by HBM: N8192 V32768 bf16 164 us for 1074 MB (6.5 TB/s) behind the forward.
// dx = -p (S + dH (log p + H)) for the vectors of one part of a row; then the elements with a
// gradient of their own, the token and the alternatives, are computed again with it.  Rows are taken
// from the last to the first: the forward has just read the last ones, and a cache may still hold
// them.  Where logits and gradient exceed the caches the gradient is stored past them, so that it
// does not drive those rows out (both steps at 8192 x 32768 bf16, forward and backward: 294 -> 262 us).
template <int F, bool ENT, bool NT>
__global__ __launch_bounds__(kThreads) void logprob_bwd_kernel(
    const typename Elem<F>::T* __restrict__ logits, long long ld, const void* __restrict__ tokens, int tok64,
    const long long* __restrict__ top_ids, const float* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ dlogp, const float* __restrict__ dent, const float* __restrict__ dtop,
    typename Elem<F>::T* __restrict__ dlogits, long long ldd, int V, int top) {
  constexpr int N = Vec<F>::N;
  const size_t n = gridDim.y - 1 - blockIdx.y;
  const auto* const row = logits + (long long)n * ld;
  auto* const drow = dlogits + (long long)n * ldd;
  const int nvec = (int)(((long long)V + N - 1) / N), first = blockIdx.x * kBwdVecs * kThreads;
  const int last = min(nvec, first + kBwdVecs * kThreads);
  Vec<F> x[kBwdVecs];  // in flight while the row's numbers arrive
#pragma unroll
  for (int k = 0; k < kBwdVecs; ++k) {
    const int i = first + k * kThreads + threadIdx.x;
    if (i < last) x[k] = load_edge<F>(row, i, V);
  }
  const float m = stats[2 * n], ls = stats[2 * n + 1];
  const bool none = m == -__builtin_inff();
  const long long tok = tokens && dlogp ? load_id(tokens, tok64, n) : -1;
  const float dl = tok >= 0 ? (tok < V ? dlogp[n] : __builtin_nanf("")) : 0.f;
  float S = dl;
  for (int k = 0; dtop && k < top; ++k) S += dtop[n * top + k];
  const float dh = ENT ? dent[n] : 0.f, SH = ENT ? __builtin_fmaf(dh, entropy[n], S) : S;
  auto grad = [&](float x) {
    const float d = x - m - ls, p = __builtin_amdgcn_exp2f(d * kLog2e);
    // p = 0: no gradient, though d may be -inf, dh d beyond fp32, or what arrives not finite
    const float pull = ENT ? __builtin_fmaf(dh, d, SH) : SH;
    return p == 0.f ? 0.f : -p * pull;
  };
#pragma unroll
  for (int k = 0; k < kBwdVecs; ++k) {
    const int i = first + k * kThreads + threadIdx.x;
    if (i >= last) break;
    float g[N];
    if (none) {
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = grad(Elem<F>::up(x[k].v[e]));
    }
    down_all<F, N>(g, x[k].v);
    auto* const out = drow + (size_t)i * N;
    if (i * N + N <= V) {
      store_vec<F, NT>(out, x[k]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i * N + e < V) out[e] = x[k].v[e];
    }
  }
  __syncthreads();  // their stores come after the part's
  const int k = threadIdx.x;
  if (none || k > top || (k < top && !dtop)) return;
  const long long v = k < top ? top_ids[n * top + k] : tok;
  if (v < (long long)first * N || v >= min((long long)V, (long long)last * N)) return;
  float g = grad(Elem<F>::up(row[v]));
  if (v == tok) g += dl;
  for (int j = 0; dtop && j < top; ++j)
    if (top_ids[n * top + j] == v) g += dtop[n * top + j];
  drow[v] = Elem<F>::down(g);
}

// Parts of a row and their vectors: one part where the rows alone fill the chip.
struct Parts {
  int count, vectors;
};
Parts plan_parts(long long N, int V, int fmt) {
  const int per = fmt == kElemF32 ? 4 : 8;
  const int nvec = (int)(((long long)V + per - 1) / per);
  // At least 9 parts: the groups of all but the last are as many as the alternatives may be.
  int count = 1;
  if (N < 512 && nvec >= 9 * kThreads) {
    const long long want = std::max((2048 + N - 1) / std::max(N, 1ll), 9ll);
    count = (int)std::min<long long>({want, kMaxParts, nvec / kThreads});
  }
  if (count == 1) return {1, nvec};
  // whole rounds of a workgroup's threads; rounded down, where that is not too many parts
  int vectors = nvec / count / kThreads * kThreads;
  if ((nvec + vectors - 1) / vectors > kMaxParts) vectors += kThreads;
  return {(nvec + vectors - 1) / vectors, vectors};
}

struct LogprobWs {
  Sums* sums;
  unsigned long long* keys;
};
size_t carve_logprob(void* ws, size_t cap, long long N, int parts, LogprobWs* o) {
  Carver c(ws, cap);
  o->sums = c.take<Sums>((size_t)N * parts);
  o->keys = c.take<unsigned long long>((size_t)N * kThreads);
  return align_up(c.off, 256);
}

int check_logprob(const char* who, long long N, int V, int top, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (N < 0 || V < 0) return fail(HSL_ERR_ARG, "%s: negative size (N=%lld V=%d)", who, N, V);
  if (top < 0 || top > kMaxTop || top > V)
    return fail(HSL_ERR_ARG, "%s: top=%d is not in 0..min(%d, V=%d)", who, top, kMaxTop, V);
  if (N >= (1ll << 31) || V > 0x7FFFF000)
    return fail(HSL_ERR_UNSUPPORTED, "%s: N=%lld rows of V=%d need 2^31 > N and V <= 2^31 - 4096", who, N, V);
  return HSL_OK;
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

size_t hsl_logprob_fwd_ws_bytes(long long N, int V, int top) {
  if (N <= 0 || V < 0) return 0;
  // the 16-bit and the fp32 cut of a row differ
  const int parts = std::max(plan_parts(N, V, kElemBf16).count, plan_parts(N, V, kElemF32).count);
  LogprobWs w;
  return parts > 1 ? carve_logprob(nullptr, 0, N, parts, &w) : 0;
}

int hsl_logprob_fwd(const void* logits, long long ld, const void* tokens, int tok64, float* logp, float* entropy,
                    float* stats, float* top_logp, long long* top_ids, void* ws, size_t ws_bytes, long long N, int V,
                    int top, int fmt, void* stream) {
  HSL_CHECK(check_logprob("hsl_logprob_fwd", N, V, top, fmt));
  if (N == 0) return HSL_OK;
  if ((V > 0 && !logits) || !entropy || !stats || (tokens && !logp) || (top && (!top_logp || !top_ids)))
    return fail(HSL_ERR_ARG, "hsl_logprob_fwd: null pointer");
  unsigned* err;
  HSL_CHECK(device_error_word(&err));
  const Parts p = plan_parts(N, V, fmt);
  LogprobWs w{};
  if (p.count > 1) {
    const size_t need = carve_logprob(ws, ws_bytes, N, p.count, &w);
    if (!ws || ws_bytes < need)
      return fail(HSL_ERR_ARG, "hsl_logprob_fwd: workspace %zu bytes, need %zu", ws_bytes, need);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Out o{tokens ? logp : nullptr, entropy, stats, top_logp, top_ids};
  return with_fmt(fmt, [&](auto f) {
    constexpr int kF = decltype(f)::value;
    const auto* x = static_cast<const typename Elem<kF>::T*>(logits);
    auto run = [&](auto t) {
      constexpr bool kTop = decltype(t)::value;
      if (p.count == 1) {
        for (long long n0 = 0; n0 < N; n0 += kLaunchRows) {
          const dim3 rows((unsigned)std::min(N - n0, kLaunchRows));
          const auto* const xn = x + n0 * ld;
          const void* const tn = tokens ? static_cast<const char*>(tokens) + n0 * (tok64 ? 8 : 4) : nullptr;
          const Out on{o.logp ? o.logp + n0 : nullptr, entropy + n0, stats + 2 * n0,
                       top ? top_logp + n0 * top : nullptr, top ? top_ids + n0 * top : nullptr};
          if (V <= kShortRow)
            hipLaunchKernelGGL((logprob_row_kernel<kF, kTop, 1>), rows, dim3(64), 0, s, xn, ld, tn, tok64, on, V, top,
                               err);
          else
            hipLaunchKernelGGL((logprob_row_kernel<kF, kTop, kWaves>), rows, dim3(kThreads), 0, s, xn, ld, tn, tok64,
                               on, V, top, err);
        }
      } else {
        auto cut = [&](auto lanes) {
          constexpr int kGL = decltype(lanes)::value;
          hipLaunchKernelGGL((logprob_part_kernel<kF, kTop, kGL>), dim3(p.count, (unsigned)N), dim3(kThreads), 0, s, x,
                             ld, w.sums, w.keys, V, p.vectors);
          hipLaunchKernelGGL((logprob_join_kernel<kF, kTop, kGL>), dim3((unsigned)N), dim3(kThreads), 0, s, x, ld,
                             w.sums, w.keys, tokens, tok64, o, V, p.vectors, p.count, top, err);
        };
        if (kTop && p.count <= kFineParts)
          cut(std::integral_constant<int, kTop ? 16 : 64>{});
        else
          cut(std::integral_constant<int, 64>{});
      }
    };
    if (top)
      run(std::true_type{});
    else
      run(std::false_type{});
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

int hsl_logprob_bwd(const void* logits, long long ld, const void* tokens, int tok64, const long long* top_ids,
                    const float* stats, const float* entropy, const float* dlogp, const float* dent, const float* dtop,
                    void* dlogits, long long ldd, long long N, int V, int top, int fmt, void* stream) {
  HSL_CHECK(check_logprob("hsl_logprob_bwd", N, V, top, fmt));
  if (N == 0 || V == 0) return HSL_OK;
  if (!logits || !stats || !dlogits || (dlogp && !tokens) || (dent && !entropy) || (dtop && !top_ids))
    return fail(HSL_ERR_ARG, "hsl_logprob_bwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  // a workgroup takes `part` vectors of a row; blockIdx.y holds fewer than 2^16 rows
  const int per = fmt == kElemF32 ? 4 : 8, part = kBwdVecs * kThreads;
  const int nvec = (int)(((long long)V + per - 1) / per);
  return with_fmt(fmt, [&](auto f) {
    constexpr int kF = decltype(f)::value;
    using T = typename Elem<kF>::T;
    const bool nt = (size_t)N * V * sizeof(T) * 2 > kCacheBytes;
    for (long long n0 = (N - 1) / 65535 * 65535; n0 >= 0; n0 -= 65535) {
      const unsigned rows = (unsigned)std::min<long long>(N - n0, 65535);
      auto run = [&](auto e, auto past) {
        hipLaunchKernelGGL((logprob_bwd_kernel<kF, decltype(e)::value, decltype(past)::value>),
                           dim3((nvec + part - 1) / part, rows), dim3(kThreads), 0, s,
                           static_cast<const T*>(logits) + n0 * ld, ld,
                           tokens ? static_cast<const char*>(tokens) + n0 * (tok64 ? 8 : 4) : nullptr, tok64,
                           top_ids ? top_ids + n0 * top : nullptr, stats + 2 * n0, entropy ? entropy + n0 : nullptr,
                           dlogp ? dlogp + n0 : nullptr, dent ? dent + n0 : nullptr, dtop ? dtop + n0 * top : nullptr,
                           static_cast<T*>(dlogits) + n0 * ldd, ldd, V, top);
      };
      using Yes = std::true_type;
      using No = std::false_type;
      if (dent)
        nt ? run(Yes{}, Yes{}) : run(Yes{}, No{});
      else
        nt ? run(No{}, Yes{}) : run(No{}, No{});
      HSL_HIP(hipGetLastError());
    }
    return (int)HSL_OK;
  });
}

}  // extern "C"
