// Log probabilities of given tokens under rows of logits, with entropy and the best alternatives.
//   m = max x,  s = sum exp(x - m),  log p_v = (x_v - m) - log s
//   H = -sum p log p = log s - (sum e d) / s  with d = x - m, e = exp(d)
// m and log s stay apart (stats): in a row of the type's lowest value m + log s would be m.
// -inf is a masked token: probability 0 and nothing to the entropy.  A row of nothing else has
// logp -inf for every token, entropy 0 and no gradient.  A row with NaN or +inf gives NaN.
// The alternatives are ordered by logit, NaN above all, the lowest id first among equals.
// A token below 0 is a position that is not scored: logp 0, no gradient through it.  One at or
// beyond V gives NaN and raises bit 1 of the sticky device word.
// Gradient, with S = dlogp + sum of dtop:
//   dx_v = dlogp [v = token] + sum_j dtop_j [v = id_j] - p_v (S + dH (log p_v + H)).
#include "lm.h"

namespace hsl {
namespace {

constexpr int kMaxTop = 32;
constexpr int kThreads = 256, kWaves = kThreads / 64;

// The order of the alternatives as whole numbers: the value's order above (-0 as 0, NaN the
// largest), the smallest index the largest below.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xFFFFFFFEu;  // (no key is all ones)
  const unsigned u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int v) {
  return (unsigned long long)order_of(x) << 32 | (0xFFFFFFFFu - (unsigned)v);
}

template <class T>
__device__ __forceinline__ T wave_max(T v) {
  for (int d = 32; d; d >>= 1) {
    const T o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// One workgroup per row; the alternatives in `top` rounds over the row.
template <int F>
__global__ __launch_bounds__(kThreads) void logprob_fwd_kernel(
    const typename Elem<F>::T* __restrict__ logits, long long ld, const void* __restrict__ tokens, int tok64,
    float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_logp,
    long long* __restrict__ top_ids, int V, int top, unsigned* err) {
  __shared__ float sm[kWaves], ss[kWaves], sw[kWaves];
  __shared__ unsigned long long sk[kWaves];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const size_t n = blockIdx.x;
  const auto* const row = logits + (long long)n * ld;
  float m = -__builtin_inff();
  for (int v = threadIdx.x; v < V; v += kThreads) m = fmaxf(m, Elem<F>::up(row[v]));
  m = wave_max(m);
  if (lane == 0) sm[w] = m;
  __syncthreads();
  for (int u = 0; u < kWaves; ++u) m = fmaxf(m, sm[u]);
  const bool empty = m == -__builtin_inff();
  const float m0 = empty ? 0.f : m;
  float s = 0.f, sd = 0.f;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    const float d = Elem<F>::up(row[v]) - m0, e = exp_f(d);
    s += e;
    sd += e == 0.f ? 0.f : e * d;
  }
  s = wave_sum(s);
  sd = wave_sum(sd);
  if (lane == 0) {
    ss[w] = s;
    sw[w] = sd;
  }
  __syncthreads();
  s = sd = 0.f;
  for (int u = 0; u < kWaves; ++u) {
    s += ss[u];
    sd += sw[u];
  }
  // no element was above -inf and the sum is 0: the row is empty (NaN is not above -inf either)
  const bool none = empty && s == 0.f;
  const float ls = logf(s);
  if (threadIdx.x == 0) {
    stats[2 * n] = none ? m : m0;
    stats[2 * n + 1] = ls;
    entropy[n] = none ? 0.f : ls - sd / s;
    if (tokens) {
      const long long t = load_id(tokens, tok64, n);
      float r = 0.f;
      if (t >= V) {
        atomicOr(err, kErrId);
        r = __builtin_nanf("");
      } else if (t >= 0) {
        r = none ? -__builtin_inff() : Elem<F>::up(row[t]) - m0 - ls;
      }
      logp[n] = r;
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int v = threadIdx.x; v < V; v += kThreads) {
      const unsigned long long c = key_of(Elem<F>::up(row[v]), v);
      if (c < last && c > best) best = c;
    }
    best = wave_max(best);
    __syncthreads();
    if (lane == 0) sk[w] = best;
    __syncthreads();
    for (int u = 0; u < kWaves; ++u) best = sk[u] > best ? sk[u] : best;
    last = best;
    if (threadIdx.x == 0) {
      const int v = (int)(0xFFFFFFFFu - (unsigned)best);
      top_ids[n * top + k] = v;
      top_logp[n * top + k] = none ? -__builtin_inff() : Elem<F>::up(row[v]) - m0 - ls;
    }
  }
}

template <int F>
__global__ __launch_bounds__(kThreads) void logprob_bwd_kernel(
    const typename Elem<F>::T* __restrict__ logits, long long ld, const void* __restrict__ tokens, int tok64,
    const long long* __restrict__ top_ids, const float* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ dlogp, const float* __restrict__ dent, const float* __restrict__ dtop,
    typename Elem<F>::T* __restrict__ dlogits, long long ldd, int V, int top) {
  const size_t n = blockIdx.x;
  const auto* const row = logits + (long long)n * ld;
  auto* const drow = dlogits + (long long)n * ldd;
  const float m = stats[2 * n], ls = stats[2 * n + 1];
  const bool none = m == -__builtin_inff();
  long long tok = tokens && dlogp ? load_id(tokens, tok64, n) : -1;
  const float dl = tok >= 0 ? (tok < V ? dlogp[n] : __builtin_nanf("")) : 0.f;
  float S = dl;
  for (int k = 0; dtop && k < top; ++k) S += dtop[n * top + k];
  const float dh = dent ? dent[n] : 0.f, H = dent ? entropy[n] : 0.f;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    const float d = Elem<F>::up(row[v]) - m - ls, p = exp_f(d);
    float g = p == 0.f ? 0.f : -p * (S + dh * (d + H));
    if (v == tok) g += dl;
    for (int k = 0; dtop && k < top; ++k)
      if (top_ids[n * top + k] == v) g += dtop[n * top + k];
    drow[v] = Elem<F>::down(none ? 0.f : g);
  }
}

int check_logprob(const char* who, long long N, int V, int top, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (N < 0 || V < 0) return fail(HSL_ERR_ARG, "%s: negative size (N=%lld V=%d)", who, N, V);
  if (top < 0 || top > kMaxTop || top > V)
    return fail(HSL_ERR_ARG, "%s: top=%d is not in 0..min(%d, V=%d)", who, top, kMaxTop, V);
  if (N >= (1ll << 31)) return fail(HSL_ERR_UNSUPPORTED, "%s: N=%lld rows need 2^31 > N", who, N);
  return HSL_OK;
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

size_t hsl_logprob_fwd_ws_bytes(long long N, int V, int top) { return 0; }

int hsl_logprob_fwd(const void* logits, long long ld, const void* tokens, int tok64, float* logp, float* entropy,
                    float* stats, float* top_logp, long long* top_ids, void* ws, size_t ws_bytes, long long N, int V,
                    int top, int fmt, void* stream) {
  HSL_CHECK(check_logprob("hsl_logprob_fwd", N, V, top, fmt));
  if (N == 0) return HSL_OK;
  if ((V > 0 && !logits) || !entropy || !stats || (tokens && !logp) || (top && (!top_logp || !top_ids)))
    return fail(HSL_ERR_ARG, "hsl_logprob_fwd: null pointer");
  unsigned* err;
  HSL_CHECK(device_error_word(&err));
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_fmt(fmt, [&](auto f) {
    using T = typename Elem<decltype(f)::value>::T;
    hipLaunchKernelGGL(logprob_fwd_kernel<decltype(f)::value>, dim3((unsigned)N), dim3(kThreads), 0, s,
                       static_cast<const T*>(logits), ld, tokens, tok64, logp, entropy, stats, top_logp, top_ids, V, top,
                       err);
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
  return with_fmt(fmt, [&](auto f) {
    using T = typename Elem<decltype(f)::value>::T;
    hipLaunchKernelGGL(logprob_bwd_kernel<decltype(f)::value>, dim3((unsigned)N), dim3(kThreads), 0, s,
                       static_cast<const T*>(logits), ld, tokens, tok64, top_ids, stats, entropy, dlogp, dent, dtop,
                       static_cast<T*>(dlogits), ldd, V, top);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
