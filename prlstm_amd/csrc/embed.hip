// Embedding of token ids with a scale, and the gradient of its table.
//   out[n] = scale W[ids[n]]          dW[v] = scale sum over n with ids[n] = v of dout[n]
// An id below 0 is a position without a token: a row of zeros, and no gradient.  An id at or
// beyond V gives a NaN row and raises bit 1 of the sticky device word; it has no gradient.
//
// The gradient sums each row's positions in their order in ids, in fp32, so it does not depend on
// timing: embed_sort_kernel lists the positions by token first.  Its workgroup w owns the tokens
// v with v mod nclass = w (frequent tokens have neighbouring ids, so residues spread them) and
// reads all ids twice: once to count, once to place.  Where its list starts in the sorted order is
// the number of ids of smaller residue, which it counts itself, so workgroups exchange nothing.
//
// embed_sum_kernel then takes 16 bytes of one row of dW per thread and adds the row's positions.
// A row of more than `chunk` positions is summed in parts, so that the work of a frequent token (9%
// of all positions, as text has them) is spread: the sorted positions are cut into chunks, each
// chunk adds what it holds of such rows (only its first and its last token can be one) into fp32
// partials, and embed_join_kernel adds a row's partials in their order.
#include <algorithm>

#include "lm.h"

namespace hsl {
namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kClassTokens = 512;  // tokens of one workgroup at most (its counters: 16 waves of them)
constexpr int kBlock = 256;
constexpr int kJoinLanes = 16, kJoinGroups = kBlock / kJoinLanes;  // 64 columns, 16 shares of the partials

// 16 bytes of a row at any element's alignment.
template <int F>
struct Vec {
  static constexpr int N = 16 / sizeof(typename Elem<F>::T);
  typename Elem<F>::T v[N];
};
// Vector c of a row of D elements: what is beyond the row is not read or written.
template <int F>
__device__ __forceinline__ Vec<F> load_vec(const typename Elem<F>::T* row, int c, int D) {
  constexpr int N = Vec<F>::N;
  Vec<F> x;
  if (c * N + N <= D) {
    __builtin_memcpy(&x, row + c * N, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x.v[e] = c * N + e < D ? row[c * N + e] : Elem<F>::down(0.f);
  }
  return x;
}
template <int F>
__device__ __forceinline__ void store_vec(typename Elem<F>::T* row, int c, int D, const Vec<F>& x) {
  constexpr int N = Vec<F>::N;
  if (c * N + N <= D) {
    __builtin_memcpy(row + c * N, &x, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c * N + e < D) row[c * N + e] = x.v[e];
  }
}

// A thread per vector of the output (`per` of them in a row).
template <int F>
__global__ __launch_bounds__(kBlock) void embed_fwd_kernel(const void* __restrict__ ids, int ids64,
                                                           const typename Elem<F>::T* __restrict__ w, long long ldw,
                                                           float scale, typename Elem<F>::T* __restrict__ out, int N,
                                                           int V, int D, int per, unsigned* err) {
  const long long i = (long long)blockIdx.x * kBlock + threadIdx.x;
  const int n = (int)(i / per), c = (int)(i - (long long)n * per);
  if (n >= N) return;
  const long long id = load_id(ids, ids64, n);
  const bool beyond = id >= V;
  if (beyond && c == 0) atomicOr(err, kErrId);
  float f[Vec<F>::N];
  if (id >= 0 && !beyond) {
    const Vec<F> x = load_vec<F>(w + id * ldw, c, D);
#pragma unroll
    for (int e = 0; e < Vec<F>::N; ++e) f[e] = scale * Elem<F>::up(x.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < Vec<F>::N; ++e) f[e] = beyond ? __builtin_nanf("") : 0.f;
  }
  Vec<F> o;
  down_all<F, Vec<F>::N>(f, o.v);
  store_vec<F>(out + (size_t)n * D, c, D, o);
}

// What the sort leaves.  Token v is token q = v / nclass of class v mod nclass; a class has
// kClassTokens + 1 entries of start.
struct Sorted {
  int* start;   // where a token's positions begin in pos; they end at the next entry
  int* pos;     // positions by token, rising within one
  int* nlong;   // of a class: its tokens of more than `chunk` positions
  int* longs;   // [class][most]
  int log2c, chunk, most;
};
__device__ __forceinline__ int2 row_range(const Sorted& s, int v) {
  const int* const p = s.start + (size_t)(v & ((1 << s.log2c) - 1)) * (kClassTokens + 1) + (v >> s.log2c);
  return {p[0], p[1]};
}

// f(i, id) for a wave's part of ids in rounds of 64, kAhead loads in flight; id -1: none.
template <class Fn>
__device__ __forceinline__ void each_id(const void* __restrict__ ids, int ids64, int lo, int hi, int V, int padding,
                                        Fn f) {
  constexpr int kAhead = 8;
  const int lane = threadIdx.x & 63;
  for (int i0 = lo; i0 < hi; i0 += kAhead * 64) {
    long long id[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * 64 + lane;
      id[k] = i < hi ? load_id(ids, ids64, i) : -1;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k * 64 >= hi) break;
      const bool there = id[k] >= 0 && id[k] < V && id[k] != padding;
      f(i0 + k * 64 + lane, there ? (int)id[k] : -1);
    }
  }
}

__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const void* __restrict__ ids, int ids64, int N,
                                                                  int V, int padding, Sorted s) {
  __shared__ int cnt[kSortWaves][kClassTokens];
  __shared__ int below_s[kSortWaves], scan_s[kSortWaves], nlong;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = threadIdx.x;
  const int cls = blockIdx.x, mask = (1 << s.log2c) - 1;
  const int tokens = V > cls ? (V - cls + mask) >> s.log2c : 0;  // of this class
  for (int u = 0; u < kSortWaves; ++u)
    if (t < tokens) cnt[u][t] = 0;
  if (t == 0) nlong = 0;
  __syncthreads();
  // the wave's part of ids, in order: its tokens' counts, and the ids of smaller residues
  const int part = ((N + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int lo = min(w * part, N), hi = min(lo + part, N);
  int below = 0;
  each_id(ids, ids64, lo, hi, V, padding, [&](int, int id) {
    if (id < 0) return;
    below += (id & mask) < cls;
    if ((id & mask) == cls) atomicAdd(&cnt[w][id >> s.log2c], 1);
  });
  for (int d = 32; d; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) below_s[w] = below;
  __syncthreads();
  // each wave's place within a token's list, the token's total, and the exclusive sums of those
  int total = 0;
  if (t < tokens)
    for (int u = 0; u < kSortWaves; ++u) {
      const int c = cnt[u][t];
      cnt[u][t] = total;
      total += c;
    }
  int sum = total;
  for (int d = 1; d < 64; d *= 2) {
    const int v = __shfl_up(sum, d);
    if (lane >= d) sum += v;
  }
  if (lane == 63) scan_s[w] = sum;
  __syncthreads();
  int first = sum - total;
  for (int u = 0; u < kSortWaves; ++u) first += below_s[u] + (u < w ? scan_s[u] : 0);
  int* const st = s.start + (size_t)cls * (kClassTokens + 1);
  if (t < tokens) {
    st[t] = first;
    if (t == tokens - 1) st[tokens] = first + total;
    for (int u = 0; u < kSortWaves; ++u) cnt[u][t] += first;
    if (total > s.chunk) s.longs[(size_t)cls * s.most + atomicAdd(&nlong, 1)] = (t << s.log2c) | cls;
  }
  __syncthreads();
  if (t == 0) s.nlong[cls] = nlong;
  each_id(ids, ids64, lo, hi, V, padding, [&](int i, int id) {
    const int q = id >= 0 && (id & mask) == cls ? id >> s.log2c : -1;
    unsigned long long left = __ballot(q >= 0);
    while (left) {  // the tokens of these 64 positions, one after the other
      const int one = __shfl(q, __ffsll(left) - 1);
      const unsigned long long same = __ballot(q == one);
      if (q == one) {
        const int at = cnt[w][one], rank = __popcll(same & ((1ull << lane) - 1));
        s.pos[at + rank] = i;
        if (rank == 0) cnt[w][one] = at + __popcll(same);  // every lane of the wave has read it
      }
      left &= ~same;
    }
  });
}

// The sum of vector c of dout over the sorted positions lo .. hi-1, in that order, four at a time.
template <int F>
__device__ __forceinline__ void sum_positions(const int* __restrict__ pos, int lo, int hi,
                                              const typename Elem<F>::T* __restrict__ dout, long long ldd, int c, int D,
                                              float (&acc)[Vec<F>::N]) {
  constexpr int kAhead = 4;
#pragma unroll
  for (int e = 0; e < Vec<F>::N; ++e) acc[e] = 0.f;
  for (int i = lo; i < hi; i += kAhead) {
    const int n = min(kAhead, hi - i);
    Vec<F> x[kAhead];
    int p[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k < n) p[k] = pos[i + k];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k < n) x[k] = load_vec<F>(dout + p[k] * ldd, c, D);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k < n) {
#pragma unroll
        for (int e = 0; e < Vec<F>::N; ++e) acc[e] += Elem<F>::up(x[k].v[e]);
      }
  }
}

// The first `chunk_items` threads each take a vector of one chunk: its parts of the chunk's first
// and last token, where those are long, to partials 2 chunk and 2 chunk + 1 (rows of `pitch`).  The
// others take a vector of a row of dW that is not long.
template <int F>
__global__ __launch_bounds__(kBlock) void embed_sum_kernel(const void* __restrict__ ids, int ids64, Sorted s,
                                                           const typename Elem<F>::T* __restrict__ dout, long long ldd,
                                                           float scale, typename Elem<F>::T* __restrict__ dw,
                                                           float* __restrict__ partial, int pitch, int V, int D,
                                                           int per, int chunk_blocks) {
  constexpr int N = Vec<F>::N;
  float acc[N];
  if ((int)blockIdx.x < chunk_blocks) {
    const int i = blockIdx.x * kBlock + threadIdx.x, k = i / per, c = i - k * per;
    const int end = min(1 << s.log2c, V) - 1;  // the last class with a token: its end is the table's
    const int count = s.start[(size_t)end * (kClassTokens + 1) + ((V - 1 - end) >> s.log2c) + 1];
    const int lo = k * s.chunk, hi = min(lo + s.chunk, count);
    if (lo >= hi) return;
    const int first = (int)load_id(ids, ids64, s.pos[lo]), last = (int)load_id(ids, ids64, s.pos[hi - 1]);
    const int2 a = row_range(s, first), b = row_range(s, last);
    auto put = [&](int row) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (c * N + e < pitch) partial[(size_t)row * pitch + c * N + e] = acc[e];
    };
    if (a.y - a.x > s.chunk) {
      sum_positions<F>(s.pos, lo, min(hi, a.y), dout, ldd, c, D, acc);
      put(2 * k);
    }
    if (last != first && b.y - b.x > s.chunk) {
      sum_positions<F>(s.pos, b.x, hi, dout, ldd, c, D, acc);
      put(2 * k + 1);
    }
    return;
  }
  const long long i = (long long)(blockIdx.x - chunk_blocks) * kBlock + threadIdx.x;
  const int v = (int)(i / per), c = (int)(i - (long long)v * per);
  if (v >= V) return;
  const int2 r = row_range(s, v);
  if (r.y - r.x > s.chunk) return;
  sum_positions<F>(s.pos, r.x, r.y, dout, ldd, c, D, acc);
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] *= scale;
  Vec<F> o;
  down_all<F, N>(acc, o.v);
  store_vec<F>(dw + (size_t)v * D, c, D, o);
}

// The long rows of class blockIdx.y, 64 columns: kJoinGroups shares of a row's partials, each added
// in order, then the shares in order.
template <int F>
__global__ __launch_bounds__(kBlock) void embed_join_kernel(Sorted s, const float* __restrict__ partial, int pitch,
                                                            float scale, typename Elem<F>::T* __restrict__ dw, int D) {
  __shared__ float4 share[kJoinGroups][kJoinLanes];
  const int cls = blockIdx.y, lane = threadIdx.x % kJoinLanes, g = threadIdx.x / kJoinLanes;
  const int col = (blockIdx.x * kJoinLanes + lane) * 4;
  const int n = s.nlong[cls];
  for (int l = 0; l < n; ++l) {
    const int v = s.longs[(size_t)cls * s.most + l];
    const int2 r = row_range(s, v);
    const int c0 = r.x / s.chunk, parts = (r.y - 1) / s.chunk - c0 + 1;
    const int each = (parts + kJoinGroups - 1) / kJoinGroups, lo = g * each, hi = min(lo + each, parts);
    float4 sum{0.f, 0.f, 0.f, 0.f};
    if (col < D) {
#pragma unroll 4
      for (int i = lo; i < hi; ++i) {
        // the chunk's first token, except where the row begins inside its first chunk
        const int row = 2 * (c0 + i) + (i == 0 && r.x != c0 * s.chunk);
        const float4 p = *reinterpret_cast<const float4*>(partial + (size_t)row * pitch + col);
        sum.x += p.x;
        sum.y += p.y;
        sum.z += p.z;
        sum.w += p.w;
      }
    }
    share[g][lane] = sum;
    __syncthreads();
    if (g == 0) {
      float t[4] = {0.f, 0.f, 0.f, 0.f};
      for (int u = 0; u < kJoinGroups; ++u) {
        const float4 p = share[u][lane];
        t[0] += p.x;
        t[1] += p.y;
        t[2] += p.z;
        t[3] += p.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < D) dw[(size_t)v * D + col + e] = Elem<F>::down(scale * t[e]);
    }
    __syncthreads();
  }
}

struct EmbedPlan {
  int nclass, log2c, chunk, nchunks, most, pitch;
};
EmbedPlan plan_embed(long long N, int V, int D) {
  EmbedPlan p;
  p.log2c = 8;
  while (((long long)kClassTokens << p.log2c) < V) ++p.log2c;
  p.nclass = 1 << p.log2c;
  p.chunk = 64;  // and at most 2048 chunks
  while ((long long)p.chunk * 2048 < N) p.chunk *= 2;
  p.nchunks = N > p.chunk ? (int)((N + p.chunk - 1) / p.chunk) : 0;  // no token is longer than a chunk
  p.most = (int)std::min<long long>(kClassTokens, N / p.chunk);
  p.pitch = (D + 3) / 4 * 4;
  return p;
}
struct EmbedWs {
  Sorted s;
  float* partial;
};
size_t carve_embed(void* ws, size_t cap, long long N, const EmbedPlan& p, EmbedWs* o) {
  Carver c(ws, cap);
  o->s.start = c.take<int>((size_t)p.nclass * (kClassTokens + 1));
  o->s.pos = c.take<int>((size_t)N);
  o->s.nlong = c.take<int>(p.nclass);
  o->s.longs = c.take<int>((size_t)p.nclass * p.most);
  o->s.log2c = p.log2c;
  o->s.chunk = p.chunk;
  o->s.most = p.most;
  o->partial = c.take<float>((size_t)2 * p.nchunks * p.pitch);
  return align_up(c.off, 256);
}

int check_embed(const char* who, long long N, int V, int D, long long ld, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (N < 0 || V < 0 || D < 0 || ld < 0) return fail(HSL_ERR_ARG, "%s: negative size (N=%lld V=%d D=%d)", who, N, V, D);
  const long long per = (D + 3ll) / 4, lim = 1ll << 31;
  if (N > 0x7FFF0000 || N * per / kBlock >= lim - 2 || V * per / kBlock >= lim - 2 || D > 0x7FFFFFF0)
    return fail(HSL_ERR_UNSUPPORTED, "%s: N=%lld V=%d D=%d is beyond 2^31 ids or a grid of 2^31 workgroups", who, N, V, D);
  return HSL_OK;
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

int hsl_embed_fwd(const void* ids, int ids64, const void* weight, long long ldw, float scale, void* out, long long N,
                  int V, int D, int fmt, void* stream) {
  HSL_CHECK(check_embed("hsl_embed_fwd", N, V, D, ldw, fmt));
  if (N == 0 || D == 0) return HSL_OK;
  if (!ids || !out || (V > 0 && !weight)) return fail(HSL_ERR_ARG, "hsl_embed_fwd: null pointer");
  unsigned* err;
  HSL_CHECK(device_error_word(&err));
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_fmt(fmt, [&](auto f) {
    using T = typename Elem<decltype(f)::value>::T;
    const int per = (D + Vec<decltype(f)::value>::N - 1) / Vec<decltype(f)::value>::N;
    hipLaunchKernelGGL(embed_fwd_kernel<decltype(f)::value>, dim3((unsigned)((N * per + kBlock - 1) / kBlock)),
                       dim3(kBlock), 0, s, ids, ids64, static_cast<const T*>(weight), ldw, scale, static_cast<T*>(out),
                       (int)N, V, D, per, err);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

size_t hsl_embed_bwd_ws_bytes(long long N, int V, int D) {
  if (N < 0 || V < 0 || D < 0) return 0;
  EmbedWs w;
  return carve_embed(nullptr, 0, N, plan_embed(N, V, D), &w);
}

int hsl_embed_bwd(const void* ids, int ids64, const void* dout, long long ldd, float scale, int padding_idx,
                  void* dweight, void* ws, size_t ws_bytes, long long N, int V, int D, int fmt, void* stream) {
  HSL_CHECK(check_embed("hsl_embed_bwd", N, V, D, ldd, fmt));
  if (V == 0 || D == 0) return HSL_OK;
  if (!dweight || (N > 0 && (!ids || !dout))) return fail(HSL_ERR_ARG, "hsl_embed_bwd: null pointer");
  const EmbedPlan p = plan_embed(N, V, D);
  EmbedWs w;
  const size_t need = carve_embed(ws, ws_bytes, N, p, &w);
  if (!ws || ws_bytes < need) return fail(HSL_ERR_ARG, "hsl_embed_bwd: workspace %zu bytes, need %zu", ws_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(embed_sort_kernel, dim3(p.nclass), dim3(kSortThreads), 0, s, ids, ids64, (int)N, V, padding_idx,
                     w.s);
  return with_fmt(fmt, [&](auto f) {
    constexpr int kF = decltype(f)::value;
    using T = typename Elem<kF>::T;
    const int per = (D + Vec<kF>::N - 1) / Vec<kF>::N;
    const long long chunk_blocks = ((long long)p.nchunks * per + kBlock - 1) / kBlock;
    const long long row_blocks = ((long long)V * per + kBlock - 1) / kBlock;
    hipLaunchKernelGGL(embed_sum_kernel<kF>, dim3((unsigned)(chunk_blocks + row_blocks)), dim3(kBlock), 0, s, ids, ids64,
                       w.s, static_cast<const T*>(dout), ldd, scale, static_cast<T*>(dweight), w.partial, p.pitch, V, D,
                       per, (int)chunk_blocks);
    if (p.nchunks)
      hipLaunchKernelGGL(embed_join_kernel<kF>, dim3((D + 4 * kJoinLanes - 1) / (4 * kJoinLanes), p.nclass),
                         dim3(kBlock), 0, s, w.s, w.partial, p.pitch, scale, static_cast<T*>(dweight), D);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
