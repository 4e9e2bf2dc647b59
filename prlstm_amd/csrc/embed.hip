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
#include <algorithm>

#include "lm.h"

namespace hsl {
namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kClassTokens = 512;  // tokens of one workgroup at most (its counters: 16 waves of them)

// Residue classes: a power of two, so that an id's class is its low bits.
int embed_classes(int V) {
  int c = 64;
  while ((long long)c * kClassTokens < V) c *= 2;
  return c;
}

template <int F>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const void* __restrict__ ids, int ids64,
                                                        const typename Elem<F>::T* __restrict__ w, long long ldw,
                                                        float scale, typename Elem<F>::T* __restrict__ out, int V,
                                                        int D, unsigned* err) {
  const size_t n = blockIdx.x;
  const long long id = load_id(ids, ids64, n);
  const bool beyond = id >= V;
  if (beyond && threadIdx.x == 0) atomicOr(err, kErrId);
  for (int d = threadIdx.x; d < D; d += 256) {
    float v = 0.f;
    if (beyond) v = __builtin_nanf("");
    else if (id >= 0) v = scale * Elem<F>::up(w[(size_t)id * ldw + d]);
    out[n * D + d] = Elem<F>::down(v);
  }
}

// Positions by token: start[w * kClassTokens + q] is where the list of token q * nclass + w
// begins in pos, and the next entry where it ends (a class has kClassTokens + 1 entries).
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const void* __restrict__ ids, int ids64, int N,
                                                                  int V, int nclass, int padding,
                                                                  int* __restrict__ start, int* __restrict__ pos) {
  __shared__ int cnt[kSortWaves][kClassTokens];
  __shared__ int below_s[kSortWaves];
  __shared__ int scan[kClassTokens];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int cls = blockIdx.x, log2c = 31 - __clz(nclass);
  const int tokens = (V - cls + nclass - 1) / nclass;  // of this class (0 when V <= cls)
  for (int i = threadIdx.x; i < kSortWaves * kClassTokens; i += kSortThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  // the wave's part of ids, in order
  const int part = ((N + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int lo = min(w * part, N), hi = min(lo + part, N);
  int below = 0;
  for (int i = lo + lane; i < hi; i += 64) {
    const long long id = load_id(ids, ids64, i);
    if (id < 0 || id >= V || id == padding) continue;
    const int c = (int)id & (nclass - 1);
    below += c < cls;
    if (c == cls) atomicAdd(&cnt[w][(int)id >> log2c], 1);
  }
  for (int d = 32; d; d >>= 1) below += __shfl_xor(below, d);
  if (lane == 0) below_s[w] = below;
  __syncthreads();
  int base = 0;
  for (int u = 0; u < kSortWaves; ++u) base += below_s[u];
  // token totals, their exclusive sums, and each wave's place within a token's list
  int total = 0;
  if (threadIdx.x < kClassTokens) {
    for (int u = 0; u < kSortWaves; ++u) {
      const int c = cnt[u][threadIdx.x];
      cnt[u][threadIdx.x] = total;
      total += c;
    }
    scan[threadIdx.x] = total;
  }
  __syncthreads();
  for (int d = 1; d < kClassTokens; d *= 2) {
    int v = 0;
    if (threadIdx.x < kClassTokens && (int)threadIdx.x >= d) v = scan[threadIdx.x - d];
    __syncthreads();
    if (threadIdx.x < kClassTokens) scan[threadIdx.x] += v;
    __syncthreads();
  }
  int* const st = start + (size_t)cls * (kClassTokens + 1);
  if (threadIdx.x < kClassTokens) {
    const int first = base + scan[threadIdx.x] - total;
    st[threadIdx.x] = first;
    for (int u = 0; u < kSortWaves; ++u) cnt[u][threadIdx.x] += first;
    if (threadIdx.x == kClassTokens - 1) st[kClassTokens] = first + total;
  }
  __syncthreads();
  if (tokens <= 0) return;
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const int i = i0 + lane;
    const long long id = i < hi ? load_id(ids, ids64, i) : -1;
    const bool mine = id >= 0 && id < V && id != padding && ((int)id & (nclass - 1)) == cls;
    const int q = mine ? (int)id >> log2c : -1;
    unsigned long long left = __ballot(mine);
    while (left) {  // the tokens of these 64 positions, one after the other
      const int t = __shfl(q, __ffsll(left) - 1);
      const unsigned long long same = __ballot(q == t);
      if (q == t) {
        const int rank = __popcll(same & ((1ull << lane) - 1));
        pos[cnt[w][t] + rank] = i;
        if (rank == 0) cnt[w][t] += __popcll(same);  // read above by every lane of the wave first
      }
      left &= ~same;
    }
  }
}

// One workgroup per row of dW.
template <int F>
__global__ __launch_bounds__(256) void embed_sum_kernel(const int* __restrict__ start, const int* __restrict__ pos,
                                                        const typename Elem<F>::T* __restrict__ dout, long long ldd,
                                                        float scale, typename Elem<F>::T* __restrict__ dw, int nclass,
                                                        int D) {
  const int v = blockIdx.x, cls = v & (nclass - 1), q = v / nclass;
  const int* const st = start + (size_t)cls * (kClassTokens + 1) + q;
  const int lo = st[0], hi = st[1];
  for (int d = threadIdx.x; d < D; d += 256) {
    float s = 0.f;
    for (int i = lo; i < hi; ++i) s += Elem<F>::up(dout[(size_t)pos[i] * ldd + d]);
    dw[(size_t)v * D + d] = Elem<F>::down(scale * s);
  }
}

struct EmbedWs {
  int* start;
  int* pos;
};
size_t carve_embed(void* ws, size_t cap, long long N, int V, EmbedWs* o) {
  Carver c(ws, cap);
  o->start = c.take<int>((size_t)embed_classes(V) * (kClassTokens + 1));
  o->pos = c.take<int>((size_t)N);
  return align_up(c.off, 256);
}

int check_embed(const char* who, long long N, int V, int D, long long ld, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (N < 0 || V < 0 || D < 0 || ld < 0) return fail(HSL_ERR_ARG, "%s: negative size (N=%lld V=%d D=%d)", who, N, V, D);
  if (N >= (1ll << 31)) return fail(HSL_ERR_UNSUPPORTED, "%s: N=%lld ids need 2^31 > N", who, N);
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
    hipLaunchKernelGGL(embed_fwd_kernel<decltype(f)::value>, dim3((unsigned)N), dim3(256), 0, s, ids, ids64,
                       static_cast<const T*>(weight), ldw, scale, static_cast<T*>(out), V, D, err);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

size_t hsl_embed_bwd_ws_bytes(long long N, int V, int D) {
  if (N < 0 || V < 0 || D < 0) return 0;
  EmbedWs w;
  return carve_embed(nullptr, 0, N, V, &w);
}

int hsl_embed_bwd(const void* ids, int ids64, const void* dout, long long ldd, float scale, int padding_idx,
                  void* dweight, void* ws, size_t ws_bytes, long long N, int V, int D, int fmt, void* stream) {
  HSL_CHECK(check_embed("hsl_embed_bwd", N, V, D, ldd, fmt));
  if (V == 0 || D == 0) return HSL_OK;
  if (!dweight || (N > 0 && (!ids || !dout))) return fail(HSL_ERR_ARG, "hsl_embed_bwd: null pointer");
  EmbedWs w;
  const size_t need = carve_embed(ws, ws_bytes, N, V, &w);
  if (!ws || ws_bytes < need) return fail(HSL_ERR_ARG, "hsl_embed_bwd: workspace %zu bytes, need %zu", ws_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int nclass = embed_classes(V);
  hipLaunchKernelGGL(embed_sort_kernel, dim3(nclass), dim3(kSortThreads), 0, s, ids, ids64, (int)N, V, nclass,
                     padding_idx, w.start, w.pos);
  return with_fmt(fmt, [&](auto f) {
    using T = typename Elem<decltype(f)::value>::T;
    hipLaunchKernelGGL(embed_sum_kernel<decltype(f)::value>, dim3(V), dim3(256), 0, s, w.start, w.pos,
                       static_cast<const T*>(dout), ldd, scale, static_cast<T*>(dweight), nclass, D);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
