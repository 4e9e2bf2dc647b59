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
constexpr int kMostTokens = 1 << 30;  // of the gradient: the sort's threads stay below 2^32
constexpr int kHits = 512;          // positions of a class that one wave lists in LDS
constexpr int kBlock = 256;
constexpr int kJoinLanes = 16, kJoinGroups = kBlock / kJoinLanes;  // 64 columns, 16 shares of the partials

// 16 bytes of a row at any element's alignment.
template <int F>
struct Vec {
  static constexpr int N = 16 / sizeof(typename Elem<F>::T);
  typename Elem<F>::T v[N];
};
// The vector at element o of a row of D elements.  SMALL: D is less than a vector, of which D
// elements are read and written.
template <int F, bool SMALL>
__device__ __forceinline__ Vec<F> load_vec(const typename Elem<F>::T* row, int o, int D) {
  constexpr int N = Vec<F>::N;
  Vec<F> x;
  if constexpr (!SMALL) {
    __builtin_memcpy(&x, row + o, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x.v[e] = e < D ? row[e] : Elem<F>::down(0.f);
  }
  return x;
}
template <int F, bool SMALL, bool NT = false>
__device__ __forceinline__ void store_vec(typename Elem<F>::T* row, int o, int D, const Vec<F>& x) {
  constexpr int N = Vec<F>::N;
  if constexpr (!SMALL) {
    if constexpr (NT)
      store16_nt(row + o, x);
    else
      __builtin_memcpy(row + o, &x, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < D) row[e] = x.v[e];
  }
}

// A row of D elements is `per` vectors, taken by 1 << log2g lanes (the power of two that holds
// them, a wave at most); a wave has 64 >> log2g rows at a time.
struct Rows {
  int n, D, per, log2g;
  unsigned tiles() const { return (unsigned)((per + (1 << log2g) - 1) >> log2g); }  // of columns
  // First element of vector c.  The last vector of a row ends with the row, beside its neighbour
  // where D is no multiple of a vector: both lanes compute and store the same values there.
  __device__ __forceinline__ int offset(int c, int vec) const { return max(min(c * vec, D - vec), 0); }
};
Rows rows_of(long long n, int D, int vec) {
  Rows r{(int)n, D, (D + vec - 1) / vec, 0};
  while (r.log2g < 6 && (1 << r.log2g) < r.per) ++r.log2g;
  return r;
}
// A wave has kWaveRows rounds of rows, whose ids (or ranges) are read ahead; the rounds are
// blocks * rows apart, so that the rows of frequent tokens, which are neighbours, go to different
// waves.
constexpr int kWaveRows = 4;
// Workgroups of a launch in x at most: HIP keeps the threads there in 32 bits, and wraps beyond.
constexpr unsigned kLaunchBlocks = (1u << 24) - 1;
unsigned row_blocks(const Rows& r) {
  const long long a_block = (long long)(kBlock >> r.log2g) * kWaveRows;
  return (unsigned)((r.n + a_block - 1) / a_block);
}
// The thread's row of round k (at or past r.n: none).
__device__ __forceinline__ long long row_at(const Rows& r, unsigned block, unsigned blocks, int k) {
  return ((long long)k * blocks + block) * (kBlock >> r.log2g) + (threadIdx.x >> r.log2g);
}

// The forward: a gather, bound by its rows' traffic; four rows a lane are in flight.  N65536 V131072
// D1024 bf16: 33 us for 134 MB written (4.1 TB/s) where the 41 MB of distinct rows are in the caches; 6
// more where they are not, and up to 15 more behind a pass whose stores are still on their way to memory
// (46 on average in training passes on inputs in turn).
template <int F, bool SMALL>
__global__ __launch_bounds__(kBlock) void embed_fwd_kernel(const void* __restrict__ ids, int ids64,
                                                           const typename Elem<F>::T* __restrict__ w, long long ldw,
                                                           float scale, typename Elem<F>::T* __restrict__ out, Rows r,
                                                           int V, unsigned* err) {
  constexpr int N = Vec<F>::N;
  long long id[kWaveRows];
#pragma unroll
  for (int k = 0; k < kWaveRows; ++k) {
    const long long n = row_at(r, blockIdx.x, gridDim.x, k);
    id[k] = n < r.n ? load_id(ids, ids64, n) : -1;
  }
  const int c = (blockIdx.y << r.log2g) + (threadIdx.x & ((1 << r.log2g) - 1));
  if (c >= r.per) return;
  const int o = r.offset(c, Vec<F>::N);
  Vec<F> x[kWaveRows];
#pragma unroll
  for (int k = 0; k < kWaveRows; ++k)
    if (id[k] >= 0 && id[k] < V) x[k] = load_vec<F, SMALL>(w + id[k] * ldw, o, r.D);
#pragma unroll
  for (int k = 0; k < kWaveRows; ++k) {
    const long long n = row_at(r, blockIdx.x, gridDim.x, k);
    if (n >= r.n) break;
    float f[N];
    if (id[k] >= 0 && id[k] < V) {
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = scale * Elem<F>::up(x[k].v[e]);
    } else {
      const bool beyond = id[k] >= V;
      if (beyond && c == 0) atomicOr(err, kErrId);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = beyond ? __builtin_nanf("") : 0.f;
    }
    Vec<F> y;
    down_all<F, N>(f, y.v);
    store_vec<F, SMALL>(out + n * r.D, o, r.D, y);
  }
}

// What the sort leaves.  Token v is token v >> log2c of class v mod 2^log2c.
struct Sorted {
  int2* range;  // of a token: where its positions begin and end in pos
  int* pos;     // positions by token (by class, then within it), rising within one
  int* nlong;   // of a class: its tokens of more than `chunk` positions
  int* longs;   // [class][most]
  int* count;   // positions in pos
  int log2c, chunk, most;
};

// f(i, there, id) for a wave's part of ids in rounds of 64; there: the id has a row and is not the
// padding.  The next kAhead rounds are loaded while kAhead are looked at.
template <class I, class Fn>
__device__ __forceinline__ void each_id(const I* __restrict__ ids, int lo, int hi, int V, int padding, Fn f) {
  constexpr int kAhead = 8;
  if (lo >= hi) return;
  const int lane = threadIdx.x & 63;
  I a[kAhead], b[kAhead];
  auto load = [&](int i0, I(&x)[kAhead]) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) x[k] = ids[min(i0 + k * 64 + lane, hi - 1)];
  };
  auto look = [&](int i0, const I(&x)[kAhead]) {
    using U = std::make_unsigned_t<I>;
    if (i0 + kAhead * 64 <= hi) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) f(i0 + k * 64 + lane, (U)x[k] < (U)V && x[k] != padding, (int)x[k]);
      return;
    }
    for (int k = 0; k < kAhead && i0 + k * 64 < hi; ++k) {
      I v = x[0];
#pragma unroll
      for (int u = 1; u < kAhead; ++u) v = u == k ? x[u] : v;
      const int i = i0 + k * 64 + lane;
      f(i, (U)v < (U)V && v != padding && i < hi, (int)v);
    }
  };
  load(lo, a);
  for (int i0 = lo; i0 < hi; i0 += 2 * kAhead * 64) {
    load(i0 + kAhead * 64, b);
    look(i0, a);
    load(i0 + 2 * kAhead * 64, a);
    look(i0 + kAhead * 64, b);
  }
}

// Places the positions of one round of a wave: q is the lane's token of the class (-1: none), of
// `bits` bits.  The lanes with the same token are found bit by bit, one ballot each.
__device__ __forceinline__ void place_round(int q, int i, int bits, int* cnt, int* __restrict__ pos) {
  const int lane = threadIdx.x & 63;
  unsigned long long same = __ballot(q >= 0);
  for (int b = 0; b < bits; ++b) {
    const bool set = q >> b & 1;
    const unsigned long long ones = __ballot(set);
    same &= set ? ones : ~ones;
  }
  if (q < 0) return;
  const int at = cnt[q], rank = __popcll(same & ((1ull << lane) - 1));
  pos[at + rank] = i;
  if (rank == 0) cnt[q] = at + __popcll(same);  // every lane of the wave has read it
}

// The sort of one class.  Every workgroup reads all ids (from its XCD's L2) rather than exchange
// anything with the others, so it is one launch; it is bound by the instructions of that look (65536
// int32 ids: 26 us, of which the loads alone are 4; 8192 int64 ids: 9; 700: 6).
template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const I* __restrict__ ids, int N, int V, int padding,
                                                                  Sorted s) {
  __shared__ int cnt[kSortWaves][kClassTokens];
  __shared__ int hit_i[kSortWaves][kHits];
  __shared__ short hit_q[kSortWaves][kHits];
  __shared__ int below_s[kSortWaves], scan_s[kSortWaves], nlong;
  const int lane = threadIdx.x & 63, t = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cls = blockIdx.x, mask = (1 << s.log2c) - 1;
  const int tokens = V > cls ? ((V - 1 - cls) >> s.log2c) + 1 : 0;  // of this class
  for (int u = 0; u < kSortWaves; ++u)
    if (t < tokens) cnt[u][t] = 0;
  if (t == 0) nlong = 0;
  __syncthreads();
  // the wave's part of ids, in order: its tokens' counts, the ids of smaller residues, and a list of
  // its own positions
  const int part = ((N + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int lo = min(w * part, N), hi = min(lo + part, N);
  int below = 0, hits = 0;
  each_id(ids, lo, hi, V, padding, [&](int i, bool there, int id) {
    const int c = id & mask;
    below += there && c < cls;
    const unsigned long long mine = __ballot(there && c == cls);
    if (mine == 0) return;
    if (there && c == cls) {
      const int q = id >> s.log2c, at = hits + __popcll(mine & ((1ull << lane) - 1));
      // one addition where all are of one token
      const unsigned long long ours = __ballot(q == __builtin_amdgcn_readfirstlane(q));
      if (ours != mine)
        atomicAdd(&cnt[w][q], 1);
      else if (at == hits)
        cnt[w][q] += __popcll(mine);
      if (at < kHits) {
        hit_i[w][at] = i;
        hit_q[w][at] = (short)q;
      }
    }
    hits += __popcll(mine);
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
  if (t < tokens) {
    const int v = (t << s.log2c) | cls;
    s.range[v] = {first, first + total};
    // the last class with a token ends where all positions do
    if (t == tokens - 1 && cls == min(mask, V - 1)) *s.count = first + total;
    for (int u = 0; u < kSortWaves; ++u) cnt[u][t] += first;
    if (total > s.chunk) s.longs[(size_t)cls * s.most + atomicAdd(&nlong, 1)] = v;
  }
  __syncthreads();
  if (t == 0) s.nlong[cls] = nlong;
  const int bits = 32 - __clz(max(tokens - 1, 0));
  if (hits <= kHits) {
    for (int k0 = 0; k0 < hits; k0 += 64) {
      const bool in = k0 + lane < hits;
      place_round(in ? hit_q[w][k0 + lane] : -1, in ? hit_i[w][k0 + lane] : 0, bits, cnt[w], s.pos);
    }
  } else {  // more than the list holds: the ids again, and the list as a ring of which 64 are placed at once
    int put = 0, got = 0;
    each_id(ids, lo, hi, V, padding, [&](int i, bool there, int id) {
      const unsigned long long mine = __ballot(there && (id & mask) == cls);
      if (mine == 0) return;
      if (there && (id & mask) == cls) {
        const int at = (put + __popcll(mine & ((1ull << lane) - 1))) % kHits;
        hit_i[w][at] = i;
        hit_q[w][at] = (short)(id >> s.log2c);
      }
      put += __popcll(mine);
      if (put - got >= 64) {
        const int at = (got + lane) % kHits;
        place_round(hit_q[w][at], hit_i[w][at], bits, cnt[w], s.pos);
        got += 64;
      }
    });
    const int at = (got + lane) % kHits;
    const bool in = got + lane < put;
    place_round(in ? hit_q[w][at] : -1, hit_i[w][at], bits, cnt[w], s.pos);
  }
}

// The sum of the vector at element o of dout over the sorted positions lo .. hi-1, in that order, three at a time.
template <int F, bool SMALL>
__device__ __forceinline__ void sum_positions(const int* __restrict__ pos, int lo, int hi,
                                              const typename Elem<F>::T* __restrict__ dout, long long ldd, int o, int D,
                                              float (&acc)[Vec<F>::N]) {
  constexpr int kAhead = 3;
#pragma unroll
  for (int e = 0; e < Vec<F>::N; ++e) acc[e] = 0.f;
  int p[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (lo + k < hi) p[k] = pos[lo + k];
  for (int i = lo; i < hi; i += kAhead) {
    Vec<F> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k < hi) x[k] = load_vec<F, SMALL>(dout + p[k] * ldd, o, D);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + kAhead + k < hi) p[k] = pos[i + kAhead + k];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k < hi) {
#pragma unroll
        for (int e = 0; e < Vec<F>::N; ++e) acc[e] += Elem<F>::up(x[k].v[e]);
      }
  }
}

// The sums, bound by dout read and dW written once: N65536 V131072 D1024 bf16 88 us for 403 MB (4.6
// TB/s).  Three positions a lane are in flight: with eight the registers halve the waves (138 us).
// The first blocks take a chunk of positions each round: its parts of the chunk's first and last
// token, where those are long, go to partials 2 chunk and 2 chunk + 1 (rows of `pitch`).  The others
// take the rows of dW that are not long.  NT: dout and dW exceed the caches, and dW is stored past them
// (N65536 V131072 D1024 bf16: 122 -> 85 us, as dout stays in them).
template <int F, bool SMALL, bool NT>
__global__ __launch_bounds__(kBlock) void embed_sum_kernel(const void* __restrict__ ids, int ids64, Sorted s,
                                                           const typename Elem<F>::T* __restrict__ dout, long long ldd,
                                                           float scale, typename Elem<F>::T* __restrict__ dw,
                                                           float* __restrict__ partial, int pitch, Rows r,
                                                           int chunk_blocks) {
  constexpr int N = Vec<F>::N;
  const int c = (blockIdx.y << r.log2g) + (threadIdx.x & ((1 << r.log2g) - 1));
  if (c >= r.per) return;
  const int o = r.offset(c, Vec<F>::N);
  float acc[N];
  if ((int)blockIdx.x < chunk_blocks) {
    const int k = blockIdx.x * (kBlock >> r.log2g) + (threadIdx.x >> r.log2g);
    const int lo = k * s.chunk, hi = min(lo + s.chunk, *s.count);
    if (lo >= hi) return;
    const int first = (int)load_id(ids, ids64, s.pos[lo]), last = (int)load_id(ids, ids64, s.pos[hi - 1]);
    const int2 a = s.range[first], b = s.range[last];
    const bool head = a.y - a.x > s.chunk, tail = last != first && b.y - b.x > s.chunk;
#pragma unroll
    for (int end = 0; end < 2; ++end) {
      if (end ? !tail : !head) continue;
      sum_positions<F, SMALL>(s.pos, end ? b.x : lo, end ? hi : min(hi, a.y), dout, ldd, o, r.D, acc);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (!SMALL || e < r.D) partial[(size_t)(2 * k + end) * pitch + o + e] = acc[e];
    }
    return;
  }
  const unsigned block = blockIdx.x - chunk_blocks, blocks = gridDim.x - chunk_blocks;
  int2 at[kWaveRows];
#pragma unroll
  for (int k = 0; k < kWaveRows; ++k) {
    const long long v = row_at(r, block, blocks, k);
    at[k] = v < r.n ? s.range[v] : int2{0, 0};
  }
#pragma unroll
  for (int k = 0; k < kWaveRows; ++k) {
    const long long v = row_at(r, block, blocks, k);
    if (v >= r.n || at[k].y - at[k].x > s.chunk) continue;
    sum_positions<F, SMALL>(s.pos, at[k].x, at[k].y, dout, ldd, o, r.D, acc);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= scale;
    Vec<F> y;
    down_all<F, N>(acc, y.v);
    store_vec<F, SMALL, NT>(dw + v * r.D, o, r.D, y);
  }
}

// The long rows of class blockIdx.x, 64 columns: kJoinGroups shares of a row's partials, each added in
// order, then the shares in order.  6.5 us at the size above, 3 to 4 of them the launch.
template <int F>
__global__ __launch_bounds__(kBlock) void embed_join_kernel(Sorted s, const float* __restrict__ partial, int pitch,
                                                            float scale, typename Elem<F>::T* __restrict__ dw, int D) {
  __shared__ float4 share[kJoinGroups][kJoinLanes];
  const int cls = blockIdx.x, lane = threadIdx.x % kJoinLanes, g = threadIdx.x / kJoinLanes;
  const int col = (blockIdx.y * kJoinLanes + lane) * 4;
  const int n = s.nlong[cls];
  for (int l = 0; l < n; ++l) {
    const int v = s.longs[(size_t)cls * s.most + l];
    const int2 r = s.range[v];
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
  // Short for short calls, whose time is that of one chunk; at most 4096.  us of the whole gradient, bf16
  // V32768, ids with a share of 1 / rank, chunks of 16 / 32 / 64:
  //   D256:  N500 16 / 18 / 19;  N8192 22 / 27 / 39;  N32768 34 / 42 / 60;  N65536 49 / 54 / 69
  //   D1024: N500 24 / 28 / 28;  N8192 29 / 32 / 42;  N32768 44 / 45 / 53;  N65536 70 / 65 / 69
  // (8: within 2 of 16, but 50 at N32768 D1024; at N131072 all are within 2 but 64 at D256, 117 to 104.)
  p.chunk = N <= 32768 ? 16 : 32;
  while ((long long)p.chunk * 4096 < N) p.chunk *= 2;
  p.nchunks = N > p.chunk ? (int)((N + p.chunk - 1) / p.chunk) : 0;  // no token is longer than a chunk
  p.most = (int)std::min<long long>(kClassTokens, N / p.chunk);
  p.pitch = (D + 3) / 4 * 4;
  return p;
}
struct EmbedWs {
  Sorted s;
  float* partial;
};
size_t carve_embed(void* ws, size_t cap, long long N, int V, const EmbedPlan& p, EmbedWs* o) {
  Carver c(ws, cap);
  o->s.range = c.take<int2>(V);
  o->s.pos = c.take<int>((size_t)N);
  o->s.nlong = c.take<int>(p.nclass);
  o->s.count = c.take<int>(1);
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
  if (N > 0x7FFF0000 || V > 0x7FFF0000 || D > 0x7FFF0000)
    return fail(HSL_ERR_UNSUPPORTED, "%s: N=%lld V=%d D=%d need less than 2^31 - 2^16 each", who, N, V, D);
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
    constexpr int kF = decltype(f)::value;
    using T = typename Elem<kF>::T;
    const auto kernel = D < Vec<kF>::N ? embed_fwd_kernel<kF, true> : embed_fwd_kernel<kF, false>;
    const long long most = (long long)kLaunchBlocks * (kBlock >> rows_of(N, D, Vec<kF>::N).log2g) * kWaveRows;
    for (long long n0 = 0; n0 < N; n0 += most) {
      const Rows r = rows_of(std::min(N - n0, most), D, Vec<kF>::N);
      hipLaunchKernelGGL(kernel, dim3(row_blocks(r), r.tiles()), dim3(kBlock), 0, s,
                         static_cast<const void*>(static_cast<const char*>(ids) + n0 * (ids64 ? 8 : 4)), ids64,
                         static_cast<const T*>(weight), ldw, scale, static_cast<T*>(out) + n0 * D, r, V, err);
    }
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

size_t hsl_embed_bwd_ws_bytes(long long N, int V, int D) {
  if (check_embed("hsl_embed_bwd_ws_bytes", N, V, D, D, kElemF32) != HSL_OK) return 0;
  EmbedWs w;
  return carve_embed(nullptr, 0, N, V, plan_embed(N, V, D), &w);
}

int hsl_embed_bwd(const void* ids, int ids64, const void* dout, long long ldd, float scale, int padding_idx,
                  void* dweight, void* ws, size_t ws_bytes, long long N, int V, int D, int fmt, void* stream) {
  HSL_CHECK(check_embed("hsl_embed_bwd", N, V, D, ldd, fmt));
  if (V == 0 || D == 0) return HSL_OK;
  if (!dweight || (N > 0 && (!ids || !dout))) return fail(HSL_ERR_ARG, "hsl_embed_bwd: null pointer");
  const EmbedPlan p = plan_embed(N, V, D);
  const Rows all = rows_of(V, D, fmt == kElemF32 ? Vec<kElemF32>::N : Vec<kElemBf16>::N);
  const int chunk_blocks = (p.nchunks + (kBlock >> all.log2g) - 1) / (kBlock >> all.log2g);
  if (V > kMostTokens || row_blocks(all) + chunk_blocks > kLaunchBlocks)
    return fail(HSL_ERR_UNSUPPORTED,
                "hsl_embed_bwd: V=%d D=%d are beyond one launch (V at most 2^30, dweight below 2^37 bytes)", V, D);
  EmbedWs w;
  const size_t need = carve_embed(ws, ws_bytes, N, V, p, &w);
  if (!ws || ws_bytes < need) return fail(HSL_ERR_ARG, "hsl_embed_bwd: workspace %zu bytes, need %zu", ws_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (ids64)
    hipLaunchKernelGGL(embed_sort_kernel<long long>, dim3(p.nclass), dim3(kSortThreads), 0, s,
                       static_cast<const long long*>(ids), (int)N, V, padding_idx, w.s);
  else
    hipLaunchKernelGGL(embed_sort_kernel<int>, dim3(p.nclass), dim3(kSortThreads), 0, s, static_cast<const int*>(ids),
                       (int)N, V, padding_idx, w.s);
  return with_fmt(fmt, [&](auto f) {
    constexpr int kF = decltype(f)::value;
    using T = typename Elem<kF>::T;
    const bool nt = (size_t)(N + V) * D * sizeof(T) > kCacheBytes;
    const auto sums = D < Vec<kF>::N ? embed_sum_kernel<kF, true, false>
                      : nt           ? embed_sum_kernel<kF, false, true>
                                     : embed_sum_kernel<kF, false, false>;
    hipLaunchKernelGGL(sums, dim3(chunk_blocks + row_blocks(all), all.tiles()), dim3(kBlock), 0, s, ids, ids64, w.s,
                       static_cast<const T*>(dout), ldd, scale, static_cast<T*>(dweight), w.partial, p.pitch, all,
                       chunk_blocks);
    if (p.nchunks)
      hipLaunchKernelGGL(embed_join_kernel<kF>, dim3(p.nclass, (D + 4 * kJoinLanes - 1) / (4 * kJoinLanes)),
                         dim3(kBlock), 0, s, w.s, w.partial, p.pitch, scale, static_cast<T*>(dweight), D);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
