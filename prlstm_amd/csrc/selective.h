// What the selective scan's kernels share (selective_fwd.hip, selective_bwd.hip).
//   dt_t = softplus(delta_t + delta_bias) (or without softplus),
//   h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t,   h_{-1} = h0, and 0 in place of h_{t-1} at a reset,
//   y_t = sum_n c_t[n] h_t[n] + d x_t,   out_t = y_t z_t sigmoid(z_t) (or y_t).
//
// A workgroup has 64 neighbouring channels of one batch row, a lane each, and W waves of S states
// each, so the states need no cross-lane sums, b and c are the same for all lanes and y is a sum over
// the waves.  It walks the time in chunks of L steps:
//   A  every wave makes dt and dt x of L / W steps of its 64 channels from loads that a chunk before
//      has issued, and leaves them in LDS, as it does its share of b and c;
//   B  every wave runs its states over the chunk and leaves its part of y in LDS;
//   C  every wave sums, gates and stores y of the steps that it had in A.
// Steps behind the last have dt = 0 and x = 0, which keeps the state.  What bounds it is the vector units
// and the latency of their chains: 6 issue slots per state and step (v_exp_f32, at half rate, takes two), about 60
// per channel and step.  T4096 B16 D1024 N16, bf16, in a training pass: forward 572 us (551 at least), the vector
// units half of it busy (0.53 ns per 1000 states; 0.35 with 32 rows), backward 1278 (1.19), two thirds; its streams
// alone would take 110 and 190.
// Streams are read and written through buffers whose bounds drop what lies outside, without branches.
#pragma once

#include "lm.h"

namespace hsl {

constexpr int kChannels = 64;  // of a workgroup
constexpr int kMaxStates = 64;

// Waves of a workgroup and states of a wave.
template <int W_, int S_>
struct ScanShape {
  static constexpr int W = W_, S = S_, N = W * S;
  // Steps of a chunk, which is also what lies between two kept states.
  static constexpr int L = N > 32 ? 8 : 16;
  static constexpr int PS = L >= W ? L / W : 1;  // steps that a wave has in A and C
};
// The states that a call's are filled up to.
inline int scan_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }
inline int scan_chunk(int N) { return N > 32 ? 8 : 16; }

struct ScanPlan {
  int tiles, nseg, seg_steps;
};
ScanPlan plan_scan(int T, int B, int D, int N);
int check_scan(const char* who, int T, int B, int D, int N, int fmt);

struct ScanArgs {
  Stream x, delta, b, c, z, reset, dout;
  OutStream y, dx, ddelta, dz;
  const float *a, *d, *bias, *h0, *dh_n;
  float *h_n, *ck, *dh0;
  // Kept states lie as [..][B][state][D].
  float* map_h;     // of [segment]: the state behind the segment if it began with zeros
  float2* map_s;    // [segment][B][D]: its sum of dt, and whether it has a reset
  float* part_bc;   // [tile][T][B][2][states]: the tile's sums for db and dc
  float* part_a;    // [B segments][state][D]
  float* part_d;    // [B segments][2][D]
  int T, B, D, N, softplus, seg_steps, nseg;
};

// softplus and its derivative from e = exp(-|u|): log(1 + e) by v_log_f32 on w = 1 + e, whose
// rounding e - (w - 1) is put back (its factor 1 / w is near 1 where the logarithm is small).
__device__ __forceinline__ float softplus_f(float u, float e) {
  const float w = 1.f + e;
  return fmaxf(u, 0.f) + __builtin_fmaf(__builtin_amdgcn_logf(w), 0.693147182464599609375f, e - (w - 1.f));
}

// A state v behind a segment that takes it times the decay exp(a S), S the sum of the segment's dt.  The power of two
// comes apart from the rest, as a decay beyond fp32's range need not make the product that: a state of 0 stays 0 and a
// small one grows as it would step by step (a above 0, or dt below), and an infinite one stays infinite.
__device__ __forceinline__ float through_segment(float a2, float S, float v) {
  const float p = fminf(fmaxf(a2 * S, -1024.f), 1024.f), whole = __builtin_ceilf(p);
  return __builtin_ldexpf(v * exp2_f(p - whole), (int)whole);
}

// A workgroup's place, and its lane's channel (clamped into the row where `ok` is false).
template <class P>
struct ScanPlace {
  int lane, w, b, tile, ch, n0;
  bool ok;
  __device__ __forceinline__ ScanPlace(const ScanArgs& a) {
    const int tiles = (a.D + kChannels - 1) / kChannels;
    lane = threadIdx.x & 63;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    b = blockIdx.x / tiles;
    tile = blockIdx.x - b * tiles;
    ch = tile * kChannels + lane;
    ok = ch < a.D;
    ch = min(ch, a.D - 1);
    n0 = w * P::S;
  }
};

// The wave's states of the lane's channel from [B, D, N], 0 beyond.
template <class P>
__device__ __forceinline__ void load_states(const float* p, const ScanPlace<P>& q, const ScanArgs& a,
                                            float (&v)[P::S]) {
  const float* r = p + ((size_t)q.b * a.D + q.ch) * a.N + q.n0;
#pragma unroll
  for (int n = 0; n < P::S; ++n) v[n] = p && q.ok && q.n0 + n < a.N ? r[n] : 0.f;
}
template <class P>
__device__ __forceinline__ void store_states(float* p, const ScanPlace<P>& q, const ScanArgs& a,
                                             const float (&v)[P::S]) {
  float* r = p + ((size_t)q.b * a.D + q.ch) * a.N + q.n0;
#pragma unroll
  for (int n = 0; n < P::S; ++n)
    if (q.ok && q.n0 + n < a.N) r[n] = v[n];
}
// The wave's states in row `row` (of B each) of kept states.
template <class P>
__device__ __forceinline__ size_t kept_at(const ScanPlace<P>& q, const ScanArgs& a, size_t row) {
  return (row * P::N + q.n0) * a.D + q.ch;
}
template <class P>
__device__ __forceinline__ void load_kept(const float* p, const ScanPlace<P>& q, const ScanArgs& a, size_t row,
                                          float (&v)[P::S]) {
#pragma unroll
  for (int n = 0; n < P::S; ++n) v[n] = p[kept_at(q, a, row) + (size_t)n * a.D];
}
template <class P>
__device__ __forceinline__ void store_kept(float* p, const ScanPlace<P>& q, const ScanArgs& a, size_t row,
                                           const float (&v)[P::S]) {
#pragma unroll
  for (int n = 0; n < P::S; ++n) __builtin_nontemporal_store(v[n], p + kept_at(q, a, row) + (size_t)n * a.D);
}
template <class P>
__device__ __forceinline__ void load_a2(const ScanPlace<P>& q, const ScanArgs& a, float (&a2)[P::S]) {
#pragma unroll
  for (int n = 0; n < P::S; ++n) a2[n] = q.n0 + n < a.N ? a.a[(size_t)q.ch * a.N + q.n0 + n] * kLog2e : 0.f;
}

// The rows of a stream that a wave has in a chunk, one every W steps; the addresses are the wave's, so
// they cost the vector units nothing, and they move on by additions.
template <int F, class P>
struct Rows {
  using T_ = typename Elem<F>::T;
  char* p;             // of the chunk's first row
  long long row, chunk;  // bytes between the wave's rows, and between chunks
  bool there;
  template <class S>
  __device__ __forceinline__ Rows(const S& s, const ScanPlace<P>& q, int t0) {
    there = s.p != nullptr;
    row = s.st * (long long)(P::W * sizeof(T_));
    chunk = s.st * (long long)(P::L * sizeof(T_));
    p = reinterpret_cast<char*>(const_cast<void*>(static_cast<const void*>(s.p))) +
        ((t0 + q.w) * s.st + q.b * s.sb) * (long long)sizeof(T_);
  }
  __device__ __forceinline__ void move(int chunks) { p += chunks * chunk; }
  // Row i; reads as zeros, and is not stored, where `in` is false.
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int i, bool in) const {
    return __builtin_amdgcn_make_buffer_rsrc(p + i * row, (short)0, in && there ? 0x7fffffff : 0, 0x00020000);
  }
  // off: the lane's bytes from the row's start, or kOffNone.
  __device__ __forceinline__ T_ load(int i, unsigned off, bool in) const {
    if constexpr (F == kElemF32)
      return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(at(i, in), (int)off, 0, 0));
    else
      return (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(at(i, in), (int)off, 0, 0);
  }
  __device__ __forceinline__ void store(int i, unsigned off, bool in, float v) const {
    if constexpr (F == kElemF32)
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), at(i, in), (int)off, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b16(Elem<F>::down(v), at(i, in), (int)off, 0, 0);
  }
};

// Lane s: whether step t0 + s begins a sequence; the lanes' answers are put together when they are
// needed (cuts_of: bit s, the same for the whole workgroup), for that waits for the load.
template <int L>
__device__ __forceinline__ unsigned char load_cut(const Stream& reset, int t0, int te, int b, int lane) {
  unsigned char cut = 0;
  if (reset.p && lane < L && t0 + lane < te)
    cut = static_cast<const unsigned char*>(reset.p)[(t0 + lane) * reset.st + b * reset.sb];
  return cut;
}
__device__ __forceinline__ unsigned cuts_of(const Stream& reset, unsigned char cut) {
  return reset.p ? (unsigned)__ballot(cut != 0) : 0u;
}

// b and c of a chunk in LDS, [step][state], 0 beyond the last state and step.
template <int F, class P>
struct BcTile {
  using T_ = typename Elem<F>::T;
  static constexpr int kEach = (P::L * P::N + P::W * 64 - 1) / (P::W * 64);
  T_ rb[kEach], rc[kEach];
  __device__ __forceinline__ void load(const ScanArgs& a, int b, int t0, int te) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = threadIdx.x + i * P::W * 64, s = k / P::N, n = k % P::N;
      const bool in = k < P::L * P::N && t0 + s < te && n < a.N;
      const int from = min(t0, te - 1);
      const T_* const bp = static_cast<const T_*>(a.b.p) + (from * a.b.st + b * a.b.sb);
      const T_* const cp = static_cast<const T_*>(a.c.p) + (from * a.c.st + b * a.c.sb);
      const int row = in ? s : 0, m = in ? n : 0;
      rb[i] = bp[row * a.b.st + m];
      rc[i] = cp[row * a.c.st + m];
      if (!in) rb[i] = rc[i] = T_{};
    }
  }
  __device__ __forceinline__ void store(float (*sb)[P::N], float (*sc)[P::N]) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = threadIdx.x + i * P::W * 64;
      if (P::L * P::N % (P::W * 64) && k >= P::L * P::N) break;
      sb[k / P::N][k % P::N] = Elem<F>::up(rb[i]);
      sc[k / P::N][k % P::N] = Elem<F>::up(rc[i]);
    }
  }
};

// A wave's S values of b or c.
template <int S>
__device__ __forceinline__ void load_row(const float* p, float (&v)[S]) {
  if constexpr (S == 1) {
    v[0] = *p;
  } else {
    typedef float V __attribute__((ext_vector_type(S)));
    const V u = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int n = 0; n < S; ++n) v[n] = u[n];
  }
}

// z sigmoid(z), 1 where there is no z.
template <int F>
__device__ __forceinline__ float gate_of(float z, bool there) {
  return there ? z * gate_sigmoid<F>(z) : 1.f;
}

}  // namespace hsl
