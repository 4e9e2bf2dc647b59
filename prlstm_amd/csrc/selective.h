// What the selective scan's kernels share (selective_fwd.hip, selective_bwd.hip).
//   dt_t = softplus(delta_t + delta_bias) (or without softplus),
//   h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t,   h_{-1} = h0, and 0 in place of h_{t-1} at a reset,
//   y_t = sum_n c_t[n] h_t[n] + d x_t,   out_t = y_t z_t sigmoid(z_t) (or y_t).
//
// A workgroup has 64 neighbouring channels of one batch row, a lane each, and W waves of kS = 4 states
// each, so the states need no cross-lane sums, b and c are the same for all lanes and y is a sum over
// the waves.  It walks the time in chunks of L steps:
//   A  every wave makes dt and dt x of L / W steps of its 64 channels from loads that a chunk before
//      has issued, and leaves them in LDS, as it does its share of b and c;
//   B  every wave runs its states over the chunk and leaves its part of y in LDS;
//   C  every wave sums, gates and stores y of the steps that it had in A.
// Steps behind the last have dt = 0 and x = 0, which keeps the state.  What bounds it is the vector
// units: 8 issue slots per state and step (v_exp_f32 takes four), about 60 per channel and step.
#pragma once

#include "lm.h"

namespace hsl {

constexpr int kS = 4;          // states of a wave
constexpr int kChannels = 64;  // of a workgroup
constexpr int kMaxStates = 64;

// Steps of a chunk, which is also what lies between two kept states.  Sixteen waves have 128
// registers each, which hold the backward's copy of 8 steps.
template <int W>
constexpr int chunk_steps() {
  return W == 16 ? 8 : 16;
}
inline int scan_waves(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
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
  float* map_h;     // [segment][B][W][D][4]: the state behind the segment if it began with zeros
  float2* map_s;    // [segment][B][D]: its sum of dt, and whether it has a reset
  float* part_bc;   // [tile][T][B][2][4 W]: the tile's sums for db and dc
  float* part_a;    // [B segments][W][D][4]
  float* part_d;    // [B segments][2][D]
  int T, B, D, N, softplus, seg_steps, nseg;
};

// softplus and its derivative from e = exp(-|u|): log(1 + e) by v_log_f32 on w = 1 + e, whose
// rounding e - (w - 1) is put back (its factor 1 / w is near 1 where the logarithm is small).
__device__ __forceinline__ float softplus_f(float u, float e) {
  const float w = 1.f + e;
  return fmaxf(u, 0.f) + __builtin_fmaf(__builtin_amdgcn_logf(w), 0.693147182464599609375f, e - (w - 1.f));
}

__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269502162933349609375f;

// The decay exp(a S) of a segment whose dt sum to S.  One that underflows is held at the smallest
// number, so that an infinite state stays infinite.
__device__ __forceinline__ float segment_decay(float a2, float S) {
  return fmaxf(exp2_f(a2 * S), __uint_as_float(1u));
}

// A workgroup's place, and its lane's channel (clamped into the row where `ok` is false).
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
    n0 = w * kS;
  }
};

// The wave's states of the lane's channel from [.., D, N], 0 beyond.
__device__ __forceinline__ void load_states(const float* p, const ScanPlace& q, const ScanArgs& a, float (&v)[kS]) {
  const float* r = p + ((size_t)q.b * a.D + q.ch) * a.N + q.n0;
#pragma unroll
  for (int n = 0; n < kS; ++n) v[n] = p && q.ok && q.n0 + n < a.N ? r[n] : 0.f;
}
__device__ __forceinline__ void store_states(float* p, const ScanPlace& q, const ScanArgs& a, const float (&v)[kS]) {
  float* r = p + ((size_t)q.b * a.D + q.ch) * a.N + q.n0;
#pragma unroll
  for (int n = 0; n < kS; ++n)
    if (q.ok && q.n0 + n < a.N) r[n] = v[n];
}
__device__ __forceinline__ void load_a2(const ScanPlace& q, const ScanArgs& a, float (&a2)[kS]) {
#pragma unroll
  for (int n = 0; n < kS; ++n) a2[n] = q.n0 + n < a.N ? a.a[(size_t)q.ch * a.N + q.n0 + n] * kLog2e : 0.f;
}

// One element of a stream per lane; 0 where `in` is false.
template <int F>
__device__ __forceinline__ typename Elem<F>::T load_at(const Stream& s, int t, int b, int j, bool in) {
  using T_ = typename Elem<F>::T;
  return in ? static_cast<const T_*>(s.p)[t * s.st + b * s.sb + j] : T_{};
}

// Bit s: whether step t0 + s begins a sequence (the same for the whole workgroup).
template <int L>
__device__ __forceinline__ unsigned load_cuts(const Stream& reset, int t0, int te, int b, int lane) {
  if (!reset.p) return 0;
  const bool cut = lane < L && t0 + lane < te &&
                   static_cast<const unsigned char*>(reset.p)[(t0 + lane) * reset.st + b * reset.sb] != 0;
  return (unsigned)__ballot(cut);
}

// b and c of a chunk in LDS, [step][state], 0 beyond the last state and step.
template <int F, int W>
struct BcTile {
  static constexpr int L = chunk_steps<W>(), kN = W * kS, kEach = (L * kN + W * 64 - 1) / (W * 64);
  typename Elem<F>::T rb[kEach], rc[kEach];
  __device__ __forceinline__ void load(const ScanArgs& a, int b, int t0, int te) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = threadIdx.x + i * W * 64, s = k / kN, n = k % kN;
      const bool in = k < L * kN && t0 + s < te && n < a.N;
      rb[i] = load_at<F>(a.b, t0 + s, b, n, in);
      rc[i] = load_at<F>(a.c, t0 + s, b, n, in);
    }
  }
  __device__ __forceinline__ void store(float (*sb)[kN], float (*sc)[kN]) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = threadIdx.x + i * W * 64;
      if (k >= L * kN) break;
      sb[k / kN][k % kN] = Elem<F>::up(rb[i]);
      sc[k / kN][k % kN] = Elem<F>::up(rc[i]);
    }
  }
};

__device__ __forceinline__ f4 load4(const float* p) { return *reinterpret_cast<const f4*>(p); }

// f(integral_constant fmt, integral_constant waves).
template <class Fn>
int with_scan(int fmt, int N, Fn f) {
  return with_fmt(fmt, [&](auto F) {
    switch (scan_waves(N)) {
      case 1: return f(F, std::integral_constant<int, 1>{});
      case 2: return f(F, std::integral_constant<int, 2>{});
      case 4: return f(F, std::integral_constant<int, 4>{});
      case 8: return f(F, std::integral_constant<int, 8>{});
      default: return f(F, std::integral_constant<int, 16>{});
    }
  });
}

}  // namespace hsl
