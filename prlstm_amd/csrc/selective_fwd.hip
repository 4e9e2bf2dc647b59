// Selective scan, forward and one step (selective.h has the formulas and the layout).
#include <algorithm>

#include "selective.h"

namespace hsl {

// Segments: where the channels give too few workgroups, the time is cut into segments that run as workgroups of
// their own, after a pass that finds each segment's state from zero and its sum of dt (the decay over it is exp(a
// times that)).  us with / without, forward and backward, bf16, 16 states, T4096:
//   128 workgroups 335, 813 / 491, 1239;  160: 375, 1121 / 520, 1247;  192: 491, 1461 / 520, 1252;
//   256: 603, 1511 / 527, 1271;  384, one and a half for a CU: 740, 2228 / 1030, 2490.
// Up to 8 states a workgroup has fewer than 8 waves, so more segments pay: T1024, 256 workgroups of 8 states 111, 240
// / 127, 277, of 4 states 98, 242 / 119, 320 (512: 165, 433 / 137, 341).  Not many more, as each one adds up the maps
// of those before it: 16 workgroups of 4 states in 32 segments 79, 161, in 128 103, 239.
ScanPlan plan_scan(int T, int B, int D, int N) {
  ScanPlan p;
  p.tiles = (D + kChannels - 1) / kChannels;
  const int chunk = scan_chunk(N), nchunks = (T + chunk - 1) / chunk, states = scan_states(N), waves = states / 2;
  const long long have = std::max(1ll, (long long)p.tiles * B);
  p.nseg = 1;
  p.seg_steps = std::max(1, nchunks) * chunk;
  long long want = 1;
  if (have < 192) want = (512 + have - 1) / have;
  if (states <= 8 && have <= 256) want = std::max(want, std::min(16ll, (4096 / waves + have - 1) / have));
  if (states == 16 && have > 256 && have <= 384) want = 2;
  if (want > 1 && nchunks >= 8) {
    want = std::min<long long>(want, nchunks / 4);
    const int per = (int)((nchunks + want - 1) / want);
    p.seg_steps = per * chunk;
    p.nseg = (nchunks + per - 1) / per;
  }
  return p;
}

int check_scan(const char* who, int T, int B, int D, int N, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (T < 0 || B < 0 || D < 0) return fail(HSL_ERR_ARG, "%s: negative size (T=%d B=%d D=%d)", who, T, B, D);
  if (N < 1 || N > kMaxStates) return fail(HSL_ERR_ARG, "%s: %d states, must be 1..%d", who, N, kMaxStates);
  // steps and channels are counted in 32 bits; a launch holds fewer than 2^32 threads
  if (T >= (1 << 30) || (long long)B * D >= (1ll << 27) ||
      (long long)B * ((D + kChannels - 1) / kChannels) * (scan_states(N) / 4) >= (1ll << 24))
    return fail(HSL_ERR_UNSUPPORTED,
                "%s: T=%d B=%d D=%d N=%d is beyond the kernels' 32-bit index range (needs T < 2^30, B*D < 2^27 and "
                "B*ceil(D/64)*ceil(N/4) < 2^24)",
                who, T, B, D, N);
  return HSL_OK;
}

namespace {

template <int F, class P>
struct FwdChunk {
  using T_ = typename Elem<F>::T;
  T_ x[P::PS], delta[P::PS], z[P::PS];
  BcTile<F, P> bc;
  unsigned char cut;
};

// MAP: only each segment's map (nothing of the last segment, whose map nothing reads).  Between two barriers a
// wave has C of the chunk before, B of this one and A of the next, which do not depend on each other, so the
// latency of each one's chains lies behind the others' work; what they exchange is kept twice.
template <int F, class P, bool MAP>
__global__ __launch_bounds__(P::W * 64) void scan_fwd_kernel(ScanArgs a) {
  constexpr int L = P::L, PS = P::PS, S = P::S, W = P::W;
  __shared__ float2 sdt[2][L][64];
  __shared__ __attribute__((aligned(16))) float sb[2][L][P::N], sc[2][L][P::N];
  __shared__ float sy[2][MAP ? 1 : W][MAP ? 1 : L][64];
  const ScanPlace<P> q(a);
  const unsigned off = q.ok ? q.ch * (unsigned)sizeof(typename Elem<F>::T) : kOffNone;
  const int seg = blockIdx.y, tb = seg * a.seg_steps, te = min(a.T, tb + a.seg_steps);
  const bool gated = a.z.p != nullptr, soft = a.softplus != 0;
  float a2[S], h[S];
  load_a2(q, a, a2);
  const float bias = a.bias ? a.bias[q.ch] : 0.f, skip = a.d ? a.d[q.ch] : 0.f;
  if (MAP) {
#pragma unroll
    for (int n = 0; n < S; ++n) h[n] = 0.f;
  } else {
    load_states(a.h0, q, a, h);
    for (int i = 0; i < seg; ++i) {
      const float2 m = a.map_s[((size_t)i * a.B + q.b) * a.D + q.ch];
      float v[S];
      load_kept(a.map_h, q, a, (size_t)i * a.B + q.b, v);
#pragma unroll
      for (int n = 0; n < S; ++n)
        h[n] = m.y != 0.f ? v[n] : through_segment(a2[n], m.x, h[n]) + v[n];
    }
  }
  float total = 0.f, low = 0.f;  // the sum of dt and what its roundings lost
  unsigned any = 0;

  FwdChunk<F, P> next;  // the loads of the chunk after the next
  Rows<F, P> xr(a.x, q, tb), dr(a.delta, q, tb), zr(a.z, q, tb), yr(a.y, q, tb - L);
  auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i;
      const bool in = s < L && t0 + s < te;
      next.x[i] = xr.load(i, off, in);
      next.delta[i] = dr.load(i, off, in);
      if (!MAP) next.z[i] = zr.load(i, off, in);
    }
    next.bc.load(a, q.b, t0, te);
    next.cut = load_cut<L>(a.reset, t0, te, q.b, q.lane);
    xr.move(1);
    dr.move(1);
    zr.move(1);
  };
  struct Kept {
    float x[PS], z[PS];
  } before, now, then;  // what A leaves for C
  auto stage = [&](int t0, int par) {  // A
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i;
      if (L < W && s >= L) break;
      const float x = Elem<F>::up(next.x[i]), u = Elem<F>::up(next.delta[i]) + bias;
      float dt = softplus_f(u, exp_f(-__builtin_fabsf(u)));
      dt = soft ? dt : u;
      dt = t0 + s < te && q.ok ? dt : 0.f;
      sdt[par][s][q.lane] = float2{dt, dt * x};
      then.x[i] = x;
      then.z[i] = MAP ? 0.f : Elem<F>::up(next.z[i]);
    }
    next.bc.store(sb[par], sc[par]);
  };
  auto run = [&](auto cut, int par, unsigned cuts) {  // B
    constexpr bool CUT = decltype(cut)::value;
    float part = 0.f;
#pragma unroll
    for (int s = 0; s < L; ++s) {
      const float2 dt = sdt[par][s][q.lane];
      float b[S], c[S], y = 0.f;
      load_row<S>(&sb[par][s][q.n0], b);
      if (!MAP) load_row<S>(&sc[par][s][q.n0], c);
      const bool zero = CUT && (cuts >> s & 1);
#pragma unroll
      for (int n = 0; n < S; ++n) {
        const float f = exp2_f(dt.x * a2[n]), e = dt.y * b[n];
        const float g = __builtin_fmaf(f, h[n], e);
        h[n] = zero ? e : g;
        if (!MAP) y = n ? __builtin_fmaf(c[n], h[n], y) : c[n] * h[n];
      }
      if (MAP) part += dt.x;
      if (!MAP) sy[par][q.w][s][q.lane] = y;
    }
    if (MAP) {  // compensated: thousands of small dt
      const float v = part - low, t = total + v;
      low = (t - total) - v;
      total = t;
    }
  };
  auto finish = [&](int t0, int par) {  // C
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i, t = t0 + s;
      if (L < W && s >= L) break;
      float y = skip * before.x[i];
#pragma unroll
      for (int v = 0; v < W; ++v) y += sy[par][v][s][q.lane];
      y *= gate_of<F>(before.z[i], gated);
      yr.store(i, off, t >= tb && t < te, y);
    }
    yr.move(1);
  };

  unsigned cuts = 0;
  now = Kept{};
  then = Kept{};
  if (tb < te) {
    load(tb);
    stage(tb, 0);
    cuts = cuts_of(a.reset, next.cut);
    load(tb + L);
  }
  lds_barrier();
  int par = 0;
  for (int t0 = tb; t0 < te; t0 += L, par ^= 1) {
    before = now;
    now = then;
    if (!MAP && a.ck && q.ok) store_kept(a.ck, q, a, (size_t)(t0 / L) * a.B + q.b, h);
    any |= cuts;
    auto all = [&](auto cut) {
      run(cut, par, cuts);
      if (!MAP) finish(t0 - L, par ^ 1);
      stage(t0 + L, par ^ 1);
    };
    if (cuts)
      all(std::true_type{});
    else
      all(std::false_type{});
    cuts = cuts_of(a.reset, next.cut);
    load(t0 + 2 * L);
    lds_barrier();
  }
  if (!MAP && tb < te) {
    before = now;
    finish(tb + (te - tb - 1) / L * L, par ^ 1);
  }
  if (MAP) {
    if (!q.ok) return;
    store_kept(a.map_h, q, a, (size_t)seg * a.B + q.b, h);
    if (q.w == 0) a.map_s[((size_t)seg * a.B + q.b) * a.D + q.ch] = float2{total, any ? 1.f : 0.f};
  } else if (te == a.T) {
    store_states(a.h_n, q, a, h);
  }
}

// f(integral_constant fmt, ScanShape).  16 states: four a wave where every CU gets two workgroups or more, whose
// barriers then hide behind each other, and two a wave (so twice the waves) where it gets fewer; us, bf16, four / two
// a wave: T4096 B16 D1024 (256 workgroups) 678 / 547, T1024 and 512 workgroups 191 / 250, fp16 T16383 B1 D1024 in 512
// segments' workgroups 117 / 147; one state a wave (16 waves): 658 for the first.  32 states: four a wave, 343 / 360
// at T1024 and 512 workgroups, 172 / 177 at 256.  8 states: two a wave, 125 with 196 for four and 107 for
// one at 256 workgroups, 153 with 249 and 221 at 512.  4 states: one a wave, 119 with 171 for two and 971 for four.
template <class Fn>
int with_fwd_shape(int fmt, int N, long long workgroups, Fn f) {
  return with_fmt(fmt, [&](auto F) {
    switch (scan_states(N)) {
      case 4: return f(F, ScanShape<4, 1>{});
      case 8: return f(F, ScanShape<4, 2>{});
      case 16: return workgroups >= 512 ? f(F, ScanShape<4, 4>{}) : f(F, ScanShape<8, 2>{});
      case 32: return f(F, ScanShape<8, 4>{});
      default: return f(F, ScanShape<16, 4>{});
    }
  });
}

constexpr int kStepStates = 4;  // of a lane of the single step

// A single step: a group of G lanes has a channel, a lane up to four of its states.  h_n may be h0.
template <int F, int G>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
  using T_ = typename Elem<F>::T;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int g = (int)(i % G);
  const long long ch = i / G;
  const bool ok = ch < (long long)a.B * a.D;  // whole groups
  const int b = ok ? (int)(ch / a.D) : 0, j = ok ? (int)(ch - (long long)b * a.D) : 0;
  float x = 0.f, u = 0.f;
  if (ok) {
    x = Elem<F>::up(static_cast<const T_*>(a.x.p)[b * a.x.sb + j]);
    u = Elem<F>::up(static_cast<const T_*>(a.delta.p)[b * a.delta.sb + j]) + (a.bias ? a.bias[j] : 0.f);
  }
  const float dt = a.softplus ? softplus_f(u, exp_f(-__builtin_fabsf(u))) : u;
  const bool cut = a.reset.p && static_cast<const unsigned char*>(a.reset.p)[b * a.reset.sb];
  float y = 0.f;
  if (ok) {
    const T_* const bp = static_cast<const T_*>(a.b.p) + b * a.b.sb;
    const T_* const cp = static_cast<const T_*>(a.c.p) + b * a.c.sb;
    const size_t row = (size_t)ch * a.N;
#pragma unroll
    for (int n4 = 0; n4 < kStepStates; ++n4) {
      const int n = g * kStepStates + n4;
      if (n >= a.N) break;
      float h = a.h0 && !cut ? a.h0[row + n] : 0.f;
      h = __builtin_fmaf(exp2_f(dt * (a.a[(size_t)j * a.N + n] * kLog2e)), h, dt * x * Elem<F>::up(bp[n]));
      if (cut) h = dt * x * Elem<F>::up(bp[n]);
      y = __builtin_fmaf(Elem<F>::up(cp[n]), h, y);
      a.h_n[row + n] = h;
    }
  }
#pragma unroll
  for (int m = 1; m < G; m *= 2) y += __shfl_xor(y, m);
  if (!ok || g) return;
  if (a.d) y = __builtin_fmaf(a.d[j], x, y);
  if (a.z.p) {
    const float z = Elem<F>::up(static_cast<const T_*>(a.z.p)[b * a.z.sb + j]);
    y *= z * sigmoid_f(z);
  }
  static_cast<T_*>(a.y.p)[b * a.y.sb + j] = Elem<F>::down(y);
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

size_t hsl_selective_ck_floats(int T, int B, int D, int N) {
  if (check_scan("hsl_selective_ck_floats", T, B, D, N, kElemF32) != HSL_OK) return 0;
  const int chunk = scan_chunk(N);
  return (size_t)((T + chunk - 1) / chunk) * B * D * scan_states(N);
}

size_t hsl_selective_fwd_ws_bytes(int T, int B, int D, int N) {
  if (check_scan("hsl_selective_fwd_ws_bytes", T, B, D, N, kElemF32) != HSL_OK || B == 0 || D == 0 || T == 1) return 0;
  return (size_t)(plan_scan(T, B, D, N).nseg - 1) * B * D * (scan_states(N) + 2) * sizeof(float);
}

int hsl_selective_fwd(const void* x, long long x_t, long long x_b, const void* delta, long long de_t, long long de_b,
                      const float* a, const void* b, long long b_t, long long b_b, const void* c, long long c_t,
                      long long c_b, const float* d, const void* z, long long z_t, long long z_b,
                      const float* delta_bias, const float* h0, const void* reset, long long rs_t, long long rs_b,
                      void* out, long long out_t, long long out_b, float* h_n, float* ck, int softplus, void* ws,
                      size_t ws_bytes, int T, int B, int D, int N, int fmt, void* stream) {
  HSL_CHECK(check_scan("hsl_selective_fwd", T, B, D, N, fmt));
  if (B == 0 || D == 0) return HSL_OK;
  if (!a || !h_n || (T > 0 && (!x || !delta || !b || !c || !out)))
    return fail(HSL_ERR_ARG, "hsl_selective_fwd: null pointer");
  const bool step = T == 1 && !ck;
  const ScanPlan p = plan_scan(T, B, D, N);
  const size_t need = step ? 0 : hsl_selective_fwd_ws_bytes(T, B, D, N);
  if (need && (!ws || ws_bytes < need))
    return fail(HSL_ERR_ARG, "hsl_selective_fwd: workspace %zu bytes, need %zu", ws_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ScanArgs g{};
  g.x = {x, x_t, x_b};
  g.delta = {delta, de_t, de_b};
  g.b = {b, b_t, b_b};
  g.c = {c, c_t, c_b};
  g.z = {z, z_t, z_b};
  g.reset = {reset, rs_t, rs_b};
  g.y = {out, out_t, out_b};
  g.a = a;
  g.d = d;
  g.bias = delta_bias;
  g.h0 = h0;
  g.h_n = h_n;
  g.ck = ck;
  g.T = T;
  g.B = B;
  g.D = D;
  g.N = N;
  g.softplus = softplus;
  g.seg_steps = p.seg_steps;
  g.nseg = p.nseg;
  g.map_h = static_cast<float*>(ws);
  return with_fwd_shape(fmt, N, (long long)p.tiles * B * p.nseg, [&](auto F, auto shape) {
    constexpr int kF = decltype(F)::value;
    using P = decltype(shape);
    if (step) {
      constexpr int kLanes = P::N / kStepStates;  // of a channel
      const long long n = (long long)B * D * kLanes;
      hipLaunchKernelGGL((scan_step_kernel<kF, kLanes>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, g);
    } else {
      if (p.nseg > 1) {
        g.map_s = reinterpret_cast<float2*>(g.map_h + (size_t)(p.nseg - 1) * B * D * P::N);
        hipLaunchKernelGGL((scan_fwd_kernel<kF, P, true>), dim3(p.tiles * B, p.nseg - 1), dim3(P::W * 64), 0, s, g);
      }
      hipLaunchKernelGGL((scan_fwd_kernel<kF, P, false>), dim3(p.tiles * B, p.nseg), dim3(P::W * 64), 0, s, g);
    }
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
