// Selective scan, forward and one step (selective.h has the formulas and the layout).
#include <algorithm>

#include "selective.h"

namespace hsl {

// Segments: where the channels give fewer than 256 workgroups' worth of waves, the time is cut into
// segments that run as workgroups of their own, after a pass that finds each segment's state from zero
// and its sum of dt (the decay over it is exp(a times that)).
ScanPlan plan_scan(int T, int B, int D, int N) {
  ScanPlan p;
  p.tiles = (D + kChannels - 1) / kChannels;
  const int chunk = scan_chunk(N), waves = scan_waves(N);
  const int nchunks = (T + chunk - 1) / chunk;
  const long long have = (long long)p.tiles * B * waves;
  p.nseg = 1;
  p.seg_steps = std::max(1, nchunks) * chunk;
  if (have < 768 && nchunks >= 8) {
    const int want = (int)std::min<long long>(nchunks / 4, (2048 + have - 1) / std::max(1ll, have));
    const int per = (nchunks + want - 1) / want;
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
      (long long)B * ((D + kChannels - 1) / kChannels) * scan_waves(N) >= (1ll << 25))
    return fail(HSL_ERR_UNSUPPORTED,
                "%s: T=%d B=%d D=%d N=%d is beyond the kernels' 32-bit index range (needs T < 2^30, B*D < 2^27 and "
                "B*ceil(D/64)*ceil(N/4) < 2^25)",
                who, T, B, D, N);
  return HSL_OK;
}

namespace {

template <int F, int W>
struct FwdChunk {
  static constexpr int L = chunk_steps<W>(), PS = L >= W ? L / W : 1;
  using T_ = typename Elem<F>::T;
  T_ x[PS], delta[PS], z[PS];
  BcTile<F, W> bc;
  unsigned cuts;
  template <bool MAP>
  __device__ __forceinline__ void load(const ScanArgs& a, const ScanPlace& q, int t0, int te) {
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i, t = t0 + s;
      const bool in = s < L && t < te && q.ok;
      x[i] = load_at<F>(a.x, t, q.b, q.ch, in);
      delta[i] = load_at<F>(a.delta, t, q.b, q.ch, in);
      if (!MAP) z[i] = load_at<F>(a.z, t, q.b, q.ch, in && a.z.p);
    }
    bc.load(a, q.b, t0, te);
    cuts = load_cuts<L>(a.reset, t0, te, q.b, q.lane);
  }
};

// MAP: only each segment's map (nothing of the last segment, whose map nothing reads).
template <int F, int W, bool MAP>
__global__ __launch_bounds__(W * 64) void scan_fwd_kernel(ScanArgs a) {
  constexpr int L = chunk_steps<W>(), PS = FwdChunk<F, W>::PS;
  using T_ = typename Elem<F>::T;
  __shared__ float2 sdt[L][64];
  __shared__ __attribute__((aligned(16))) float sb[L][W * kS], sc[L][W * kS];
  __shared__ float sy[MAP ? 1 : W][MAP ? 1 : L][64];
  const ScanPlace q(a);
  const int seg = blockIdx.y, tb = seg * a.seg_steps, te = min(a.T, tb + a.seg_steps);
  float a2[kS], h[kS];
  load_a2(q, a, a2);
  const float bias = a.bias ? a.bias[q.ch] : 0.f, skip = a.d ? a.d[q.ch] : 0.f;
  const size_t row4 = ((size_t)q.w * a.D + q.ch) * kS, rows4 = (size_t)W * a.D * kS;  // of a [B][W][D][4]
  if (MAP) {
#pragma unroll
    for (int n = 0; n < kS; ++n) h[n] = 0.f;
  } else {
    load_states(a.h0, q, a, h);
    for (int i = 0; i < seg; ++i) {
      const float2 m = a.map_s[((size_t)i * a.B + q.b) * a.D + q.ch];
      const f4 v = load4(a.map_h + ((size_t)i * a.B + q.b) * rows4 + row4);
#pragma unroll
      for (int n = 0; n < kS; ++n)
        h[n] = m.y != 0.f ? v[n] : __builtin_fmaf(segment_decay(a2[n], m.x), h[n], v[n]);
    }
  }
  float total = 0.f, low = 0.f;  // the sum of dt and what its roundings lost
  unsigned any = 0;

  FwdChunk<F, W> now, next;
  // what A leaves for C
  float keep_x[PS], keep_z[PS];
  auto stage = [&](const FwdChunk<F, W>& m, int t0) {
    now.cuts = m.cuts;
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i;
      if (s >= L) break;
      const float x = Elem<F>::up(m.x[i]), u = Elem<F>::up(m.delta[i]) + bias;
      float dt = a.softplus ? softplus_f(u, exp_f(-__builtin_fabsf(u))) : u;
      if (t0 + s >= te || !q.ok) dt = 0.f;
      sdt[s][q.lane] = float2{dt, dt * x};
      keep_x[i] = x;
      if (!MAP) keep_z[i] = Elem<F>::up(m.z[i]);
    }
    m.bc.store(sb, sc);
  };
  auto run = [&](auto cut) {
    constexpr bool CUT = decltype(cut)::value;
    float part = 0.f;
#pragma unroll
    for (int s = 0; s < L; ++s) {
      const float2 dt = sdt[s][q.lane];
      const f4 b = load4(&sb[s][q.n0]), c = MAP ? f4{} : load4(&sc[s][q.n0]);
      const bool zero = CUT && (now.cuts >> s & 1);
      float y = 0.f;
#pragma unroll
      for (int n = 0; n < kS; ++n) {
        const float f = exp2_f(dt.x * a2[n]), v = dt.y * b[n];
        const float g = __builtin_fmaf(f, h[n], v);
        h[n] = zero ? v : g;
        if (!MAP) y = n ? __builtin_fmaf(c[n], h[n], y) : c[n] * h[n];
      }
      if (MAP) part += dt.x;
      if (!MAP) sy[q.w][s][q.lane] = y;
    }
    if (MAP) {  // compensated: thousands of small dt
      const float v = part - low, t = total + v;
      low = (t - total) - v;
      total = t;
      any |= now.cuts;
    }
  };

  if (tb < te) {
    next.template load<MAP>(a, q, tb, te);
    stage(next, tb);
  }
  lds_barrier();
  for (int t0 = tb; t0 < te; t0 += L) {
    const bool more = t0 + L < te;
    if (more) next.template load<MAP>(a, q, t0 + L, te);
    if (!MAP && a.ck && q.ok) {
      const f4 v = {h[0], h[1], h[2], h[3]};
      __builtin_nontemporal_store(v, reinterpret_cast<f4*>(a.ck + ((size_t)(t0 / L) * a.B + q.b) * rows4 + row4));
    }
    if (now.cuts)
      run(std::true_type{});
    else
      run(std::false_type{});
    lds_barrier();
    if (!MAP) {
#pragma unroll
      for (int i = 0; i < PS; ++i) {
        const int s = q.w + W * i, t = t0 + s;
        if (s >= L || t >= te || !q.ok) continue;
        float y = skip * keep_x[i];
#pragma unroll
        for (int v = 0; v < W; ++v) y += sy[v][s][q.lane];
        if (a.z.p) y *= keep_z[i] * sigmoid_f(keep_z[i]);
        static_cast<T_*>(a.y.p)[t * a.y.st + q.b * a.y.sb + q.ch] = Elem<F>::down(y);
      }
    }
    if (more) stage(next, t0 + L);
    lds_barrier();
  }
  if (MAP) {
    if (!q.ok) return;
    const f4 v = {h[0], h[1], h[2], h[3]};
    *reinterpret_cast<f4*>(a.map_h + ((size_t)seg * a.B + q.b) * rows4 + row4) = v;
    if (q.w == 0) a.map_s[((size_t)seg * a.B + q.b) * a.D + q.ch] = float2{total, any ? 1.f : 0.f};
  } else if (te == a.T) {
    store_states(a.h_n, q, a, h);
  }
}

// A single step: a group of G lanes has a channel, a lane up to four of its states.  h_n may be h0.
template <int F, int G>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a) {
  using T_ = typename Elem<F>::T;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int g = (int)(i % G);
  const long long ch = i / G;
  const bool ok = ch < (long long)a.B * a.D;  // whole groups
  const int b = ok ? (int)(ch / a.D) : 0, j = ok ? (int)(ch - (long long)b * a.D) : 0;
  const float x = Elem<F>::up(load_at<F>(a.x, 0, b, j, ok));
  const float u = Elem<F>::up(load_at<F>(a.delta, 0, b, j, ok)) + (a.bias ? a.bias[j] : 0.f);
  const float dt = a.softplus ? softplus_f(u, exp_f(-__builtin_fabsf(u))) : u;
  const bool cut = a.reset.p && static_cast<const unsigned char*>(a.reset.p)[b * a.reset.sb];
  float y = 0.f;
  if (ok) {
    const T_* const bp = static_cast<const T_*>(a.b.p) + b * a.b.sb;
    const T_* const cp = static_cast<const T_*>(a.c.p) + b * a.c.sb;
    const size_t row = (size_t)ch * a.N;
#pragma unroll
    for (int n4 = 0; n4 < kS; ++n4) {
      const int n = g * kS + n4;
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
  return (size_t)((T + chunk - 1) / chunk) * B * D * scan_waves(N) * kS;
}

size_t hsl_selective_fwd_ws_bytes(int T, int B, int D, int N) {
  if (check_scan("hsl_selective_fwd_ws_bytes", T, B, D, N, kElemF32) != HSL_OK || B == 0 || D == 0 || T == 1) return 0;
  return (size_t)(plan_scan(T, B, D, N).nseg - 1) * B * D * (scan_waves(N) * kS + 2) * sizeof(float);
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
  return with_scan(fmt, N, [&](auto F, auto WW) {
    constexpr int kF = decltype(F)::value, kW = decltype(WW)::value;
    if (step) {
      const long long n = (long long)B * D * kW;
      hipLaunchKernelGGL((scan_step_kernel<kF, kW>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, g);
    } else {
      if (p.nseg > 1) {
        g.map_s = reinterpret_cast<float2*>(g.map_h + (size_t)(p.nseg - 1) * B * D * kW * kS);
        hipLaunchKernelGGL((scan_fwd_kernel<kF, kW, true>), dim3(p.tiles * B, p.nseg - 1), dim3(kW * 64), 0, s, g);
      }
      hipLaunchKernelGGL((scan_fwd_kernel<kF, kW, false>), dim3(p.tiles * B, p.nseg), dim3(kW * 64), 0, s, g);
    }
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
