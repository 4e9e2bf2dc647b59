// Selective scan, backward (selective.h has the forward's formulas and the layout).
// With dy_t the gradient of y_t and U_T = dh_n:
//   G_t = c_t dy_t + U_{t+1},  U_t = exp(dt_t a) G_t (0 at a reset),  P_t = U_t h_{t-1},
//   db_t = sum_d G_t dt_t x_t,  dc_t = sum_d dy_t h_t,  da = sum_{t, b} dt_t P_t,
//   dx_t = dt_t sum_n G_t b_t + d dy_t,  d(dt_t) = x_t sum_n G_t b_t + sum_n a P_t,  dh0 = U_0.
//
// A workgroup walks its chunks from the last to the first: it runs a chunk's steps again from the
// state that the forward kept, with every decay and state in registers, and then backwards.  The sums
// over states go through LDS as y does in the forward.  db and dc are sums over channels, which are
// lanes: four values of a step (the wave's states) are added over the four rows of 16 lanes while the
// rows are exchanged between registers, which leaves one register with a state in each row, and the 16
// such registers of a chunk are added over the 16 lanes of a row the same way (a lane keeps half of
// what it has and hands on the other half), so that each lane ends with one finished sum; about 2 issue
// slots a value instead of 6.  The workgroups' sums are added by a second kernel in their order.
#include <algorithm>

#include "selective.h"

namespace hsl {
namespace {

// A sum of many terms that keeps what its roundings lose.
struct Acc {
  float sum = 0.f, low = 0.f;
  __device__ __forceinline__ void add(float v) {
    const float u = v - low, t = sum + u;
    low = (t - sum) - u;
    sum = t;
  }
};

// The state of the wave that add16(add32(v0, v1), add32(v2, v3)) leaves in row r.
__device__ __forceinline__ int state_of_row(int r) { return (r & 1) * 2 + (r >> 1); }

template <int F, int W>
struct BwdChunk {
  static constexpr int L = chunk_steps<W>(), PS = L >= W ? L / W : 1;
  using T_ = typename Elem<F>::T;
  T_ x[PS], delta[PS], z[PS], dout[PS];
  BcTile<F, W> bc;
  unsigned cuts;
  f4 h;
  template <bool MAP>
  __device__ __forceinline__ void load(const ScanArgs& a, const ScanPlace& q, int t0, int te, size_t row4) {
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i, t = t0 + s;
      const bool in = s < L && t < te && q.ok;
      if (!MAP) x[i] = load_at<F>(a.x, t, q.b, q.ch, in);
      delta[i] = load_at<F>(a.delta, t, q.b, q.ch, in);
      z[i] = load_at<F>(a.z, t, q.b, q.ch, in && a.z.p);
      dout[i] = load_at<F>(a.dout, t, q.b, q.ch, in && a.dout.p);
    }
    bc.load(a, q.b, t0, te);
    cuts = load_cuts<L>(a.reset, t0, te, q.b, q.lane);
    if (!MAP) {
      h = f4{};
      if (q.ok) h = load4(a.ck + ((size_t)(t0 / L) * a.B + q.b) * W * a.D * kS + row4);
    }
  }
};

// U as it leaves the segments behind this one.
template <int W>
__device__ __forceinline__ void enter_reverse(const ScanArgs& a, const ScanPlace& q, int seg, const float (&a2)[kS],
                                              float (&U)[kS]) {
  load_states(a.dh_n, q, a, U);
  for (int i = a.nseg - 1; i > seg; --i) {
    const float2 m = a.map_s[((size_t)(i - 1) * a.B + q.b) * a.D + q.ch];
    const f4 v = load4(a.map_h + (((size_t)(i - 1) * a.B + q.b) * W * a.D + (size_t)q.w * a.D + q.ch) * kS);
#pragma unroll
    for (int n = 0; n < kS; ++n)
      U[n] = m.y != 0.f ? v[n] : __builtin_fmaf(segment_decay(a2[n], m.x), U[n], v[n]);
    if (!q.ok)
#pragma unroll
      for (int n = 0; n < kS; ++n) U[n] = 0.f;
  }
}

// The reverse map of segment blockIdx.y + 1.
template <int F, int W>
__global__ __launch_bounds__(W * 64) void scan_bwd_map_kernel(ScanArgs a) {
  using Chunk = BwdChunk<F, W>;
  constexpr int L = Chunk::L, PS = Chunk::PS;
  __shared__ float2 sdt[L][64];  // dt, dy
  __shared__ __attribute__((aligned(16))) float sb[L][W * kS], sc[L][W * kS];
  const ScanPlace q(a);
  const int seg = blockIdx.y + 1, tb = seg * a.seg_steps, te = min(a.T, tb + a.seg_steps);
  const size_t row4 = ((size_t)q.w * a.D + q.ch) * kS;
  float a2[kS], U[kS] = {};
  load_a2(q, a, a2);
  const float bias = a.bias ? a.bias[q.ch] : 0.f;
  Acc total;
  unsigned any = 0;
  Chunk m;
  const int first = tb + (te - tb - 1) / L * L;
  m.template load<true>(a, q, first, te, row4);
  for (int t0 = first; t0 >= tb; t0 -= L) {
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i;
      if (s >= L) break;
      const float u = Elem<F>::up(m.delta[i]) + bias, z = Elem<F>::up(m.z[i]);
      float dt = a.softplus ? softplus_f(u, exp_f(-__builtin_fabsf(u))) : u, dy = Elem<F>::up(m.dout[i]);
      if (t0 + s >= te || !q.ok) dt = 0.f;
      if (a.z.p) dy *= z * sigmoid_f(z);
      sdt[s][q.lane] = float2{dt, dy};
    }
    m.bc.store(sb, sc);
    const unsigned cuts = m.cuts;
    any |= cuts;
    lds_barrier();
    if (t0 > tb) m.template load<true>(a, q, t0 - L, te, row4);
    float part = 0.f;
#pragma unroll
    for (int s = L - 1; s >= 0; --s) {
      const float2 d = sdt[s][q.lane];
      const f4 c = load4(&sc[s][q.n0]);
#pragma unroll
      for (int n = 0; n < kS; ++n) {
        const float v = exp2_f(d.x * a2[n]) * __builtin_fmaf(c[n], d.y, U[n]);
        U[n] = cuts >> s & 1 ? 0.f : v;
      }
      part += d.x;
    }
    total.add(part);
    lds_barrier();
  }
  if (!q.ok) return;
  const f4 v = {U[0], U[1], U[2], U[3]};
  *reinterpret_cast<f4*>(a.map_h + ((size_t)blockIdx.y * a.B + q.b) * W * a.D * kS + row4) = v;
  if (q.w == 0) a.map_s[((size_t)blockIdx.y * a.B + q.b) * a.D + q.ch] = float2{total.sum, any ? 1.f : 0.f};
}

template <int F, int W>
__global__ __launch_bounds__(W * 64) void scan_bwd_kernel(ScanArgs a) {
  using Chunk = BwdChunk<F, W>;
  using T_ = typename Elem<F>::T;
  constexpr int L = Chunk::L, PS = Chunk::PS;
  __shared__ float2 sdt[L][64];  // dt, dt x
  __shared__ float sdy[L][64];
  __shared__ __attribute__((aligned(16))) float sb[L][W * kS], sc[L][W * kS];
  __shared__ float sp[3][W][L][64];  // the waves' parts of sum G b, sum a P and y
  const ScanPlace q(a);
  const int seg = blockIdx.y, tb = seg * a.seg_steps, te = min(a.T, tb + a.seg_steps);
  const size_t row4 = ((size_t)q.w * a.D + q.ch) * kS;
  const bool tail = (q.tile + 1) * kChannels > a.D;  // lanes without a channel
  float a2[kS], an[kS], U[kS];
  load_a2(q, a, a2);
#pragma unroll
  for (int n = 0; n < kS; ++n) an[n] = q.n0 + n < a.N ? a.a[(size_t)q.ch * a.N + q.n0 + n] : 0.f;
  const float bias = a.bias ? a.bias[q.ch] : 0.f, skip = a.d ? a.d[q.ch] : 0.f;
  enter_reverse<W>(a, q, seg, a2, U);
  Acc da[kS], dskip, dbias;

  Chunk m;
  // what A leaves for C
  float kx[PS], kdt[PS], ksig[PS], kdy[PS], kdo[PS], kz[PS];
  unsigned cuts = 0;
  f4 h0v{};
  auto stage = [&](int t0) {
    cuts = m.cuts;
    h0v = m.h;
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i;
      if (s >= L) break;
      const float x = Elem<F>::up(m.x[i]), u = Elem<F>::up(m.delta[i]) + bias, z = Elem<F>::up(m.z[i]);
      float dt = u, sig = 1.f, dy = Elem<F>::up(m.dout[i]);
      kdo[i] = dy;
      if (a.softplus) {
        const float e = exp_f(-__builtin_fabsf(u)), r = __builtin_amdgcn_rcpf(1.f + e);
        dt = softplus_f(u, e);
        sig = u >= 0.f ? r : e * r;
        if (u != u) sig = u;
      }
      if (t0 + s >= te || !q.ok) dt = 0.f;
      if (a.z.p) dy *= z * sigmoid_f(z);
      sdt[s][q.lane] = float2{dt, dt * x};
      sdy[s][q.lane] = dy;
      kx[i] = x;
      kdt[i] = dt;
      ksig[i] = sig;
      kdy[i] = dy;
      kz[i] = z;
    }
    m.bc.store(sb, sc);
  };
  // SLOW: a reset in the chunk, or lanes without a channel
  auto run = [&](auto slow, int t0) {
    constexpr bool SLOW = decltype(slow)::value;
    float f[L][kS], hs[L][kS], h[kS] = {h0v[0], h0v[1], h0v[2], h0v[3]};
#pragma unroll
    for (int s = 0; s < L; ++s) {
      const float2 dt = sdt[s][q.lane];
      const f4 b = load4(&sb[s][q.n0]);
#pragma unroll
      for (int n = 0; n < kS; ++n) {
        f[s][n] = exp2_f(dt.x * a2[n]);
        const float v = dt.y * b[n], g = __builtin_fmaf(f[s][n], h[n], v);
        h[n] = SLOW && (cuts >> s & 1) ? v : g;
        hs[s][n] = h[n];
      }
    }
    float rb[16], rc[16], cda[kS] = {};
#pragma unroll
    for (int s = L - 1; s >= 0; --s) {
      const float2 dt = sdt[s][q.lane];
      const float dy = sdy[s][q.lane];
      const f4 b = load4(&sb[s][q.n0]), c = load4(&sc[s][q.n0]);
      const bool cut = SLOW && (cuts >> s & 1);
      float gb = 0.f, ap = 0.f, y = 0.f, vb[kS], vc[kS];
#pragma unroll
      for (int n = 0; n < kS; ++n) {
        const float G = __builtin_fmaf(c[n], dy, U[n]);
        y = __builtin_fmaf(c[n], hs[s][n], y);
        gb = __builtin_fmaf(G, b[n], gb);
        vb[n] = G * dt.y;
        vc[n] = dy * hs[s][n];
        U[n] = G * f[s][n];
        float p = U[n] * (s ? hs[s ? s - 1 : 0][n] : h0v[n]);
        if (cut) U[n] = p = 0.f;
        ap = __builtin_fmaf(an[n], p, ap);
        cda[n] = __builtin_fmaf(dt.x, p, cda[n]);
        if (SLOW && !q.ok) vb[n] = vc[n] = 0.f;
      }
      sp[0][q.w][s][q.lane] = gb;
      sp[1][q.w][s][q.lane] = ap;
      sp[2][q.w][s][q.lane] = y;
      const float sum_b = add16(add32(vb[0], vb[1]), add32(vb[2], vb[3]));
      const float sum_c = add16(add32(vc[0], vc[1]), add32(vc[2], vc[3]));
      if constexpr (L == 16) {
        rb[s] = sum_b;
        rc[s] = sum_c;
      } else {
        rb[s] = sum_b;
        rb[8 + s] = sum_c;
      }
    }
#pragma unroll
    for (int n = 0; n < kS; ++n) da[n].add(cda[n]);
    const int i = q.lane & 15, n = q.n0 + state_of_row(q.lane >> 4);
    float* const out = a.part_bc + ((size_t)q.tile * a.T * a.B + q.b) * (2 * W * kS) + n;
    const size_t step = (size_t)a.B * (2 * W * kS);
    if constexpr (L == 16) {
      const float vb = sum_rows(rb, q.lane), vc = sum_rows(rc, q.lane);
      if (t0 + i < te) {
        out[(t0 + i) * step] = vb;
        out[(t0 + i) * step + W * kS] = vc;
      }
    } else {
      const float v = sum_rows(rb, q.lane);
      const int s = i & 7;
      if (t0 + s < te) out[(t0 + s) * step + (i >> 3) * (W * kS)] = v;
    }
  };

  const int first = te > tb ? tb + (te - tb - 1) / L * L : tb - L;
  if (te > tb) {
    m.template load<false>(a, q, first, te, row4);
    stage(first);
  }
  lds_barrier();
  for (int t0 = first; t0 >= tb; t0 -= L) {
    if (t0 > tb) m.template load<false>(a, q, t0 - L, te, row4);
    if (cuts || tail)
      run(std::true_type{}, t0);
    else
      run(std::false_type{}, t0);
    lds_barrier();
    float cskip = 0.f, cbias = 0.f;
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i, t = t0 + s;
      if (s >= L || t >= te || !q.ok) continue;
      float gb = 0.f, ap = 0.f, y = skip * kx[i];
#pragma unroll
      for (int v = 0; v < W; ++v) {
        gb += sp[0][v][s][q.lane];
        ap += sp[1][v][s][q.lane];
        y += sp[2][v][s][q.lane];
      }
      const float ddelta = __builtin_fmaf(kx[i], gb, ap) * ksig[i];
      cskip = __builtin_fmaf(kdy[i], kx[i], cskip);
      cbias += ddelta;
      const float dx = __builtin_fmaf(kdt[i], gb, skip * kdy[i]);
      static_cast<T_*>(a.dx.p)[t * a.dx.st + q.b * a.dx.sb + q.ch] = Elem<F>::down(dx);
      static_cast<T_*>(a.ddelta.p)[t * a.ddelta.st + q.b * a.ddelta.sb + q.ch] = Elem<F>::down(ddelta);
      if (a.z.p) {
        const float sg = sigmoid_f(kz[i]), slope = __builtin_fmaf(kz[i] * sg, 1.f - sg, sg);
        static_cast<T_*>(a.dz.p)[t * a.dz.st + q.b * a.dz.sb + q.ch] = Elem<F>::down(kdo[i] * y * slope);
      }
    }
    dskip.add(cskip);
    dbias.add(cbias);
    if (t0 > tb) stage(t0 - L);
    lds_barrier();
  }
  if (seg == 0 && a.dh0) store_states(a.dh0, q, a, U);
  const size_t part = (size_t)q.b * a.nseg + seg;
  if (q.ok) {
    const f4 v = {da[0].sum, da[1].sum, da[2].sum, da[3].sum};
    *reinterpret_cast<f4*>(a.part_a + part * W * a.D * kS + row4) = v;
  }
  sp[0][q.w][0][q.lane] = dskip.sum;
  sp[1][q.w][0][q.lane] = dbias.sum;
  lds_barrier();
  if (q.w == 0 && q.ok) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) {
      s0 += sp[0][v][0][q.lane];
      s1 += sp[1][v][0][q.lane];
    }
    a.part_d[part * 2 * a.D + q.ch] = s0;
    a.part_d[(part * 2 + 1) * a.D + q.ch] = s1;
  }
}

// db and dc from the tiles' sums, in the tiles' order.
template <int F>
__global__ __launch_bounds__(256) void scan_bc_kernel(const float* __restrict__ part, OutStream db, OutStream dc, int T,
                                                      int B, int N, int pad, int tiles) {
  using T_ = typename Elem<F>::T;
  const long long all = (long long)T * B * 2 * pad, stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += stride) {
    const int n = (int)(i % pad);
    if (n >= N) continue;
    const long long row = i / pad, tb = row >> 1;
    float v = 0.f;
    for (int k = 0; k < tiles; ++k) v += part[k * all + i];
    const OutStream& o = row & 1 ? dc : db;
    static_cast<T_*>(o.p)[tb / B * o.st + tb % B * o.sb + n] = Elem<F>::down(v);
  }
}

// da [D][N], dd and ddelta_bias [D] from the workgroups' sums, in fp64.
__global__ __launch_bounds__(256) void scan_sum_kernel(const float* __restrict__ part_a,
                                                       const float* __restrict__ part_d, float* da, float* dd,
                                                       float* dbias, int rows, int D, int N, int W) {
  __shared__ double sm[4][64];
  const int c = threadIdx.x & 63, strip = threadIdx.x >> 6;
  const long long na = (long long)W * D * kS, all = na + 2 * D, i = (long long)blockIdx.x * 64 + c;
  double v = 0.0;
  if (i < all)
    for (int r = strip; r < rows; r += 4)
      v += i < na ? part_a[(long long)r * na + i] : part_d[(long long)r * 2 * D + (i - na)];
  sm[strip][c] = v;
  __syncthreads();
  if (strip || i >= all) return;
  const float s = (float)((sm[0][c] + sm[1][c]) + (sm[2][c] + sm[3][c]));
  if (i < na) {
    const long long wd = i / kS;
    const int n = (int)(wd / D) * kS + (int)(i % kS);
    if (n < N) da[wd % D * N + n] = s;
  } else {
    const long long j = i - na;
    float* const o = j < D ? dd : dbias;
    if (o) o[j % D] = s;
  }
}

// The pieces of a workspace, in floats.
struct BwdLayout {
  size_t map_h, map_s, bc, a, d, all;
};
BwdLayout bwd_layout(int T, int B, int D, int N) {
  const ScanPlan p = plan_scan(T, B, D, N);
  const size_t states = (size_t)scan_waves(N) * kS, bd = (size_t)B * D;
  BwdLayout l;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off += align_up(n, 64);
    return at;
  };
  l.map_h = take((p.nseg - 1) * bd * states);
  l.map_s = take((p.nseg - 1) * bd * 2);
  l.bc = take((size_t)p.tiles * T * B * 2 * states);
  l.a = take(p.nseg * bd * states);
  l.d = take(p.nseg * bd * 2);
  l.all = off;
  return l;
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

size_t hsl_selective_bwd_ws_bytes(int T, int B, int D, int N) {
  if (check_scan("hsl_selective_bwd_ws_bytes", T, B, D, N, kElemF32) != HSL_OK || B == 0 || D == 0) return 0;
  return bwd_layout(T, B, D, N).all * sizeof(float);
}

int hsl_selective_bwd(const void* x, long long x_t, long long x_b, const void* delta, long long de_t, long long de_b,
                      const float* a, const void* b, long long b_t, long long b_b, const void* c, long long c_t,
                      long long c_b, const float* d, const void* z, long long z_t, long long z_b,
                      const float* delta_bias, const void* reset, long long rs_t, long long rs_b, const float* ck,
                      const void* dout, long long do_t, long long do_b, const float* dh_n, void* dx, long long dx_t,
                      long long dx_b, void* ddelta, long long dd_t, long long dd_b, float* da, void* db,
                      long long db_t, long long db_b, void* dc, long long dc_t, long long dc_b, float* dd, void* dz,
                      long long dz_t, long long dz_b, float* ddelta_bias, float* dh0, int softplus, void* ws,
                      size_t ws_bytes, int T, int B, int D, int N, int fmt, void* stream) {
  HSL_CHECK(check_scan("hsl_selective_bwd", T, B, D, N, fmt));
  if (D > 0 && (!a || !da || (T > 0 && B > 0 && (!x || !delta || !b || !c || !ck || !dx || !ddelta || (z && !dz)))))
    return fail(HSL_ERR_ARG, "hsl_selective_bwd: null pointer");
  if (T > 0 && B > 0 && (!db || !dc))
    return fail(HSL_ERR_ARG, "hsl_selective_bwd: null pointer");
  const size_t need = hsl_selective_bwd_ws_bytes(T, B, D, N);
  if (need && (!ws || ws_bytes < need))
    return fail(HSL_ERR_ARG, "hsl_selective_bwd: workspace %zu bytes, need %zu", ws_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const ScanPlan p = plan_scan(T, B, D, N);
  const BwdLayout l = bwd_layout(T, B, D, N);
  float* const base = static_cast<float*>(ws);
  ScanArgs g{};
  g.x = {x, x_t, x_b};
  g.delta = {delta, de_t, de_b};
  g.b = {b, b_t, b_b};
  g.c = {c, c_t, c_b};
  g.z = {z, z_t, z_b};
  g.reset = {reset, rs_t, rs_b};
  g.dout = {dout, do_t, do_b};
  g.dx = {dx, dx_t, dx_b};
  g.ddelta = {ddelta, dd_t, dd_b};
  g.dz = {dz, dz_t, dz_b};
  g.a = a;
  g.d = d;
  g.bias = delta_bias;
  g.dh_n = dh_n;
  g.dh0 = dh0;
  g.ck = const_cast<float*>(ck);
  g.map_h = base + l.map_h;
  g.map_s = reinterpret_cast<float2*>(base + l.map_s);
  g.part_bc = base + l.bc;
  g.part_a = base + l.a;
  g.part_d = base + l.d;
  g.T = T;
  g.B = B;
  g.D = D;
  g.N = N;
  g.softplus = softplus;
  g.seg_steps = p.seg_steps;
  g.nseg = p.nseg;
  const int W = scan_waves(N);
  if (B > 0)
    HSL_CHECK(with_scan(fmt, N, [&](auto F, auto WW) {
      constexpr int kF = decltype(F)::value, kW = decltype(WW)::value;
      if (p.nseg > 1 && D > 0)
        hipLaunchKernelGGL((scan_bwd_map_kernel<kF, kW>), dim3(p.tiles * B, p.nseg - 1), dim3(kW * 64), 0, s, g);
      if (D > 0)
        hipLaunchKernelGGL((scan_bwd_kernel<kF, kW>), dim3(p.tiles * B, p.nseg), dim3(kW * 64), 0, s, g);
      if (T > 0) {  // zeros where there is no channel
        const long long n = ((long long)T * B * 2 * kW * kS + 255) / 256;
        hipLaunchKernelGGL((scan_bc_kernel<kF>), dim3((unsigned)std::min<long long>(n, 1 << 20)), dim3(256), 0, s,
                           g.part_bc, OutStream{db, db_t, db_b}, OutStream{dc, dc_t, dc_b}, T, B, N, kW * kS, p.tiles);
      }
      HSL_HIP(hipGetLastError());
      return (int)HSL_OK;
    }));
  if (D == 0) return HSL_OK;
  const long long cols = (long long)W * D * kS + 2 * D;
  hipLaunchKernelGGL(scan_sum_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(256), 0, s, g.part_a, g.part_d, da, dd,
                     ddelta_bias, B * p.nseg, D, N, W);
  HSL_HIP(hipGetLastError());
  return HSL_OK;
}

}  // extern "C"
