// Selective scan, backward (selective.h has the forward's formulas and the layout).
// With dy_t the gradient of y_t and U_T = dh_n:
//   G_t = c_t dy_t + U_{t+1},  U_t = exp(dt_t a) G_t (0 at a reset),  P_t = U_t h_{t-1},
//   db_t = sum_d G_t dt_t x_t,  dc_t = sum_d dy_t h_t,  da = sum_{t, b} dt_t P_t,
//   dx_t = dt_t sum_n G_t b_t + d dy_t,  d(dt_t) = x_t sum_n G_t b_t + sum_n a P_t,  dh0 = U_0.
//
// A workgroup walks its chunks from the last to the first: it runs a chunk's steps again from the
// state that the forward kept, with every decay and state in registers, and then backwards.  The sums
// over states go through LDS as y does in the forward.  db and dc are sums over channels, which are
// lanes: four values of a step are added over the four rows of 16 lanes while the rows are exchanged
// between registers, which leaves one register with a value in each row, and the 16 such registers of a
// chunk are added over the 16 lanes of a row the same way (a lane keeps half of what it has and hands on
// the other half), so that each lane ends with one finished sum; about 2 issue slots a value instead
// of 6.  The workgroups' sums are added by a second kernel in their order.
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

template <int F, class P>
struct BwdChunk {
  using T_ = typename Elem<F>::T;
  T_ x[P::PS], delta[P::PS], z[P::PS], dout[P::PS];
  BcTile<F, P> bc;
  unsigned char cut;
  float h[P::S];
};

// The streams' rows of a wave, from the chunk that is loaded next, towards the first.
template <int F, class P, bool MAP>
struct BwdRows {
  Rows<F, P> x, delta, z, dout;
  __device__ __forceinline__ BwdRows(const ScanArgs& a, const ScanPlace<P>& q, int t0)
      : x(a.x, q, t0), delta(a.delta, q, t0), z(a.z, q, t0), dout(a.dout, q, t0) {}
  __device__ __forceinline__ void load(const ScanArgs& a, const ScanPlace<P>& q, unsigned off, int t0, int te,
                                       BwdChunk<F, P>& m) {
#pragma unroll
    for (int i = 0; i < P::PS; ++i) {
      const int s = q.w + P::W * i;
      const bool in = s < P::L && t0 + s < te;
      if (!MAP) m.x[i] = x.load(i, off, in);
      m.delta[i] = delta.load(i, off, in);
      m.z[i] = z.load(i, off, in);
      m.dout[i] = dout.load(i, off, in);
    }
    m.bc.load(a, q.b, t0, te);
    m.cut = load_cut<P::L>(a.reset, t0, te, q.b, q.lane);
    if (!MAP) load_kept(a.ck, q, a, (size_t)(t0 / P::L) * a.B + q.b, m.h);
    x.move(-1);
    delta.move(-1);
    z.move(-1);
    dout.move(-1);
  }
};

// U as it leaves the segments behind this one.
template <class P>
__device__ __forceinline__ void enter_reverse(const ScanArgs& a, const ScanPlace<P>& q, int seg,
                                              const float (&a2)[P::S], float (&U)[P::S]) {
  load_states(a.dh_n, q, a, U);
  for (int i = a.nseg - 1; i > seg; --i) {
    const float2 m = a.map_s[((size_t)(i - 1) * a.B + q.b) * a.D + q.ch];
    float v[P::S];
    load_kept(a.map_h, q, a, (size_t)(i - 1) * a.B + q.b, v);
#pragma unroll
    for (int n = 0; n < P::S; ++n) {
      const float u = m.y != 0.f ? v[n] : through_segment(a2[n], m.x, U[n]) + v[n];
      U[n] = q.ok ? u : 0.f;
    }
  }
}

// The reverse map of segment blockIdx.y + 1.
template <int F, class P>
__global__ __launch_bounds__(P::W * 64) void scan_bwd_map_kernel(ScanArgs a) {
  constexpr int L = P::L, S = P::S;
  __shared__ float2 sdt[L][64];  // dt, dy
  __shared__ __attribute__((aligned(32))) float sb[L][P::N], sc[L][P::N];
  const ScanPlace<P> q(a);
  const unsigned off = q.ok ? q.ch * (unsigned)sizeof(typename Elem<F>::T) : kOffNone;
  const int seg = blockIdx.y + 1, tb = seg * a.seg_steps, te = min(a.T, tb + a.seg_steps);
  const bool gated = a.z.p != nullptr, soft = a.softplus != 0;
  float a2[S], U[S] = {};
  load_a2(q, a, a2);
  const float bias = a.bias ? a.bias[q.ch] : 0.f;
  Acc total;
  unsigned any = 0;
  BwdChunk<F, P> m;
  const int first = tb + (te - tb - 1) / L * L;
  BwdRows<F, P, true> rows(a, q, first);
  rows.load(a, q, off, first, te, m);
  for (int t0 = first; t0 >= tb; t0 -= L) {
#pragma unroll
    for (int i = 0; i < P::PS; ++i) {
      const int s = q.w + P::W * i;
      if (L < P::W && s >= L) break;
      const float u = Elem<F>::up(m.delta[i]) + bias;
      float dt = softplus_f(u, exp_f(-__builtin_fabsf(u)));
      dt = soft ? dt : u;
      dt = t0 + s < te && q.ok ? dt : 0.f;
      sdt[s][q.lane] = float2{dt, Elem<F>::up(m.dout[i]) * gate_of<F>(Elem<F>::up(m.z[i]), gated)};
    }
    m.bc.store(sb, sc);
    const unsigned cuts = cuts_of(a.reset, m.cut);
    any |= cuts;
    lds_barrier();
    if (t0 > tb) rows.load(a, q, off, t0 - L, te, m);
    float part = 0.f;
#pragma unroll
    for (int s = L - 1; s >= 0; --s) {
      const float2 d = sdt[s][q.lane];
      float c[S];
      load_row<S>(&sc[s][q.n0], c);
#pragma unroll
      for (int n = 0; n < S; ++n) {
        const float v = exp2_f(d.x * a2[n]) * __builtin_fmaf(c[n], d.y, U[n]);
        U[n] = cuts >> s & 1 ? 0.f : v;
      }
      part += d.x;
    }
    total.add(part);
    lds_barrier();
  }
  if (!q.ok) return;
  store_kept(a.map_h, q, a, (size_t)blockIdx.y * a.B + q.b, U);
  if (q.w == 0) a.map_s[((size_t)blockIdx.y * a.B + q.b) * a.D + q.ch] = float2{total.sum, any ? 1.f : 0.f};
}

template <int F, class P>
__global__ __launch_bounds__(P::W * 64) void scan_bwd_kernel(ScanArgs a) {
  constexpr int L = P::L, PS = P::PS, S = P::S, W = P::W;
  __shared__ float2 sdt[L][64];  // dt, dt x
  __shared__ float sdy[L][64];
  __shared__ __attribute__((aligned(32))) float sb[L][P::N], sc[L][P::N];
  __shared__ float sp[3][W][L][64];  // the waves' parts of sum G b, sum a P and y
  const ScanPlace<P> q(a);
  const unsigned off = q.ok ? q.ch * (unsigned)sizeof(typename Elem<F>::T) : kOffNone;
  const int seg = blockIdx.y, tb = seg * a.seg_steps, te = min(a.T, tb + a.seg_steps);
  const bool gated = a.z.p != nullptr, soft = a.softplus != 0;
  const bool tail = (q.tile + 1) * kChannels > a.D;  // lanes without a channel
  float a2[S], an[S], U[S];
  load_a2(q, a, a2);
#pragma unroll
  for (int n = 0; n < S; ++n) an[n] = q.n0 + n < a.N ? a.a[(size_t)q.ch * a.N + q.n0 + n] : 0.f;
  const float bias = a.bias ? a.bias[q.ch] : 0.f, skip = a.d ? a.d[q.ch] : 0.f;
  enter_reverse(a, q, seg, a2, U);
  Acc da[S], dskip, dbias;

  BwdChunk<F, P> m;  // the loads of the next chunk
  // what A leaves for C
  float kx[PS], kdt[PS], ksig[PS], kdo[PS], kz[PS];
  unsigned cuts = 0;
  float hin[S];
  auto stage = [&](int t0) {
    cuts = cuts_of(a.reset, m.cut);
#pragma unroll
    for (int n = 0; n < S; ++n) hin[n] = q.ok ? m.h[n] : 0.f;
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i;
      if (L < W && s >= L) break;
      const float x = Elem<F>::up(m.x[i]), u = Elem<F>::up(m.delta[i]) + bias;
      const float e = exp_f(-__builtin_fabsf(u)), r = __builtin_amdgcn_rcpf(1.f + e);
      float dt = softplus_f(u, e), sig = u >= 0.f ? r : e * r;
      dt = soft ? dt : u;
      ksig[i] = soft ? sig : 1.f;
      dt = t0 + s < te && q.ok ? dt : 0.f;
      kdo[i] = Elem<F>::up(m.dout[i]);
      kz[i] = Elem<F>::up(m.z[i]);
      sdt[s][q.lane] = float2{dt, dt * x};
      sdy[s][q.lane] = kdo[i] * gate_of<F>(kz[i], gated);
      kx[i] = x;
      kdt[i] = dt;
    }
    m.bc.store(sb, sc);
  };
  // A chunk's steps forwards with their decays and states kept, then backwards: in two parts where four states a wave
  // would not leave the registers for all of it, in four where eight are (a part's steps run once more for each part
  // behind it).
  // SLOW: a reset in the chunk, or lanes without a channel
  constexpr int kParts = S == 8 ? 4 : S == 4 ? 2 : 1, H = L / kParts;
  constexpr int G = S >= 4 ? 1 : 4;  // steps whose operands are read from LDS ahead
  auto run = [&](auto slow, int t0) {
    constexpr bool SLOW = decltype(slow)::value;
    float f[H][S], hs[H][S], start[S], cda[S] = {};
    // the states behind steps s0 .. s0 + H - 1, from `start`
    auto forwards = [&](int s0, auto keep) {
      constexpr bool KEEP = decltype(keep)::value;
      struct Ahead {
        float2 dt[G];
        float b[G][S];
      } r[2];
      auto read = [&](int s1, Ahead& v) {
#pragma unroll
        for (int s = 0; s < G; ++s) {
          v.dt[s] = sdt[s1 + s][q.lane];
          load_row<S>(&sb[s1 + s][q.n0], v.b[s]);
        }
      };
      float h[S];
#pragma unroll
      for (int n = 0; n < S; ++n) h[n] = start[n];
      read(s0, r[0]);
#pragma unroll
      for (int g = 0; g < H; g += G) {
        if (g + G < H) read(s0 + g + G, r[(g / G + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead
        const Ahead& v = r[(g / G) & 1];
#pragma unroll
        for (int k = 0; k < G; ++k)
#pragma unroll
          for (int n = 0; n < S; ++n) {
            const float decay = exp2_f(v.dt[k].x * a2[n]), e = v.dt[k].y * v.b[k][n];
            const float w = __builtin_fmaf(decay, h[n], e);
            h[n] = SLOW && (cuts >> (s0 + g + k) & 1) ? e : w;
            if (KEEP) {
              f[g + k][n] = decay;
              hs[g + k][n] = h[n];
            }
          }
      }
      if (!KEEP) {
#pragma unroll
        for (int n = 0; n < S; ++n) start[n] = h[n];
      }
    };
    // Sums over rows, four values each; they are finished when there are 16.
    static_assert(L * S / 2 % 16 == 0 && (H * S / 2 % 16 == 0 || 16 % (H * S / 2) == 0), "sum_rows takes 16");
    float sums[16];
    auto finish_sums = [&](int s0) {
      const int row = q.lane >> 4;
      float* const out = a.part_bc + (((size_t)q.tile * a.T + t0) * a.B + q.b) * (2 * P::N) + (row & 1) * P::N +
                         q.n0 + (row >> 1);
      const float v = sum_rows(sums, q.lane);
      const int r = q.lane & 15, s = s0 + r / (S / 2), n = r % (S / 2) * 2;
      if (t0 + s < te) out[(size_t)s * a.B * (2 * P::N) + n] = v;
    };
#pragma unroll
    for (int part = kParts - 1; part >= 0; --part) {
      const int s0 = part * H;
#pragma unroll
      for (int n = 0; n < S; ++n) start[n] = hin[n];
#pragma unroll
      for (int before = 0; before < part; ++before) {
        forwards(before * H, std::false_type{});
        asm volatile("" ::: "memory");  // what it read is read again rather than kept for the other parts
      }
      forwards(s0, std::true_type{});
      struct Ahead {
        float2 dt[G];
        float dy[G], b[G][S], c[G][S];
      } r[2];
      auto read = [&](int s1, Ahead& v) {
#pragma unroll
        for (int s = 0; s < G; ++s) {
          v.dt[s] = sdt[s1 + s][q.lane];
          v.dy[s] = sdy[s1 + s][q.lane];
          load_row<S>(&sb[s1 + s][q.n0], v.b[s]);
          load_row<S>(&sc[s1 + s][q.n0], v.c[s]);
        }
      };
      read(s0 + H - G, r[(H / G - 1) & 1]);
#pragma unroll
      for (int k = H - 1; k >= 0; --k) {
        const int s = s0 + k;
        if (k % G == G - 1) {
          if (k >= G) read(s0 + k / G * G - G, r[(k / G - 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);  // the reads stay ahead
        }
        const Ahead& v = r[(k / G) & 1];
        const float2 dt = v.dt[k % G];
        const float dy = v.dy[k % G];
        const float(&b)[S] = v.b[k % G];
        const float(&c)[S] = v.c[k % G];
        const bool cut = SLOW && (cuts >> s & 1);
        float gb = 0.f, ap = 0.f, y = 0.f, vb[S], vc[S];
#pragma unroll
        for (int n = 0; n < S; ++n) {
          const float g = __builtin_fmaf(c[n], dy, U[n]);
          y = __builtin_fmaf(c[n], hs[k][n], y);
          gb = __builtin_fmaf(g, b[n], gb);
          vb[n] = g * dt.y;
          vc[n] = dy * hs[k][n];
          U[n] = g * f[k][n];
          float p = U[n] * (k ? hs[k ? k - 1 : 0][n] : start[n]);
          if (cut) U[n] = p = 0.f;
          ap = __builtin_fmaf(an[n], p, ap);
          cda[n] = __builtin_fmaf(dt.x, p, cda[n]);
          if (SLOW && !q.ok) vb[n] = vc[n] = 0.f;
        }
        sp[0][q.w][s][q.lane] = gb;
        sp[1][q.w][s][q.lane] = ap;
        sp[2][q.w][s][q.lane] = y;
        // rows 0..3: b of state n, c of state n, b of state n + 1, c of state n + 1
#pragma unroll
        for (int n = 0; n < S; n += 2)
          sums[(s * (S / 2) + n / 2) % 16] = add16(add32(vb[n], vb[n + 1]), add32(vc[n], vc[n + 1]));
        if (s * (S / 2) % 16 == 0) finish_sums(s);
      }
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int n = 0; n < S; ++n) da[n].add(cda[n]);
  };

  const int first = te > tb ? tb + (te - tb - 1) / L * L : tb - L;
  BwdRows<F, P, false> rows(a, q, first);
  Rows<F, P> dxr(a.dx, q, first), ddr(a.ddelta, q, first), dzr(a.dz, q, first);
  if (te > tb) {
    rows.load(a, q, off, first, te, m);
    stage(first);
  }
  lds_barrier();
  for (int t0 = first; t0 >= tb; t0 -= L) {
    if (t0 > tb) rows.load(a, q, off, t0 - L, te, m);
    if (cuts || tail)
      run(std::true_type{}, t0);
    else
      run(std::false_type{}, t0);
    lds_barrier();
    float cskip = 0.f, cbias = 0.f;
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int s = q.w + W * i, t = t0 + s;
      if (L < W && s >= L) break;
      float gb = 0.f, ap = 0.f, y = skip * kx[i];
#pragma unroll
      for (int v = 0; v < W; ++v) {
        gb += sp[0][v][s][q.lane];
        ap += sp[1][v][s][q.lane];
        y += sp[2][v][s][q.lane];
      }
      const float sg = gate_sigmoid<F>(kz[i]), slope = __builtin_fmaf(kz[i] * sg, 1.f - sg, sg);
      const float dy = kdo[i] * (gated ? kz[i] * sg : 1.f);
      const float ddelta = __builtin_fmaf(kx[i], gb, ap) * ksig[i];
      const bool in = t < te;
      cskip = __builtin_fmaf(dy, kx[i], cskip);
      cbias += in && q.ok ? ddelta : 0.f;
      dxr.store(i, off, in, __builtin_fmaf(kdt[i], gb, skip * dy));
      ddr.store(i, off, in, ddelta);
      dzr.store(i, off, in && gated, kdo[i] * y * slope);
    }
    dskip.add(cskip);
    dbias.add(cbias);
    dxr.move(-1);
    ddr.move(-1);
    dzr.move(-1);
    if (t0 > tb) stage(t0 - L);
    lds_barrier();
  }
  if (seg == 0 && a.dh0) store_states(a.dh0, q, a, U);
  const size_t part = (size_t)q.b * a.nseg + seg;
  if (q.ok) {
    float v[S];
#pragma unroll
    for (int n = 0; n < S; ++n) v[n] = da[n].sum;
    store_kept(a.part_a, q, a, part, v);
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
                                                       float* dbias, int rows, int D, int N, int states) {
  __shared__ double sm[4][64];
  const int c = threadIdx.x & 63, strip = threadIdx.x >> 6;
  const long long na = (long long)states * D, all = na + 2 * D, i = (long long)blockIdx.x * 64 + c;
  double v = 0.0;
  if (i < all)
    for (int r = strip; r < rows; r += 4)
      v += i < na ? part_a[(long long)r * na + i] : part_d[(long long)r * 2 * D + (i - na)];
  sm[strip][c] = v;
  __syncthreads();
  if (strip || i >= all) return;
  const float s = (float)((sm[0][c] + sm[1][c]) + (sm[2][c] + sm[3][c]));
  if (i < na) {
    const int n = (int)(i / D);
    if (n < N) da[i % D * N + n] = s;
  } else {
    const long long j = i - na;
    float* const o = j < D ? dd : dbias;
    if (o) o[j % D] = s;
  }
}

// f(integral_constant fmt, ScanShape): two states a wave up to 16 (four a wave, in half the waves and two workgroups a
// CU, took 3152 us for 2547, T4096 B32 D1024 N16 bf16: its registers leave one wave a SIMD).  64 states: eight a wave,
// 2891 us at T1024 B32 D1024 in four parts, 3308 in two; four a wave, whose 16 waves have 128 registers each, 5253.
template <class Fn>
int with_bwd_shape(int fmt, int N, Fn f) {
  return with_fmt(fmt, [&](auto F) {
    switch (scan_states(N)) {
      case 4: return f(F, ScanShape<2, 2>{});
      case 8: return f(F, ScanShape<4, 2>{});
      case 16: return f(F, ScanShape<8, 2>{});
      case 32: return f(F, ScanShape<8, 4>{});
      default: return f(F, ScanShape<8, 8>{});
    }
  });
}

// The pieces of a workspace, in floats.
struct BwdLayout {
  size_t map_h, map_s, bc, a, d, all;
};
BwdLayout bwd_layout(int T, int B, int D, int N) {
  const ScanPlan p = plan_scan(T, B, D, N);
  const size_t states = scan_states(N), bd = (size_t)B * D;
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
  if (B > 0)
    HSL_CHECK(with_bwd_shape(fmt, N, [&](auto F, auto shape) {
      constexpr int kF = decltype(F)::value;
      using P = decltype(shape);
      if (p.nseg > 1 && D > 0)
        hipLaunchKernelGGL((scan_bwd_map_kernel<kF, P>), dim3(p.tiles * B, p.nseg - 1), dim3(P::W * 64), 0, s, g);
      if (D > 0)
        hipLaunchKernelGGL((scan_bwd_kernel<kF, P>), dim3(p.tiles * B, p.nseg), dim3(P::W * 64), 0, s, g);
      if (T > 0) {  // zeros where there is no channel
        const long long n = ((long long)T * B * 2 * P::N + 255) / 256;
        hipLaunchKernelGGL((scan_bc_kernel<kF>), dim3((unsigned)std::min<long long>(n, 1 << 20)), dim3(256), 0, s,
                           g.part_bc, OutStream{db, db_t, db_b}, OutStream{dc, dc_t, dc_b}, T, B, N, P::N, p.tiles);
      }
      HSL_HIP(hipGetLastError());
      return (int)HSL_OK;
    }));
  if (D == 0) return HSL_OK;
  const long long cols = ((long long)scan_states(N) + 2) * D;
  hipLaunchKernelGGL(scan_sum_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(256), 0, s, g.part_a, g.part_d, da, dd,
                     ddelta_bias, B * p.nseg, D, N, scan_states(N));
  HSL_HIP(hipGetLastError());
  return HSL_OK;
}

}  // extern "C"
