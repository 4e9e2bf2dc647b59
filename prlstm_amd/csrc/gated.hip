// Gated linear recurrence, forward, backward and one step.
//   f = sigmoid(z), w = sigmoid(-z) = 1 - f,   h_t = f_t h'_{t-1} + w_t v_t,
//   h'_{t-1} = 0 where reset_t is set (a new sequence begins at t), else h_{t-1};  h_{-1} = h0.
// Backward, with U_T = dh_n:  G_t = dout_t + U_{t+1},  U_t = reset_t ? 0 : f_t G_t,
//   dv_t = w_t G_t,  dz_t = G_t (h'_{t-1} - v_t) f_t w_t,  dh0 = U_0.
// zv holds z in its first H and v in its last H channels.  The state is fp32 throughout; out is
// h rounded once.  ck keeps h as it enters every 16th step, in fp32, from which the backward runs
// the steps again (the rounded out would cost dz its precision where h and v are close).
//
// Both directions are first-order recurrences, so runs of steps compose into affine maps
// x -> A x + V.  A workgroup owns kLanes * E neighbouring channels and walks the time in chunks:
// each of its groups of kLanes lanes takes 8 steps of the chunk, composes them, the maps are
// joined by one cross-lane move and through LDS, and the group runs its steps again from the
// state that enters them, all from registers; the next chunk's loads are issued first.  Every
// stream is read and written once.  With few channels the time is cut into segments that run as
// workgroups of their own after a pass that composes each segment's map.
#include <algorithm>
#include <initializer_list>

#include "lm.h"

namespace hsl {
namespace {

constexpr int kSteps = 8;    // of a group in a chunk
constexpr int kCkSteps = 2 * kSteps;  // of a wave's two groups: one checkpoint row
constexpr int kLanes = 32;   // of a group
constexpr int kMaxWaves = 8;

struct Gates {
  float f, w;
};
// e = exp(-|z|) is at most 1, so neither gate is a difference: the larger is 1 / (1 + e), the
// smaller e / (1 + e).  A 16-bit z has an error of 2^-9 (bf16) or 2^-12 of itself, against which
// that of rounding z log2 e to fp32 (|z| 2^-24 of e) does not count, so exp is one product and
// v_exp_f32 there; an fp32 z gets the corrected exp_f.
template <int F>
__device__ __forceinline__ Gates gates_of(float z) {
  float e;
  if constexpr (F == kElemF32)
    e = exp_f(-__builtin_fabsf(z));
  else
    e = __builtin_amdgcn_exp2f(-__builtin_fabsf(z) * 1.44269502162933349609375f);
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  return z >= 0.f ? Gates{big, small} : Gates{small, big};
}

// A of a map with a reset in it is -0 (all others are >= +0): nothing of the state before it
// passes, not even what is infinite or NaN, where 0 * x would.
constexpr unsigned kCutBits = 0x80000000u;
template <bool RESET>
__device__ __forceinline__ float apply(float A, float V, float x) {
  const float y = __builtin_fmaf(A, x, V);
  if constexpr (RESET) return __float_as_uint(A) == kCutBits ? V : y;
  return y;
}
// A of a composed map.  A product of gates is held at the smallest number once it underflows,
// unless a factor is 0, so that an infinite state stays infinite; a cut stays a cut.
template <bool RESET>
__device__ __forceinline__ float compose(float a, float b) {
  const float p = fmaxf(a * b, fminf(fminf(a, b), __uint_as_float(1u)));
  if constexpr (RESET)
    return __float_as_uint(a) == kCutBits || __float_as_uint(b) == kCutBits ? __uint_as_float(kCutBits) : p;
  return p;
}

// Strides are in elements.
struct Stream {
  const void* p;
  long long st, sb;
};
struct OutStream {
  void* p;
  long long st, sb;
};

// E neighbouring elements, at any element's alignment (global memory takes unaligned accesses).
template <int F, int E>
struct Pack {
  typename Elem<F>::T v[E];
};
// NT: non-temporal, for streams that no cache holds until their next use.
template <int N>
struct RawOf;
template <>
struct RawOf<2> {
  using T = unsigned short;
};
template <>
struct RawOf<4> {
  using T = unsigned;
};
template <>
struct RawOf<8> {
  using T = unsigned __attribute__((ext_vector_type(2)));
};
template <int F, int E, bool NT = false>
__device__ __forceinline__ Pack<F, E> load_pack(const typename Elem<F>::T* p) {
  Pack<F, E> r;
  if constexpr (NT) {
    typedef typename RawOf<sizeof(r)>::T Raw __attribute__((aligned(alignof(Pack<F, E>)), may_alias));
    const auto u = __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p));
    __builtin_memcpy(&r, &u, sizeof(r));
  } else {
    __builtin_memcpy(&r, p, sizeof(r));
  }
  return r;
}
template <int F, int E>
__device__ __forceinline__ void store_pack(typename Elem<F>::T* p, const Pack<F, E>& v) {
  typedef typename RawOf<sizeof(v)>::T Raw __attribute__((aligned(alignof(Pack<F, E>)), may_alias));
  typename RawOf<sizeof(v)>::T u;
  __builtin_memcpy(&u, &v, sizeof(v));
  __builtin_nontemporal_store(u, reinterpret_cast<Raw*>(p));
}
template <int E>
struct Floats {
  float v[E];
};
template <int E>
__device__ __forceinline__ Floats<E> load_floats(const float* p) {
  Floats<E> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <int E>
__device__ __forceinline__ void store_floats(float* p, const float (&v)[E]) {
  __builtin_memcpy(p, v, sizeof(v));
}

// A thread's place: E neighbouring channels j .. j+E-1 of batch row b.  Where H is odd the last
// thread of a row takes the last two channels, one of them beside its neighbour: both compute and
// store the same values.
template <int E>
struct Place {
  int lane, w, c, g, nw;  // lane in the wave, wave, lane in the group, group in the workgroup, waves
  int ch, b, j;           // ch = b H + j; clamped into range
  bool ok;
  __device__ __forceinline__ void channels(int i, int B, int H) {
    const int per = (H + E - 1) / E;
    ok = i < B * per;
    i = ok ? i : B * per - 1;
    b = i / per;
    j = min((i - b * per) * E, H - E);
    ch = b * H + j;
  }
  __device__ __forceinline__ Place(int B, int H) {
    lane = threadIdx.x & 63;
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    nw = blockDim.x >> 6;
    c = lane % kLanes;
    g = threadIdx.x / kLanes;
    channels(blockIdx.x * kLanes + c, B, H);
  }
};

// The reset flags of the 8 steps from t0 on, p at its first (flags of steps past T are not used).
template <bool TAIL>
__device__ __forceinline__ void load_resets(const unsigned char* p, long long st, int t0, int T,
                                            unsigned char (&r)[kSteps]) {
  if (!TAIL && st == 1) {
    __builtin_memcpy(r, p, kSteps);
    return;
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) r[s] = TAIL && t0 + s >= T ? 0 : p[s * st];
}

// Whether any lane of the wave has one (most groups of 8 steps have none).
__device__ __forceinline__ bool any_reset(const unsigned char (&r)[kSteps]) {
  unsigned any = 0;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) any |= r[s];
  return __any((int)any);
}

// A of the composed map of a group's steps, from the product and the smallest of the gates.
__device__ __forceinline__ float held(float prod, float least) {
  return fmaxf(prod, fminf(least, __uint_as_float(1u)));
}

// Joins the maps of a chunk's groups: from each thread's map (A, V) of its group, first (REV:
// last) group nearest to the incoming state x, returns the state that enters the thread's group
// and leaves in x the state behind the chunk.  sm is this chunk's [waves][kLanes] part of LDS.
template <int E, bool RESET, bool REV>
__device__ __forceinline__ void join(const Place<E>& q, float (&A)[E], float (&V)[E], float (&x)[E], float (&in)[E],
                                     Floats<2 * E> (*sm)[kLanes]) {
  // the wave's other group's map; the group further from the state continues the nearer one's
  float oA[E], oV[E];
  const bool far = REV ? q.lane < kLanes : q.lane >= kLanes;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    oA[e] = __shfl_xor(A[e], kLanes);
    oV[e] = __shfl_xor(V[e], kLanes);
  }
  if (far) {
    Floats<2 * E> m;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      m.v[2 * e + 1] = apply<RESET>(A[e], V[e], oV[e]);
      m.v[2 * e] = compose<RESET>(A[e], oA[e]);
    }
    sm[q.w][q.c] = m;
  }
  lds_barrier();
  float cur[E];
#pragma unroll
  for (int e = 0; e < E; ++e) cur[e] = x[e];
  for (int i = 0; i < q.nw; ++i) {
    const int u = REV ? q.nw - 1 - i : i;
    const Floats<2 * E> m = sm[u][q.c];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (u == q.w) in[e] = cur[e];
      cur[e] = apply<RESET>(m.v[2 * e], m.v[2 * e + 1], cur[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[e] = cur[e];
    if (far) in[e] = apply<RESET>(oA[e], oV[e], in[e]);
  }
}

// The state that enters a segment: the first (REV: last) state through the maps of the segments
// before it, maps[i][C] of segment i + 1 (REV) or i.
template <int E, bool RESET, bool REV>
__device__ __forceinline__ void enter_segment(const float2* __restrict__ maps, int C, int ch, int seg, int nseg,
                                              float (&x)[E]) {
  const int n = REV ? nseg - 1 - seg : seg;
  for (int i0 = 0; i0 < n; i0 += 8) {
    float2 m[8][E];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = min(i0 + i, n - 1), row = REV ? nseg - 2 - k : k;
#pragma unroll
      for (int e = 0; e < E; ++e) m[i][e] = maps[(size_t)row * C + ch + e];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < n) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = apply<RESET>(m[i][e].x, m[i][e].y, x[e]);
      }
  }
}

// Forward.  Bound by HBM: T4096 B16 H1024 bf16 74 us for 419 MB (5.7 TB/s, a large copy has 5.1; 79 to 83
// on average in training passes on inputs in turn), fp32 150 us for 822 MB.  Two channels a lane make
// 128-byte (bf16) and 256-byte (fp32) rows of a group.
template <int F, int E, bool RESET, bool NT>
__global__ __launch_bounds__(kMaxWaves * 64) void gated_fwd_kernel(Stream zv, const float* h0, Stream reset,
                                                                  OutStream out, float* h_n, float* __restrict__ ck,
                                                                  const float2* __restrict__ maps, int T, int B, int H,
                                                                  int seg_steps) {
  using T_ = typename Elem<F>::T;
  __shared__ Floats<2 * E> sm[2][kMaxWaves][kLanes];
  const Place<E> q(B, H);
  const int C = B * H, chunk = q.nw * 2 * kSteps;
  const int seg = blockIdx.y, tb = seg * seg_steps, te = min(T, tb + seg_steps);
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = h0 ? h0[q.ch + e] : 0.f;
  enter_segment<E, RESET, false>(maps, C, q.ch, seg, gridDim.y, x);
  // the group's first step of the chunk that is loaded (zp, rp) and of the one that is run (op)
  const T_* zp = static_cast<const T_*>(zv.p) + q.b * zv.sb + (tb + q.g * kSteps) * zv.st + q.j;
  const unsigned char* rp =
      static_cast<const unsigned char*>(reset.p) + q.b * reset.sb + (tb + q.g * kSteps) * reset.st;
  T_* op = static_cast<T_*>(out.p) + q.b * out.sb + (tb + q.g * kSteps) * out.st + q.j;
  float* cp = ck + (size_t)(tb / kCkSteps + q.w) * C + q.ch;

  Pack<F, E> rz[2][kSteps], rv[2][kSteps];
  unsigned char rr[2][kSteps];
  auto load = [&](int t1, Pack<F, E>(&z)[kSteps], Pack<F, E>(&v)[kSteps], unsigned char(&r)[kSteps]) {
    if (t1 + chunk <= te) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        z[s] = load_pack<F, E, NT>(zp + s * zv.st);
        v[s] = load_pack<F, E, NT>(zp + s * zv.st + H);
      }
      if constexpr (RESET) load_resets<false>(rp, reset.st, 0, T, r);
    } else {  // the last chunk: steps past T are not read
      const int t0 = t1 + q.g * kSteps;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        z[s] = v[s] = Pack<F, E>{};
        if (t0 + s < te) {
          z[s] = load_pack<F, E, NT>(zp + s * zv.st);
          v[s] = load_pack<F, E, NT>(zp + s * zv.st + H);
        }
      }
      if constexpr (RESET) load_resets<true>(rp, reset.st, t0, te, r);
    }
    zp += chunk * zv.st;
    if constexpr (RESET) rp += chunk * reset.st;
  };
  auto step = [&](auto tail, auto resets, int t1, int par, Pack<F, E>(&z)[kSteps], Pack<F, E>(&v)[kSteps],
                  unsigned char(&r)[kSteps]) {
    constexpr bool TAIL = decltype(tail)::value;  // the chunk with step T-1: later ones keep the state
    constexpr bool CUTS = decltype(resets)::value;  // a reset among the wave's steps
    const int t0 = t1 + q.g * kSteps;
    float f[kSteps][E], wv[kSteps][E], A[E], V[E], h[E], least[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      A[e] = least[e] = 1.f;
      V[e] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const bool in = !TAIL || t0 + s < te;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const Gates g = gates_of<F>(Elem<F>::up(z[s].v[e]));
        f[s][e] = in ? g.f : 1.f;
        wv[s][e] = in ? g.w * Elem<F>::up(v[s].v[e]) : 0.f;
        if (CUTS && in && r[s]) f[s][e] = __uint_as_float(kCutBits);
        V[e] = apply<CUTS>(f[s][e], wv[s][e], V[e]);
        if constexpr (CUTS) {
          A[e] = compose<CUTS>(f[s][e], A[e]);
        } else {
          A[e] *= f[s][e];
          least[e] = fminf(least[e], f[s][e]);
        }
      }
    }
    if constexpr (!CUTS) {
#pragma unroll
      for (int e = 0; e < E; ++e) A[e] = held(A[e], least[e]);
    }
    join<E, RESET, false>(q, A, V, x, h, sm[par]);
    T_* const o0 = op;
    float* const c0 = cp;
    op += chunk * out.st;
    cp += (size_t)(chunk / kCkSteps) * C;
    if (!q.ok || (TAIL && t0 >= te)) return;
    if (ck && q.lane < kLanes) store_floats(c0, h);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      Pack<F, E> o;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[e] = apply<CUTS>(f[s][e], wv[s][e], h[e]);
        o.v[e] = Elem<F>::down(h[e]);
      }
      if (!TAIL || t0 + s < te) store_pack<F, E>(o0 + s * out.st, o);
    }
    if (TAIL && te == T && T - t0 <= kSteps) store_floats(h_n + q.ch, h);
  };
  auto run = [&](int t, int i) {
    if (t + chunk < te) {
      load(t + chunk, rz[i ^ 1], rv[i ^ 1], rr[i ^ 1]);
      if (RESET && any_reset(rr[i]))
        step(std::false_type{}, std::integral_constant<bool, RESET>{}, t, i, rz[i], rv[i], rr[i]);
      else
        step(std::false_type{}, std::false_type{}, t, i, rz[i], rv[i], rr[i]);
    } else {
      step(std::true_type{}, std::integral_constant<bool, RESET>{}, t, i, rz[i], rv[i], rr[i]);
    }
  };
  if (tb < te) load(tb, rz[0], rv[0], rr[0]);
  for (int t = tb; t < te; t += 2 * chunk) {
    run(t, 0);
    if (t + chunk < te) run(t + chunk, 1);
  }
  if (T == 0 && q.g == 0 && q.ok) store_floats(h_n + q.ch, x);
}

// The map of segment blockIdx.y (never the last, so every step is below T), of whole 8-step parts
// for each group.
template <int F, int E, bool RESET>
__global__ __launch_bounds__(kMaxWaves * 64) void gated_fwd_map_kernel(Stream zv, Stream reset,
                                                                      float2* __restrict__ maps, int T, int B, int H,
                                                                      int seg_steps) {
  using T_ = typename Elem<F>::T;
  __shared__ Floats<2 * E> sm[kMaxWaves][kLanes];
  const Place<E> q(B, H);
  const int part = seg_steps / (q.nw * 2), t0 = blockIdx.y * seg_steps + q.g * part;
  const T_* zp = static_cast<const T_*>(zv.p) + q.b * zv.sb + t0 * zv.st + q.j;
  const unsigned char* rp = static_cast<const unsigned char*>(reset.p) + q.b * reset.sb + t0 * reset.st;
  float A[E], V[E], x[E], in[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    A[e] = 1.f;
    V[e] = x[e] = 0.f;
  }
  for (int k = 0; k < part; k += kSteps) {
    Pack<F, E> z[kSteps], v[kSteps];
    unsigned char r[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      z[s] = load_pack<F, E>(zp + s * zv.st);
      v[s] = load_pack<F, E>(zp + s * zv.st + H);
    }
    zp += kSteps * zv.st;
    if constexpr (RESET) {
      load_resets<false>(rp, reset.st, 0, T, r);
      rp += kSteps * reset.st;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        Gates g = gates_of<F>(Elem<F>::up(z[s].v[e]));
        if (RESET && r[s]) g.f = __uint_as_float(kCutBits);
        V[e] = apply<RESET>(g.f, g.w * Elem<F>::up(v[s].v[e]), V[e]);
        A[e] = compose<RESET>(g.f, A[e]);
      }
  }
  join<E, RESET, false>(q, A, V, x, in, sm);  // x: V of the whole segment
  if (threadIdx.x < kLanes && q.ok) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a = 1.f;
      for (int u = 0; u < q.nw; ++u) a = compose<RESET>(sm[u][q.c].v[2 * e], a);
      maps[(size_t)blockIdx.y * B * H + q.ch + e] = float2{a, x[e]};
    }
  }
}

// Backward: the group's steps forward from the checkpoint (by way of the wave's first group for its
// second), then the reverse map and, from the joined U, the gradients.  T4096 B16 H1024 bf16 136 us for
// 688 MB (5.1 TB/s; 141 to 145 on average in training passes on inputs in turn), fp32 228 us for 1359 MB
// (6.0).  A third or fourth chunk in flight changes nothing.
template <int F, int E, bool RESET, bool NT>
__global__ __launch_bounds__(kMaxWaves * 64) void gated_bwd_kernel(Stream zv, Stream reset,
                                                                  const float* __restrict__ ck, Stream dout,
                                                                  const float* __restrict__ dh_n, OutStream dzv,
                                                                  float* __restrict__ dh0,
                                                                  const float2* __restrict__ maps, int T, int B, int H,
                                                                  int seg_steps) {
  using T_ = typename Elem<F>::T;
  __shared__ Floats<2 * E> sm[2][kMaxWaves][kLanes];
  const Place<E> q(B, H);
  const int C = B * H, chunk = q.nw * 2 * kSteps;
  const int seg = blockIdx.y, tb = seg * seg_steps, te = min(T, tb + seg_steps);
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = dh_n ? dh_n[q.ch + e] : 0.f;
  enter_segment<E, RESET, true>(maps, C, q.ch, seg, gridDim.y, x);
  // pointers at the group's first step of the chunk that is loaded (gp: run), from the last one on
  const int n = (te - tb + chunk - 1) / chunk;
  const long long last = tb + (n - 1) * chunk + q.g * kSteps;
  const T_* zp = static_cast<const T_*>(zv.p) + q.b * zv.sb + last * zv.st + q.j;
  const T_* dp = static_cast<const T_*>(dout.p) + q.b * dout.sb + last * dout.st + q.j;
  const unsigned char* rp = static_cast<const unsigned char*>(reset.p) + q.b * reset.sb + last * reset.st;
  const float* cp = ck + (last / kCkSteps) * C + q.ch;
  T_* gp = static_cast<T_*>(dzv.p) + q.b * dzv.sb + last * dzv.st + q.j;

  struct Chunk {  // of the group, in registers
    Pack<F, E> z[kSteps], v[kSteps], d[kSteps];
    Floats<E> h;
    unsigned char r[kSteps];
  };
  auto load = [&](auto tail, int t1, Chunk& m) {
    constexpr bool TAIL = decltype(tail)::value;  // steps past T are not read
    const int t0 = t1 + q.g * kSteps;
    m.h = Floats<E>{};
    if (!TAIL || t0 < te) m.h = load_floats<E>(cp);  // of the wave's first group
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (TAIL) m.z[s] = m.v[s] = Pack<F, E>{};
      m.d[s] = Pack<F, E>{};
      if (!TAIL || t0 + s < te) {
        m.z[s] = load_pack<F, E, NT>(zp + s * zv.st);
        m.v[s] = load_pack<F, E, NT>(zp + s * zv.st + H);
        if (dout.p) m.d[s] = load_pack<F, E, NT>(dp + s * dout.st);
      }
    }
    if constexpr (RESET) load_resets<TAIL>(rp, reset.st, t0, te, m.r);
    zp -= chunk * zv.st;
    dp -= chunk * dout.st;
    if constexpr (RESET) rp -= chunk * reset.st;
    cp -= (size_t)(chunk / kCkSteps) * C;
  };
  auto step = [&](auto tail, auto resets, int t1, int par, Chunk& m) {
    constexpr bool TAIL = decltype(tail)::value;  // the chunk with step T-1: U passes later ones
    constexpr bool CUTS = decltype(resets)::value;  // a reset among the wave's steps
    const int t0 = t1 + q.g * kSteps;
    float f[kSteps][E], w[kSteps][E], hp[kSteps][E], A[E], V[E], U[E], h[E], least[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      A[e] = least[e] = 1.f;
      V[e] = 0.f;
      h[e] = m.h.v[e];
    }
    float wv[kSteps][E];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const Gates g = gates_of<F>(Elem<F>::up(m.z[s].v[e]));
        f[s][e] = g.f;
        w[s][e] = g.w;
        wv[s][e] = g.w * Elem<F>::up(m.v[s].v[e]);
        h[e] = CUTS && m.r[s] ? wv[s][e] : __builtin_fmaf(g.f, h[e], wv[s][e]);
      }
    }
    // the state behind the wave's first group enters its second
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float behind = __shfl_xor(h[e], kLanes);
      h[e] = q.lane < kLanes ? m.h.v[e] : behind;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        hp[s][e] = CUTS && m.r[s] ? 0.f : h[e];
        h[e] = CUTS && m.r[s] ? wv[s][e] : __builtin_fmaf(f[s][e], h[e], wv[s][e]);
      }
    }
#pragma unroll
    for (int s = kSteps - 1; s >= 0; --s) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool cut = CUTS && m.r[s];
        const float d = Elem<F>::up(m.d[s].v[e]);
        if (!TAIL || t0 + s < te) {
          V[e] = cut ? 0.f : f[s][e] * (d + V[e]);
          if constexpr (CUTS) {
            A[e] = compose<CUTS>(cut ? __uint_as_float(kCutBits) : f[s][e], A[e]);
          } else {
            A[e] *= f[s][e];
            least[e] = fminf(least[e], f[s][e]);
          }
        }
      }
    }
    if constexpr (!CUTS) {
#pragma unroll
      for (int e = 0; e < E; ++e) A[e] = held(A[e], least[e]);
    }
    join<E, RESET, true>(q, A, V, x, U, sm[par]);
    T_* const p0 = gp;
    gp -= chunk * dzv.st;
    if (!q.ok || (TAIL && t0 >= te)) return;
#pragma unroll
    for (int s = kSteps - 1; s >= 0; --s) {
      if (!TAIL || t0 + s < te) {
        Pack<F, E> oz, ov;
        float dz[E], dv[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float G = Elem<F>::up(m.d[s].v[e]) + U[e];
          dv[e] = w[s][e] * G;
          dz[e] = dv[e] * ((hp[s][e] - Elem<F>::up(m.v[s].v[e])) * f[s][e]);
          U[e] = CUTS && m.r[s] ? 0.f : f[s][e] * G;
        }
        down_all<F, E>(dz, oz.v);
        down_all<F, E>(dv, ov.v);
        store_pack<F, E>(p0 + s * dzv.st, oz);
        store_pack<F, E>(p0 + s * dzv.st + H, ov);
      }
    }
    if (t0 == 0 && dh0) store_floats(dh0 + q.ch, U);
  };
  auto whole = [&](int t1, int par, Chunk& m) {
    if (RESET && any_reset(m.r))
      step(std::false_type{}, std::integral_constant<bool, RESET>{}, t1, par, m);
    else
      step(std::false_type{}, std::false_type{}, t1, par, m);
  };
  Chunk m0, m1;
  if (n > 0) {
    load(std::true_type{}, tb + (n - 1) * chunk, m0);
    if (n > 1) load(std::false_type{}, tb + (n - 2) * chunk, m1);
    step(std::true_type{}, std::integral_constant<bool, RESET>{}, tb + (n - 1) * chunk, 0, m0);
  }
  for (int k = n - 2; k >= 0; k -= 2) {
    if (k >= 1) load(std::false_type{}, tb + (k - 1) * chunk, m0);
    whole(tb + k * chunk, 1, m1);
    if (k < 1) break;
    if (k >= 2) load(std::false_type{}, tb + (k - 2) * chunk, m1);
    whole(tb + (k - 1) * chunk, 0, m0);
  }
  if (T == 0 && dh0 && q.g == 0 && q.ok) store_floats(dh0 + q.ch, x);
}

// The reverse map of segment blockIdx.y + 1, which ends at min(T, ..).
template <int F, int E, bool RESET>
__global__ __launch_bounds__(kMaxWaves * 64) void gated_bwd_map_kernel(Stream zv, Stream reset, Stream dout,
                                                                      float2* __restrict__ maps, int T, int B, int H,
                                                                      int seg_steps) {
  using T_ = typename Elem<F>::T;
  __shared__ Floats<2 * E> sm[kMaxWaves][kLanes];
  const Place<E> q(B, H);
  const int part = seg_steps / (q.nw * 2), t0 = ((int)blockIdx.y + 1) * seg_steps + q.g * part;
  const T_* const zp = static_cast<const T_*>(zv.p) + q.b * zv.sb + t0 * zv.st + q.j;
  const T_* const dp = static_cast<const T_*>(dout.p) + q.b * dout.sb + t0 * dout.st + q.j;
  const unsigned char* const rp = static_cast<const unsigned char*>(reset.p) + q.b * reset.sb + t0 * reset.st;
  float A[E], V[E], x[E], in[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    A[e] = 1.f;
    V[e] = x[e] = 0.f;
  }
  for (int k = part - kSteps; k >= 0; k -= kSteps) {
    if (t0 + k >= T) continue;
    Pack<F, E> z[kSteps], d[kSteps];
    unsigned char r[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      z[s] = d[s] = Pack<F, E>{};
      if (t0 + k + s < T) {
        z[s] = load_pack<F, E>(zp + (k + s) * zv.st);
        if (dout.p) d[s] = load_pack<F, E>(dp + (k + s) * dout.st);
      }
    }
    if constexpr (RESET) load_resets<true>(rp + k * reset.st, reset.st, t0 + k, T, r);
#pragma unroll
    for (int s = kSteps - 1; s >= 0; --s)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (t0 + k + s < T) {
          const float f = gates_of<F>(Elem<F>::up(z[s].v[e])).f;
          const bool cut = RESET && r[s];
          V[e] = cut ? 0.f : f * (Elem<F>::up(d[s].v[e]) + V[e]);
          A[e] = cut ? __uint_as_float(kCutBits) : compose<RESET>(f, A[e]);
        }
  }
  join<E, RESET, true>(q, A, V, x, in, sm);
  if (threadIdx.x < kLanes && q.ok) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a = 1.f;
      for (int u = q.nw - 1; u >= 0; --u) a = compose<RESET>(sm[u][q.c].v[2 * e], a);
      maps[(size_t)blockIdx.y * B * H + q.ch + e] = float2{a, x[e]};
    }
  }
}

// A single step, bound by its launch (2.5 us for B32 H1024): one thread per E channels (H is a multiple
// of E).  h_n may be h0.
template <int F, int E, bool RESET>
__global__ __launch_bounds__(256) void gated_step_kernel(Stream zv, const float* h0, Stream reset, OutStream out,
                                                         float* h_n, float* ck, int B, int H) {
  using T_ = typename Elem<F>::T;
  const int ch = (blockIdx.x * 256 + threadIdx.x) * E;
  if (ch >= B * H) return;
  const int b = ch / H, j = ch - b * H;
  const T_* p = static_cast<const T_*>(zv.p) + b * zv.sb + j;
  const Pack<F, E> z = load_pack<F, E>(p), v = load_pack<F, E>(p + H);
  Floats<E> h{};
  if (h0) h = load_floats<E>(h0 + ch);
  if (ck) store_floats(ck + ch, h.v);
  const bool cut = RESET && static_cast<const unsigned char*>(reset.p)[b * reset.sb];
  Pack<F, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const Gates g = gates_of<F>(Elem<F>::up(z.v[e]));
    const float wv = g.w * Elem<F>::up(v.v[e]);
    h.v[e] = cut ? wv : __builtin_fmaf(g.f, h.v[e], wv);
    o.v[e] = Elem<F>::down(h.v[e]);
  }
  store_pack<F, E>(static_cast<T_*>(out.p) + b * out.sb + j, o);
  store_floats(h_n + ch, h.v);
}

// The shape of a call's launches: waves of a workgroup, workgroups over the channels, segments.
struct GatedPlan {
  int waves, tiles, nseg, seg_steps;
};
// Waves: 8 (chunks of 128 steps) where a CU gets one or two workgroups, 4 where it gets more or the
// time is cut, 1 and 2 for short sequences.  us forward, backward, 8 waves / 4 waves, H1024:
//   bf16 T4096 B16 (256 workgroups): 73, 152 / 87, 166;  16 waves: 119, 275 (registers)
//   bf16 T4096 B20 (320): 132, 244 / 137, 209;  B28 (448): 142, 263 / 146, 248;  B32 (512): 158, 281 / 167, 272
//   fp32 T4096 B20 (320): 260, 389 / 238, 387;  B28 (448): 284, 444 / 268, 461;  B32 (512): 306, 482 / 291, 499
//   bf16 T256  B20 (320): 12, 17 / 11, 14;  B64 (1024): 25, 39 / 22, 31;   T2048 B32 (512): 79, 150 / 81, 140
// so that between 257 and 511 workgroups 4 waves would gain up to a fifth of a bf16 backward.
// Segments: of at least two chunks, for about 512 workgroups, where the channels alone give fewer
// than 192.  us of T16383 B2 H256 fp32, 8 tiles: 36, 40 for 512; 47, 45 for 256; 38, 46 for 1024.  With
// segments / without, T4096 H1024:
//   bf16 B8 H512 (64 workgroups): 32, 46 / 56, 79;  B8 (128): 57, 83 / 56, 107;  B10 (160): 73, 114 / 57, 117;
//        B12 (192): 96, 162 / 68, 121
//   fp32 B8 H512: 65, 75 / 75, 148;  B8: 126, 149 / 117, 167;  B10: 170, 206 / 124, 181;  B12: 240, 263 / 130, 192
// so that the two meet at about 128 workgroups, and those from there to 191 would gain a little without.
GatedPlan plan_gated(int T, int B, int H, int E) {
  GatedPlan p;
  p.tiles = (int)(((long)B * ((H + E - 1) / E) + kLanes - 1) / kLanes);
  const int most = p.tiles >= 512 ? kMaxWaves / 2 : kMaxWaves;
  p.waves = 1;
  while (p.waves < most && p.waves * 2 * kSteps < T) p.waves *= 2;
  int chunk = p.waves * 2 * kSteps, nchunks = (T + chunk - 1) / chunk;
  p.nseg = 1;
  p.seg_steps = std::max(1, nchunks) * chunk;
  if (p.tiles < 192 && nchunks >= 4) {
    p.waves = std::min(p.waves, kMaxWaves / 2);
    chunk = p.waves * 2 * kSteps;
    nchunks = (T + chunk - 1) / chunk;
    const int want = std::min(nchunks / 2, (512 + p.tiles - 1) / p.tiles);
    const int per = (nchunks + want - 1) / want;
    p.seg_steps = per * chunk;
    p.nseg = (nchunks + per - 1) / per;
  }
  return p;
}

int check_gated(const char* who, int T, int B, int H, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (T < 0 || B < 0 || H < 0) return fail(HSL_ERR_ARG, "%s: negative size (T=%d B=%d H=%d)", who, T, B, H);
  // steps and channels are counted in 32 bits, and 2^27 channels are 2^30 threads
  if (T >= (1 << 30) || (long long)B * H >= (1ll << 27))
    return fail(HSL_ERR_UNSUPPORTED,
                "%s: T=%d B=%d H=%d is beyond the kernels' 32-bit index range (needs T < 2^30 and B*H < 2^27)", who, T,
                B, H);
  return HSL_OK;
}

// Channels of a thread.  (The single step's stay within a row, for its state may be updated in place.)
int channels_each(int T, int H) { return T == 1 ? 2 - H % 2 : std::min(H, 2); }

// Whether a call's streams (`bytes` in all) are read without keeping them in the caches: where they
// exceed those and every workgroup's rows are whole 128-byte lines.
bool streams_past_cache(size_t bytes, int H, int es, std::initializer_list<Stream> streams) {
  if (bytes <= kCacheBytes || (size_t)H * es % 128) return false;
  for (const Stream& s : streams)
    if (reinterpret_cast<uintptr_t>(s.p) % 128 || s.st * es % 128 || s.sb * es % 128) return false;
  return true;
}

// f(fmt, channels each, reset, non-temporal) as integral constants.
template <class Fn>
int with_instance(int fmt, int e, bool reset, bool nt, Fn f) {
  return with_fmt(fmt, [&](auto F) {
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Yes = std::true_type;
    using No = std::false_type;
    if (e == 1) return reset ? f(F, One{}, Yes{}, No{}) : f(F, One{}, No{}, No{});
    if (nt) return reset ? f(F, Two{}, Yes{}, Yes{}) : f(F, Two{}, No{}, Yes{});
    return reset ? f(F, Two{}, Yes{}, No{}) : f(F, Two{}, No{}, No{});
  });
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

int hsl_gated_ck_rows(int T) { return T <= 0 ? 0 : (T + kCkSteps - 1) / kCkSteps; }

size_t hsl_gated_ws_bytes(int T, int B, int H) {
  if (check_gated("hsl_gated_ws_bytes", T, B, H, kElemF32) != HSL_OK || B == 0 || H == 0) return 0;
  return (size_t)(plan_gated(T, B, H, std::min(H, 2)).nseg - 1) * B * H * sizeof(float2);
}

int hsl_gated_fwd(const void* zv, long long zv_t, long long zv_b, const float* h0, const void* reset, long long rs_t,
                  long long rs_b, void* out, long long out_t, long long out_b, float* h_n, float* ck, void* ws,
                  size_t ws_bytes, int T, int B, int H, int fmt, void* stream) {
  HSL_CHECK(check_gated("hsl_gated_fwd", T, B, H, fmt));
  if (B == 0 || H == 0) return HSL_OK;
  if (!h_n || (T > 0 && (!zv || !out))) return fail(HSL_ERR_ARG, "hsl_gated_fwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int e = channels_each(T, H);
  const GatedPlan p = plan_gated(T, B, H, e);
  if (p.nseg > 1 && (!ws || ws_bytes < hsl_gated_ws_bytes(T, B, H)))
    return fail(HSL_ERR_ARG, "hsl_gated_fwd: workspace %zu bytes, need %zu", ws_bytes, hsl_gated_ws_bytes(T, B, H));
  float2* const maps = static_cast<float2*>(ws);
  const Stream z{zv, zv_t, zv_b}, r{reset, rs_t, rs_b};
  const OutStream o{out, out_t, out_b};
  const int es = fmt == kElemF32 ? 4 : 2;
  const bool nt = p.nseg == 1 && streams_past_cache((size_t)3 * T * B * H * es, H, es, {z});
  return with_instance(fmt, e, reset != nullptr, nt, [&](auto F, auto E, auto R, auto N) {
    constexpr int kF = decltype(F)::value, kE = decltype(E)::value;
    constexpr bool kR = decltype(R)::value, kN = decltype(N)::value;
    if (T == 1) {
      const int n = (B * H + kE * 256 - 1) / (kE * 256);
      hipLaunchKernelGGL((gated_step_kernel<kF, kE, kR>), dim3(n), dim3(256), 0, s, z, h0, r, o, h_n, ck, B, H);
    } else {
      if (p.nseg > 1)
        hipLaunchKernelGGL((gated_fwd_map_kernel<kF, kE, kR>), dim3(p.tiles, p.nseg - 1), dim3(p.waves * 64), 0, s, z,
                           r, maps, T, B, H, p.seg_steps);
      hipLaunchKernelGGL((gated_fwd_kernel<kF, kE, kR, kN>), dim3(p.tiles, p.nseg), dim3(p.waves * 64), 0, s, z, h0, r,
                         o, h_n, ck, maps, T, B, H, p.seg_steps);
    }
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

int hsl_gated_bwd(const void* zv, long long zv_t, long long zv_b, const void* reset, long long rs_t, long long rs_b,
                  const float* ck, const void* dout, long long do_t, long long do_b, const float* dh_n, void* dzv,
                  long long dz_t, long long dz_b, float* dh0, void* ws, size_t ws_bytes, int T, int B, int H, int fmt,
                  void* stream) {
  HSL_CHECK(check_gated("hsl_gated_bwd", T, B, H, fmt));
  if (B == 0 || H == 0) return HSL_OK;
  if (T > 0 && (!zv || !ck || !dzv)) return fail(HSL_ERR_ARG, "hsl_gated_bwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int e = std::min(H, 2);
  const GatedPlan p = plan_gated(T, B, H, e);
  if (p.nseg > 1 && (!ws || ws_bytes < hsl_gated_ws_bytes(T, B, H)))
    return fail(HSL_ERR_ARG, "hsl_gated_bwd: workspace %zu bytes, need %zu", ws_bytes, hsl_gated_ws_bytes(T, B, H));
  float2* const maps = static_cast<float2*>(ws);
  const Stream z{zv, zv_t, zv_b}, r{reset, rs_t, rs_b}, d{dout, do_t, do_b};
  const OutStream g{dzv, dz_t, dz_b};
  const int es = fmt == kElemF32 ? 4 : 2;
  const bool nt = p.nseg == 1 && streams_past_cache((size_t)5 * T * B * H * es, H, es, {z, d});
  return with_instance(fmt, e, reset != nullptr, nt, [&](auto F, auto E, auto R, auto N) {
    constexpr int kF = decltype(F)::value, kE = decltype(E)::value;
    constexpr bool kR = decltype(R)::value, kN = decltype(N)::value;
    if (p.nseg > 1)
      hipLaunchKernelGGL((gated_bwd_map_kernel<kF, kE, kR>), dim3(p.tiles, p.nseg - 1), dim3(p.waves * 64), 0, s, z, r,
                         d, maps, T, B, H, p.seg_steps);
    hipLaunchKernelGGL((gated_bwd_kernel<kF, kE, kR, kN>), dim3(p.tiles, p.nseg), dim3(p.waves * 64), 0, s, z, r, ck, d,
                       dh_n, g, dh0, maps, T, B, H, p.seg_steps);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
