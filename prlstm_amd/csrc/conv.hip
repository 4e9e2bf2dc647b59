// Causal depthwise convolution of K <= 4 taps over time, forward, backward and one step.
//   u_t = bias + sum_j w[:, j] x_{t-K+1+j},   y_t = u_t sigmoid(u_t) (or u_t),
// where an input before the first step comes from the state, and one before the last reset is 0.
// Backward: du_t = dy_t s (1 + u_t (1 - s)) with s = sigmoid(u_t),
//   dx_t = sum_j w[:, j] du_{t+K-1-j} over the steps of t's own sequence,
//   dw[:, j] = sum_{t, b} du_t x_{t-K+1+j},   dbias = sum_{t, b} du_t.
//
// Each direction reads every stream once: a thread owns E neighbouring channels of one batch row and
// walks a segment of the time forwards with the last K-1 inputs in registers; the backward keeps the
// K-1 gradients that later steps still add to, and runs K-1 steps past its segment to finish them.
// u is computed again in the backward rather than kept.  The weights' sums are fp32 over a segment
// (256 steps at most) and the workgroup's rows, fp64 beyond, in an order that the sizes alone set.
#include <algorithm>

#include "lm.h"

namespace hsl {
namespace {

constexpr int kBlock = 8;      // steps whose loads are issued together
constexpr int kMaxTaps = 4;
constexpr int kMaxSeg = 256;   // steps that an fp32 sum runs over
constexpr int kWaves = 4;        // of a workgroup

// A call's split: a row of the work is one segment of one batch row, row = segment * B + b; a wave
// holds 64 >> log2g rows of 1 << log2g vectors each, and `tiles` waves cover a row's vectors.
struct ConvPlan {
  int per, log2g, tiles, seg, nseg;
  long long rows;
  int row_blocks() const {
    const int each = kWaves * (64 >> log2g);
    return (int)((rows + each - 1) / each);
  }
};

struct ConvArgs {
  Stream x, dy, reset;
  OutStream y, dx;
  const float *w, *bias;
  const void *state, *dstate_n;
  void *state_n, *dstate;
  float* part;  // [row blocks][K + 1][D]
  int T, B, D, silu;
  ConvPlan p;
};

// A thread's place.  Where E does not divide D the last vector of a row ends with the row, beside its
// neighbour: both lanes compute and store the same values.
template <int E>
struct ConvPlace {
  int lane, wave, j, b, t0, te;
  bool ok;
  __device__ __forceinline__ ConvPlace(const ConvArgs& a) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = blockIdx.x % a.p.tiles;
    const long long block = blockIdx.x / a.p.tiles;
    const long long row = (block * (blockDim.x >> 6) + wave) * (64 >> a.p.log2g) + (lane >> a.p.log2g);
    const int vec = (tile << a.p.log2g) + (lane & ((1 << a.p.log2g) - 1));
    ok = row < a.p.rows && vec < a.p.per;
    const long long r = row < a.p.rows ? row : a.p.rows - 1;
    j = min(vec * E, a.D - E);
    b = (int)(r % a.B);
    t0 = (int)(r / a.B) * a.p.seg;
    te = min(a.T, t0 + a.p.seg);
  }
};

// The last K-1 inputs before a step, the oldest first.
template <int F, int E, int K>
struct Window {
  float v[K][E];  // v[K-1] is the step's own input
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = 0.f;
  }
  // The next step's input; with `cut` a new sequence begins with it.
  template <bool RESET>
  __device__ __forceinline__ void push(const Pack<F, E>& x, bool cut) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = RESET && cut ? 0.f : v[k + 1][e];
#pragma unroll
    for (int e = 0; e < E; ++e) v[K - 1][e] = Elem<F>::up(x.v[e]);
  }
};

template <int F, int E, int K, bool RESET>
struct Walk {
  using T_ = typename Elem<F>::T;
  const T_* xp;
  const unsigned char* rp;
  const T_* sp;  // the state's rows of this batch row, or null
  long long xs, rs;
  int D;
  __device__ __forceinline__ Walk(const ConvArgs& a, const ConvPlace<E>& q)
      : xp(static_cast<const T_*>(a.x.p) + q.b * a.x.sb + q.j),
        rp(static_cast<const unsigned char*>(a.reset.p) + q.b * a.reset.sb),
        sp(a.state ? static_cast<const T_*>(a.state) + (long long)q.b * (K - 1) * a.D + q.j : nullptr),
        xs(a.x.st),
        rs(a.reset.st),
        D(a.D) {}
  __device__ __forceinline__ bool cut(int t) const { return RESET && rp[t * rs]; }
  // The window before step t0 and how many steps (K at most) its sequence has had by then.
  __device__ __forceinline__ int enter(int t0, Window<F, E, K>& w) const {
    w.clear();
    int since = K;
#pragma unroll
    for (int i = 1 - K; i < 0; ++i) {
      Pack<F, E> v{};
      bool c = false;
      if (t0 > 0) {  // a segment has at least kBlock >= K - 1 steps
        v = load_pack<F, E>(xp + (t0 + i) * xs);
        c = cut(t0 + i);
      } else if (sp) {
        v = load_pack<F, E>(sp + (long long)(K - 1 + i) * D);
      }
      w.template push<RESET>(v, c);
      since = c ? 0 : min(since + 1, K);
    }
    return since;
  }
};

template <int E, int K>
__device__ __forceinline__ void load_taps(const ConvArgs& a, int j, float (&w)[K][E], float (&bias)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    bias[e] = a.bias ? a.bias[j + e] : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][e] = a.w[(long long)(j + e) * K + k];
  }
}

// Forward.  Bound by HBM: 63 us at T4096 B16 D1024 K4, bf16 (268 MB, 4.3 TB/s), 50 on an input of which the caches
// hold a part.  Whole blocks of steps run without a test per step: with the tests, and exp in full precision, the
// latter was 66 us.
template <int F, int E, int K, bool RESET>
__global__ __launch_bounds__(kWaves * 64) void conv_fwd_kernel(ConvArgs a) {
  using T_ = typename Elem<F>::T;
  const ConvPlace<E> q(a);
  if (!q.ok) return;
  const Walk<F, E, K, RESET> walk(a, q);
  float w[K][E], bias[E];
  load_taps<E, K>(a, q.j, w, bias);
  Window<F, E, K> win;
  walk.enter(q.t0, win);
  T_* const yp = static_cast<T_*>(a.y.p) + q.b * a.y.sb + q.j;
  auto block = [&](int t, auto whole) {  // steps t .. t + kBlock - 1; the segment may end within if not `whole`
    constexpr bool kWhole = decltype(whole)::value;
    Pack<F, E> x[kBlock];
    bool cut[kBlock];
#pragma unroll
    for (int s = 0; s < kBlock; ++s) {
      if (!kWhole) {
        x[s] = Pack<F, E>{};
        cut[s] = false;
        if (t + s >= q.te) continue;
      }
      x[s] = load_pack<F, E>(walk.xp + (t + s) * walk.xs);
      cut[s] = walk.cut(t + s);
    }
#pragma unroll
    for (int s = 0; s < kBlock; ++s) {
      if (!kWhole && t + s >= q.te) break;
      win.template push<RESET>(x[s], cut[s]);
      float u[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        u[e] = bias[e];
#pragma unroll
        for (int k = 0; k < K; ++k) u[e] = __builtin_fmaf(w[k][e], win.v[k][e], u[e]);
        if (a.silu) u[e] *= gate_sigmoid<F>(u[e]);
      }
      Pack<F, E> y;
      down_all<F, E>(u, y.v);
      store_pack<F, E>(yp + (t + s) * a.y.st, y);
    }
  };
  int t = q.t0;
  for (; t + kBlock <= q.te; t += kBlock) block(t, std::true_type{});
  if (t < q.te) block(t, std::false_type{});
  if (K > 1 && q.te == a.T) {
    T_* const np = static_cast<T_*>(a.state_n) + (long long)q.b * (K - 1) * a.D + q.j;
#pragma unroll
    for (int k = 1; k < K; ++k) {
      Pack<F, E> v;
      down_all<F, E>(win.v[k], v.v);
      __builtin_memcpy(np + (long long)(k - 1) * a.D, &v, sizeof(v));
    }
  }
}

// Backward.  E = 4: the window, the taps and both kinds of sums take 150 registers, so 3 waves share a SIMD
// (held to 128 registers for a fourth, they spill: 127 us for the call).  93 us at T4096 B16 D1024 K4, bf16
// (403 MB, 4.3 TB/s); with a test per step, and of every weight's sum for the steps behind the segment, it
// was 117 us, the vector units as busy as the memory.
template <int F, int E, int K, bool RESET>
__global__ __launch_bounds__(kWaves * 64) void conv_bwd_kernel(ConvArgs a) {
  using T_ = typename Elem<F>::T;
  __shared__ float sm[kWaves][K + 1][64 * E];
  const ConvPlace<E> q(a);
  const Walk<F, E, K, RESET> walk(a, q);
  float w[K][E], bias[E], dw[K + 1][E];  // dw[K]: the bias's
  load_taps<E, K>(a, q.j, w, bias);
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[k][e] = 0.f;
  if (q.ok) {
    Window<F, E, K> win;
    int since = walk.enter(q.t0, win);
    float acc[K][E];  // gradients of the inputs t-K+1 .. t that the steps so far give
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[k][e] = 0.f;
    const T_* const dyp = static_cast<const T_*>(a.dy.p) + q.b * a.dy.sb + q.j;
    T_* const dxp = static_cast<T_*>(a.dx.p) + q.b * a.dx.sb + q.j;
    T_* const dsp = a.dstate ? static_cast<T_*>(a.dstate) + (long long)q.b * (K - 1) * a.D + q.j : nullptr;
    // stores the gradient of input t, if it is this segment's
    auto emit = [&](int t, const float(&g)[E]) {
      T_* p = nullptr;
      if (t >= q.t0 && t < q.te)
        p = dxp + t * a.dx.st;
      else if (t < 0 && dsp)
        p = dsp + (long long)(K - 1 + t) * a.D;
      if (!p) return;
      Pack<F, E> v;
      down_all<F, E>(g, v.v);
      store_pack<F, E>(p, v);
    };
    auto shift = [&]() {
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[k][e] = acc[k + 1][e];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[K - 1][e] = 0.f;
    };
    const int stop = min(a.T, q.te + K - 1);
    // Steps t .. t + kBlock - 1, all of them the segment's if `whole`; else the walk may end within, and
    // the steps behind the segment only finish its inputs' gradients.
    auto block = [&](int t, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      Pack<F, E> x[kBlock], dy[kBlock];
      bool cut[kBlock];
#pragma unroll
      for (int s = 0; s < kBlock; ++s) {
        x[s] = dy[s] = Pack<F, E>{};
        cut[s] = false;
        if (!kWhole && t + s >= stop) continue;
        x[s] = load_pack<F, E>(walk.xp + (t + s) * walk.xs);
        if (a.dy.p) dy[s] = load_pack<F, E>(dyp + (t + s) * a.dy.st);
        cut[s] = walk.cut(t + s);
      }
#pragma unroll
      for (int s = 0; s < kBlock; ++s) {
        if (!kWhole && t + s >= stop) break;
        win.template push<RESET>(x[s], cut[s]);
        if (RESET) since = cut[s] ? 0 : min(since + 1, K);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float du = Elem<F>::up(dy[s].v[e]);
          if (a.silu) {
            float u = bias[e];
#pragma unroll
            for (int k = 0; k < K; ++k) u = __builtin_fmaf(w[k][e], win.v[k][e], u);
            const float sg = gate_sigmoid<F>(u);
            du *= __builtin_fmaf(u * sg, 1.f - sg, sg);
          }
#pragma unroll
          for (int k = 0; k < K; ++k) {
            // input t-(K-1-k) of the same sequence
            const float g = __builtin_fmaf(w[k][e], du, acc[k][e]);
            acc[k][e] = !RESET || since >= K - 1 - k ? g : acc[k][e];
            if (kWhole || t + s < q.te) dw[k][e] = __builtin_fmaf(du, win.v[k][e], dw[k][e]);
          }
          if (kWhole || t + s < q.te) dw[K][e] += du;
        }
        emit(t + s - (K - 1), acc[0]);
        shift();
      }
    };
    int t = q.t0;
    for (; t + kBlock <= q.te; t += kBlock) block(t, std::true_type{});
    for (; t < stop; t += kBlock) block(t, std::false_type{});
    // the inputs that no step is left for, with the gradient of the state that the call returned
    if (stop == a.T) {
#pragma unroll
      for (int k = 0; k < K - 1; ++k) {
        if (a.dstate_n && (!RESET || since >= K - 2 - k)) {
          const T_* np = static_cast<const T_*>(a.dstate_n) + ((long long)q.b * (K - 1) + k) * a.D + q.j;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[k][e] += Elem<F>::up(np[e]);
        }
        emit(a.T - (K - 1) + k, acc[k]);
      }
    }
  }
  // the sums of the wave's rows, then of the workgroup's
  const int g = 1 << a.p.log2g;
#pragma unroll
  for (int k = 0; k <= K; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float v = dw[k][e];
      for (int m = g; m < 64; m *= 2) v += __shfl_xor(v, m);
      sm[q.wave][k][q.lane * E + e] = v;
    }
  __syncthreads();
  const int tile = blockIdx.x % a.p.tiles;
  float* const out = a.part + (long long)(blockIdx.x / a.p.tiles) * (K + 1) * a.D;
  for (int i = threadIdx.x; i < (K + 1) * g * E; i += kWaves * 64) {
    const int k = i / (g * E), l = i % (g * E), vec = (tile << a.p.log2g) + l / E;
    if (vec >= a.p.per) continue;
    float v = 0.f;
#pragma unroll
    for (int n = 0; n < kWaves; ++n) v += sm[n][k][l];
    out[(long long)k * a.D + min(vec * E, a.D - E) + l % E] = v;
  }
}

// dw [D][K] and dbias [D] from the workgroups' sums part[n][K + 1][D], in fp64.
constexpr int kSumStrips = 16;
__global__ __launch_bounds__(kSumStrips * 64) void conv_sum_kernel(const float* __restrict__ part, float* dw,
                                                                   float* dbias, int n, int K, int D) {
  __shared__ double sm[kSumStrips][64];
  const int c = threadIdx.x & 63, strip = threadIdx.x >> 6;
  const long long i = (long long)blockIdx.x * 64 + c, all = (long long)(K + 1) * D;
  double v = 0.0;
  if (i < all) {
#pragma unroll 8
    for (int r = strip; r < n; r += kSumStrips) v += part[r * all + i];
  }
  sm[strip][c] = v;
  __syncthreads();
  if (strip || i >= all) return;
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kSumStrips; ++k) sum += sm[k][c];
  const float s = (float)sum;
  const int k = (int)(i / D);
  const long long d = i % D;
  if (k < K)
    dw[d * K + k] = s;
  else if (dbias)
    dbias[d] = s;
}

// A single step, bound by its launch: one thread per E channels (E divides D).  state_n may be state.
template <int F, int E, int K, bool RESET>
__global__ __launch_bounds__(256) void conv_step_kernel(Stream x, Stream reset, OutStream y, const float* w,
                                                        const float* bias, const void* state, void* state_n, int silu,
                                                        int B, int D) {
  using T_ = typename Elem<F>::T;
  const int ch = (blockIdx.x * 256 + threadIdx.x) * E;
  if (ch >= B * D) return;
  const int b = ch / D, j = ch - b * D;
  const bool cut = RESET && static_cast<const unsigned char*>(reset.p)[b * reset.sb];
  const long long row = (long long)b * (K - 1) * D + j;
  Pack<F, E> v[K];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) {
    v[k] = Pack<F, E>{};
    if (state && !cut) v[k] = load_pack<F, E>(static_cast<const T_*>(state) + row + (long long)k * D);
  }
  v[K - 1] = load_pack<F, E>(static_cast<const T_*>(x.p) + b * x.sb + j);
  Pack<F, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float u = bias ? bias[j + e] : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) u = __builtin_fmaf(w[(long long)(j + e) * K + k], Elem<F>::up(v[k].v[e]), u);
    if (silu) u *= gate_sigmoid<F>(u);
    o.v[e] = Elem<F>::down(u);
  }
  store_pack<F, E>(static_cast<T_*>(y.p) + b * y.sb + j, o);
#pragma unroll
  for (int k = 1; k < K; ++k)
    __builtin_memcpy(static_cast<T_*>(state_n) + row + (long long)(k - 1) * D, &v[k], sizeof(v[k]));
}

ConvPlan plan_conv(int T, int B, int D, int E) {
  ConvPlan p;
  p.per = (D + E - 1) / E;
  p.log2g = 0;
  while (p.log2g < 6 && (1 << p.log2g) < p.per) ++p.log2g;
  p.tiles = (p.per + (1 << p.log2g) - 1) >> p.log2g;
  // 16 waves for each of 256 CUs
  const long long at_once = (long long)p.tiles * B, rows = 4096ll << (6 - p.log2g);
  const long long want = std::max(1ll, rows / std::max(1ll, at_once));
  const long long least = (T + want - 1) / want;
  p.seg = (int)std::min<long long>(kMaxSeg, std::max<long long>(16, (least + kBlock - 1) / kBlock * kBlock));
  p.nseg = std::max(1, (T + p.seg - 1) / p.seg);
  p.rows = (long long)p.nseg * B;
  return p;
}

int fwd_vec(int D, int fmt) {
  const int e = fmt == kElemF32 ? 4 : 8;
  return D < e ? 1 : e;
}
int bwd_vec(int D) { return D < 4 ? 1 : 4; }

int check_conv(const char* who, int T, int B, int D, int K, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (T < 0 || B < 0 || D < 0) return fail(HSL_ERR_ARG, "%s: negative size (T=%d B=%d D=%d)", who, T, B, D);
  if (K < 1 || K > kMaxTaps) return fail(HSL_ERR_ARG, "%s: %d taps, must be 1..%d", who, K, kMaxTaps);
  // rows and channels are counted in 32 bits; a launch holds fewer than 2^32 threads
  if (T >= (1 << 30) || (long long)B * D >= (1ll << 27) || (long long)T * B * D >= (1ll << 38))
    return fail(HSL_ERR_UNSUPPORTED,
                "%s: T=%d B=%d D=%d is beyond the kernels' 32-bit index range (needs T < 2^30, B*D < 2^27 and T*B*D < "
                "2^38)",
                who, T, B, D);
  return HSL_OK;
}

// f(fmt, taps, reset) as integral constants.
template <class Fn>
int with_conv(int fmt, int K, bool reset, Fn f) {
  return with_fmt(fmt, [&](auto F) {
    auto with_reset = [&](auto k) { return reset ? f(F, k, std::true_type{}) : f(F, k, std::false_type{}); };
    switch (K) {
      case 1: return with_reset(std::integral_constant<int, 1>{});
      case 2: return with_reset(std::integral_constant<int, 2>{});
      case 3: return with_reset(std::integral_constant<int, 3>{});
      default: return with_reset(std::integral_constant<int, 4>{});
    }
  });
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

int hsl_conv_fwd(const void* x, long long x_t, long long x_b, const float* w, const float* bias, const void* state,
                 const void* reset, long long rs_t, long long rs_b, void* y, long long y_t, long long y_b,
                 void* state_n, int silu, int T, int B, int D, int K, int fmt, void* stream) {
  HSL_CHECK(check_conv("hsl_conv_fwd", T, B, D, K, fmt));
  if (B == 0 || D == 0) return HSL_OK;
  if (!w || (K > 1 && !state_n) || (T > 0 && (!x || !y))) return fail(HSL_ERR_ARG, "hsl_conv_fwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_conv(fmt, K, reset != nullptr, [&](auto F, auto KK, auto R) {
    constexpr int kF = decltype(F)::value, kK = decltype(KK)::value;
    constexpr bool kR = decltype(R)::value;
    constexpr int kE = kF == kElemF32 ? 4 : 8;
    if (T == 1) {
      const Stream xs{x, 0, x_b}, rs{reset, 0, rs_b};
      const OutStream ys{y, 0, y_b};
      const dim3 grid((B * (D % 2 ? D : D / 2) + 255) / 256), block(256);
      if (D % 2)
        hipLaunchKernelGGL((conv_step_kernel<kF, 1, kK, kR>), grid, block, 0, s, xs, rs, ys, w, bias, state, state_n,
                           silu, B, D);
      else
        hipLaunchKernelGGL((conv_step_kernel<kF, 2, kK, kR>), grid, block, 0, s, xs, rs, ys, w, bias, state, state_n,
                           silu, B, D);
    } else {
      ConvArgs a{};
      a.x = {x, x_t, x_b};
      a.reset = {reset, rs_t, rs_b};
      a.y = {y, y_t, y_b};
      a.w = w;
      a.bias = bias;
      a.state = state;
      a.state_n = state_n;
      a.T = T;
      a.B = B;
      a.D = D;
      a.silu = silu;
      const int e = fwd_vec(D, fmt);
      a.p = plan_conv(T, B, D, e);
      const dim3 grid((unsigned)a.p.row_blocks() * a.p.tiles), block(kWaves * 64);
      if (e == 1)
        hipLaunchKernelGGL((conv_fwd_kernel<kF, 1, kK, kR>), grid, block, 0, s, a);
      else
        hipLaunchKernelGGL((conv_fwd_kernel<kF, kE, kK, kR>), grid, block, 0, s, a);
    }
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

size_t hsl_conv_ws_bytes(int T, int B, int D, int K) {
  if (check_conv("hsl_conv_ws_bytes", T, B, D, K, kElemF32) != HSL_OK || B == 0 || D == 0) return 0;
  return (size_t)plan_conv(T, B, D, bwd_vec(D)).row_blocks() * (K + 1) * D * sizeof(float);
}

int hsl_conv_bwd(const void* x, long long x_t, long long x_b, const float* w, const float* bias, const void* state,
                 const void* reset, long long rs_t, long long rs_b, const void* dy, long long dy_t, long long dy_b,
                 const void* dstate_n, void* dx, long long dx_t, long long dx_b, float* dw, float* dbias, void* dstate,
                 int silu, void* ws, size_t ws_bytes, int T, int B, int D, int K, int fmt, void* stream) {
  HSL_CHECK(check_conv("hsl_conv_bwd", T, B, D, K, fmt));
  if (D == 0) return HSL_OK;
  if (!w || !dw || (T > 0 && B > 0 && (!x || !dx))) return fail(HSL_ERR_ARG, "hsl_conv_bwd: null pointer");
  const size_t need = hsl_conv_ws_bytes(T, B, D, K);
  if (need && (!ws || ws_bytes < need))
    return fail(HSL_ERR_ARG, "hsl_conv_bwd: workspace %zu bytes, need %zu", ws_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int parts = 0;
  if (B > 0) {
    ConvArgs a{};
    a.x = {x, x_t, x_b};
    a.dy = {dy, dy_t, dy_b};
    a.reset = {reset, rs_t, rs_b};
    a.dx = {dx, dx_t, dx_b};
    a.w = w;
    a.bias = bias;
    a.state = state;
    a.dstate_n = dstate_n;
    a.dstate = dstate;
    a.part = static_cast<float*>(ws);
    a.T = T;
    a.B = B;
    a.D = D;
    a.silu = silu;
    a.p = plan_conv(T, B, D, bwd_vec(D));
    parts = a.p.row_blocks();
    HSL_CHECK(with_conv(fmt, K, reset != nullptr, [&](auto F, auto KK, auto R) {
      constexpr int kF = decltype(F)::value, kK = decltype(KK)::value;
      constexpr bool kR = decltype(R)::value;
      const dim3 grid((unsigned)parts * a.p.tiles), block(kWaves * 64);
      if (bwd_vec(D) == 1)
        hipLaunchKernelGGL((conv_bwd_kernel<kF, 1, kK, kR>), grid, block, 0, s, a);
      else
        hipLaunchKernelGGL((conv_bwd_kernel<kF, 4, kK, kR>), grid, block, 0, s, a);
      HSL_HIP(hipGetLastError());
      return (int)HSL_OK;
    }));
  }
  const long long cols = (long long)(K + 1) * D;
  hipLaunchKernelGGL(conv_sum_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(kSumStrips * 64), 0, s,
                     static_cast<const float*>(ws), dw, dbias, parts, K, D);
  HSL_HIP(hipGetLastError());
  return HSL_OK;
}

}  // extern "C"
