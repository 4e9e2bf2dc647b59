// Gated linear recurrence, forward, backward and one step.
//   f = sigmoid(z), w = sigmoid(-z) = 1 - f,   h_t = f_t h'_{t-1} + w_t v_t,
//   h'_{t-1} = 0 where reset_t is set (a new sequence begins at t), else h_{t-1};  h_{-1} = h0.
// Backward, with U_T = dh_n:  G_t = dout_t + U_{t+1},  U_t = reset_t ? 0 : f_t G_t,
//   dv_t = w_t G_t,  dz_t = G_t (h'_{t-1} - v_t) f_t w_t,  dh0 = U_0.
// zv holds z in its first H and v in its last H channels.  The state is fp32 throughout; out is
// h rounded once.  ck keeps h as it enters every 8th step, in fp32, from which the backward runs
// the steps again (the rounded out would cost dz its precision where h and v are close).
#include "lm.h"

namespace hsl {
namespace {

constexpr int kGatedCk = 8;  // steps per checkpoint row

struct Gates {
  float f, w;
};
// e = exp(-|z|) is at most 1, so neither gate is a difference: the larger is 1 / (1 + e), the
// smaller e / (1 + e).
__device__ __forceinline__ Gates gates_of(float z) {
  const float e = exp_f(-__builtin_fabsf(z));
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  return z >= 0.f ? Gates{big, small} : Gates{small, big};
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

template <int F>
__global__ __launch_bounds__(256) void gated_fwd_kernel(Stream zv, const float* h0, Stream reset, OutStream out,
                                                        float* h_n, float* __restrict__ ck, int T, int B, int H) {
  using E = Elem<F>;
  const int ch = blockIdx.x * 256 + threadIdx.x;
  if (ch >= B * H) return;
  const int b = ch / H, j = ch % H;
  float h = h0 ? h0[ch] : 0.f;
  for (int t = 0; t < T; ++t) {
    if (ck && t % kGatedCk == 0) ck[(size_t)(t / kGatedCk) * B * H + ch] = h;
    const auto* row = static_cast<const typename E::T*>(zv.p) + t * zv.st + b * zv.sb;
    const Gates g = gates_of(E::up(row[j]));
    const float wv = g.w * E::up(row[H + j]);
    const bool cut = reset.p && static_cast<const unsigned char*>(reset.p)[t * reset.st + b * reset.sb];
    h = cut ? wv : __builtin_fmaf(g.f, h, wv);
    static_cast<typename E::T*>(out.p)[t * out.st + b * out.sb + j] = E::down(h);
  }
  h_n[ch] = h;
}

template <int F>
__global__ __launch_bounds__(256) void gated_bwd_kernel(Stream zv, Stream reset, const float* __restrict__ ck,
                                                        Stream dout, const float* __restrict__ dh_n, OutStream dzv,
                                                        float* __restrict__ dh0, int T, int B, int H) {
  using E = Elem<F>;
  const int ch = blockIdx.x * 256 + threadIdx.x;
  if (ch >= B * H) return;
  const int b = ch / H, j = ch % H;
  float U = dh_n ? dh_n[ch] : 0.f;
  for (int k = (T - 1) / kGatedCk; k >= 0; --k) {
    float prev[kGatedCk];
    float h = ck[(size_t)k * B * H + ch];
    const int n = min(kGatedCk, T - k * kGatedCk);
    for (int s = 0; s < n; ++s) {
      const int t = k * kGatedCk + s;
      const auto* row = static_cast<const typename E::T*>(zv.p) + t * zv.st + b * zv.sb;
      const Gates g = gates_of(E::up(row[j]));
      const float wv = g.w * E::up(row[H + j]);
      const bool cut = reset.p && static_cast<const unsigned char*>(reset.p)[t * reset.st + b * reset.sb];
      prev[s] = cut ? 0.f : h;
      h = cut ? wv : __builtin_fmaf(g.f, h, wv);
    }
    for (int s = n - 1; s >= 0; --s) {
      const int t = k * kGatedCk + s;
      const auto* row = static_cast<const typename E::T*>(zv.p) + t * zv.st + b * zv.sb;
      const Gates g = gates_of(E::up(row[j]));
      const float v = E::up(row[H + j]);
      const bool cut = reset.p && static_cast<const unsigned char*>(reset.p)[t * reset.st + b * reset.sb];
      const float G =
          dout.p ? E::up(static_cast<const typename E::T*>(dout.p)[t * dout.st + b * dout.sb + j]) + U : U;
      auto* drow = static_cast<typename E::T*>(dzv.p) + t * dzv.st + b * dzv.sb;
      drow[j] = E::down(G * (prev[s] - v) * (g.f * g.w));
      drow[H + j] = E::down(g.w * G);
      U = cut ? 0.f : g.f * G;
    }
  }
  if (dh0) dh0[ch] = U;
}

int check_gated(const char* who, int T, int B, int H, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  return check_shape(who, T, B, 0, H);
}

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

int hsl_gated_ck_rows(int T) { return T <= 0 ? 0 : (T + kGatedCk - 1) / kGatedCk; }

size_t hsl_gated_ws_bytes(int T, int B, int H) { return 0; }

int hsl_gated_fwd(const void* zv, long long zv_t, long long zv_b, const float* h0, const void* reset, long long rs_t,
                  long long rs_b, void* out, long long out_t, long long out_b, float* h_n, float* ck, void* ws,
                  size_t ws_bytes, int T, int B, int H, int fmt, void* stream) {
  HSL_CHECK(check_gated("hsl_gated_fwd", T, B, H, fmt));
  if (B == 0 || H == 0) return HSL_OK;
  if (!h_n || (T > 0 && (!zv || !out))) return fail(HSL_ERR_ARG, "hsl_gated_fwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return with_fmt(fmt, [&](auto f) {
    hipLaunchKernelGGL(gated_fwd_kernel<decltype(f)::value>, dim3((B * H + 255) / 256), dim3(256), 0, s,
                       Stream{zv, zv_t, zv_b}, h0, Stream{reset, rs_t, rs_b}, OutStream{out, out_t, out_b}, h_n, ck, T,
                       B, H);
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
  return with_fmt(fmt, [&](auto f) {
    hipLaunchKernelGGL(gated_bwd_kernel<decltype(f)::value>, dim3((B * H + 255) / 256), dim3(256), 0, s,
                       Stream{zv, zv_t, zv_b}, Stream{reset, rs_t, rs_b}, ck, Stream{dout, do_t, do_b}, dh_n,
                       OutStream{dzv, dz_t, dz_b}, dh0, T, B, H);
    HSL_HIP(hipGetLastError());
    return (int)HSL_OK;
  });
}

}  // extern "C"
