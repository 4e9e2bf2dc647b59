// Helpers shared by the language-model operators (embed.hip, gated.hip, logprob.hip, conv.hip,
// selective_fwd.hip and selective_bwd.hip through selective.h, xent.hip through mm16.h).
#pragma once

#include <type_traits>

#include "hsl_internal.h"

namespace hsl {

// Element formats of the operators' streams, as the C ABI numbers them.
enum ElemFmt { kElemBf16 = 0, kElemF16 = 1, kElemF32 = 2 };
inline bool elem_fmt_ok(int fmt) { return fmt >= kElemBf16 && fmt <= kElemF32; }

// Elements are widened to fp32 when they are read and rounded to nearest even once when they
// are stored.
template <int F>
struct Elem;
template <>
struct Elem<kElemBf16> {
  using T = unsigned short;
  static __device__ __forceinline__ float up(T u) { return __uint_as_float((unsigned)u << 16); }
  static __device__ __forceinline__ T down(float v) { return __builtin_bit_cast(T, (__bf16)v); }
};
template <>
struct Elem<kElemF16> {
  using T = unsigned short;
  static __device__ __forceinline__ float up(T u) { return (float)__builtin_bit_cast(_Float16, u); }
  static __device__ __forceinline__ T down(float v) {
    asm("" : "+v"(v));  // not fused into a mixed-precision multiply that would skip fp32's rounding
    return __builtin_bit_cast(T, (_Float16)v);
  }
};
template <>
struct Elem<kElemF32> {
  using T = float;
  static __device__ __forceinline__ float up(T u) { return u; }
  static __device__ __forceinline__ T down(float v) { return v; }
};

// N values rounded into N neighbouring elements (two bf16 ones are one conversion).
template <int F, int N>
__device__ __forceinline__ void down_all(const float (&f)[N], typename Elem<F>::T (&out)[N]) {
  if constexpr (F == kElemBf16 && N % 2 == 0) {
    typedef float F2 __attribute__((ext_vector_type(2)));
    typedef __bf16 B2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const B2 b = __builtin_convertvector((F2){f[i], f[i + 1]}, B2);
      __builtin_memcpy(&out[i], &b, sizeof(b));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = Elem<F>::down(f[i]);
  }
}

// 16 bytes to any element's alignment (global memory takes unaligned accesses), non-temporal.
template <class V>
__device__ __forceinline__ void store16_nt(void* p, const V& x) {
  typedef unsigned U4 __attribute__((ext_vector_type(4)));
  typedef U4 Raw __attribute__((aligned(2), may_alias));
  static_assert(sizeof(V) == sizeof(U4), "16 bytes");
  U4 u;
  __builtin_memcpy(&u, &x, sizeof(u));
  __builtin_nontemporal_store(u, static_cast<Raw*>(p));
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
template <>
struct RawOf<16> {
  using T = unsigned __attribute__((ext_vector_type(4)));
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

// What a call streams through beyond this is not kept in the caches (the last-level one has 256 MB).
constexpr size_t kCacheBytes = 256u << 20;

// The sticky device word that hsl_device_errors reads, for a kernel's argument (recurrent.hip).
// Bit 1: an id beyond the vocabulary (bit 0 is the persistent kernels').
int device_error_word(unsigned** word);
constexpr unsigned kErrId = 2u;

// Token ids are int32 or int64.
__device__ __forceinline__ long long load_id(const void* ids, int ids64, size_t i) {
  return ids64 ? static_cast<const long long*>(ids)[i] : (long long)static_cast<const int*>(ids)[i];
}

// Sums over lanes that many values need at once: an exchange of halves between two registers and an
// addition leave one register with half of each value's lanes, so n values take about 2 n operations
// where a sum of each alone takes 6 n.
// Lower half-wave: a over lanes l and l + 32; upper half-wave: b.
__device__ __forceinline__ float add32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Even rows of 16 lanes: a over the pair of rows; odd rows: b.
__device__ __forceinline__ float add16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// r[i] over the 16 lanes of a row, i = lane % 16.
__device__ __forceinline__ float sum_rows(float (&r)[16], int lane) {
  const bool b8 = lane & 8, b4 = lane & 4, b2 = lane & 2, b1 = lane & 1;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (b8 ? r[i + 8] : r[i]) + lane_move<0x128>(b8 ? r[i] : r[i + 8]);  // row_ror:8
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (b4 ? r[i + 4] : r[i]) + lane_move<0x141>(b4 ? r[i] : r[i + 4]);  // half mirror
#pragma unroll
  for (int i = 0; i < 2; ++i) r[i] = (b2 ? r[i + 2] : r[i]) + lane_move<0x4e>(b2 ? r[i] : r[i + 2]);  // quad 2,3,0,1
  return (b1 ? r[1] : r[0]) + lane_move<0xb1>(b1 ? r[0] : r[1]);                                       // quad 1,0,3,2
}

__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269502162933349609375f;

// sigmoid(z) next to values of format F.  Rounding z log2 e to fp32 counts as one more rounding of z, which
// 16-bit results (2^-9 or 2^-12 of themselves) do not show, so exp is one product and v_exp_f32 there.
template <int F>
__device__ __forceinline__ float gate_sigmoid(float z) {
  if constexpr (F == kElemF32) return sigmoid_f(z);
  return __builtin_amdgcn_rcpf(1.f + exp2_f(-kLog2e * z));
}

// f(integral_constant<int, fmt>) for the element format of a call.
template <class Fn>
int with_fmt(int fmt, Fn f) {
  switch (fmt) {
    case kElemBf16: return f(std::integral_constant<int, kElemBf16>{});
    case kElemF16: return f(std::integral_constant<int, kElemF16>{});
    default: return f(std::integral_constant<int, kElemF32>{});
  }
}

}  // namespace hsl
