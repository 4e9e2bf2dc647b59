// Helpers shared by the language-model operators (embed.hip, gated.hip, logprob.hip).
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
