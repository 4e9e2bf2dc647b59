// A 256 x 256 tile of a product of 16-bit operands (bf16 or fp16) with fp32 sums, for kernels with
// their own epilogues (xent.hip): C[i][j] = sum_k A(i, k) B(j, k).
//
// Workgroup = 8 waves, 2 (rows) x 4 (columns) of 128 x 64 each, in 4 x 2 fragments of the 32x32x16
// instruction.  A slice is 64 deep; two slices are in LDS (128 KB), and the next one is copied from
// memory straight to LDS while this one multiplies.  A copy instruction moves 64 pieces of 16 bytes to
// consecutive addresses, so the layout in LDS is made by choosing which piece each lane fetches:
//   an operand whose k are neighbours in memory ([row][k]) lies as [256 rows][8 pieces of 8 k], piece p of
//   row r at place p ^ f(r), f(r) = (r ^ r >> 3) & 7, so that the 16 rows that a read serves at a time are
//   in different banks;
//   an operand whose rows are neighbours ([k][row]) lies as [64 k][32 pieces of 8 rows], piece p of k at
//   place p ^ 4 (k & 3), and is read by the transposing LDS read, which gives lane i of 16 the four
//   values (k .. k+3, row i) from 16 addresses of 4 rows each.
// Pieces beyond the operand's rows or k read as zeros (a buffer's bounds), nothing outside is touched.
// Operands have 16-byte aligned rows.
#pragma once

#include "lm.h"

namespace hsl {

constexpr int kMmTile = 256, kMmSlice = 64, kMmThreads = 512;
constexpr int kMmOperand = kMmTile * kMmSlice * 2;  // bytes of one operand's slice
constexpr int kMmLds = 4 * kMmOperand;

typedef __bf16 mm_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 mm_h8 __attribute__((ext_vector_type(8)));
typedef unsigned mm_u4 __attribute__((ext_vector_type(4)));
typedef short mm_s4 __attribute__((ext_vector_type(4)));

// An operand from its tile's first row and first k on: `rows` of its tile's 256 exist, and k of them.
// ld (elements) is between rows in memory, or between k where TRANS.
struct MmOperand {
  const unsigned short* p;
  long long ld;
  int rows, k;
};

template <bool TRANS>
struct MmLoad {
  unsigned off[4];  // bytes from the slice's first element
  int at[4];        // the piece's first k (TRANS: its k) in the slice; beyond every k where no row exists
  __device__ __forceinline__ void init(const MmOperand& o, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = (wave * 4 + j) * 64 + lane;
      if constexpr (TRANS) {
        const int k = p >> 5, c = (p & 31) ^ (4 * (k & 3));
        off[j] = (unsigned)((k * o.ld + c * 8) * 2);
        at[j] = c * 8 < o.rows ? k : 0x7fffffff;
      } else {
        const int r = p >> 3, c = (p & 7) ^ ((r ^ (r >> 3)) & 7);
        off[j] = (unsigned)((r * o.ld + c * 8) * 2);
        at[j] = r < o.rows ? c * 8 : 0x7fffffff;
      }
    }
  }
  // Copies the slice from k0 on to the operand's place in LDS.
  __device__ __forceinline__ void copy(const MmOperand& o, int k0, char* lds, int wave) const {
    const unsigned short* base = o.p + (TRANS ? k0 * o.ld : (long long)k0);
    const int left = o.k - k0;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(base), (short)0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned v = at[j] < left ? off[j] : kOffNone;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(lds + (wave * 4 + j) * 1024), 16, (int)v, 0, 0, 0);
    }
  }
};

// Reads one 32-row fragment (row or column fragment i of the wave) of k-step ks.
template <bool TRANS>
struct MmRead {
  int base, x[4];
  __device__ __forceinline__ void init(int first, int lane) {  // first row of the wave: a multiple of 64
    if constexpr (TRANS) {
      const int j = lane & 15, g = lane >> 4;
      base = (8 * (g >> 1) + (j >> 2)) * 512 + (j & 1) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = ((first / 8 + i * 4 + 2 * (g & 1) + ((j & 3) >> 1)) ^ (4 * (j >> 2))) * 16;
    } else {
      const int r = lane & 31, half = lane >> 5;
      base = (first + r) * 128;
      const int f = (r ^ ((first + r) >> 3)) & 7;
#pragma unroll
      for (int s = 0; s < 4; ++s) x[s] = ((s * 2 + half) ^ f) * 16;
    }
  }
  __device__ __forceinline__ mm_u4 read(const char* lds, int i, int ks) const {
    if constexpr (TRANS) {
      typedef __attribute__((address_space(3))) mm_s4* P;
      const char* p = lds + base + x[i] + ks * (16 * 512);
      const mm_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p));
      const mm_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * 512));
      mm_u4 r;
      __builtin_memcpy(&r, &lo, 8);
      __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
      return r;
    } else {
      // rows 32 further have f with bit 2 turned over, which is the step two further
      return *reinterpret_cast<const mm_u4*>(lds + base + i * (32 * 128) + x[i & 1 ? ks ^ 2 : ks]);
    }
  }
};

template <bool FP16>
__device__ __forceinline__ f16v mm_mfma(mm_u4 a, mm_u4 b, f16v c) {
  if constexpr (FP16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(mm_h8, a), __builtin_bit_cast(mm_h8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(mm_bf8, a), __builtin_bit_cast(mm_bf8, b), c, 0,
                                                   0, 0);
}

// acc[i][j]: rows 32 i, columns 32 j of the wave's block (rows from 128 (wave / 4), columns from
// 64 (wave % 4)): lane l, register r is row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32.
// nk: slices.  lds: kMmLds bytes, free when the call returns (after a barrier).
template <bool FP16, bool TA, bool TB>
__device__ __forceinline__ void mm_tile(const MmOperand& A, const MmOperand& B, int nk, char* lds, f16v (&acc)[4][2]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  MmLoad<TA> la;
  MmLoad<TB> lb;
  la.init(A, wave, lane);
  lb.init(B, wave, lane);
  MmRead<TA> ra;
  MmRead<TB> rb;
  ra.init((wave >> 2) * 128, lane);
  rb.init((wave & 3) * 64, lane);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f16v{};
  la.copy(A, 0, lds, wave);
  lb.copy(B, 0, lds + kMmOperand, wave);
  __syncthreads();
  for (int it = 0; it < nk; ++it) {
    char* const now = lds + (it & 1) * (2 * kMmOperand);
    char* const next = lds + (~it & 1) * (2 * kMmOperand);
    if (it + 1 < nk) {
      la.copy(A, (it + 1) * kMmSlice, next, wave);
      lb.copy(B, (it + 1) * kMmSlice, next + kMmOperand, wave);
    }
#pragma unroll
    for (int ks = 0; ks < kMmSlice / 16; ++ks) {
      mm_u4 a[4], b[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) b[j] = rb.read(now + kMmOperand, j, ks);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = ra.read(now, i, ks);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mm_mfma<FP16>(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
}

}  // namespace hsl
