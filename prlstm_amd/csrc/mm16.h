// A 256 x 256 tile of a product of 16-bit operands (bf16 or fp16) with fp32 sums, for kernels with
// their own epilogues (xent.hip): C[i][j] = sum_k A(i, k) B(j, k).
//
// Workgroup = 8 waves, two a SIMD, 2 (rows) x 4 (columns) of 128 x 64 each, in 4 x 2 fragments of the
// 32x32x16 instruction.  A slice is 32 deep; four are in LDS (128 KB), copied from memory straight to LDS.
// While half a slice multiplies, the other half's operands, or the next slice's first ones, are read
// from LDS; the one barrier a slice, between its halves, says that the next slice has arrived and that this
// one's place is free for the slice four further.
//
// A copy instruction moves 64 pieces of 16 bytes to consecutive addresses, so the layout in LDS is made
// by choosing which piece each lane fetches:
//   an operand whose k are neighbours in memory ([row][k]) lies as [256 rows][4 pieces of 8 k], piece p of
//   row r at place p ^ (r >> 2 & 3), so that the 16 rows that a read serves at a time are in different
//   banks;
//   an operand whose rows are neighbours ([k][row]) lies as [32 k][32 pieces of 8 rows], piece p of k at
//   place p ^ 4 (k & 3), and is read by the transposing LDS read, which gives lane i of 16 the four
//   values (k .. k+3, row i) from 16 addresses of 4 rows each.
// Pieces beyond the operand's rows or k read as zeros (a buffer's bounds), nothing outside is touched.
// Operands have 16-byte aligned rows.
//
// AF = 2 in place of 4: a tile of 128 rows, for products that have too few tiles of 256 for the chip's CUs.
//
// SPLIT: fp32 operands as three bf16 pieces each (x = x0 + x1 + x2, 8 bits a piece), in planes: the product is six
// products of pieces, the smallest first, of each slice in turn (so that a piece's slice, which three of them take, comes
// from the caches); what is left out, x1 w2, x2 w1 and x2 w2, is below 2^-25 of |x| |w|.
//
// The copies are written in assembly because the compiler, which cannot tell the four slices apart, would
// wait for all copies before each read.  So the waits for them are written too: a wave's copies, loads and
// stores end in order, so a wait for all but the last n is right where at least n were issued behind
// those that it is for.
#pragma once

#include "lm.h"

namespace hsl {

constexpr int kMmTile = 256, kMmSlice = 32, kMmThreads = 512, kMmStages = 4;
constexpr int kMmFrag = 64 * kMmSlice * 2;        // bytes of a slice's 64 rows: 32 of each of A's two rows of waves
constexpr int kMmOperand = 4 * kMmFrag;           // of one operand's slice
constexpr int mm_lds(int af) { return kMmStages * (af * kMmFrag + kMmOperand); }
constexpr int kMmLds = mm_lds(4);
// Instructions of a wave for the slice of an operand of n fragments.
constexpr int mm_copies(int n) { return n * kMmFrag / 1024 / (kMmThreads / 64); }
static_assert(mm_copies(4) == 2 && mm_copies(2) == 1, "whole instructions");

typedef __bf16 mm_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 mm_h8 __attribute__((ext_vector_type(8)));
typedef unsigned mm_u4 __attribute__((ext_vector_type(4)));
typedef short mm_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char mm_lds_char;

// acc[i][j]: rows 32 i, columns 32 j of the wave's block (rows from 128 (wave / 4), columns from
// 64 (wave % 4)): lane l, register r is row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32.
template <int AF>
using MmAccOf = float[AF][2][16];
typedef MmAccOf<4> MmAcc;

// An operand from its tile's first row and first k on: `rows` of its tile's 256 exist, and k of them.
// ld (elements) is between rows in memory, or between k where TRANS.
struct MmOperand {
  const unsigned short* p;
  long long ld;
  int rows, k;
  long long plane = 0;  // elements between pieces
};

// For an operand of assembly that has to be in a scalar register.
__device__ __forceinline__ unsigned mm_uniform(unsigned v) { return (unsigned)__builtin_amdgcn_readfirstlane((int)v); }

template <bool TRANS, int N>  // N fragments
struct MmLoad {
  unsigned row, ld;  // bytes: of the lane's row (TRANS: k) among a copy's 16 (2), between rows
  int lane;
  __device__ __forceinline__ void init(const MmOperand& o, int l) {
    lane = l;
    ld = (unsigned)(o.ld * 2);
    row = (TRANS ? lane >> 5 : lane >> 2) * ld;
  }
  // Copies piece `piece`'s slice from k0 on to the operand's place in LDS.
  __device__ __forceinline__ void copy(const MmOperand& o, int piece, int k0, unsigned lds, int wave) const {
    const unsigned long long base =
        (unsigned long long)(o.p + piece * o.plane + (TRANS ? k0 * o.ld : (long long)k0));
    const unsigned lo = mm_uniform((unsigned)base), hi = mm_uniform((unsigned)(base >> 32));
    const mm_u4 rsrc = {lo, hi & 0xffffu, 0x7fffffffu, 0x00020000u};
    const unsigned step = mm_uniform(ld), to = mm_uniform(lds);
    const int left = o.k - k0;
#pragma unroll
    for (int j = 0; j < mm_copies(N); ++j) {
      const int n = wave * mm_copies(N) + j;  // of the operand's 4 N copies
      int c, first;
      bool in;
      if constexpr (TRANS) {
        first = n * 2;
        c = (lane & 31) ^ (4 * ((first + (lane >> 5)) & 3));
        in = c * 8 < o.rows && (lane >> 5) < left - first;
      } else {
        first = n * 16;
        c = (lane & 3) ^ ((lane >> 4) & 3);
        in = c * 8 < left && (lane >> 2) < o.rows - first;
      }
      const unsigned off = in ? row + c * 16 : kOffNone;
      // (m0 is never kept by the compiler; a write of it may not be followed at once by a copy to LDS)
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "buffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to + n * 1024),
          "v"(off), "s"(rsrc), "s"(first * step)
          : "memory");
    }
  }
};

// Wave `wave` copies the 1 KB at `from` (16-byte aligned) to piece `wave` of `to`, or zeros.
__device__ __forceinline__ void mm_copy_kb(const void* from, bool in, const void* to, int wave) {
  const unsigned long long base = (unsigned long long)from;
  const unsigned lo = mm_uniform((unsigned)base), hi = mm_uniform((unsigned)(base >> 32));
  const mm_u4 rsrc = {lo, hi & 0xffffu, 0x7fffffffu, 0x00020000u};
  const unsigned at = mm_uniform((unsigned)(unsigned long long)(const mm_lds_char*)to + wave * 1024);
  const unsigned off = in ? (threadIdx.x & 63) * 16 : kOffNone;
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(rsrc)
      : "memory");
}

// Reads a wave's N 32-row fragments of a slice's two k-steps.
template <bool TRANS, int N>
struct MmRead {
  int x[TRANS ? N : 2];  // bytes: of fragment i where TRANS, otherwise of k-step ks
  __device__ __forceinline__ void init(int first, int lane) {  // first row of the wave
    if constexpr (TRANS) {
      const int j = lane & 15, g = lane >> 4;
#pragma unroll
      for (int i = 0; i < N; ++i)
        x[i] = (8 * (g >> 1) + (j >> 2)) * 512 + (j & 1) * 8 +
               ((first / 8 + i * 4 + 2 * (g & 1) + ((j & 3) >> 1)) ^ (4 * (j >> 2))) * 16;
    } else {
      const int r = lane & 31, half = lane >> 5;
#pragma unroll
      for (int s = 0; s < 2; ++s) x[s] = (first + r) * 64 + ((s * 2 + half) ^ ((r >> 2) & 3)) * 16;
    }
  }
  __device__ __forceinline__ mm_u4 read(const char* lds, int ks, int i) const {
    if constexpr (TRANS) {
      typedef __attribute__((address_space(3))) mm_s4* P;
      const char* p = lds + x[i] + ks * (16 * 512);
      const mm_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p));
      const mm_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * 512));
      mm_u4 f;
      __builtin_memcpy(&f, &lo, 8);
      __builtin_memcpy(reinterpret_cast<char*>(&f) + 8, &hi, 8);
      return f;
    } else {
      return *reinterpret_cast<const mm_u4*>(lds + x[ks] + i * (32 * 64));
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

// The products of a workgroup's tiles, one after the other: while a tile's last slices multiply, the next
// one's first are copied, so that they have arrived when its product begins.  lds: kMmLds bytes that hold
// nothing else from begin() on.
template <bool FP16, bool TA, bool TB, bool SPLIT = false, int AF = 4>
struct MmPipe {
  static_assert(AF == 4 || (AF == 2 && !TA), "a transposed slice has 256 rows");
  static constexpr int kA = AF * kMmFrag, kStage = kA + kMmOperand, kCopies = mm_copies(AF) + mm_copies(4);
  MmOperand A, B;
  MmLoad<TA, AF> la;
  MmLoad<TB, 4> lb;
  MmRead<TA, AF> ra;
  MmRead<TB, 2> rb;
  const char* lds;
  int wave, stage, slices;  // stage: where the tile's first slice lies; slices: of a tile

  __device__ __forceinline__ void copy(const MmOperand& a, const MmOperand& b, int slice, int at) const {
    const unsigned p = (unsigned)(unsigned long long)(const mm_lds_char*)lds + (at % kMmStages) * kStage;
    int pa = 0, pb = 0;
    if constexpr (SPLIT) {
      const int pair = (unsigned)slice % 6;
      slice = (unsigned)slice / 6;
      pa = 0x118 >> (2 * pair) & 3;  // 0 2 1 0 1 0
      pb = 0x052 >> (2 * pair) & 3;  // 2 0 1 1 0 0
    }
    la.copy(a, pa, slice * kMmSlice, p, wave);
    lb.copy(b, pb, slice * kMmSlice, p + kA, wave);
  }
  // Every tile has k up to K and the same strides as this first one.
  __device__ __forceinline__ void begin(const char* space, const MmOperand& a, const MmOperand& b, int K) {
    const int lane = threadIdx.x & 63;
    A = a;
    B = b;
    lds = space;
    stage = 0;
    slices = max(kMmStages, (SPLIT ? 6 : 1) * ((K + kMmSlice - 1) / kMmSlice));  // slices beyond K are zeros
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    la.init(A, lane);
    lb.init(B, lane);
    ra.init((wave >> 2) * 32 * AF, lane);
    rb.init((wave & 3) * 64, lane);
#pragma unroll
    for (int s = 0; s < kMmStages; ++s) copy(A, B, s, s);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(3 * kCopies) : "memory");  // 3 slices may be on their way
  }
  // acc = this tile's product; nextA, nextB: the next tile, or operands without k.  with_next() is called
  // before the first copy for it: where a tile has no more slices than are in LDS, before any barrier of run(), so
  // that other waves may still be behind the tile before.  LATER (a count): loads and stores that the wave has issued for sure since the
  // product before, which the waits for the copies before them leave out; later: whether there was one.
  template <int LATER, class Fn>
  __device__ __forceinline__ void run(MmAccOf<AF>& acc, const MmOperand& nextA, const MmOperand& nextB, bool later,
                                      Fn with_next) {
    f16v sum[AF][2];
#pragma unroll
    for (int i = 0; i < AF; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) sum[i][j] = f16v{};
    auto place = [&](int slice) { return lds + ((stage + slice) % kMmStages) * kStage; };
    mm_u4 a0[AF], b0[2], a1[AF], b1[2];
#pragma unroll
    for (int i = 0; i < AF; ++i) a0[i] = ra.read(place(0), 0, i);
#pragma unroll
    for (int j = 0; j < 2; ++j) b0[j] = rb.read(place(0) + kA, 0, j);
    // The order is fixed: between two products there is always something to issue, and there is a product
    // to run while the wave is at the barrier.
    auto fixed = [] { __builtin_amdgcn_sched_barrier(0); };
    auto product = [&](mm_u4 a, const mm_u4(&b)[2], int i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) sum[i][j] = mm_mfma<FP16>(a, b[j], sum[i][j]);
      fixed();
    };
    auto slice = [&](int it, const MmOperand& from_a, const MmOperand& from_b, int ahead) {
      const char* const now = place(it);
      const char* const next = place(it + 1);
      product(a0[0], b0, 0);
      b1[0] = rb.read(now + kA, 1, 0);
      b1[1] = rb.read(now + kA, 1, 1);
      a1[0] = ra.read(now, 1, 0);
      fixed();
      product(a0[1], b0, 1);
#pragma unroll
      for (int i = 1; i < AF; ++i) a1[i] = ra.read(now, 1, i);
      fixed();
#pragma unroll
      for (int i = 2; i < AF; ++i) product(a0[i], b0, i);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      product(a1[0], b1, 0);
      // this slice is in registers and the next one has arrived: 2 more may be on their way, and behind the
      // slices that were copied before it, what `later` says
      if (LATER > 0 && later && it < kMmStages - 1)
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(2 * kCopies + LATER) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(2 * kCopies) : "memory");
      fixed();
      // (the last time, of the next tile: they are read again behind the epilogue rather than kept)
      b0[0] = rb.read(next + kA, 0, 0);
      b0[1] = rb.read(next + kA, 0, 1);
      a0[0] = ra.read(next, 0, 0);
      fixed();
      if constexpr (AF > 2) product(a1[1], b1, 1);
#pragma unroll
      for (int i = 1; i < AF; ++i) a0[i] = ra.read(next, 0, i);
      fixed();
      if constexpr (AF > 2) product(a1[2], b1, 2);
      copy(from_a, from_b, ahead, stage + it);  // to where this slice lay
      fixed();
      product(a1[AF - 1], b1, AF - 1);
    };
    int it = 0;
    for (; it < slices - kMmStages; ++it) slice(it, A, B, it + kMmStages);
    with_next();
    for (; it < slices; ++it) slice(it, nextA, nextB, it + kMmStages - slices);
#pragma unroll
    for (int i = 0; i < AF; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = sum[i][j][r];
    stage = (stage + slices) % kMmStages;
    A = nextA;
    B = nextB;
  }
};

}  // namespace hsl
