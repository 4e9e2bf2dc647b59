// Cross entropy of a projection on the vocabulary, without keeping the logits:
//   l[n][v] = x[n] . w[v] + bias[v],   loss[n] = log sum_v exp l[n][v] - l[n][target[n]],
//   dl[n][v] = g[n] (exp(l[n][v]) / sum - [v = target[n]]),   g = dloss (0 for a target < 0),
//   dx = dl w,   dw = dl^T x,   dbias = sum_n dl.
//
// One kernel multiplies 256 x 256 tiles (mm16.h) whose rows are tokens of the
// vocabulary and whose columns are the positions, so that a lane has 64 logits of each of 2 positions in
// registers.  The forward reduces them to the tile's largest logit and sum of exponentials, from which a
// second kernel makes the loss; no logit leaves the registers.  The backward computes the logits again,
// a piece of the vocabulary at a time, and writes the piece's dl, for 16-bit operands in fp16, from which one launch
// makes the piece's dw and adds to dx, both in fp32.
//   Rounding dl is the one error that a sum of two roundings' size in dx and dw would show, and fp16's is
// 2^-11 where bf16's, 2^-8, is as large as that of the results themselves (with it bf16 gradients were 1.4
// times as far from the exact ones as when rounded once, few rows' up to twice).  So bf16 operands enter
// these two products as fp16 too, which holds their 8 bits.  Range is made up for by powers of two: a row of dl
// is scaled to |g| = 2^14 .. 2^15, x to as large an element less what its row's g is below the largest one, a
// bf16 w to as large an element; the results take them back.  What is then below fp16's 2^-24 counts as 0: a
// probability below 2^-38, an element 2^-38 of its operand's largest (of x: times its row's |g| over the largest |g|).
//   For few rows dl is kept as two rows, its value and the rest, whose products the sums join: a bf16 one in bf16
// up to 128 rows (2^-17 of it remain), which leave half of a tile empty, so that no copy of w is made for them; an
// fp16 one up to 512 (2^-22), whose error would otherwise be 1.4 times that of one rounding, and by chance more
// where few rows' are added (0.00035 for 0.00021), at the cost of twice the products (8192 rows would take half as
// long again).
// fp32 operands: the same in three bf16 pieces each (mm16.h), dl too; the weight's are made for a piece of the
// vocabulary at a time.
#include <algorithm>
#include <cmath>

#include "mm16.h"

namespace hsl {
namespace {

constexpr size_t kPieceBytes = 256u << 20;  // of a piece's dl
constexpr int kPieceWidth = 1 << 21;        // tokens at most: 256 rows of dl lie within 2^31 bytes

constexpr float kPieceEnd = 0x1.ffp127f;  // the least number that bf16 rounds to infinity

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// A row of nothing but masks (m is -inf beside a sum of NaN where every logit is NaN).
__device__ __forceinline__ bool all_masked(float m, float s) { return m == neg_inf() && s == 0.f; }

// exp(l - m).  (A fused l log2 e - m log2 e would spare the difference, but is off by 2^-24 of l's and m's size rather
// than of their difference's: 1e-6 of a probability at logits of 20.)
__device__ __forceinline__ float exp_from(float l, float m) { return __builtin_amdgcn_exp2f((l - m) * kLog2e); }

// Joins (m, sum exp(l - m)) of two parts of a row.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float big = fmaxf(m, m2), r = big == neg_inf() ? 0.f : big;
  s = s * exp_from(m, r) + s2 * exp_from(m2, r);
  m = big;
}

struct LogitArgs {
  MmOperand w, x;   // from the piece's first token on; from the first position on
  // Filled up to whole tiles:
  const float* bias;  // the piece's, zeros where there is none; -inf beyond the vocabulary
  const int* target;  // the positions' targets (of the whole vocabulary)
  const float4* rows;  // backward: as of row_of(), beyond N of row_beyond()
  int v_first;        // the piece's first token
  int V, N, D, tiles_v, tiles_n;
  float2* part;     // forward: [tile_v or workgroup][N]
  float* own;       // forward: [N], the target's logit
  unsigned short* dl;  // backward: [parts][N][tiles_v * 256]
  float* dbias;        // backward: [tile_n][tiles_v * 256], or null
  float* dl_rows;      // backward of few rows: [V][R]
};

__device__ __forceinline__ void xent_tile_order(int tiles_m, int tiles_n, int id, int* tm, int* tn) {
  // workgroup i runs on XCD i % 8: each XCD takes a contiguous range of the tiles, which go down 8 row
  // panels before they move to the next column
  const int total = tiles_m * tiles_n, even = total & ~7;
  if (id < even) id = (id % 8) * (even / 8) + id / 8;
  constexpr int GM = 8;
  const int group = id / (GM * tiles_n), first = group * GM, rows = min(GM, tiles_m - first);
  const int in = id - group * GM * tiles_n;
  *tm = first + in % rows;
  *tn = in / rows;
}

// What a tile's epilogue needs, copied to LDS with the tile's first slice.
struct TileInfo {
  float4 rows[kMmTile];
  int target[kMmTile];
  float bias[kMmTile];
  char rest[2048];  // of the two waves that have nothing to copy
};
static_assert(sizeof(TileInfo) == 8 * 1024, "a copy of 1 KB by each wave");

// One workgroup's walk over the tiles of 64 AF tokens by 256 positions.
template <int AF>
struct LogitWalk {
  const LogitArgs& a;
  int id, tv, tn;
  __device__ __forceinline__ LogitWalk(const LogitArgs& args) : a(args), id(blockIdx.x) { find(); }
  __device__ __forceinline__ void find() { xent_tile_order(a.tiles_v, a.tiles_n, id, &tv, &tn); }
  __device__ __forceinline__ bool there() const { return id < a.tiles_v * a.tiles_n; }
  __device__ __forceinline__ void next() {
    id += gridDim.x;
    if (there()) find();
  }
  __device__ __forceinline__ MmOperand rows_of(const MmOperand& o, int tile, int rows) const {
    const int first = tile * rows;
    return {o.p + first * o.ld, o.ld, min(rows, o.rows - first), there() ? o.k : 0, o.plane};
  }
  __device__ __forceinline__ MmOperand w() const { return rows_of(a.w, there() ? tv : 0, 64 * AF); }
  __device__ __forceinline__ MmOperand x() const { return rows_of(a.x, there() ? tn : 0, kMmTile); }
  // Wave w copies piece w of the tile's information.
  __device__ __forceinline__ void info(TileInfo* to, int wave) const {
    const char* from = reinterpret_cast<const char*>(a.target + tn * kMmTile);
    bool in = there() && wave < 6;
    if (wave < 4) {
      from = reinterpret_cast<const char*>(a.rows + tn * kMmTile) + wave * 1024;
      in = in && a.rows;
    } else if (wave == 5) {
      from = reinterpret_cast<const char*>(a.bias + tv * 64 * AF);  // 256 of them, the last tile's too
    }
    mm_copy_kb(from, in, to, wave);
  }
};

// A lane's place in a tile: tokens v0 + 32 i + 8 q + e (q, e < 4) and positions n0 + 32 j.
template <int AF>
struct LogitPlace {
  int lane, wave, half, v, c, v0, n0;
  __device__ __forceinline__ LogitPlace(int tv, int tn) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    half = lane >> 5;
    v = (wave >> 2) * 32 * AF;
    c = (wave & 3) * 64 + (lane & 31);
    v0 = tv * 64 * AF + v + 4 * half;
    n0 = tn * kMmTile + c;
  }
};

// Adds the bias, which is there for every call: a branch around it would have the compiler move all sums.
template <int AF>
__device__ __forceinline__ void add_bias(const LogitPlace<AF>& q, const float* bias, MmAccOf<AF>& acc) {
#pragma unroll
  for (int i = 0; i < AF; ++i) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f4 b = *reinterpret_cast<const f4*>(bias + q.v + 4 * q.half + i * 32 + 8 * k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j][4 * k + e] += b[e];
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int F, int AF>
__global__ __launch_bounds__(kMmThreads) void xent_stats_kernel(LogitArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[mm_lds(AF)];
  __shared__ __attribute__((aligned(1024))) TileInfo info[2];
  __shared__ float2 sm[2][kMmTile];
  MmPipe<F == kElemF16, false, false, F == kElemF32, AF> mm;
  LogitWalk<AF> walk(a);
  walk.info(&info[0], __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  mm.begin(lds, walk.w(), walk.x(), a.D);
  for (int par = 0; walk.there(); par ^= 1) {
    const int tv = walk.tv, tn = walk.tn;
    walk.next();
    MmAccOf<AF> acc;
    mm.template run<0>(acc, walk.w(), walk.x(), false, [&] { walk.info(&info[par ^ 1], mm.wave); });
    const LogitPlace<AF> q(tv, tn);
    add_bias(q, info[par].bias, acc);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = q.n0 + j * 32, own = info[par].target[q.c + j * 32] - a.v_first - q.v0;
      float m = neg_inf();
#pragma unroll
      for (int i = 0; i < AF; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
      if (__any((unsigned)own < 32u * AF)) {  // few waves have a target among their tokens
        float l = 0.f;
        bool found = false;
#pragma unroll
        for (int i = 0; i < AF; ++i) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool here = own == i * 32 + 8 * (r >> 2) + (r & 3);
            l = here ? acc[i][j][r] : l;
            found |= here;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (found && n < a.N) a.own[n] = l;
      }
      const float ref = m == neg_inf() ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < AF; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s += exp_from(acc[i][j][r], ref);
        __builtin_amdgcn_sched_barrier(0);
      }
      join(m, s, __shfl_xor(m, 32), __shfl_xor(s, 32));
      if (q.half == 0) sm[q.wave >> 2][q.c + j * 32] = float2{m, s};
    }
    lds_barrier();
    const int n = tn * kMmTile + threadIdx.x;
    if (threadIdx.x < kMmTile && n < a.N) {
      float2 p = sm[0][threadIdx.x];
      join(p.x, p.y, sm[1][threadIdx.x].x, sm[1][threadIdx.x].y);
      a.part[(size_t)tv * a.N + n] = p;
    }
  }
}

// The forward of few rows, which would leave a tile of 256 empty: 32 tokens times 32 rows a workgroup and step,
// whose operands go from memory to the registers of the matrix instructions (the rows' from the caches), 64 of the
// width at a time by each of 4 waves and the next ones already on their way.  The waves' sums meet in LDS, where each
// takes the logits of a quarter of the registers.  Bound by reading w: 11 us at 8 rows and 32768 tokens of width 512
// in bf16 (33 MB, 3.0 TB/s).  Calls of so many rows in this way / in tiles, us, w from memory (from the caches):
//   131072 of 1024:  8 rows 75 / 66 (59 / 59), 16 rows 87 / 67 (67 / 60)
//   131072 of 512:   46 / 43 (37 / 38), 51 / 43 (40 / 38);  of 256: 30 / 31 (25 / 28), 31 / 31 (27 / 28)
//   32768 of 512:    19 / 18 (15.0 / 15.4), 20 / 18 (16 / 16)
//   68480 of 576:    32 / 37 (27 / 35), 36 / 37 (29 / 35);  10000 of 2048: 23 / 33 (20 / 32), 27 / 34 (21 / 32)
// so up to 16 rows where the tiles would leave a fifth of the CUs idle (the last line) or the width is 256 or less,
// otherwise up to 8; at 32 rows, whose reads cost as much as w's, 131072 of 1024 take 84.  (64 tokens a step halve
// those, but leave fewer workgroups: 67, 43 and 35 at 16 rows and 131072 of 1024 and 512 and 68480 of 576.)
// fp32 operands: w is read as it is and cut into its three pieces (mm16.h) in registers, 32 of the width at a time; x's
// pieces are made before.  Up to 64 rows, 32 at a time: 83328 tokens of width 256 take 45 us at 16 rows, 82 at 64 and
// 112 at 96 in this way, 113 in tiles, for which w's pieces are made; 131072 of 1024 265, 523 and 775, 620 in tiles.
constexpr int kFewBlocks = 1024;
constexpr int kFewRows = 8, kFewRowsUnfilled = 16, kFewRowsF32 = 64;
template <int F>
struct FewChunk {  // a lane's operands of kSteps instructions' 16 k
  static constexpr bool kSplit = F == kElemF32;
  static constexpr int kSteps = kSplit ? 2 : 4, kPieces = kSplit ? 3 : 1;
  mm_u4 x[kSteps][kPieces], w[kSteps][kSplit ? 2 : 1];
  // The lane's eight k from `at` on in step 0; xr, wr: its rows of x and w.
  __device__ __forceinline__ void load(const LogitArgs& a, const unsigned short* xr, const void* wr, int at) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i, at += 16) {
      const bool in = at < a.x.k;
#pragma unroll
      for (int q = 0; q < kPieces; ++q)
        x[i][q] = in ? *reinterpret_cast<const mm_u4*>(xr + q * a.x.plane + at) : mm_u4{};
      if constexpr (!kSplit) {
        w[i][0] = in ? *reinterpret_cast<const mm_u4*>(static_cast<const unsigned short*>(wr) + at) : mm_u4{};
      } else {
        const float* const p = static_cast<const float*>(wr) + at;
        if (at + 8 <= a.D) {
          __builtin_memcpy(w[i], p, 32);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[i][e / 4][e % 4] = at + e < a.D ? __float_as_uint(p[e]) : 0u;
        }
      }
    }
  }
  __device__ __forceinline__ f16v product(f16v acc) const {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if constexpr (!kSplit) {
        acc = mm_mfma<F == kElemF16>(w[i][0], x[i][0], acc);
      } else {
        float f[8];
        mm_u4 v[3];
        __builtin_memcpy(f, w[i], 32);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          unsigned short h[8];
          down_all<kElemBf16, 8>(f, h);
          __builtin_memcpy(&v[q], h, 16);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] -= Elem<kElemBf16>::up(h[e]);
        }
        acc = mm_mfma<false>(v[0], x[i][2], acc);
        acc = mm_mfma<false>(v[2], x[i][0], acc);
        acc = mm_mfma<false>(v[1], x[i][1], acc);
        acc = mm_mfma<false>(v[0], x[i][1], acc);
        acc = mm_mfma<false>(v[1], x[i][0], acc);
        acc = mm_mfma<false>(v[0], x[i][0], acc);
      }
    }
    return acc;
  }
};
// R: 0 for the statistics; otherwise the backward's logits, of which it leaves dl as [token][R] in fp32.
template <int F, int R>
__global__ __launch_bounds__(256) void xent_few_kernel(LogitArgs a) {
  constexpr int kChunk = 16 * FewChunk<F>::kSteps;
  constexpr size_t kBytes = F == kElemF32 ? 4 : 2;
  __shared__ float sm[4][16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, n = blockIdx.y * 32 + col, half = lane >> 5;
  const int groups = (a.V + 31) / 32, width = a.x.k;
  const int target = n < a.N ? a.target[n] - a.v_first : -1;
  const float4 row = R > 0 && n < a.N ? a.rows[n] : float4{0.f, 0.f, 0.f, 0.f};
  const unsigned short* const xr = a.x.p + min(n, a.N - 1) * a.x.ld;
  auto load = [&](int group, int k, FewChunk<F>& c) {
    const char* const wr = reinterpret_cast<const char*>(a.w.p) + min(group * 32 + col, a.V - 1) * a.w.ld * kBytes;
    c.load(a, xr, wr, k + 8 * half);
  };
  float m = neg_inf(), sum = 0.f;
  FewChunk<F> now, next;
  load(blockIdx.x, wave * kChunk, now);
  for (int group = blockIdx.x; group < groups; group += gridDim.x) {
    f16v acc{};
    for (int k = wave * kChunk; k < width; k += 4 * kChunk) {
      const bool last = k + 4 * kChunk >= width;
      const int to = last ? group + (int)gridDim.x : group;
      if (to < groups) load(to, last ? wave * kChunk : k + 4 * kChunk, next);
      acc = now.product(acc);
      now = next;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) sm[wave][r][lane] = acc[r];
    __syncthreads();
    float l[4], big = m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int reg = 4 * wave + r, v = group * 32 + 8 * wave + 4 * half + r;
      l[r] = (sm[0][reg][lane] + sm[1][reg][lane]) + (sm[2][reg][lane] + sm[3][reg][lane]) + a.bias[v];
      if constexpr (R == 0) {
        if (v == target) a.own[n] = l[r];
        big = fmaxf(big, l[r]);
      } else {
        float d = exp_from(l[r], row.x) * row.y;
        d = row.z == 0.f || l[r] == neg_inf() ? 0.f : d;
        if (v == target) d -= __float_as_int(row.w) < 0 ? 0.f : row.z;
        if (n < R && v < a.V) a.dl_rows[(size_t)v * R + n] = d;
      }
    }
    if constexpr (R == 0) {
      const float ref = big == neg_inf() ? 0.f : big;
      sum *= exp_from(m, ref);  // (0 for the first m, -inf)
      m = big;
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += exp_from(l[r], ref);
    }
    __syncthreads();
  }
  if constexpr (R > 0) return;
  join(m, sum, __shfl_xor(m, 32), __shfl_xor(sum, 32));
  sm[wave][0][lane] = m;
  sm[wave][1][lane] = sum;
  __syncthreads();
  if (wave || half || n >= a.N) return;
#pragma unroll
  for (int k = 1; k < 4; ++k) join(m, sum, sm[k][0][lane], sm[k][1][lane]);
  a.part[(size_t)blockIdx.x * a.N + n] = float2{m, sum};
}

// dx and dw of few fp32 rows from dl [V][R], which is uniform: a thread has 4 columns (2 at 32 rows) of all rows
// of x and of its sums for dx in registers, and takes a range of the tokens' rows of w, whose dw it leaves.
// Bound by reading w and writing dw: 204 us at 5 rows and 131072 tokens of width 1024 (1.07 GB, 5.3 TB/s).  The
// pass takes 683 us there, 844 at 16 rows and 1017 at 32, on tiles, for which all of w's pieces are made, 1563;
// at 64 rows with a column a thread 1846, so that up to 32 go this way.
// dx: planes [range][N][D]; dw, dx: may be null.
struct FewOutArgs {
  const float *w, *x, *dl;
  const float4* rows;
  long long ldw, ldx;
  float *dw, *dx;
  int V, N, D, per, add;  // per: tokens of a range
};
template <int R>
__global__ __launch_bounds__(256) void xent_few_out_kernel(FewOutArgs a) {
  constexpr int E = R <= 16 ? 4 : 2;
  typedef const __attribute__((address_space(4))) float Uniform;  // for scalar loads; nothing is stored there

  const int own = (blockIdx.x * 256 + threadIdx.x) * E;
  if (own >= a.D) return;
  const int d = min(own, a.D - E);  // the last columns, beside the neighbour's: both store the same of dw
  const int v0 = blockIdx.y * a.per, v1 = min(a.V, v0 + a.per);
  float x[R][E], acc[R][E];
#pragma unroll
  for (int n = 0; n < R; ++n)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[n][e] = n < a.N && a.rows[n].z != 0.f ? a.x[n * a.ldx + d + e] : 0.f;
      acc[n][e] = 0.f;
    }
  constexpr int kAhead = 4;
  Pack<kElemF32, E> w[kAhead];
  auto load = [&](int v) { return load_pack<kElemF32, E>(a.w + min(v, a.V - 1) * a.ldw + d); };
#pragma unroll
  for (int k = 0; k < kAhead; ++k) w[k] = load(v0 + k);
  for (int v = v0; v < v1; v += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (v + k >= v1) break;
      Uniform* const g = (Uniform*)(unsigned long long)(a.dl + (size_t)(v + k) * R);
      Pack<kElemF32, E> o;
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] = 0.f;
#pragma unroll
      for (int n = 0; n < R; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          acc[n][e] = __builtin_fmaf(g[n], w[k].v[e], acc[n][e]);
          o.v[e] = __builtin_fmaf(g[n], x[n][e], o.v[e]);
        }
      w[k] = load(v + k + kAhead);
      if (a.dw) __builtin_memcpy(a.dw + (size_t)(v + k) * a.D + d, &o, sizeof(o));
    }
  }
  if (!a.dx) return;
  float* const to = a.dx + (size_t)blockIdx.y * a.N * a.D + d;
#pragma unroll
  for (int n = 0; n < R; ++n) {
    if (n >= a.N) continue;  // (a break would have the compiler keep the loop, and the sums in memory)
    float* const row = to + (size_t)n * a.D;
    if (d == own) {
      Pack<kElemF32, E> o{};
      if (a.add) o = load_pack<kElemF32, E>(row);
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] += acc[n][e];
      __builtin_memcpy(row, &o, sizeof(o));
    } else {  // a sum that is added to has one owner
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (d + e >= own) row[e] = (a.add ? row[e] : 0.f) + acc[n][e];
    }
  }
}
template <int R>
__global__ __launch_bounds__(256) void xent_few_bias_kernel(const float* __restrict__ dl, float* dbias, int V) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= V) return;
  double s = 0.0;
#pragma unroll
  for (int n = 0; n < R; ++n) s += dl[(size_t)v * R + n];
  dbias[v] = (float)s;
}

// Targets as 32-bit numbers (-1: not scored, -2: beyond the vocabulary), and the bias, up to whole tiles.
__global__ __launch_bounds__(256) void xent_prepare_kernel(const void* targets, int tgt64, const float* bias,
                                                          int* target, float* bias_out, int N, int V) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < (N + kMmTile - 1) / kMmTile * kMmTile) {
    const long long t = i < N ? load_id(targets, tgt64, i) : -1;
    target[i] = t < 0 ? -1 : t >= V ? -2 : (int)t;
  }
  if (i < (V + kMmTile - 1) / kMmTile * kMmTile) bias_out[i] = i >= V ? neg_inf() : bias ? bias[i] : 0.f;
}

// The loss and the row's (m, sum exp(l - m)) from its parts: 8 positions by 32 strips of them.
__global__ __launch_bounds__(256) void xent_join_kernel(const float2* __restrict__ part, const float* __restrict__ own,
                                                        const int* __restrict__ target, float* loss, float2* stats,
                                                        unsigned* err, int N, int parts) {
  __shared__ float2 sm[4][8];
  const int c = threadIdx.x & 7, strip = threadIdx.x >> 3, n = blockIdx.x * 8 + c;
  float m = neg_inf(), s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int t = strip; t < parts; t += 32) {
      const float2 p = part[(size_t)t * N + n];
      join(m, s, p.x, p.y);
    }
  }
#pragma unroll
  for (int k = 8; k < 64; k *= 2) join(m, s, __shfl_xor(m, k), __shfl_xor(s, k));
  if ((threadIdx.x & 63) < 8) sm[threadIdx.x >> 6][c] = float2{m, s};
  __syncthreads();
  if (strip || n >= N) return;
  for (int k = 1; k < 4; ++k) join(m, s, sm[k][c].x, sm[k][c].y);
  if (stats) stats[n] = float2{m, s};
  const bool masked = all_masked(m, s);
  const int t = target[n];
  float v = 0.f;
  if (t >= 0)
    v = masked ? __builtin_inff() : (m - own[n]) + logf(s);
  else if (t == -2) {
    v = __builtin_nanf("");
    atomicOr(err, kErrId);
  }
  loss[n] = v;
}


// Rows' gradients: none where the target is outside of the vocabulary or nothing but masks is in the row.  What such a
// row of x holds (padding that nothing has written, say) must not reach dw, neither NaN times 0 nor by the scale, and a
// masked token's weight sets no scale either.
struct RowGradients {
  const float2* stats;
  const int* target;
  const float* dloss;
  __device__ __forceinline__ float operator()(long long n) const {
    const float2 s = stats[n];
    const float g = dloss[n];  // (three loads at a time)
    return target[n] >= 0 && !all_masked(s.x, s.y) ? g : 0.f;
  }
};
// What the backward needs of each row: the largest logit, g / sum, g, and 2^(its exponent less the largest row's),
// negative where the target is masked.
__device__ __forceinline__ float4 row_of(float2 s, float g, int t, const float* bias, float part) {
  return float4{s.x, g * (1.f / s.y), g, t >= 0 && bias && bias[t] == neg_inf() ? -part : part};
}
// A row beyond the last one has no gradient, and its logits are the bias alone, whose exponential may be infinite: its
// reference has it computed with a test.
__device__ __forceinline__ float4 row_beyond() { return float4{__builtin_inff(), 0.f, 0.f, 0.f}; }
// 16-bit operands' scales.  The rows of a matrix among the threads of `blocks` workgroups: 1 << lg of them a row.
struct RowSplit {
  int lg, blocks;
  long long rows;
};
constexpr int kTopExp = 14;  // of the largest element of what is scaled
struct ScaleArgs {
  const unsigned short *x, *w;  // of width elements, a multiple of 8, at ldx and ldw
  long long ldx, ldw;
  int width;
  RowSplit rx, rw;              // rw: no workgroups for an fp16 w
  int blocks_g;                 // for the rows' gradients
  RowGradients g;
  const float* bias;
  unsigned* part;               // the workgroups' largest magnitudes
  int* exps;                    // [3]: exponents of the largest g, of x's scale and of w's
  unsigned short *hx, *hw;      // the scaled operands in fp16, dense
  float4* rows;
  int* row_exp;
  int N, twice;                 // twice: hx has x again behind it
  // Whether a row is multiplied by anything but 0: a position that has a gradient, a token that is not masked.
  __device__ __forceinline__ bool counts(bool is_x, long long row) const {
    return is_x ? g(row) != 0.f : !bias || bias[row] != neg_inf();
  }
};

__device__ __forceinline__ unsigned block_max(unsigned m) {
  __shared__ unsigned sm[4];
#pragma unroll
  for (int k = 1; k < 64; k *= 2) m = max(m, (unsigned)__shfl_xor((int)m, k));
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  return max(max(sm[0], sm[1]), max(sm[2], sm[3]));
}
__device__ __forceinline__ int exp_of(float v) { return (int)((__float_as_uint(v) >> 23) & 0xff) - 127; }
// f(row, vector) for the vectors of 8 elements of workgroup `block`'s rows, 4 rows at a time; there is no such
// row where it is -1.
template <class Fn>
__device__ __forceinline__ void for_rows(const RowSplit& r, int vecs, int block, Fn f) {
  const long long step = (long long)r.blocks * (256 >> r.lg);
  const int mine = threadIdx.x & ((1 << r.lg) - 1);
  for (long long row = (long long)block * (256 >> r.lg) + (threadIdx.x >> r.lg); row < r.rows; row += 4 * step)
    for (int c = mine; c < vecs; c += 1 << r.lg) {
      long long at[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) at[k] = row + k * step < r.rows ? row + k * step : -1;
      f(at, c);
    }
}

// The largest finite magnitudes, as bits: of elements in a workgroup's rows that count, or of rows' gradients in fp32.
template <bool FP16>
__global__ __launch_bounds__(256) void xent_max_kernel(ScaleArgs a) {
  constexpr unsigned kInf = FP16 ? 0x7c00 : 0x7f80;
  const int b = blockIdx.x;
  unsigned m = 0;
  if (b < a.rx.blocks + a.rw.blocks) {
    const bool is_x = b < a.rx.blocks;
    const unsigned short* const p = is_x ? a.x : a.w;
    const long long ld = is_x ? a.ldx : a.ldw;
    for_rows(is_x ? a.rx : a.rw, a.width / 8, is_x ? b : b - a.rx.blocks, [&](const long long(&row)[4], int c) {
      mm_u4 v[4];
      bool counts[4];  // (not a condition of the loads, which then would wait for it)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = row[k] < 0 ? mm_u4{} : *reinterpret_cast<const mm_u4*>(p + row[k] * ld + c * 8);
        counts[k] = row[k] >= 0 && a.counts(is_x, row[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned lo = v[k][e] & 0x7fff, hi = (v[k][e] >> 16) & 0x7fff;
          most = max(most, max(lo < kInf ? lo : 0, hi < kInf ? hi : 0));
        }
        m = max(m, counts[k] ? most : 0);
      }
    });
  } else {
    for (long long n = (b - a.rx.blocks - a.rw.blocks) * 256 + threadIdx.x; n < a.N; n += a.blocks_g * 256) {
      const unsigned g = __float_as_uint(a.g(n)) & 0x7fffffff;
      m = max(m, g < 0x7f800000 ? g : 0);
    }
  }
  m = block_max(m);
  if (threadIdx.x == 0) a.part[b] = m;
}

// The scaled operands, and the rows.
template <bool FP16>
__global__ __launch_bounds__(256) void xent_scaled_kernel(ScaleArgs a) {
  using E = Elem<FP16 ? kElemF16 : kElemBf16>;
  const int b = blockIdx.x;
  const bool is_x = b < a.rx.blocks, is_w = !is_x && b < a.rx.blocks + a.rw.blocks;
  const int first = is_x ? 0 : a.rx.blocks, count = is_x ? a.rx.blocks : a.rw.blocks;
  unsigned g = 0, m = 0;
  if (!is_w)
    for (int i = threadIdx.x; i < a.blocks_g; i += 256) g = max(g, a.part[a.rx.blocks + a.rw.blocks + i]);
  if (is_x || is_w)
    for (int i = threadIdx.x; i < count; i += 256) m = max(m, a.part[first + i]);
  g = block_max(g);
  __syncthreads();
  m = block_max(m);
  constexpr int kLeast = kTopExp - 126;  // 2^126 is the largest power of two that a row of small g is scaled by
  const int top = g ? max(kLeast, exp_of(__uint_as_float(g))) : 0;
  const int up = m ? kTopExp - exp_of(E::up((unsigned short)m)) : 0;
  auto exponent = [&](float g) {
    return g == 0.f || !(__builtin_fabsf(g) < __builtin_inff()) ? top : max(kLeast, exp_of(g));
  };
  if (is_x || is_w) {
    if (threadIdx.x == 0 && b == first) a.exps[is_x ? 1 : 2] = up;
    const unsigned short* const p = is_x ? a.x : a.w;
    unsigned short* const out = is_x ? a.hx : a.hw;
    const long long ld = is_x ? a.ldx : a.ldw;
    for_rows(is_x ? a.rx : a.rw, a.width / 8, b - first, [&](const long long(&row)[4], int c) {
      mm_u4 v[4];
      int e[4];
      bool counts[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (row[k] < 0) continue;
        v[k] = *reinterpret_cast<const mm_u4*>(p + row[k] * ld + c * 8);
        counts[k] = a.counts(is_x, row[k]);
        e[k] = up + (is_x ? exponent(a.g(row[k])) - top : 0);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (row[k] < 0) continue;
        if (!counts[k]) v[k] = mm_u4{};
        unsigned short h[8];
        __builtin_memcpy(h, &v[k], 16);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __builtin_ldexpf(E::up(h[i]), e[k]);
        down_all<kElemF16, 8>(f, h);
        __builtin_memcpy(&v[k], h, 16);
        *reinterpret_cast<mm_u4*>(out + row[k] * a.width + c * 8) = v[k];
        if (is_x && a.twice) *reinterpret_cast<mm_u4*>(out + (row[k] + a.N) * a.width + c * 8) = v[k];
      }
    });
    return;
  }
  const int blocks = gridDim.x - a.rx.blocks - a.rw.blocks, block = b - a.rx.blocks - a.rw.blocks;
  if (block == 0 && threadIdx.x == 0) {
    a.exps[0] = top;
    if (a.rw.blocks == 0) a.exps[2] = 0;
  }
  const int all = (a.N + kMmTile - 1) / kMmTile * kMmTile;
  for (int n = block * 256 + threadIdx.x; n < all; n += blocks * 256) {  // up to whole tiles
    if (n >= a.N) {
      a.rows[n] = row_beyond();
      continue;
    }
    const float g = a.g(n);
    const int e = exponent(g);
    a.rows[n] = row_of(a.g.stats[n], __builtin_ldexpf(g, kTopExp - e), a.g.target[n], a.bias,
                       __builtin_ldexpf(1.f, e - top));
    a.row_exp[n] = e;
  }
}

// The rows where nothing is scaled.
__global__ __launch_bounds__(256) void xent_rows_kernel(ScaleArgs a) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n < 3) a.exps[n] = n == 0 ? kTopExp : 0;
  if (n >= a.N) {  // up to whole tiles
    a.rows[n] = row_beyond();
    return;
  }
  a.rows[n] = row_of(a.g.stats[n], a.g(n), a.g.target[n], a.bias, 1.f);
  a.row_exp[n] = kTopExp;
}

// x twice, for a bf16 dl in two rows.  A workgroup a row.
__global__ __launch_bounds__(256) void xent_twice_kernel(ScaleArgs a) {
  const int n = blockIdx.x, row = n < a.N ? n : n - a.N;
  const unsigned short* const from = a.x + row * a.ldx;
  const bool there = a.g(row) != 0.f;
  for (int c = threadIdx.x * 8; c < a.width; c += 2048)
    *reinterpret_cast<mm_u4*>(a.hx + (size_t)n * a.width + c) =
        there ? *reinterpret_cast<const mm_u4*>(from + c) : mm_u4{};
}

// The three pieces of fp32 rows, in planes of rows of `width` with zeros behind `cols`.  ROWS: of x for the backward;
// its rows without a gradient lose what no piece holds (the rest stays: their logits must not exceed the forward's).
template <bool ROWS>
__global__ __launch_bounds__(256) void xent_split_kernel(const float* __restrict__ src, long long ld,
                                                         unsigned short* dst, RowSplit r, int cols, int width,
                                                         RowGradients g) {
  const size_t plane = (size_t)r.rows * width;
  for_rows(r, width / 8, blockIdx.x, [&](const long long(&row)[4], int c) {
    float f[4][8];
    bool none[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      none[k] = ROWS && row[k] >= 0 && g(row[k]) == 0.f;
      const float* const p = src + row[k] * ld + c * 8;
      if (row[k] >= 0 && c * 8 + 8 <= cols) {
        const Pack<kElemF32, 4> lo = load_pack<kElemF32, 4>(p), hi = load_pack<kElemF32, 4>(p + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[k][e] = e < 4 ? lo.v[e] : hi.v[e - 4];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[k][e] = row[k] >= 0 && c * 8 + e < cols ? p[e] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (row[k] < 0) continue;
      if (ROWS && none[k]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[k][e] = __builtin_fabsf(f[k][e]) < kPieceEnd ? f[k][e] : 0.f;
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        unsigned short h[8];
        down_all<kElemBf16, 8>(f[k], h);
        mm_u4 v;
        __builtin_memcpy(&v, h, 16);
        *reinterpret_cast<mm_u4*>(dst + q * plane + (size_t)row[k] * width + c * 8) = v;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[k][e] -= Elem<kElemBf16>::up(h[e]);
      }
    }
  });
}

// The tile's dl goes from the registers to memory: an exchange between the half-waves gives every lane 8
// neighbouring tokens of a position.  A lane's stores, 4 AF a part, are always issued, whatever lies outside, so
// that the next product's waits can leave them out.
// PARTS: how many numbers of the product's type a dl is kept in.
template <int F, int PARTS, int AF>
__global__ __launch_bounds__(kMmThreads) void xent_grad_kernel(LogitArgs a) {
  constexpr int kStores = 4 * AF * PARTS, kDl = PARTS > 1 && F != kElemF16 ? kElemBf16 : kElemF16;
  __shared__ __attribute__((aligned(1024))) char lds[mm_lds(AF)];
  __shared__ __attribute__((aligned(1024))) TileInfo info[2];
  __shared__ float sums[4][64 * AF];
  constexpr int kTokens = 64 * AF;
  const long long ld = (long long)a.tiles_v * kTokens;
  MmPipe<F == kElemF16, false, false, F == kElemF32, AF> mm;
  LogitWalk<AF> walk(a);
  walk.info(&info[0], __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  mm.begin(lds, walk.w(), walk.x(), a.D);
  bool first = true;
  for (int par = 0; walk.there(); par ^= 1, first = false) {
    const int tv = walk.tv, tn = walk.tn;
    walk.next();
    MmAccOf<AF> acc;
    mm.template run<kStores>(acc, walk.w(), walk.x(), !first, [&] { walk.info(&info[par ^ 1], mm.wave); });
    const LogitPlace<AF> q(tv, tn);
    add_bias(q, info[par].bias, acc);
    auto out_of = [&](int part) {
      unsigned short* const p = a.dl + ((long long)part * a.N + tn * kMmTile) * ld + tv * kTokens;
      return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, 0x7fffffff, 0x00020000);
    };
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 row = info[par].rows[q.c + j * 32];
      const int own = info[par].target[q.c + j * 32] - a.v_first - q.v0;
      const float gi = row.y, ref = row.x;
      const float hot = __float_as_int(row.w) < 0 ? 0.f : row.z;
      const bool owns = __any((unsigned)own < 32u * AF);  // few waves have a target among their tokens
      // a masked logit has none whatever arrives, nor has a row without a gradient whatever it holds
      const bool plain =
          __all(__builtin_fabsf(gi) < __builtin_inff() && __builtin_fabsf(row.x) < __builtin_inff());
      // the lower half-wave takes the 8 tokens from 16 k on, the upper one those 8 further
      const unsigned off =
          q.n0 + j * 32 < a.N ? (unsigned)((q.c + j * 32) * ld + q.v + 8 * q.half) * 2 : kOffNone;
#pragma unroll
      for (int i = 0; i < AF; ++i) {
        __builtin_amdgcn_sched_barrier(0);  // 16 values at a time in registers beside the rest
        if (plain) {
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = exp_from(acc[i][j][r], ref) * gi;
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float d = exp_from(acc[i][j][r], ref) * gi;
            acc[i][j][r] = row.z == 0.f || acc[i][j][r] == neg_inf() ? 0.f : d;
          }
        }
        if (owns) {
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] -= own == i * 32 + 8 * (r >> 2) + (r & 3) ? hot : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mm_u4 v[PARTS];
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // 2 tokens of groups 2 k and 2 k + 1
            float f[4] = {acc[i][j][8 * k + 2 * e], acc[i][j][8 * k + 2 * e + 1], acc[i][j][8 * k + 4 + 2 * e],
                          acc[i][j][8 * k + 5 + 2 * e]};
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
              unsigned short h[4];
              unsigned lo, hi;
              down_all<kDl, 4>(f, h);
              __builtin_memcpy(&lo, h, 4);
              __builtin_memcpy(&hi, h + 2, 4);
              const auto x = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
              v[part][e] = x[0];
              v[part][2 + e] = x[1];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float top = Elem<kDl>::up(h[c]);
                f[c] = __builtin_fabsf(top) < __builtin_inff() ? f[c] - top : 0.f;
              }
            }
          }
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            __builtin_amdgcn_raw_buffer_store_b128(v[part], out_of(part), (int)off + (i * 32 + 16 * k) * 2, 0, 0);
        }
      }
    }
    if (a.dbias) {  // in fp32, from before the rounding
      float f[AF / 2][16];
      const float p0 = __builtin_fabsf(info[par].rows[q.c].w), p1 = __builtin_fabsf(info[par].rows[q.c + 32].w);
#pragma unroll
      for (int k = 0; k < 8 * AF; ++k) {
        const int u = 2 * k, i = u / 16, r = u % 16;
        f[k / 16][k % 16] = add16(acc[i][0][r] * p0 + acc[i][1][r] * p1, acc[i][0][r + 1] * p0 + acc[i][1][r + 1] * p1);
      }
#pragma unroll
      for (int k = 0; k < AF / 2; ++k) {
        const float v = sum_rows(f[k], q.lane);
        const int u = 2 * (16 * k + (q.lane & 15)) + ((q.lane >> 4) & 1), i = u / 16, r = u % 16;
        sums[q.wave & 3][q.v + i * 32 + 8 * (r >> 2) + 4 * q.half + (r & 3)] = v;
      }
      lds_barrier();
      const int c = threadIdx.x;
      if (c < kTokens)
        a.dbias[(size_t)tn * ld + tv * kTokens + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
    } else if (mm.slices == kMmStages) {
      lds_barrier();  // the next product copies over info[par] at once; a longer one has a barrier before it does
    }
  }
}

// dbias of a piece from its tiles' sums, in fp64: 32 tokens by 8 strips of the tiles.
__global__ __launch_bounds__(256) void xent_bias_kernel(const float* __restrict__ part, const int* exps, float* dbias,
                                                        int V, long long ld, int tiles) {
  __shared__ double sm[8][32];
  const int c = threadIdx.x & 31, strip = threadIdx.x >> 5, v = blockIdx.x * 32 + c;
  double s = 0.0;
  if (v < V)
    for (int t = strip; t < tiles; t += 8) s += part[t * ld + v];
  sm[strip][c] = s;
  __syncthreads();
  if (strip || v >= V) return;
  for (int k = 1; k < 8; ++k) s += sm[k][c];
  dbias[v] = (float)ldexp(s, exps[0] - kTopExp);
}

struct OutArgs {
  const unsigned short *dl, *w, *x;  // of the product's type
  long long ld, ldw, ldx;   // of dl (the piece's padded width), w and x
  long long plane_w;        // between w's pieces
  float *dx, *dw;           // planes [split][N][D] and [split][ld][D] (one: dw itself); dw null: straight to dw16
  unsigned short* dw16;
  const int* exps;
  int N, V, D, Dk;          // V: the piece's tokens; Dk: the width that x and w have in memory
  int tiles_n, tiles_d, tiles_v, splits_x, splits_w, k_x, k_w, add;
};

// One piece's share of dx = dl w (the first splits_x tiles_n tiles_d workgroups) and its dw = dl^T x.  A tile's
// rows are the width's, so that a lane has 4 neighbouring elements of a result's row in registers and, from an
// exchange between the half-waves, 8 of a 16-bit one.
template <int F, bool FP16>  // of the results, and whether the product's type is fp16
__global__ __launch_bounds__(kMmThreads) void xent_out_kernel(OutArgs a) {
  constexpr bool kSplit = F == kElemF32;
  __shared__ __attribute__((aligned(1024))) char lds[kMmLds];
  const int count_x = a.splits_x * a.tiles_n * a.tiles_d;
  const bool is_x = (int)blockIdx.x < count_x;
  int id = is_x ? blockIdx.x : blockIdx.x - count_x;
  {  // workgroups i and i + 8 share an XCD and its L2: each XCD has a contiguous range, whose tiles of the width take
     // the same dl (515 -> 502 us for a piece of 16384 tokens at 8192 rows of width 1024)
    const int even = (is_x ? count_x : (int)gridDim.x - count_x) & ~7;
    if (id < even) id = (id % 8) * (even / 8) + id / 8;
  }
  const int td = id % a.tiles_d;
  id /= a.tiles_d;
  const int tiles = is_x ? a.tiles_n : a.tiles_v, tm = id % tiles, split = id / tiles;
  MmAcc acc;
  const int dcols = a.Dk - td * kMmTile;
  if (is_x) {
    const int k0 = split * a.k_x, k1 = min((int)a.ld, k0 + a.k_x);
    const MmOperand A{a.w + k0 * a.ldw + td * kMmTile, a.ldw, dcols, min(a.V, k1) - k0, a.plane_w};
    const MmOperand B{a.dl + (long long)tm * kMmTile * a.ld + k0, a.ld, min(kMmTile, a.N - tm * kMmTile), k1 - k0,
                      a.N * a.ld};
    MmPipe<FP16, true, false, kSplit> mm;
    mm.begin(lds, A, B, k1 - k0);
    mm.template run<0>(acc, MmOperand{A.p, A.ld, 0, 0}, MmOperand{B.p, B.ld, 0, 0}, false, [] {});
  } else {
    const int k0 = split * a.k_w, k1 = min(a.N, k0 + a.k_w);
    const MmOperand A{a.x + k0 * a.ldx + td * kMmTile, a.ldx, dcols, k1 - k0, a.N * a.ldx};
    const MmOperand B{a.dl + k0 * a.ld + tm * kMmTile, a.ld, kMmTile, k1 - k0, a.N * a.ld};
    MmPipe<FP16, true, true, kSplit> mm;
    mm.begin(lds, A, B, k1 - k0);
    mm.template run<0>(acc, MmOperand{A.p, A.ld, 0, 0}, MmOperand{B.p, B.ld, 0, 0}, false, [] {});
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const int d0 = td * kMmTile + (wave >> 2) * 128, r0 = tm * kMmTile + (wave & 3) * 64 + (lane & 31);
  const int rows = is_x ? a.N : a.V;
  const int back = a.exps[0] - kTopExp - a.exps[1];
  float* const plane = is_x ? a.dx + (size_t)split * a.N * a.D : a.dw ? a.dw + (size_t)split * a.ld * a.D : nullptr;
  const bool add = is_x && a.add;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = r0 + j * 32;
    if (plane) {
      if (row >= rows) continue;
      float* const to = plane + (size_t)row * a.D;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d = d0 + i * 32 + 8 * q + 4 * half;
          float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          if (d + 4 <= a.D) {
            Pack<kElemF32, 4> w;
            if (add) {
              w = load_pack<kElemF32, 4>(to + d);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] += w.v[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) w.v[e] = v[e];
            __builtin_memcpy(to + d, &w, sizeof(w));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d + e < a.D) to[d + e] = add ? to[d + e] + v[e] : v[e];
          }
        }
    } else if constexpr (!kSplit) {
      unsigned short* const to = a.dw16 + (size_t)row * a.D;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mm_u4 v;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f[4] = {__builtin_ldexpf(acc[i][j][8 * k + 2 * e], back),
                                __builtin_ldexpf(acc[i][j][8 * k + 2 * e + 1], back),
                                __builtin_ldexpf(acc[i][j][8 * k + 4 + 2 * e], back),
                                __builtin_ldexpf(acc[i][j][8 * k + 5 + 2 * e], back)};
            unsigned short h[4];
            unsigned lo, hi;
            down_all<F, 4>(f, h);
            __builtin_memcpy(&lo, h, 4);
            __builtin_memcpy(&hi, h + 2, 4);
            const auto x = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
            v[e] = x[0];
            v[2 + e] = x[1];
          }
          const int d = d0 + i * 32 + 16 * k + 8 * half;
          if (row < rows && d + 8 <= a.D) {
            __builtin_memcpy(to + d, &v, 16);
          } else if (row < rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (d + e < a.D) to[d + e] = (unsigned short)(v[e / 2] >> (16 * (e % 2)));
          }
        }
    }
  }
}

// Rows of `cols` of the sum of the planes, in their order, without their scales (row_exp: those of the rows).
template <int F>
__global__ __launch_bounds__(256) void xent_planes_kernel(const float* __restrict__ planes, size_t plane, int splits,
                                                          const int* exps, const int* row_exp, void* out, RowSplit r,
                                                          int cols) {
  const long long step = (long long)r.blocks * (256 >> r.lg);
  for (long long row = (long long)blockIdx.x * (256 >> r.lg) + (threadIdx.x >> r.lg); row < r.rows; row += step) {
    const int back = row_exp ? row_exp[row] - kTopExp - exps[2] : exps[0] - kTopExp - exps[1];
    for (int c = threadIdx.x & ((1 << r.lg) - 1); c < cols; c += 1 << r.lg) {
      const size_t i = (size_t)row * cols + c;
      float v = planes[i];
      for (int s = 1; s < splits; ++s) v += planes[s * plane + i];
      static_cast<typename Elem<F>::T*>(out)[i] = Elem<F>::down(__builtin_ldexpf(v, back));
    }
  }
}

// The same of many planes of few rows, for which a thread an element is neither enough of them nor of the loads:
// 4 strips of the planes, 8 loads at a time (104 planes of 7 rows of 576: 5 us, 59 as above).
constexpr int kManyPlanes = 8;
template <int F>
__global__ __launch_bounds__(256) void xent_many_planes_kernel(const float* __restrict__ planes, size_t plane,
                                                               int splits, const int* exps, const int* row_exp,
                                                               void* out, size_t n, int cols) {
  __shared__ float sm[4][64];
  const int c = threadIdx.x & 63, strip = threadIdx.x >> 6;
  const size_t i = (size_t)blockIdx.x * 64 + c;
  float v = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int s = strip; s < splits; s += 4) v += planes[s * plane + i];
  }
  sm[strip][c] = v;
  __syncthreads();
  if (strip || i >= n) return;
  v = (sm[0][c] + sm[1][c]) + (sm[2][c] + sm[3][c]);
  const int back = row_exp ? row_exp[i / cols] - kTopExp - exps[2] : exps[0] - kTopExp - exps[1];
  static_cast<typename Elem<F>::T*>(out)[i] = Elem<F>::down(__builtin_ldexpf(v, back));
}

template <int F>
__global__ __launch_bounds__(256) void xent_zero_kernel(void* out, size_t n) {
  const size_t stride = (size_t)gridDim.x * 256;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride)
    static_cast<typename Elem<F>::T*>(out)[i] = typename Elem<F>::T{};
}

// Rows of 16-bit elements with zeros up to a width that is a multiple of 8.
__global__ __launch_bounds__(256) void xent_pack_kernel(const unsigned short* __restrict__ src, long long ld,
                                                        unsigned short* dst, long long rows, int cols, int width) {
  const size_t all = (size_t)rows * width, stride = (size_t)gridDim.x * 256;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += stride) {
    const size_t r = i / width;
    const int c = (int)(i - r * width);
    dst[i] = c < cols ? src[(long long)r * ld + c] : (unsigned short)0;
  }
}

// ---- host ---------------------------------------------------------------------------------

int up_to(long long n, int unit) { return (int)((n + unit - 1) / unit * unit); }
unsigned grid_of(size_t n) { return (unsigned)std::min<size_t>((n + 255) / 256, 1 << 16); }

RowSplit split_rows(long long rows, int units, int most) {
  RowSplit r{0, 0, rows};
  while (r.lg < 8 && (1 << r.lg) < units) ++r.lg;
  const int each = 256 >> r.lg;
  r.blocks = (int)std::min<long long>(most, (rows + each - 1) / each);
  return r;
}
constexpr int kScaleBlocks = 1024;  // for an operand

// When 256 CUs that take `nx` workgroups of length x and then `nw` of length w, in order, are done.
double rounds_time(double nx, double x, double nw, double w) {
  const double full = std::floor(nx / 256);
  double late = nx - 256 * full, time[2] = {full * x, (full + 1) * x}, cus[2] = {256 - late, late};
  if (late == 0) time[1] = time[0];
  if (nw > 256 * 64) {  // so many that their lengths do not tell
    time[0] += std::floor(nw / 256) * w;
    time[1] += std::floor(nw / 256) * w;
    nw -= 256 * std::floor(nw / 256);
  }
  double done = std::max(time[0], cus[1] > 0 ? time[1] : 0);
  while (nw > 0) {
    const int g = cus[1] == 0 || time[0] <= time[1] ? 0 : 1;
    nw -= cus[g];
    time[g] += w;
    done = std::max(done, time[g]);
  }
  return done;
}

struct XentPlan {
  int piece, pieces;  // tokens of a piece: a multiple of 256
  int tiles_n, tiles_d, tiles_v;
  int splits_x, splits_w, k_x, k_w;
};
XentPlan plan_xent(int N, int V, int D, int fmt) {
  XentPlan p;
  const bool split = fmt == kElemF32;
  const int all = up_to(V, kMmTile);
  long long room = std::min<long long>(kPieceWidth, kPieceBytes / (split ? 6 : 2) / std::max(1, N));
  if (split) room = std::min<long long>(room, kPieceBytes / 6 / up_to(D, 8));  // the weight's pieces are no larger
  const long long fit = std::max<long long>(1, room / kMmTile) * kMmTile;
  p.piece = (int)std::min<long long>(all, fit);
  p.pieces = (all + p.piece - 1) / p.piece;
  p.piece = up_to((all + p.pieces - 1) / p.pieces, kMmTile);
  p.pieces = (all + p.piece - 1) / p.piece;
  p.tiles_n = (N + kMmTile - 1) / kMmTile;
  p.tiles_d = (D + kMmTile - 1) / kMmTile;
  p.tiles_v = p.piece / kMmTile;
  // k of a workgroup: the two products' work in about 256 equal shares, or 384, 512 or 768 where those should end a
  // quarter sooner (2500 fp32 rows, 3100 tokens of width 1999: 264 of the first would take two rounds of the 256 CUs,
  // 448 smaller ones two of half the length, 1152 -> 1070 us for the pass; by less they lose, as the last workgroups
  // of a round run faster than a full chip's: 5227 bf16 rows, 53383 tokens of width 299 1120 -> 1215).  An fp32 k is
  // six, and a share's start and end cost about 400.
  const double total = (double)p.tiles_d * ((double)p.tiles_n * p.piece + (double)p.tiles_v * N);
  const int least = split ? 128 : 512, ends = split ? 64 : 400;
  double best = 0;
  for (int parts : {256, 384, 512, 768}) {
    const int share = std::max(least, (int)std::min(1e9, total / parts));
    auto share_out = [&](int k, int* splits, int* each) {
      *splits = std::max(1, (int)(((long long)k + share / 2) / share));
      *each = std::max(kMmSlice, up_to((k + *splits - 1) / *splits, kMmSlice));
      *splits = std::max(1, (k + *each - 1) / *each);
    };
    int sx, kx, sw, kw;
    share_out(p.piece, &sx, &kx);
    share_out(N, &sw, &kw);
    const double time = rounds_time((double)sx * p.tiles_n * p.tiles_d, kx + ends, (double)sw * p.tiles_v * p.tiles_d,
                                    kw + ends);
    if (parts > 256 && time > 0.75 * best) continue;
    best = time;
    p.splits_x = sx;
    p.k_x = kx;
    p.splits_w = sw;
    p.k_w = kw;
  }
  return p;
}

int few_blocks(int V) { return std::min(kFewBlocks, (V + 31) / 32); }
bool in_two(int N, int fmt) { return fmt == kElemF32 ? false : N <= (fmt == kElemBf16 ? kMmTile / 2 : 512); }

// Whether the backward runs on xent_few_kernel and xent_few_out_kernel.
bool takes_few_back(int N, int D, int fmt) { return fmt == kElemF32 && N <= 32 && D >= 4; }
// Whether the forward runs on xent_few_kernel.  Not where a backward on tiles follows: its logits are rounded in
// another order, and a probability of them against the other ones' sum would be off by as much (dbias of 12 fp16 rows:
// 3.3e-7, 2.1e-7 from the same ones).
bool takes_few(int N, int V, int D, int fmt, bool alone) {
  if (!alone) return takes_few_back(N, D, fmt);
  if (fmt == kElemF32) return N <= kFewRowsF32;
  const long long tiles = ((long long)V + 127) / 128, rounds = (tiles + 255) / 256;  // of 128 tokens, one column
  return N <= kFewRows || (N <= kFewRowsUnfilled && (D <= 256 || 5 * tiles < 4 * 256 * rounds));
}
// The backward of few fp32 rows: R of its rows of dl, the tokens it takes at a time, and their ranges.
struct FewPlan {
  int R, piece, columns, ranges, per;
};
FewPlan plan_few(int N, int V, int D) {
  FewPlan p;
  p.R = N <= 8 ? 8 : N <= 16 ? 16 : 32;
  const int each = p.R <= 16 ? 1024 : 512;  // columns of a workgroup
  p.piece = (int)std::min<long long>(V, kPieceBytes / 4 / p.R);
  p.columns = (D + each - 1) / each;
  p.ranges = std::max(1, std::min((p.piece + 31) / 32, 1024 / p.columns));
  p.per = (p.piece + p.ranges - 1) / p.ranges;
  return p;
}
// The tokens that the forward takes at a time.
int forward_piece(int N, int V, int D, int fmt) {
  return fmt == kElemF32 ? std::min(V, plan_xent(N, V, D, fmt).piece) : V;
}
// Fragments of 64 tokens of the logits' tiles, 2 where that takes less rounds of the 256 CUs: half a tile costs a
// little more than half (700 fp32 rows, 10007 tokens of width 650, 120 tiles: 105 -> 83 us).
int logit_frags(int N, int V) {
  const long long tiles = (long long)((N + kMmTile - 1) / kMmTile) * ((V + kMmTile - 1) / kMmTile);
  return 11 * ((2 * tiles + 255) / 256) < 20 * ((tiles + 255) / 256) ? 2 : 4;
}
// The parts that the forward's statistics of a row are joined from.
int forward_parts(int N, int V, int D, int fmt, bool alone) {
  const int tokens = 64 * logit_frags(N, forward_piece(N, V, D, fmt));
  return takes_few(N, V, D, fmt, alone) ? few_blocks(V) : (V + tokens - 1) / tokens;
}

int check_xent(const char* who, long long N, int V, int D, int fmt) {
  if (!elem_fmt_ok(fmt)) return fail(HSL_ERR_ARG, "%s: format %d is not 0 (bf16), 1 (fp16) or 2 (fp32)", who, fmt);
  if (N < 0 || V < 0 || D < 0) return fail(HSL_ERR_ARG, "%s: negative size (N=%lld V=%d D=%d)", who, N, V, D);
  if (V == 0 || D == 0) return fail(HSL_ERR_ARG, "%s: an empty projection (V=%d D=%d)", who, V, D);
  // a launch holds fewer than 2^32 threads (256 a row at most), and rows of a tile lie within 2^31 bytes
  if (N >= (1ll << 24) || V >= 0x7fffffff - 256 || D >= (1 << 20) ||
      ((N + 255) / 256) * (((long long)V + 255) / 256) >= (1ll << 22) ||
      ((N + 255) / 256 + ((long long)V + 255) / 256) * ((D + 255) / 256) >= (1ll << 22))
    return fail(HSL_ERR_UNSUPPORTED,
                "%s: N=%lld V=%d D=%d is beyond one launch (needs N < 2^24, D < 2^20 and fewer than 2^22 tiles of 256 "
                "x 256 of each product)",
                who, N, V, D);
  return HSL_OK;
}

int check_rows(const char* who, long long ldx, long long ldw, int D) {
  if (ldx < D || ldw < D || ldx >= (1ll << 31) || ldw >= (1ll << 31))
    return fail(HSL_ERR_ARG, "%s: row strides %lld and %lld, must be D=%d or more and below 2^31", who, ldx, ldw, D);
  return HSL_OK;
}

int check_begin(const char* who, const void* x, long long ldx, const void* w, long long ldw, int D, int fmt) {
  auto readable = [](const void* p, long long ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld < (1 << 21);
  };
  if (fmt != kElemF32 && D % 8 == 0 && (!readable(x, ldx) || !readable(w, ldw)))
    return fail(HSL_ERR_ARG,
                "%s: rows of D=%d must begin at multiples of 16 bytes, fewer than 2^21 elements apart (row strides "
                "%lld and %lld)",
                who, D, ldx, ldw);
  return HSL_OK;
}

// The pieces of a call's workspace.  base = nullptr: to find its size.
struct XentSpace {
  int* target;
  float* own;
  float2* part;
  float4* rows;
  unsigned* part_max;
  int *exps, *row_exp;
  unsigned short *own_x, *own_w;  // the operands as the tiles read them, where they are not that
  unsigned short *scaled_x, *scaled_w, *dl;
  float *bias, *dbias, *dx, *dw, *dl_rows;
  size_t bytes;
};

XentSpace xent_space(void* base, int N, int V, int D, int fmt, bool backward) {
  XentSpace s{};
  const bool two = backward && in_two(N, fmt), split = fmt == kElemF32;
  const XentPlan p = plan_xent(two ? 2 * N : N, V, D, fmt);
  const int width = up_to(D, 8);
  Carver c(base, 0);
  s.target = c.take<int>(up_to(N, kMmTile));
  s.bias = c.take<float>(up_to(V, kMmTile) + kMmTile / 2);  // a last tile of 128 has 256 copied
  if (split) {
    s.own_x = c.take<unsigned short>((size_t)3 * N * width);
    if (!(backward && takes_few_back(N, D, fmt)))
      s.own_w = c.take<unsigned short>((size_t)3 * std::min(V, p.piece) * width);
  } else if (D % 8) {
    s.own_x = c.take<unsigned short>((size_t)N * width);
    s.own_w = c.take<unsigned short>((size_t)V * width);
  }
  if (!backward) {
    s.own = c.take<float>(N);
    const int parts = std::max(forward_parts(N, V, D, fmt, true), forward_parts(N, V, D, fmt, false));
    s.part = c.take<float2>((size_t)N * parts);
    s.bytes = c.off;
    return s;
  }
  s.rows = c.take<float4>(up_to(N, kMmTile));
  if (takes_few_back(N, D, fmt)) {
    const FewPlan f = plan_few(N, V, D);
    s.exps = c.take<int>(3);
    s.row_exp = c.take<int>(N);
    s.dl_rows = c.take<float>((size_t)f.piece * f.R);
    s.dx = c.take<float>((size_t)f.ranges * N * D);
    s.bytes = c.off;
    return s;
  }
  s.part_max = c.take<unsigned>(3 * kScaleBlocks);
  s.exps = c.take<int>(3);
  s.row_exp = c.take<int>(N);
  const size_t rows = two ? 2 * N : N, parts = split ? 3 : 1;
  if (!split) s.scaled_x = c.take<unsigned short>(rows * width);
  if (fmt == kElemBf16 && !two) s.scaled_w = c.take<unsigned short>((size_t)V * width);
  s.dl = c.take<unsigned short>(parts * rows * p.piece);
  s.dbias = c.take<float>((size_t)p.tiles_n * p.piece);
  if (!split || p.splits_x > 1) s.dx = c.take<float>(p.splits_x * rows * D);
  if (p.splits_w > 1) s.dw = c.take<float>((size_t)p.splits_w * p.piece * D);
  s.bytes = c.off;
  return s;
}

// Operands as the tiles read them: rows of a multiple of 8 elements at 16-byte steps, of fp32 ones the pieces.
struct XentOperands {
  const void *x0, *w0;
  const unsigned short *x, *w;
  long long ldx, ldw, ldw0;
  int N, D, width, fmt;
  unsigned short* own_w;

  int init(const void* x_, long long ldx_, const void* w_, long long ldw_, const XentSpace& s, int N_, int V, int D_,
           int fmt_, const RowGradients& g, hipStream_t st) {
    x0 = x_;
    w0 = w_;
    ldw0 = ldw_;
    N = N_;
    D = D_;
    fmt = fmt_;
    width = up_to(D, 8);
    own_w = s.own_w;
    x = static_cast<const unsigned short*>(x_);
    w = static_cast<const unsigned short*>(w_);
    ldx = ldx_;
    ldw = ldw_;
    if (s.own_x) x = s.own_x;
    if (s.own_w) w = s.own_w;
    if (s.own_x) ldx = ldw = width;
    if (fmt == kElemF32) {
      split(static_cast<const float*>(x0), ldx_, s.own_x, N, g, st);
    } else if (D % 8) {
      hipLaunchKernelGGL(xent_pack_kernel, dim3(grid_of((size_t)N * width)), dim3(256), 0, st,
                         static_cast<const unsigned short*>(x0), ldx_, s.own_x, (long long)N, D, width);
      hipLaunchKernelGGL(xent_pack_kernel, dim3(grid_of((size_t)V * width)), dim3(256), 0, st,
                         static_cast<const unsigned short*>(w0), ldw_, s.own_w, (long long)V, D, width);
    }
    HSL_HIP(hipGetLastError());
    return HSL_OK;
  }
  void split(const float* src, long long ld, unsigned short* dst, int rows, const RowGradients& g,
             hipStream_t st) const {
    const RowSplit r = split_rows(rows, width / 8, 1 << 16);
    if (g.stats)
      hipLaunchKernelGGL(xent_split_kernel<true>, dim3(r.blocks), dim3(256), 0, st, src, ld, dst, r, D, width, g);
    else
      hipLaunchKernelGGL(xent_split_kernel<false>, dim3(r.blocks), dim3(256), 0, st, src, ld, dst, r, D, width, g);
  }
  // The v tokens from v0 on.
  MmOperand tokens(int v0, int v, hipStream_t st) const {
    if (fmt != kElemF32) return {w + v0 * ldw, ldw, v, width};
    split(static_cast<const float*>(w0) + v0 * ldw0, ldw0, own_w, v, RowGradients{}, st);
    return {own_w, ldw, v, width, (long long)v * width};
  }
  MmOperand positions() const { return {x, ldx, N, width, (long long)N * width}; }
};

}  // namespace
}  // namespace hsl

using namespace hsl;

extern "C" {

size_t hsl_xent_ws_bytes(long long N, int V, int D, int fmt, int backward) {
  if (check_xent("hsl_xent_ws_bytes", N, V, D, fmt) != HSL_OK || N == 0) return 0;
  return xent_space(nullptr, (int)N, V, D, fmt, backward != 0).bytes;
}

int hsl_xent_fwd(const void* x, long long ldx, const void* w, long long ldw, const float* bias, const void* targets,
                 int tgt64, float* loss, float* stats, void* ws, size_t ws_bytes, long long N, int V, int D, int fmt,
                 void* stream) {
  HSL_CHECK(check_xent("hsl_xent_fwd", N, V, D, fmt));
  if (N == 0) return HSL_OK;
  if (!targets || !loss || !x || !w) return fail(HSL_ERR_ARG, "hsl_xent_fwd: null pointer");
  HSL_CHECK(check_rows("hsl_xent_fwd", ldx, ldw, D));
  const int n = (int)N;
  XentSpace s = xent_space(ws, n, V, D, fmt, false);
  if (!ws || ws_bytes < s.bytes)
    return fail(HSL_ERR_ARG, "hsl_xent_fwd: workspace %zu bytes, need %zu", ws_bytes, s.bytes);
  HSL_CHECK(check_begin("hsl_xent_fwd", x, ldx, w, ldw, D, fmt));
  hipStream_t st = static_cast<hipStream_t>(stream);
  unsigned* err = nullptr;
  HSL_CHECK(device_error_word(&err));
  DeviceInfo info;
  HSL_CHECK(device_info(&info));
  hipLaunchKernelGGL(xent_prepare_kernel, dim3((std::max(n, V) + 255) / 256), dim3(256), 0, st, targets,
                     tgt64, bias, s.target, s.bias, n, V);
  XentOperands o;
  HSL_CHECK(o.init(x, ldx, w, ldw, s, n, V, D, fmt, RowGradients{}, st));
  LogitArgs a{};
  a.x = o.positions();
  a.target = s.target;
  a.N = n;
  a.D = D;
  a.tiles_n = (n + kMmTile - 1) / kMmTile;
  a.own = s.own;
  const bool few = takes_few(n, V, D, fmt, !stats);
  const int piece = few ? V : forward_piece(n, V, D, fmt), frags = logit_frags(n, piece);
  for (int v0 = 0; v0 < V; v0 += piece) {
    const int v = std::min(piece, V - v0);
    a.w = few && fmt == kElemF32 ? MmOperand{static_cast<const unsigned short*>(w), ldw, V, D} : o.tokens(v0, v, st);
    a.bias = s.bias + v0;
    a.v_first = v0;
    a.V = v;
    a.tiles_v = (v + 64 * frags - 1) / (64 * frags);
    a.part = s.part + (size_t)(v0 / (64 * frags)) * n;
    const dim3 grid(std::min(a.tiles_v * a.tiles_n, info.num_cus)), block(kMmThreads);
    HSL_CHECK(with_fmt(fmt, [&](auto F) {
      constexpr int kF = decltype(F)::value;
      if (few)
        hipLaunchKernelGGL((xent_few_kernel<kF, 0>), dim3(few_blocks(V), (n + 31) / 32), dim3(256), 0, st, a);
      else if (frags == 2)
        hipLaunchKernelGGL((xent_stats_kernel<kF, 2>), grid, block, 0, st, a);
      else
        hipLaunchKernelGGL((xent_stats_kernel<kF, 4>), grid, block, 0, st, a);
      return (int)HSL_OK;
    }));
  }
  hipLaunchKernelGGL(xent_join_kernel, dim3((n + 7) / 8), dim3(256), 0, st, s.part, s.own, s.target, loss,
                     reinterpret_cast<float2*>(stats), err, n, forward_parts(n, V, D, fmt, !stats));
  HSL_HIP(hipGetLastError());
  return HSL_OK;
}

int hsl_xent_bwd(const void* x, long long ldx, const void* w, long long ldw, const float* bias, const void* targets,
                 int tgt64, const float* stats, const float* dloss, void* dx, void* dw, float* dbias, void* ws,
                 size_t ws_bytes, long long N, int V, int D, int fmt, void* stream) {
  HSL_CHECK(check_xent("hsl_xent_bwd", N, V, D, fmt));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int n = (int)N;
  if (N > 0 && (!targets || !stats || !dloss || !x || !w))
    return fail(HSL_ERR_ARG, "hsl_xent_bwd: null pointer");
  if (N > 0) HSL_CHECK(check_rows("hsl_xent_bwd", ldx, ldw, D));
  const bool two = in_two(n, fmt);
  const XentPlan p = plan_xent(two ? 2 * n : n, V, D, fmt);
  XentSpace s = xent_space(ws, n, V, D, fmt, true);
  if (N > 0 && (!ws || ws_bytes < s.bytes))
    return fail(HSL_ERR_ARG, "hsl_xent_bwd: workspace %zu bytes, need %zu", ws_bytes, s.bytes);
  if (N > 0) HSL_CHECK(check_begin("hsl_xent_bwd", x, ldx, w, ldw, D, fmt));
  if (N == 0) {  // no position: the weights' gradients are zeros
    if (!dw && !dbias) return HSL_OK;
    const size_t count = (size_t)V * D;
    if (dw) {
      HSL_CHECK(with_fmt(fmt, [&](auto F) {
        hipLaunchKernelGGL((xent_zero_kernel<decltype(F)::value>), dim3(grid_of(count)), dim3(256), 0, st, dw, count);
        HSL_HIP(hipGetLastError());
        return (int)HSL_OK;
      }));
    }
    if (dbias) hipLaunchKernelGGL((xent_zero_kernel<kElemF32>), dim3(grid_of(V)), dim3(256), 0, st, dbias, (size_t)V);
    HSL_HIP(hipGetLastError());
    return HSL_OK;
  }
  hipLaunchKernelGGL(xent_prepare_kernel, dim3((std::max(n, V) + 255) / 256), dim3(256), 0, st, targets,
                     tgt64, bias, s.target, s.bias, n, V);
  HSL_HIP(hipGetLastError());
  DeviceInfo info;
  HSL_CHECK(device_info(&info));
  XentOperands o;
  const RowGradients rows{reinterpret_cast<const float2*>(stats), s.target, dloss};
  HSL_CHECK(o.init(x, ldx, w, ldw, s, n, V, D, fmt, rows, st));
  const bool split = fmt == kElemF32;
  ScaleArgs sc{};
  sc.x = o.x;
  sc.w = o.w;
  sc.ldx = o.ldx;
  sc.ldw = o.ldw;
  sc.width = o.width;
  sc.rx = split_rows(n, o.width / 8, kScaleBlocks);
  if (fmt == kElemBf16) sc.rw = split_rows(V, o.width / 8, kScaleBlocks);
  sc.blocks_g = std::min(kScaleBlocks, (n + 1023) / 1024);
  sc.g = rows;
  sc.bias = bias;
  sc.part = s.part_max;
  sc.exps = s.exps;
  sc.hx = s.scaled_x;
  sc.hw = s.scaled_w;
  sc.rows = s.rows;
  sc.row_exp = s.row_exp;
  sc.N = n;
  sc.twice = two;
  const int scaled = sc.rx.blocks + sc.rw.blocks, row_blocks = (n + 255) / 256;
  if (split || (two && fmt == kElemBf16)) {
    hipLaunchKernelGGL(xent_rows_kernel, dim3(row_blocks), dim3(256), 0, st, sc);
    if (two) hipLaunchKernelGGL(xent_twice_kernel, dim3(2 * n), dim3(256), 0, st, sc);
  } else if (fmt == kElemF16) {
    hipLaunchKernelGGL(xent_max_kernel<true>, dim3(scaled + sc.blocks_g), dim3(256), 0, st, sc);
    hipLaunchKernelGGL(xent_scaled_kernel<true>, dim3(scaled + std::min(kScaleBlocks, row_blocks)), dim3(256), 0, st,
                       sc);
  } else {
    hipLaunchKernelGGL(xent_max_kernel<false>, dim3(scaled + sc.blocks_g), dim3(256), 0, st, sc);
    hipLaunchKernelGGL(xent_scaled_kernel<false>, dim3(scaled + std::min(kScaleBlocks, row_blocks)), dim3(256), 0, st,
                       sc);
  }
  HSL_HIP(hipGetLastError());
  auto sum_planes = [&](const float* planes, size_t plane, int count, const int* row_exp, void* out, long long rows) {
    HSL_CHECK(with_fmt(fmt, [&](auto F) {
      constexpr int kF = decltype(F)::value;
      const RowSplit r = split_rows(rows, D, 1 << 16);
      if (count < kManyPlanes)
        hipLaunchKernelGGL(xent_planes_kernel<kF>, dim3(r.blocks), dim3(256), 0, st, planes, plane, count, s.exps,
                           row_exp, out, r, D);
      else
        hipLaunchKernelGGL(xent_many_planes_kernel<kF>, dim3((unsigned)(((size_t)rows * D + 63) / 64)), dim3(256), 0,
                           st, planes, plane, count, s.exps, row_exp, out, (size_t)rows * D, D);
      HSL_HIP(hipGetLastError());
      return (int)HSL_OK;
    }));
    return (int)HSL_OK;
  };
  if (s.dl_rows) {  // few fp32 rows
    const FewPlan f = plan_few(n, V, D);
    for (int v0 = 0; v0 < V; v0 += f.piece) {
      const int v = std::min(f.piece, V - v0);
      const float* const wp = static_cast<const float*>(w) + v0 * ldw;
      LogitArgs a{};
      a.w = {reinterpret_cast<const unsigned short*>(wp), ldw, v, D};
      a.x = o.positions();
      a.bias = s.bias + v0;
      a.target = s.target;
      a.v_first = v0;
      a.V = v;
      a.N = n;
      a.D = D;
      a.rows = s.rows;
      a.dl_rows = s.dl_rows;
      FewOutArgs g{};
      g.w = wp;
      g.x = static_cast<const float*>(x);
      g.dl = s.dl_rows;
      g.rows = s.rows;
      g.ldw = ldw;
      g.ldx = ldx;
      g.dw = dw ? static_cast<float*>(dw) + (size_t)v0 * D : nullptr;
      g.dx = dx ? s.dx : nullptr;
      g.V = v;
      g.N = n;
      g.D = D;
      g.per = f.per;
      g.add = v0 > 0;
      auto run = [&](auto RR) {
        constexpr int kR = decltype(RR)::value;
        hipLaunchKernelGGL((xent_few_kernel<kElemF32, kR>), dim3(few_blocks(v)), dim3(256), 0, st, a);
        if (dw || dx)
          hipLaunchKernelGGL(xent_few_out_kernel<kR>, dim3(f.columns, f.ranges), dim3(256), 0, st, g);
        if (dbias)
          hipLaunchKernelGGL(xent_few_bias_kernel<kR>, dim3((v + 255) / 256), dim3(256), 0, st, s.dl_rows, dbias + v0,
                             v);
      };
      if (f.R == 8)
        run(std::integral_constant<int, 8>{});
      else if (f.R == 16)
        run(std::integral_constant<int, 16>{});
      else
        run(std::integral_constant<int, 32>{});
      HSL_HIP(hipGetLastError());
    }
    if (dx) HSL_CHECK(sum_planes(s.dx, (size_t)n * D, f.ranges, s.row_exp, dx, n));
    return HSL_OK;
  }
  float* const planes_x = s.dx ? s.dx : static_cast<float*>(dx);  // fp32: one plane is dx itself
  const int frags = logit_frags(n, std::min(V, p.piece));
  for (int v0 = 0; v0 < V; v0 += p.piece) {
    const int v = std::min(p.piece, V - v0);
    const int tiles_v = (v + kMmTile - 1) / kMmTile;  // the last piece may have fewer
    LogitArgs a{};
    a.w = o.tokens(v0, v, st);
    a.x = o.positions();
    a.bias = s.bias + v0;
    a.target = s.target;
    a.v_first = v0;
    a.V = v;
    a.N = n;
    a.D = D;
    a.tiles_v = tiles_v * (4 / frags);  // dl and dbias to whole tiles of 256
    a.tiles_n = (n + kMmTile - 1) / kMmTile;
    a.rows = s.rows;
    a.dl = s.dl;
    a.dbias = dbias ? s.dbias : nullptr;
    OutArgs g{};
    g.dl = a.dl;
    g.w = s.scaled_w ? s.scaled_w + (size_t)v0 * o.width : a.w.p;
    g.x = split ? o.x : s.scaled_x;
    g.ld = (long long)tiles_v * kMmTile;
    g.ldw = s.scaled_w ? o.width : a.w.ld;
    g.ldx = o.width;
    g.plane_w = a.w.plane;
    g.dx = planes_x;
    g.dw = p.splits_w > 1 ? s.dw : split && dw ? static_cast<float*>(dw) + (size_t)v0 * D : nullptr;
    g.dw16 = static_cast<unsigned short*>(dw) + (size_t)v0 * D;
    g.exps = s.exps;
    g.N = two ? 2 * n : n;
    g.V = v;
    g.D = D;
    g.Dk = o.width;
    g.tiles_n = p.tiles_n;
    g.tiles_d = p.tiles_d;
    g.tiles_v = tiles_v;
    g.splits_x = dx ? p.splits_x : 0;
    g.splits_w = dw ? p.splits_w : 0;
    g.k_x = p.k_x;
    g.k_w = p.k_w;
    g.add = v0 > 0;
    const dim3 grid(std::min(a.tiles_v * a.tiles_n, info.num_cus)), block(kMmThreads);
    const dim3 grid_out((g.splits_x * g.tiles_n + g.splits_w * tiles_v) * g.tiles_d);
    auto run = [&](auto F, auto PARTS, auto FP16) {
      constexpr int kF = decltype(F)::value, kParts = decltype(PARTS)::value;
      if (frags == 2)
        hipLaunchKernelGGL((xent_grad_kernel<kF, kParts, 2>), grid, block, 0, st, a);
      else
        hipLaunchKernelGGL((xent_grad_kernel<kF, kParts, 4>), grid, block, 0, st, a);
      if (grid_out.x)
        hipLaunchKernelGGL((xent_out_kernel<kF, decltype(FP16)::value>), grid_out, block, 0, st, g);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Bf16 = std::integral_constant<int, kElemBf16>;
    using F16 = std::integral_constant<int, kElemF16>;
    if (split)
      run(std::integral_constant<int, kElemF32>{}, std::integral_constant<int, 3>{}, std::false_type{});
    else if (fmt == kElemF16 && two)
      run(F16{}, Two{}, std::true_type{});
    else if (fmt == kElemF16)
      run(F16{}, One{}, std::true_type{});
    else if (two)
      run(Bf16{}, Two{}, std::false_type{});
    else
      run(Bf16{}, One{}, std::true_type{});
    if (dbias)
      hipLaunchKernelGGL(xent_bias_kernel, dim3((v + 31) / 32), dim3(256), 0, st, s.dbias, s.exps, dbias + v0, v, g.ld,
                         a.tiles_n);
    HSL_HIP(hipGetLastError());
    if (dw && p.splits_w > 1) {
      void* const out = split ? static_cast<void*>(static_cast<float*>(dw) + (size_t)v0 * D) : g.dw16;
      HSL_CHECK(sum_planes(s.dw, (size_t)g.ld * D, p.splits_w, nullptr, out, v));
    }
  }
  if (dx && s.dx) HSL_CHECK(sum_planes(s.dx, (size_t)n * D, two ? 2 * p.splits_x : p.splits_x, s.row_exp, dx, n));
  return HSL_OK;
}

}  // extern "C"
