// Orthogonalised updates: X <- aX + (b XX' + c (XX')^2) X, some steps from
// X = U / (|U|_F + eps), for many matrices at once, each with a short side r (an
// adapter's rank) and a long side K.
//
// With G_k = X_k X_k' on the short side and Q_k = aI + b G_k + c G_k^2,
//   X_n = P_n U,  P_0 = I / (|U|_F + eps),  P_{k+1} = Q_k P_k,  G_{k+1} = Q_k G_k Q_k,
// so the long side is walked twice, once for G_0 and once for P_n U, whatever the
// number of steps; in between stand r x r matrices alone.
//
// Everything between the loads and the stores is in 64 bits, on the matrix cores
// (v_mfma_f64_16x16x4: 77 TFLOP/s measured and dependent ones 27 ns apart with the sums
// in vector registers, 26 and 81 in the accumulation ones).  In 32 bits
// G loses the squares of singular values below 2^-12 of the largest, and the steps
// then multiply what was lost by a^2 each.  64 bits bound the steps too: an error of
// 2^-53 grows by a^2 a step, so |a|^(2 steps) may reach 1e13 (12 steps at a = 3.4445).
//
// The instruction takes A[i][k] from lane i + 16 k, B[k][j] from lane j + 16 k and
// gives D[4 v + q][j] in register v of lane j + 16 q.  The r x r matrices are
// symmetric, so a tile read as B[k][j] is at once the operand A of its transpose:
// rows of 16 doubles, no bank conflicts, no transposition anywhere.  For that G stays
// symmetric to the bit: its upper half is written to both places.  (What rounding
// leaves between G and its transpose grows by a^2 a step as well: without this, 7 steps
// are off by 5e-12 and 12 by 6e-7 of the largest entry, with it by 3e-15.)
#include <cmath>
#include <type_traits>

#include "common.h"

namespace {

typedef double d4 __attribute__((ext_vector_type(4)));
typedef double d2 __attribute__((ext_vector_type(2)));
constexpr int NTH = 256;
constexpr int MAXE = 44;        // entries of a launch's table (kernel arguments: 4 KB)
constexpr int64_t MAXR = 1024;  // short side

// A batch of equal matrices, back to back.
struct Entry {
  const void* x;
  void* out;
  int64_t part, poly;      // its first matrix's place in the two scratch areas (doubles)
  int32_t K, r;            // long and short side
  int32_t CH, chunks;      // long elements of a workgroup in gram, and its workgroups
                           // (of matrices done whole CH is their number)
  int32_t AL;              // long elements of a workgroup in apply (all three: r <= 32)
  int16_t tall;            // the short side is the contiguous one
  int16_t vec;             // rows may be read four elements at a time
};
enum { IN_GRAM, IN_SUM, IN_NORM, IN_POLY, IN_APPLY, PHASES };
// Equal shares of all units of a phase, one behind the other, for `wgs` workgroups: the
// first `rem` take q + 1 units, the others q.
struct Shares {
  uint32_t wgs, q, rem;
  __host__ __device__ uint32_t begin(uint32_t b) const { return b * q + (b < rem ? b : rem); }
  __host__ __device__ uint32_t owner(uint32_t u) const {
    return u < rem * (q + 1) ? u / (q + 1) : rem + (u - rem * (q + 1)) / q;
  }
};
struct Table {
  Entry e[MAXE];
  uint32_t tile0[PHASES][64];  // the entries' first workgroups (units) in a phase, then ~0
  Shares gram, apply;          // r > 32
  int32_t n, steps;
  double a, b, c, eps;
};
static_assert(sizeof(Table) <= 3840 && sizeof(Table) % 4 == 0, "kernel arguments");

// Kernel arguments lie in the host's memory: gram, the first launch, copies the table
// beside the sums, where the others find it in a third of the time.

// The last entry with tile0 <= b and its place among the entry's workgroups: one
// load for all entries (a search would be six dependent ones, 1 us of each
// workgroup's time).
__device__ __forceinline__ const Entry& find(const Table& t, int phase, uint32_t b, uint32_t& w) {
  const uint32_t mine = t.tile0[phase][threadIdx.x & 63];
  const int i = __popcll(__ballot(mine <= b)) - 1;
  w = b - __builtin_amdgcn_readlane(mine, i);
  return t.e[i];
}
// The workgroup's number among all, counted XCD by XCD: neighbours, which read the same
// matrix, share an L2.
__device__ __forceinline__ uint32_t neighbours() {
  const uint32_t x = blockIdx.x % 8, each = gridDim.x / 8, rem = gridDim.x % 8;
  return x * each + min(x, rem) + blockIdx.x / 8;
}
// The long side of short sides beyond 32 goes in units of this many elements, of which a
// workgroup takes an equal share; it may end inside one matrix and begin inside another.
constexpr int UNIT = 128;
__host__ __device__ inline uint32_t units_of(const Entry& e, int unit) {
  return (uint32_t)(e.K + unit - 1) / unit;
}
// In gram the pairs of a block with itself come first, whose ten tiles of sixteen make
// a unit of 192 elements cost as much (28 factors of rank 128: with units of 128 for both
// 78 us, so 69).
constexpr int SELF = 192;
struct Pairs {
  uint32_t nb, self, other, each;  // blocks, units of either kind of pair, of a matrix
  __host__ __device__ explicit Pairs(const Entry& e)
      : nb((uint32_t)(e.r + 63) / 64), self(units_of(e, SELF)), other(units_of(e, UNIT)),
        each(nb * self + nb * (nb - 1) / 2 * other) {}
  __host__ __device__ uint32_t many() const { return nb * (nb + 1) / 2; }
  // pair p's first unit in its matrix
  __host__ __device__ uint32_t begin(uint32_t p) const {
    return p < nb ? p * self : nb * self + (p - nb) * other;
  }
  // pair p's blocks
  __device__ void blocks(uint32_t p, int& I, int& J) const {
    I = J = (int)p;
    if (p < nb) return;
    I = 0, J = (int)(p - nb);  // (0,1..nb-1), (1,2..nb-1), ...
    while (J >= (int)nb - 1 - I) J -= (int)nb - 1 - I, ++I;
    J += I + 1;
  }
};

// Pointers that were read from memory, said to be ones to device memory: otherwise
// their loads are flat ones, which are counted as LDS reads too and waited for with them.
#define GLOBAL(T) __attribute__((address_space(1))) T
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <bool BF>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (BF)
    return st::bf16_to_f32(((const GLOBAL(uint16_t)*)p)[i]);
  else
    return ((const GLOBAL(float)*)p)[i];
}
template <bool BF>
__device__ __forceinline__ void load4(const void* p, int64_t i, float* f) {
  if constexpr (BF) {
    const u32x2 w = *(const GLOBAL(u32x2)*)((const uint16_t*)p + i);
    f[0] = __uint_as_float(w.x << 16), f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16), f[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const f32x4 w = *(const GLOBAL(f32x4)*)((const float*)p + i);
    f[0] = w.x, f[1] = w.y, f[2] = w.z, f[3] = w.w;
  }
}
// four elements from i on, the first `n` of them inside (n may be 0 or less)
template <bool BF>
__device__ __forceinline__ void load_upto4(const void* p, int64_t i, int n, bool vec, float* f) {
  if (vec && n >= 4) {
    load4<BF>(p, i, f);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = e < n ? load1<BF>(p, i + e) : 0.0f;
}
template <bool BF>
__device__ __forceinline__ void store4(void* p, int64_t i, const float* f) {
  if constexpr (BF)
    *(GLOBAL(u32x2)*)((uint16_t*)p + i) =
        u32x2{st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3])};
  else
    *(GLOBAL(f32x4)*)((float*)p + i) = f32x4{f[0], f[1], f[2], f[3]};
}
template <bool BF>
__device__ __forceinline__ void store_upto4(void* p, int64_t i, int n, bool vec, const float* f) {
  if (vec && n >= 4) {
    store4<BF>(p, i, f);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) {
      if constexpr (BF)
        ((GLOBAL(uint16_t)*)p)[i + e] = st::f32_to_bf16(f[e]);
      else
        ((GLOBAL(float)*)p)[i + e] = f[e];
    }
}

// ---------------------------------------------------------------- G = U U'
// One workgroup: a chunk of the long side and one block pair (I <= J) of 16 T short
// rows each, of which the tiles on and above the diagonal are formed.  A wave takes 32
// long elements at a time, of which lane group q holds eight: in a wide matrix
// 8q..8q+7 (128 contiguous bytes a row), in a tall one 4s + q, s = 0..7 (whole
// contiguous rows).  Which element is which k does not matter to a sum over all of
// them, as long as both operands agree.
//
// FULL: all 32 are inside and may be read four at a time.  Then there is no branch
// around a load, which would make the wave wait for it at the branch's end; the elements
// that follow are under way while the present ones are multiplied.  Rows past the short
// side read the last one; their sums are cleared.
template <bool BF, int T, bool TALL, bool FULL>
__device__ __forceinline__ void gram_rows(const Entry& e, const void* x, int row0, int64_t k0,
                                          int64_t kend, int lane, float (&u)[T][8]) {
  const int m = lane & 15, q = lane >> 4;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int i = row0 + 16 * t + m, at = i < e.r ? i : e.r - 1;
    if constexpr (TALL) {
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const int64_t k = k0 + 4 * s + q;
        u[t][s] = FULL || k < kend ? load1<BF>(x, k * e.r + at) : 0.0f;
      }
    } else {
      const int64_t k = k0 + 8 * q;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (FULL) {
          load4<BF>(x, (int64_t)at * e.K + k + 4 * h, u[t] + 4 * h);
        } else {
          const int64_t left = kend - k - 4 * h;
          load_upto4<BF>(x, (int64_t)at * e.K + k + 4 * h, (int)(left < 4 ? left : 4), e.vec,
                         u[t] + 4 * h);
        }
      }
    }
  }
}
// acc[i][j] += rows rowa + 16 i times rows rowb + 16 j over k0, k0 + step, .. < k1;
// SAME: the two are one, and the tiles below the diagonal stay out.
template <bool BF, int TA, int TB, bool TALL, bool SAME>
__device__ __forceinline__ void gram_walk(const Entry& e, const void* x, int rowa, int rowb,
                                          int64_t k0, int64_t k1, int step, int lane,
                                          d4 (&acc)[TA][TB]) {
  auto multiply = [&](float (&a)[TA][8], float (&b)[TB][8]) {
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = SAME ? i : 0; j < TB; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(
              (double)a[i][s], (double)(SAME ? a[j < TA ? j : 0][s] : b[j][s]), acc[i][j], 0, 0, 0);
  };
  float a[TA][8], b[TB][8], na[TA][8], nb[TB][8];
  if (e.vec || TALL) {
    if (k0 + 32 <= k1) {
      gram_rows<BF, TA, TALL, true>(e, x, rowa, k0, k1, lane, na);
      if constexpr (!SAME) gram_rows<BF, TB, TALL, true>(e, x, rowb, k0, k1, lane, nb);
    }
    for (; k0 + 32 <= k1; k0 += step) {
      const int64_t next = k0 + step + 32 <= k1 ? k0 + step : k0;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
#pragma unroll
        for (int i = 0; i < TA; ++i) a[i][s] = na[i][s];
#pragma unroll
        for (int i = 0; i < TB; ++i) b[i][s] = SAME ? 0.0f : nb[i][s];
      }
      gram_rows<BF, TA, TALL, true>(e, x, rowa, next, k1, lane, na);
      if constexpr (!SAME) gram_rows<BF, TB, TALL, true>(e, x, rowb, next, k1, lane, nb);
      multiply(a, b);
    }
  }
  for (; k0 < k1; k0 += step) {
    gram_rows<BF, TA, TALL, false>(e, x, rowa, k0, k1, lane, a);
    if constexpr (!SAME) gram_rows<BF, TB, TALL, false>(e, x, rowb, k0, k1, lane, b);
    multiply(a, b);
  }
}
// 1 / (|U|_F + eps), or 0 of a zero matrix without eps, which stays zero.
__device__ __forceinline__ double over(double trace, double eps) {
  const double norm = sqrt(trace) + eps;
  return norm == 0.0 ? 0.0 : 1.0 / norm;
}
// A sum of the Gram matrix, or 0 past the short side.
__device__ __forceinline__ double inside(const Entry& e, double sum, int row, int col) {
  return row < e.r && col < e.r ? sum : 0.0;
}
// One wave's tiles of a block of 4 x 4, from tile (ti, tj) on, over a chunk.
template <bool BF, int TA, int TB, bool SAME>
__device__ __forceinline__ void gram_tiles(const Entry& e, const void* x, int rowI, int rowJ, int ti,
                                           int tj, int64_t k0, int64_t k1, int lane, double* to) {
  d4 acc[TA][TB] = {};
  rowI += 16 * ti, rowJ += 16 * tj;
  if (rowI < e.r && rowJ < e.r) {  // (zeros past the short side are read, too)
    if (e.tall)
      gram_walk<BF, TA, TB, true, SAME>(e, x, rowI, rowJ, k0, k1, 32, lane, acc);
    else
      gram_walk<BF, TA, TB, false, SAME>(e, x, rowI, rowJ, k0, k1, 32, lane, acc);
  }
#pragma unroll
  for (int i = 0; i < TA; ++i)
#pragma unroll
    for (int j = SAME ? i : 0; j < TB; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        to[((ti + i) * 4 + tj + j) * 256 + v * 64 + lane] =
            inside(e, acc[i][j][v], rowI + 16 * i + 4 * v + (lane >> 4), rowJ + 16 * j + (lane & 15));
}

template <int T, bool BF>
__global__ __launch_bounds__(NTH) void gram(Table tab, double* __restrict__ part,
                                            uint32_t* __restrict__ copy) {
  __shared__ double sum[T < 4 ? T * T * 256 : 1];
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < (int)(sizeof(Table) / 4); i += NTH)
      copy[i] = ((const uint32_t*)&tab)[i];
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t w;
  if constexpr (T == 4) {
    // a unit is 128 long elements of a block pair; the sums of a workgroup's units of
    // one pair go to the place numbered by both
    const uint32_t b = neighbours(), end = tab.gram.begin(b + 1);
    for (uint32_t u = tab.gram.begin(b); u < end;) {
      const Entry& e = find(tab, IN_GRAM, u, w);
      const Pairs pairs(e);
      const uint32_t mat = w / pairs.each, in = w % pairs.each, selves = pairs.nb * pairs.self;
      const uint32_t pair = in < selves ? in / pairs.self : pairs.nb + (in - selves) / pairs.other;
      const uint32_t first = in - pairs.begin(pair);
      const uint32_t many = min((pair < pairs.nb ? pairs.self : pairs.other) - first, end - u);
      const int unit = pair < pairs.nb ? SELF : UNIT;
      u += many;
      int I, J;
      pairs.blocks(pair, I, J);
      const void* x = (const char*)e.x + mat * e.r * (int64_t)e.K * (BF ? 2 : 4);
      const int64_t k0 = (int64_t)first * unit, k1 = min(k0 + (int64_t)many * unit, (int64_t)e.K);
      double* to = part + e.part + ((int64_t)mat * pairs.many() + pair + b) * 4096;
      // what a lane reads is worked out here, each time: kept over the loop, the three
      // forms' addresses below would take the third wave's registers
      int mine = lane;
      asm volatile("" : "+v"(mine));
      // Each wave a quarter of the block, two tiles by two: 32 registers of sums leave
      // room for more waves, and for the elements under way.  Of a block with itself,
      // two waves take its two ends (three tiles each) and two the rest, other waves in
      // every other block.
      const int as = wave ^ (pair & 1 ? 2 : 0);
      if (I != J)
        gram_tiles<BF, 2, 2, false>(e, x, I * 64, J * 64, wave >> 1 << 1, (wave & 1) << 1, k0, k1,
                                    mine, to);
      else if (as < 2)
        gram_tiles<BF, 2, 2, true>(e, x, I * 64, I * 64, 2 * as, 2 * as, k0, k1, mine, to);
      else
        gram_tiles<BF, 1, 2, false>(e, x, I * 64, I * 64, as - 2, 2, k0, k1, mine, to);
    }
  } else {
    const Entry& e = find(tab, IN_GRAM, blockIdx.x, w);
    const int64_t mat = w / e.chunks, chunk = w % e.chunks;
    const void* x = (const char*)e.x + mat * e.r * (int64_t)e.K * (BF ? 2 : 4);
    const int64_t k0 = chunk * e.CH, k1 = k0 + e.CH < e.K ? k0 + e.CH : e.K;
    double* to = part + e.part + (int64_t)w * (T * T * 256);
    d4 acc[T][T] = {};
    if (e.tall)
      gram_walk<BF, T, T, true, true>(e, x, 0, 0, k0 + 32 * wave, k1, 128, lane, acc);
    else
      gram_walk<BF, T, T, false, true>(e, x, 0, 0, k0 + 32 * wave, k1, 128, lane, acc);
    // the waves' sums in their order, so that the result does not depend on the time
    for (int o = 0; o < NTH / 64; ++o) {
      if (wave == o) {
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = i; j < T; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const int at = (i * T + j) * 256 + v * 64 + lane;
              sum[at] = o ? sum[at] + acc[i][j][v] : acc[i][j][v];
            }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < T * T * 256; i += NTH) {
      const int row = i / 256 / T, col = i / 256 % T;
      if (row <= col)
        to[i] = inside(e, sum[i], 16 * row + i % 256 / 16, 16 * col + i % 16);
    }
  }
}

// Element (row, col) of U U' from sums over blocks of 64 short rows; what lies below
// the diagonal was not formed, or is not the upper half's to the bit.
__device__ __forceinline__ double gram_at(const double* part, int nb, int row, int col) {
  if (row > col) {
    const int s = row;
    row = col, col = s;
  }
  const int bi = row / 64, bj = col / 64;
  const int pair = bi * nb - bi * (bi - 1) / 2 + bj - bi;
  const int tile = row / 16 % 4 * 4 + col / 16 % 4, m = row % 16;
  return part[(int64_t)pair * 4096 + tile * 256 + m / 4 * 64 + m % 4 * 16 + col % 16];
}

// ---------------------------------------------------------------- P, r <= 16
// One wave holds everything in registers: register v of lane (m, q) is element
// [4v + q][m], which is what a product wants of either operand, so a product of two
// symmetric matrices is four instructions on the registers they lie in.  Two sums
// each, as an instruction waits 27 ns for the sum before it.
__device__ __forceinline__ d4 product16(d4 a, d4 b) {
  d4 x = {0.0, 0.0, 0.0, 0.0}, y = x;
  x = __builtin_amdgcn_mfma_f64_16x16x4f64(a[0], b[0], x, 0, 0, 0);
  y = __builtin_amdgcn_mfma_f64_16x16x4f64(a[1], b[1], y, 0, 0, 0);
  x = __builtin_amdgcn_mfma_f64_16x16x4f64(a[2], b[2], x, 0, 0, 0);
  y = __builtin_amdgcn_mfma_f64_16x16x4f64(a[3], b[3], y, 0, 0, 0);
  return x + y;
}
// The upper half in both places; `turn` is 16 x 17 doubles of this wave's own.
__device__ __forceinline__ d4 mirrored(d4 g, double* turn, int m, int q) {
#pragma unroll
  for (int v = 0; v < 4; ++v) turn[(4 * v + q) * 17 + m] = g[v];
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const double t = turn[m * 17 + 4 * v + q];
    if (4 * v + q > m) g[v] = t;
  }
  __builtin_amdgcn_wave_barrier();
  return g;
}
// P of the sums `g` (register v of lane (m, q): [4v + q][m], zero from r on).
__device__ __forceinline__ d4 steps16(const Table& tab, d4 g, double* turn, int m, int q) {
  double trace = 0.0;
#pragma unroll
  for (int v = 0; v < 4; ++v) trace += 4 * v + q == m ? g[v] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) trace += __shfl_xor(trace, o);
  const double inv = over(trace, tab.eps);
  d4 one, P;
#pragma unroll
  for (int v = 0; v < 4; ++v) one[v] = 4 * v + q == m ? 1.0 : 0.0;
  d4 G = mirrored(g * inv * inv, turn, m, q);
  P = one * inv;
  for (int s = 0; s < tab.steps; ++s) {
    const d4 Q = product16(G, G) * tab.c + G * tab.b + one * tab.a;
    P = product16(Q, P);
    if (s + 1 < tab.steps) G = mirrored(product16(product16(Q, G), Q), turn, m, q);
  }
  return P;
}

__global__ __launch_bounds__(64) void poly16(const Table* __restrict__ table,
                                             const double* __restrict__ part,
                                             double* __restrict__ poly) {
  __shared__ double turn[16 * 17];
  const Table& tab = *table;
  uint32_t mat;
  const Entry& e = find(tab, IN_POLY, blockIdx.x, mat);
  const int lane = threadIdx.x, m = lane & 15, q = lane >> 4;
  const double* p = part + e.part + (int64_t)mat * e.chunks * 256 + lane;
  d4 g = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
  for (int c = 0; c < e.chunks; ++c)
#pragma unroll
    for (int v = 0; v < 4; ++v) g[v] += p[c * 256 + v * 64];
  const d4 P = steps16(tab, g, turn, m, q);
#pragma unroll
  for (int v = 0; v < 4; ++v) poly[e.poly + (int64_t)mat * 256 + v * 64 + lane] = P[v];
}

// ---------------------------------------------------------------- P, r <= 32
// One workgroup of four waves a matrix, everything in LDS; T tiles of 16 rows, tile
// (w, j) the work of wave (w T + j) % 4.
template <int T>
__device__ __forceinline__ d4 product_tile(const double* A, const double* B, int w, int j, int lane) {
  constexpr int R = 16 * T;
  const int m = lane & 15, q = lane >> 4;
  d4 x = {0.0, 0.0, 0.0, 0.0}, y = x;
#pragma unroll
  for (int k = 0; k < R; k += 8) {
    x = __builtin_amdgcn_mfma_f64_16x16x4f64(A[(k + q) * R + 16 * w + m],  // A symmetric
                                             B[(k + q) * R + 16 * j + m], x, 0, 0, 0);
    y = __builtin_amdgcn_mfma_f64_16x16x4f64(A[(k + 4 + q) * R + 16 * w + m],
                                             B[(k + 4 + q) * R + 16 * j + m], y, 0, 0, 0);
  }
  return x + y;
}

template <int T>
__global__ __launch_bounds__(NTH) void poly_small(const Table* __restrict__ table,
                                                  const double* __restrict__ part,
                                                  double* __restrict__ poly) {
  constexpr int R = 16 * T, N = R * R, OWN = T * T / 4;  // tiles of a wave
  __shared__ double G[N], Q[N], P[N];
  const Table& tab = *table;
  uint32_t mat;
  const Entry& e = find(tab, IN_POLY, blockIdx.x, mat);
  const double* mine = part + e.part + (int64_t)mat * e.chunks * N;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
  // the tiles on and above the diagonal, as the waves of gram left them
  for (int i = threadIdx.x; i < N; i += NTH) {
    const int row = i / 256 / T * 16 + (i & 255) / 64 * 4 + (i & 63) / 16;
    const int col = i / 256 % T * 16 + (i & 15);
    if (row > col) continue;
    double s = 0.0;
#pragma unroll 4
    for (int c = 0; c < e.chunks; ++c) s += mine[(int64_t)c * N + i];
    G[row * R + col] = G[col * R + row] = s;
  }
  __syncthreads();
  double trace = 0.0;
  for (int i = 0; i < e.r; ++i) trace += G[i * R + i];
  __syncthreads();
  const double inv = over(trace, tab.eps);
  for (int i = threadIdx.x; i < N; i += NTH) {
    G[i] = G[i] * inv * inv;
    P[i] = i / R == i % R ? inv : 0.0;
  }
  __syncthreads();
  for (int s = 0; s < tab.steps; ++s) {
    const bool more = s + 1 < tab.steps;
    d4 x[OWN], h[OWN];
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int t = o * 4 + wave, w = t / T, j = t % T;
      x[o] = product_tile<T>(G, G, w, j, lane);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = (16 * w + 4 * v + q) * R + 16 * j + m;
        Q[at] = tab.c * x[o][v] + tab.b * G[at] + (16 * w + 4 * v + q == 16 * j + m ? tab.a : 0.0);
      }
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int t = o * 4 + wave;
      x[o] = product_tile<T>(Q, P, t / T, t % T, lane);
      if (more) h[o] = product_tile<T>(Q, G, t / T, t % T, lane);
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int t = o * 4 + wave;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = (16 * (t / T) + 4 * v + q) * R + 16 * (t % T) + m;
        P[at] = x[o][v];
        if (more) G[at] = h[o][v];  // Q G
      }
    }
    __syncthreads();
    if (!more) break;
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int t = o * 4 + wave;
      if (t / T <= t % T) x[o] = product_tile<T>(G, Q, t / T, t % T, lane);
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int t = o * 4 + wave;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int row = 16 * (t / T) + 4 * v + q, col = 16 * (t % T) + m;
        if (row <= col) G[row * R + col] = G[col * R + row] = x[o][v];
      }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < N; i += NTH) poly[e.poly + (int64_t)mat * N + i] = P[i];
}

// ---------------------------------------------------------------- P, r > 32
// Matrices of R = 64 nb in scratch, one behind the other: G, Q (or the other G), P (two,
// in turn) and H = Q G.
enum { SLOT_G, SLOT_Q, SLOT_P0, SLOT_P1, SLOT_H, SLOTS };

// The workgroups' sums of a block pair joined, in their order, in the place of H.
__global__ __launch_bounds__(NTH) void poly_sum(const Table* __restrict__ table,
                                                const double* __restrict__ part,
                                                double* __restrict__ poly) {
  const Table& tab = *table;
  uint32_t w, at;
  const Entry& e = find(tab, IN_SUM, blockIdx.x, w);
  const Pairs pairs(e);
  const uint32_t combo = w / 8, piece = w % 8, mat = combo / pairs.many();
  const uint32_t pair = combo % pairs.many(), R = 64 * pairs.nb;
  int I, J;
  pairs.blocks(pair, I, J);
  const uint32_t u0 = tab.tile0[IN_GRAM][&e - tab.e] + mat * pairs.each + pairs.begin(pair);
  const uint32_t b0 = tab.gram.owner(u0);
  const uint32_t many =
      tab.gram.owner(u0 + (pair < pairs.nb ? pairs.self : pairs.other) - 1) - b0 + 1;
  at = piece * NTH + threadIdx.x;
  const double2* p = (const double2*)(part + e.part + ((int64_t)combo + b0) * 4096) + at;
  double2 s = make_double2(0.0, 0.0);
#pragma unroll 4
  for (uint32_t c = 0; c < many; ++c) {
    const double2 x = p[(int64_t)c * 2048];
    s.x += x.x, s.y += x.y;
  }
  // (gram_at counts the pairs row by row)
  const int64_t place = I * pairs.nb - I * (I - 1) / 2 + J - I;
  double* to = poly + e.poly + ((int64_t)mat * SLOTS + SLOT_H) * R * R;
  ((double2*)(to + place * 4096))[at] = s;
}

// G = U U' / (|U|_F + eps)^2 and P = I / (|U|_F + eps), from the joined sums.
__global__ __launch_bounds__(NTH) void poly_norm(const Table* __restrict__ table,
                                                 double* __restrict__ poly) {
  __shared__ double red[NTH / 64];
  const Table& tab = *table;
  uint32_t w;
  const Entry& e = find(tab, IN_NORM, blockIdx.x, w);
  const int nb = (e.r + 63) / 64, R = 64 * nb;
  const uint32_t per = (uint32_t)R * R / 1024;
  double* base = poly + e.poly + (int64_t)(w / per) * SLOTS * R * R;
  const double* mine = base + (int64_t)SLOT_H * R * R;
  double trace = 0.0;
  for (int i = threadIdx.x; i < e.r; i += NTH) trace += gram_at(mine, nb, i, i);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) trace += __shfl_xor(trace, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = trace;
  __syncthreads();
  trace = red[0] + red[1] + red[2] + red[3];
  const double inv = over(trace, tab.eps);
  for (int i = threadIdx.x; i < 1024; i += NTH) {
    const int at = (int)(w % per) * 1024 + i;
    base[at] = gram_at(mine, nb, at / R, at % R) * inv * inv;  // SLOT_G
    base[(int64_t)SLOT_P0 * R * R + at] = at / R == at % R ? inv : 0.0;
  }
}

// Short sides of 64 and 128: a step is one launch.  A workgroup holds all of G in LDS
// and forms 16 rows of the next G and P by themselves,
//   H = aG + b GG + c GGG,  G' = aH + b HG + c HGG,  P' = aP + b PG + c PGG,
// each product those rows times G.  That is six products of 16 rows in the place of
// four of all, but nothing waits for another workgroup within a step: 21 us at 28
// matrices of 128 (10 us of products, the rest G's way into LDS and the barriers; 25
// with a matrix's workgroups on all XCDs) where the three launches of the tiles below
// took 33.  (G' as one polynomial of G, whose coefficients reach 37, lost two more
// digits.)
// Wave j forms columns 16 j..; the rows that are multiplied next stand transposed in
// LDS, rows of 17 doubles.  G' is written from its upper half to both places.
template <int R>
__global__ __launch_bounds__(4 * R) void poly_panel(const Table* __restrict__ table, int turn,
                                                    int more, double* __restrict__ poly) {
  __shared__ double G[R * R];
  __shared__ double T[R * 17];
  const Table& tab = *table;
  uint32_t w;
  const Entry& e = find(tab, IN_POLY, neighbours(), w);
  const int I = (int)(w % (R / 16));
  double* base = poly + e.poly + (int64_t)(w / (R / 16)) * SLOTS * R * R;
  const double* Gold = base + (int64_t)(turn ? SLOT_Q : SLOT_G) * R * R;
  double* Gnew = base + (int64_t)(turn ? SLOT_G : SLOT_Q) * R * R;
  const double* Pold = base + (int64_t)(turn ? SLOT_P1 : SLOT_P0) * R * R;
  double* Pnew = base + (int64_t)(turn ? SLOT_P0 : SLOT_P1) * R * R;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int j = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  d2 in[R / 8];
#pragma unroll
  for (int i = 0; i < R / 8; ++i) in[i] = ((const d2*)Gold)[threadIdx.x + 4 * R * i];
  for (int i = threadIdx.x; i < 16 * R; i += 4 * R)
    T[i / 16 * 17 + i % 16] = Pold[(int64_t)(i / 16) * R + 16 * I + i % 16];  // P symmetric
#pragma unroll
  for (int i = 0; i < R / 8; ++i) ((d2*)G)[threadIdx.x + 4 * R * i] = in[i];
  double p[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) p[v] = Pold[(int64_t)(16 * I + 4 * v + q) * R + 16 * j + m];
  __syncthreads();
  auto times = [&](const double* A, int ld) {  // the rows A[k][i] times G's columns 16 j..
    d4 x = {0.0, 0.0, 0.0, 0.0}, y = x;
#pragma unroll 8
    for (int k = 0; k < R; k += 8) {
      x = __builtin_amdgcn_mfma_f64_16x16x4f64(A[(k + q) * ld + m], G[(k + q) * R + 16 * j + m], x, 0,
                                               0, 0);
      y = __builtin_amdgcn_mfma_f64_16x16x4f64(A[(k + 4 + q) * ld + m],
                                               G[(k + 4 + q) * R + 16 * j + m], y, 0, 0, 0);
    }
    return x + y;
  };
  auto next = [&](d4 x) {  // x times G
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v) T[(16 * j + m) * 17 + 4 * v + q] = x[v];
    __syncthreads();
    return times(T, 17);
  };
  const double ca = tab.a, cb = tab.b, cc = tab.c;
  const d4 z1 = times(T, 17);
  d4 y = z1;
  if (more) y = times(G + 16 * I, R);  // G symmetric
  const d4 z2 = next(z1);
#pragma unroll
  for (int v = 0; v < 4; ++v)
    Pnew[(int64_t)(16 * I + 4 * v + q) * R + 16 * j + m] = ca * p[v] + cb * z1[v] + cc * z2[v];
  if (!more) return;
  d4 h;
#pragma unroll
  for (int v = 0; v < 4; ++v) h[v] = ca * G[(16 * I + 4 * v + q) * R + 16 * j + m];
  h += y * cb;
  h += next(y) * cc;
  y = next(h);
  const d4 g = h * ca + y * cb + next(y) * cc;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int row = 16 * I + 4 * v + q, col = 16 * j + m;
    if (row <= col)
      Gnew[(int64_t)row * R + col] = Gnew[(int64_t)col * R + row] = g[v];
  }
}

// Short sides beyond 128, in tiles of 32 x 32 and three launches a step.
// mode 0: Q = aI + bG + cGG;  mode 1: P' = Q P and (blockIdx.y = 1) H = Q G;
// mode 2: G = H Q.  All are polynomials of one symmetric matrix, so symmetric: the tiles on
// and above the diagonal are formed and written to both places, turned over in LDS, a
// matrix's workgroups on one XCD (a launch of mode 0 at 4 matrices of 1024: 135 us, every
// tile formed 216; at 16 of 256 16 and 22).
__global__ __launch_bounds__(NTH) void poly_step(const Table* __restrict__ table, int mode, int turn,
                                                 double* __restrict__ poly) {
  __shared__ double As[128 * 32], Bs[128 * 32];
  const Table& tab = *table;
  uint32_t w;
  const Entry& e = find(tab, IN_POLY, neighbours(), w);
  const int R = (e.r + 63) / 64 * 64;
  const int nt = R / 32, per = nt * (nt + 1) / 2;
  double* base = poly + e.poly + (int64_t)(w / per) * SLOTS * R * R;
  int i0 = 0, j0 = (int)(w % per);  // (0,0..nt-1), (1,1..nt-1), ...
  while (j0 >= nt - i0) j0 -= nt - i0, ++i0;
  j0 = 32 * (j0 + i0), i0 *= 32;
  const int64_t RR = (int64_t)R * R;
  const int from = turn ? SLOT_P1 : SLOT_P0, into = turn ? SLOT_P0 : SLOT_P1;
  const bool h = mode == 1 && blockIdx.y == 1;
  const double* A = base + (mode == 0 ? SLOT_G : mode == 1 ? SLOT_Q : SLOT_H) * RR;
  const double* B = base + (mode == 0 || h ? SLOT_G : mode == 1 ? from : SLOT_Q) * RR;
  double* D = base + (mode == 0 ? SLOT_Q : h ? SLOT_H : mode == 1 ? into : SLOT_G) * RR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = lane & 15, q = lane >> 4, wi = 16 * (wave >> 1), wj = 16 * (wave & 1);
  d4 acc = {0.0, 0.0, 0.0, 0.0}, odd = acc;
  const int lr = threadIdx.x / 16, lc = threadIdx.x % 16 * 2;
  const d2* pa = (const d2*)(A + (int64_t)lr * R + i0 + lc);  // A symmetric
  const d2* pb = (const d2*)(B + (int64_t)lr * R + j0 + lc);
  const int64_t by = 8 * (int64_t)R;  // 16 rows
  d2* wa = (d2*)(As + lr * 32 + lc);
  d2* wb = (d2*)(Bs + lr * 32 + lc);
  for (int k0 = 0; k0 < R; k0 += 128) {
    // 128 rows of either operand under way at once: what a launch takes is one round
    // trip to memory (with 64 rows and the next 64 behind them 9 us, so 6)
    d2 ta[8], tb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = k0 + 16 * i < R ? k0 / 16 + i : 0;
      ta[i] = pa[at * by], tb[i] = pb[at * by];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[256 * i] = ta[i], wb[256 * i] = tb[i];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 128; h += 64) {
      if (k0 + h >= R) break;
#pragma unroll
      for (int k = h; k < h + 64; k += 8) {
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(As[(k + q) * 32 + wi + m],
                                                   Bs[(k + q) * 32 + wj + m], acc, 0, 0, 0);
        odd = __builtin_amdgcn_mfma_f64_16x16x4f64(As[(k + 4 + q) * 32 + wi + m],
                                                   Bs[(k + 4 + q) * 32 + wj + m], odd, 0, 0, 0);
      }
    }
  }
  acc += odd;
  __syncthreads();
  double* tile = As;  // rows of 33
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int row = wi + 4 * v + q, col = wj + m;
    const int64_t at = (int64_t)(i0 + row) * R + j0 + col;
    tile[row * 33 + col] =
        mode ? acc[v] : tab.c * acc[v] + tab.b * A[at] + (i0 + row == j0 + col ? tab.a : 0.0);
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 1024; i += NTH) {
    const int row = i / 32, col = i % 32;
    const double up = tile[row * 33 + col], low = tile[col * 33 + row];
    D[(int64_t)(i0 + row) * R + j0 + col] = i0 == j0 && row > col ? low : up;
    if (i0 != j0) D[(int64_t)(j0 + row) * R + i0 + col] = low;
  }
}

// ---------------------------------------------------------------- out = P U
// A wave takes 64 long elements at a time.  Wide: lane (m, q) reads four long elements
// 4m.. of short row 4t + q, which is B[k = 4t + q][j = m] of four products, and
// stores four long elements of rows 4v + q.  Tall: it reads the short elements
// 4q.. of long row m, so that step t's k is 4q + t, and with P's rows taken in the
// order 4 (m % 4) + m / 4 it holds the short elements 4q.. of that row again.
// u[n]: wide, of row 4n + q; tall, of the n-th 16 long rows.  FULL as in gram.
template <bool BF, bool TALL, bool FULL>
__device__ __forceinline__ void apply_rows(const Entry& e, const void* x, int row0, int64_t k0,
                                           int64_t l1, int m, int q, float (&u)[4][4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if constexpr (TALL) {
      const int64_t k = k0 + 16 * n + m;
      const int i = row0 + 4 * q;
      if constexpr (FULL)
        load4<BF>(x, k * e.r + (i < e.r ? i : 0), u[n]);
      else
        load_upto4<BF>(x, k * e.r + i, k < l1 ? e.r - i : 0, e.vec, u[n]);
    } else {
      const int i = row0 + 4 * n + q;
      const int64_t k = k0 + 4 * m, left = i < e.r ? l1 - k : 0;
      if constexpr (FULL)
        load4<BF>(x, (int64_t)(i < e.r ? i : 0) * e.K + k, u[n]);
      else
        load_upto4<BF>(x, (int64_t)i * e.K + k, (int)(left < 4 ? left : 4), e.vec, u[n]);
    }
  }
}
// acc[i][c] += of one tile of 16 short elements: Ps is P's block, its rows k0.. taken, N
// tiles of its columns from col0 on.  Past the short side P is zero off its diagonal, and
// U's place holds others of its elements.
template <int N, bool TALL>
__device__ __forceinline__ void apply_tile(const double* Ps, int ld, int k0, int col0, int m, int q,
                                           const float (&u)[4][4], d4 (&acc)[N][4]) {
  const int prow = TALL ? 4 * (m & 3) + (m >> 2) : m;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int k = TALL ? 4 * q + t : 4 * t + q;
    double b[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) b[c] = (double)(TALL ? u[c][t] : u[t][c]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double a = Ps[(k0 + k) * ld + col0 + 16 * i + prow];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        acc[i][c] = __builtin_amdgcn_mfma_f64_16x16x4f64(a, b[c], acc[i][c], 0, 0, 0);
    }
  }
}
template <int N, bool BF, bool TALL, bool FULL>
__device__ __forceinline__ void apply_store(const Entry& e, void* out, int row0, int64_t k0,
                                            int64_t l1, int m, int q, const d4 (&acc)[N][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float f[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) f[n] = (float)(TALL ? acc[i][s][n] : acc[i][n][s]);
      if constexpr (TALL) {
        const int64_t k = k0 + 16 * s + m;
        const int row = row0 + 16 * i + 4 * q;
        if constexpr (!FULL)
          store_upto4<BF>(out, k * e.r + row, k < l1 ? e.r - row : 0, e.vec, f);
        else if (row < e.r)
          store4<BF>(out, k * e.r + row, f);
      } else {
        const int row = row0 + 16 * i + 4 * s + q;
        const int64_t k = k0 + 4 * m, left = row < e.r ? l1 - k : 0;
        if constexpr (!FULL)
          store_upto4<BF>(out, (int64_t)row * e.K + k, (int)(left < 4 ? left : 4), e.vec, f);
        else if (row < e.r)
          store4<BF>(out, (int64_t)row * e.K + k, f);
      }
    }
}

// (Entries are copied: read where they are used, behind a store, they would be vector
// loads, and waiting for those waits for the tiles under way.)

// Short sides of one block, 16 T: a workgroup takes e.AL long elements, a wave every
// fourth 64 of them, its next ones on their way while the present ones are multiplied.
template <int T, bool BF, bool TALL>
__device__ __forceinline__ void apply_walk(const Entry& e, const void* x, void* out,
                                           const double* P, double* Ps, int64_t k0, int64_t l1,
                                           int m, int q) {
  constexpr int R = 16 * T;
  float u[T][4][4], next[T][4][4];
  const bool fast = e.vec && k0 + 64 <= l1;
  if (fast) {
#pragma unroll
    for (int t = 0; t < T; ++t) apply_rows<BF, TALL, true>(e, x, 16 * t, k0, l1, m, q, next[t]);
  }
  for (int i = threadIdx.x; i < R * R; i += NTH) Ps[i] = P[i];
  __syncthreads();
  if (fast) {
    for (; k0 + 64 <= l1; k0 += 256) {
      const int64_t kn = k0 + 256 + 64 <= l1 ? k0 + 256 : k0;
#pragma unroll
      for (int t = 0; t < T; ++t) {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
          for (int b = 0; b < 4; ++b) u[t][a][b] = next[t][a][b];
        apply_rows<BF, TALL, true>(e, x, 16 * t, kn, l1, m, q, next[t]);
      }
      d4 acc[T][4] = {};
#pragma unroll
      for (int t = 0; t < T; ++t)
        apply_tile<T, TALL>(Ps, R, 16 * t, 0, m, q, u[t], acc);
      apply_store<T, BF, TALL, true>(e, out, 0, k0, l1, m, q, acc);
    }
  }
  for (; k0 < l1; k0 += 256) {
    d4 acc[T][4] = {};
#pragma unroll
    for (int t = 0; t < T; ++t) {
      apply_rows<BF, TALL, false>(e, x, 16 * t, k0, l1, m, q, u[t]);
      apply_tile<T, TALL>(Ps, R, 16 * t, 0, m, q, u[t], acc);
    }
    apply_store<T, BF, TALL, false>(e, out, 0, k0, l1, m, q, acc);
  }
}

template <int T, bool BF>
__global__ __launch_bounds__(NTH) void apply(const Table* __restrict__ table,
                                             const double* __restrict__ poly) {
  constexpr int R = 16 * T;
  __shared__ double Ps[R * R];
  const Table& tab = *table;
  uint32_t w;
  const Entry e = find(tab, IN_APPLY, blockIdx.x, w);
  const uint32_t tiles = (uint32_t)((e.K + e.AL - 1) / e.AL);
  const int64_t mat = w / tiles, l0 = (int64_t)(w % tiles) * e.AL;
  const int64_t l1 = l0 + e.AL < e.K ? l0 + e.AL : e.K;
  const int64_t off = mat * e.r * (int64_t)e.K * (BF ? 2 : 4);
  const void* x = (const char*)e.x + off;
  void* out = (char*)e.out + off;
  const double* P = poly + e.poly + mat * R * R;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (e.tall)
    apply_walk<T, BF, true>(e, x, out, P, Ps, l0 + 64 * wave, l1, lane & 15, lane >> 4);
  else
    apply_walk<T, BF, false>(e, x, out, P, Ps, l0 + 64 * wave, l1, lane & 15, lane >> 4);
}

// Short sides of blocks of 64: a workgroup takes its share of units of 128 long elements
// of one block, a unit at a time, a wave half of the block's rows and 64 of them.  P's
// blocks stay in LDS where there are at most two.  The tile of U that follows, be it of
// the next unit, is on its way while the present one is multiplied.
template <bool BF, bool TALL>
__device__ __forceinline__ void apply64_walk(const Entry& e, const void* x, void* out,
                                             const double* P, double* Pall, int nb, int I,
                                             int64_t l0, int64_t l1, int wave, int m, int q) {
  const int R = 64 * nb, wi = wave & 1, wl = wave >> 1, rows = I * 64 + 32 * wi;
  const bool idle = rows >= e.r;  // (of the last block; the others wait for it below)
  auto fill = [&](double* Ps, int kb) {
    d2 in[8];
    const d2* from = (const d2*)(P + (int64_t)(kb * 64 + threadIdx.x / 32) * R + I * 64) +
                     threadIdx.x % 32;
#pragma unroll
    for (int i = 0; i < 8; ++i) in[i] = from[(int64_t)i * 4 * R];
#pragma unroll
    for (int i = 0; i < 8; ++i) ((d2*)Ps)[threadIdx.x + 256 * i] = in[i];
  };
  int64_t k0 = l0 + 64 * wl;  // a wave past the end loads nothing and stores nothing
  const bool fast = e.vec && k0 + 64 <= l1;
  float next[4][4];
  if (fast) apply_rows<BF, TALL, true>(e, x, 0, k0, l1, m, q, next);
  __syncthreads();  // P's places are free again
  if (nb <= 2) {
    fill(Pall, 0);
    if (nb == 2) fill(Pall + 4096, 1);
    __syncthreads();
  }
  // one unit; the two kinds of loads in loops of their own: where they meet, the wave
  // waits for the loads under way (28 factors of rank 128: 124 us, so 103)
  auto unit = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    const int64_t kn = k0 + UNIT + 64 <= l1 ? k0 + UNIT : k0;
    d4 acc[2][4] = {};
    for (int kb = 0; kb < nb; ++kb) {
      double* Ps = Pall + (nb <= 2 ? kb : 0) * 4096;
      if (nb > 2) {
        __syncthreads();
        fill(Ps, kb);
        __syncthreads();
      }
      if (idle) continue;
      const int stop = min(e.r, kb * 64 + 64);
#pragma unroll 1
      for (int row = kb * 64; row < stop; row += 16) {
        float u[4][4];
        if constexpr (FULL) {
          const bool end = row + 16 >= e.r;
#pragma unroll
          for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) u[a][b] = next[a][b];
          apply_rows<BF, TALL, true>(e, x, end ? 0 : row + 16, end ? kn : k0, l1, m, q, next);
        } else {
          apply_rows<BF, TALL, false>(e, x, row, k0, l1, m, q, u);
        }
        apply_tile<2, TALL>(Ps, 64, row % 64, 32 * wi, m, q, u, acc);
      }
    }
    if (!idle) apply_store<2, BF, TALL, FULL>(e, out, rows, k0, l1, m, q, acc);
    k0 += UNIT;
  };
  int64_t step = l0;
  if (fast)
    for (; step < l1 && k0 + 64 <= l1; step += UNIT) unit(std::true_type());
  for (; step < l1; step += UNIT) unit(std::false_type());
}

template <bool BF>
__global__ __launch_bounds__(NTH) void apply64(const Table* __restrict__ table, int last,
                                               const double* __restrict__ poly) {
  __shared__ double Pall[2 * 4096];
  const Table& tab = *table;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t b = neighbours(), end = tab.apply.begin(b + 1);
  for (uint32_t at = tab.apply.begin(b); at < end;) {
    uint32_t w;
    const Entry e = find(tab, IN_APPLY, at, w);
    const uint32_t units = units_of(e, UNIT), mb = w / units, first = w % units;
    const uint32_t many = min(units - first, end - at);
    at += many;
    const int nb = (e.r + 63) / 64, R = 64 * nb, I = (int)(mb % nb);
    const int64_t mat = mb / nb, l0 = (int64_t)first * UNIT;
    const int64_t l1 = min(l0 + (int64_t)many * UNIT, (int64_t)e.K);
    const int64_t off = mat * e.r * (int64_t)e.K * (BF ? 2 : 4);
    const void* x = (const char*)e.x + off;
    void* out = (char*)e.out + off;
    const double* P = poly + e.poly + (mat * SLOTS + (last ? SLOT_P1 : SLOT_P0)) * R * R;
    if (e.tall)
      apply64_walk<BF, true>(e, x, out, P, Pall, nb, I, l0, l1, wave, lane & 15, lane >> 4);
    else
      apply64_walk<BF, false>(e, x, out, P, Pall, nb, I, l0, l1, wave, lane & 15, lane >> 4);
  }
}

// ---------------------------------------------------------------- all of it, r <= 16
// Matrices with long sides up to WHOLE: a workgroup of eight waves holds one in its
// registers, or two, four or eight shorter ones, so it is read once and nothing goes
// through memory in between (a call on 128 experts' factors at rank 16: 49 us, with the
// three launches of longer ones 55; on 14 factors of rank 4 37 and 47).
// Registers hold U as the last product wants it; for the Gram matrix each wave turns 64
// long elements at a time over in LDS.  One wave a matrix does the steps; two workgroups a
// CU cover for one another.
constexpr int WAVES = 8, BLOCKS = 4, WHOLE = 64 * WAVES * BLOCKS;
constexpr int LD = 68;  // floats of a row that is turned over
static_assert(LD * sizeof(float) >= 17 * sizeof(double), "a tile is the room of steps16, too");
// waves that hold a matrix
__host__ __device__ inline int waves_of(const Entry& e) {
  int w = WAVES;
  while (w > 1 && e.K <= 32 * w * BLOCKS) w /= 2;
  return w;
}

// 64 long elements from k0 on, as apply_rows; what lies behind the end is cleared where it
// is first used, so that nothing waits for all loads.
template <bool BF, bool TALL>
__device__ __forceinline__ void whole_rows(const Entry& e, const void* x, int k0, int m, int q,
                                           float (&u)[4][4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int k = TALL ? k0 + 16 * n + m : k0 + 4 * m, i = TALL ? 4 * q : 4 * n + q;
    const uint32_t at = TALL ? k * e.r + i : i * e.K + k;  // below 16 WHOLE
    load4<BF>(x, k < e.K && i < e.r ? at : 0, u[n]);
  }
}
template <bool TALL>
__device__ __forceinline__ void whole_clear(const Entry& e, int k0, int m, float (&u)[4][4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const bool in = (TALL ? k0 + 16 * n + m : k0 + 4 * m) < e.K;
#pragma unroll
    for (int c = 0; c < 4; ++c) u[n][c] = in ? u[n][c] : 0.0f;
  }
}

// `wave` of the `waves` that hold the matrix; `sum` and `tile` are its own, the sums of the
// others behind the first one's.  `live`: there is one.
template <bool BF, bool TALL>
__device__ __forceinline__ void whole_walk(const Table& tab, const Entry& e, const void* x,
                                           void* out, double* sum, float* tile, int wave, int waves,
                                           bool live, int lane) {
  const int m = lane & 15, q = lane >> 4;
  float u[BLOCKS][4][4];
  if (e.vec) {
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j)
      whole_rows<BF, TALL>(e, x, 64 * (wave + waves * j), m, q, u[j]);
  } else {
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j)
      apply_rows<BF, TALL, false>(e, x, 0, 64 * (wave + waves * j), e.K, m, q, u[j]);
  }
  d4 g = {0.0, 0.0, 0.0, 0.0}, odd = g;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    const int k0 = 64 * (wave + waves * j);
    if (k0 >= e.K) break;
    if (e.vec) whole_clear<TALL>(e, k0, m, u[j]);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if constexpr (TALL) {
#pragma unroll
        for (int c = 0; c < 4; ++c) tile[(4 * q + c) * LD + 16 * n + m] = u[j][n][c];
      } else {
        *(f32x4*)(tile + (4 * n + q) * LD + 4 * m) =
            f32x4{u[j][n][0], u[j][n][1], u[j][n][2], u[j][n][3]};
      }
    }
    __builtin_amdgcn_wave_barrier();
    // lane (m, q) takes row m's elements 16q..: which is which k does not matter
    f32x4 a[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) a[n] = *(const f32x4*)(tile + m * LD + 16 * q + 4 * n);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        const double v = a[n][c], w = a[n][c + 1];
        g = __builtin_amdgcn_mfma_f64_16x16x4f64(v, v, g, 0, 0, 0);
        odd = __builtin_amdgcn_mfma_f64_16x16x4f64(w, w, odd, 0, 0, 0);
      }
  }
  g += odd;
#pragma unroll
  for (int v = 0; v < 4; ++v) sum[v * 64 + lane] = g[v];
  __syncthreads();
  double* Ps = sum - wave * 256;  // the first wave's, which it has read by then
  if (wave == 0) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      double s = sum[v * 64 + lane];
      for (int w = 1; w < waves; ++w) s += sum[w * 256 + v * 64 + lane];
      g[v] = inside(e, s, 4 * v + q, m);
    }
    const d4 P = steps16(tab, g, (double*)tile, m, q);
#pragma unroll
    for (int v = 0; v < 4; ++v) Ps[v * 64 + lane] = P[v];
  }
  __syncthreads();
  if (!live) return;
#pragma unroll
  for (int j = 0; j < BLOCKS; ++j) {
    const int64_t k0 = 64 * (wave + waves * j);
    if (k0 >= e.K) break;
    d4 acc[1][4] = {};
    apply_tile<1, TALL>(Ps, 16, 0, 0, m, q, u[j], acc);
    if (e.vec && k0 + 64 <= e.K)
      apply_store<1, BF, TALL, true>(e, out, 0, k0, e.K, m, q, acc);
    else
      apply_store<1, BF, TALL, false>(e, out, 0, k0, e.K, m, q, acc);
  }
}

template <bool BF>
__global__ __launch_bounds__(64 * WAVES, 4) void whole(Table tab) {
  __shared__ double sums[WAVES][256];
  __shared__ f32x4 tiles[WAVES][4 * LD];
  uint32_t w;
  const Entry e = find(tab, IN_POLY, blockIdx.x, w);
  const int at = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = waves_of(e);
  // (a workgroup's last matrices may not be there: their waves work on the last one)
  const uint32_t mat = w * (WAVES / waves) + at / waves, last = (uint32_t)e.CH - 1;
  const int64_t off = (int64_t)min(mat, last) * e.r * (int64_t)e.K * (BF ? 2 : 4);
  const void* x = (const char*)e.x + off;
  void* out = (char*)e.out + off;
  if (e.tall)
    whole_walk<BF, true>(tab, e, x, out, sums[at], (float*)tiles[at], at % waves, waves, mat <= last,
                         threadIdx.x & 63);
  else
    whole_walk<BF, false>(tab, e, x, out, sums[at], (float*)tiles[at], at % waves, waves,
                          mat <= last, threadIdx.x & 63);
}

// ---------------------------------------------------------------- host
struct Plan {  // one table's launches
  Table tab;
  int T = 1;
  bool whole = false;
  int64_t count[MAXE];
  int64_t part = 0, poly = 0;  // doubles
};

// Equal pieces of at most about `most` of a long side, in whole units.
int64_t piece(int64_t K, int64_t most, int64_t unit) {
  return st::cdiv(st::cdiv(K, st::cdiv(K, most)), unit) * unit;
}
// Long elements of a workgroup at short sides up to 32: the length whose rounds of
// `slots` workgroups at a time take least, each as long as its longest piece and `start`
// elements more.
int64_t pick(const Plan& p, int64_t unit, int64_t slots, int64_t start) {
  int64_t best = unit, least = INT64_MAX;
  for (const int k : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24}) {
    int64_t n = 0, longest = 0;
    for (int i = 0; i < p.tab.n; ++i) {
      const int64_t K = p.tab.e[i].K, l = piece(K, k * unit, unit);
      n += p.count[i] * st::cdiv(K, l);
      longest = l > longest ? l : longest;
    }
    const int64_t cost = st::cdiv(n, slots) * (longest + start);
    if (cost < least) least = cost, best = k * unit;
    if (n <= slots) break;  // one round: longer ones only take longer
  }
  return best;
}

// Workgroups of gram and apply64 at short sides beyond 32: two a CU run at once.
constexpr int64_t GRAM_WGS = 512, APPLY_WGS = 512;
Shares shares(int64_t units, int64_t wgs) {
  if (wgs > units) wgs = units;
  return {(uint32_t)wgs, (uint32_t)(units / wgs), (uint32_t)(units % wgs)};
}

// The next table: entries from `at` on whose short sides are of one class (up to 16, 32,
// 64, 128, more).  Returns the entries taken.
int make_plan(const st_matrix_batch* in, int32_t n, int32_t at, int32_t dtype, Plan& p) {
  p = Plan();
  Table& t = p.tab;
  int taken = 0;
  int kind = 0;
  t.n = 0;
  for (; at + taken < n && t.n < MAXE; ++taken) {
    const st_matrix_batch& b = in[at + taken];
    if (b.count == 0 || b.rows == 0 || b.cols == 0) continue;
    const int64_t r = b.rows < b.cols ? b.rows : b.cols, K = b.rows < b.cols ? b.cols : b.rows;
    const int mine = r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 3 : r <= 128 ? 4 : 5;
    if (!kind) kind = mine, p.T = kind < 3 ? kind : 4;
    if (mine != kind) break;
    Entry& e = t.e[t.n];
    e.x = b.x, e.out = b.out;
    e.K = (int32_t)K, e.r = (int32_t)r, e.tall = b.rows > b.cols;
    const uintptr_t mask = dtype == ST_DTYPE_BF16 ? 7 : 15;
    e.vec = (e.tall ? r : K) % 4 == 0 && (((uintptr_t)b.x | (uintptr_t)b.out) & mask) == 0;
    p.count[t.n++] = b.count;
  }
  int64_t all = 0;
  p.whole = p.T == 1;
  for (int i = 0; i < t.n; ++i) {
    p.whole = p.whole && t.e[i].K <= WHOLE;
    all += p.count[i];
  }
  if (all * 64 * WAVES >= (int64_t)1 << 32) p.whole = false;  // more than a launch takes
  for (int i = 0; p.whole && i < t.n; ++i) t.e[i].CH = (int32_t)p.count[i];
  if (p.whole) return taken;
  // places: 256 CUs and as many workgroups each as the kernels' registers and LDS allow
  const int64_t ch = p.T == 4 ? 0 : pick(p, 128, p.T == 1 ? 2048 : 1280, 256);
  const int64_t al = p.T == 4 ? 0 : pick(p, 256, p.T == 1 ? 1280 : 512, 256);
  int64_t combos = 0;  // block pairs of matrices
  for (int i = 0; i < t.n; ++i) {
    Entry& e = t.e[i];
    e.poly = p.poly;
    if (p.T == 4) {
      const int64_t nb = st::cdiv(e.r, 64);
      e.part = 4096 * combos;
      combos += p.count[i] * nb * (nb + 1) / 2;
      p.poly += p.count[i] * SLOTS * 4096 * nb * nb;
    } else {
      e.CH = (int32_t)piece(e.K, ch, 128), e.AL = (int32_t)piece(e.K, al, 256);
      e.chunks = (int32_t)st::cdiv(e.K, e.CH);
      e.part = p.part;
      p.part += p.count[i] * e.chunks * p.T * p.T * 256;
      p.poly += p.count[i] * p.T * p.T * 256;
    }
  }
  if (p.T == 4 && t.n) p.part = 4096 * (combos + GRAM_WGS);
  return taken;
}

// Workgroups (units) of a matrix in a phase.
int64_t each_of(const Plan& p, int phase, const Entry& e) {
  const int64_t nb = st::cdiv(e.r, 64);
  switch (phase) {
    case IN_GRAM: return p.T < 4 ? (int64_t)e.chunks : (int64_t)Pairs(e).each;
    case IN_SUM: return p.T < 4 ? 0 : nb * (nb + 1) / 2 * 8;
    case IN_NORM: return p.T < 4 ? 0 : nb * nb * 4;
    case IN_POLY: return p.T < 4 ? 1 : nb <= 2 ? 4 * nb : nb * (2 * nb + 1);
    default: return p.T < 4 ? st::cdiv(e.K, e.AL) : st::cdiv(e.K, UNIT) * nb;
  }
}
// Every phase's workgroups fit a launch.
bool fits(const Plan& p) {
  for (int phase = 0; phase < PHASES; ++phase) {
    int64_t all = 0;
    for (int i = 0; i < p.tab.n; ++i) all += p.count[i] * each_of(p, phase, p.tab.e[i]);
    if (all * NTH >= (int64_t)1 << 32) return false;
  }
  return true;
}
// Numbers the workgroups of a phase; their count.
int64_t number(Plan& p, int phase) {
  int64_t at = 0;
  for (int i = 0; i < 64; ++i) p.tab.tile0[phase][i] = ~0u;
  for (int i = 0; i < p.tab.n; ++i) {
    p.tab.tile0[phase][i] = (uint32_t)at;
    at += p.count[i] * each_of(p, phase, p.tab.e[i]);
  }
  return at;
}

constexpr int64_t TABLE_BYTES = (sizeof(Table) + 15) / 16 * 16;

template <bool BF>
int launch_whole(Plan& p, hipStream_t stream) {
  for (int i = 0; i < p.tab.n; ++i) p.count[i] = st::cdiv(p.count[i], WAVES / waves_of(p.tab.e[i]));
  const int64_t n = number(p, IN_POLY);
  whole<BF><<<(unsigned)n, 64 * WAVES, 0, stream>>>(p.tab);
  return st::check_launch("st_orthogonalize");
}

template <int T, bool BF>
int launch(Plan& p, char* workspace, hipStream_t stream) {
  const int nb = (p.tab.e[0].r + 63) / 64;  // 1, 2 or more for all entries
  int64_t ng = number(p, IN_GRAM), na = number(p, IN_APPLY);
  const int64_t np = number(p, IN_POLY), ns = number(p, IN_SUM), nn = number(p, IN_NORM);
  if (T == 4) {
    p.tab.gram = shares(ng, GRAM_WGS), ng = p.tab.gram.wgs;
    p.tab.apply = shares(na, APPLY_WGS), na = p.tab.apply.wgs;
  }
  const Table* tab = (const Table*)workspace;
  double* part = (double*)(workspace + TABLE_BYTES);
  double* poly = part + p.part;
  gram<T, BF><<<(unsigned)ng, NTH, 0, stream>>>(p.tab, part, (uint32_t*)workspace);
  int turn = 0;
  if constexpr (T == 1) {
    poly16<<<(unsigned)np, 64, 0, stream>>>(tab, part, poly);
  } else if constexpr (T == 2) {
    poly_small<T><<<(unsigned)np, NTH, 0, stream>>>(tab, part, poly);
  } else {
    poly_sum<<<(unsigned)ns, NTH, 0, stream>>>(tab, part, poly);
    poly_norm<<<(unsigned)nn, NTH, 0, stream>>>(tab, poly);
    for (int s = 0; s < p.tab.steps; ++s, turn ^= 1) {
      const int more = s + 1 < p.tab.steps;
      if (nb == 1) {
        poly_panel<64><<<(unsigned)np, 256, 0, stream>>>(tab, turn, more, poly);
      } else if (nb == 2) {
        poly_panel<128><<<(unsigned)np, 512, 0, stream>>>(tab, turn, more, poly);
      } else {
        poly_step<<<(unsigned)np, NTH, 0, stream>>>(tab, 0, turn, poly);
        poly_step<<<dim3((unsigned)np, more ? 2 : 1), NTH, 0, stream>>>(tab, 1, turn, poly);
        if (more) poly_step<<<(unsigned)np, NTH, 0, stream>>>(tab, 2, turn, poly);
      }
    }
  }
  if constexpr (T == 4)
    apply64<BF><<<(unsigned)na, NTH, 0, stream>>>(tab, turn, poly);
  else
    apply<T, BF><<<(unsigned)na, NTH, 0, stream>>>(tab, poly);
  return st::check_launch("st_orthogonalize");
}

int check_table(int32_t n, const st_matrix_batch* table) {
  ST_CHECK_ARG(n >= 0 && (n == 0 || table), "st_orthogonalize: NULL table");
  for (int32_t i = 0; i < n; ++i) {
    const st_matrix_batch& b = table[i];
    ST_CHECK_ARG(b.count >= 0 && b.rows >= 0 && b.cols >= 0, "matrices %d: negative size", i);
    if (b.count == 0 || b.rows == 0 || b.cols == 0) continue;
    const int64_t r = b.rows < b.cols ? b.rows : b.cols, K = b.rows < b.cols ? b.cols : b.rows;
    if (r > MAXR)
      return st::fail(ST_EUNSUPPORTED, "matrices %d: the shorter side is %lld, at most %lld", i,
                      (long long)r, (long long)MAXR);
    if (K >= (int64_t)1 << 30 || b.count >= (int64_t)1 << 24)
      return st::fail(ST_EUNSUPPORTED, "matrices %d: a side of 2^30 or 2^24 matrices and more", i);
  }
  return ST_OK;
}
// The sizes of all tables, checked before the first launch, and their workspace.
int survey(int32_t n, const st_matrix_batch* table, int64_t& bytes) {
  const int rc = check_table(n, table);
  if (rc != ST_OK) return rc;
  int64_t most = 0;
  Plan p;
  for (int32_t at = 0; at < n;) {
    at += make_plan(table, n, at, ST_DTYPE_F32, p);
    if (p.tab.n && !p.whole && !fits(p))
      return st::fail(ST_EUNSUPPORTED, "too many matrices for a launch: call with fewer at a time");
    if (p.part + p.poly > most) most = p.part + p.poly;
  }
  bytes = most ? most * 8 + TABLE_BYTES : 0;
  return ST_OK;
}

}  // namespace

extern "C" int64_t st_orthogonalize_workspace_bytes(int32_t n, const st_matrix_batch* table) {
  int64_t bytes = 0;
  return survey(n, table, bytes) == ST_OK ? bytes : -1;
}

extern "C" int st_orthogonalize(int32_t n, const st_matrix_batch* table, int32_t dtype,
                                int32_t steps, double a, double b, double c, double eps,
                                void* workspace, int64_t workspace_bytes, st_stream_t stream) {
  int64_t need = 0;
  const int rc = survey(n, table, need);
  if (rc != ST_OK) return rc;
  ST_CHECK_ARG(dtype == ST_DTYPE_BF16 || dtype == ST_DTYPE_F32, "dtype codes are bf16 and fp32");
  ST_CHECK_ARG(std::isfinite(a) && std::isfinite(b) && std::isfinite(c) && std::isfinite(eps) &&
                   eps >= 0,
               "coefficients must be finite, eps not negative");
  ST_CHECK_ARG(steps >= 1 && steps <= 64 &&
                   2.0 * steps * std::log10(std::fabs(a) > 1.0 ? std::fabs(a) : 1.0) <= 13.0,
               "steps must be 1..64 with |a|^(2 steps) at most 1e13, got %d", steps);
  for (int32_t i = 0; i < n; ++i) {
    const st_matrix_batch& m = table[i];
    const uintptr_t mask = dtype == ST_DTYPE_BF16 ? 1 : 3;
    if (m.count == 0 || m.rows == 0 || m.cols == 0) continue;
    ST_CHECK_ARG(m.x && m.out, "matrices %d: NULL", i);
    ST_CHECK_ARG((((uintptr_t)m.x | (uintptr_t)m.out) & mask) == 0, "matrices %d: misaligned", i);
  }
  if (need > 0 && (!workspace || workspace_bytes < need))
    return st::fail(ST_EWORKSPACE, "st_orthogonalize needs %lld workspace bytes", (long long)need);
  ST_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
  Plan p;
  for (int32_t at = 0; at < n;) {
    at += make_plan(table, n, at, dtype, p);
    if (!p.tab.n) continue;
    p.tab.steps = steps, p.tab.a = a, p.tab.b = b, p.tab.c = c, p.tab.eps = eps;
    char* ws = (char*)workspace;
    const hipStream_t s = (hipStream_t)stream;
    const bool bf = dtype == ST_DTYPE_BF16;
    const int r = p.whole    ? (bf ? launch_whole<true>(p, s) : launch_whole<false>(p, s))
                  : p.T == 1 ? (bf ? launch<1, true>(p, ws, s) : launch<1, false>(p, ws, s))
                  : p.T == 2 ? (bf ? launch<2, true>(p, ws, s) : launch<2, false>(p, ws, s))
                             : (bf ? launch<4, true>(p, ws, s) : launch<4, false>(p, ws, s));
    if (r != ST_OK) return r;
  }
  return ST_OK;
}
