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
// (v_mfma_f64_16x16x4: 46 TFLOP/s measured, dependent ones 75 ns apart).  In 32 bits
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

#include "common.h"

namespace {

typedef double d4 __attribute__((ext_vector_type(4)));
constexpr int NTH = 256;
constexpr int MAXE = 60;        // entries of a launch's table (kernel arguments: 4 KB)
constexpr int64_t MAXR = 1024;  // short side

// A batch of equal matrices, back to back.
struct Entry {
  const void* x;
  void* out;
  int64_t part, poly;      // its first matrix's place in the two scratch areas (doubles)
  int32_t K, r, chunks;    // long and short side, chunks of the long side in gram
  int32_t tall;            // the short side is the contiguous one
  uint32_t tile0;          // its first workgroup in the present launch
  int32_t vec;             // rows may be read four elements at a time
};
struct Table {
  Entry e[MAXE];
  int32_t n, steps;
  int32_t CH, AL;  // long elements of a workgroup in gram and apply
  double a, b, c, eps;
};

__device__ __forceinline__ const Entry& find(const Table& t, uint32_t b) {
  int lo = 0, hi = t.n - 1;  // the last entry with tile0 <= b
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].tile0 <= b)
      lo = mid;
    else
      hi = mid - 1;
  }
  return t.e[lo];
}

template <bool BF>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (BF)
    return st::bf16_to_f32(((const uint16_t*)p)[i]);
  else
    return ((const float*)p)[i];
}
template <bool BF>
__device__ __forceinline__ void load4(const void* p, int64_t i, float* f) {
  if constexpr (BF) {
    const uint2 w = *(const uint2*)((const uint16_t*)p + i);
    f[0] = __uint_as_float(w.x << 16), f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16), f[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const float4 w = *(const float4*)((const float*)p + i);
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
__device__ __forceinline__ void store_upto4(void* p, int64_t i, int n, bool vec, const float* f) {
  if (vec && n >= 4) {
    if constexpr (BF)
      *(uint2*)((uint16_t*)p + i) =
          make_uint2(st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3]));
    else
      *(float4*)((float*)p + i) = make_float4(f[0], f[1], f[2], f[3]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) {
      if constexpr (BF)
        ((uint16_t*)p)[i + e] = st::f32_to_bf16(f[e]);
      else
        ((float*)p)[i + e] = f[e];
    }
}

// ---------------------------------------------------------------- G = U U'
// One workgroup: a chunk of the long side and one block pair (I <= J) of 16 T short
// rows each.  A wave takes 32 long elements at a time, of which lane group q holds
// eight: in a wide matrix 8q..8q+7 (128 contiguous bytes a row), in a tall one
// 4s + q, s = 0..7 (whole contiguous rows).  Which element is which k does not
// matter to a sum over all of them, as long as both operands agree.
template <bool BF, int T>
__device__ __forceinline__ void gram_rows(const Entry& e, const void* x, int row0, int64_t k0,
                                          int64_t kend, int lane, float (&u)[T][8]) {
  const int m = lane & 15, q = lane >> 4;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int i = row0 + 16 * t + m;
    if (i >= e.r) {
#pragma unroll
      for (int s = 0; s < 8; ++s) u[t][s] = 0.0f;
    } else if (e.tall) {
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const int64_t k = k0 + 4 * s + q;
        u[t][s] = k < kend ? load1<BF>(x, k * e.r + i) : 0.0f;
      }
    } else {
      const int64_t k = k0 + 8 * q;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t left = kend - k - 4 * h;
        load_upto4<BF>(x, (int64_t)i * e.K + k + 4 * h, (int)(left < 4 ? left : 4), e.vec,
                       u[t] + 4 * h);
      }
    }
  }
}

template <int T, bool BF>
__global__ __launch_bounds__(NTH) void gram(Table tab, double* __restrict__ part) {
  __shared__ double sum[T * T * 256];
  const Entry& e = find(tab, blockIdx.x);
  const int nb = T < 4 ? 1 : (e.r + 63) / 64, pairs = nb * (nb + 1) / 2;
  const uint32_t w = blockIdx.x - e.tile0;
  const int pair = (int)(w % pairs);
  const uint32_t mc = w / pairs;  // matrix * chunks + chunk
  const int64_t mat = mc / e.chunks, chunk = mc % e.chunks;
  int I = 0, J = pair;  // pairs row by row: (0,0..nb-1), (1,1..nb-1), ...
  while (J >= nb - I) J -= nb - I, ++I;
  J += I;
  const void* x = (const char*)e.x + mat * e.r * (int64_t)e.K * (BF ? 2 : 4);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t k1 = (chunk + 1) * tab.CH < e.K ? (chunk + 1) * tab.CH : e.K;
  const bool diag = I == J;
  d4 acc[T][T] = {};
  for (int64_t k0 = chunk * tab.CH + 32 * wave; k0 < k1; k0 += 128) {
    float a[T][8], b[T][8];
    gram_rows<BF, T>(e, x, I * 16 * T, k0, k1, lane, a);
    if (T == 4 && !diag) {
      gram_rows<BF, T>(e, x, J * 16 * T, k0, k1, lane, b);
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = 0; j < T; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)a[i][s], (double)b[j][s],
                                                             acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = i; j < T; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)a[i][s], (double)a[j][s],
                                                             acc[i][j], 0, 0, 0);
    }
  }
  // the waves' sums in their order, so that the result does not depend on the time
  for (int o = 0; o < NTH / 64; ++o) {
    if (wave == o) {
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int at = (i * T + j) * 256 + v * 64 + lane;
            sum[at] = o ? sum[at] + acc[i][j][v] : acc[i][j][v];
          }
    }
    __syncthreads();
  }
  double* to = part + e.part + ((int64_t)mc * pairs + pair) * (T * T * 256);
  for (int i = threadIdx.x; i < T * T * 256; i += NTH) to[i] = sum[i];
}

// Element (row, col) of G from the chunks' partial sums; tiles below a diagonal
// block's diagonal were not formed.
template <int T>
__device__ __forceinline__ double gram_at(const double* part, int chunks, int nb, int row, int col) {
  int bi = row / (16 * T), bj = col / (16 * T);
  if (bi > bj || (bi == bj && row / 16 > col / 16)) {
    const int s = row;
    row = col, col = s;
    bi = row / (16 * T), bj = col / (16 * T);
  }
  const int pair = bi * nb - bi * (bi - 1) / 2 + bj - bi, pairs = nb * (nb + 1) / 2;
  const int i = row / 16 % T, j = col / 16 % T, m = row % 16;
  const double* p = part + (int64_t)pair * (T * T * 256) + (i * T + j) * 256 + m / 4 * 64 +
                    m % 4 * 16 + col % 16;
  double s = 0.0;
  for (int c = 0; c < chunks; ++c) s += p[(int64_t)c * pairs * (T * T * 256)];
  return s;
}

// ---------------------------------------------------------------- P, r <= 64
// One workgroup of T waves a matrix, everything in LDS; wave w forms tile row w.
template <int T>
__device__ __forceinline__ void small_product(const double* A, const double* B, int w, int lane,
                                              d4 (&acc)[T]) {
  constexpr int R = 16 * T;
  const int m = lane & 15, q = lane >> 4;
#pragma unroll
  for (int j = 0; j < T; ++j) acc[j] = d4{0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int k = 0; k < R; k += 4) {
    const double a = A[(k + q) * R + 16 * w + m];  // A symmetric
#pragma unroll
    for (int j = 0; j < T; ++j)
      acc[j] = __builtin_amdgcn_mfma_f64_16x16x4f64(a, B[(k + q) * R + 16 * j + m], acc[j], 0, 0, 0);
  }
}
template <int T>
__device__ __forceinline__ void small_store(double* D, int w, int lane, const d4 (&acc)[T]) {
  constexpr int R = 16 * T;
#pragma unroll
  for (int j = 0; j < T; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v)
      D[(16 * w + 4 * v + (lane >> 4)) * R + 16 * j + (lane & 15)] = acc[j][v];
}

template <int T>
__global__ __launch_bounds__(64 * T) void poly_small(Table tab, const double* __restrict__ part,
                                                     double* __restrict__ poly) {
  constexpr int R = 16 * T, N = R * R;
  __shared__ double G[N], Q[N], P[N];
  const Entry& e = find(tab, blockIdx.x);
  const int64_t mat = blockIdx.x - e.tile0;
  const double* mine = part + e.part + mat * e.chunks * (T * T * 256);
  for (int i = threadIdx.x; i < N; i += 64 * T)
    G[i] = gram_at<T>(mine, e.chunks, 1, i / R, i % R);
  __syncthreads();
  double trace = 0.0;
  for (int i = 0; i < e.r; ++i) trace += G[i * R + i];
  __syncthreads();
  const double inv = 1.0 / (sqrt(trace) + tab.eps);
  for (int i = threadIdx.x; i < N; i += 64 * T) {
    G[i] = G[i] * inv * inv;
    P[i] = i / R == i % R ? inv : 0.0;
  }
  __syncthreads();
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int s = 0; s < tab.steps; ++s) {
    d4 x[T], h[T];
    small_product<T>(G, G, w, lane, x);
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int row = 16 * w + 4 * v + (lane >> 4), col = 16 * j + (lane & 15);
        Q[row * R + col] =
            tab.c * x[j][v] + tab.b * G[row * R + col] + (row == col ? tab.a : 0.0);
      }
    __syncthreads();
    small_product<T>(Q, P, w, lane, x);
    if (s + 1 < tab.steps) small_product<T>(Q, G, w, lane, h);
    __syncthreads();
    small_store<T>(P, w, lane, x);
    if (s + 1 < tab.steps) {
      small_store<T>(G, w, lane, h);  // Q G
      __syncthreads();
      small_product<T>(G, Q, w, lane, x);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < T; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int row = 16 * w + 4 * v + (lane >> 4), col = 16 * j + (lane & 15);
          if (row <= col) G[row * R + col] = G[col * R + row] = x[j][v];
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < N; i += 64 * T) poly[e.poly + mat * N + i] = P[i];
}

// ---------------------------------------------------------------- P, larger r
// The same in tiles of 32 x 32, a workgroup each, over matrices of R = 64 nb in
// scratch: G, Q, P (two, in turn) and H = Q G, one behind the other.
enum { SLOT_G, SLOT_Q, SLOT_P0, SLOT_P1, SLOT_H, SLOTS };

__global__ __launch_bounds__(NTH) void poly_sum(Table tab, const double* __restrict__ part,
                                                double* __restrict__ poly) {
  const Entry& e = find(tab, blockIdx.x);
  const int nb = (e.r + 63) / 64, R = 64 * nb;
  const uint32_t w = blockIdx.x - e.tile0, per = (uint32_t)R * R / 1024;
  const int64_t mat = w / per;
  const double* mine = part + e.part + mat * e.chunks * (nb * (nb + 1) / 2) * 4096;
  double* to = poly + e.poly + mat * SLOTS * R * R + (int64_t)SLOT_H * R * R;
  for (int i = threadIdx.x; i < 1024; i += NTH) {
    const int at = (int)(w % per) * 1024 + i;
    to[at] = gram_at<4>(mine, e.chunks, nb, at / R, at % R);
  }
}

__global__ __launch_bounds__(NTH) void poly_norm(Table tab, double* __restrict__ poly) {
  const Entry& e = find(tab, blockIdx.x);
  const int R = (e.r + 63) / 64 * 64;
  const uint32_t w = blockIdx.x - e.tile0, per = (uint32_t)R * R / 1024;
  double* base = poly + e.poly + (int64_t)(w / per) * SLOTS * R * R;
  const double* raw = base + (int64_t)SLOT_H * R * R;
  double trace = 0.0;
  for (int i = 0; i < e.r; ++i) trace += raw[(int64_t)i * R + i];
  const double inv = 1.0 / (sqrt(trace) + tab.eps);
  for (int i = threadIdx.x; i < 1024; i += NTH) {
    const int at = (int)(w % per) * 1024 + i;
    base[at] = raw[at] * inv * inv;  // SLOT_G
    base[(int64_t)SLOT_P0 * R * R + at] = at / R == at % R ? inv : 0.0;
  }
}

// mode 0: Q = aI + bG + cGG;  mode 1: P' = Q P and (blockIdx.y = 1) H = Q G;
// mode 2: G = H Q, its upper half in both places.
__global__ __launch_bounds__(NTH) void poly_step(Table tab, int mode, int turn,
                                                 double* __restrict__ poly) {
  __shared__ double As[64 * 32], Bs[64 * 32];
  const Entry& e = find(tab, blockIdx.x);
  const int R = (e.r + 63) / 64 * 64;
  const uint32_t w = blockIdx.x - e.tile0, per = (uint32_t)R * R / 1024;
  double* base = poly + e.poly + (int64_t)(w / per) * SLOTS * R * R;
  const int i0 = (int)(w % per) / (R / 32) * 32, j0 = (int)(w % per) % (R / 32) * 32;
  const int64_t RR = (int64_t)R * R;
  if (mode == 2 && i0 > j0) return;
  const int from = turn ? SLOT_P1 : SLOT_P0, into = turn ? SLOT_P0 : SLOT_P1;
  const bool h = mode == 1 && blockIdx.y == 1;
  const double* A = base + (mode == 0 ? SLOT_G : mode == 1 ? SLOT_Q : SLOT_H) * RR;
  const double* B = base + (mode == 0 || h ? SLOT_G : mode == 1 ? from : SLOT_Q) * RR;
  double* D = base + (mode == 0 ? SLOT_Q : h ? SLOT_H : mode == 1 ? into : SLOT_G) * RR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = lane & 15, q = lane >> 4, wi = 16 * (wave >> 1), wj = 16 * (wave & 1);
  d4 acc = {0.0, 0.0, 0.0, 0.0};
  for (int k0 = 0; k0 < R; k0 += 64) {
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 32; i += NTH) {
      const int64_t row = (int64_t)(k0 + i / 32) * R;
      As[i] = A[row + i0 + i % 32];  // A symmetric
      Bs[i] = B[row + j0 + i % 32];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 64; k += 4)
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64(As[(k + q) * 32 + wi + m], Bs[(k + q) * 32 + wj + m],
                                                 acc, 0, 0, 0);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int row = i0 + wi + 4 * v + q, col = j0 + wj + m;
    const int64_t at = (int64_t)row * R + col;
    if (mode == 2) {
      if (row <= col) D[at] = D[(int64_t)col * R + row] = acc[v];
    } else {
      D[at] = mode == 0 ? tab.c * acc[v] + tab.b * A[at] + (row == col ? tab.a : 0.0) : acc[v];
    }
  }
}

// ---------------------------------------------------------------- out = P U
// One workgroup: tab.AL long elements and one block of 16 T short rows; a wave
// takes 64 long elements at a time.  Wide: lane (m, q) reads four long elements
// 4m.. of short row 4t + q, which is B[k = 4t + q][j = m] of four products, and
// stores four long elements of rows 4v + q.  Tall: it reads the short elements
// 4q.. of long row m, so that step t's k is 4q + t, and with P's rows taken in the
// order 4 (m % 4) + m / 4 it holds the short elements 4q.. of that row again.
template <int T, bool BF>
__global__ __launch_bounds__(NTH) void apply(Table tab, int last, const double* __restrict__ poly) {
  constexpr int R16 = 16 * T;
  __shared__ double Ps[R16 * R16];
  const Entry& e = find(tab, blockIdx.x);
  const int nb = T < 4 ? 1 : (e.r + 63) / 64, R = R16 * nb;
  const uint32_t w = blockIdx.x - e.tile0, tiles = (uint32_t)((e.K + tab.AL - 1) / tab.AL);
  const int I = (int)(w % nb);
  const uint32_t mt = w / nb;
  const int64_t mat = mt / tiles, l0 = (int64_t)(mt % tiles) * tab.AL;
  const int64_t l1 = l0 + tab.AL < e.K ? l0 + tab.AL : e.K;
  const int64_t off = mat * e.r * (int64_t)e.K * (BF ? 2 : 4);
  const void* x = (const char*)e.x + off;
  void* out = (char*)e.out + off;
  const double* P = poly + e.poly;
  P += nb == 1 ? mat * R * R : (mat * SLOTS + (last ? SLOT_P1 : SLOT_P0)) * R * R;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
  const int prow = e.tall ? 4 * (m & 3) + (m >> 2) : m;
  for (int64_t step = l0; step < l1; step += 4 * 64) {
    const int64_t k0 = step + 64 * wave;  // a wave past the end loads nothing and stores nothing
    d4 acc[T][4] = {};
    for (int kb = 0; kb < nb; ++kb) {
      if (nb > 1 || step == l0) {
        __syncthreads();
        for (int i = threadIdx.x; i < R16 * R16; i += NTH)
          Ps[i] = P[(int64_t)(kb * R16 + i / R16) * R + I * R16 + i % R16];
        __syncthreads();
      }
      float u[T][4][4];  // wide: [kt][t][c], tall: [kt][c][t]
#pragma unroll
      for (int kt = 0; kt < T; ++kt)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (e.tall) {
            const int64_t k = k0 + 16 * t + m;
            const int i = kb * R16 + 16 * kt + 4 * q, left = k < l1 ? e.r - i : 0;
            load_upto4<BF>(x, k * e.r + i, left, e.vec, u[kt][t]);
          } else {
            const int i = kb * R16 + 16 * kt + 4 * t + q;
            const int64_t k = k0 + 4 * m, left = i < e.r ? l1 - k : 0;
            load_upto4<BF>(x, (int64_t)i * e.K + k, (int)(left < 4 ? left : 4), e.vec, u[kt][t]);
          }
        }
#pragma unroll
      for (int kt = 0; kt < T; ++kt)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int k = 16 * kt + (e.tall ? 4 * q + t : 4 * t + q);
          double b[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) b[c] = (double)(e.tall ? u[kt][c][t] : u[kt][t][c]);
#pragma unroll
          for (int i = 0; i < T; ++i) {
            const double a = Ps[k * R16 + 16 * i + prow];
#pragma unroll
            for (int c = 0; c < 4; ++c)
              acc[i][c] = __builtin_amdgcn_mfma_f64_16x16x4f64(a, b[c], acc[i][c], 0, 0, 0);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float f[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) f[n] = (float)(e.tall ? acc[i][s][n] : acc[i][n][s]);
        if (e.tall) {
          const int64_t k = k0 + 16 * s + m;
          const int row = I * R16 + 16 * i + 4 * q;
          store_upto4<BF>(out, k * e.r + row, k < l1 ? e.r - row : 0, e.vec, f);
        } else {
          const int row = I * R16 + 16 * i + 4 * s + q;
          const int64_t k = k0 + 4 * m, left = row < e.r ? l1 - k : 0;
          store_upto4<BF>(out, (int64_t)row * e.K + k, (int)(left < 4 ? left : 4), e.vec, f);
        }
      }
  }
}

// ---------------------------------------------------------------- host
struct Plan {  // one table's launches
  Table tab;
  int T = 1;
  int64_t count[MAXE];
  int64_t part = 0, poly = 0;  // doubles
};

int tiles_of(int64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : 4; }

// The next table: entries from `at` on whose short sides take tiles of one size and
// are either all within one block or all beyond it.  Returns the entries taken.
int make_plan(const st_matrix_batch* in, int32_t n, int32_t at, int32_t dtype, Plan& p) {
  p = Plan();
  Table& t = p.tab;
  int64_t total = 0;
  int taken = 0;
  bool large = false, first = true;
  t.n = 0;
  for (; at + taken < n && t.n < MAXE; ++taken) {
    const st_matrix_batch& b = in[at + taken];
    if (b.count == 0 || b.rows == 0 || b.cols == 0) continue;
    const int64_t r = b.rows < b.cols ? b.rows : b.cols, K = b.rows < b.cols ? b.cols : b.rows;
    if (first) p.T = tiles_of(r), large = r > 64, first = false;
    if (tiles_of(r) != p.T || (r > 64) != large) break;
    Entry& e = t.e[t.n];
    e.x = b.x, e.out = b.out;
    e.K = (int32_t)K, e.r = (int32_t)r, e.tall = b.rows > b.cols;
    const uintptr_t mask = dtype == ST_DTYPE_BF16 ? 7 : 15;
    e.vec = (e.tall ? r : K) % 4 == 0 && (((uintptr_t)b.x | (uintptr_t)b.out) & mask) == 0;
    p.count[t.n++] = b.count;
    total += b.count * K;
  }
  // Long elements of a workgroup: about 2048 workgroups where there is that much
  // work, never less than one round of its four waves.
  const int64_t ch = st::cdiv(total, 2048);
  t.CH = (int32_t)(st::cdiv(ch < 256 ? 256 : ch > 4096 ? 4096 : ch, 128) * 128);
  t.AL = (int32_t)(st::cdiv(ch < 256 ? 256 : ch > 2048 ? 2048 : ch, 256) * 256);
  for (int i = 0; i < t.n; ++i) {
    Entry& e = t.e[i];
    const int64_t nb = (e.r + 16 * p.T - 1) / (16 * p.T);
    e.chunks = (int32_t)st::cdiv(e.K, t.CH);
    e.part = p.part, e.poly = p.poly;
    p.part += p.count[i] * e.chunks * (nb * (nb + 1) / 2) * p.T * p.T * 256;
    const int64_t R = 16 * p.T * nb;
    p.poly += p.count[i] * R * R * (nb > 1 ? SLOTS : 1);
  }
  return taken;
}

// Numbers the workgroups of a launch; their count, or -1 beyond a launch's limit.
template <typename F>
int64_t number(Plan& p, F per_matrix) {
  int64_t at = 0;
  for (int i = 0; i < p.tab.n; ++i) {
    p.tab.e[i].tile0 = (uint32_t)at;
    at += p.count[i] * per_matrix(p.tab.e[i]);
    if (at * NTH >= (int64_t)1 << 32) return -1;
  }
  return at;
}

template <int T, bool BF>
int launch(Plan& p, double* part, double* poly, hipStream_t stream) {
  auto blocks = [](const Entry& e) { return T < 4 ? (int64_t)1 : ((int64_t)e.r + 63) / 64; };
  const bool large = T == 4 && p.tab.e[0].r > 64;
  auto tiles = [&](const Entry& e) { return blocks(e) * blocks(e) * 4; };
  const int64_t ng = number(p, [&](const Entry& e) {
    return e.chunks * blocks(e) * (blocks(e) + 1) / 2;
  });
  const int64_t np = ng < 0 ? -1 : number(p, [&](const Entry& e) { return large ? tiles(e) : 1; });
  const int64_t na = np < 0 ? -1 : number(p, [&](const Entry& e) {
    return st::cdiv(e.K, p.tab.AL) * blocks(e);
  });
  if (na < 0)
    return st::fail(ST_EUNSUPPORTED, "too many matrices for a launch: call with fewer at a time");
  number(p, [&](const Entry& e) { return e.chunks * blocks(e) * (blocks(e) + 1) / 2; });
  gram<T, BF><<<dim3((unsigned)ng), NTH, 0, stream>>>(p.tab, part);
  number(p, [&](const Entry& e) { return large ? tiles(e) : 1; });
  int turn = 0;
  if (!large) {
    poly_small<T><<<dim3((unsigned)np), 64 * T, 0, stream>>>(p.tab, part, poly);
  } else {
    poly_sum<<<dim3((unsigned)np), NTH, 0, stream>>>(p.tab, part, poly);
    poly_norm<<<dim3((unsigned)np), NTH, 0, stream>>>(p.tab, poly);
    for (int s = 0; s < p.tab.steps; ++s) {
      const bool more = s + 1 < p.tab.steps;
      poly_step<<<dim3((unsigned)np), NTH, 0, stream>>>(p.tab, 0, turn, poly);
      poly_step<<<dim3((unsigned)np, more ? 2 : 1), NTH, 0, stream>>>(p.tab, 1, turn, poly);
      if (more) poly_step<<<dim3((unsigned)np), NTH, 0, stream>>>(p.tab, 2, turn, poly);
      turn ^= 1;
    }
  }
  number(p, [&](const Entry& e) { return st::cdiv(e.K, p.tab.AL) * blocks(e); });
  apply<T, BF><<<dim3((unsigned)na), NTH, 0, stream>>>(p.tab, turn, poly);
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

}  // namespace

extern "C" int64_t st_orthogonalize_workspace_bytes(int32_t n, const st_matrix_batch* table) {
  if (check_table(n, table) != ST_OK) return 0;
  int64_t most = 0;
  Plan p;
  for (int32_t at = 0; at < n;) {
    at += make_plan(table, n, at, ST_DTYPE_F32, p);
    if (p.part + p.poly > most) most = p.part + p.poly;
  }
  return most * 8;
}

extern "C" int st_orthogonalize(int32_t n, const st_matrix_batch* table, int32_t dtype,
                                int32_t steps, double a, double b, double c, double eps,
                                void* workspace, int64_t workspace_bytes, st_stream_t stream) {
  const int rc = check_table(n, table);
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
  const int64_t need = st_orthogonalize_workspace_bytes(n, table);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return st::fail(ST_EWORKSPACE, "st_orthogonalize needs %lld workspace bytes", (long long)need);
  ST_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
  Plan p;
  for (int32_t at = 0; at < n;) {
    at += make_plan(table, n, at, dtype, p);
    if (!p.tab.n) continue;
    p.tab.steps = steps, p.tab.a = a, p.tab.b = b, p.tab.c = c, p.tab.eps = eps;
    double* part = (double*)workspace;
    double* poly = part + p.part;
    const hipStream_t s = (hipStream_t)stream;
    const bool bf = dtype == ST_DTYPE_BF16;
    const int r = p.T == 1 ? (bf ? launch<1, true>(p, part, poly, s) : launch<1, false>(p, part, poly, s))
                : p.T == 2 ? (bf ? launch<2, true>(p, part, poly, s) : launch<2, false>(p, part, poly, s))
                           : (bf ? launch<4, true>(p, part, poly, s) : launch<4, false>(p, part, poly, s));
    if (r != ST_OK) return r;
  }
  return ST_OK;
}
