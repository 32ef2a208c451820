// Attention in which query i of a row sees the keys [key_start[i], key_end[i]):
// packed documents, bidirectional runs inside them, sliding windows, padding
// (an empty run) -- and, optionally, scores capped by a tanh and a bias that
// falls with the distance.  Forward and deterministic backward.
//
//   x[i,j] = cap * tanh(scale * q_i.k_j / cap) - slope[h] * |i - j|
//   P[i,:] = softmax of x[i,:] over the seen keys,   o_i = sum_j P[i,j] v_j
//   dP = dO V^T,  delta_i = sum_j P dP = dO_i . o_i,  dx = P (dP - delta)
//   dS = dx * (1 - tanh^2),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Layout as the causal kernels (attention.hip): q [B,H,S,DQ], k [B,Hkv,S,DQ],
// v [B,Hkv,S,DV] head-major bf16, out and dout token-major [B,S,H*DV], lse
// [B,H,S] fp32 the base-2 log-sum-exp (+inf for a query that sees no key, so
// every probability recomputed from it is 0).  Scores, statistics and sums are
// fp32.  Probabilities are rounded to bf16 for their MFMA products, dS is split
// into two bf16 parts (2^-17): the second product reads no operand of its own
// and cost 3-7% of a pass.  delta from the rounded output is off by 2^-9 of
// |dO||o|, which counts where few keys share the weight, so a tile whose queries
// see at most SHORT keys in all sums P dP itself, in a sweep of its own before
// dQ's (for no tile, those, and every one: 544, 550 and 600 us a training pass of
// 2048 tokens and 128 heads of 192/128).  A query that sees one key has dS = 0,
// and gets exactly that.
//
// A plan (span_plan below, made once per mask) holds for each 32-query block
// the extremes of its runs, for each 128-key tile the query blocks that see it,
// and the tiles by falling work, so a workgroup walks only the tiles that some
// of its queries see and the long ones start first.
//
// Masked places never reach a result: a masked score is replaced, not added to,
// but an infinity or NaN in a key, value or gradient row that a 32-row block
// partly sees does meet a zero probability inside an MFMA product.  A workgroup
// in which a wave's sums are not finite therefore walks its tile once more
// (CAREFUL), with products in which a masked pair adds nothing whatever its rows
// hold (add_seen), and those waves' rows are taken from there.  What is not finite
// then is the answer.  A training pass of 4096 tokens in one document whose values
// are all NaN, 8/2 heads of 128: 2.5 ms, of finite ones 0.38 (rows summed pair by
// pair instead took 62 ms at 1024 tokens, 0.2 finite, and grew with their square).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_tile.h"

namespace {

using namespace attn;

constexpr int NT = 256;
constexpr int TILE = 128;  // queries (dQ, forward) or keys (dK, dV) per workgroup
constexpr int BKT = 64;    // keys per step of the forward and dQ passes
constexpr int QT = 64;     // queries per step of the dK/dV pass
constexpr int LEAD = 6;  // LDS reads ahead of the MFMAs (see fed)
constexpr int SHORT = 256;   // keys of a tile whose delta is summed from P dP
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_LOG2 = 8.0f;  // the running maximum may lag by up to 2^8

// ---------------------------------------------------------------- plan
// Int32 regions, in order: blocks int4 [B, nb] (least and greatest run start,
// least and greatest run end of 32 queries; an empty run makes the greatest
// start INT_MAX and the least end 0, so the block is never taken for wholly
// visible), key tiles int2 [B, nt] (first query block that sees the tile, end),
// query and key tiles [B*nt] by falling work, their work (keys of the tile's
// queries; query blocks of the tile's keys), the key tiles' sum (0 where the
// tiles were not sorted).
struct Plan {
  const int4* blk;
  const int2* keys;
  const int32_t *qorder, *korder;
  int32_t *qwork, *kwork, *ktotal;
  int nb, nt;
  int64_t bytes;
};
Plan plan_of(const void* base, int64_t B, int64_t S) {
  Plan p;
  const int64_t nb = st::cdiv(S, 32), nt = st::cdiv(S, TILE);
  int32_t* w = (int32_t*)base;
  p.nb = (int)nb;
  p.nt = (int)nt;
  p.blk = (const int4*)w;
  w += 4 * B * nb;
  p.keys = (const int2*)w;
  w += 2 * B * nt;
  p.qorder = w;
  w += B * nt;
  p.korder = w;
  w += B * nt;
  p.qwork = w;
  w += B * nt;
  p.kwork = w;
  w += B * nt;
  p.ktotal = w;
  w += 1;
  p.bytes = (char*)w - (char*)base;
  return p;
}

__device__ __forceinline__ int2 clamp_run(int2 r, int S) {
  const int a = min(max(r.x, 0), S), z = min(max(r.y, 0), S);
  return a < z ? make_int2(a, z) : make_int2(0, 0);
}
__device__ __forceinline__ int2 run_of(const int32_t* __restrict__ lo, const int32_t* __restrict__ hi,
                                       int64_t at, int S) {
  return clamp_run(make_int2(lo[at], hi[at]), S);
}

// one 32-lane half per block of 32 queries
__global__ __launch_bounds__(NT) void span_blocks(const int32_t* __restrict__ lo,
                                                  const int32_t* __restrict__ hi, int S, int nb,
                                                  int64_t total, int4* __restrict__ blk) {
  const int64_t id = ((int64_t)blockIdx.x * NT + threadIdx.x) >> 5;
  if (id >= total) return;
  const int64_t b = id / nb;
  const int i = (int)(id % nb) * 32 + (threadIdx.x & 31);
  int2 r = i < S ? run_of(lo, hi, b * S + i, S) : make_int2(0, 0);
  const bool some = r.x < r.y;
  int4 x = some ? make_int4(r.x, r.x, r.y, r.y) : make_int4(INT_MAX, INT_MAX, 0, 0);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    x.x = min(x.x, __shfl_xor(x.x, d));
    x.y = max(x.y, __shfl_xor(x.y, d));
    x.z = min(x.z, __shfl_xor(x.z, d));
    x.w = max(x.w, __shfl_xor(x.w, d));
  }
  if ((threadIdx.x & 31) == 0) blk[id] = x;
}

// per 128-row tile: the query blocks that see it as keys, and the work of both kinds
__global__ __launch_bounds__(64) void span_tiles(const int4* __restrict__ blk, int nb, int nt,
                                                 int2* __restrict__ keys, int32_t* __restrict__ qwork,
                                                 int32_t* __restrict__ kwork) {
  const int64_t t = blockIdx.x;
  const int64_t b = t / nt;
  const int k0 = (int)(t % nt) * TILE, lane = threadIdx.x;
  const int4* row = blk + b * nb;
  int first = INT_MAX, end = 0;
  for (int i = lane; i < nb; i += 64) {
    const int4 x = row[i];
    if (x.x < k0 + TILE && x.w > k0) {
      first = min(first, i);
      end = max(end, i + 1);
    }
  }
  const int q = (int)(t % nt) * 4 + lane;
  int a = INT_MAX, z = 0;
  if (lane < 4 && q < nb) {
    a = row[q].x;
    z = row[q].w;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    first = min(first, __shfl_xor(first, d));
    end = max(end, __shfl_xor(end, d));
    a = min(a, __shfl_xor(a, d));
    z = max(z, __shfl_xor(z, d));
  }
  if (lane == 0) {
    keys[t] = first < end ? make_int2(first, end) : make_int2(0, 0);
    kwork[t] = first < end ? end - first : 0;
    qwork[t] = a < z ? z - a : 0;
  }
}

// Tiles by falling work (ties by index): each counts those before it.  Training
// pass in us, in this order and in the tiles' own, heads of 128: 8192 tokens, 32/8
// heads, 16 equal documents 294 : 363, one document 2675 : 2799; 16384 tokens of 2
// documents, 16/2 heads, 3201 : 3593.  The count is quadratic, 1.1 ms for 16384
// tiles: more than SORT_LIMIT keep their own order, and no tile's group is split.
constexpr int64_t SORT_LIMIT = 16384;
__global__ __launch_bounds__(NT) void span_order(const int32_t* __restrict__ qwork,
                                                 const int32_t* __restrict__ kwork, int64_t n,
                                                 int32_t* __restrict__ qorder,
                                                 int32_t* __restrict__ korder,
                                                 int32_t* __restrict__ ktotal) {
  const bool keys = blockIdx.y != 0;
  const int32_t* w = keys ? kwork : qwork;
  int32_t* o = keys ? korder : qorder;
  const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (i >= n) return;
  if (n > SORT_LIMIT) {
    o[i] = (int32_t)i;
    if (keys && i == 0) *ktotal = 0;
    return;
  }
  const int mine = w[i];
  int64_t rank = 0, sum = 0;
  for (int64_t j = 0; j < n; ++j) {
    rank += w[j] > mine || (w[j] == mine && j < i);
    sum += w[j];
  }
  o[rank] = (int32_t)i;
  if (keys && i == 0) *ktotal = (int32_t)min(sum, (int64_t)INT_MAX);
}

// ---------------------------------------------------------------- shared
struct Args {
  const uint16_t *q, *k, *v;
  const int32_t *lo, *hi;
  const float* slopes;  // [H] or NULL
  Plan plan;
  int S, H, Hkv;
  float scale, sl2;          // scale, scale * log2(e)
  float cap_in, cap_out;     // with a cap: 2 log2(e) scale / cap, cap * log2(e)
  float cap_small, cap_r;    // |s| up to which score_small holds, scale / cap
  float cap_p[3];            // score_small's coefficients, in powers of y^2
  float cap_s[3];            // in powers of s^2; 0 where those leave fp32
};

// Workgroup head index -> head, so that the query heads of a KV head share an
// XCD (blocks go to the 8 XCDs in turn) and its L2 holds that KV head's rows
// (forward of 8192 packed tokens, 32/8 heads of 128: 88 us, by rising index 97).
__device__ __forceinline__ int head_of(int x, int H, int Hkv) {
  if (Hkv % 8) return x;
  const int group = H / Hkv, y = x / 8;
  return (x % 8 + 8 * (y / group)) * group + y % group;
}

// MODE: what is done to a score, CAP and BIAS
constexpr int CAP = 1, BIAS = 2;
// tanh(y) = y + y z P(z), z = y^2, for |y| <= 0.35: P by least squares on
// Chebyshev points, reweighted to level the relative error (4e-8).  Most capped
// scores are there, and the polynomial takes half of the time of the exponential
// and the reciprocal: the forward chooses it alone where a whole wave's are.
// In powers of s^2 it is one product shorter (SQUARES; 16384 tokens, window 4096:
// 1070 us against 1118), but s^2 and the coefficients can leave fp32 where the
// score does not (scale / cap below 1e-19 or far from 1 with an extreme scale).
template <bool SQUARES>
__device__ __forceinline__ float score_small(const Args& a, float s) {
  const float y = SQUARES ? s : s * a.cap_r, z = y * y;
  const float* c = SQUARES ? a.cap_s : a.cap_p;
  float p = __builtin_fmaf(c[2], z, c[1]);
  p = __builtin_fmaf(p, z, c[0]);
  return s * __builtin_fmaf(p, z, a.sl2);
}

// Base-2 score of a raw product s at distance `far` (>= 0); `grad`: d x / d (scale s).
template <int MODE>
__device__ __forceinline__ float score(const Args& a, float slope2, float s, float far, float& grad) {
  grad = 1.0f;
  float x = s * a.sl2;
  if constexpr ((MODE & CAP) != 0) {
    // tanh(y) = 1 - 2 r, r = 1 / (1 + e^2y); absolute error of a few 2^-24, which a
    // large cap would multiply: small scores take the polynomial
    const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * a.cap_in));
    const float far_out = __builtin_fmaf(-2.0f * a.cap_out, r, a.cap_out);
    x = fabsf(s) <= a.cap_small ? score_small<false>(a, s) : far_out;
    grad = 4.0f * r * (1.0f - r);
  }
  if constexpr ((MODE & BIAS) != 0) x = __builtin_fmaf(-slope2, far, x);
  return x;
}
// Instruction order of a run of MFMAs fed from LDS: LEAD reads ahead, then PER
// after each MFMA.  Left alone the compiler reads an operand just before its use
// and every pair of MFMAs waits for the LDS (a training pass of 8192 packed tokens
// 479 us against 461; 192/128 heads 553 against 534; 3 or 9 ahead as 6).
template <int READS, int MFMAS, int LEAD, int PER>
__device__ __forceinline__ void fed() {
  __builtin_amdgcn_sched_group_barrier(0x100, LEAD, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (LEAD + i * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
  }
}

__device__ __forceinline__ bool finite(float x) { return x - x == 0.0f; }
// the greater of this lane's value and of the lane's 32 on or back
__device__ __forceinline__ float half_max(float x) {
  // the swap leaves the lower half's values in both halves of r[0], the upper's in r[1]
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// 0 if every value is finite
template <int N>
__device__ __forceinline__ float probe_of(const f32x16 (&acc)[N]) {
  float p = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) p = __builtin_fmaf(acc[i][v], 0.0f, p);
  return p;
}
// eight fp32 values as bf16 `hi` and what the rounding left as bf16 `lo`
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8& hi, bf16x8& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = st::pack_bf16x2(x[2 * e], x[2 * e + 1]);
    l[e] = st::pack_bf16x2(x[2 * e] - __uint_as_float(h[e] << 16),
                           x[2 * e + 1] - __uint_as_float(h[e] & 0xffff0000u));
  }
  hi = as_bf16x8(make_uint4(h[0], h[1], h[2], h[3]));
  lo = as_bf16x8(make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ bf16x8 pack8(const float (&x)[8]) {
  return as_bf16x8(make_uint4(st::pack_bf16x2(x[0], x[1]), st::pack_bf16x2(x[2], x[3]),
                              st::pack_bf16x2(x[4], x[5]), st::pack_bf16x2(x[6], x[7])));
}

// copies of the K and V tiles of a step, as RowCopy lays them out
template <int D, int NTHR, int ROWS>
struct TileCopy {
  using C = RowCopy<D, NTHR>;
  static constexpr int PER = ROWS * D / 8 / NTHR;
  static_assert(PER * NTHR * 8 == ROWS * D, "tiles are whole thread copies");
  uint32_t off[C::uniform ? 1 : PER];
  __device__ __forceinline__ TileCopy(int tid, int64_t ld) {
#pragma unroll
    for (int i = 0; i < (C::uniform ? 1 : PER); ++i) {
      const int P = i * NTHR + tid, row = P / (D / 8);
      off[i] = (uint32_t)(row * ld + ((P % (D / 8)) ^ swz<D>(row)) * 8) * 2;
    }
  }
  // rows [r0, r0 + ROWS) of a [n][ld] matrix at `base` (rows past n read zeros)
  __device__ __forceinline__ void operator()(const uint16_t* base, int64_t ld, int r0, int n,
                                             uint16_t* tile, int wave) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = r0 + (C::uniform ? i * C::rows : 0);
      const int left = min(max(n - r, 0), C::uniform ? C::rows : ROWS);
      const int64_t bytes = left > 0 ? ((left - 1) * ld + D) * 2 : 0;
      b2lds16(st::make_rsrc(base + (int64_t)r * ld, bytes), off[C::uniform ? 0 : i],
              tile + (i * NTHR + wave * 64) * 8);
    }
  }
};

// O^T or dQ^T accumulators of a wave's 32 queries -> rows of `out` (row stride
// ld) through the wave's own LDS space; rows for which `keep` is false get zeros
template <int D>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[D / 32], float mul, bool keep,
                                           uint16_t* os, int lane, int rows, uint16_t* out,
                                           int64_t ld) {
  constexpr int LDO = D + 8;
  const int g = lane >> 5, c = lane & 31;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int v4 = 0; v4 < 4; ++v4) {
      const int d = db * 32 + v4 * 8 + g * 4;
      u32x2 w = {st::pack_bf16x2(acc[db][4 * v4] * mul, acc[db][4 * v4 + 1] * mul),
                 st::pack_bf16x2(acc[db][4 * v4 + 2] * mul, acc[db][4 * v4 + 3] * mul)};
      if (!keep) w = u32x2{0, 0};
      *(u32x2*)(os + c * LDO + d) = w;
    }
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_wave_barrier();  // each wave reads back only its own rows
  for (int i = lane; i < 32 * (D / 8); i += 64) {
    const int r = i / (D / 8), ch = i % (D / 8);
    if (r < rows) {
      const u32x2 a = *(const u32x2*)(os + r * LDO + ch * 8);
      const u32x2 b = *(const u32x2*)(os + r * LDO + ch * 8 + 4);
      *(uint4*)(out + r * ld + ch * 8) = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
}

// a value that every lane of the wave holds alike, in scalar registers
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A value at a wave-uniform address that no one writes during the kernel, by a
// scalar load: a vector load behind the tile copies would wait for all of them.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
  typedef const __attribute__((address_space(4))) T* sp;
  return *(sp)(uintptr_t)p;
}

// LDS values that no copy in flight writes (as read_row's tiles)
__device__ __forceinline__ float4 lds4(const float* __restrict__ p) { return *(const float4*)p; }
template <typename T>
__device__ __forceinline__ T lds1(const T* __restrict__ p) {
  return *p;
}

// the same in fp32 (`os`: 32 rows of D + 4 floats)
template <int D>
__device__ __forceinline__ void store_rows_f32(const f32x16 (&acc)[D / 32], float mul, float* os,
                                               int lane, int rows, float* out) {
  constexpr int LDO = D + 4;
  const int g = lane >> 5, c = lane & 31;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int v4 = 0; v4 < 4; ++v4)
      *(float4*)(os + c * LDO + db * 32 + v4 * 8 + g * 4) =
          make_float4(acc[db][4 * v4] * mul, acc[db][4 * v4 + 1] * mul, acc[db][4 * v4 + 2] * mul,
                      acc[db][4 * v4 + 3] * mul);
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_wave_barrier();
  for (int i = lane; i < 32 * (D / 4); i += 64) {
    const int r = i / (D / 4), ch = i % (D / 4);
    if (r < rows) *(float4*)(out + r * D + ch * 4) = *(const float4*)(os + r * LDO + ch * 4);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int4 extremes(const int4* p) {
  typedef int i4 __attribute__((ext_vector_type(4)));
  const i4 x = scalar_load((const i4*)p);
  return make_int4(x.x, x.y, x.z, x.w);
}

// Key range of a 128-query tile and the wave's own block of extremes.
struct Walk {
  int4 mine;       // of this wave's 32 queries
  int first, end;  // keys that some query of the tile sees
};
__device__ __forceinline__ Walk walk_of(const Plan& p, int b, int qt, int wave) {
  Walk w{make_int4(INT_MAX, INT_MAX, 0, 0), INT_MAX, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = qt * 4 + i;
    if (n >= p.nb) break;
    const int4 x = extremes(p.blk + (int64_t)b * p.nb + n);
    w.first = min(w.first, x.x);
    w.end = max(w.end, x.w);
    if (i == wave) w.mine = x;
  }
  return w;
}

// ---------------------------------------------------------------- careful pass
// whether any wave of the workgroup says so; `flags`: LDS that no wave needs
template <int NTH>
__device__ __forceinline__ bool any_wave(bool x, int* flags) {
  __syncthreads();
  if ((threadIdx.x & 63) == 0) flags[threadIdx.x >> 6] = x;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < NTH / 64; ++w) any |= flags[w];
  __syncthreads();
  return uniform(any) != 0;
}
// The careful pass reads its arguments and forms its indexes again: kept from the
// first one they would take registers through its loop (a training pass of 8192
// packed tokens 514 us against 477).
template <typename T>  // T: the kernel's only argument
__device__ __forceinline__ T arguments_again() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const T*)p;
}
template <bool AGAIN>
__device__ __forceinline__ int block_index() {
  int x = blockIdx.x;
  if constexpr (AGAIN) asm volatile("" : "+s"(x));
  return x;
}
template <bool AGAIN>
__device__ __forceinline__ int thread_index() {
  int x = threadIdx.x;
  if constexpr (AGAIN) asm volatile("" : "+v"(x));
  return x;
}
// a lane's rows of an operand in registers, or read again at each use
template <int N, bool AGAIN>
struct Rows {
  bf16x8 held[AGAIN || N == 0 ? 1 : N];
  const uint16_t* at;  // NULL: zeros
  __device__ __forceinline__ bf16x8 read(int s) const {
    return as_bf16x8(at ? ld_global16(at + 16 * s) : make_uint4(0, 0, 0, 0));
  }
  __device__ __forceinline__ explicit Rows(const uint16_t* p) : at(p) {
    if constexpr (!AGAIN)
#pragma unroll
      for (int s = 0; s < N; ++s) held[s] = read(s);
  }
  __device__ __forceinline__ void forget() {  // or the reads would leave the loop
    if constexpr (AGAIN) asm volatile("" : "+v"(at));
  }
  __device__ __forceinline__ bf16x8 operator[](int s) const {
    if constexpr (AGAIN) return read(s);
    else return held[s];
  }
};

// acc += A B over the seen pairs of a block, where A's rows may hold infinities and
// NaN; B's weights of masked pairs are 0.  The infinities and NaN are taken out of
// A, so a masked pair adds 0, and what they make of a sum is found by a second
// product: of their kind (+inf 1, -inf 2^10, NaN 2^20) with 1 for a seen pair,
// 2^20 for one of weight 0 (0 * inf), 0 for a masked one.  At most 64 pairs meet,
// so the kinds do not run into each other.
constexpr uint32_t ONE = 0x3f80, NEG = 0x4480, NAN20 = 0x4980;  // bf16 1, 2^10, 2^20
__device__ __forceinline__ void part_kinds(bf16x8 x, bf16x8& rest, bf16x8& kind) {
  uint4 w = __builtin_bit_cast(uint4, x), k;
  auto one = [](uint32_t& v, uint32_t& to) {
    auto half = [](uint32_t h) {
      return (h & 0x7f80) != 0x7f80 ? 0u : (h & 0x7f) ? NAN20 : (h & 0x8000) ? NEG : ONE;
    };
    const uint32_t lo = half(v & 0xffff), hi = half(v >> 16);
    to = lo | hi << 16;
    v &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
  };
  one(w.x, k.x);
  one(w.y, k.y);
  one(w.z, k.z);
  one(w.w, k.w);
  rest = as_bf16x8(w);
  kind = as_bf16x8(k);
}
// The pairs of a lane: bit i of `seen`, and of `none` where the weight is 0.
struct Pairs {
  uint32_t seen = 0, none = 0;
  __device__ __forceinline__ void put(int i, bool sees, float weight) {
    seen |= sees ? 1u << i : 0u;
    none |= weight == 0.0f ? 1u << i : 0u;
    asm volatile("" : "+v"(seen), "+v"(none));  // or every pair keeps two lane masks
  }
  // what pairs 8 i .. 8 i + 7 say to the second product
  __device__ __forceinline__ bf16x8 kinds(int i) const {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      auto half = [&](int bit) { return !(seen >> bit & 1) ? 0u : none >> bit & 1 ? NAN20 : ONE; };
      w[e] = half(8 * i + 2 * e) | half(8 * i + 2 * e + 1) << 16;
    }
    return as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
  }
};
__device__ __forceinline__ float of_kinds(float c) {
  const float nan = __uint_as_float(0x7fc00000u);
  const bool neg = c >= 1024.0f, pos = c - 1024.0f * floorf(c * (1.0f / 1024.0f)) > 0.0f;
  return c >= 1048576.0f || (neg && pos) ? nan : neg ? -INFINITY : pos ? INFINITY : 0.0f;
}
// N steps of 16 rows: a(i) the A operand of step i, b and lo its weights in one or
// two parts
template <int N, bool TWO, typename F>
__device__ __forceinline__ void add_seen(f32x16& acc, F&& a, const bf16x8 (&b)[N], const bf16x8 (&lo)[N],
                                         const Pairs& pairs) {
  f32x16 count;
#pragma unroll
  for (int e = 0; e < 16; ++e) count[e] = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    bf16x8 rest, kind;
    part_kinds(a(i), rest, kind);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rest, b[i], acc, 0, 0, 0);
    if constexpr (TWO) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rest, lo[i], acc, 0, 0, 0);
    count = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kind, pairs.kinds(i), count, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);  // one at a time: the first pass needs the registers
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] += of_kinds(count[e]);
  __builtin_amdgcn_sched_barrier(0);
}

// ---------------------------------------------------------------- forward
// 4 waves of 32 queries over steps of 64 keys from the first key that the tile
// sees; K and V tiles [key][D] in LDS, two buffers, one barrier a step.  Every
// MFMA tile is S^T = K Q^T (a lane owns a query column), O^T += V^T P^T with
// V^T read by the transposing LDS loads.  Two waves a SIMD: one's exponentials run
// under the other's MFMAs.  Bound by that overlap: the MFMA pipes are busy 38% of
// the time, the vector units 43%, LDS without conflicts in the loop.  8192 packed
// tokens (7 documents, 32/8 heads of 128): 88 us, 0.73 PFLOP/s of what the runs
// need; 16384 tokens, window 4096, capped: 1068 us, 0.90 PFLOP/s; 2048 tokens and
// 128 heads of 192/128: 98 us, 0.50 PFLOP/s.
// Returns whether the wave's sums are not finite (its rows are then not stored);
// the careful pass stores the rows of waves with `again`.
template <int DQ, int DV, int MODE, bool CAREFUL>
__device__ __forceinline__ bool fwd_pass(const Args& a, uint16_t* lds, bool again,
                                         uint16_t* __restrict__ out, float* __restrict__ lse) {
  constexpr int DS = DQ / 16, DB = DV / 32, LK = BKT * DQ, LV = BKT * DV;
  static_assert(4 * 32 * (DV + 8) <= 2 * (LK + LV), "output staging fits");
  const int S = a.S, H = a.H, block = block_index<CAREFUL>();
  const int id = uniform(a.plan.qorder[block / H]), h = head_of(block % H, H, a.Hkv);
  const int b = id / a.plan.nt, qt = id % a.plan.nt;
  const int tid = thread_index<CAREFUL>(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, c = lane & 31, hk = h / (H / a.Hkv);
  const uint16_t* qb = a.q + (int64_t)(b * H + h) * S * DQ;
  const uint16_t* kb = a.k + (int64_t)(b * a.Hkv + hk) * S * DQ;
  const uint16_t* vb = a.v + (int64_t)(b * a.Hkv + hk) * S * DV;
  const int q0 = qt * TILE + wave * 32, myq = q0 + c;
  const Walk w = walk_of(a.plan, b, qt, wave);
  const int2 run = myq < S ? run_of(a.lo, a.hi, (int64_t)b * S + myq, S) : make_int2(0, 0);
  const float slope2 = (MODE & BIAS) ? a.slopes[h] * LOG2E : 0.0f;

  Rows<DS, CAREFUL> qf(myq < S ? qb + (int64_t)myq * DQ + 8 * g : nullptr);
  f32x16 oacc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) oacc[i][v] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  const uint32_t lr = lane_row<DQ>(c, g), lt = lane_tr<DV>(lane);

  const TileCopy<DQ, NT, BKT> ck(tid, DQ);
  const TileCopy<DV, NT, BKT> cv(tid, DV);
  auto issue = [&](int k0, int buf) {
    uint16_t* ks = lds + buf * (LK + LV);
    ck(kb, DQ, k0, S, ks, wave);
    cv(vb, DV, k0, S, ks + LK, wave);
  };
  if (w.first < w.end) issue(w.first, 0);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  // the buffer is a constant of each half of the unrolled loop: LDS addresses
  // are then a lane's own and an offset within the instruction
  auto step = [&](int k0, auto which) {
    const int buf = which;
    if (k0 + BKT < w.end) issue(k0 + BKT, buf ^ 1);
    const uint16_t* ks = lds + buf * (LK + LV);
    const uint16_t* vs = ks + LK;
    if (k0 < w.mine.w && k0 + BKT > w.mine.x) {  // some query of the wave sees some key
      const bool edge = CAREFUL || k0 < w.mine.y || k0 + BKT > w.mine.z;  // wave-uniform
      qf.forget();
      f32x16 sacc[2];
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int v = 0; v < 16; ++v) sacc[jb][v] = 0.0f;
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
          sacc[jb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_row<DQ>(ks, lr, jb * 32, s),
                                                             qf[s], sacc[jb], 0, 0, 0);
      if constexpr (!CAREFUL) fed<2 * DS, 2 * DS, LEAD, 1>();
      if constexpr (CAREFUL && MODE == 0) {
        // rounded before the maximum is taken off: of scores beyond 2^31 a fused
        // product would leave more than an exponent holds
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int v = 0; v < 16; ++v) sacc[jb][v] *= a.sl2;
      }
      if constexpr ((MODE & CAP) != 0) {
        float top = 0.0f;
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int v = 0; v < 16; ++v) top = fmaxf(top, fabsf(sacc[jb][v]));
        // (a NaN product passes either way: both forms keep it)
        auto all = [&](auto squares) {
#pragma unroll
          for (int jb = 0; jb < 2; ++jb)
#pragma unroll
            for (int v = 0; v < 16; ++v)
              sacc[jb][v] = score_small<decltype(squares)::value>(a, sacc[jb][v]);
        };
        if (__ballot(top > a.cap_small) == 0) {
          if (a.cap_s[2] != 0.0f)
            all(std::true_type{});
          else
            all(std::false_type{});
        } else {
#pragma unroll
          for (int jb = 0; jb < 2; ++jb)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              float grad;
              sacc[jb][v] = score<CAP>(a, 0.0f, sacc[jb][v], 0.0f, grad);
            }
        }
      }
      if constexpr ((MODE & BIAS) != 0) {
        const float far0 = (float)(myq - k0 - 4 * g);
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float x = (MODE & CAP) ? sacc[jb][v] : sacc[jb][v] * a.sl2;
            sacc[jb][v] = __builtin_fmaf(
                -slope2, fabsf(far0 - (float)(jb * 32 + (v >> 2) * 8 + (v & 3))), x);
          }
      }
      if (edge) {
        const int base = run.x - k0 - 4 * g;
        const unsigned width = (unsigned)(run.y - run.x);
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            sacc[jb][v] = (unsigned)(jb * 32 + (v >> 2) * 8 + (v & 3) - base) < width
                              ? sacc[jb][v] : -INFINITY;
      }
      const float mul = MODE || CAREFUL ? 1.0f : a.sl2;
      float mt = sacc[0][0];
#pragma unroll
      for (int jb = 0; jb < 2; ++jb)
#pragma unroll
        for (int v = 0; v < 16; ++v) mt = fmaxf(mt, sacc[jb][v]);
      mt = half_max(mt) * mul;
      if (__ballot(mt > m_run + RESCALE_LOG2)) {
        const float m_new = fmaxf(m_run, mt);
        // a row with no key yet: -inf - -inf is not a number, its sums are 0
        const float alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) oacc[i][v] *= alpha;
        l_run *= alpha;
        m_run = m_new;
      }
      const float m_use = m_run == -INFINITY ? 0.0f : m_run;
      bf16x8 pf[4];
      Pairs pairs;  // of the careful pass
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(
              __builtin_fmaf(sacc[cc >> 1][8 * (cc & 1) + e], mul, -m_use));
          l_run += p[e];
          if constexpr (CAREFUL) {
            const int v = 8 * (cc & 1) + e, key = k0 + (cc >> 1) * 32 + (v >> 2) * 8 + (v & 3) + 4 * g;
            pairs.put(8 * cc + e, key >= run.x && key < run.y, p[e]);
          }
        }
        pf[cc] = as_bf16x8(make_uint4(st::pack_bf16x2(p[0], p[1]), st::pack_bf16x2(p[2], p[3]),
                                      st::pack_bf16x2(p[4], p[5]), st::pack_bf16x2(p[6], p[7])));
      }
      if constexpr (CAREFUL) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
          add_seen<4, false>(oacc[db], [&](int cc) { return read_tr<DV>(vs, lt, cc * 16, db); }, pf, pf,
                             pairs);
      } else {
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
          for (int db = 0; db < DB; ++db)
            oacc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_tr<DV>(vs, lt, cc * 16, db), pf[cc],
                                                               oacc[db], 0, 0, 0);
        fed<8 * DB, 4 * DB, 2 * LEAD, 2>();
      }
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  if constexpr (CAREFUL) {
    int buf = 0;
#pragma unroll 1
    for (int k0 = w.first; k0 < w.end; k0 += BKT, buf ^= 1) step(k0, buf);
  } else {
#pragma unroll 1
    for (int k0 = w.first; k0 < w.end; k0 += 2 * BKT) {
      step(k0, std::integral_constant<int, 0>{});
      if (k0 + BKT < w.end) step(k0 + BKT, std::integral_constant<int, 1>{});
    }
  }

  const float l_tot = l_run + __shfl_xor(l_run, 32);
  const bool some = run.x < run.y;
  bool bad = false;
  if constexpr (!CAREFUL)
    bad = __ballot(some && !(probe_of(oacc) == 0.0f && finite(l_tot) && l_tot > 0.0f)) != 0;
  if (CAREFUL ? again : !bad) {
    if (g == 0 && myq < S)
      lse[(int64_t)(b * H + h) * S + myq] = some ? m_run + log2f(l_tot) : INFINITY;
    store_rows<DV>(oacc, 1.0f / l_tot, some, lds + wave * 32 * (DV + 8), lane, S - q0,
                   out + ((int64_t)b * S + q0) * H * DV + (int64_t)h * DV, (int64_t)H * DV);
  }
  return bad;
}

// (heads of 64 without a cap: the first pass runs four waves a SIMD, 72 us for 8192
// packed tokens of 32/8 heads; with the registers that the careful one would like,
// three and 77.)
struct FwdCall {
  Args a;
  uint16_t* out;
  float* lse;
};
template <int DQ, int DV, int MODE>
__global__ __launch_bounds__(NT, DQ == 64 && !(MODE & CAP) ? 4 : 2) void span_fwd(FwdCall c) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * BKT * (DQ + DV)];
  const bool bad = fwd_pass<DQ, DV, MODE, false>(c.a, lds, false, c.out, c.lse);
  if (!any_wave<NT>(bad, (int*)lds)) return;
  const FwdCall d = arguments_again<FwdCall>();
  fwd_pass<DQ, DV, MODE, true>(d.a, lds, bad, d.out, d.lse);
}

// ---------------------------------------------------------------- backward
// dQ (and delta) of a 128-query tile: S^T and dP^T = V dO^T as in the forward,
// dQ^T += K^T dS^T.  Bound as the forward (MFMA pipes 44% busy): 174 us in a
// trace, 0.55 PFLOP/s, at its 8192 packed tokens, 191 us at its heads of 192/128.
// Unrolled by two steps as the forward is, it spilled (495 us a training pass
// against 467).
template <int DQ, int DV, int MODE, bool CAREFUL>
__device__ __forceinline__ bool dq_pass(const Args& a, uint16_t* lds, bool again,
                                        const uint16_t* __restrict__ o,
                                        const uint16_t* __restrict__ dout,
                                        const float* __restrict__ lse, float* __restrict__ delta,
                                        uint16_t* __restrict__ dq) {
  constexpr int DSQ = DQ / 16, DSV = DV / 16, DB = DQ / 32, LK = BKT * DQ, LV = BKT * DV;
  static_assert(4 * 32 * (DQ + 8) <= 2 * (LK + LV), "output staging fits");
  const int S = a.S, H = a.H, block = block_index<CAREFUL>();
  const int id = uniform(a.plan.qorder[block / H]), h = head_of(block % H, H, a.Hkv);
  const int b = id / a.plan.nt, qt = id % a.plan.nt;
  const int tid = thread_index<CAREFUL>(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, c = lane & 31, hk = h / (H / a.Hkv);
  const int64_t ldt = (int64_t)H * DV;
  const uint16_t* qb = a.q + (int64_t)(b * H + h) * S * DQ;
  const uint16_t* kb = a.k + (int64_t)(b * a.Hkv + hk) * S * DQ;
  const uint16_t* vb = a.v + (int64_t)(b * a.Hkv + hk) * S * DV;
  const int q0 = qt * TILE + wave * 32, myq = q0 + c;
  const bool qok = myq < S;
  const Walk w = walk_of(a.plan, b, qt, wave);
  const int2 run = qok ? run_of(a.lo, a.hi, (int64_t)b * S + myq, S) : make_int2(0, 0);
  const float slope2 = (MODE & BIAS) ? a.slopes[h] * LOG2E : 0.0f;
  const int64_t srow = (int64_t)(b * H + h) * S;
  const int64_t trow = ((int64_t)b * S + myq) * ldt + (int64_t)h * DV;

  Rows<DSQ, CAREFUL> qf(qok ? qb + (int64_t)myq * DQ + 8 * g : nullptr);
  Rows<DSV, CAREFUL> dof(qok ? dout + trow + 8 * g : nullptr);
  const bool shortrow = w.end - w.first <= SHORT;  // uniform over the workgroup
  float dl = 0.0f;
#pragma unroll
  for (int s = 0; s < DSV; ++s) {
    if (shortrow) continue;
    const uint4 gv = __builtin_bit_cast(uint4, dof[s]);
    const uint4 ov = qok ? ld_global16(o + trow + 16 * s + 8 * g) : make_uint4(0, 0, 0, 0);
    const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w}, ow[4] = {ov.x, ov.y, ov.z, ov.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      dl += st::bf16_to_f32((uint16_t)(gw[e >> 1] >> (16 * (e & 1)))) *
            st::bf16_to_f32((uint16_t)(ow[e >> 1] >> (16 * (e & 1))));
  }
  dl += __shfl_xor(dl, 32);
  const float lq = qok ? lse[srow + myq] : INFINITY;
  const uint32_t lrq = lane_row<DQ>(c, g), lrv = lane_row<DV>(c, g), lt = lane_tr<DQ>(lane);

  f32x16 dqacc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dqacc[i][e] = 0.0f;

  const TileCopy<DQ, NT, BKT> ck(tid, DQ);
  const TileCopy<DV, NT, BKT> cv(tid, DV);
  auto issue = [&](int k0, int buf) {
    uint16_t* ks = lds + buf * (LK + LV);
    ck(kb, DQ, k0, S, ks, wave);
    cv(vb, DV, k0, S, ks + LK, wave);
  };
  if (w.first < w.end) issue(w.first, 0);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  int buf = 0;
#pragma unroll 1
  for (int sweep = shortrow ? 0 : 1; sweep < 2; ++sweep) {
  const bool only_delta = sweep == 0;
#pragma unroll 1
  for (int k0 = w.first; k0 < w.end; k0 += BKT, buf ^= 1) {
    if (k0 + BKT < w.end)
      issue(k0 + BKT, buf ^ 1);
    else if (only_delta)
      issue(w.first, buf ^ 1);
    const uint16_t* ks = lds + buf * (LK + LV);
    const uint16_t* vs = ks + LK;
#pragma unroll
    for (int jb = 0; jb < 2; ++jb) {
      const int kb0 = k0 + jb * 32;
      if (kb0 >= w.mine.w || kb0 + 32 <= w.mine.x) continue;  // wave-uniform
      const bool edge = CAREFUL || kb0 < w.mine.y || kb0 + 32 > w.mine.z;
      // an edge keeps the offsets of the lane's run (of more than one key, or
      // dS is 0), other blocks keep all
      const int base = edge ? run.x - kb0 - 4 * g : 0;
      const unsigned width = edge ? (run.y - run.x > 1 ? (unsigned)(run.y - run.x) : 0u) : 32u;
      const float far0 = (float)(myq - kb0 - 4 * g);
      f32x16 sacc, pacc;
#pragma unroll
      for (int e = 0; e < 16; ++e) { sacc[e] = 0.0f; pacc[e] = 0.0f; }
      qf.forget();
      dof.forget();
#pragma unroll
      for (int s = 0; s < DSQ; ++s) {
        sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_row<DQ>(ks, lrq, jb * 32, s), qf[s],
                                                       sacc, 0, 0, 0);
        if (s < DSV)
          pacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_row<DV>(vs, lrv, jb * 32, s),
                                                         dof[s], pacc, 0, 0, 0);
      }
      if constexpr (DQ != 192 && !CAREFUL) fed<DSQ + DSV, DSQ + DSV, LEAD, 1>();
      bf16x8 dsf[2], dsl[2];
      Pairs pairs;  // of the careful pass
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float ds[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int vv = 8 * hh + e, ro = (vv >> 2) * 8 + (vv & 3);
          float p, grad = 1.0f;
          if constexpr (MODE != 0 || CAREFUL)
            p = __builtin_amdgcn_exp2f(
                score<MODE>(a, slope2, sacc[vv], fabsf(far0 - (float)ro), grad) - lq);
          else
            p = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[vv], a.sl2, -lq));
          // in the first sweep dl is 0 and P dP is what is summed
          const float d = p * (pacc[vv] - (only_delta ? 0.0f : dl));
          const float kept = (unsigned)(ro - base) < width ? d : 0.0f;
          if (only_delta) dl += kept;
          ds[e] = MODE ? kept * grad : kept;
          if constexpr (CAREFUL) {
            const bool sees = (unsigned)(ro - base) < width;
            if (!sees) ds[e] = 0.0f;  // not 0 times a masked pair's slope
            pairs.put(vv, sees, ds[e]);
          }
        }
        split8(ds, dsf[hh], dsl[hh]);
      }
      if (only_delta) continue;
      if constexpr (CAREFUL) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
          add_seen<2, true>(dqacc[db], [&](int hh) { return read_tr<DQ>(ks, lt, jb * 32 + 16 * hh, db); },
                            dsf, dsl, pairs);
        continue;
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        // operands in registers at once; at DQ = 192 all six, or reads ordered
        // ahead of the MFMAs, spilled (the pass 561 us against 540 at one
        // sequence of 2048 tokens and 128 heads)
        constexpr int GRP = DQ == 192 ? 2 : DB;
#pragma unroll
        for (int d0 = 0; d0 < DB; d0 += GRP) {
          bf16x8 ktr[GRP];
#pragma unroll
          for (int e = 0; e < GRP; ++e) ktr[e] = read_tr<DQ>(ks, lt, jb * 32 + 16 * hh, d0 + e);
#pragma unroll
          for (int e = 0; e < GRP; ++e)
            dqacc[d0 + e] =
                __builtin_amdgcn_mfma_f32_32x32x16_bf16(ktr[e], dsf[hh], dqacc[d0 + e], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < GRP; ++e)
            dqacc[d0 + e] =
                __builtin_amdgcn_mfma_f32_32x32x16_bf16(ktr[e], dsl[hh], dqacc[d0 + e], 0, 0, 0);
        }
      }
      if constexpr (DQ != 192 && !CAREFUL) fed<4 * DB, 4 * DB, 6, 2>();
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  if (only_delta) dl += __shfl_xor(dl, 32);
  }
  if (g == 0 && qok && (!CAREFUL || again)) delta[srow + myq] = dl;
  const bool some = run.x < run.y;
  bool bad = false;
  if constexpr (!CAREFUL) bad = __ballot(some && probe_of(dqacc) != 0.0f) != 0;
  if (CAREFUL ? again : !bad)
    store_rows<DQ>(dqacc, a.scale, some, lds + wave * 32 * (DQ + 8), lane, S - q0,
                   dq + (srow + q0) * DQ, DQ);
  return bad;
}

struct DqCall {
  Args a;
  const uint16_t *o, *dout;
  const float* lse;
  float* delta;
  uint16_t* dq;
};
template <int DQ, int DV, int MODE>
__global__ __launch_bounds__(NT, 2) void span_bwd_dq(DqCall c) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * BKT * (DQ + DV)];
  const bool bad = dq_pass<DQ, DV, MODE, false>(c.a, lds, false, c.o, c.dout, c.lse, c.delta, c.dq);
  if (!any_wave<NT>(bad, (int*)lds)) return;
  const DqCall d = arguments_again<DqCall>();
  dq_pass<DQ, DV, MODE, true>(d.a, lds, bad, d.o, d.dout, d.lse, d.delta, d.dq);
}

// dK, dV of a 128-key tile of one KV head over the query heads of one part of
// its group: steps of 64 queries of each head in turn, from the first query
// block that sees the tile.  S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T +=
// Q^T dS.  DQ <= 128: 8 waves (4 key quarters x 2 query halves, two waves a
// SIMD), K and V tiles in LDS, the halves' sums meet in LDS at the end.  (4 waves
// with their K and V rows in registers and two workgroups a CU spilled 37 of 256
// registers: 857 us against 306 for 8192 packed tokens, 32/8 heads of 128.)
// DQ = 192: 4 waves, one a key quarter, each taking both query halves in turn,
// its K and V rows in registers.
// The whole group in one workgroup needs no partial sums in memory; a tile with
// much more work than a CU's share has its group split over several workgroups
// (parts_of), and span_reduce adds their fp32 sums in order.
// Bound as the forward for DQ <= 128 (MFMA pipes 43% busy): 226 us in a trace,
// 0.57 PFLOP/s, at its 8192 packed tokens.  DQ = 192 has one wave a SIMD and one
// workgroup a CU, so nothing covers a tile's start and end (MFMA pipes 24% busy):
// 273 us, 0.36 PFLOP/s (both query halves in one run of instructions took as long).
// A tile stays whole up to a CU's share of all work (256 CUs) or 16 steps (of 2
// blocks each); a heavier one is split, by a divisor of the group, into parts of
// at most three quarters of a share.  Training pass in us, against parts of at
// most half a share whatever the tile: 8192 tokens, 32/8 heads of 128, 16 equal
// documents 283 : 316, documents of 60 to 2500 tokens 463 : 479; one document 2718
// : 2800; 16384 tokens of 2 documents, 16/2 heads, 3282 : 3036.
__device__ __forceinline__ int parts_of(const Plan& p, int id, int group, int Hkv, int most) {
  if (most == 1) return 1;
  const int64_t w = (int64_t)uniform(p.kwork[id]) * group;
  const int64_t share = (int64_t)uniform(*p.ktotal) * group * Hkv;  // of 256 CUs
  if (w * 256 <= share || w <= 32) return 1;
  const int64_t piece = max(share * 3 / 1024, (int64_t)32);
  int n = 1;
  while (n < most && (group % n || w > piece * n)) ++n;
  return n;
}

template <int DQ>
constexpr int dkdv_waves() {
  return DQ <= 128 ? 8 : 4;
}
// elements of the LDS array that holds the K and V tiles, later the sums' meeting
// place and each wave's rows on their way out (fp32 rows of 192 do not fit)
template <int DQ, int DV>
constexpr int dkdv_lds() {
  constexpr int tiles = TILE * (DQ + DV), sums = 4 * 32 * (DQ + 4) * 2, rows = 4 * 32 * (DQ + 8);
  return dkdv_waves<DQ>() == 4 ? rows : tiles > sums ? tiles : sums;
}

// (arrays of their own: a read of one is not taken for a read of what the copies
// into another still write, and does not wait for them)
template <int DQ, int DV>
struct DkdvTiles {
  uint16_t *lds, *q_a, *q_b, *g_a, *g_b;
  float (*lse)[QT], (*dl)[QT];
  int (*lo)[QT], (*wd)[QT];
};

template <int DQ, int DV, int MODE, bool CAREFUL>
__device__ __forceinline__ bool dkdv_pass(const Args& a, const DkdvTiles<DQ, DV>& tiles, bool again,
                                          const uint16_t* __restrict__ dout,
                                          const float* __restrict__ lse,
                                          const float* __restrict__ delta, int most,
                                          float* __restrict__ dk_part, float* __restrict__ dv_part,
                                          uint16_t* __restrict__ dk, uint16_t* __restrict__ dv) {
  constexpr int DSQ = DQ / 16, DSV = DV / 16, DBQ = DQ / 32, DBV = DV / 32;
  constexpr int LK = TILE * DQ, LQ = QT * DQ, LG = QT * DV;
  constexpr int NW = dkdv_waves<DQ>(), NTH = 64 * NW, QH = 8 / NW;
  constexpr bool KREG = NW == 4;
  uint16_t *lds = tiles.lds, *q_a = tiles.q_a, *q_b = tiles.q_b, *g_a = tiles.g_a, *g_b = tiles.g_b;
  float (*lse_s)[QT] = tiles.lse, (*dl_s)[QT] = tiles.dl;
  int (*lo_s)[QT] = tiles.lo, (*wd_s)[QT] = tiles.wd;
  const int S = a.S, H = a.H, nb = a.plan.nb, group = H / a.Hkv;
  // an XCD's shader engines take its workgroups in turn: the parts that a tile
  // does not have are rotated from tile to tile, or one engine got all the work
  const int block = block_index<CAREFUL>();
  const int slot = block / (a.Hkv * most), rest = block % (a.Hkv * most);
  const int id = uniform(a.plan.korder[slot]), hk = rest % a.Hkv;
  const int part = (rest / a.Hkv + slot) % most;
  const int parts = parts_of(a.plan, id, group, a.Hkv, most);
  if (part >= parts) return false;
  const int b = id / a.plan.nt, kt = id % a.plan.nt;
  const int tid = thread_index<CAREFUL>(), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, c = lane & 31;
  const int kq = wave & 3, qh0 = NW == 8 ? wave >> 2 : 0;
  const int heads = group / parts, h0 = hk * group + part * heads;
  const int64_t ldt = (int64_t)H * DV;
  const uint16_t* kb = a.k + (int64_t)(b * a.Hkv + hk) * S * DQ;
  const uint16_t* vb = a.v + (int64_t)(b * a.Hkv + hk) * S * DV;
  uint16_t* Ks = lds;
  uint16_t* Vs = lds + LK;
  const int k0 = kt * TILE, kw0 = k0 + kq * 32, mykey = kw0 + c;
  const int2 seen = make_int2(uniform(a.plan.keys[id].x), uniform(a.plan.keys[id].y));
  const int4* blk = a.plan.blk + (int64_t)b * nb;
  const uint32_t lrq = lane_row<DQ>(c, g), lrv = lane_row<DV>(c, g);
  const uint32_t ltq = lane_tr<DQ>(lane), ltv = lane_tr<DV>(lane);
  Rows<KREG ? DSQ : 0, CAREFUL> kfr(KREG && mykey < S ? kb + (int64_t)mykey * DQ + 8 * g : nullptr);
  Rows<KREG ? DSV : 0, CAREFUL> vfr(KREG && mykey < S ? vb + (int64_t)mykey * DV + 8 * g : nullptr);
  if constexpr (!KREG) {
    const TileCopy<DQ, NTH, TILE> ck(tid, DQ);
    const TileCopy<DV, NTH, TILE> cv(tid, DV);
    ck(kb, DQ, k0, S, Ks, wave);
    cv(vb, DV, k0, S, Vs, wave);
  }
  f32x16 dvacc[DBV], dkacc[DBQ];
#pragma unroll
  for (int i = 0; i < DBV; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dvacc[i][e] = 0.0f;
#pragma unroll
  for (int i = 0; i < DBQ; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dkacc[i][e] = 0.0f;

  const int qfirst = seen.x * 32, nq = (seen.y - seen.x + 1) / 2;  // 64-query steps of a head
  const int steps = nq * heads;
  const TileCopy<DQ, NTH, QT> cq(tid, DQ);
  const TileCopy<DV, NTH, QT> cg(tid, ldt);
  float lr = INFINITY, dr = 0.0f;
  int2 rr = make_int2(0, 0);
  auto issue = [&](int h, int q0, auto which) {
    constexpr int buf = decltype(which)::value;
    cq(a.q + (int64_t)(b * H + h) * S * DQ, DQ, q0, S, buf ? q_b : q_a, wave);
    cg(dout + (int64_t)b * S * ldt + (int64_t)h * DV, ldt, q0, S, buf ? g_b : g_a, wave);
    if (tid < QT) {  // used at the end of the step, when the copies have landed too
      const int i = q0 + tid;
      const bool in = i < S;
      const int64_t at = (int64_t)(b * H + h) * S + i, row = (int64_t)b * S + i;
      lr = in ? lse[at] : INFINITY;
      dr = in ? delta[at] : 0.0f;
      rr = in ? make_int2(a.lo[row], a.hi[row]) : make_int2(0, 0);
    }
  };
  // FOLD: the accumulators of S and dP start from -lse / sl2 and -delta of their
  // rows, read from LDS as they lie, so the statistics take no registers of their
  // own and no instruction (a cap needs the bare product)
  constexpr bool FOLD = (MODE & CAP) == 0 && !CAREFUL;
  const float over = 1.0f / a.sl2;
  auto stats = [&](int buf) {
    if (tid < QT) {
      const int2 r = clamp_run(rr, S);
      lse_s[buf][tid] = FOLD ? -lr * over : -lr;
      dl_s[buf][tid] = -dr;
      lo_s[buf][tid] = r.x;
      wd_s[buf][tid] = r.y - r.x;
    }
  };
  if (steps > 0) {
    issue(h0, qfirst, std::integral_constant<int, 0>{});
    stats(0);
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  int j = 0, u = 0;  // head of the part, step of the head
  auto step = [&](int n, auto which) {
    constexpr int buf = decltype(which)::value;
    const int q0 = qfirst + u * QT;
    const float slope2 = (MODE & BIAS) ? scalar_load(a.slopes + h0 + j) * LOG2E : 0.0f;
    if (++u == nq) {
      u = 0;
      ++j;
    }
    if (n + 1 < steps) issue(h0 + j, qfirst + u * QT, std::integral_constant<int, buf ^ 1>{});
    const uint16_t* qs = buf ? q_b : q_a;
    const uint16_t* gs = buf ? g_b : g_a;
#pragma unroll
    for (int hq = 0; hq < QH; ++hq) {
      const int qh = NW == 8 ? qh0 : hq;
      const int qw0 = q0 + qh * 32;  // this wave's queries
      const int4 x = qw0 < S ? extremes(blk + (qw0 >> 5)) : make_int4(INT_MAX, INT_MAX, 0, 0);
      if (kw0 < x.w && kw0 + 32 > x.x) {  // some query sees some key
        const bool edge = CAREFUL || kw0 < x.y || kw0 + 32 > x.z;
        const float far0 = (float)(qw0 + 4 * g - mykey);
        // this wave's rows of the tiles, through its lane addresses
        const uint32_t q_row = lrq + qh * 32 * DQ * 2, g_row = lrv + qh * 32 * DV * 2;
        const uint32_t q_tr = ltq + qh * 32 * DQ * 2, g_tr = ltv + qh * 32 * DV * 2;
        const uint32_t k_row = lrq + kq * 32 * DQ * 2, v_row = lrv + kq * 32 * DV * 2;
        const int r0 = qh * 32 + g * 4;
        f32x16 sacc, pacc;
        kfr.forget();
        vfr.forget();
#pragma unroll
        for (int v4 = 0; v4 < 4; ++v4) {
          const float4 l = lds4(&lse_s[buf][r0 + 8 * v4]);
          const float4 d = lds4(&dl_s[buf][r0 + 8 * v4]);
          const float lv[4] = {l.x, l.y, l.z, l.w}, dv4[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sacc[4 * v4 + e] = FOLD ? lv[e] : 0.0f;
            pacc[4 * v4 + e] = dv4[e];
          }
        }
#pragma unroll
        for (int s = 0; s < DSQ; ++s) {
          sacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              read_row<DQ>(qs, q_row, 0, s),
              KREG ? kfr[s] : read_row<DQ>(Ks, k_row, 0, s), sacc, 0, 0, 0);
          if (s < DSV)
            pacc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                read_row<DV>(gs, g_row, 0, s),
                KREG ? vfr[s] : read_row<DV>(Vs, v_row, 0, s), pacc, 0, 0, 0);
        }
        if constexpr (!CAREFUL)
          fed<8 + (KREG ? 1 : 2) * (DSQ + DSV), DSQ + DSV, 8 + (KREG ? 4 : 6), KREG ? 1 : 2>();
        bf16x8 pf[2], dsf[2], dsl[2];
        Pairs pairs_p, pairs_d;  // of the careful pass
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float p8[8], d8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int vv = 8 * hh + e, ro = (vv >> 2) * 8 + (vv & 3);
            if constexpr (FOLD) {
              float y = sacc[vv] * a.sl2;
              if constexpr ((MODE & BIAS) != 0) y = __builtin_fmaf(-slope2, fabsf(far0 + (float)ro), y);
              p8[e] = __builtin_amdgcn_exp2f(y);
              d8[e] = p8[e] * pacc[vv];
            } else {
              float grad;
              const float y = score<MODE>(a, slope2, sacc[vv], fabsf(far0 + (float)ro), grad);
              p8[e] = __builtin_amdgcn_exp2f(y + lds1(&lse_s[buf][r0 + ro]));
              d8[e] = p8[e] * pacc[vv] * grad;
            }
          }
          if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int vv = 8 * hh + e, r = r0 + (vv >> 2) * 8 + (vv & 3);
              const int width = lds1(&wd_s[buf][r]);
              const bool keep = (unsigned)(mykey - lds1(&lo_s[buf][r])) < (unsigned)width;
              p8[e] = keep ? p8[e] : 0.0f;
              d8[e] = keep && width > 1 ? d8[e] : 0.0f;
              if constexpr (CAREFUL) {
                pairs_p.put(vv, keep, p8[e]);
                pairs_d.put(vv, keep && width > 1, d8[e]);
              }
            }
          }
          pf[hh] = pack8(p8);
          split8(d8, dsf[hh], dsl[hh]);
        }
        if constexpr (CAREFUL) {
#pragma unroll
          for (int db = 0; db < DBV; ++db)
            add_seen<2, false>(dvacc[db], [&](int hh) { return read_tr<DV>(gs, g_tr, 16 * hh, db); }, pf, pf,
                               pairs_p);
#pragma unroll
          for (int db = 0; db < DBQ; ++db)
            add_seen<2, true>(dkacc[db], [&](int hh) { return read_tr<DQ>(qs, q_tr, 16 * hh, db); }, dsf, dsl,
                              pairs_d);
          continue;
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
          for (int db = 0; db < DBV; ++db)
            dvacc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_tr<DV>(gs, g_tr, 16 * hh, db),
                                                                pf[hh], dvacc[db], 0, 0, 0);
#pragma unroll
          for (int db = 0; db < DBQ; db += 2) {
            bf16x8 qtr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) qtr[e] = read_tr<DQ>(qs, q_tr, 16 * hh, db + e);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              dkacc[db + e] =
                  __builtin_amdgcn_mfma_f32_32x32x16_bf16(qtr[e], dsf[hh], dkacc[db + e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              dkacc[db + e] =
                  __builtin_amdgcn_mfma_f32_32x32x16_bf16(qtr[e], dsl[hh], dkacc[db + e], 0, 0, 0);
          }
        }
        if constexpr (!CAREFUL) fed<4 * (DBV + DBQ), 2 * DBV + 4 * DBQ, 6, 2>();
      }
    }
    if (n + 1 < steps) stats(buf ^ 1);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
#pragma unroll 1
  for (int n = 0; n < steps; n += 2) {
    step(n, std::integral_constant<int, 0>{});
    if (n + 1 < steps) step(n + 1, std::integral_constant<int, 1>{});
  }
  // 8 waves: query half 1 parks its sums in LDS, half 0 adds them; dV first, then dK
  float* red = (float*)lds;
  auto meet = [&](auto& acc, auto blocks) {
    constexpr int DB = decltype(blocks)::value;
    static_assert(NW == 4 || 4 * DB * 16 * 64 * 4 <= dkdv_lds<DQ, DV>() * 2, "sums fit in LDS");
    if (qh0 == 1) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) red[(kq * DB * 16 + db * 16 + e) * 64 + lane] = acc[db][e];
    }
    __syncthreads();
    if (qh0 == 0) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[db][e] += red[(kq * DB * 16 + db * 16 + e) * 64 + lane];
    }
    __syncthreads();
  };
  if constexpr (NW == 8) {
    meet(dvacc, std::integral_constant<int, DBV>{});
    meet(dkacc, std::integral_constant<int, DBQ>{});
  }
  bool bad = false;
  if constexpr (!CAREFUL)
    bad = __ballot(qh0 == 0 && mykey < S && probe_of(dvacc) + probe_of(dkacc) != 0.0f) != 0;
  const int64_t krow = (int64_t)(b * a.Hkv + hk) * S;                  // of dk, dv
  const int64_t prow = ((int64_t)(b * a.Hkv + hk) * most + part) * S;  // of the partials
  if (qh0 == 0 && (CAREFUL ? again : !bad) && kw0 < S) {
    // staged by each wave in its own LDS space
    uint16_t* os = lds + kq * (dkdv_lds<DQ, DV>() / 4);
    static_assert(32 * (DQ + 8) <= dkdv_lds<DQ, DV>() / 4 && 32 * (DV + 8) <= dkdv_lds<DQ, DV>() / 4,
                  "bf16 staging fits");
    if (parts == 1) {
      store_rows<DV>(dvacc, 1.0f, true, os, lane, S - kw0, dv + (krow + kw0) * DV, DV);
      __builtin_amdgcn_s_waitcnt(0);
      __builtin_amdgcn_wave_barrier();
      store_rows<DQ>(dkacc, a.scale, true, os, lane, S - kw0, dk + (krow + kw0) * DQ, DQ);
    } else {
      constexpr bool whole = 32 * (DQ + 4) * 2 <= dkdv_lds<DQ, DV>() / 4;
      if constexpr (whole) {
        store_rows_f32<DV>(dvacc, 1.0f, (float*)os, lane, S - kw0, dv_part + (prow + kw0) * DV);
        store_rows_f32<DQ>(dkacc, a.scale, (float*)os, lane, S - kw0, dk_part + (prow + kw0) * DQ);
      } else if (mykey < S) {  // heads of 192: the tile's LDS does not hold fp32 rows
#pragma unroll
        for (int v = 0; v < DBV * 4; ++v)
          *(float4*)(dv_part + (prow + mykey) * DV + v / 4 * 32 + v % 4 * 8 + g * 4) =
              make_float4(dvacc[v / 4][v % 4 * 4], dvacc[v / 4][v % 4 * 4 + 1],
                          dvacc[v / 4][v % 4 * 4 + 2], dvacc[v / 4][v % 4 * 4 + 3]);
#pragma unroll
        for (int v = 0; v < DBQ * 4; ++v)
          *(float4*)(dk_part + (prow + mykey) * DQ + v / 4 * 32 + v % 4 * 8 + g * 4) =
              make_float4(dkacc[v / 4][v % 4 * 4] * a.scale, dkacc[v / 4][v % 4 * 4 + 1] * a.scale,
                          dkacc[v / 4][v % 4 * 4 + 2] * a.scale, dkacc[v / 4][v % 4 * 4 + 3] * a.scale);
      }
    }
  }
  return bad;
}

struct DkdvCall {
  Args a;
  const uint16_t* dout;
  const float *lse, *delta;
  int most;
  float *dk_part, *dv_part;
  uint16_t *dk, *dv;
};
template <int DQ, int DV, int MODE>
__global__ __launch_bounds__(64 * dkdv_waves<DQ>(), dkdv_waves<DQ>() == 8 ? 2 : 1)
void span_bwd_dkdv(DkdvCall c) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[dkdv_lds<DQ, DV>()];
  __shared__ __attribute__((aligned(16))) uint16_t q_a[QT * DQ], q_b[QT * DQ], g_a[QT * DV], g_b[QT * DV];
  __shared__ __attribute__((aligned(16))) float lse_s[2][QT], dl_s[2][QT];
  __shared__ __attribute__((aligned(16))) int lo_s[2][QT], wd_s[2][QT];
  const DkdvTiles<DQ, DV> tiles{lds, q_a, q_b, g_a, g_b, lse_s, dl_s, lo_s, wd_s};
  const bool bad = dkdv_pass<DQ, DV, MODE, false>(c.a, tiles, false, c.dout, c.lse, c.delta, c.most,
                                                  c.dk_part, c.dv_part, c.dk, c.dv);
  if (!any_wave<64 * dkdv_waves<DQ>()>(bad, (int*)lds)) return;
  const DkdvCall d = arguments_again<DkdvCall>();
  dkdv_pass<DQ, DV, MODE, true>(d.a, tiles, bad, d.dout, d.lse, d.delta, d.most, d.dk_part, d.dv_part, d.dk,
                                d.dv);
}

// dk = bf16(sum over the parts, in order), same for dv, of the tiles in parts
__global__ __launch_bounds__(NT) void span_reduce(Plan plan, const float* __restrict__ dk_part,
                                                  const float* __restrict__ dv_part, int group,
                                                  int Hkv, int most, int S, int DQ, int DV,
                                                  uint16_t* __restrict__ dk,
                                                  uint16_t* __restrict__ dv) {
  const int id = uniform(plan.korder[blockIdx.x / Hkv]), hk = blockIdx.x % Hkv;
  const int parts = parts_of(plan, id, group, Hkv, most);
  if (parts == 1) return;
  constexpr int ROWS = TILE / 8;  // few tiles are in parts: 8 workgroups each
  const int k0 = id % plan.nt * TILE + blockIdx.y * ROWS, rows = min(ROWS, S - k0);
  const int64_t bhk = (int64_t)(id / plan.nt) * Hkv + hk;
  auto add = [&](const float* part, uint16_t* out, int D) {
    for (int i = threadIdx.x; i < rows * D / 4; i += NT) {
      float4 s = make_float4(0, 0, 0, 0);
      for (int j = 0; j < parts; ++j) {
        const float4 x = *(const float4*)(part + ((bhk * most + j) * S + k0) * D + i * 4);
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
      }
      *(u32x2*)(out + (bhk * S + k0) * D + i * 4) =
          u32x2{st::pack_bf16x2(s.x, s.y), st::pack_bf16x2(s.z, s.w)};
    }
  };
  add(dk_part, dk, DQ);
  add(dv_part, dv, DV);
}

// ---------------------------------------------------------------- host
bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// Most parts that a KV head's group may be split into: none where a tile has at
// most 16 steps anyway or the tiles are many.  (None at all: 513 us against 472
// for a training pass of 8192 packed tokens, 32/8 heads of 128.)
int most_parts(int64_t B, int64_t S, int64_t H, int64_t Hkv) {
  const int64_t group = H / Hkv;
  return st::cdiv(S, QT) * group <= 16 || B * st::cdiv(S, TILE) * Hkv > 8192 ? 1 : (int)group;
}

struct Space {
  int64_t delta, dkp, dvp, bytes;  // byte offsets
  int most;
};
Space space_of(int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t DQ, int64_t DV) {
  Space s{};
  s.most = most_parts(B, S, H, Hkv);
  s.delta = 0;
  int64_t at = up256(B * H * S * 4);
  if (s.most > 1) {
    s.dkp = at;
    at += up256(B * Hkv * s.most * S * DQ * 4);
    s.dvp = at;
    at += up256(B * Hkv * s.most * S * DV * 4);
  }
  s.bytes = at + 256;
  return s;
}

bool dims_ok(int64_t DQ, int64_t DV) {
  return (DQ == 64 && DV == 64) || (DQ == 128 && DV == 128) || (DQ == 192 && DV == 128);
}

int check_common(const char* name, int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t DQ,
                 int64_t DV, float scale, float cap) {
  ST_CHECK_ARG(B >= 0 && S >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0, "%s: bad head counts", name);
  if (!dims_ok(DQ, DV))
    return st::fail(ST_EUNSUPPORTED, "%s: head dims %lld/%lld (64/64, 128/128 or 192/128 only)",
                    name, (long long)DQ, (long long)DV);
  ST_CHECK_ARG(std::isfinite(scale) && scale > 0, "%s: scale must be positive and finite", name);
  ST_CHECK_ARG(std::isfinite(cap) && cap >= 0, "%s: cap must be finite, 0 for none", name);
  // the kernels divide by the scale, and multiply the cap and the scale by constants
  if (scale < 1e-30f || scale > 1e30f || (cap > 0 && (cap > 1e30f || scale / cap > 1e4f)))
    return st::fail(ST_EUNSUPPORTED, "%s: scale %g or cap %g out of range (scale 1e-30 to 1e30, cap up "
                    "to 1e30 and at least scale / 1e4)", name, scale, cap);
  // tiles by 32-bit ids, one grid of tiles x heads, and 64 token-major rows
  // within a 32-bit byte offset
  const int64_t lim = (int64_t)1 << 31;
  if (S >= (1 << 30) || H >= (1 << 16) || B >= (1 << 24) || B * st::cdiv(S, 32) >= lim ||
      B * st::cdiv(S, 32) * H >= lim || 64 * H * DV * 2 >= lim)
    return st::fail(ST_EUNSUPPORTED, "%s: B=%lld S=%lld H=%lld is too large", name, (long long)B,
                    (long long)S, (long long)H);
  return ST_OK;
}

Args args_of(const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t B, int64_t S,
             int64_t H, int64_t Hkv, float scale, float cap, const float* slopes,
             const int32_t* lo, const int32_t* hi, const void* plan) {
  Args a{};
  a.q = q; a.k = k; a.v = v;
  a.lo = lo; a.hi = hi;
  a.slopes = slopes;
  a.plan = plan_of(plan, B, S);
  a.S = (int)S; a.H = (int)H; a.Hkv = (int)Hkv;
  a.scale = scale;
  a.sl2 = scale * LOG2E;
  if (cap > 0) {
    a.cap_in = 2.0f * LOG2E * scale / cap;
    a.cap_out = cap * LOG2E;
    const float r = scale / cap;
    a.cap_small = 0.35f / r;
    a.cap_r = r;
    const float c[3] = {-0.33332663774490356f, 0.1329982578754425f, -0.049148499965667725f};
    for (int i = 0; i < 3; ++i) a.cap_p[i] = a.sl2 * c[i];
    // (the greatest s^2 used is 0.35^2 / r^2; the smallest and greatest coefficient)
    const double last = (double)a.cap_p[2] * pow((double)r, 6.0), first = (double)a.cap_p[0] * r * r;
    if (r > 1e-19f && std::min(fabs(first), fabs(last)) > 1e-36 && std::max(fabs(first), fabs(last)) < 1e36)
      for (int i = 0; i < 3; ++i) a.cap_s[i] = (float)(a.cap_p[i] * pow((double)r, 2.0 * (i + 1)));
  }
  return a;
}

// a dimension of a launch holds less than 2^32 threads
int fits(const char* name, int64_t groups, int64_t threads) {
  if (groups * threads >= (int64_t)1 << 32)
    return st::fail(ST_EUNSUPPORTED, "%s: %lld workgroups of %lld threads are too large a launch", name,
                    (long long)groups, (long long)threads);
  return ST_OK;
}

template <int DQ, int DV, int MODE>
int run_fwd(const Args& a, int64_t B, uint16_t* out, float* lse, hipStream_t s) {
  if (int rc = fits("st_span_attn_fwd", B * a.plan.nt * a.H, NT)) return rc;
  span_fwd<DQ, DV, MODE><<<(unsigned)(B * a.plan.nt * a.H), NT, 0, s>>>({a, out, lse});
  return st::check_launch("span_fwd");
}

template <int DQ, int DV, int MODE>
int run_bwd(const Args& a, int64_t B, const uint16_t* out, const float* lse, const uint16_t* dout,
            uint16_t* dq, uint16_t* dk, uint16_t* dv, char* ws, hipStream_t s) {
  const Space sp = space_of(B, a.S, a.H, a.Hkv, DQ, DV);
  float* delta = (float*)(ws + sp.delta);
  float *dkp = (float*)(ws + sp.dkp), *dvp = (float*)(ws + sp.dvp);
  constexpr int NTH = 64 * dkdv_waves<DQ>();
  const int64_t tiles = B * a.plan.nt * a.Hkv;
  if (int rc = fits("st_span_attn_bwd", B * a.plan.nt * a.H, NT)) return rc;
  if (int rc = fits("st_span_attn_bwd", tiles * sp.most, NTH)) return rc;
  if (int rc = fits("st_span_attn_bwd", sp.most > 1 ? tiles : 0, NT)) return rc;
  span_bwd_dq<DQ, DV, MODE><<<(unsigned)(B * a.plan.nt * a.H), NT, 0, s>>>(
      {a, out, dout, lse, delta, dq});
  if (int rc = st::check_launch("span_bwd_dq")) return rc;
  span_bwd_dkdv<DQ, DV, MODE><<<(unsigned)(tiles * sp.most), NTH, 0, s>>>(
      {a, dout, lse, delta, sp.most, dkp, dvp, dk, dv});
  int rc = st::check_launch("span_bwd_dkdv");
  if (rc || sp.most == 1) return rc;
  span_reduce<<<dim3((unsigned)tiles, 8), NT, 0, s>>>(a.plan, dkp, dvp, a.H / a.Hkv, a.Hkv, sp.most, a.S,
                                                     DQ, DV, dk, dv);
  return st::check_launch("span_reduce");
}

// fn(DQ, DV, MODE) of a call as compile-time values
template <typename F>
int by_kind(int64_t DQ, float cap, const float* slopes, F&& fn) {
  auto with = [&](auto dq, auto dv) {
    const int mode = (cap > 0 ? CAP : 0) | (slopes ? BIAS : 0);
    switch (mode) {
      case 0: return fn(dq, dv, std::integral_constant<int, 0>{});
      case CAP: return fn(dq, dv, std::integral_constant<int, CAP>{});
      case BIAS: return fn(dq, dv, std::integral_constant<int, BIAS>{});
      default: return fn(dq, dv, std::integral_constant<int, CAP | BIAS>{});
    }
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (DQ == 64) return with(D64{}, D64{});
  if (DQ == 128) return with(D128{}, D128{});
  return with(std::integral_constant<int, 192>{}, D128{});
}

}  // namespace

extern "C" int64_t st_span_plan_bytes(int64_t B, int64_t S) {
  if (B <= 0 || S <= 0) return 0;
  return plan_of(nullptr, B, S).bytes;
}

extern "C" int st_span_plan(const int32_t* key_start, const int32_t* key_end, int64_t B, int64_t S,
                            void* plan, int64_t plan_bytes, st_stream_t stream) {
  ST_CHECK_ARG(B >= 0 && S >= 0 && S < (1 << 30), "st_span_plan: bad shape");
  if (B == 0 || S == 0) return ST_OK;
  if (B >= (1 << 24) || B * st::cdiv(S, 32) >= (int64_t)1 << 31)
    return st::fail(ST_EUNSUPPORTED, "st_span_plan: too many rows");
  ST_CHECK_ARG(key_start && key_end && plan && al16(plan), "st_span_plan: NULL or unaligned pointer");
  const Plan p = plan_of(plan, B, S);
  if (plan_bytes < p.bytes)
    return st::fail(ST_EWORKSPACE, "st_span_plan: needs %lld bytes", (long long)p.bytes);
  hipStream_t s = (hipStream_t)stream;
  const int64_t blocks = B * p.nb, tiles = B * p.nt;
  if (int rc = fits("st_span_plan", st::cdiv(blocks * 32, NT), NT)) return rc;
  if (int rc = fits("st_span_plan", tiles, 64)) return rc;
  span_blocks<<<(unsigned)st::cdiv(blocks * 32, NT), NT, 0, s>>>(key_start, key_end, (int)S, p.nb,
                                                                 blocks, (int4*)p.blk);
  if (int rc = st::check_launch("span_blocks")) return rc;
  span_tiles<<<(unsigned)tiles, 64, 0, s>>>(p.blk, p.nb, p.nt, (int2*)p.keys, p.qwork, p.kwork);
  if (int rc = st::check_launch("span_tiles")) return rc;
  span_order<<<dim3((unsigned)st::cdiv(tiles, NT), 2), NT, 0, s>>>(
      p.qwork, p.kwork, tiles, (int32_t*)p.qorder, (int32_t*)p.korder, p.ktotal);
  return st::check_launch("span_order");
}

extern "C" int64_t st_span_attn_workspace_bytes(int64_t B, int64_t S, int64_t H, int64_t Hkv,
                                                int64_t DQ, int64_t DV) {
  if (B <= 0 || S <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || !dims_ok(DQ, DV)) return 0;
  return space_of(B, S, H, Hkv, DQ, DV).bytes;
}

extern "C" int st_span_attn_fwd(const uint16_t* q, const uint16_t* k, const uint16_t* v, int64_t B,
                                int64_t S, int64_t H, int64_t Hkv, int64_t DQ, int64_t DV,
                                float scale, float cap, const float* slopes,
                                const int32_t* key_start, const int32_t* key_end, const void* plan,
                                uint16_t* out, float* lse, st_stream_t stream) {
  const char* name = "st_span_attn_fwd";
  if (int rc = check_common(name, B, S, H, Hkv, DQ, DV, scale, cap)) return rc;
  if (B == 0 || S == 0) return ST_OK;
  ST_CHECK_ARG(q && k && v && out && lse && key_start && key_end && plan && al16(q) && al16(k) &&
                   al16(v) && al16(out) && al16(plan), "%s: NULL or unaligned pointer", name);
  const Args a = args_of(q, k, v, B, S, H, Hkv, scale, cap, slopes, key_start, key_end, plan);
  return by_kind(DQ, cap, slopes, [&](auto dq, auto dv, auto mode) {
    return run_fwd<decltype(dq)::value, decltype(dv)::value, decltype(mode)::value>(
        a, B, out, lse, (hipStream_t)stream);
  });
}

extern "C" int st_span_attn_bwd(const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                const uint16_t* out, const float* lse, const uint16_t* dout,
                                int64_t B, int64_t S, int64_t H, int64_t Hkv, int64_t DQ,
                                int64_t DV, float scale, float cap, const float* slopes,
                                const int32_t* key_start, const int32_t* key_end, const void* plan,
                                uint16_t* dq, uint16_t* dk, uint16_t* dv, void* workspace,
                                int64_t workspace_bytes, st_stream_t stream) {
  const char* name = "st_span_attn_bwd";
  if (int rc = check_common(name, B, S, H, Hkv, DQ, DV, scale, cap)) return rc;
  if (B == 0 || S == 0) return ST_OK;
  ST_CHECK_ARG(q && k && v && out && lse && dout && dq && dk && dv && key_start && key_end && plan &&
                   al16(q) && al16(k) && al16(v) && al16(out) && al16(dout) && al16(dq) &&
                   al16(dk) && al16(dv) && al16(plan), "%s: NULL or unaligned pointer", name);
  const int64_t need = space_of(B, S, H, Hkv, DQ, DV).bytes;
  if (!workspace || workspace_bytes < need)
    return st::fail(ST_EWORKSPACE, "%s: needs %lld workspace bytes", name, (long long)need);
  const Args a = args_of(q, k, v, B, S, H, Hkv, scale, cap, slopes, key_start, key_end, plan);
  char* ws = (char*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  return by_kind(DQ, cap, slopes, [&](auto dq_, auto dv_, auto mode) {
    return run_bwd<decltype(dq_)::value, decltype(dv_)::value, decltype(mode)::value>(
        a, B, out, lse, dout, dq, dk, dv, ws, (hipStream_t)stream);
  });
}
