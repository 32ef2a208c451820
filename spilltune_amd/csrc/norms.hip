// Norms after and before a part of a decoder block, fused with its gate and
// residual scale, and their backward:
//
//   z = y  or  y r1 post,              r1 = rsqrt(mean(y^2) + eps)
//   h = residual + scale gate z
//   normed = h r2 pre,                 r2 = rsqrt(mean(h^2) + eps)
//
//   g = dnormed pre,  dH = dh + r2 (g - h r2^2 mean(g h)),  dresidual = dH
//   q = scale gate dH,  dgate = scale dH z,  dpost = q y r1,  dpre = dnormed h r2
//   dy = q  or  r1 (w - y r1^2 mean(w y)),  w = q post
//
// Bound by HBM: the forward reads y and residual and writes h and normed once (8
// bytes an element), the backward reads y, residual, dh and dnormed and writes dy
// and dresidual once (12 bytes): a row stays in the registers of its workgroup
// between its two sums, and h is formed again from what z needs anyway instead of
// being read (its bf16 copy would also be off by half a step).  All in fp32, each
// result rounded once; normed comes from the unrounded h.
//
// Sums over rows (dpost, dpre, and dgate where a gate is shared by rows): a
// workgroup walks a run of rows with the columns' sums in registers, and a second
// kernel joins the runs in their order.
#include <cmath>

#include "common.h"

namespace {

enum {
  GATE_NONE = ST_GATE_NONE,
  GATE_COLUMNS = ST_GATE_COLUMNS,
  GATE_TOKENS = ST_GATE_TOKENS,
  GATE_FULL = ST_GATE_FULL
};
constexpr int64_t MAXH = 16384;

struct Args {
  const uint16_t *y, *res, *post, *pre;
  const void* gate;
  int32_t gate_mode, gate_f32;
  int64_t rows_per;  // rows that share a gate row (GATE_COLUMNS)
  int64_t rows, H;
  float scale, eps;
  float *r1, *r2;
  // forward
  uint16_t *h, *normed;
  // backward
  const uint16_t *dh, *dn;
  uint16_t *dy, *dres;
  void* dgate;     // of the gate's type
  float* partial;  // [runs][3][H]: dpost, dpre, dgate of the run's rows
  int64_t runs, per_run;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Sum over the workgroup, in every thread; `red` is free again after the next one.
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v += red[i];
  }
  return v;
}

// VEC bf16 as they lie.  Elements past the row (`in` false) read its first ones and are
// cleared: a load under a branch would be waited for at the branch's end.
template <int VEC>
struct Raw {
  uint4 v;
};
template <>
struct Raw<1> {
  uint32_t v;
};
template <int VEC>
__device__ __forceinline__ Raw<VEC> raw(const uint16_t* row, int64_t i, bool in) {
  Raw<VEC> r;
  if constexpr (VEC == 8)
    r.v = *(const uint4*)(row + (in ? i : 0));
  else
    r.v = row[in ? i : 0];
  return r;
}
template <int VEC>
__device__ __forceinline__ void unpack(const Raw<VEC>& r, bool in, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    const uint32_t w[4] = {in ? r.v.x : 0, in ? r.v.y : 0, in ? r.v.z : 0, in ? r.v.w : 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
    f[0] = in ? __uint_as_float(r.v << 16) : 0.0f;
  }
}
template <int VEC>
__device__ __forceinline__ void load_bf16(const uint16_t* row, int64_t i, bool in,
                                          float (&f)[VEC]) {
  unpack<VEC>(raw<VEC>(row, i, in), in, f);
}
template <int VEC>
__device__ __forceinline__ void store_bf16(uint16_t* p, int64_t i, const float (&f)[VEC]) {
  if constexpr (VEC == 8)
    *(uint4*)(p + i) = make_uint4(st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3]),
                                  st::pack_bf16x2(f[4], f[5]), st::pack_bf16x2(f[6], f[7]));
  else
    p[i] = st::f32_to_bf16(f[0]);
}
template <int VEC>
__device__ __forceinline__ void load_f32(const float* row, int64_t i, bool in, float (&f)[VEC]) {
  const float* p = row + (in ? i : 0);
  if constexpr (VEC == 8) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    f[0] = *p;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = in ? f[e] : 0.0f;
}
template <int VEC>
__device__ __forceinline__ void store_f32(float* p, int64_t i, const float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    *(float4*)(p + i) = make_float4(f[0], f[1], f[2], f[3]);
    *(float4*)(p + i + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    p[i] = f[0];
  }
}

// scale * gate of one chunk
template <int VEC>
__device__ __forceinline__ void gate_of(const Args& a, int64_t row, int64_t i, bool in,
                                        float (&f)[VEC]) {
  if (a.gate_mode == GATE_NONE) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = a.scale;
    return;
  }
  if (a.gate_mode == GATE_TOKENS) {
    const float g = a.gate_f32 ? ((const float*)a.gate)[row]
                               : st::bf16_to_f32(((const uint16_t*)a.gate)[row]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = a.scale * g;
    return;
  }
  const int64_t at = (a.gate_mode == GATE_FULL ? row : row / a.rows_per) * a.H;
  if (a.gate_f32)
    load_f32<VEC>((const float*)a.gate + at, i, in, f);
  else
    load_bf16<VEC>((const uint16_t*)a.gate + at, i, in, f);
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] *= a.scale;
}

template <int VEC, int NT, int NV>
__global__ __launch_bounds__(NT) void norms_fwd(Args a) {
  __shared__ float red[2][NT / 64];
  const float over = 1.0f / (float)a.H;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t base = row * a.H;
    float y[NV][VEC], h[NV][VEC];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
      load_bf16<VEC>(a.y + base, i, i < a.H, y[n]);
      load_bf16<VEC>(a.res + base, i, i < a.H, h[n]);
    }
    float r1 = 1.0f;
    if (a.post) {
      float ss = 0.0f;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += y[n][e] * y[n][e];
      r1 = 1.0f / sqrtf(block_sum<NT>(ss, red[0]) * over + a.eps);
      if (a.r1 && threadIdx.x == 0) a.r1[row] = r1;
    }
    float ss = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
      float w[VEC], g[VEC];
      if (a.post) load_bf16<VEC>(a.post, i, i < a.H, w);
      gate_of<VEC>(a, row, i, i < a.H, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = a.post ? y[n][e] * r1 * w[e] : y[n][e];
        h[n][e] += g[e] * z;
        ss += h[n][e] * h[n][e];
      }
      if (i < a.H) store_bf16<VEC>(a.h + base, i, h[n]);
    }
    if (a.pre) {  // the same way for the whole launch
      const float r2 = 1.0f / sqrtf(block_sum<NT>(ss, red[1]) * over + a.eps);
      if (a.r2 && threadIdx.x == 0) a.r2[row] = r2;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
        float w[VEC];
        load_bf16<VEC>(a.pre, i, i < a.H, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= h[n][e] * r2;
        if (i < a.H) store_bf16<VEC>(a.normed + base, i, w);
      }
    }
    if constexpr (NT > 64) __syncthreads();  // the sums' places are free again
  }
}

// SUMS: run blockIdx.x of `per_run` rows (all of one gate row), columns' sums kept.
// GATE: there is one.  The next row is read while the present one is worked on (up to
// 16 elements a thread: beyond, registers are short), and rows wait as the bf16 they
// are: with them in fp32, fewer waves fit.
template <int VEC, int NT, int NV, bool SUMS, bool GATE>
__global__ __launch_bounds__(NT) void norms_bwd(Args a) {
  __shared__ float red[3][NT / 64];
  constexpr bool EARLY = SUMS && VEC * NV <= 16;
  const float over = 1.0f / (float)a.H;
  float dpost[NV][VEC] = {}, dpre[NV][VEC] = {}, dgate[NV][VEC] = {};
  int64_t row, end, by;
  if constexpr (SUMS) {
    const int64_t in_group = a.runs / (a.rows / a.rows_per);  // runs of a gate row
    const int64_t g = blockIdx.x / in_group, k = blockIdx.x % in_group;
    row = g * a.rows_per + k * a.per_run;
    end = min(row + a.per_run, (g + 1) * a.rows_per), by = 1;
  } else {
    row = blockIdx.x, end = a.rows, by = gridDim.x;
  }
  // (a gradient that is not there: y in its place, cleared)
  const bool has_dh = a.dh, has_dn = a.dn;
  const uint16_t *dh = has_dh ? a.dh : a.y, *dn = has_dn ? a.dn : a.y;
  Raw<VEC> ny[NV], nh[NV], nd[NV], nn[NV];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC, base = r * a.H;
      ny[n] = raw<VEC>(a.y + base, i, i < a.H);
      nh[n] = raw<VEC>(a.res + base, i, i < a.H);
      nd[n] = raw<VEC>(dh + base, i, i < a.H);
      nn[n] = raw<VEC>(dn + base, i, i < a.H);
    }
  };
  fetch(row);
  for (; row < end; row += by) {
    const int64_t base = row * a.H;
    Raw<VEC> ry[NV], rh[NV], rd[NV], rn[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) ry[n] = ny[n], rh[n] = nh[n], rd[n] = nd[n], rn[n] = nn[n];
    if (EARLY) fetch(row + by < end ? row + by : row);
    const float r1 = a.post ? a.r1[row] : 1.0f, r2 = has_dn ? a.r2[row] : 0.0f;
    float d[NV][VEC];
    if (has_dn) {
      float h[NV][VEC], gn[NV][VEC], dot = 0.0f;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
        const bool in = i < a.H;
        float y[VEC], w[VEC], g[VEC], p[VEC];
        unpack<VEC>(ry[n], in, y);
        unpack<VEC>(rh[n], in, h[n]);
        unpack<VEC>(rn[n], in, gn[n]);
        if (a.post) load_bf16<VEC>(a.post, i, in, w);
        load_bf16<VEC>(a.pre, i, in, p);
        if (GATE) gate_of<VEC>(a, row, i, in, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float z = a.post ? y[e] * r1 * w[e] : y[e];
          h[n][e] = __builtin_fmaf(GATE ? g[e] : a.scale, z, h[n][e]);
          if constexpr (SUMS) dpre[n][e] = __builtin_fmaf(gn[n][e], h[n][e] * r2, dpre[n][e]);
          gn[n][e] *= p[e];
          dot = __builtin_fmaf(gn[n][e], h[n][e], dot);
        }
      }
      const float c = block_sum<NT>(dot, red[0]) * over * r2 * r2;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const bool in = ((int64_t)n * NT + threadIdx.x) * VEC < a.H;
        unpack<VEC>(rd[n], in && has_dh, d[n]);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          d[n][e] = __builtin_fmaf(r2, __builtin_fmaf(-c, h[n][e], gn[n][e]), d[n][e]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        unpack<VEC>(rd[n], ((int64_t)n * NT + threadIdx.x) * VEC < a.H && has_dh, d[n]);
    }
    float dot = 0.0f, gdot = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
      const bool in = i < a.H;
      if (a.dres && in) store_bf16<VEC>(a.dres + base, i, d[n]);
      float y[VEC], w[VEC], g[VEC], dz[VEC];
      unpack<VEC>(ry[n], in, y);
      if (a.post) load_bf16<VEC>(a.post, i, in, w);
      if (GATE) gate_of<VEC>(a, row, i, in, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float yn = y[e] * r1;
        if (GATE) {
          dz[e] = a.scale * d[n][e] * (a.post ? yn * w[e] : yn);
          gdot += dz[e];
        }
        float q = (GATE ? g[e] : a.scale) * d[n][e];
        if constexpr (SUMS) {
          if (GATE) dgate[n][e] += dz[e];
          dpost[n][e] = __builtin_fmaf(q, yn, dpost[n][e]);
        }
        if (a.post) q *= w[e];
        dot = __builtin_fmaf(q, y[e], dot);
        d[n][e] = q;
      }
      if (GATE && a.gate_mode == GATE_FULL && a.dgate && in) {
        if (a.gate_f32)
          store_f32<VEC>((float*)a.dgate + base, i, dz);
        else
          store_bf16<VEC>((uint16_t*)a.dgate + base, i, dz);
      }
    }
    if (GATE && a.gate_mode == GATE_TOKENS && a.dgate) {
      gdot = block_sum<NT>(gdot, red[1]);
      if (threadIdx.x == 0) {
        if (a.gate_f32)
          ((float*)a.dgate)[row] = gdot;
        else
          ((uint16_t*)a.dgate)[row] = st::f32_to_bf16(gdot);
      }
    }
    if (a.dy) {
      float c = 0.0f;
      if (a.post) c = block_sum<NT>(dot, red[2]) * over * r1 * r1;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
        const bool in = i < a.H;
        if (a.post) {
          float y[VEC];
          unpack<VEC>(ry[n], in, y);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[n][e] = r1 * __builtin_fmaf(-c, y[e], d[n][e]);
        }
        if (in) store_bf16<VEC>(a.dy + base, i, d[n]);
      }
    }
    if (!EARLY && row + by < end) fetch(row + by);
    if constexpr (NT > 64) __syncthreads();  // the sums' places are free again
  }
  if constexpr (SUMS) {
    float* to = a.partial + (int64_t)blockIdx.x * 3 * a.H;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
      if (i >= a.H) continue;
      store_f32<VEC>(to, i, dpost[n]);
      store_f32<VEC>(to + a.H, i, dpre[n]);
      if (GATE) store_f32<VEC>(to + 2 * a.H, i, dgate[n]);
    }
  }
}

// The runs' sums joined: 64 columns a workgroup, sixteen of its waves a share of the
// runs each.  blockIdx.y: dpost, dpre, then dgate's rows.
__global__ __launch_bounds__(1024) void norms_join(const float* __restrict__ partial, int64_t H,
                                                   int64_t runs, int64_t groups,
                                                   uint16_t* __restrict__ dpost,
                                                   uint16_t* __restrict__ dpre,
                                                   void* __restrict__ dgate, int gate_f32) {
  __shared__ float red[16][64];
  const int col = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + col, what = blockIdx.y;
  void* out = what == 0 ? dpost : what == 1 ? dpre : dgate;
  if (!out) return;
  const int64_t many = what < 2 ? runs : runs / groups, first = what < 2 ? 0 : (what - 2) * many;
  const int64_t share = (many + 15) / 16, a = part * share, z = min(a + share, many);
  float s = 0.0f;
  if (i < H) {
    const float* p = partial + (first * 3 + (what < 2 ? what : 2)) * H + i;
#pragma unroll 8
    for (int64_t k = a; k < z; ++k) s += p[k * 3 * H];
  }
  red[part][col] = s;
  __syncthreads();
  if (part == 0 && i < H) {
    s = red[0][col];
    for (int k = 1; k < 16; ++k) s += red[k][col];
    const int64_t at = (what < 2 ? 0 : what - 2) * H + i;
    if (what >= 2 && gate_f32)
      ((float*)out)[at] = s;
    else
      ((uint16_t*)out)[at] = st::f32_to_bf16(s);
  }
}

// ---------------------------------------------------------------- host
// Runs of rows in a backward that sums over rows, never across gate rows: as many as
// workgroups run at once, so that none waits for a second turn (2103 rows of 7168: 421
// runs of 5 rows 76 us, 234 of 9 rows 66).
void plan_runs(int64_t rows, int64_t rows_per, int64_t H, int64_t& runs, int64_t& per_run) {
  const int64_t groups = rows / rows_per;
  int64_t each = st::cdiv(H > 4096 ? 256 : 512, groups);
  if (each > rows_per) each = rows_per;
  per_run = st::cdiv(rows_per, each);
  runs = groups * st::cdiv(rows_per, per_run);
}

template <int VEC, int NT, int NV>
void go(const Args& a, bool bwd, bool sums, hipStream_t s) {
  const unsigned grid = (unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20);
  if (!bwd)
    norms_fwd<VEC, NT, NV><<<grid, NT, 0, s>>>(a);
  else if (sums && a.gate)
    norms_bwd<VEC, NT, NV, true, true><<<(unsigned)a.runs, NT, 0, s>>>(a);
  else if (sums)
    norms_bwd<VEC, NT, NV, true, false><<<(unsigned)a.runs, NT, 0, s>>>(a);
  else if (a.gate)
    norms_bwd<VEC, NT, NV, false, true><<<grid, NT, 0, s>>>(a);
  else
    norms_bwd<VEC, NT, NV, false, false><<<grid, NT, 0, s>>>(a);
}

// A row in one wave where it fits (no barriers), in two to sixteen waves otherwise;
// rows of whole 16-byte chunks eight elements a lane at a time, others one by one.  The
// forward and the sums over rows do better with sixteen elements a thread (fewer waves
// at a barrier; 8192 rows of 4096 forward 47 us against 52), the plain backward with
// eight (84 against 95).
void dispatch(const Args& a, bool bwd, bool sums, hipStream_t s) {
  const int64_t H = a.H;
  if (H % 8 == 0) {
    if (H <= 512) go<8, 64, 1>(a, bwd, sums, s);
    else if (H <= 1024) go<8, 128, 1>(a, bwd, sums, s);
    else if (H <= 2048) go<8, 256, 1>(a, bwd, sums, s);
    else if (H <= 4096 && bwd) go<8, 512, 1>(a, bwd, sums, s);
    else if (H <= 4096) go<8, 256, 2>(a, bwd, sums, s);
    else if (H <= 8192 && bwd && !sums) go<8, 1024, 1>(a, bwd, sums, s);
    else if (H <= 8192) go<8, 512, 2>(a, bwd, sums, s);
    else if (bwd && sums) go<8, 512, 4>(a, bwd, sums, s);
    else go<8, 1024, 2>(a, bwd, sums, s);
  } else {
    if (H <= 256) go<1, 64, 4>(a, bwd, sums, s);
    else if (H <= 1024) go<1, 256, 4>(a, bwd, sums, s);
    else if (H <= 4096) go<1, 512, 8>(a, bwd, sums, s);
    else go<1, 1024, 16>(a, bwd, sums, s);
  }
}

int check_args(const Args& a, const char* what) {
  ST_CHECK_ARG(a.rows >= 0 && a.H >= 1, "%s: rows %lld, hidden %lld", what, (long long)a.rows,
               (long long)a.H);
  if (a.H > MAXH)
    return st::fail(ST_EUNSUPPORTED, "%s: hidden size %lld, at most %lld", what, (long long)a.H,
                    (long long)MAXH);
  if (a.rows >= (int64_t)1 << 40)
    return st::fail(ST_EUNSUPPORTED, "%s: 2^40 rows and more", what);
  ST_CHECK_ARG(a.gate_mode >= GATE_NONE && a.gate_mode <= GATE_FULL, "%s: unknown gate", what);
  ST_CHECK_ARG((a.gate_mode == GATE_NONE) == (a.gate == nullptr), "%s: gate and its kind differ",
               what);
  ST_CHECK_ARG(a.gate_mode != GATE_COLUMNS || a.rows == 0 ||
                   (a.rows_per >= 1 && a.rows % a.rows_per == 0),
               "%s: rows of a gate must divide the rows", what);
  ST_CHECK_ARG(std::isfinite(a.scale) && std::isfinite(a.eps) && a.eps >= 0,
               "%s: scale must be finite, eps not negative", what);
  if (a.rows) {
    ST_CHECK_ARG(a.y && a.res, "%s: NULL y or residual", what);
    const uintptr_t all = (uintptr_t)a.y | (uintptr_t)a.res | (uintptr_t)a.post | (uintptr_t)a.pre |
                          (a.gate_mode == GATE_TOKENS ? 0 : (uintptr_t)a.gate) | (uintptr_t)a.h |
                          (uintptr_t)a.normed | (uintptr_t)a.dh | (uintptr_t)a.dn |
                          (uintptr_t)a.dy | (uintptr_t)a.dres |
                          (a.gate_mode == GATE_FULL ? (uintptr_t)a.dgate : 0);
    ST_CHECK_ARG((all & 15) == 0, "%s: tensors must start on 16-byte boundaries", what);
  }
  return ST_OK;
}

}  // namespace

extern "C" int st_residual_norms_fwd(const uint16_t* y, const uint16_t* residual,
                                     const uint16_t* post, const uint16_t* pre, const void* gate,
                                     int32_t gate_mode, int32_t gate_dtype, int64_t rows_per,
                                     int64_t rows, int64_t hidden, float scale, float eps,
                                     uint16_t* h, uint16_t* normed, float* rstd_post,
                                     float* rstd_pre, st_stream_t stream) {
  Args a = {};
  a.y = y, a.res = residual, a.post = post, a.pre = pre, a.gate = gate, a.gate_mode = gate_mode;
  a.gate_f32 = gate_dtype == ST_DTYPE_F32, a.rows_per = rows_per, a.rows = rows, a.H = hidden;
  a.scale = scale, a.eps = eps, a.h = h, a.normed = normed, a.r1 = rstd_post, a.r2 = rstd_pre;
  const int rc = check_args(a, "st_residual_norms_fwd");
  if (rc != ST_OK) return rc;
  if (rows == 0) return ST_OK;
  ST_CHECK_ARG(h && (normed || !pre), "st_residual_norms_fwd: NULL output");
  dispatch(a, false, false, (hipStream_t)stream);
  return st::check_launch("st_residual_norms_fwd");
}

extern "C" int64_t st_residual_norms_workspace_bytes(int64_t rows, int64_t hidden, int64_t rows_per) {
  if (rows < 1 || hidden < 1 || rows_per < 1 || rows % rows_per) return 0;
  int64_t runs, per_run;
  plan_runs(rows, rows_per, hidden, runs, per_run);
  return runs * 3 * hidden * 4;
}

extern "C" int st_residual_norms_bwd(const uint16_t* y, const uint16_t* residual,
                                     const uint16_t* post, const uint16_t* pre, const void* gate,
                                     int32_t gate_mode, int32_t gate_dtype, int64_t rows_per,
                                     int64_t rows, int64_t hidden, float scale, float eps,
                                     const float* rstd_post, const float* rstd_pre,
                                     const uint16_t* dh, const uint16_t* dnormed, uint16_t* dy,
                                     uint16_t* dresidual, void* dgate, uint16_t* dpost, uint16_t* dpre,
                                     void* workspace, int64_t workspace_bytes,
                                     st_stream_t stream) {
  Args a = {};
  a.y = y, a.res = residual, a.post = post, a.pre = pre, a.gate = gate, a.gate_mode = gate_mode;
  a.gate_f32 = gate_dtype == ST_DTYPE_F32, a.rows_per = rows_per, a.rows = rows, a.H = hidden;
  a.scale = scale, a.eps = eps, a.dh = dh, a.dn = dnormed, a.dy = dy, a.dres = dresidual;
  a.r1 = (float*)rstd_post, a.r2 = (float*)rstd_pre, a.dgate = dgate;
  const int rc = check_args(a, "st_residual_norms_bwd");
  if (rc != ST_OK) return rc;
  ST_CHECK_ARG((!post || rstd_post) && (!dnormed || (pre && rstd_pre)),
               "st_residual_norms_bwd: NULL statistics or weight");
  ST_CHECK_ARG((!dpost || post) && (!dpre || dnormed) && (!dgate || gate),
               "st_residual_norms_bwd: a gradient of what is not there");
  if (rows == 0) return ST_OK;
  const bool columns = dgate && gate_mode == GATE_COLUMNS, sums = dpost || dpre || columns;
  if (sums) {
    // gate rows only bound the runs where their sums are asked for
    if (!columns) a.rows_per = gate_mode == GATE_COLUMNS ? rows_per : rows;
    plan_runs(rows, a.rows_per, hidden, a.runs, a.per_run);
    const int64_t need = a.runs * 3 * hidden * 4;
    if (!workspace || workspace_bytes < need)
      return st::fail(ST_EWORKSPACE, "st_residual_norms_bwd needs %lld workspace bytes",
                      (long long)need);
    ST_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
    const int64_t groups = rows / a.rows_per;
    if (a.runs >= (int64_t)1 << 22 || groups + 2 >= 65536)
      return st::fail(ST_EUNSUPPORTED, "st_residual_norms_bwd: 65534 gate rows and more");
    a.partial = (float*)workspace;
    dispatch(a, true, true, (hipStream_t)stream);
    norms_join<<<dim3((unsigned)st::cdiv(hidden, 64), (unsigned)(columns ? groups + 2 : 2)), 1024, 0,
                 (hipStream_t)stream>>>(a.partial, hidden, a.runs, groups, dpost, dpre,
                                        columns ? dgate : nullptr, a.gate_f32);
  } else {
    dispatch(a, true, false, (hipStream_t)stream);
  }
  return st::check_launch("st_residual_norms_bwd");
}
