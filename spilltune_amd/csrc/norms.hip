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
// workgroup walks a run of rows with the columns' sums in registers or LDS, and a
// second kernel joins the runs in their order.
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

// A thread's n-th chunk of a row.  Where the row is no multiple of a chunk (RAG), the last
// chunk is moved back to end with it: its first `skip` elements are the chunk's before,
// worked out and stored by both alike, and counted in no sum here.  Elements past the row
// (`in` false) read its first ones and are cleared: a load under a branch would be waited
// for at the branch's end.  (4096 rows of 4097: 47 us forward, 87 backward; one element a
// load took 640 and 1245.)
struct Place {
  int64_t i;
  bool in;
  int skip;
};
template <int VEC, int NT, bool RAG>
__device__ __forceinline__ Place place(int n, int64_t H) {
  Place c;
  const int64_t i = ((int64_t)n * NT + threadIdx.x) * VEC;
  c.in = i < H;
  c.i = !c.in ? 0 : RAG && i + VEC > H ? H - VEC : i;
  c.skip = RAG && c.in ? (int)(i - c.i) : 0;
  return c;
}
// Ragged rows start on any element.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// VEC bf16 as they lie.
template <int VEC>
struct Raw {
  u32x4 v;
};
template <>
struct Raw<1> {
  uint32_t v;
};
template <int VEC, bool RAG>
__device__ __forceinline__ Raw<VEC> raw(const uint16_t* row, const Place& c) {
  Raw<VEC> r;
  if constexpr (VEC == 1)
    r.v = row[c.i];
  else if constexpr (RAG)
    r.v = *(const u32x4_any*)(row + c.i);
  else
    r.v = *(const u32x4*)(row + c.i);
  return r;
}
template <int VEC>
__device__ __forceinline__ void unpack(const Raw<VEC>& r, bool in, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = in ? r.v[e] : 0;
      f[2 * e] = __uint_as_float(w << 16);
      f[2 * e + 1] = __uint_as_float(w & 0xffff0000u);
    }
  } else {
    f[0] = in ? __uint_as_float(r.v << 16) : 0.0f;
  }
}
template <int VEC, bool RAG>
__device__ __forceinline__ void load_bf16(const uint16_t* row, const Place& c, float (&f)[VEC]) {
  unpack<VEC>(raw<VEC, RAG>(row, c), c.in, f);
}
template <int VEC, bool RAG>
__device__ __forceinline__ void store_bf16(uint16_t* row, const Place& c, const float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    const u32x4 w = {st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3]),
                     st::pack_bf16x2(f[4], f[5]), st::pack_bf16x2(f[6], f[7])};
    if constexpr (RAG)
      *(u32x4_any*)(row + c.i) = w;
    else
      *(u32x4*)(row + c.i) = w;
  } else {
    row[c.i] = st::f32_to_bf16(f[0]);
  }
}
template <int VEC, bool RAG>
__device__ __forceinline__ void load_f32(const float* row, const Place& c, float (&f)[VEC]) {
  const float* p = row + c.i;
  if constexpr (VEC == 8) {
    f32x4 a, b;
    if constexpr (RAG)
      a = *(const f32x4_any*)p, b = *(const f32x4_any*)(p + 4);
    else
      a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
  } else {
    f[0] = *p;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = c.in ? f[e] : 0.0f;
}
template <int VEC, bool RAG>
__device__ __forceinline__ void store_f32(float* row, const Place& c, const float (&f)[VEC]) {
  float* p = row + c.i;
  if constexpr (VEC == 8) {
    const f32x4 a = {f[0], f[1], f[2], f[3]}, b = {f[4], f[5], f[6], f[7]};
    if constexpr (RAG)
      *(f32x4_any*)p = a, *(f32x4_any*)(p + 4) = b;
    else
      *(f32x4*)p = a, *(f32x4*)(p + 4) = b;
  } else {
    p[0] = f[0];
  }
}

// scale * gate of one chunk
template <int VEC, bool RAG>
__device__ __forceinline__ void gate_of(const Args& a, int64_t row, const Place& c,
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
    load_f32<VEC, RAG>((const float*)a.gate + at, c, f);
  else
    load_bf16<VEC, RAG>((const uint16_t*)a.gate + at, c, f);
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] *= a.scale;
}

template <int VEC, int NT, int NV, bool RAG>
__global__ __launch_bounds__(NT) void norms_fwd(Args a) {
  __shared__ float red[2][NT / 64];
  const float over = 1.0f / (float)a.H;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t base = row * a.H;
    float y[NV][VEC], h[NV][VEC];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const Place c = place<VEC, NT, RAG>(n, a.H);
      load_bf16<VEC, RAG>(a.y + base, c, y[n]);
      load_bf16<VEC, RAG>(a.res + base, c, h[n]);
    }
    float r1 = 1.0f;
    if (a.post) {
      float ss = 0.0f;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const Place c = place<VEC, NT, RAG>(n, a.H);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += e < c.skip ? 0.0f : y[n][e] * y[n][e];
      }
      r1 = 1.0f / sqrtf(block_sum<NT>(ss, red[0]) * over + a.eps);
      if (a.r1 && threadIdx.x == 0) a.r1[row] = r1;
    }
    float ss = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const Place c = place<VEC, NT, RAG>(n, a.H);
      float w[VEC], g[VEC];
      if (a.post) load_bf16<VEC, RAG>(a.post, c, w);
      gate_of<VEC, RAG>(a, row, c, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = a.post ? y[n][e] * r1 * w[e] : y[n][e];
        h[n][e] = __builtin_fmaf(g[e], z, h[n][e]);  // as the backward forms it again
        ss += e < c.skip ? 0.0f : h[n][e] * h[n][e];
      }
      if (c.in) store_bf16<VEC, RAG>(a.h + base, c, h[n]);
    }
    if (a.pre) {  // the same way for the whole launch
      const float r2 = 1.0f / sqrtf(block_sum<NT>(ss, red[1]) * over + a.eps);
      if (a.r2 && threadIdx.x == 0) a.r2[row] = r2;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const Place c = place<VEC, NT, RAG>(n, a.H);
        float w[VEC];
        load_bf16<VEC, RAG>(a.pre, c, w);
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[e] *= h[n][e] * r2;
        if (c.in) store_bf16<VEC, RAG>(a.normed + base, c, w);
      }
    }
    if constexpr (NT > 64) __syncthreads();  // the sums' places are free again
  }
}

// SUMS: run blockIdx.x of `per_run` rows (all of one gate row), columns' sums kept.
// GATE: there is one.  Rows wait in registers as the bf16 they are (in fp32, fewer waves
// fit).  The columns' sums of rows over more than one wave lie in LDS, each read and
// written by its own thread alone: in registers they left a CU 8 to 12 waves in the place
// of 16 (8192 x 4096 with learnt norms and gate 140 us, so 105; 2103 x 7168 takes 59).  Rows
// of one wave keep them, and the next row is under way (30000 x 512: 39, in LDS 55).
// Beyond 8192 columns (WIDE) a thread has no registers for its row either: it reads its
// chunks again where it needs them, out of the caches (2048 x 16384: a training pass 165
// us, with all of it in registers 470).
template <int VEC, int NT, int NV, bool SUMS, bool GATE, bool RAG>
__global__ __launch_bounds__(NT, SUMS && NT > 64 && NV == 1 ? 4 : 1) void norms_bwd(Args a) {
  __shared__ float red[3][NT / 64];
  constexpr bool WIDE = NT * NV * VEC > 8192, LDS = SUMS && NT > 64, EARLY = SUMS && !LDS;
  // dpost, dpre and, where there is room, dgate
  constexpr int KEPT = !LDS ? 0 : GATE && !WIDE ? 3 : 2;
  __shared__ f32x4 kept[LDS ? KEPT * NV * VEC / 4 * NT : 1];
  const float over = 1.0f / (float)a.H;
  float dpost[NV][VEC] = {}, dpre[NV][VEC] = {}, dgate[NV][VEC] = {};
  float one[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) one[e] = 1.0f;
  auto add = [&](int which, int n, float (&sum)[VEC], const float (&x)[VEC],
                 const float (&y)[VEC]) {
    if (which < KEPT) {
#pragma unroll
      for (int q = 0; q < VEC / 4; ++q) {
        f32x4& k = kept[((which * NV + n) * (VEC / 4) + q) * NT + threadIdx.x];
        f32x4 v = k;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(x[4 * q + e], y[4 * q + e], v[e]);
        k = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] = __builtin_fmaf(x[e], y[e], sum[e]);
    }
  };
  if constexpr (LDS) {
#pragma unroll
    for (int k = 0; k < KEPT * NV * VEC / 4; ++k) kept[k * NT + threadIdx.x] = f32x4{};
  }
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
    if (WIDE) return;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const Place c = place<VEC, NT, RAG>(n, a.H);
      const int64_t base = r * a.H;
      ny[n] = raw<VEC, RAG>(a.y + base, c);
      nh[n] = raw<VEC, RAG>(a.res + base, c);
      nd[n] = raw<VEC, RAG>(dh + base, c);
      nn[n] = raw<VEC, RAG>(dn + base, c);
    }
  };
  fetch(row);
  for (; row < end; row += by) {
    const int64_t base = row * a.H;
    Raw<VEC> ry[NV], rh[NV], rd[NV], rn[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) ry[n] = ny[n], rh[n] = nh[n], rd[n] = nd[n], rn[n] = nn[n];
    if (EARLY) fetch(row + by < end ? row + by : row);
    auto chunk = [&](const Raw<VEC>(&r)[NV], const uint16_t* p, int n) {
      if constexpr (WIDE)
        return raw<VEC, RAG>(p + base, place<VEC, NT, RAG>(n, a.H));
      else
        return r[n];
    };
    const float r1 = a.post ? a.r1[row] : 1.0f, r2 = has_dn ? a.r2[row] : 0.0f;
    float d[NV][VEC];
    if (has_dn) {
      float h[NV][VEC], gn[NV][VEC], dot = 0.0f;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const Place c = place<VEC, NT, RAG>(n, a.H);
        float y[VEC], w[VEC], g[VEC], p[VEC], hr[VEC];
        unpack<VEC>(chunk(ry, a.y, n), c.in, y);
        unpack<VEC>(chunk(rh, a.res, n), c.in, h[n]);
        unpack<VEC>(chunk(rn, dn, n), c.in, gn[n]);
        if (a.post) load_bf16<VEC, RAG>(a.post, c, w);
        load_bf16<VEC, RAG>(a.pre, c, p);
        if (GATE) gate_of<VEC, RAG>(a, row, c, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float z = a.post ? y[e] * r1 * w[e] : y[e];
          h[n][e] = __builtin_fmaf(GATE ? g[e] : a.scale, z, h[n][e]);
          hr[e] = h[n][e] * r2;
        }
        if constexpr (SUMS) add(1, n, dpre[n], gn[n], hr);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          gn[n][e] *= p[e];
          dot = e < c.skip ? dot : __builtin_fmaf(gn[n][e], h[n][e], dot);
        }
      }
      const float c = block_sum<NT>(dot, red[0]) * over * r2 * r2;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        unpack<VEC>(chunk(rd, dh, n), place<VEC, NT, RAG>(n, a.H).in && has_dh, d[n]);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          d[n][e] = __builtin_fmaf(r2, __builtin_fmaf(-c, h[n][e], gn[n][e]), d[n][e]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        unpack<VEC>(chunk(rd, dh, n), place<VEC, NT, RAG>(n, a.H).in && has_dh, d[n]);
    }
    float dot = 0.0f, gdot = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const Place c = place<VEC, NT, RAG>(n, a.H);
      if (a.dres && c.in) store_bf16<VEC, RAG>(a.dres + base, c, d[n]);
      float y[VEC], yn[VEC], w[VEC], g[VEC], dz[VEC];
      unpack<VEC>(chunk(ry, a.y, n), c.in, y);
      if (a.post) load_bf16<VEC, RAG>(a.post, c, w);
      if (GATE) gate_of<VEC, RAG>(a, row, c, g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        yn[e] = y[e] * r1;
        if (GATE) {
          dz[e] = a.scale * d[n][e] * (a.post ? yn[e] * w[e] : yn[e]);
          gdot += e < c.skip ? 0.0f : dz[e];
        }
        d[n][e] *= GATE ? g[e] : a.scale;
      }
      if constexpr (SUMS && GATE) add(2, n, dgate[n], dz, one);
      if constexpr (SUMS) add(0, n, dpost[n], d[n], yn);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (a.post) d[n][e] *= w[e];
        dot = e < c.skip ? dot : __builtin_fmaf(d[n][e], y[e], dot);
      }
      if (GATE && a.gate_mode == GATE_FULL && a.dgate && c.in) {
        if (a.gate_f32)
          store_f32<VEC, RAG>((float*)a.dgate + base, c, dz);
        else
          store_bf16<VEC, RAG>((uint16_t*)a.dgate + base, c, dz);
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
        const Place at = place<VEC, NT, RAG>(n, a.H);
        if (a.post) {
          float y[VEC];
          unpack<VEC>(chunk(ry, a.y, n), at.in, y);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[n][e] = r1 * __builtin_fmaf(-c, y[e], d[n][e]);
        }
        if (at.in) store_bf16<VEC, RAG>(a.dy + base, at, d[n]);
      }
    }
    if (!EARLY && row + by < end) fetch(row + by);
    if constexpr (NT > 64) __syncthreads();  // the sums' places are free again
  }
  if constexpr (SUMS) {
    float* to = a.partial + (int64_t)blockIdx.x * 3 * a.H;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const Place c = place<VEC, NT, RAG>(n, a.H);
      if (!c.in) continue;
      if constexpr (LDS) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dpost[n][e] = kept[(n * (VEC / 4) + e / 4) * NT + threadIdx.x][e % 4];
          dpre[n][e] = kept[((NV + n) * (VEC / 4) + e / 4) * NT + threadIdx.x][e % 4];
          if (KEPT == 3)
            dgate[n][e] = kept[((2 * NV + n) * (VEC / 4) + e / 4) * NT + threadIdx.x][e % 4];
        }
      }
      store_f32<VEC, RAG>(to, c, dpost[n]);
      store_f32<VEC, RAG>(to + a.H, c, dpre[n]);
      if (GATE) store_f32<VEC, RAG>(to + 2 * a.H, c, dgate[n]);
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
// workgroups run at once, so that none waits for a second turn and no CU idles (30000
// rows of 512: two runs a CU 140 us, twelve 39).  A CU holds 12 waves that keep their sums in
// registers, or 16, or one workgroup beyond 4096 columns.  Runs of at least two rows where
// there are as many: each costs as much as a row again in partial sums.
void plan_runs(int64_t rows, int64_t rows_per, int64_t H, int64_t& runs, int64_t& per_run) {
  const int64_t groups = rows / rows_per;
  const int64_t at_once = H > 4096  ? 256
                          : H > 2048 ? 512
                          : H > 512  ? 256 * 16 / st::cdiv(H, 512)
                                     : 256 * 12;
  int64_t each = st::cdiv(at_once, groups);
  if (each > rows_per / 2) each = rows_per > 1 ? rows_per / 2 : 1;
  per_run = st::cdiv(rows_per, each);
  runs = groups * st::cdiv(rows_per, per_run);
}

template <int VEC, int NT, int NV, bool RAG>
void go(const Args& a, bool bwd, bool sums, hipStream_t s) {
  const unsigned grid = (unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20);
  if (!bwd)
    norms_fwd<VEC, NT, NV, RAG><<<grid, NT, 0, s>>>(a);
  else if (sums && a.gate)
    norms_bwd<VEC, NT, NV, true, true, RAG><<<(unsigned)a.runs, NT, 0, s>>>(a);
  else if (sums)
    norms_bwd<VEC, NT, NV, true, false, RAG><<<(unsigned)a.runs, NT, 0, s>>>(a);
  else if (a.gate)
    norms_bwd<VEC, NT, NV, false, true, RAG><<<grid, NT, 0, s>>>(a);
  else
    norms_bwd<VEC, NT, NV, false, false, RAG><<<grid, NT, 0, s>>>(a);
}

// A row in one wave where it fits (no barriers), in two to sixteen waves otherwise, in
// chunks of eight elements.  From 2049 columns on the forward does better with sixteen
// elements a thread (fewer waves at a barrier; 8192 rows of 4096 47 us against 52), the
// backward with eight (84 against 95).  Rows of fewer than 512 columns leave lanes idle:
// 100000 of 64 take 45 us forward and 59 backward, of 128 46 and 60.
template <bool RAG>
void by_size(const Args& a, bool bwd, bool sums, hipStream_t s) {
  const int64_t H = a.H;
  if (H <= 512) go<8, 64, 1, RAG>(a, bwd, sums, s);
  else if (H <= 1024) go<8, 128, 1, RAG>(a, bwd, sums, s);
  else if (H <= 2048) go<8, 256, 1, RAG>(a, bwd, sums, s);
  else if (H <= 4096 && bwd) go<8, 512, 1, RAG>(a, bwd, sums, s);
  else if (H <= 4096) go<8, 256, 2, RAG>(a, bwd, sums, s);
  else if (H <= 8192 && bwd) go<8, 1024, 1, RAG>(a, bwd, sums, s);
  else if (H <= 8192) go<8, 512, 2, RAG>(a, bwd, sums, s);
  else if (bwd && a.gate) go<8, 512, 4, RAG>(a, bwd, sums, s);
  else go<8, 1024, 2, RAG>(a, bwd, sums, s);
}
void dispatch(const Args& a, bool bwd, bool sums, hipStream_t s) {
  if (a.H < 8) go<1, 64, 1, false>(a, bwd, sums, s);
  else if (a.H % 8 == 0) by_size<false>(a, bwd, sums, s);
  else by_size<true>(a, bwd, sums, s);
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
    // no run crosses a gate row, so that the kernel finds one gate row a run where their
    // sums are asked for (with a frozen gate the same runs)
    if (!columns) a.rows_per = gate_mode == GATE_COLUMNS ? rows_per : rows;
    plan_runs(rows, a.rows_per, hidden, a.runs, a.per_run);
    const int64_t need = a.runs * 3 * hidden * 4;
    if (!workspace || workspace_bytes < need)
      return st::fail(ST_EWORKSPACE, "st_residual_norms_bwd needs %lld workspace bytes",
                      (long long)need);
    ST_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
    const int64_t groups = rows / a.rows_per;
    if (columns && groups + 2 >= 65536)
      return st::fail(ST_EUNSUPPORTED, "st_residual_norms_bwd: 65534 gate rows and more");
    if (a.runs >= (int64_t)1 << 22)
      return st::fail(ST_EUNSUPPORTED, "st_residual_norms_bwd: 2^22 frozen gate rows and more");
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
