// Rotary embedding of a fused q|k|v projection output by per-token positions,
// with the relayout to heads: any rotated part of the head, half or interleaved
// pairs, any frequencies (the caller's scaling for long contexts), optionally
// after each query and key head's RMS norm.  One launch each way.
//
//   n = x * rsqrt(mean(x^2) + eps) * w            (norms only, per head)
//   a' = a cos - b sin,  b' = b cos + a sin       (pairs (a, b) of the rotated part)
//   cos, sin = amplitude * (cos, sin)(position * inv_freq)
//
// The angle of a far position loses all its digits in fp32 (position 10^6 is
// off by up to 0.06 rad), so it is formed and reduced to [-pi, pi] in fp64 and
// only its sine and cosine are fp32.  Everything else is fp32 and rounded to
// bf16 once.  Bound by HBM: each element is read and written once.
//
// A workgroup takes one token and makes its table in LDS once for all heads;
// then each thread turns 8 elements at a time, its pair partners read beside them
// (from L1: the neighbouring thread's elements).  Four tokens a workgroup, for
// longer runs of memory in each head's rows, took 15.1 us against 10.7 for 2048
// tokens of 48 heads of 128, and for 8192 (202 MB; in a trace, cold) 46 against 41
// forward, 41 against 47 back.
#include <algorithm>

#include "common.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_ROT = 256;

struct Rot {
  const uint16_t *x, *wq, *wk;   // token rows (fwd: input; bwd: the forward's, with norms)
  const void* pos;
  const double* inv;
  int64_t ldx, S, total;  // total: tokens
  int heads, kv, D, rot, pos64, inter;
  float amplitude, eps;
};

__device__ __forceinline__ void load8(const uint16_t* p, float (&f)[8]) {
  const uint4 v = *(const uint4*)p;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = __uint_as_float(w[e] << 16);
    f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&f)[8]) {
  *(uint4*)p = make_uint4(st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3]),
                          st::pack_bf16x2(f[4], f[5]), st::pack_bf16x2(f[6], f[7]));
}

// (cos, sin) of token t's angles, [rot/2]
__device__ __forceinline__ void table(const Rot& a, int64_t t, float2* cs) {
  const double p = a.pos64 ? (double)((const int64_t*)a.pos)[t] : (double)((const int32_t*)a.pos)[t];
  for (int i = threadIdx.x; i < a.rot / 2; i += NT) {
    const double angle = p * a.inv[i];
    // 2 pi in two parts; n < 2^31 keeps n * hi within half an ulp of the angle
    const double n = rint(angle * 0.15915494309189535);
    const double r = __builtin_fma(-n, 2.4492935982947064e-16, __builtin_fma(-n, 6.283185307179586, angle));
    float s, c;
    sincosf((float)r, &s, &c);
    cs[i] = make_float2(c * a.amplitude, s * a.amplitude);
  }
}

// f: this chunk's 8 elements, from column d0 of the head; `other(d)` the value
// of column d of the same head; sign = 1 turns forward, -1 back
template <typename F1, typename F8>
__device__ __forceinline__ void turn(const Rot& a, const float2* cs, int d0, float sign, float (&f)[8],
                                     F1&& other, F8&& other8) {
  const int half = a.rot / 2;
  if (d0 >= a.rot) return;
  if (a.inter) {  // d0 is even: a chunk holds whole pairs
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (d0 + 2 * e >= a.rot) break;
      const float2 t = cs[d0 / 2 + e];
      const float u = f[2 * e], w = f[2 * e + 1], sn = t.y * sign;
      f[2 * e] = u * t.x - w * sn;
      f[2 * e + 1] = w * t.x + u * sn;
    }
    return;
  }
  if (half % 8 == 0) {
    const bool first = d0 < half;
    const int j = first ? d0 : d0 - half;
    float o[8];
    other8(first ? d0 + half : j, o);
    const float sg = first ? -sign : sign;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 t = cs[j + e];
      f[e] = f[e] * t.x + o[e] * (t.y * sg);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {  // halves that end inside a chunk
    const int d = d0 + e;
    if (d >= a.rot) break;
    const bool first = d < half;
    const float2 t = cs[first ? d : d - half];
    f[e] = f[e] * t.x + other(first ? d + half : d - half) * (t.y * (first ? -sign : sign));
  }
}

// A launch of 2^32 threads or more in one dimension is refused by the runtime:
// tokens past 2^23 continue in the grid's third.
constexpr int64_t MAX_X = (int64_t)1 << 23;
__device__ __forceinline__ int64_t token_of() {
  return (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
}

// CH: chunks of a head when known (0: a.D / 8)
template <int CH, bool NORM>
__global__ __launch_bounds__(NT) void rope_pos_fwd(Rot a, uint16_t* __restrict__ q,
                                                   uint16_t* __restrict__ k, uint16_t* __restrict__ v,
                                                   float* __restrict__ rstd) {
  __shared__ float2 cs[MAX_ROT / 2];
  const int64_t t = token_of();
  if (t >= a.total) return;  // the whole workgroup
  table(a, t, cs);
  __syncthreads();
  const int ch = CH ? CH : a.D / 8;
  const int64_t b = (unsigned)t / (unsigned)a.S, s = (unsigned)t % (unsigned)a.S;
  const int all = (a.heads + 2 * a.kv) * ch;
  for (int i = blockIdx.y * NT + threadIdx.x; i < all; i += gridDim.y * NT) {
    const int c = i % ch, h = i / ch;
    const uint16_t* x = a.x + t * a.ldx + (int64_t)h * a.D;
    uint16_t* out = h < a.heads ? q + ((b * a.heads + h) * a.S + s) * a.D
                    : h < a.heads + a.kv ? k + ((b * a.kv + h - a.heads) * a.S + s) * a.D
                                         : v + ((b * a.kv + h - a.heads - a.kv) * a.S + s) * a.D;
    if (h >= a.heads + a.kv) {
      *(uint4*)(out + c * 8) = *(const uint4*)(x + c * 8);
      continue;
    }
    float f[8];
    load8(x + c * 8, f);
    float rs = 1.0f;
    const uint16_t* w = h < a.heads ? a.wq : a.wk;
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[e], f[e], ss);
#pragma unroll
      for (int o = CH / 2; o >= 1; o >>= 1) ss += __shfl_xor(ss, o);
      rs = rsqrtf(ss / (float)(CH * 8) + a.eps);
      if (c == 0) rstd[t * (a.heads + a.kv) + h] = rs;
      float g[8];
      load8(w + c * 8, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * rs * g[e];
    }
    turn(a, cs, c * 8, 1.0f, f,
         [&](int d) {
           const float o = st::bf16_to_f32(x[d]);
           return NORM ? o * rs * st::bf16_to_f32(w[d]) : o;
         },
         [&](int d, float (&o)[8]) {
           load8(x + d, o);
           if constexpr (NORM) {
             float g[8];
             load8(w + d, g);
#pragma unroll
             for (int e = 0; e < 8; ++e) o[e] = o[e] * rs * g[e];
           }
         });
    store8(out + c * 8, f);
  }
}

// dx of the above: the turn back, then the norm's VJP
//   dn = w * turned gradient,  dx = rs * (dn - n * mean(dn * n)),  n = x * rs
template <int CH, bool NORM>
__global__ __launch_bounds__(NT) void rope_pos_bwd(Rot a, const uint16_t* __restrict__ dq,
                                                   const uint16_t* __restrict__ dk,
                                                   const uint16_t* __restrict__ dv,
                                                   const float* __restrict__ rstd,
                                                   uint16_t* __restrict__ dx, int64_t lddx) {
  __shared__ float2 cs[MAX_ROT / 2];
  const int64_t t = token_of();
  if (t >= a.total) return;  // the whole workgroup
  table(a, t, cs);
  __syncthreads();
  const int ch = CH ? CH : a.D / 8;
  const int64_t b = (unsigned)t / (unsigned)a.S, s = (unsigned)t % (unsigned)a.S;
  const int all = (a.heads + 2 * a.kv) * ch;
  for (int i = blockIdx.y * NT + threadIdx.x; i < all; i += gridDim.y * NT) {
    const int c = i % ch, h = i / ch;
    const uint16_t* g = h < a.heads ? dq + ((b * a.heads + h) * a.S + s) * a.D
                        : h < a.heads + a.kv ? dk + ((b * a.kv + h - a.heads) * a.S + s) * a.D
                                             : dv + ((b * a.kv + h - a.heads - a.kv) * a.S + s) * a.D;
    uint16_t* out = dx + t * lddx + (int64_t)h * a.D;
    if (h >= a.heads + a.kv) {
      *(uint4*)(out + c * 8) = *(const uint4*)(g + c * 8);
      continue;
    }
    float f[8];
    load8(g + c * 8, f);
    turn(a, cs, c * 8, -1.0f, f, [&](int d) { return st::bf16_to_f32(g[d]); },
         [&](int d, float (&o)[8]) { load8(g + d, o); });
    if constexpr (NORM) {
      float w[8], x[8];
      load8((h < a.heads ? a.wq : a.wk) + c * 8, w);
      load8(a.x + t * a.ldx + (int64_t)h * a.D + c * 8, x);
      const float rs = rstd[t * (a.heads + a.kv) + h];
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] *= w[e];
        x[e] *= rs;
        m = __builtin_fmaf(f[e], x[e], m);
      }
#pragma unroll
      for (int o = CH / 2; o >= 1; o >>= 1) m += __shfl_xor(m, o);
      m /= (float)(CH * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = rs * (f[e] - x[e] * m);
    }
    store8(out + c * 8, f);
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int check_rot(const char* name, Rot& a, const void* positions, int32_t pos64, const double* inv_freq,
              double amplitude, int64_t B, int64_t S, int64_t heads, int64_t kv, int64_t D,
              int64_t rot, int32_t inter, const uint16_t* wq, const uint16_t* wk, float eps) {
  ST_CHECK_ARG(B >= 0 && S >= 0 && heads > 0 && kv > 0, "%s: bad shape", name);
  ST_CHECK_ARG(D > 0 && rot > 0 && rot <= D && rot % 2 == 0,
               "%s: the rotated part (%lld) must be even and within the head (%lld)", name,
               (long long)rot, (long long)D);
  if (D % 8 || D > 512 || rot > MAX_ROT || heads > 4096 || kv > 4096)
    return st::fail(ST_EUNSUPPORTED, "%s: head_dim %lld (multiples of 8 up to 512, rotated part up to %d)",
                    name, (long long)D, MAX_ROT);
  if (S > 0 && B >= ((int64_t)1 << 31) / S)
    return st::fail(ST_EUNSUPPORTED, "%s: 2^31 tokens or more", name);
  ST_CHECK_ARG(!wq == !wk, "%s: norm weights of queries and keys come together", name);
  if (wq && D != 64 && D != 128 && D != 256)
    return st::fail(ST_EUNSUPPORTED, "%s: norms with head_dim %lld (64, 128 or 256)", name, (long long)D);
  if (B == 0 || S == 0) return ST_OK;
  ST_CHECK_ARG(positions && inv_freq && (!wq || (al16(wq) && al16(wk))),
               "%s: NULL or unaligned pointer", name);
  a.wq = wq; a.wk = wk;
  a.pos = positions; a.pos64 = pos64;
  a.inv = inv_freq;
  a.S = S;
  a.total = B * S;
  a.heads = (int)heads; a.kv = (int)kv; a.D = (int)D; a.rot = (int)rot; a.inter = inter;
  a.amplitude = (float)amplitude;
  a.eps = eps;
  return ST_OK;
}

// a token's workgroups: one, or as many as its chunks fill where few tokens
// leave CUs without work (16 tokens of 48 heads of 128: 3.2 us against 4.1; 400:
// 4.7 against 5.0; 600: 5.6 either way)
dim3 grid_of(const Rot& a) {
  const int64_t chunks = (int64_t)(a.heads + 2 * a.kv) * (a.D / 8), x = std::min(a.total, MAX_X);
  return dim3((unsigned)x, (unsigned)(a.total >= 512 ? 1 : st::cdiv(chunks, NT)),
              (unsigned)st::cdiv(a.total, x));
}
template <typename F>
void by_head(const Rot& a, F&& go) {
  const bool norm = a.wq != nullptr;
  switch (a.D) {
    case 64: norm ? go(std::integral_constant<int, 8>{}, std::true_type{})
                  : go(std::integral_constant<int, 8>{}, std::false_type{}); break;
    case 128: norm ? go(std::integral_constant<int, 16>{}, std::true_type{})
                   : go(std::integral_constant<int, 16>{}, std::false_type{}); break;
    case 256: norm ? go(std::integral_constant<int, 32>{}, std::true_type{})
                   : go(std::integral_constant<int, 32>{}, std::false_type{}); break;
    default: go(std::integral_constant<int, 0>{}, std::false_type{});
  }
}

}  // namespace

extern "C" int st_rope_pos_fwd(const uint16_t* x, int64_t ldx, const void* positions, int32_t pos64,
                               const double* inv_freq, double amplitude, int64_t B, int64_t S,
                               int64_t heads, int64_t kv_heads, int64_t D, int64_t rotary_dim,
                               int32_t interleave, const uint16_t* wq, const uint16_t* wk, float eps,
                               uint16_t* q, uint16_t* k, uint16_t* v, float* rstd,
                               st_stream_t stream) {
  const char* name = "st_rope_pos_fwd";
  Rot a{};
  if (int rc = check_rot(name, a, positions, pos64, inv_freq, amplitude, B, S, heads, kv_heads, D,
                         rotary_dim, interleave, wq, wk, eps)) return rc;
  if (B == 0 || S == 0) return ST_OK;
  ST_CHECK_ARG(x && q && k && v && (!wq || rstd) && al16(x) && al16(q) && al16(k) && al16(v) &&
                   ldx % 8 == 0 && ldx >= (heads + 2 * kv_heads) * D,
               "%s: NULL or unaligned pointer, or rows below (heads + 2 kv_heads) * head_dim", name);
  a.x = x;
  a.ldx = ldx;
  by_head(a, [&](auto ch, auto norm) {
    rope_pos_fwd<decltype(ch)::value, decltype(norm)::value>
        <<<grid_of(a), NT, 0, (hipStream_t)stream>>>(a, q, k, v, rstd);
  });
  return st::check_launch(name);
}

extern "C" int st_rope_pos_bwd(const uint16_t* dq, const uint16_t* dk, const uint16_t* dv,
                               const uint16_t* x, int64_t ldx, const void* positions, int32_t pos64,
                               const double* inv_freq, double amplitude, int64_t B, int64_t S,
                               int64_t heads, int64_t kv_heads, int64_t D, int64_t rotary_dim,
                               int32_t interleave, const uint16_t* wq, const uint16_t* wk,
                               const float* rstd, uint16_t* dx, int64_t lddx, st_stream_t stream) {
  const char* name = "st_rope_pos_bwd";
  Rot a{};
  if (int rc = check_rot(name, a, positions, pos64, inv_freq, amplitude, B, S, heads, kv_heads, D,
                         rotary_dim, interleave, wq, wk, 0.0f)) return rc;
  if (B == 0 || S == 0) return ST_OK;
  const int64_t width = (heads + 2 * kv_heads) * D;
  ST_CHECK_ARG(dq && dk && dv && dx && al16(dq) && al16(dk) && al16(dv) && al16(dx) &&
                   lddx % 8 == 0 && lddx >= width,
               "%s: NULL or unaligned pointer, or rows below (heads + 2 kv_heads) * head_dim", name);
  ST_CHECK_ARG(!wq || (x && rstd && al16(x) && ldx % 8 == 0 && ldx >= width),
               "%s: norms need the forward's rows and rstd", name);
  a.x = x;
  a.ldx = ldx;
  by_head(a, [&](auto ch, auto norm) {
    rope_pos_bwd<decltype(ch)::value, decltype(norm)::value>
        <<<grid_of(a), NT, 0, (hipStream_t)stream>>>(a, dq, dk, dv, rstd, dx, lddx);
  });
  return st::check_launch(name);
}
