// Log probabilities of given tokens under the vocabulary head, with entropy and
// top alternatives, and the gradient of the hidden states.
//
//   l = hidden head^T,  x = cap * tanh(l / cap) / temperature
//   logprob = x_y - lse(x),  entropy = lse(x) - sum_c p_c x_c,  p = softmax(x)
//   dx_c = g_lp ([c = y] - p_c) + sum_j g_top_j ([c = top_j] - p_c)
//          - g_ent p_c (x_c - lse + entropy)
//   dl = dx (1 - tanh^2) / temperature,  dhidden = dl head
//
// Forward: one pass over the head.  The GEMM's tiles (bf16 products, fp32 sums)
// are reduced in registers: each tile of 256 vocabulary columns reduces its x to
// (max, sum of e^(x - max), sum of e^(x - max) (x - max)) per row, and a second
// kernel joins the tiles.  All three are kept relative to the maximum, so
// nothing cancels: the entropy is log(sum) less a sum of terms below zero.
// The vocabulary is the GEMM's row axis, so a lane owns token columns and its
// reductions run down its own accumulators (two exchanges between lanes per
// token; the other way round took four for each of its 32 rows).
// Top alternatives are chosen on l before cap and temperature (ties to the
// lowest index): only then, or for a caller that keeps them for the backward, the
// tiles also write l (fp32); the join reads back just the tiles that hold the
// largest maxima.
//
// Backward: l read back, or formed again by the same GEMM, becomes dl (bf16: a
// choice, half a step of 2^-8 on values that are then summed over the
// vocabulary); the given token's and the alternatives' entries, the large ones,
// come from the saved log probabilities, and what their rounding leaves is kept in
// fp32.  dl head is a GEMM split over the vocabulary so
// that few rows fill the GPU; its fp32 partials are summed in order and the
// picked entries' remainders times their rows of the head added.
#include <algorithm>
#include <cmath>

#include "gemm_dma.h"

namespace {

constexpr int NT = 256;
constexpr int VT = 256;  // vocabulary columns of a tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Transform {
  float cap, inv_cap, inv_t;  // cap = 0: none
};

// tanh: an odd polynomial up to 0.625 (least squares on Chebyshev points,
// reweighted to level the relative error: 7e-8), 1 - 2 / (1 + e^2y) beyond
__device__ __forceinline__ float tanh32(float y) {
  const float z = y * y;
  float p = -0.005704985465854406f;
  p = __builtin_fmaf(p, z, 0.02063908614218235f);
  p = __builtin_fmaf(p, z, -0.05373971536755562f);
  p = __builtin_fmaf(p, z, 0.13331441581249237f);
  p = __builtin_fmaf(p, z, -0.3333328068256378f);
  const float small = __builtin_fmaf(y * z, p, y);
  const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * (2.0f * LOG2E)));
  return fabsf(y) <= 0.625f ? small : __builtin_fmaf(-2.0f, r, 1.0f);
}
__device__ __forceinline__ float value(const Transform& t, float l) {
  if (t.cap != 0.0f) l = t.cap * tanh32(l * t.inv_cap);
  return l * t.inv_t;
}
// d x / d l
__device__ __forceinline__ float slope(const Transform& t, float l) {
  if (t.cap == 0.0f) return t.inv_t;
  const float y = tanh32(l * t.inv_cap);
  return (1.0f - y) * (1.0f + y) * t.inv_t;
}

// A part of a row: its maximum, the sum of e^(x - max) less the maximum's own 1,
// the sum of e^(x - max) (x - max).  Without the 1 a sure token keeps the digits
// of the others' sum, and so does log1p of it.  A part of -inf alone (or of
// nothing) has rest = -1.
struct Stats {
  float m, rest, u;
};
__device__ __forceinline__ Stats join(Stats a, Stats b) {
  const Stats hi = a.m >= b.m ? a : b, lo = a.m >= b.m ? b : a;
  const float all = 1.0f + lo.rest;
  // nothing but -inf adds nothing (0 * -inf is not a number), but NaN its NaN
  if (lo.m == -INFINITY) return {hi.m, hi.rest + all, hi.u};
  const float d = lo.m - hi.m, f = __builtin_amdgcn_exp2f(d * LOG2E);
  return {hi.m, __builtin_fmaf(f, all, hi.rest), __builtin_fmaf(f, __builtin_fmaf(d, all, lo.u), hi.u)};
}

struct Head {
  const uint16_t *hidden, *head;
  const int64_t* tokens;
  int64_t ldh, ldw, rows, V;
  int H, vtiles, rtiles;
  Transform tf;
};

// Tile of a workgroup: the row tiles of one vocabulary tile one after the other
// on one XCD, so its L2 serves that panel of the head to all of them.
__device__ __forceinline__ bool tile_of(const Head& h, int64_t& vt, int64_t& rt) {
  const unsigned t = st::xcd_remap(blockIdx.x, gridDim.x);  // the grid is a multiple of 8
  vt = t / (unsigned)h.rtiles;
  rt = t % (unsigned)h.rtiles;
  return vt < h.vtiles;
}
template <class LP>
__device__ __forceinline__ void products(const Head& h, int64_t vt, int64_t rt, uint4* lds, int wave,
                                         int lane, int& vn, int& rn, f32x4 (&acc)[LP::FM][LP::FN]) {
  const int64_t v0 = vt * LP::BM, r0 = rt * LP::BN;
  vn = (int)min((int64_t)LP::BM, h.V - v0);
  rn = (int)min((int64_t)LP::BN, h.rows - r0);
  const st::DmaOperands o{h.head + v0 * h.ldw, h.hidden + r0 * h.ldh, h.ldw, h.ldh,
                          ((vn - 1) * h.ldw + h.H) * 2, ((rn - 1) * h.ldh + h.H) * 2};
  LP::run(o, lds, 0, vn, 0, rn, h.H, wave, lane, acc);
}

// part[row][vtile] = (Stats of x, max of l); xy[row] = x of the given token.
// Many rows are bound by the matrix pipes: 2048 x 4096 x 151936 in 2.10 ms, 1.21
// PFLOP/s, as the library's large product.  Few rows are bound by reading the head:
// 61 x 7168 x 129280 in 324 us, 5.7 TB/s; 5 x 1024 x 32000 (125 tiles, 65 MB) in
// 20 us, 3.3 TB/s.
template <class LP>
__global__ __launch_bounds__(LP::NT, LP::MIN_WG_WAVES) void lp_tiles(Head h, float4* __restrict__ part,
                                                                     float* __restrict__ xy,
                                                                     float* __restrict__ logits,
                                                                     int64_t ldl, int top) {
  constexpr int WMS = LP::WAVES / LP::WAVES_N;
  __shared__ uint4 lds[LP::LDS16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t vt, rt;
  if (!tile_of(h, vt, rt)) return;
  int vn, rn;
  f32x4 acc[LP::FM][LP::FN];
  products<LP>(h, vt, rt, lds, wave, lane, vn, rn, acc);

  const int wm = wave / LP::WAVES_N, wn = wave % LP::WAVES_N, lr = lane & 15, lh = lane >> 4;
  const int64_t v0 = vt * LP::BM, r0 = rt * LP::BN;
  const int vw = wm * LP::WM + lh * 4;  // this lane's first column of the tile
  float4* red = (float4*)lds;           // [WMS][BN]
#pragma unroll
  for (int j = 0; j < LP::FN; ++j) {
    const int r = wn * LP::WN + j * 16 + lr;
    const int64_t row = r0 + r;
    const bool in = r < rn;
    if (logits && in) {
#pragma unroll
      for (int i = 0; i < LP::FM; ++i)
        if (vw + i * 16 < vn)  // rows of `logits` are padded to whole float4
          *(float4*)(logits + row * ldl + v0 + vw + i * 16) =
              make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
    }
    float raw = -INFINITY, m = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP::FM; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const bool ok = vn == LP::BM || vw + i * 16 + v < vn;
        if (top) raw = fmaxf(raw, ok ? acc[i][j][v] : -INFINITY);
        const float x = value(h.tf, acc[i][j][v]);
        acc[i][j][v] = ok ? x : -INFINITY;
        m = fmaxf(m, acc[i][j][v]);
      }
    const int64_t y = in ? h.tokens[row] - v0 - vw : -1;  // the given token's place in this lane
    if (y >= 0 && y < LP::WM && (y & 15) < 4) {
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < LP::FM; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) x = y == i * 16 + v ? acc[i][j][v] : x;
      xy[row] = x;
    }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float base = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < LP::FM; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float d = acc[i][j][v] - base, e = __builtin_amdgcn_exp2f(d * LOG2E);
        s += e;
        u = __builtin_fmaf(e, fmaxf(d, -1e30f), u);  // 0 for x = -inf, not 0 * -inf
      }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    u += __shfl_xor(u, 16);
    u += __shfl_xor(u, 32);
    float rest = s - 1.0f;
    if (__ballot(s < 1.0078125f)) {  // some token's others have lost digits to its 1
      float ties = 0.0f, less = 0.0f;
#pragma unroll
      for (int i = 0; i < LP::FM; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float d = acc[i][j][v] - base;
          less += d < 0.0f ? __builtin_amdgcn_exp2f(d * LOG2E) : 0.0f;
          ties += d == 0.0f ? 1.0f : 0.0f;
        }
      less += __shfl_xor(less, 16);
      less += __shfl_xor(less, 32);
      ties += __shfl_xor(ties, 16);
      ties += __shfl_xor(ties, 32);
      if (s < 1.0078125f) rest = less + (ties - 1.0f);
    }
    if (top) {
      raw = fmaxf(raw, __shfl_xor(raw, 16));
      raw = fmaxf(raw, __shfl_xor(raw, 32));
    }
    if (lh == 0) red[wm * LP::BN + r] = make_float4(m, rest, u, raw);
  }
  __syncthreads();
  for (int r = tid; r < rn; r += LP::NT) {
    const float4 a = red[r];
    Stats x{a.x, a.y, a.z};
    float raw = a.w;
#pragma unroll
    for (int w = 1; w < WMS; ++w) {
      const float4 b = red[w * LP::BN + r];
      x = join(x, {b.x, b.y, b.z});
      raw = fmaxf(raw, b.w);
    }
    part[(r0 + r) * h.vtiles + vt] = make_float4(x.m, x.rest, x.u, raw);
  }
}

// Maximum over the wave without LDS: within rows of 16 lanes, then across them;
// the last lane holds it.  (No NaN comes here.)
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_from(float x) {
  const int v = __float_as_int(x);
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = max_from<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8
  x = max_from<0x112, 0xf>(x);
  x = max_from<0x114, 0xf>(x);
  x = max_from<0x118, 0xf>(x);
  x = max_from<0x142, 0xa>(x);  // row_bcast:15, 31
  x = max_from<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
// the first lane that holds the greatest value
__device__ __forceinline__ int first_of(float x, float most) {
  return __ffsll((unsigned long long)__ballot(x == most)) - 1;
}

// Bound by the latency of a row's reads, one after the other: 9 us for 5 rows of
// 125 tiles and five alternatives, 22 us for 1000 rows of 501 tiles and eight.
// One wave a row: joins the tiles, then picks `top` alternatives one by one
// from the tile with the greatest value left.
__global__ __launch_bounds__(NT) void lp_join(Head h, int64_t ignore, const float4* __restrict__ part,
                                              const float* __restrict__ xy,
                                              const float* __restrict__ logits, int64_t ldl, int top,
                                              float* __restrict__ logprobs, float* __restrict__ entropy,
                                              float* __restrict__ lse, float* __restrict__ top_lp,
                                              int64_t* __restrict__ top_idx) {
  extern __shared__ float tile_max[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * (NT / 64) + wave;
  if (row >= h.rows) return;
  float* tm = tile_max + (int64_t)wave * h.vtiles;
  const float4* p = part + row * h.vtiles;
  Stats a{-INFINITY, -1.0f, 0.0f};
  for (int t = lane; t < h.vtiles; t += 64) {
    const float4 x = p[t];
    a = join(a, {x.x, x.y, x.z});
    if (top) tm[t] = x.w;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1)
    a = join(a, {__shfl_xor(a.m, d), __shfl_xor(a.rest, d), __shfl_xor(a.u, d)});
  const float logs = log1pf(a.rest), nan = __uint_as_float(0x7fc00000u);
  if (lane == 0) {
    const int64_t y = h.tokens[row];
    logprobs[row] = y == ignore ? 0.0f : y >= 0 && y < h.V ? (xy[row] - a.m) - logs : nan;
    entropy[row] = logs - a.u / (1.0f + a.rest);
    lse[row] = a.m + logs;
  }
  // a lane's tiles are neighbours: the first lane with a maximum has the lowest
  // index, of tiles as of columns
  const int per = (h.vtiles + 63) / 64, t0 = lane * per, t1 = min(t0 + per, h.vtiles);
  __builtin_amdgcn_s_waitcnt(0);
  __builtin_amdgcn_wave_barrier();
  float lv = INFINITY;  // the last pick: what is left comes after it
  int li = -1;
  for (int k = 0; k < top; ++k) {
    float bv = -INFINITY;
    int bt = 0;
    for (int t = t0; t < t1; ++t)
      if (tm[t] > bv) {
        bv = tm[t];
        bt = t;
      }
    const float best = wave_max(bv);
    if (!(best > -INFINITY)) {  // nothing left that is a number
      if (lane == 0) {
        top_lp[row * top + k] = nan;
        top_idx[row * top + k] = -1;
      }
      continue;
    }
    bt = __builtin_amdgcn_readlane(bt, first_of(bv, best));
    constexpr int PER = VT / 64;
    const int c0 = bt * VT + lane * PER;
    float f[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) f[e] = -INFINITY;
    if (c0 < h.V) {  // rows of `logits` are padded to whole float4
      typedef float fv __attribute__((ext_vector_type(PER)));
      const fv x = *(const fv*)(logits + row * ldl + c0);
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (c0 + e < h.V && (x[e] < lv || (x[e] == lv && c0 + e > li))) f[e] = x[e];
    }
    float v = -INFINITY;
    int i = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (f[e] > v) {
        v = f[e];
        i = c0 + e;
      }
    li = __builtin_amdgcn_readlane(i, first_of(v, best));
    lv = best;  // the tile's maximum is one of its columns
    float next = -INFINITY;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (c0 + e != li) next = fmaxf(next, f[e]);
    next = wave_max(next);
    if (lane == 0) {
      tm[bt] = next;
      top_lp[row * top + k] = (value(h.tf, lv) - a.m) - logs;
      top_idx[row * top + k] = li;
    }
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_wave_barrier();
  }
}

// Upstream gradients of a row: its sum over the picked tokens, and the entropy's.
struct Upstream {
  const float *lp, *ent, *top;  // each may be NULL
  int ntop;
};
__device__ __forceinline__ float given(const Head& h, const Upstream& g, int64_t row, int64_t ignore) {
  return g.lp && h.tokens[row] != ignore ? g.lp[row] : 0.0f;
}

// (sum over the picked, of the entropy, lse, entropy) of a row
__device__ __forceinline__ float4 upstream(const Head& h, const Upstream& g, int64_t row, int64_t ignore,
                                           const int64_t* top_idx, const float* lse, const float* ent) {
  float sum = given(h, g, row, ignore);
  if (g.top)
    for (int k = 0; k < g.ntop; ++k)
      sum += top_idx[row * g.ntop + k] >= 0 ? g.top[row * g.ntop + k] : 0.0f;
  return make_float4(sum, g.ent ? g.ent[row] : 0.0f, lse[row], ent[row]);
}
// dl of a logit but for a picked token's own term; a row without an upstream
// gradient has none, whatever it holds
__device__ __forceinline__ float dlogit(const Transform& t, float4 c, float l) {
  const float lp = value(t, l) - c.z, p = __builtin_amdgcn_exp2f(lp * LOG2E);
  const float d = -p * __builtin_fmaf(c.y, lp + c.w, c.x) * slope(t, l);
  return c.x == 0.0f && c.y == 0.0f ? 0.0f : d;
}

// Column of pick k of a row (alternative k, or the given token for k = ntop), -1
// for none.
struct Picks {
  const int64_t* top_idx;
  const float *top_lp, *logprobs, *lse, *ent;
};
__device__ __forceinline__ int64_t column_of(const Head& h, const Upstream& g, int64_t ignore,
                                             const Picks& p, int64_t row, int k) {
  if (k < g.ntop) return p.top_idx[row * g.ntop + k];
  const int64_t y = h.tokens[row];
  return y != ignore && y >= 0 && y < h.V ? y : -1;
}
// dl of pick k, in column c of logit l (read with a cap only), from the saved log
// probability; a token picked twice gets one value from both.  Returns whether the
// entry is to be replaced; `left`: what its rounding leaves, once for each entry.
// (The tanh is not taken back from lp + lse: those are of the size of log V, and a
// temperature far above the cap would multiply their rounding.)
__device__ __forceinline__ bool picked(const Head& h, const Upstream& g, int64_t ignore, const Picks& p,
                                       int64_t row, int k, int64_t c, float l, uint16_t& value,
                                       float& left) {
  left = 0.0f;
  const int64_t y = column_of(h, g, ignore, p, row, g.ntop);
  const float lp = k < g.ntop ? p.top_lp[row * g.ntop + k] : p.logprobs[row];
  const float own_lp = given(h, g, row, ignore);
  float sum = own_lp, own = c == y ? own_lp : 0.0f;
  bool again = false;  // the given token among the alternatives
  for (int j = 0; j < g.ntop; ++j) {
    const int64_t t = p.top_idx[row * g.ntop + j];
    const float w = g.top ? g.top[row * g.ntop + j] : 0.0f;
    if (t >= 0) sum += w;
    if (t == c) own += w;
    again |= k == g.ntop && t == c;
  }
  const float pr = __builtin_amdgcn_exp2f(lp * LOG2E), ge = g.ent ? g.ent[row] : 0.0f;
  if (own == 0.0f && sum == 0.0f && ge == 0.0f) return false;  // as the other columns
  const float d = (own - pr * __builtin_fmaf(ge, lp + p.ent[row], sum)) * slope(h.tf, l);
  value = st::f32_to_bf16(d);
  if (!again) left = d - st::bf16_to_f32(value);
  return true;
}

// dl from logits formed again
template <class LP>
__global__ __launch_bounds__(LP::NT, LP::MIN_WG_WAVES) void lp_dlogits(Head h, Upstream g,
                                                                       int64_t ignore,
                                                                       const int64_t* __restrict__ top_idx,
                                                                       const float* __restrict__ lse,
                                                                       const float* __restrict__ ent,
                                                                       uint16_t* __restrict__ dl,
                                                                       int64_t ldd) {
  __shared__ uint4 lds[LP::LDS16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t vt, rt;
  if (!tile_of(h, vt, rt)) return;
  int vn, rn;
  f32x4 acc[LP::FM][LP::FN];
  products<LP>(h, vt, rt, lds, wave, lane, vn, rn, acc);

  const int wm = wave / LP::WAVES_N, wn = wave % LP::WAVES_N, lr = lane & 15, lh = lane >> 4;
  const int64_t v0 = vt * LP::BM, r0 = rt * LP::BN;
  float4* up = (float4*)lds;
  for (int r = tid; r < rn; r += LP::NT) up[r] = upstream(h, g, r0 + r, ignore, top_idx, lse, ent);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < LP::FN; ++j) {
    const int r = wn * LP::WN + j * 16 + lr;
    if (r >= rn) continue;
    const float4 c = up[r];
    uint16_t* out = dl + (r0 + r) * ldd + v0 + wm * LP::WM + lh * 4;
#pragma unroll
    for (int i = 0; i < LP::FM; ++i) {
      const int col = wm * LP::WM + lh * 4 + i * 16;
      float d[4];
#pragma unroll
      for (int v = 0; v < 4; ++v)  // a column past the vocabulary (up to the row's padding) gets 0
        d[v] = col + v < vn ? dlogit(h.tf, c, acc[i][j][v]) : 0.0f;
      if (v0 + col < ldd)
        *(uint2*)(out + i * 16) = make_uint2(st::pack_bf16x2(d[0], d[1]), st::pack_bf16x2(d[2], d[3]));
    }
  }
}
// dl from kept logits, the picked entries in the same pass (by the thread that
// holds the column): 4 + 2 bytes a logit, bound by HBM (2048 x 151936: 297 us,
// 6.3 TB/s)
constexpr int KEPT = 8;  // logits of a thread
__global__ __launch_bounds__(NT) void lp_dlogits_kept(Head h, Upstream g, int64_t ignore, Picks p,
                                                      const float* __restrict__ logits, int64_t ldl,
                                                      uint16_t* __restrict__ dl, int64_t ldd,
                                                      float* __restrict__ left) {
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= h.rows) return;
  const float4 c = upstream(h, g, row, ignore, p.top_idx, p.lse, p.ent);
  const int64_t c0 = ((int64_t)blockIdx.x * NT + threadIdx.x) * KEPT;
  if (c0 >= ldd) return;
  float l[KEPT], d[KEPT];
#pragma unroll
  for (int e = 0; e < KEPT; e += 4) {
    float4 x = make_float4(0, 0, 0, 0);
    if (c0 + e < ldl) x = *(const float4*)(logits + row * ldl + c0 + e);
    l[e] = x.x; l[e + 1] = x.y; l[e + 2] = x.z; l[e + 3] = x.w;
  }
#pragma unroll
  for (int e = 0; e < KEPT; ++e) d[e] = c0 + e < h.V ? dlogit(h.tf, c, l[e]) : 0.0f;
  for (int k = 0; k <= g.ntop; ++k) {
    const int64_t at = column_of(h, g, ignore, p, row, k);
    if (at < 0 ? c0 != 0 : at < c0 || at >= c0 + KEPT) continue;
    uint16_t value;
    float rest = 0.0f;
    float raw = 0.0f;
#pragma unroll
    for (int e = 0; e < KEPT; ++e)
      if (at == c0 + e) raw = l[e];
    if (at >= 0 && picked(h, g, ignore, p, row, k, at, raw, value, rest)) {
#pragma unroll
      for (int e = 0; e < KEPT; ++e)
        if (at == c0 + e) d[e] = st::bf16_to_f32(value);
    }
    left[row * (g.ntop + 1) + k] = rest;
  }
  *(uint4*)(dl + row * ldd + c0) = make_uint4(st::pack_bf16x2(d[0], d[1]), st::pack_bf16x2(d[2], d[3]),
                                              st::pack_bf16x2(d[4], d[5]), st::pack_bf16x2(d[6], d[7]));
}

// the picked tokens' entries whole, over what lp_dlogits wrote: thread k of a row
// takes pick k; with a cap wave k does, and forms the logit again.  left[row][k]:
// see picked
template <bool CAP>
__global__ __launch_bounds__(NT) void lp_picked(Head h, Upstream g, int64_t ignore, Picks p,
                                                uint16_t* __restrict__ dl, int64_t ldd,
                                                float* __restrict__ left) {
  constexpr int OF = CAP ? 64 : 1;  // threads of a pick
  const int per = g.ntop + 1, lane = threadIdx.x & 63;
  for (int64_t n = ((int64_t)blockIdx.x * NT + threadIdx.x) / OF; n < h.rows * per;
       n += (int64_t)gridDim.x * NT / OF) {
    const int64_t row = n / per;
    const int k = (int)(n % per);
    const int64_t c = column_of(h, g, ignore, p, row, k);
    float l = 0.0f;
    if (CAP && c >= 0) {
      for (int i = lane * 8; i < h.H; i += 64 * 8) {
        const uint4 a = *(const uint4*)(h.hidden + row * h.ldh + i);
        const uint4 b = *(const uint4*)(h.head + c * h.ldw + i);
        const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          l = __builtin_fmaf(__uint_as_float(x[e] << 16), __uint_as_float(y[e] << 16), l);
          l = __builtin_fmaf(__uint_as_float(x[e] & 0xffff0000u), __uint_as_float(y[e] & 0xffff0000u), l);
        }
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
    }
    if (CAP && lane != 0) continue;
    uint16_t value;
    float rest = 0.0f;
    if (c >= 0 && picked(h, g, ignore, p, row, k, c, l, value, rest)) dl[row * ldd + c] = value;
    left[n] = rest;
  }
}

// dhidden partials: part[split][row][h] = sum over the split's columns of dl head.
// 2048 x 151936 x 4096: 1.71 ms, 1.49 PFLOP/s; 61 x 129280 x 7168: 318 us, 5.8 TB/s
// of the head.
struct Dgrad {
  const uint16_t *dl, *head;
  int64_t ldd, ldw, rows, V;
  int H, rtiles, htiles, splits;
  int64_t per;  // columns of a split, a multiple of 64
};
template <class LP>
__global__ __launch_bounds__(LP::NT, LP::MIN_WG_WAVES) void lp_dhidden(Dgrad g, float* __restrict__ part) {
  __shared__ uint4 lds[LP::LDS16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the tiles of one split one after the other on one XCD: they share its rows
  const unsigned t = st::xcd_remap(blockIdx.x, gridDim.x);
  const unsigned tiles = (unsigned)g.rtiles * g.htiles, sp = t / tiles, in = t % tiles;
  if (sp >= (unsigned)g.splits) return;
  const int64_t r0 = (int64_t)(in % g.rtiles) * LP::BM, c0 = (int64_t)(in / g.rtiles) * LP::BN;
  const int64_t q0 = sp * g.per;
  const int qn = (int)max((int64_t)0, min(g.per, g.V - q0));
  const int rn = (int)min((int64_t)LP::BM, g.rows - r0), cn = (int)min((int64_t)LP::BN, g.H - c0);
  const st::DmaOperands o{g.dl + r0 * g.ldd + q0, g.head + q0 * g.ldw + c0, g.ldd, g.ldw,
                          // whole 16-byte chunks of dl: its rows are padded with zeros
                          ((rn - 1) * g.ldd + (qn + 7) / 8 * 8) * 2, qn ? ((qn - 1) * g.ldw + cn) * 2 : 0};
  f32x4 acc[LP::FM][LP::FN];
  LP::run(o, lds, 0, rn, 0, cn, qn, wave, lane, acc);
  const int wm = wave / LP::WAVES_N, wn = wave % LP::WAVES_N, lr = lane & 15, lh = lane >> 4;
  float* out = part + (sp * g.rows + r0) * g.H + c0;
#pragma unroll
  for (int i = 0; i < LP::FM; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = wm * LP::WM + i * 16 + lh * 4 + v;
#pragma unroll
      for (int j = 0; j < LP::FN; ++j) {
        const int c = wn * LP::WN + j * 16 + lr;
        if (r < rn && c < cn) out[(int64_t)r * g.H + c] = acc[i][j][v];
      }
    }
}
// dhidden = the splits' sums in order, and the picked entries' remainders
__global__ __launch_bounds__(NT) void lp_reduce(Head h, const float* __restrict__ part, int splits,
                                                const float* __restrict__ left, int ntop,
                                                const int64_t* __restrict__ top_idx,
                                                uint16_t* __restrict__ out, int64_t ldo) {
  const int64_t per = h.rows * h.H, n = per / 4;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < n; i += (int64_t)gridDim.x * NT) {
    const int64_t row = i * 4 / h.H, col = i * 4 % h.H;
    float4 s = make_float4(0, 0, 0, 0);
    auto add = [&](const float4& x) { s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w; };
    int k = 0;
    for (; k + 8 <= splits; k += 8) {  // eight reads in flight, added in order
      float4 x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = *(const float4*)(part + (k + e) * per + i * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) add(x[e]);
    }
    for (; k < splits; ++k) add(*(const float4*)(part + k * per + i * 4));
    for (int k = 0; k <= ntop; ++k) {
      const float w = left[row * (ntop + 1) + k];
      if (w == 0.0f) continue;
      const int64_t c = k < ntop ? top_idx[row * ntop + k] : h.tokens[row];
      const uint2 x = *(const uint2*)(h.head + c * h.ldw + col);
      s.x = __builtin_fmaf(w, __uint_as_float(x.x << 16), s.x);
      s.y = __builtin_fmaf(w, __uint_as_float(x.x & 0xffff0000u), s.y);
      s.z = __builtin_fmaf(w, __uint_as_float(x.y << 16), s.z);
      s.w = __builtin_fmaf(w, __uint_as_float(x.y & 0xffff0000u), s.w);
    }
    *(uint2*)(out + row * ldo + col) = make_uint2(st::pack_bf16x2(s.x, s.y), st::pack_bf16x2(s.z, s.w));
  }
}

// ---------------------------------------------------------------- host
bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Row tile of the vocabulary GEMM: cost of a k-step of its 256-column tile
// relative to 256 rows (a 256x128 tile takes 0.57 of it; a 256x64 one is bound
// by the head's rows, 0.4).
// (64 rows with 128 columns and a deeper ring, so that a vocabulary of 32000
// fills the CUs, took as long: 20.5 against 20.4 us for 5 x 1024.)
int row_tile(int64_t rows) {
  const double c256 = (double)st::cdiv(rows, 256), c128 = 0.57 * (double)st::cdiv(rows, 128),
               c64 = 0.4 * (double)st::cdiv(rows, 64);
  return c64 <= c128 && c64 <= c256 ? 64 : c128 <= c256 ? 128 : 256;
}

// Tile and split of dl head: rounds of 256 workgroups, each a split's k-steps
// and about 10 of fill, at the tile's microseconds a k-step, and the partials'
// traffic; a split's rows of the head stay within a 32-bit byte offset.
struct Split {
  int bm, bn, splits;
  int64_t per;
};
Split split_of(int64_t rows, int64_t H, int64_t ldw, int64_t V) {
  struct Kind {
    int bm, bn;
    double us;
  };
  static const Kind kinds[] = {{256, 256, 1.35}, {256, 128, 0.8}, {64, 256, 0.55}};
  const int64_t steps = st::cdiv(V, 64);
  Split best{};
  double least = 1e300;
  for (const Kind& k : kinds) {
    const int64_t tiles = st::cdiv(rows, k.bm) * st::cdiv(H, k.bn);
    for (int64_t s = 1; s <= 64; ++s) {
      const int64_t per = st::cdiv(steps, s) * 64;
      if (s > 1 && per < 512) break;
      if (per * ldw * 2 >= (int64_t)1 << 31) continue;
      const int64_t n = st::cdiv(V, per);
      const double us = (double)st::cdiv(tiles * n, 256) * ((double)per / 64 + 10) * k.us +
                        (double)(n * rows * H) * 8e-6 / 5.0;
      if (us < least) {
        least = us;
        best = {k.bm, k.bn, (int)n, per};
      }
    }
  }
  return best;
}

struct Space {
  int64_t part, xy, logits, bytes, ldl;
};
Space fwd_space(int64_t rows, int64_t V, int64_t top, bool kept) {
  Space s{};
  s.part = 0;
  s.xy = up(rows * st::cdiv(V, VT) * 16, 256);
  s.logits = s.xy + up(rows * 4, 256);
  s.ldl = up(V, 4);
  s.bytes = s.logits + (top > 0 && !kept ? rows * s.ldl * 4 : 0) + 256;
  return s;
}
// dl rows padded to 64 columns: whole k-steps start on 128-byte lines
struct BwdSpace {
  int64_t left, part, bytes, ldd;
  Split split;
};
BwdSpace bwd_space(int64_t rows, int64_t H, int64_t ldw, int64_t V, int64_t top) {
  BwdSpace s{};
  s.ldd = up(V, 64);
  s.split = split_of(rows, H, ldw, V);
  s.left = up(rows * s.ldd * 2, 256);
  s.part = s.left + up(rows * (top + 1) * 4, 256);
  s.bytes = s.part + s.split.splits * rows * H * 4 + 256;
  return s;
}

int check(const char* name, Head& h, const uint16_t* hidden, int64_t rows, int64_t H, int64_t ldh,
          const uint16_t* head, int64_t V, int64_t ldw, const int64_t* tokens, float temperature,
          float cap, int64_t top) {
  ST_CHECK_ARG(rows >= 0 && H > 0 && V > 0 && H % 8 == 0 && ldh % 8 == 0 && ldw % 8 == 0 &&
                   ldh >= H && ldw >= H, "%s: rows must be 16-byte multiples of at least H", name);
  ST_CHECK_ARG(std::isfinite(temperature) && temperature > 0 && std::isfinite(cap) && cap >= 0,
               "%s: temperature must be positive, cap 0 (none) or positive", name);
  ST_CHECK_ARG(top >= 0 && top <= V, "%s: top must be within the vocabulary", name);
  if (temperature < 1e-30f || temperature > 1e30f || (cap > 0 && (cap < 1e-30f || cap > 1e30f)))
    return st::fail(ST_EUNSUPPORTED, "%s: temperature %g or cap %g out of range (1e-30 to 1e30)", name,
                    temperature, cap);
  if (top > 64 || V > (1 << 21) || (top && V > (1 << 20)) || H > (1 << 20) || ldw > (1 << 20) ||
      ldh > (1 << 20) || rows > (1 << 22))
    return st::fail(ST_EUNSUPPORTED, "%s: rows=%lld H=%lld V=%lld top=%lld is too large (top <= 64)",
                    name, (long long)rows, (long long)H, (long long)V, (long long)top);
  if (rows == 0) return ST_OK;
  ST_CHECK_ARG(hidden && head && tokens && al16(hidden) && al16(head), "%s: NULL or unaligned pointer",
               name);
  h.hidden = hidden; h.head = head; h.tokens = tokens;
  h.ldh = ldh; h.ldw = ldw; h.rows = rows; h.V = V;
  h.H = (int)H;
  h.vtiles = (int)st::cdiv(V, VT);
  h.tf = {cap, cap > 0 ? 1.0f / cap : 0.0f, 1.0f / temperature};
  return ST_OK;
}

// a dimension of a launch holds less than 2^32 threads
bool fits(int64_t groups, int threads) { return groups * threads < (int64_t)1 << 32; }

// fn(loop type, grid) with the row tile that suits the rows
template <typename F>
int by_rows(Head& h, F&& fn) {
  const int bn = row_tile(h.rows);
  h.rtiles = (int)st::cdiv(h.rows, bn);
  const int64_t tiles = up((int64_t)h.rtiles * h.vtiles, 8);
  if (!fits(tiles, 512)) return st::fail(ST_EUNSUPPORTED, "token_logprobs: too many tiles");
  const dim3 grid((unsigned)tiles);
  if (bn == 256) fn(st::DmaLoop256<false, false>{}, grid);
  else if (bn == 128) fn(st::DmaLoop64<false, false, 4, 2, 3>{}, grid);
  else fn(st::DmaLoop64<false, false, 4, 1, 4>{}, grid);
  return ST_OK;
}

}  // namespace

extern "C" int64_t st_token_logprobs_workspace_bytes(int64_t rows, int64_t H, int64_t V, int64_t ldw,
                                                     int64_t top, int32_t kept, int32_t backward) {
  if (rows <= 0 || H <= 0 || V <= 0 || ldw < H || ldw > (1 << 20) || top < 0) return 0;
  return backward ? bwd_space(rows, H, ldw, V, top).bytes : fwd_space(rows, V, top, kept != 0).bytes;
}

extern "C" int st_token_logprobs_fwd(const uint16_t* hidden, int64_t rows, int64_t H, int64_t ldh,
                                     const uint16_t* head, int64_t V, int64_t ldw,
                                     const int64_t* tokens, int64_t ignore_index, float temperature,
                                     float cap, int64_t top, float* logprobs, float* entropy,
                                     float* lse, float* top_logprobs, int64_t* top_tokens,
                                     float* logits, void* workspace, int64_t workspace_bytes,
                                     st_stream_t stream) {
  const char* name = "st_token_logprobs_fwd";
  Head h{};
  if (int rc = check(name, h, hidden, rows, H, ldh, head, V, ldw, tokens, temperature, cap, top)) return rc;
  if (rows == 0) return ST_OK;
  ST_CHECK_ARG(logprobs && entropy && lse && (!top || (top_logprobs && top_tokens)) && al16(logits),
               "%s: NULL or unaligned pointer", name);
  const Space sp = fwd_space(rows, V, top, logits != nullptr);
  if (!workspace || workspace_bytes < sp.bytes)
    return st::fail(ST_EWORKSPACE, "%s: needs %lld workspace bytes", name, (long long)sp.bytes);
  char* ws = (char*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  float4* part = (float4*)(ws + sp.part);
  float* xy = (float*)(ws + sp.xy);
  if (top && !logits) logits = (float*)(ws + sp.logits);
  hipStream_t s = (hipStream_t)stream;
  if (int rc = by_rows(h, [&](auto lp, dim3 grid) {
        using LP = decltype(lp);
        lp_tiles<LP><<<grid, LP::NT, 0, s>>>(h, part, xy, logits, sp.ldl, top > 0);
      })) return rc;
  if (int rc = st::check_launch(name)) return rc;
  const dim3 grid((unsigned)st::cdiv(rows, NT / 64));
  const size_t lds = top ? (NT / 64) * h.vtiles * 4 : 0;
  lp_join<<<grid, NT, lds, s>>>(h, ignore_index, part, xy, logits, sp.ldl, (int)top, logprobs, entropy,
                                lse, top_logprobs, top_tokens);
  return st::check_launch("lp_join");
}

extern "C" int st_token_logprobs_bwd(const uint16_t* hidden, int64_t rows, int64_t H, int64_t ldh,
                                     const uint16_t* head, int64_t V, int64_t ldw,
                                     const int64_t* tokens, int64_t ignore_index, float temperature,
                                     float cap, int64_t top, const float* logprobs,
                                     const float* entropy, const float* lse,
                                     const float* top_logprobs, const int64_t* top_tokens,
                                     const float* logits, const float* g_logprobs,
                                     const float* g_entropy, const float* g_top, uint16_t* dhidden,
                                     int64_t ldd, void* workspace, int64_t workspace_bytes,
                                     st_stream_t stream) {
  const char* name = "st_token_logprobs_bwd";
  Head h{};
  if (int rc = check(name, h, hidden, rows, H, ldh, head, V, ldw, tokens, temperature, cap, top)) return rc;
  if (rows == 0) return ST_OK;
  ST_CHECK_ARG(logprobs && entropy && lse && (!top || (top_logprobs && top_tokens)) && dhidden &&
                   al16(dhidden) && al16(logits) && ldd % 8 == 0 && ldd >= H,
               "%s: NULL or unaligned pointer", name);
  const BwdSpace sp = bwd_space(rows, H, ldw, V, top);
  if (!workspace || workspace_bytes < sp.bytes)
    return st::fail(ST_EWORKSPACE, "%s: needs %lld workspace bytes", name, (long long)sp.bytes);
  if (sp.split.splits == 0)
    return st::fail(ST_EUNSUPPORTED, "%s: 64 columns of the head span 2 GiB", name);
  char* ws = (char*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  uint16_t* dl = (uint16_t*)ws;
  float *left = (float*)(ws + sp.left), *part = (float*)(ws + sp.part);
  hipStream_t s = (hipStream_t)stream;
  const Split& k = sp.split;
  const Dgrad d{dl, head, sp.ldd, ldw, rows, V, (int)H, (int)st::cdiv(rows, k.bm),
                (int)st::cdiv(H, k.bn), k.splits, k.per};
  const int64_t parts = up((int64_t)d.rtiles * d.htiles * d.splits, 8);
  if (!fits(parts, 512)) return st::fail(ST_EUNSUPPORTED, "%s: too many tiles", name);
  const Upstream g{g_logprobs, g_entropy, top ? g_top : nullptr, (int)top};
  const Picks p{top_tokens, top_logprobs, logprobs, lse, entropy};
  if (logits) {
    const unsigned y = (unsigned)std::min<int64_t>(rows, 32768);
    lp_dlogits_kept<<<dim3((unsigned)st::cdiv(sp.ldd, NT * KEPT), y, (unsigned)st::cdiv(rows, y)), NT, 0,
                      s>>>(h, g, ignore_index, p, logits, up(V, 4), dl, sp.ldd, left);
    if (int rc = st::check_launch("lp_dlogits_kept")) return rc;
  } else {
    if (int rc = by_rows(h, [&](auto lp, dim3 grid) {
          using LP = decltype(lp);
          lp_dlogits<LP><<<grid, LP::NT, 0, s>>>(h, g, ignore_index, top_tokens, lse, entropy, dl, sp.ldd);
        })) return rc;
    if (int rc = st::check_launch("lp_dlogits")) return rc;
    const int64_t picks = rows * (top + 1);
    const unsigned groups = (unsigned)std::min<int64_t>(st::cdiv(picks, h.tf.cap != 0.0f ? NT / 64 : NT), 1 << 20);
    if (h.tf.cap != 0.0f)
      lp_picked<true><<<groups, NT, 0, s>>>(h, g, ignore_index, p, dl, sp.ldd, left);
    else
      lp_picked<false><<<groups, NT, 0, s>>>(h, g, ignore_index, p, dl, sp.ldd, left);
    if (int rc = st::check_launch("lp_picked")) return rc;
  }
  const dim3 grid((unsigned)parts);
  if (k.bm == 64)
    lp_dhidden<st::DmaLoop64<true, false, 1, 4, 4>><<<grid, 256, 0, s>>>(d, part);
  else if (k.bn == 128)
    lp_dhidden<st::DmaLoop64<true, false, 4, 2, 3>><<<grid, 512, 0, s>>>(d, part);
  else
    lp_dhidden<st::DmaLoop256<true, false>><<<grid, 512, 0, s>>>(d, part);
  if (int rc = st::check_launch("lp_dhidden")) return rc;
  lp_reduce<<<(unsigned)std::min<int64_t>(st::cdiv(rows * H / 4, NT), 4096), NT, 0, s>>>(
      h, part, k.splits, left, (int)top, top_tokens, dhidden, ldd);
  return st::check_launch("lp_reduce");
}
