// Balance loss of a router and its per-expert counts, and the gradient of its logits.
//
//   p = softmax(l)  or  sigma(l) / (sum sigma(l) + 1e-20)
//   a group of tokens (all of them, or a row's) with n valid ones:
//     c_e picks of expert e,  P_e = mean of p_e,  L_g = E sum_e c_e / (k n) P_e
//   L = mean of L_g over the groups with a valid token (1 when balanced)
//   dp_e = a_e = dL E c_e / (k n^2 groups);  dl_e = p_e (a_e - sum a p)  or
//          (a_e - sum a p) / (sum sigma + 1e-20) sigma_e (1 - sigma_e)
//
// A wave holds a token's logits (up to 512 experts, PER = 1, 2, 4 or 8 a lane), so each
// is read once forward and once backward, the next token's while the present one's are
// worked on; picks are counted in LDS (whole numbers: their order does not matter),
// probabilities summed in fp32 in registers over a workgroup's tokens and joined over the
// workgroups in their order.  16384 tokens of 256 experts (17 MB): the sums 13 us, the join
// 8 in four rows and 19 as one group (one workgroup a group), the mean over rows 1.5,
// backward 12.  The sums' waves have one token ahead and are eight a CU: 2 MB in flight in
// all, which a round trip to memory of about 1.5 us makes the 1.3 TB/s measured.
#include "common.h"

namespace {

constexpr int NTH = 256, WAVES = NTH / 64, JOIN = 1024;
constexpr int MAXE = 512;
constexpr float TINY = 1e-20f;

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

struct Args {
  const void* logits;
  const int32_t* picks;  // words of 32 bits, `wide` of them a pick
  int32_t wide;
  const uint8_t* valid;
  int64_t groups, per_group;  // tokens of a group
  int32_t E, k, sigmoid;
  int64_t chunk, chunks;  // tokens of a workgroup, workgroups of a group
  float* probs;           // [groups][chunks][E]
  int32_t* counted;       // [groups][chunks][E + 1], the last: valid tokens
  float* terms;           // [groups]
  float* loss;
  int64_t* counts;  // [groups][E]
  int32_t* tokens;  // [groups] valid tokens, and behind them the groups that have some
  const float* dloss;
  void* dlogits;
};

// A token's logits; lane + 64 i is the expert.  Lanes past the experts read the first
// ones (a load under a branch would be waited for at its end).
template <bool BF, int PER>
__device__ __forceinline__ void fetch(const Args& a, int64_t t, int lane, float (&v)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t at = t * a.E + (lane + 64 * i < a.E ? lane + 64 * i : 0);
    v[i] = BF ? st::bf16_to_f32(((const uint16_t*)a.logits)[at]) : ((const float*)a.logits)[at];
  }
}
// The scores e of a token in the place of its logits, and the reciprocal of their sum:
// p = e * inv.
template <int PER>
__device__ __forceinline__ float scores(const Args& a, int lane, float (&v)[PER]) {
  float sum = 0.0f;
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = lane + 64 * i < a.E ? 1.0f / (1.0f + expf(-v[i])) : 0.0f;
      sum += v[i];
    }
    return 1.0f / (wave_sum(sum) + TINY);
  }
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) mx = fmaxf(mx, v[i]);
  mx = wave_max(mx);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = lane + 64 * i < a.E ? expf(v[i] - mx) : 0.0f;
    sum += v[i];
  }
  return 1.0f / wave_sum(sum);
}

template <bool BF, int PER>
__global__ __launch_bounds__(NTH) void balance_sums(Args a) {
  __shared__ float sums[WAVES][64 * PER];
  __shared__ int32_t count[64 * PER + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t g = blockIdx.y, c = blockIdx.x;
  for (int i = threadIdx.x; i <= 64 * PER; i += NTH) count[i] = 0;
  __syncthreads();
  float p[PER] = {}, next[PER];
  int n = 0;
  const int64_t z = min((c + 1) * a.chunk, a.per_group), t0 = g * a.per_group;
  int64_t i = c * a.chunk + wave;
  const int64_t last = a.per_group - 1;
  // what the next token needs, also where there is none (the last one's then)
  auto ahead = [&](int64_t k, bool& valid, int& pick, int& high) {
    const int64_t t = t0 + (k < z ? k : last);
    fetch<BF, PER>(a, t, lane, next);
    valid = !a.valid || a.valid[t];
    const int32_t* p = a.picks + (t * a.k + (lane < a.k ? lane : 0)) * a.wide;
    pick = p[0], high = a.wide == 2 ? p[a.wide - 1] : 0;
  };
  bool valid;
  int pick, high;
  ahead(i, valid, pick, high);
  for (; i < z; i += WAVES) {
    float v[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = next[j];
    const bool live = valid;
    const int e = high ? -1 : pick;
    ahead(i + WAVES, valid, pick, high);
    if (!live) continue;  // the same for the whole wave
    const float inv = scores<PER>(a, lane, v);
#pragma unroll
    for (int j = 0; j < PER; ++j) p[j] += v[j] * inv;
    if (lane < a.k && e >= 0 && e < a.E) atomicAdd(&count[e], 1);
    ++n;
  }
  if (lane == 0) atomicAdd(&count[64 * PER], n);
#pragma unroll
  for (int j = 0; j < PER; ++j) sums[wave][lane + 64 * j] = p[j];
  __syncthreads();
  float* to = a.probs + (g * a.chunks + c) * a.E;
  int32_t* nt = a.counted + (g * a.chunks + c) * (a.E + 1);
  for (int e = threadIdx.x; e < a.E; e += NTH) {
    float s = sums[0][e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += sums[w][e];
    to[e] = s;
    nt[e] = count[e];
  }
  if (threadIdx.x == 0) nt[a.E] = count[64 * PER];
}

// Sums of the chunks of a group, one wave each 64 experts at a time: wave w takes the
// chunks w, w + WAVES, .., whose loads do not wait for one another; the waves' sums are
// added in their order.
__global__ __launch_bounds__(JOIN) void balance_join(Args a) {
  constexpr int W = JOIN / 64;
  __shared__ float probs[W][64];
  __shared__ int32_t count[W][64], total[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t g = blockIdx.x;
  const int32_t* counted = a.counted + g * a.chunks * (a.E + 1);
  const float* sums = a.probs + g * a.chunks * a.E;
  int n = 0;  // fewer than 2^25 tokens a group
  for (int64_t c = threadIdx.x; c < a.chunks; c += JOIN) n += counted[c * (a.E + 1) + a.E];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) n += __shfl_xor(n, d);
  if (lane == 0) total[wave] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) n += total[w];
  const float many = (float)(n > 0 ? n : 1);
  float loss = 0.0f;
  for (int e0 = 0; e0 < a.E; e0 += 64) {
    const int e = e0 + lane;
    float p = 0.0f;
    int32_t picks = 0;
    if (e < a.E) {
#pragma unroll 8
      for (int64_t c = wave; c < a.chunks; c += W) {
        p += sums[c * a.E + e];
        picks += counted[c * (a.E + 1) + e];
      }
    }
    __syncthreads();
    probs[wave][lane] = p;
    count[wave][lane] = picks;
    __syncthreads();
    if (wave == 0) {
      int64_t all = 0;
      p = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) p += probs[w][lane], all += count[w][lane];
      if (e < a.E) {
        a.counts[g * a.E + e] = all;
        loss += (float)all * (float)a.E / ((float)a.k * many) * (p / many);
      }
    }
  }
  if (wave) return;
  loss = wave_sum(loss);
  if (lane == 0) {
    a.tokens[g] = n;
    if (a.groups == 1) {
      *a.loss = loss;
      a.tokens[1] = n > 0;
    } else {
      a.terms[g] = loss;
    }
  }
}

__global__ __launch_bounds__(64) void balance_mean(Args a) {
  float s = 0.0f;
  int some = 0;
  for (int64_t g = threadIdx.x; g < a.groups; g += 64) {
    s += a.terms[g];
    some += a.tokens[g] > 0;
  }
  s = wave_sum(s);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) some += __shfl_xor(some, d);
  if (threadIdx.x == 0) {
    *a.loss = s / (float)(some > 0 ? some : 1);
    a.tokens[a.groups] = some;
  }
}

template <bool BF, int PER>
__global__ __launch_bounds__(NTH) void balance_bwd(Args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t g = blockIdx.y, z = min((int64_t)(blockIdx.x + 1) * a.chunk, a.per_group);
  const int64_t t0 = g * a.per_group, last = a.per_group - 1;
  int64_t i = blockIdx.x * a.chunk + wave;
  float next[PER];
  auto ahead = [&](int64_t k, bool& valid) {
    const int64_t t = t0 + (k < z ? k : last);
    fetch<BF, PER>(a, t, lane, next);
    valid = !a.valid || a.valid[t];
  };
  bool valid;
  ahead(i, valid);
  const float n = (float)a.tokens[g];
  const float each = *a.dloss * (float)a.E / ((float)a.k * n * n * (float)a.tokens[a.groups]);
  float w[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + 64 * j;
    w[j] = e < a.E ? each * (float)a.counts[g * a.E + e] : 0.0f;
  }
  for (; i < z; i += WAVES) {
    const int64_t t = t0 + i;
    float v[PER], d[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = next[j], d[j] = 0.0f;
    const bool live = valid;
    ahead(i + WAVES, valid);
    if (live) {  // the same for the whole wave
      const float inv = scores<PER>(a, lane, v);
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) dot += w[j] * (v[j] * inv);
      dot = wave_sum(dot);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        d[j] = v[j] * inv * (w[j] - dot) * (a.sigmoid ? 1.0f - v[j] : 1.0f);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = lane + 64 * j;
      if (e >= a.E) continue;
      if (BF)
        ((uint16_t*)a.dlogits)[t * a.E + e] = st::f32_to_bf16(d[j]);
      else
        ((float*)a.dlogits)[t * a.E + e] = d[j];
    }
  }
}

// Tokens of a workgroup: about 512 workgroups in all, at least four tokens a wave.
void plan(Args& a) {
  const int64_t want = st::cdiv(512, a.groups);
  a.chunk = st::cdiv(st::cdiv(a.per_group, want), 4 * WAVES) * 4 * WAVES;
  a.chunks = st::cdiv(a.per_group, a.chunk);
}

int check_args(const Args& a, int32_t dtype, const char* what) {
  ST_CHECK_ARG(dtype == ST_DTYPE_BF16 || dtype == ST_DTYPE_F32, "dtype codes are bf16 and fp32");
  ST_CHECK_ARG(a.groups >= 1 && a.per_group >= 1, "%s: groups %lld of %lld tokens", what,
               (long long)a.groups, (long long)a.per_group);
  ST_CHECK_ARG(a.E >= 1 && a.E <= MAXE && a.k >= 1 && a.k <= 64, "%s: experts 1..512, picks 1..64",
               what);
  if (a.groups >= 65536 || a.per_group >= (int64_t)1 << 25)
    return st::fail(ST_EUNSUPPORTED, "%s: 65536 groups or 2^25 tokens a group and more", what);
  return ST_OK;
}

}  // namespace

extern "C" int64_t st_balance_workspace_bytes(int64_t groups, int64_t per_group, int32_t experts) {
  Args a = {};
  a.groups = groups, a.per_group = per_group, a.E = experts, a.k = 1;
  if (check_args(a, ST_DTYPE_F32, "st_balance") != ST_OK) return 0;
  plan(a);
  return (groups * a.chunks * (2 * (int64_t)experts + 1) + groups) * 4;
}

extern "C" int st_balance_fwd(const void* logits, int32_t dtype, const void* picks,
                              int32_t picks64, const uint8_t* valid, int64_t groups,
                              int64_t per_group, int32_t experts, int32_t top_k, int32_t sigmoid, float* loss,
                              int64_t* counts, int32_t* tokens, void* workspace,
                              int64_t workspace_bytes, st_stream_t stream) {
  Args a = {};
  a.logits = logits, a.picks = (const int32_t*)picks, a.wide = picks64 ? 2 : 1, a.valid = valid;
  a.groups = groups, a.per_group = per_group;
  a.E = experts, a.k = top_k, a.sigmoid = sigmoid, a.loss = loss, a.counts = counts;
  a.tokens = tokens;
  const int rc = check_args(a, dtype, "st_balance_fwd");
  if (rc != ST_OK) return rc;
  ST_CHECK_ARG(logits && picks && loss && counts && tokens, "st_balance_fwd: NULL");
  const int64_t need = st_balance_workspace_bytes(groups, per_group, experts);
  if (!workspace || workspace_bytes < need)
    return st::fail(ST_EWORKSPACE, "st_balance_fwd needs %lld workspace bytes", (long long)need);
  ST_CHECK_ARG(((uintptr_t)workspace & 3) == 0, "workspace must be 4-byte aligned");
  plan(a);
  a.probs = (float*)workspace;
  a.counted = (int32_t*)(a.probs + groups * a.chunks * experts);
  a.terms = (float*)(a.counted + groups * a.chunks * (experts + 1));
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)a.chunks, (unsigned)groups);
  auto run = [&](auto bf, auto f32) {
    if (dtype == ST_DTYPE_BF16)
      bf<<<grid, NTH, 0, s>>>(a);
    else
      f32<<<grid, NTH, 0, s>>>(a);
  };
  if (experts <= 64)
    run(balance_sums<true, 1>, balance_sums<false, 1>);
  else if (experts <= 128)
    run(balance_sums<true, 2>, balance_sums<false, 2>);
  else if (experts <= 256)
    run(balance_sums<true, 4>, balance_sums<false, 4>);
  else
    run(balance_sums<true, 8>, balance_sums<false, 8>);
  balance_join<<<(unsigned)groups, JOIN, 0, s>>>(a);
  if (groups > 1) balance_mean<<<1, 64, 0, s>>>(a);
  return st::check_launch("st_balance_fwd");
}

extern "C" int st_balance_bwd(const void* logits, int32_t dtype, const uint8_t* valid,
                              int64_t groups, int64_t per_group, int32_t experts, int32_t top_k,
                              int32_t sigmoid, const int64_t* counts, const int32_t* tokens,
                              const float* dloss, void* dlogits, st_stream_t stream) {
  Args a = {};
  a.logits = logits, a.valid = valid, a.groups = groups, a.per_group = per_group;
  a.E = experts, a.k = top_k, a.sigmoid = sigmoid, a.counts = (int64_t*)counts;
  a.tokens = (int32_t*)tokens, a.dloss = dloss, a.dlogits = dlogits;
  const int rc = check_args(a, dtype, "st_balance_bwd");
  if (rc != ST_OK) return rc;
  ST_CHECK_ARG(logits && counts && tokens && dloss && dlogits, "st_balance_bwd: NULL");
  // about 2048 workgroups, two tokens a wave at least: its weights are read per wave
  a.chunk = st::cdiv(st::cdiv(per_group, st::cdiv(2048, groups)), 2 * WAVES) * 2 * WAVES;
  a.chunks = st::cdiv(per_group, a.chunk);
  const dim3 grid((unsigned)a.chunks, (unsigned)groups);
  auto run = [&](auto bf, auto f32) {
    if (dtype == ST_DTYPE_BF16)
      bf<<<grid, NTH, 0, (hipStream_t)stream>>>(a);
    else
      f32<<<grid, NTH, 0, (hipStream_t)stream>>>(a);
  };
  if (experts <= 64)
    run(balance_bwd<true, 1>, balance_bwd<false, 1>);
  else if (experts <= 128)
    run(balance_bwd<true, 2>, balance_bwd<false, 2>);
  else if (experts <= 256)
    run(balance_bwd<true, 4>, balance_bwd<false, 4>);
  else
    run(balance_bwd<true, 8>, balance_bwd<false, 8>);
  return st::check_launch("st_balance_bwd");
}
