// Token embedding: scaled lookup, and the table's gradient by sorted tokens.
//
//   out[t] = scale table[id_t];   dtable[v] = scale sum_{t: id_t = v} dout[t]
//
// Both are bound by HBM.  The gradient's sums must not depend on the order in which
// workgroups arrive, so no float is added atomically: (token, position) pairs are
// sorted by token (least significant digit first, nine bits a pass, stable, so each
// token's positions rise), and chunks of the sorted list are summed in that order,
// each row of dout read once.  A token whose positions reach over a chunk's end
// leaves partial sums, which a last kernel joins from chunk to chunk.  A dense
// gradient is cleared by the launch that sorts: up to 16384 tokens are sorted by one
// workgroup in LDS while the others clear.
#include <cmath>

#include "common.h"

namespace {

constexpr int NTH = 256;
constexpr int BITS = 9, BINS = 1 << BITS;
constexpr int64_t SMALL = 16384;  // tokens one workgroup sorts (16 a thread)
// 16-byte words up to which the launch that sorts in LDS also clears, one workgroup a
// CU beside it: 64 MB in the sort's time, 2.1 GB in 364 us instead of 310 and 25
constexpr int64_t CLEAR_APART = (64 << 20) / 16;
constexpr int TILE = 2048;        // keys of a workgroup beyond that

__device__ __forceinline__ int64_t id_at(const void* ids, int ids32, int64_t i) {
  return ids32 ? (int64_t)((const int32_t*)ids)[i] : ((const int64_t*)ids)[i];
}
// The sort key: tokens outside the table and the padding token come last.
__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t V, int64_t padding) {
  return id < 0 || id >= V || id == padding ? (uint32_t)V : (uint32_t)id;
}

// A row that is no multiple of VEC columns (RAG) starts on any element; its last VEC are
// moved back to end with it: the first `skip` of them are another thread's too, worked
// out alike and stored twice, or added to the gradient by that one alone.  (8192 tokens,
// 32000 rows of 1001 columns: sums 9.1 us, of 1000 columns 8.9.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

template <typename V, typename ANY, bool RAG>
__device__ __forceinline__ V load(const void* p) {
  if constexpr (RAG)
    return *(const ANY*)p;
  else
    return *(const V*)p;
}
template <typename V, typename ANY, bool RAG>
__device__ __forceinline__ void store(void* p, V v) {
  if constexpr (RAG)
    *(ANY*)p = v;
  else
    *(V*)p = v;
}
template <bool RAG>
__device__ __forceinline__ void store_bf16x8(uint16_t* p, const float (&f)[8]) {
  store<u32x4, u32x4_any, RAG>(p, u32x4{st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3]),
                                        st::pack_bf16x2(f[4], f[5]), st::pack_bf16x2(f[6], f[7])});
}

// ---------------------------------------------------------------- lookup
template <int VEC, bool F32, bool RAG>
__global__ __launch_bounds__(NTH) void lookup(const void* __restrict__ table,
                                              const void* __restrict__ ids, int ids32, int64_t n,
                                              int64_t V, int64_t H, float scale,
                                              uint16_t* __restrict__ out) {
  for (int64_t t = blockIdx.x; t < n; t += gridDim.x) {
    const int64_t id = id_at(ids, ids32, t);
    const bool in = id >= 0 && id < V;
    for (int64_t col = threadIdx.x * VEC; col < H; col += (int64_t)blockDim.x * VEC) {
      const int64_t i = RAG && col + VEC > H ? H - VEC : col;
      float f[VEC];
      const int64_t at = (in ? id : 0) * H + i;
      if constexpr (VEC == 8) {
        if constexpr (F32) {
          const float* p = (const float*)table + at;
          const f32x4 a = load<f32x4, f32x4_any, RAG>(p), b = load<f32x4, f32x4_any, RAG>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
        } else {
          const u32x4 w = load<u32x4, u32x4_any, RAG>((const uint16_t*)table + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[2 * e] = __uint_as_float(w[e] << 16);
            f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          }
        }
      } else {
        f[0] = F32 ? ((const float*)table)[at] : st::bf16_to_f32(((const uint16_t*)table)[at]);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = in ? f[e] * scale : NAN;
      uint16_t* to = out + t * H + i;
      if constexpr (VEC == 8)
        store_bf16x8<RAG>(to, f);
      else
        *to = st::f32_to_bf16(f[0]);
    }
  }
}

// ---------------------------------------------------------------- clear
// Workgroup `b` of `many` clears its share: one 16-byte word a thread and as many
// workgroups as that takes (2.1 GB: 310 us, where loops of any kind took 350 to 420).
template <int NT>
__device__ __forceinline__ void clear_share(uint4* p, int64_t words, int64_t b, int64_t many) {
  for (int64_t i = b * NT + threadIdx.x; i < words; i += many * NT) p[i] = make_uint4(0, 0, 0, 0);
}
unsigned clear_blocks(int64_t words) {
  const int64_t b = st::cdiv(words, NTH);
  return (unsigned)(b < (1 << 23) ? b : 1 << 23);
}

// ---------------------------------------------------------------- sort
// Rank of each lane's key among its wave's keys of one digit, those of earlier
// calls first (count[] starts at zero).  Lanes that are not `live` take no part.
__device__ __forceinline__ uint32_t wave_rank(uint32_t digit, bool live, uint32_t* count) {
  const int lane = threadIdx.x & 63;
  unsigned long long same = __ballot(live);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const unsigned long long set = __ballot((digit >> b) & 1u);
    same &= (digit >> b) & 1u ? set : ~set;
  }
  uint32_t base = 0;
  const int first = __ffsll((long long)same) - 1;
  if (live && lane == first) base = atomicAdd(&count[digit], (uint32_t)__popcll(same));
  base = __shfl(base, live ? first : 0);
  return base + (uint32_t)__popcll(same & ((1ull << lane) - 1));
}

// Exclusive sums of count[wave][digit] over digits, then waves, in place; 64 W
// threads.
template <int W>
__device__ __forceinline__ void scan_counts(uint32_t (*count)[BINS], uint32_t* totals) {
  constexpr int PER = BINS * W / (64 * W);  // counters a thread: 8 bins of one wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // thread order = digit-major: entry e = digit * W + w
  uint32_t v[PER], sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int e = threadIdx.x * PER + k;
    v[k] = count[e % W][e / W];
    sum += v[k];
  }
  uint32_t inc = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t x = __shfl_up(inc, d);
    if (lane >= d) inc += x;
  }
  if (lane == 63) totals[wave] = inc;
  __syncthreads();
  uint32_t base = inc - sum;
  for (int w = 0; w < wave; ++w) base += totals[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int e = threadIdx.x * PER + k;
    count[e % W][e / W] = base;
    base += v[k];
  }
  __syncthreads();
}

// Up to 16384 tokens: workgroup 0 sorts, the others clear `words` 16-byte words.
__global__ __launch_bounds__(1024) void sort_small(const void* __restrict__ ids, int ids32, int n,
                                                   int64_t V, int64_t padding, int passes,
                                                   uint32_t* __restrict__ tok,
                                                   uint32_t* __restrict__ pos,
                                                   uint4* __restrict__ clear, int64_t words) {
  if (blockIdx.x) return clear_share<1024>(clear, words, blockIdx.x - 1, gridDim.x - 1);
  __shared__ uint32_t count[16][BINS];
  __shared__ uint32_t totals[16];
  __shared__ uint32_t keys[SMALL];
  __shared__ uint16_t where[SMALL];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int steps = (n + 1023) / 1024, first = wave * steps * 64 + lane;
  uint32_t key[16], rank[16];
  uint16_t at[16];
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    const int i = first + s * 64;
    const bool live = s < steps && i < n;
    key[s] = live ? key_of(id_at(ids, ids32, i), V, padding) : 0;
    at[s] = (uint16_t)i;
  }
  for (int p = 0; p < passes; ++p) {
    for (int i = threadIdx.x; i < 16 * BINS; i += 1024) (&count[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 16; ++s)
      if (s < steps) rank[s] = wave_rank((key[s] >> (BITS * p)) & (BINS - 1), first + s * 64 < n,
                                         count[wave]);
    __syncthreads();
    scan_counts<16>(count, totals);
#pragma unroll
    for (int s = 0; s < 16; ++s)
      if (s < steps && first + s * 64 < n) {
        const uint32_t to = count[wave][(key[s] >> (BITS * p)) & (BINS - 1)] + rank[s];
        keys[to] = key[s];
        where[to] = at[s];
      }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 16; ++s)
      if (s < steps && first + s * 64 < n) {
        key[s] = keys[first + s * 64];
        at[s] = where[first + s * 64];
      }
    __syncthreads();
  }
#pragma unroll
  for (int s = 0; s < 16; ++s)
    if (s < steps && first + s * 64 < n) {
      tok[first + s * 64] = key[s];
      pos[first + s * 64] = at[s];
    }
}

// More tokens: per pass the tiles' digit counts [digit][tile], their exclusive sums,
// and the move.  The first pass reads the ids themselves, and its workgroups behind
// the tiles' clear the gradient.
__global__ __launch_bounds__(NTH) void tile_counts(const void* __restrict__ ids, int ids32,
                                                   const uint32_t* __restrict__ tok, int64_t n,
                                                   int64_t V, int64_t padding, int shift,
                                                   int64_t tiles, uint32_t* __restrict__ counts,
                                                   uint4* __restrict__ clear, int64_t words) {
  __shared__ uint32_t hist[BINS];
  if (blockIdx.x >= tiles)
    return clear_share<NTH>(clear, words, blockIdx.x - tiles, gridDim.x - tiles);
  for (int i = threadIdx.x; i < BINS; i += NTH) hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int s = 0; s < TILE / NTH; ++s) {
    const int64_t i = (int64_t)blockIdx.x * TILE + s * NTH + threadIdx.x;
    if (i < n) {
      const uint32_t key = tok ? tok[i] : key_of(id_at(ids, ids32, i), V, padding);
      atomicAdd(&hist[(key >> shift) & (BINS - 1)], 1u);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NTH) counts[i * tiles + blockIdx.x] = hist[i];
}

// Exclusive sums of all counts in place, 8192 at a time.
__global__ __launch_bounds__(1024) void tile_scan(uint32_t* __restrict__ counts, int64_t many) {
  __shared__ uint32_t totals[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t carry = 0;
  for (int64_t i0 = 0; i0 < many; i0 += 8192) {
    const int64_t at = i0 + threadIdx.x * 8;
    uint32_t v[8], sum = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = at + k < many ? counts[at + k] : 0;
      sum += v[k];
    }
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t x = __shfl_up(inc, d);
      if (lane >= d) inc += x;
    }
    if (lane == 63) totals[wave] = inc;
    __syncthreads();
    uint32_t base = carry + inc - sum;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const uint32_t t = totals[w];
      if (w < wave) base += t;
      carry += t;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (at + k < many) counts[at + k] = base;
      base += v[k];
    }
    __syncthreads();
  }
}

// SUMMED: counts are exclusive sums already.  Otherwise each workgroup forms its own
// from the counts themselves (up to MOVE_TILES tiles: 2 us in the place of a launch of
// one workgroup, 7 us).
constexpr int64_t MOVE_TILES = 64;
template <bool SUMMED>
__global__ __launch_bounds__(NTH) void tile_move(const void* __restrict__ ids, int ids32,
                                                 const uint32_t* __restrict__ tok,
                                                 const uint32_t* __restrict__ pos, int64_t n,
                                                 int64_t V, int64_t padding, int shift,
                                                 int64_t tiles,
                                                 const uint32_t* __restrict__ counts,
                                                 uint32_t* __restrict__ tok_out,
                                                 uint32_t* __restrict__ pos_out) {
  constexpr int W = NTH / 64, STEPS = TILE / NTH, OWN = BINS / NTH;
  __shared__ uint32_t count[W][BINS];
  __shared__ uint32_t totals[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < W * BINS; i += NTH) (&count[0][0])[i] = 0;
  const int64_t first = (int64_t)blockIdx.x * TILE + wave * (TILE / W) + lane;
  uint32_t key[STEPS], at[STEPS], rank[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int64_t i = first + s * 64;
    key[s] = i >= n ? 0 : tok ? tok[i] : key_of(id_at(ids, ids32, i), V, padding);
    at[s] = i >= n ? 0 : tok ? pos[i] : (uint32_t)i;
  }
  // the tile's place of the digits OWN threadIdx.x ..
  uint32_t place[OWN];
  if constexpr (SUMMED) {
#pragma unroll
    for (int o = 0; o < OWN; ++o)
      place[o] = counts[(threadIdx.x * OWN + o) * tiles + blockIdx.x];
  } else {
    uint32_t sum = 0, all[OWN];
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const uint32_t* p = counts + (threadIdx.x * OWN + o) * tiles;
      uint32_t before = 0;
      all[o] = 0;
#pragma unroll 8
      for (int t = 0; t < (int)tiles; ++t) {
        const uint32_t c = p[t];
        all[o] += c;
        before += t < (int)blockIdx.x ? c : 0;
      }
      place[o] = before;
      sum += all[o];
    }
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t x = __shfl_up(inc, d);
      if (lane >= d) inc += x;
    }
    if (lane == 63) totals[wave] = inc;
    __syncthreads();
    uint32_t base = inc - sum;
    for (int w = 0; w < wave; ++w) base += totals[w];
#pragma unroll
    for (int o = 0; o < OWN; ++o) place[o] += base, base += all[o];
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
    rank[s] = wave_rank((key[s] >> shift) & (BINS - 1), first + s * 64 < n, count[wave]);
  __syncthreads();
  // then the waves' before this one
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int d = threadIdx.x * OWN + o;
    for (int w = 0; w < W; ++w) {
      const uint32_t v = count[w][d];
      count[w][d] = place[o];
      place[o] += v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
    if (first + s * 64 < n) {
      const uint32_t to = count[wave][(key[s] >> shift) & (BINS - 1)] + rank[s];
      tok_out[to] = key[s];
      pos_out[to] = at[s];
    }
}

__global__ __launch_bounds__(NTH) void clear_words(uint4* __restrict__ p, int64_t words) {
  clear_share<NTH>(p, words, blockIdx.x, gridDim.x);
}
// what 16-byte words leave of a gradient
__global__ __launch_bounds__(64) void clear_tail(uint16_t* __restrict__ p, int halves) {
  if ((int)threadIdx.x < halves) p[threadIdx.x] = 0;
}

// ---------------------------------------------------------------- sums
struct Sums {
  const uint16_t* dout;
  const uint32_t *tok, *pos;
  int64_t n, V, H;
  int64_t chunk;  // sorted entries of a workgroup
  float scale;
  int32_t grad_f32, accumulate;
  void* grad;
  float* partial;  // [chunks][2][H]: of the run from the chunk before, of the run into the next
};

template <int VEC, bool RAG>
__device__ __forceinline__ void store_f(float* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    p[0] = f[0];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 4)
      store<f32x4, f32x4_any, RAG>(p + e, f32x4{f[e], f[e + 1], f[e + 2], f[e + 3]});
  }
}
template <int VEC, bool RAG>
__device__ __forceinline__ void write_row(const Sums& a, uint32_t token, int64_t i, int skip,
                                          const float (&acc)[VEC]) {
  const int64_t at = (int64_t)token * a.H + i;
  float f[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = a.scale * acc[e];
  if (a.grad_f32) {
    float* p = (float*)a.grad + at;
    if (RAG && a.accumulate && skip) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (e >= skip) p[e] += f[e];
      return;
    }
    if (a.accumulate) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] += p[e];
    }
    store_f<VEC, RAG>(p, f);
  } else {
    uint16_t* p = (uint16_t*)a.grad + at;
    if constexpr (VEC == 8)
      store_bf16x8<RAG>(p, f);
    else if constexpr (VEC == 4)
      store<u32x2, u32x2_any, RAG>(
          p, u32x2{st::pack_bf16x2(f[0], f[1]), st::pack_bf16x2(f[2], f[3])});
    else
      *p = st::f32_to_bf16(f[0]);
  }
}

// A chunk of the sorted list: sums of its runs of one token.  Each wave has the
// chunk's tokens and positions in its lanes (lane l: entry e0 - 1 + l, so the
// neighbours' too), and eight rows are read at once.
constexpr int AHEAD = 8;
template <int VEC>
struct Raw {
  u32x4 v;
};
template <>
struct Raw<4> {
  u32x2 v;
};
template <>
struct Raw<1> {
  uint16_t v;
};
template <int VEC, bool RAG>
__device__ __forceinline__ void read_row(const uint16_t* p, Raw<VEC>& r) {
  if constexpr (VEC == 8)
    r.v = load<u32x4, u32x4_any, RAG>(p);
  else if constexpr (VEC == 4)
    r.v = load<u32x2, u32x2_any, RAG>(p);
  else
    r.v = *p;
}
template <int VEC>
__device__ __forceinline__ void add_row(const Raw<VEC>& r, float (&acc)[VEC]) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      acc[2 * e] += __uint_as_float(r.v[e] << 16);
      acc[2 * e + 1] += __uint_as_float(r.v[e] & 0xffff0000u);
    }
  } else {
    acc[0] += st::bf16_to_f32(r.v);
  }
}

template <int VEC, bool RAG>
__global__ __launch_bounds__(NTH) void sum_runs(Sums a) {
  const int lane = threadIdx.x & 63;
  const int64_t c = blockIdx.x, e0 = c * a.chunk;
  const int many = (int)(e0 + a.chunk < a.n ? a.chunk : a.n - e0);
  const int64_t mine = e0 - 1 + lane;
  const bool here = mine >= 0 && mine < a.n && lane <= many + 1;
  // before the first and after the last stands a token of no one's
  const uint32_t tok = here ? a.tok[mine] : ~0u, pos = here ? a.pos[mine] : 0;
  const uint32_t V = (uint32_t)a.V;
  // entries from the first one that takes no part on are behind the end
  const int count = __popcll(__ballot(here && lane >= 1 && lane <= many && tok < V));
  if (!count) return;  // the same for the whole wave
  // lanes past the columns stay, since the others read their tokens: they add the row's
  // first columns and write nothing
  const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool in = col < a.H;
  const int64_t i = !in ? 0 : RAG && col + VEC > a.H ? a.H - VEC : col;
  const int skip = RAG && in ? (int)(col - i) : 0;
  auto token = [&](int e) { return __builtin_amdgcn_readlane(tok, e + 1); };  // -1..many
  auto row = [&](int e) {
    return a.dout + (int64_t)__builtin_amdgcn_readlane(pos, e + 1) * a.H + i;
  };
  bool from = token(-1) == token(0);  // the run began in an earlier chunk
  float acc[VEC] = {};
  for (int b = 0; b < count; b += AHEAD) {
    Raw<VEC> now[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) read_row<VEC, RAG>(row(b + k < count ? b + k : b), now[k]);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int e = b + k;
      if (e >= count) break;
      add_row<VEC>(now[k], acc);
      const bool end = token(e + 1) != token(e);
      if (!end && e + 1 < many) continue;
      const uint32_t whose = token(e);
      if (in) {
        if (from)
          store_f<VEC, RAG>(a.partial + c * 2 * a.H + i, acc);
        else if (!end)
          store_f<VEC, RAG>(a.partial + (c * 2 + 1) * a.H + i, acc);
        else
          write_row<VEC, RAG>(a, whose, i, skip, acc);
      }
      from = false;
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
    }
  }
}

// The same for few tokens, without partial sums and the launch that joins them: a
// workgroup sums the runs that begin in its chunk to their ends, wherever these are
// (at most WHOLE entries, 64 rounds of loads).
constexpr int64_t WHOLE = 512;
template <int VEC, bool RAG>
__global__ __launch_bounds__(NTH) void sum_whole(Sums a) {
  const int lane = threadIdx.x & 63;
  const int n = (int)a.n, e0 = (int)(blockIdx.x * a.chunk), stop = e0 + (int)a.chunk;
  const uint32_t V = (uint32_t)a.V;
  // lanes past the columns stay, as in sum_runs: every lane holds a token
  const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool in = col < a.H;
  const int64_t i = !in ? 0 : RAG && col + VEC > a.H ? a.H - VEC : col;
  const int skip = RAG && in ? (int)(col - i) : 0;
  bool open = false;  // within a run of this workgroup's
  float acc[VEC] = {};
  for (int w = e0;; w += 56) {  // lane l: entry w - 1 + l, up to the one behind w + 56
    const int mine = w - 1 + lane;
    const bool here = mine >= 0 && mine < n;
    const uint32_t tok = here ? a.tok[mine] : ~0u, pos = here ? a.pos[mine] : 0;
    for (int b = 0; b < 56; b += AHEAD) {
      Raw<VEC> now[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        read_row<VEC, RAG>(a.dout + (int64_t)__builtin_amdgcn_readlane(pos, b + k + 1) * a.H + i,
                           now[k]);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int e = w + b + k;
        const uint32_t token = __builtin_amdgcn_readlane(tok, b + k + 1);
        if (!open) {
          if (e >= stop || token >= V) return;  // (~0 behind the last entry)
          if (__builtin_amdgcn_readlane(tok, b + k) == token) continue;  // begun before e0
          open = true;
        }
        add_row<VEC>(now[k], acc);
        if (__builtin_amdgcn_readlane(tok, b + k + 2) == token) continue;
        if (in) write_row<VEC, RAG>(a, token, i, skip, acc);
        open = false;
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
      }
    }
  }
}

// The run that begins in chunk c and goes on behind it: the partial sums of the
// chunks whose first token it is, 64 chunks' tokens looked up at once.
template <int VEC, bool RAG>
__global__ __launch_bounds__(NTH) void join_runs(Sums a) {
  const int lane = threadIdx.x & 63;
  const int64_t c = blockIdx.x, e0 = c * a.chunk, next = e0 + a.chunk;  // next < n by the grid
  const uint32_t token = a.tok[next], last = a.tok[next - 1], first = a.tok[e0];
  const uint32_t before = e0 > 0 ? a.tok[e0 - 1] : ~0u;
  const int64_t col = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  const bool in = col < a.H;
  const int64_t i = !in ? 0 : RAG && col + VEC > a.H ? a.H - VEC : col;
  const int skip = RAG && in ? (int)(col - i) : 0;
  // (lanes past the columns stay: the others ask for their chunks)
  if (token >= a.V || last != token) return;
  if (first == token && before == token) return;  // began earlier
  float acc[VEC] = {};
  const float* p = a.partial + (c * 2 + 1) * a.H + i;
  if (in) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = p[k];
  }
  for (int64_t d0 = c + 1;; d0 += 64) {
    const int64_t e = (d0 + lane) * a.chunk;
    const unsigned long long same = __ballot(e < a.n && a.tok[e < a.n ? e : 0] == token);
    const int run = ~same ? __ffsll((long long)~same) - 1 : 64;
    if (in) {
      p = a.partial + d0 * 2 * a.H + i;
#pragma unroll 8
      for (int d = 0; d < run; ++d) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += p[d * 2 * a.H + k];
      }
    }
    if (run < 64) break;
  }
  if (in) write_row<VEC, RAG>(a, token, i, skip, acc);
}

// ---------------------------------------------------------------- host
int64_t chunk_of(int64_t n) { return n <= 16384 ? 8 : n <= 65536 ? 16 : 32; }
int passes_of(int64_t V) {  // of keys 0..V
  int bits = 1;
  while (V >> bits) ++bits;
  return (bits + BITS - 1) / BITS;
}
int64_t align16(int64_t b) { return (b + 15) & ~(int64_t)15; }

struct Layout {
  int64_t tok[2], pos[2], counts, partial, bytes;
};
Layout layout(int64_t n, int64_t H) {
  Layout l = {};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t a = at;
    at += align16(bytes);
    return a;
  };
  const int two = n > SMALL ? 2 : 1;
  for (int k = 0; k < two; ++k) l.tok[k] = take(4 * n), l.pos[k] = take(4 * n);
  if (n > SMALL) l.counts = take(4 * BINS * st::cdiv(n, TILE));
  l.partial = take(st::cdiv(n, chunk_of(n)) * 2 * H * 4);
  l.bytes = at;
  return l;
}

int check_sizes(const char* what, int64_t n, int64_t V, int64_t H) {
  ST_CHECK_ARG(n >= 0 && V >= 1 && H >= 1, "%s: %lld tokens, table %lld x %lld", what, (long long)n,
               (long long)V, (long long)H);
  if (n >= (int64_t)1 << 31 || V >= (int64_t)1 << 31 || H >= (int64_t)1 << 24)
    return st::fail(ST_EUNSUPPORTED, "%s: 2^31 tokens or rows, or 2^24 columns, and more", what);
  return ST_OK;
}

// Threads of a workgroup over the columns of a row, VEC at a time.
unsigned threads_of(int64_t H, int VEC) {
  const int64_t t = st::cdiv(st::cdiv(H, VEC), 64) * 64;
  return (unsigned)(t < NTH ? t : NTH);
}

}  // namespace

extern "C" int st_embedding_fwd(const void* table, int32_t dtype, const void* ids, int32_t ids32,
                                int64_t n, int64_t vocab, int64_t hidden, float scale,
                                uint16_t* out, st_stream_t stream) {
  const int rc = check_sizes("st_embedding_fwd", n, vocab, hidden);
  if (rc != ST_OK) return rc;
  ST_CHECK_ARG(dtype == ST_DTYPE_BF16 || dtype == ST_DTYPE_F32, "dtype codes are bf16 and fp32");
  if (n == 0) return ST_OK;
  ST_CHECK_ARG(table && ids && out, "st_embedding_fwd: NULL");
  const bool whole = hidden % 8 == 0 && (((uintptr_t)table | (uintptr_t)out) & 15) == 0;
  const unsigned grid = (unsigned)(n < (1 << 20) ? n : 1 << 20);
  const unsigned th = threads_of(hidden, hidden < 8 ? 1 : 8);
  const hipStream_t s = (hipStream_t)stream;
  auto run = [&](auto kernel) {
    kernel<<<grid, th, 0, s>>>(table, ids, ids32, n, vocab, hidden, scale, out);
  };
  const bool f32 = dtype == ST_DTYPE_F32;
  if (hidden < 8)
    f32 ? run(lookup<1, true, false>) : run(lookup<1, false, false>);
  else if (whole)
    f32 ? run(lookup<8, true, false>) : run(lookup<8, false, false>);
  else
    f32 ? run(lookup<8, true, true>) : run(lookup<8, false, true>);
  return st::check_launch("st_embedding_fwd");
}

extern "C" int64_t st_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t hidden) {
  if (n < 1 || check_sizes("st_embedding_bwd", n, vocab, hidden) != ST_OK) return 0;
  return layout(n, hidden).bytes;
}

extern "C" int st_embedding_bwd(const uint16_t* dout, const void* ids, int32_t ids32, int64_t n,
                                int64_t vocab, int64_t hidden, float scale, int64_t padding_idx,
                                void* grad, int32_t grad_dtype, int32_t accumulate, void* workspace,
                                int64_t workspace_bytes, st_stream_t stream) {
  const int rc = check_sizes("st_embedding_bwd", n, vocab, hidden);
  if (rc != ST_OK) return rc;
  ST_CHECK_ARG(grad_dtype == ST_DTYPE_BF16 || grad_dtype == ST_DTYPE_F32,
               "dtype codes are bf16 and fp32");
  ST_CHECK_ARG(!accumulate || grad_dtype == ST_DTYPE_F32,
               "st_embedding_bwd adds to fp32 gradients only");
  ST_CHECK_ARG(grad && ((uintptr_t)grad & 15) == 0, "st_embedding_bwd: NULL or misaligned gradient");
  // as many columns a lane as make 16 bytes of the gradient
  const int vec = hidden < 8 ? 1 : grad_dtype == ST_DTYPE_F32 ? 4 : 8;
  const unsigned th = threads_of(hidden, vec);
  const int64_t chunks = st::cdiv(n, chunk_of(n)), slices = st::cdiv(hidden, (int64_t)th * vec);
  if (chunks * slices * th >= (int64_t)1 << 32)
    return st::fail(ST_EUNSUPPORTED, "st_embedding_bwd: more threads than a launch takes");
  const hipStream_t s = (hipStream_t)stream;
  const int64_t bytes = vocab * hidden * (grad_dtype == ST_DTYPE_F32 ? 4 : 2);
  const int64_t words = accumulate ? 0 : bytes / 16;
  const int tail = accumulate ? 0 : (int)(bytes % 16 / 2);
  if (n > 0) {
    ST_CHECK_ARG(dout && ids, "st_embedding_bwd: NULL");
    const int64_t need = layout(n, hidden).bytes;
    if (!workspace || workspace_bytes < need)
      return st::fail(ST_EWORKSPACE, "st_embedding_bwd needs %lld workspace bytes", (long long)need);
    ST_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
  }
  const unsigned fill = clear_blocks(words);
  if (tail)
    clear_tail<<<1, 64, 0, s>>>((uint16_t*)((char*)grad + bytes - 2 * tail), tail);
  if (n == 0) {
    if (words) clear_words<<<fill, NTH, 0, s>>>((uint4*)grad, words);
    return st::check_launch("st_embedding_bwd");
  }
  const Layout l = layout(n, hidden);
  char* w = (char*)workspace;
  const int passes = passes_of(vocab);
  int last = 0;
  if (n <= SMALL) {
    const bool apart = words > CLEAR_APART;
    if (apart) clear_words<<<fill, NTH, 0, s>>>((uint4*)grad, words);
    sort_small<<<1 + (apart ? 0 : (fill + 3) / 4), 1024, 0, s>>>(
        ids, ids32, (int)n, vocab, padding_idx, passes, (uint32_t*)(w + l.tok[0]),
        (uint32_t*)(w + l.pos[0]), (uint4*)grad, apart ? 0 : words);
  } else {
    const int64_t tiles = st::cdiv(n, TILE);
    uint32_t* counts = (uint32_t*)(w + l.counts);
    for (int p = 0; p < passes; ++p) {
      const uint32_t* tok = p ? (const uint32_t*)(w + l.tok[last]) : nullptr;
      const uint32_t* pos = p ? (const uint32_t*)(w + l.pos[last]) : nullptr;
      const int to = p & 1;
      tile_counts<<<(unsigned)(tiles + (p ? 0 : fill)), NTH, 0, s>>>(
          ids, ids32, tok, n, vocab, padding_idx, BITS * p, tiles, counts, (uint4*)grad, words);
      auto move = [&](auto kernel) {
        kernel<<<(unsigned)tiles, NTH, 0, s>>>(ids, ids32, tok, pos, n, vocab, padding_idx, BITS * p,
                                               tiles, counts, (uint32_t*)(w + l.tok[to]),
                                               (uint32_t*)(w + l.pos[to]));
      };
      if (tiles <= MOVE_TILES) {
        move(tile_move<false>);
      } else {
        tile_scan<<<1, 1024, 0, s>>>(counts, BINS * tiles);
        move(tile_move<true>);
      }
      last = to;
    }
  }
  Sums a = {};
  a.dout = dout, a.tok = (const uint32_t*)(w + l.tok[last]), a.pos = (const uint32_t*)(w + l.pos[last]);
  a.n = n, a.V = vocab, a.H = hidden, a.chunk = chunk_of(n), a.scale = scale;
  a.grad_f32 = grad_dtype == ST_DTYPE_F32, a.accumulate = accumulate, a.grad = grad;
  a.partial = (float*)(w + l.partial);
  const bool even = hidden % 8 == 0 && ((uintptr_t)dout & 15) == 0;
  const dim3 grid((unsigned)chunks, (unsigned)slices), more((unsigned)chunks - 1, (unsigned)slices);
  auto sums = [&](auto whole, auto runs, auto join) {
    if (n <= WHOLE) {
      whole<<<grid, th, 0, s>>>(a);
    } else {
      runs<<<grid, th, 0, s>>>(a);
      if (chunks > 1) join<<<more, th, 0, s>>>(a);
    }
  };
  if (vec == 1)
    sums(sum_whole<1, false>, sum_runs<1, false>, join_runs<1, false>);
  else if (vec == 4 && even)
    sums(sum_whole<4, false>, sum_runs<4, false>, join_runs<4, false>);
  else if (vec == 4)
    sums(sum_whole<4, true>, sum_runs<4, true>, join_runs<4, true>);
  else if (even)
    sums(sum_whole<8, false>, sum_runs<8, false>, join_runs<8, false>);
  else
    sums(sum_whole<8, true>, sum_runs<8, true>, join_runs<8, true>);
  return st::check_launch("st_embedding_bwd");
}
