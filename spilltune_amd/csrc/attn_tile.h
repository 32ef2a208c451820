// LDS tiles of the attention kernels: buffer copies into them and the MFMA
// operands read from them.
#pragma once
#include "common.h"

namespace attn {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint4 ld_global16(const uint16_t* p) { return *(const uint4*)p; }

__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

// Buffer copy of 16 bytes per lane into LDS, the 64 lanes of a wave filling
// 1 KiB contiguously from `lds_wave` (wave-uniform); an offset at or past the
// resource's extent reads zeros.  Tiles move the resource base (scalar work)
// and keep each lane's offset fixed, so a copy costs no vector instructions.
__device__ __forceinline__ void b2lds16(__amdgpu_buffer_rsrc_t rs, uint32_t off,
                                        uint16_t* lds_wave) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      rs, (__attribute__((address_space(3))) void*)lds_wave, 16, off, 0, 0, 0);
}

// Thread chunks of a row-major [rows][D] tile (tswz layout) copied by NT
// threads, copy i covering rows i*R .. i*R+R-1 (R = NT/(D/8)).  When R is a
// multiple of 16 every copy puts a thread at the same in-row position (the
// swizzle repeats every 16 rows): one lane offset serves all copies, and
// copy i moves the resource base by i*R rows instead.
template <int D, int NT>
struct RowCopy {
  static constexpr bool uniform = NT % (D / 8) == 0 && (NT / (D / 8)) % 16 == 0;
  static constexpr int rows = NT / (D / 8);
};

// Row-major [rows][D] LDS tile, 16-byte chunks XOR-swizzled by row.  A
// quarter-wave 16-byte read (tile_row: one chunk of 16 rows) and a half-wave
// transposing 8-byte read (tile_tr: 4 chunks of 4 rows, both aligned) must each
// land on 16 distinct positions of the 64 banks.  D = 128: a row is 256 bytes
// and starts at bank 0, so the XOR value ((row & 3) << 2) | ((row >> 2) & 3), a
// permutation of row & 15, serves both (rows apart in bits 2-3, chunks in bits
// 0-1).  D = 64 and 192: rows start at bank 0 and 32 in turn, the XOR value must
// stay below 8 and differ among the 8 rows of one parity, in bit 2 among
// neighbours of one parity: ((row & 2) << 1) | ((row >> 2) & 3).  Measured
// without bank conflicts (SQ_LDS_BANK_CONFLICT).
template <int D>
__device__ __forceinline__ int swz(int row) {
  static_assert(D == 64 || D == 128 || D == 192, "row lengths");
  if constexpr (D == 128)
    return ((row & 3) << 2) | ((row >> 2) & 3);
  else
    return ((row & 2) << 1) | ((row >> 2) & 3);
}
template <int D>
__device__ __forceinline__ int tswz(int row, int chunk) {
  return row * D + ((chunk ^ swz<D>(row)) << 3);
}
template <int D>
__device__ __forceinline__ bf16x8 tile_row(const uint16_t* t, int row, int s, int g) {
  return as_bf16x8(*(const uint4*)(t + tswz<D>(row, 2 * s + g)));
}
// Transposed MFMA operand from a row-major tile: lane (row n = nb + lane%32,
// half g = lane/32) gets tile[kb + (s>>2)*8 + g*4 + (s&3)][n] for s = 0..7,
// the contraction order of a probability block held in MFMA accumulators.
// ds_read_b64_tr_b16: within 16 lanes, lane i receives element (i % 4) of the
// 4-element rows supplied by lanes 4j + i/4, j = 0..3.
template <int D>
__device__ __forceinline__ bf16x8 tile_tr(const uint16_t* t, int kb, int nb, int lane) {
  const int G = lane >> 4, i = lane & 15, g = lane >> 5;
  const int col = nb + 16 * (G & 1) + 4 * (i & 3);
  typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
  v4bf r[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = kb + 8 * h + 4 * g + (i >> 2);
    const uint16_t* p = t + tswz<D>(row, col >> 3) + (col & 7);
    r[h] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) v4bf*)p);
  }
  return __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

// The same two operands by a lane's own address: `lane_row` / `lane_tr` once,
// then one exclusive-or with a constant per read, the rest in the instruction's
// offset (the row's chunks stay within aligned bits of the byte address).  The
// tile comes through a __restrict__ pointer: the caller has waited for its DMAs
// and passed the barrier, and without it the compiler waits for every DMA in
// flight before the first read.
template <int D>
__device__ __forceinline__ uint32_t lane_row(int row, int g) {
  return (uint32_t)(row * D * 2 + ((g ^ swz<D>(row)) << 4));
}
template <int D>  // chunk 2 s + g of row `row0` + the lane's, row0 a multiple of 16
__device__ __forceinline__ bf16x8 read_row(const uint16_t* __restrict__ t, uint32_t lane, int row0, int s) {
  constexpr int IN = D == 128 ? 15 : 7;  // chunks that the swizzle permutes
  const uint32_t at = (lane ^ (uint32_t)((2 * s & IN) << 4)) + (2 * s & ~IN) * 16 + row0 * D * 2;
  return as_bf16x8(*(const uint4*)((const char*)t + at));
}
template <int D>
__device__ __forceinline__ uint32_t lane_tr(int lane) {
  const int G = lane >> 4, i = lane & 15, g = lane >> 5, row = 4 * g + (i >> 2);
  const int chunk = 2 * (G & 1) + ((i & 3) >> 1);
  return (uint32_t)(row * D * 2 + ((chunk ^ swz<D>(row)) << 4) + (i & 1) * 8);
}
template <int D>  // tile_tr(t, kb, 32 db), kb a multiple of 16
__device__ __forceinline__ bf16x8 read_tr(const uint16_t* __restrict__ t, uint32_t lane, int kb, int db) {
  constexpr int IN = D == 128 ? 15 : 7;
  typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
  v4bf r[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // 8 rows on, swz flips bit 1
    const uint32_t at = (lane ^ (uint32_t)(((4 * db & IN) ^ (2 * h)) << 4)) + (4 * db & ~IN) * 16 +
                        (kb + 8 * h) * D * 2;
    r[h] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) v4bf*)((const char*)t + at));
  }
  return __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace attn
