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

// Row-major [rows][D] LDS tile, 16-byte chunks XOR-swizzled by row.  For
// D = 128 (rows of 256 bytes, each starting at bank 0) the XOR value
// ((row & 3) << 2) | ((row >> 2) & 3) is a permutation of row & 15, so the
// 16 rows of a quarter-wave 16-byte read (tile_row) land on 16 distinct chunk
// positions, and the 4 rows x 4 chunks of a half-wave transposing 8-byte read
// (tile_tr: rows 4 apart in bits 2-3 of the XOR value, chunks in bits 0-1)
// land on 16 distinct chunks: both are free of bank conflicts.  Other widths
// keep the XOR value ((row & 7) << 1), which stays inside the row's chunks.
template <int D>
__device__ __forceinline__ int swz(int row) {
  if constexpr (D == 128)
    return ((row & 3) << 2) | ((row >> 2) & 3);
  else
    return ((row & 7) << 1) & (D / 8 - 1);
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

}  // namespace attn
