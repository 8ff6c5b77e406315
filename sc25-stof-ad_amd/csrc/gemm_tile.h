// Pieces shared by the GEMM kernels (16-bit: gemm_epilogue_gfx950.hip, 8-bit: gemm_i8_gfx950.hip): LDS tiles of
// 128-byte rows filled by direct-to-LDS loads, fragment reads, and the order in which workgroups take output tiles.
#pragma once
#include "stof_common.h"

namespace {

typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(1))) const void gptr_t;

// chunk c (16 B) of tile row r is stored at chunk position c ^ swz(r)
__device__ __forceinline__ int swz(int row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

__device__ __forceinline__ half8_t lds_frag(const lds_byte* tile, int byte_off) {
  return *reinterpret_cast<const __attribute__((address_space(3))) half8_t*>(tile + byte_off);
}
__device__ __forceinline__ void dma16(const half_t* src, lds_byte* dst) {
  __builtin_amdgcn_global_load_lds((gptr_t*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
// The operand tiles of the K loops are addressed through buffer resources: the tile's first row as
// a wave-uniform base in scalar registers (set up once per workgroup), the lane's place inside the
// tile as a 32-bit byte offset computed once, the position along K as a scalar offset - no 64-bit
// vector add per load instruction.  (Extent 2^32 - 1: every address is in range by construction,
// rows past the edge re-read the last row.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const half_t* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t*>(base), 0, -1, 0x00020000);
}
__device__ __forceinline__ void dma16b(__amdgpu_buffer_rsrc_t rsrc, uint32_t lane_off, uint32_t k_off, lds_byte* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)dst, 16, lane_off, k_off, 0, 0);
}

// Workgroup index -> output tile.  Workgroups go round-robin to the 8 XCDs, each with an L2 of
// its own, and about 64 of them run on an XCD at a time.  XCD x = index % 8 owns the token tiles
// tm = 8 q + x and takes its tiles in bands of kRasterRows values of q, feature tile after feature
// tile inside a band: the 64 workgroups in flight on an XCD then cover 8 token tiles x 8 feature
// tiles and bring 8 + 8 operand tiles through its L2 instead of 64 + 1 (token tile after token
// tile for one feature tile re-read the activations once per feature tile from memory:
// 65536 x 3072 x 768 470 us = 660 TFLOP/s where 8192 rows reach 840).
// The grid is 8 * ceil(tiles_m / 8) * tiles_n; false = padding of the last token tiles.
constexpr int kRasterRows = 8;
__device__ __forceinline__ bool raster_tile(int index, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int x = index & 7, i = index >> 3;
  const int rows_x = (tiles_m + 7) >> 3;
  const int band = i / (kRasterRows * tiles_n), r = i - band * (kRasterRows * tiles_n);
  const int first = band * kRasterRows;
  const int rows = min(kRasterRows, rows_x - first);
  tn = r / rows;
  tm = 8 * (first + r - tn * rows) + x;
  return tm < tiles_m;
}
inline unsigned raster_grid(int tiles_m, int tiles_n) { return 8u * (unsigned)((tiles_m + 7) / 8) * (unsigned)tiles_n; }

}  // namespace
