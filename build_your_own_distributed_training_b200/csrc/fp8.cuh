// Shared by the 8-bit kernels: the layout of scale tiles, and launches that overlap their predecessor's end.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace dtb {
namespace fp8 {

constexpr int SF_STEP = 4;  // blocks of 128 of K that a scale tile holds

// plain e8m0 scales [row groups, k blocks] (strides in bytes) and the tiles to make of them
struct TileJob {
  const uint8_t* s;
  long row_stride, blk_stride;
  int gran, rows, kb, kq;  // rows per group (1 or 128), rows, k blocks, tiles per row block
  uint32_t* tiles;
  int count;               // tiles in all
};

// word of row r (0..127) of tile `t`; blocks past K get scale 1, rows past the matrix the last row's
__device__ __forceinline__ void make_tile_word(const TileJob& a, int t, int r) {
  const int mt = t / a.kq, k = t % a.kq * SF_STEP;
  const int row = min(mt * 128 + r, a.rows - 1);
  const uint8_t* p = a.s + (long)(a.gran == 1 ? row : mt) * a.row_stride + k * a.blk_stride;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < SF_STEP; ++i) w |= (k + i < a.kb ? (uint32_t)p[i * a.blk_stride] : 127u) << (8 * i);
  a.tiles[(long)t * 128 + (r & 31) * 4 + (r >> 5)] = w;
}

// The product's kernels are launched so that they may start while the kernel before them in the stream still
// runs (their set-up then costs no time of its own): they wait here before they touch memory.  A kernel lets
// its successor start early with the other call; without it the successor starts at its end.  The product
// and the small kernels before it make that call (48 x 4096 x 11008: 17.8 -> 16.0 us); the tile quantisation
// does not, as early blocks of the product would take the shared memory that its own still need (8192 x
// 11008 x 4096 with its quantisation 290 -> 317 us).
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_successor_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace fp8
}  // namespace dtb
