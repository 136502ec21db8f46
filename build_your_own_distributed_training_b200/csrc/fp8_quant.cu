// Quantisation to 8-bit floating point (e4m3) with one power-of-two scale for each block of 128.
//
// A block's scale is the least 2^e with max|x| <= 448 * 2^e (448 = 1.75 * 2^8 is the largest e4m3
// number), stored as its biased exponent (e8m0); x * 2^-e is exact, so the only rounding is the one to
// e4m3 (nearest even).  Blocks are 1 x 128 along the axis that a product sums over (activations and
// gradients) or 128 x 128 (weights, whose codes then serve both products that read them).  A block whose
// largest magnitude is below 2^-100, zeros included, takes the scale for 2^-100; NaN or infinity in a
// block makes its scale NaN, so every product it enters is NaN.
//
// Training needs each operand along two axes: activations along features (forward) and along tokens
// (weight gradient).  One kernel reads a 128 x 128 tile once, holds it in registers (8 x 8 elements per
// thread), and writes the codes as they lie and transposed, so that both products get operands whose
// summed axis is contiguous.  2 bytes in, 1 or 2 bytes out per element: 8192 x 4096 bf16 takes 24 us as it
// lies, 34 us both ways (4.0 TB/s), 25 us both ways in 128 x 128 blocks, whose one scale lets the transposed
// codes be byte permutes of the others.  The 1 x 128 form uses 67% of the issue slots: a product by the
// scale and a conversion for each of an element's two codes.  Magnitudes go two elements at a time (71 us before).  The transposed
// codes go through 16 KB of shared memory in 8-byte chunks (8 rows of one column) at chunk
// rg ^ (column / 8), which is free of bank conflicts on the way in, and leave as 16-byte stores.
//
// Scales leave twice: plain (1 x 128 blocks block-major, s[block][row]), for whoever reads the codes, and
// as the 512-byte tiles that the product copies to tensor memory as they are (fp8_gemm.cu).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>
#include <torch/extension.h>

#include <algorithm>

#include "common.cuh"
#include "fp8.cuh"
#include "vecio.cuh"

namespace dtb {
namespace fp8 {

// |x| as ordered bits: infinity and NaN compare above every finite magnitude
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// biased exponent of the block's scale from the bits of its largest magnitude
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255u;             // NaN
  amax = max(amax, 27u << 23);                      // 2^-100
  // amax = f * 2^E, 1 <= f < 2: e = E - 8 where f <= 1.75, E - 7 above
  return (amax >> 23) - 8u + ((amax & 0x7fffffu) > 0x600000u ? 1u : 0u);
}
// 2^-e, the factor that brings the block into range (NaN for a NaN scale)
__device__ __forceinline__ float inv_scale(uint32_t byte) {
  return byte == 255u ? __int_as_float(0x7fc00000) : __uint_as_float((254u - byte) << 23);
}

__device__ __forceinline__ uint32_t cvt4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

struct QuantArgs {
  const void* x;      // [R, C], row stride ld
  long ld;
  int R, C;
  uint8_t* q;         // [R, q_ld] codes as they lie, or null
  long q_ld;
  uint8_t* s;         // 1 x 128: [C / 128][R]; 128 x 128: [R / 128][C / 128]; or null (tiles alone)
  uint8_t* qt;        // [C, qt_ld] transposed codes, or null
  long qt_ld;
  uint8_t* st;        // 1 x 128 of the transpose: [R / 128][C], or null
  uint8_t* t;         // scale tiles of the codes as they lie: [R / 128][C / 512][512]
  uint8_t* tt;        // and of the transpose: [C / 128][R / 512][512]
};

// Byte of (row r of 128, k block `kb`) from the start of its row block's scale tiles.
__device__ __forceinline__ long tile_byte(int r, long kb) {
  return (kb >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (kb & 3);
}

// Two 16-bit magnitudes (sign bits cleared, so ordered as integers: infinity and NaN above every finite) at a time.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.s16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// fp32 bits of a 16-bit magnitude
template <typename T>
__device__ __forceinline__ uint32_t widen(uint32_t m);
template <>
__device__ __forceinline__ uint32_t widen<__nv_bfloat16>(uint32_t m) { return m << 16; }
template <>
__device__ __forceinline__ uint32_t widen<__half>(uint32_t m) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}

// Largest magnitudes (fp32 bits) of a thread's 8 x 8 elements: of each row over the 16 lanes of the row
// (ROWS), of each column over the thread's rows (COLS).  16-bit types go two at a time.
template <typename T, bool ROWS, bool COLS>
__device__ __forceinline__ void magnitudes(const Pack<T, 8> (&v)[8], uint32_t (&rmax)[8], uint32_t (&cmax)[8]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t c[4] = {0, 0, 0, 0}, r[4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      uint32_t m[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint4& q = v[i + p].w[0];
        const uint32_t a0 = q.x & 0x7fff7fffu, a1 = q.y & 0x7fff7fffu, a2 = q.z & 0x7fff7fffu, a3 = q.w & 0x7fff7fffu;
        if (COLS) c[0] = max2(c[0], a0), c[1] = max2(c[1], a1), c[2] = max2(c[2], a2), c[3] = max2(c[3], a3);
        m[p] = max2(max2(a0, a1), max2(a2, a3));
      }
      r[i / 2] = max2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));  // row i low, i + 1 high
    }
    if (ROWS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) r[i] = max2(r[i], __shfl_xor_sync(0xffffffffu, r[i], o));
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) rmax[i] = widen<T>((i & 1) ? r[i / 2] >> 16 : r[i / 2] & 0xffffu);
    if (COLS) {
#pragma unroll
      for (int k = 0; k < 8; ++k) cmax[k] = widen<T>((k & 1) ? c[k / 2] >> 16 : c[k / 2] & 0xffffu);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rmax[i] = cmax[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t m = mag(v[i].at(k));
        rmax[i] = max(rmax[i], m);
        cmax[k] = max(cmax[k], m);
      }
    if (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) rmax[i] = max(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
    }
  }
}

template <typename T>
__device__ __forceinline__ uint2 codes8(const Pack<T, 8>& v, float f) {
  return make_uint2(cvt4(v.at(0) * f, v.at(1) * f, v.at(2) * f, v.at(3) * f),
                    cvt4(v.at(4) * f, v.at(5) * f, v.at(6) * f, v.at(7) * f));
}

// bytes (row i, column k) of four words a[i] -> words (column k)
__device__ __forceinline__ void transpose4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t (&c)[4]) {
  const uint32_t t0 = __byte_perm(a0, a1, 0x5140), t1 = __byte_perm(a2, a3, 0x5140);
  const uint32_t t2 = __byte_perm(a0, a1, 0x7362), t3 = __byte_perm(a2, a3, 0x7362);
  c[0] = __byte_perm(t0, t1, 0x5410);
  c[1] = __byte_perm(t0, t1, 0x7632);
  c[2] = __byte_perm(t2, t3, 0x5410);
  c[3] = __byte_perm(t2, t3, 0x7632);
}

// One 128 x 128 tile per block of 256 threads: thread (rg, cg) holds rows rg * 8 + i, columns cg * 8 + k.
template <typename T, bool SQUARE, bool WIDE>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) quant_tile_kernel(const QuantArgs a) {
  __shared__ __align__(16) uint8_t sh[128 * 128];
  __shared__ __align__(16) uint32_t colmax[8][128];
  const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4, warp = tid >> 5, lane = tid & 31;
  const int r0 = blockIdx.y * 128 + rg * 8, c0 = blockIdx.x * 128 + cg * 8;
  const long tq = (gridDim.x + 3) >> 2, ttq = (gridDim.y + 3) >> 2;  // scale tiles per row block
  const T* x = reinterpret_cast<const T*>(a.x);
  Pack<T, 8> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + i;
    if (WIDE && row < a.R && c0 + 8 <= a.C) {
      v[i].load(x + row * a.ld + c0);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[i].e[k] = (row < a.R && c0 + k < a.C) ? x[row * a.ld + c0 + k] : from_float<T>(0.f);
    }
  }
  uint32_t rmax[8], cmax[8];
  if constexpr (SQUARE) {
    magnitudes<T, false, false>(v, rmax, cmax);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, rmax[i]);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) colmax[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, colmax[0][w]);
    const uint8_t b = (uint8_t)scale_byte(m);
    if (tid == 0 && a.s != nullptr) a.s[(long)blockIdx.y * gridDim.x + blockIdx.x] = b;
    if (tid < 128 && a.t != nullptr) a.t[blockIdx.y * tq * 512 + tile_byte(tid, blockIdx.x)] = b;
    if (tid >= 128 && a.tt != nullptr) a.tt[blockIdx.x * ttq * 512 + tile_byte(tid - 128, blockIdx.y)] = b;
    const float f = inv_scale(b);
    uint2 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = codes8(v[i], f);
      // q_ld is a multiple of 16: the padding columns get zeros
      if (a.q != nullptr && r0 + i < a.R && c0 < a.q_ld)
        *reinterpret_cast<uint2*>(a.q + (long)(r0 + i) * a.q_ld + c0) = o[i];
    }
    if (a.qt == nullptr) return;
    // one scale: the transposed codes are the same codes
    uint32_t lo[4], hi[4];
    transpose4(o[0].x, o[1].x, o[2].x, o[3].x, lo);
    transpose4(o[4].x, o[5].x, o[6].x, o[7].x, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<uint2*>(sh + (cg * 8 + k) * 128 + ((rg ^ cg) << 3)) = make_uint2(lo[k], hi[k]);
    transpose4(o[0].y, o[1].y, o[2].y, o[3].y, lo);
    transpose4(o[4].y, o[5].y, o[6].y, o[7].y, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<uint2*>(sh + (cg * 8 + 4 + k) * 128 + ((rg ^ cg) << 3)) = make_uint2(lo[k], hi[k]);
  } else {
    if (a.q != nullptr) {
      magnitudes<T, true, true>(v, rmax, cmax);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = scale_byte(rmax[i]);
        if (cg == i) {
          if (r0 + i < a.R && a.s != nullptr) a.s[(long)blockIdx.x * a.R + r0 + i] = (uint8_t)b;
          a.t[blockIdx.y * tq * 512 + tile_byte(rg * 8 + i, blockIdx.x)] = (uint8_t)b;
        }
        if (r0 + i < a.R && c0 < a.q_ld)
          *reinterpret_cast<uint2*>(a.q + (long)(r0 + i) * a.q_ld + c0) = codes8(v[i], inv_scale(b));
      }
    } else {
      magnitudes<T, false, true>(v, rmax, cmax);
    }
    if (a.qt == nullptr) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) cmax[k] = max(cmax[k], __shfl_xor_sync(0xffffffffu, cmax[k], 16));
    if (lane < 16) {
      uint4* d = reinterpret_cast<uint4*>(&colmax[warp][cg * 8]);
      d[0] = make_uint4(cmax[0], cmax[1], cmax[2], cmax[3]);
      d[1] = make_uint4(cmax[4], cmax[5], cmax[6], cmax[7]);
    }
    __syncthreads();
    if (tid < 128) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) m = max(m, colmax[w][tid]);
      const uint32_t b = scale_byte(m);
      const int col = blockIdx.x * 128 + tid;
      if (col < a.C && a.st != nullptr) a.st[(long)blockIdx.y * a.C + col] = (uint8_t)b;
      a.tt[blockIdx.x * ttq * 512 + tile_byte(tid, blockIdx.y)] = (uint8_t)b;
      colmax[0][tid] = __float_as_uint(inv_scale(b));
    }
    __syncthreads();
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(colmax[0][cg * 8 + k]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint2 o;
      o.x = cvt4(v[0].at(k) * f[k], v[1].at(k) * f[k], v[2].at(k) * f[k], v[3].at(k) * f[k]);
      o.y = cvt4(v[4].at(k) * f[k], v[5].at(k) * f[k], v[6].at(k) * f[k], v[7].at(k) * f[k]);
      *reinterpret_cast<uint2*>(sh + (cg * 8 + k) * 128 + ((rg ^ cg) << 3)) = o;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (tid >> 3) + i * 32, j = tid & 7;  // column of x, pair of chunks (16 rows)
    const int col = blockIdx.x * 128 + c;
    const long row = (long)blockIdx.y * 128 + j * 16;
    if (col >= a.C || row >= a.qt_ld) continue;
    const uint8_t* src = sh + c * 128;
    const uint2 lo = *reinterpret_cast<const uint2*>(src + (((2 * j) ^ (c >> 3)) << 3));
    const uint2 hi = *reinterpret_cast<const uint2*>(src + (((2 * j + 1) ^ (c >> 3)) << 3));
    *reinterpret_cast<uint4*>(a.qt + (long)col * a.qt_ld + row) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}

// A few rows alone (1 x 128, codes as they lie): 16 lanes per block of 128.  Blocks from `quant_blocks` on make
// the scale tiles of the other operand, so that a few tokens against kept weights need one launch before the
// product.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantArgs a, int quant_blocks, const TileJob job) {
  let_successor_start();
  if ((int)blockIdx.x >= quant_blocks) {
    const int t = ((int)blockIdx.x - quant_blocks) * 2 + (threadIdx.x >> 7);
    if (t < job.count) make_tile_word(job, t, threadIdx.x & 127);
    return;
  }
  const int cb = (a.C + 127) / 128;
  const int item = blockIdx.x * 16 + (threadIdx.x >> 4), cg = threadIdx.x & 15;  // (row, block) pair
  const bool live = item < a.R * cb;
  const int row = live ? item / cb : 0, blk = live ? item % cb : 0;
  const int c0 = blk * 128 + cg * 8;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  Pack<T, 8> v;
  if (WIDE && live && c0 + 8 <= a.C) {
    v.load(x + c0);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v.e[k] = (live && c0 + k < a.C) ? x[c0 + k] : from_float<T>(0.f);
  }
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, mag(v.at(k)));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (!live) return;
  const uint32_t b = scale_byte(m);
  if (cg == 0) {
    if (a.s != nullptr) a.s[(long)blk * a.R + row] = (uint8_t)b;
    a.t[tile_byte(row, blk)] = (uint8_t)b;  // fewer than 128 rows: one row block
  }
  if (c0 < a.q_ld) *reinterpret_cast<uint2*>(a.q + row * a.q_ld + c0) = codes8(v, inv_scale(b));
}

}  // namespace fp8
}  // namespace dtb

using namespace dtb;

// x [R, C] -> {codes [R, C], scales, scale tiles, transposed codes [C, R], their scales, their scale tiles}.
// square: 128 x 128 blocks, scales [R/128, C/128] and their transpose; else 1 x 128 along the last axis of
// each output, scales [R, C/128] and [C, R/128] (block-major in memory).  Codes lie in rows padded to 16
// bytes.  `plain` / `transposed` select which of the two are made (undefined tensors stand for the other).
static std::vector<torch::Tensor> quantize(torch::Tensor x, bool square, bool plain, bool transposed, fp8::TileJob job,
                                           bool scales = true) {
  DTB_CHECK(x.is_cuda() && x.dim() == 2 && is_float_type(x.scalar_type()) && (x.numel() == 0 || x.size(1) == 1 || x.stride(1) == 1), "fp8_quantize: x must be a 2-D CUDA tensor of fp32, bf16 or fp16 with contiguous columns");
  DTB_CHECK(plain || transposed, "fp8_quantize: nothing asked for");
  DTB_CHECK(x.size(0) < (1L << 31) - 256 && x.size(1) < (1L << 31) - 256, "fp8_quantize: too large");
  const c10::cuda::CUDAGuard guard(x.device());
  const long R = x.size(0), C = x.size(1), RB = (R + 127) / 128, CB = (C + 127) / 128;
  auto codes = [&](long rows, long cols) {
    const long pitch = (cols + 15) / 16 * 16;
    return torch::empty({rows, pitch}, x.options().dtype(at::kFloat8_e4m3fn)).narrow(1, 0, cols);
  };
  auto opts = x.options().dtype(at::kFloat8_e8m0fnu);
  auto tiles = [&](long rb, long cb) { return torch::empty({rb, (cb + 3) / 4, 512}, x.options().dtype(at::kByte)); };
  torch::Tensor q, s, t, qt, st, tt;
  if (plain) t = tiles(RB, CB);
  if (transposed) tt = tiles(CB, RB);
  if (plain) q = codes(R, C);
  if (transposed) qt = codes(C, R);
  if (square && scales) {
    s = torch::empty({RB, CB}, opts);
    st = s.t();
  } else if (scales) {
    if (plain) s = torch::empty({CB, R}, opts).t();
    if (transposed) st = torch::empty({RB, C}, opts).t();
  }
  if (R == 0 || C == 0) return {q, s, t, qt, st, tt};
  fp8::QuantArgs a{};
  a.x = x.data_ptr();
  a.ld = x.stride(0);
  a.R = (int)R;
  a.C = (int)C;
  if (plain) {
    a.q = reinterpret_cast<uint8_t*>(q.data_ptr());
    a.q_ld = (C + 15) / 16 * 16;
  }
  if (plain) a.t = t.data_ptr<uint8_t>();
  if (transposed) a.tt = tt.data_ptr<uint8_t>();
  if (scales && (square || plain)) a.s = reinterpret_cast<uint8_t*>(s.data_ptr());
  if (transposed) {
    a.qt = reinterpret_cast<uint8_t*>(qt.data_ptr());
    a.qt_ld = (R + 15) / 16 * 16;
    if (scales && !square) a.st = reinterpret_cast<uint8_t*>(st.data_ptr());
  }
  const bool wide = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && (a.ld * (long)x.element_size()) % 16 == 0;
  auto stream = at::cuda::getCurrentCUDAStream();
  // Under 128 rows a tile per block would leave most of its threads without rows; from there on the tile
  // kernel also writes the scales together (8192 x 4096: 34 us by rows, 28 by tiles).
  const bool tile = square || transposed || R >= 128;
  DTB_CHECK(!tile || RB <= 65535, "fp8_quantize: more than 8388480 rows");
  const dim3 grid((unsigned)CB, (unsigned)RB);
  const unsigned items = (unsigned)((R * CB + 15) / 16);
  DTB_FLOAT_TYPES(x.scalar_type(), {
    if (tile && square) {
      if (wide) fp8::quant_tile_kernel<T, true, true><<<grid, 256, 0, stream>>>(a);
      else fp8::quant_tile_kernel<T, true, false><<<grid, 256, 0, stream>>>(a);
    } else if (tile) {
      if (wide) fp8::quant_tile_kernel<T, false, true><<<grid, 256, 0, stream>>>(a);
      else fp8::quant_tile_kernel<T, false, false><<<grid, 256, 0, stream>>>(a);
    } else {
      const unsigned n = items + (unsigned)((job.count + 1) / 2);
      if (wide) fp8::quant_rows_kernel<T, true><<<n, 256, 0, stream>>>(a, (int)items, job);
      else fp8::quant_rows_kernel<T, false><<<n, 256, 0, stream>>>(a, (int)items, job);
    }
  });
  DTB_LAUNCH_CHECK();
  return {q, s, t, qt, st, tt};
}

std::vector<torch::Tensor> fp8_quantize(torch::Tensor x, bool square, bool plain, bool transposed) {
  return quantize(x, square, plain, transposed, fp8::TileJob{});
}

// fp8_quantize of x's rows, and in the same launch (under 128 rows) the scale tiles of `rows` rows of codes with
// the plain scales s: {codes, scales, tiles of x, tiles of s}.
torch::Tensor fp8_scale_tiles(torch::Tensor s, int64_t gran, int64_t rows);
std::vector<torch::Tensor> fp8_quantize_with_tiles(torch::Tensor x, torch::Tensor s, int64_t rows) {
  DTB_CHECK(x.dim() == 2, "fp8: a matrix of rows");
  const long mt = (rows + 127) / 128, kb = (x.size(1) + 127) / 128, kq = (kb + fp8::SF_STEP - 1) / fp8::SF_STEP;
  const int64_t gran = s.dim() == 2 && s.size(0) == mt ? 128 : 1;
  DTB_CHECK(s.device() == x.device() && s.scalar_type() == at::kFloat8_e8m0fnu && s.dim() == 2 && s.size(0) == (rows + gran - 1) / gran && s.size(1) == kb && mt * kq < (1L << 31), "fp8: scales must be e8m0 [%ld or %ld, %ld] on x's device", (long)rows, mt, kb);
  if (x.size(0) == 0 || x.size(0) >= 128 || x.size(1) == 0 || rows == 0) {
    auto q = quantize(x, false, true, false, fp8::TileJob{});
    return {q[0], q[1], q[2], fp8_scale_tiles(s, gran, rows)};
  }
  auto t = torch::empty({mt, kq, 512}, x.options().dtype(at::kByte));
  auto q = quantize(x, false, true, false, fp8::TileJob{reinterpret_cast<const uint8_t*>(s.data_ptr()), s.stride(0), s.stride(1), (int)gran,
                                                        (int)rows, (int)kb, (int)kq, reinterpret_cast<uint32_t*>(t.data_ptr()), (int)(mt * kq)});
  return {q[0], q[1], q[2], t};
}

// fp8_quantize without the plain scales: {codes, tiles, transposed codes, their tiles}.
std::vector<torch::Tensor> fp8_quantize_tiles(torch::Tensor x, bool square, bool plain, bool transposed) {
  auto q = quantize(x, square, plain, transposed, fp8::TileJob{}, false);
  return {q[0], q[2], q[3], q[5]};
}
