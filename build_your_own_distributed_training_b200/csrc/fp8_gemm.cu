// Matrix product of 8-bit operands with one power-of-two scale for each block of 128 (sm_100a).
//
//   D[m, n] = sum_k A[m, k] sA[m, k / 128] B[n, k] sB[n / g, k / 128]      (g = 1 or 128; also A may have g = 128)
//
// A [M, K] and B [N, K] are e4m3 codes with the summed axis contiguous; the scales are e8m0.
//
// Persistent tcgen05 kernel, one CTA per SM, 12 warps:
//   warp 0       TMA: 128 x 128-byte tiles of A and B (128-byte swizzle) into a 4-stage ring;
//   warp 1       one thread issues, per stage, three tcgen05.cp (the stage's scales, shared memory ->
//                tensor memory) and four block-scaled MMAs (kind::mxf8f6f4, 128 x BN x 32);
//   warps 2, 3   gather the scale bytes of A's and B's rows of the stage from global memory, four stages
//                ahead in registers, and lay them out for tcgen05.cp;
//   warps 4-11   epilogue: two warpgroups, each half of the tile's columns.
// The hardware applies a scale to 32 elements; a block of 128 is four of them, so a 128-deep stage has one
// scale byte per row, repeated in the four byte places of its 32-bit word, and every MMA of the stage reads
// the word's byte 0.  Powers of two make the scaling exact: the sum is the fp32 accumulation of the codes'
// products in tensor memory, over all of K, with no promotion pass through registers.
//
// Tensor memory: the accumulator takes 256 columns (one 128 x 256 tile, or two 128 x 128 tiles in turn), the
// scales 16 columns per stage.  With 256-column tiles the accumulator is read into registers as bf16 before
// the tile is stored, so the MMAs of the next tile wait only for that read.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>
#include <torch/extension.h>

#include <algorithm>

#include "common.cuh"
#include "vecio.cuh"

namespace dtb {
namespace fp8 {

enum Out : int { OUT_BF16 = 0, OUT_F32 = 1, OUT_ACC_F32 = 2 };

struct Scale {
  const uint8_t* s;
  long row, blk;  // strides of the row group and of the 128-block of K, in bytes
  int gran;       // rows per group: 1 or 128
};

struct GemmArgs {
  int M, N, K;
  Scale sa, sb;
  void* D;
  long ldd;
  const __nv_bfloat16* R;  // OUT_BF16: residual, or null
  long ldr;
  int m_blocks, n_blocks, k_iters, num_tiles;
  int vec;                 // D (and R) rows start on 16 bytes
  int* err;
};

constexpr int BM = 128, BK = 128, STAGES = 4, GROUP_M = 16;
constexpr uint32_t TMEM_COLS = 512, SF_COL = 256;

template <int BN>
struct Smem {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int SF_OFF = STAGES * STAGE;
  static constexpr int SF_STAGE = 512 * (1 + BN / 128);  // 512 bytes for each 128 rows of A and of B
  static constexpr int STG_OFF = SF_OFF + STAGES * SF_STAGE;
  static constexpr int STG_BYTES = 8 * 2048;             // per epilogue warp: 32 rows x 64 bytes
  static constexpr int BAR_OFF = STG_OFF + STG_BYTES;
  static constexpr int TOTAL = BAR_OFF + 256 + 1024;     // + alignment slack
  static_assert(TOTAL <= 232448, "shared memory per CTA");
};

// kind::mxf8f6f4: e4m3 x e4m3 -> fp32, both K-major, e8m0 scales, scale byte 0 of either operand
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N) {
  return (1u << 23) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_mxf8(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 512 bytes (32 lanes x 16 bytes) of shared memory to 4 columns of every 32-lane quarter
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint32_t saddr) {
  // no swizzle, 8 x 16-byte core matrices one after the other
  const uint64_t desc = (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 16) |
                        ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tile_coords(int tile, int mblocks, int nblocks, int& mb, int& nb) {
  const int per_group = GROUP_M * nblocks;
  const int g = tile / per_group, first = g * GROUP_M;
  const int gm = min(GROUP_M, mblocks - first);
  const int r = tile - g * per_group;
  mb = first + r % gm;
  nb = r / gm;
}

// the scale byte of a row, 1.0 outside the matrix
__device__ __forceinline__ uint32_t scale_of(const Scale& s, int row, int rows, int kb) {
  if (row >= rows) return 127u;
  return __ldg(s.s + (long)(s.gran == 1 ? row : row >> 7) * s.row + (long)kb * s.blk);
}

// 32 rows x 64 bytes staged by the warp (16-byte chunks swizzled by the row) -> global rows
__device__ __forceinline__ uint32_t stg_off(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

template <int OUT>
__device__ __forceinline__ void store_segment(const GemmArgs& a, uint8_t* stg, int row0, int col, int lane) {
  // lane covers rows lane / 4 + 8 i, 16-byte chunk lane % 4: eight 64-byte row pieces per access
  constexpr int ES = OUT == OUT_BF16 ? 2 : 4, PER = 16 / ES;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (lane >> 2) + 8 * i, row = row0 + r, c = col + (lane & 3) * PER;
    if (row >= a.M || c >= a.N) continue;
    uint4 v = *reinterpret_cast<const uint4*>(stg + stg_off(r, lane & 3));
    const bool vec = a.vec && c + PER <= a.N;
    if constexpr (OUT == OUT_BF16) {
      __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(a.D) + (long)row * a.ldd + c;
      if (vec) {
        *reinterpret_cast<uint4*>(d) = v;
      } else {
        const __nv_bfloat16* e = reinterpret_cast<const __nv_bfloat16*>(&v);
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (c + k < a.N) d[k] = e[k];
      }
    } else {
      float* d = reinterpret_cast<float*>(a.D) + (long)row * a.ldd + c;
      float e[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
      if (vec) {
        if constexpr (OUT == OUT_ACC_F32) {
          const float4 o = *reinterpret_cast<const float4*>(d);
          e[0] += o.x, e[1] += o.y, e[2] += o.z, e[3] += o.w;
        }
        *reinterpret_cast<float4*>(d) = make_float4(e[0], e[1], e[2], e[3]);
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (c + k < a.N) d[k] = OUT == OUT_ACC_F32 ? d[k] + e[k] : e[k];
      }
    }
  }
  __syncwarp();
}

// the residual is added in fp32, before the one rounding
__device__ __forceinline__ void add_residual(const GemmArgs& a, int row, int col, float (&v)[32]) {
  if (row >= a.M) return;
  const __nv_bfloat16* r = a.R + (long)row * a.ldr + col;
  if (a.vec && col + 32 <= a.N) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(r + i));
      const uint32_t* u = &q.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = unpack_bf16x2(u[k]);
        v[i + 2 * k] += f.x;
        v[i + 2 * k + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (col + i < a.N) v[i] += __bfloat162float(r[i]);
  }
}

template <int BN, int OUT>
__global__ void __launch_bounds__(384, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const GemmArgs args) {
  using L = Smem<BN>;
  constexpr int ACCS = BN == 256 ? 1 : 2;  // accumulators of BN columns in 256
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 3);  // the TMA thread and the two scale warps
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t issued = 0, issued_phase = 0;  // bit per stage
      bool ok = true;
      for (int tile = blockIdx.x; tile < args.num_tiles && ok; tile += gridDim.x) {
        int mb, nb;
        tile_coords(tile, args.m_blocks, args.n_blocks, mb, nb);
        for (int k = 0; k < args.k_iters; ++k) {
          if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1, args.err)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * L::STAGE;
          mbar_arrive_expect_tx(&full[stage], L::STAGE);
          tma_load_2d(sa, &tmA, &full[stage], k * BK, mb * BM);
#pragma unroll
          for (int j = 0; j < BN / 128; ++j)
            tma_load_2d(sa + L::A_BYTES + j * 16384, &tmB, &full[stage], k * BK, nb * BN + j * 128);
          issued |= 1u << stage;
          issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
      }
      if (!ok)  // copies in flight land before the shared memory goes away
        for (int s = 0; s < STAGES; ++s)
          if (issued >> s & 1) mbar_wait(&full[s], issued_phase >> s & 1, args.err);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, t = 0;
      uint32_t phase = 0;
      bool ok = true;
      constexpr uint32_t IDESC = idesc_mxf8(BM, BN);
      for (int tile = blockIdx.x; tile < args.num_tiles && ok; tile += gridDim.x, ++t) {
        const int acc = t % ACCS;
        const uint32_t acc_phase = (t / ACCS) & 1;
        if (*abort_flag || !mbar_wait(&acc_empty[acc], acc_phase ^ 1, args.err)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        for (int k = 0; k < args.k_iters; ++k) {
          if (*abort_flag || !mbar_wait(&full[stage], phase, args.err)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + stage * L::STAGE), b0 = a0 + L::A_BYTES;
          const uint32_t sf = smem_u32(smem + L::SF_OFF + stage * L::SF_STAGE);
          const uint32_t sfa = tmem + SF_COL + stage * 16, sfb = sfa + 4;
          tmem_copy_scales(sfa, sf);
#pragma unroll
          for (int j = 0; j < BN / 128; ++j) tmem_copy_scales(sfb + 4 * j, sf + 512 * (1 + j));
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk)
            umma_mxf8(tmem + acc * BN, sdesc_sw128(a0 + kk * 32, 16, 1024), sdesc_sw128(b0 + kk * 32, 16, 1024), IDESC,
                      sfa, sfb, k != 0 || kk != 0);
          umma_commit(&empty[stage]);
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
        umma_commit(&acc_full[acc]);
      }
    }
  } else if (warp < 4) {
    // scale bytes: lane l holds rows l, l + 32, l + 64, l + 96 of each 128, PF stages ahead of their use
    constexpr int PF = 4;
    const bool isb = warp == 3;
    const int parts = isb ? BN / 128 : 1;
    const Scale sc = isb ? args.sb : args.sa;
    const int rows = isb ? args.N : args.M;
    uint32_t w[PF][BN / 128][4];
    int ltile = blockIdx.x, lk = 0;  // the next stage to load
    auto load = [&](uint32_t (&d)[BN / 128][4]) {
      if (ltile >= args.num_tiles) return;
      int mb, nb;
      tile_coords(ltile, args.m_blocks, args.n_blocks, mb, nb);
      const int base = isb ? nb * BN : mb * BM;
#pragma unroll
      for (int p = 0; p < BN / 128; ++p)
        if (p < parts) {
#pragma unroll
          for (int j = 0; j < 4; ++j) d[p][j] = scale_of(sc, base + p * 128 + j * 32 + lane, rows, lk);
        }
      if (++lk == args.k_iters) lk = 0, ltile += gridDim.x;
    };
#pragma unroll
    for (int i = 0; i < PF; ++i) load(w[i]);
    const long mine = (args.num_tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1;  // grid <= num_tiles
    const long total = mine * args.k_iters;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (long it = 0; it < total && ok; it += PF) {
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        if (it + i >= total || !ok) break;
        if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1, args.err)) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t* sf = smem + L::SF_OFF + stage * L::SF_STAGE + (isb ? 512 : 0);
#pragma unroll
        for (int p = 0; p < BN / 128; ++p)
          if (p < parts)
            *reinterpret_cast<uint4*>(sf + p * 512 + lane * 16) =
                make_uint4(w[i][p][0] * 0x01010101u, w[i][p][1] * 0x01010101u, w[i][p][2] * 0x01010101u,
                           w[i][p][3] * 0x01010101u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[stage]);
        load(w[i]);
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 4) >> 2;  // TMEM lanes 32 quad .., columns half * BN / 2 ..
    uint8_t* stg = smem + L::STG_OFF + (warp - 4) * 2048;
    constexpr int COLS = BN / 2;
    int t = 0;
    for (int tile = blockIdx.x; tile < args.num_tiles; tile += gridDim.x, ++t) {
      const int acc = t % ACCS;
      const uint32_t acc_phase = (t / ACCS) & 1;
      int mb, nb;
      tile_coords(tile, args.m_blocks, args.n_blocks, mb, nb);
      if (*abort_flag || !mbar_wait(&acc_full[acc], acc_phase, args.err)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t tb = tmem + ((uint32_t)(quad * 32) << 16) + acc * BN + half * COLS;
      const int row0 = mb * BM + quad * 32, col0 = nb * BN + half * COLS;
      if constexpr (OUT == OUT_BF16) {
        uint32_t h[COLS / 2];
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          float v[32];
          tmem_ld32(tb + c, v);
          if (args.R != nullptr) add_residual(args, row0 + lane, col0 + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) h[c / 2 + i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stg + stg_off(lane, i)) =
                make_uint4(h[c / 2 + 4 * i], h[c / 2 + 4 * i + 1], h[c / 2 + 4 * i + 2], h[c / 2 + 4 * i + 3]);
          store_segment<OUT>(args, stg, row0, col0 + c, lane);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < COLS; c += 32) {
          float v[32];
          tmem_ld32(tb + c, v);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float4*>(stg + stg_off(lane, i)) =
                  make_float4(v[16 * g + 4 * i], v[16 * g + 4 * i + 1], v[16 * g + 4 * i + 2], v[16 * g + 4 * i + 3]);
            store_segment<OUT>(args, stg, row0, col0 + c + 16 * g, lane);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[acc]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------- host side
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    DTB_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
    DTB_CHECK(q == cudaDriverEntryPointSuccess && p, "cuTensorMapEncodeTiled not available");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// [rows, inner] bytes, boxes of 128 rows x 128 bytes; bytes past the matrix read as zero
static CUtensorMap make_map(const void* base, long inner, long rows, long pitch) {
  static thread_local bool bound = false;
  if (!bound) {  // the driver call needs a current context on this thread (autograd's workers)
    DTB_CUDA(cudaFree(nullptr));
    bound = true;
  }
  CUtensorMap m;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {128, 128};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  DTB_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d): inner=%ld rows=%ld pitch=%ld base=%p", (int)r, inner, rows, pitch, base);
  return m;
}

template <int BN, int OUT>
static void launch(const CUtensorMap& ta, const CUtensorMap& tb, GemmArgs& g, cudaStream_t st) {
  using L = Smem<BN>;
  auto kern = fp8_gemm_kernel<BN, OUT>;
  DTB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
  g.n_blocks = (g.N + BN - 1) / BN;
  g.num_tiles = g.m_blocks * g.n_blocks;
  kern<<<std::min(g.num_tiles, device_sm_count()), 384, L::TOTAL, st>>>(ta, tb, g);
  DTB_LAUNCH_CHECK();
}

}  // namespace fp8
}  // namespace dtb

using namespace dtb;

static fp8::Scale fp8_scale(const char* which, const torch::Tensor& q, const torch::Tensor& s, int64_t gran) {
  const long kb = (q.size(1) + 127) / 128, groups = (q.size(0) + gran - 1) / gran;
  DTB_CHECK(gran == 1 || gran == 128, "fp8_gemm: %s: blocks have 1 or 128 rows", which);
  DTB_CHECK(s.device() == q.device() && s.scalar_type() == at::kFloat8_e8m0fnu && s.dim() == 2 && s.size(0) == groups && s.size(1) == kb, "fp8_gemm: %s: scales must be e8m0 [%ld, %ld]", which, groups, kb);
  return {reinterpret_cast<const uint8_t*>(s.data_ptr()), s.stride(0), s.stride(1), (int)gran};
}

// D [M, N] = A [M, K] B [N, K]^T (+ R): D bf16 (R bf16, optional) or fp32 (accumulate: D += the product).
void fp8_gemm(torch::Tensor A, torch::Tensor sA, int64_t granA, torch::Tensor B, torch::Tensor sB, int64_t granB,
              torch::Tensor D, c10::optional<torch::Tensor> R, bool accumulate) {
  for (const torch::Tensor* t : {&A, &B})
    DTB_CHECK(t->is_cuda() && t->device() == A.device() && t->scalar_type() == at::kFloat8_e4m3fn && t->dim() == 2 && (t->numel() == 0 || ((t->size(1) == 1 || t->stride(1) == 1) && t->stride(0) % 16 == 0 && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0)), "fp8_gemm: operands must be 2-D e4m3 on one GPU, rows contiguous and starting on 16-byte boundaries");
  const long M = A.size(0), N = B.size(0), K = A.size(1);
  DTB_CHECK(B.size(1) == K && D.dim() == 2 && D.size(0) == M && D.size(1) == N && D.device() == A.device() && (N == 1 || M == 0 || D.stride(1) == 1), "fp8_gemm: shapes do not match");
  DTB_CHECK(D.scalar_type() == at::kBFloat16 || D.scalar_type() == at::kFloat, "fp8_gemm: the result is bf16 or fp32");
  DTB_CHECK(!accumulate || D.scalar_type() == at::kFloat, "fp8_gemm: accumulation is fp32");
  DTB_CHECK(M < (1L << 30) && N < (1L << 30) && K < (1L << 30), "fp8_gemm: too large");
  const c10::cuda::CUDAGuard guard(A.device());
  fp8::GemmArgs g{};
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.sa = fp8_scale("A", A, sA, granA);
  g.sb = fp8_scale("B", B, sB, granB);
  g.D = D.data_ptr();
  g.ldd = M > 1 ? D.stride(0) : N;
  g.err = dtb_error_word();
  const long es = (long)D.element_size();
  g.vec = (reinterpret_cast<uintptr_t>(g.D) & 15) == 0 && (g.ldd * es) % 16 == 0;
  if (R.has_value()) {
    DTB_CHECK(R->device() == A.device() && R->scalar_type() == at::kBFloat16 && D.scalar_type() == at::kBFloat16 && R->sizes() == D.sizes() && (N == 1 || M == 0 || R->stride(1) == 1), "fp8_gemm: the residual must be bf16 with the result's shape");
    g.R = reinterpret_cast<const __nv_bfloat16*>(R->data_ptr());
    g.ldr = M > 1 ? R->stride(0) : N;
    g.vec = g.vec && (reinterpret_cast<uintptr_t>(g.R) & 15) == 0 && (g.ldr * 2) % 16 == 0;
  }
  if (M == 0 || N == 0) return;
  if (K == 0) {
    if (R.has_value()) D.copy_(*R);
    else if (!accumulate) D.zero_();
    return;
  }
  g.m_blocks = (g.M + fp8::BM - 1) / fp8::BM;
  g.k_iters = (g.K + fp8::BK - 1) / fp8::BK;
  auto st = at::cuda::getCurrentCUDAStream();
  const CUtensorMap ta = fp8::make_map(A.data_ptr(), K, M, M > 1 ? A.stride(0) : (K + 15) / 16 * 16);
  const CUtensorMap tb = fp8::make_map(B.data_ptr(), K, N, N > 1 ? B.stride(0) : (K + 15) / 16 * 16);
  // 256-column tiles once they fill the SMs
  const bool wide = (long)g.m_blocks * ((N + 255) / 256) >= device_sm_count();
  const int out = D.scalar_type() == at::kBFloat16 ? fp8::OUT_BF16 : accumulate ? fp8::OUT_ACC_F32 : fp8::OUT_F32;
  if (out == fp8::OUT_BF16) wide ? fp8::launch<256, fp8::OUT_BF16>(ta, tb, g, st) : fp8::launch<128, fp8::OUT_BF16>(ta, tb, g, st);
  else if (out == fp8::OUT_F32) wide ? fp8::launch<256, fp8::OUT_F32>(ta, tb, g, st) : fp8::launch<128, fp8::OUT_F32>(ta, tb, g, st);
  else wide ? fp8::launch<256, fp8::OUT_ACC_F32>(ta, tb, g, st) : fp8::launch<128, fp8::OUT_ACC_F32>(ta, tb, g, st);
}
