// Matrix product of 8-bit operands with one power-of-two scale for each block of 128 (sm_100a).
//
//   D[m, n] = sum_k A[m, k] sA[m, k / 128] B[n, k] sB[n / g, k / 128]      (g = 1 or 128; also A may have g = 128)
//
// A [M, K] and B [N, K] are e4m3 codes with the summed axis contiguous; the scales are e8m0.
//
// Persistent tcgen05 kernel, 10 warps per CTA, one CTA per SM.  Large products run on CTA pairs: a (2,1,1)
// cluster computes a 256 x 256 tile with cta_group::2 MMAs that the even CTA issues; each CTA holds its 128
// rows of A and 128 columns of B.  Small ones run on single CTAs with 128 x 128 tiles.
//   warp 0       TMA: 128 x 128-byte tiles of A and B (128-byte swizzle) and their scale tiles into a 6-stage
//                ring;
//   warp 1       an elected lane issues, per stage, the tcgen05.cp of the stage's scales (shared memory -> tensor
//                memory) and four block-scaled MMAs (kind::mxf8f6f4, 32 deep);
//   warps 2-9    epilogue: two warpgroups, each half of the tile's columns.
// The hardware applies a scale to 32 elements, one byte of a row's 32-bit scale word; a block of 128 is four
// of them, so the four MMAs of a 128-deep stage read the same byte, and a word serves four stages.  Powers of
// two make the scaling exact: the sum is the fp32 accumulation of the codes' products in tensor memory, over
// all of K, with no promotion pass through registers.
//
// Scale tiles: for each 128 rows and each 512 of K the 512 bytes that tcgen05.cp takes (row r: the 32-bit
// word at (r % 32) * 16 + (r / 32) * 4, byte i the scale of the i-th block of 128), written by the
// quantisation kernels.  They come with every fourth stage.  Gathering scale bytes from a plain [rows,
// blocks] tensor in this kernel was measured and left: two warps per CTA could not keep up (their loads'
// latency came back once per stage), 1230 TFLOP/s at 8192 x 11008 x 4096 where the rest ran at 2290.
//
// 8192 x 11008 x 4096: bf16 result 264 us (2.80 PFLOP/s), fp32 288 us.
//
// What bounds it: a 128 x 256 x 128 step takes the tensor cores 512 cycles, in which one CTA alone would
// move 48 KB into shared memory and read 48 KB from it, 192 bytes a cycle against the 128 there are.  A pair
// halves B's share: 64 KB per CTA and step, 128 bytes a cycle.  At about 1.5 GHz under the power limit a step
// takes some 700 cycles.
//
// Tensor memory: the accumulator takes 256 columns (one 256-column tile, or two 128-column tiles in turn),
// the scales 16 columns for each of eight 512-deep steps in turn.  The accumulator is read into registers
// before the tile is stored, so with 256-column tiles the MMAs of the next tile wait only for that read.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cudaTypedefs.h>
#include <torch/extension.h>

#include <algorithm>

#include "common.cuh"
#include "fp8.cuh"
#include "vecio.cuh"

namespace dtb {
namespace fp8 {

enum Out : int { OUT_BF16 = 0, OUT_F32 = 1, OUT_ACC_F32 = 2 };

struct GemmArgs {
  int M, N, K;
  void* D;
  long ldd;
  const __nv_bfloat16* R;  // OUT_BF16: residual, or null
  long ldr;
  int m_blocks, n_blocks, k_iters, k_quads, num_tiles;
  int a_bytes;             // bytes of A's box: fewer than 128 rows of it when M is smaller
  int splits, k_per;       // K in `splits` parts of k_per blocks (a multiple of SF_STEP); part p writes D + p * M * ldd
  int vec;                 // D (and R) rows start on 16 bytes
  int* err;
};

constexpr int BM = 128, BK = 128, STAGES = 6, GROUP_M = 16;
constexpr int SF_SLOTS = 8;  // places in tensor memory: a slot comes round after 8 stages at least, when the MMAs
                             // of the ring's 6 earlier ones have been waited for
constexpr uint32_t TMEM_COLS = 512, SF_COL = 256;

// PAIR: each CTA of a pair holds half of B's columns
template <int BN, bool PAIR>
struct Smem {
  static constexpr int A_BYTES = BM * BK, B_BYTES = (PAIR ? BN / 2 : BN) * BK;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int SF_OFF = STAGES * STAGE;
  static constexpr int SF_STAGE = 512 * (1 + BN / 128);  // 512 bytes for each 128 rows of A and of B
  static constexpr int STG_OFF = SF_OFF + STAGES * SF_STAGE;
  static constexpr int STG_BYTES = 8 * 2048;             // per epilogue warp: 32 rows x 64 bytes
  static constexpr int BAR_OFF = STG_OFF + STG_BYTES;
  static constexpr int TOTAL = BAR_OFF + 256 + 1024;     // + alignment slack
  static_assert(TOTAL <= 232448, "shared memory per CTA");
};

// kind::mxf8f6f4: e4m3 x e4m3 -> fp32, both K-major, e8m0 scales, byte `sf` of either operand's scale words
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N, uint32_t sf) {
  return (sf << 4) | (sf << 29) | (1u << 23) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
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
__device__ __forceinline__ void umma_mxf8_pair(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa,
                                               uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 512 bytes (32 lanes x 16 bytes) of shared memory to 4 columns of every 32-lane quarter
// (of each CTA of a pair, from its own shared memory)
template <bool PAIR>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint32_t saddr) {
  // no swizzle, 8 x 16-byte core matrices one after the other
  const uint64_t desc = (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(128 >> 4) << 16) |
                        ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// The issuing warps run their loops with all 32 lanes and let one elected lane issue, so that addresses,
// descriptors and branches stay warp-uniform: with a single-lane loop an MMA took 95 cycles to issue and a
// stage's bookkeeping 400, more than the tensor cores need for the stage.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
// mbar_wait for a whole warp: the same answer in every lane, false after 2 s (error word set)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u64 t, u;\n\t"
      "mov.u32 %0, 1;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 t, %%globaltimer;\n\t"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra DONE;\n\t"
      "mov.u64 u, %%globaltimer;\n\t"
      "sub.u64 u, u, t;\n\t"
      "setp.lt.u64 q, u, 2000000000;\n\t"
      "@q bra AGAIN;\n\t"
      "mov.u32 %0, 0;\n\t"
      "DONE:\n\t}"
      : "=&r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, ok != 0)) return true;
  if (err) atomicExch(err, ERR_MBAR_TIMEOUT);
  return false;
}

__device__ __forceinline__ void tile_coords(int tile, int mblocks, int nblocks, int& mb, int& nb) {
  const int per_group = GROUP_M * nblocks;
  const int g = tile / per_group, first = g * GROUP_M;
  const int gm = min(GROUP_M, mblocks - first);
  const int r = tile - g * per_group;
  mb = first + r % gm;
  nb = r / gm;
}

// 32 rows x 64 bytes staged by the warp (16-byte chunks swizzled by the row) -> global rows
__device__ __forceinline__ uint32_t stg_off(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

// Vector stores: lane covers rows lane / 4 + 8 i, 16-byte chunk lane % 4, eight 64-byte row pieces per
// access.  Rows that do not start on 16 bytes: an element per lane, consecutive lanes on consecutive columns.
template <int OUT>
__device__ __forceinline__ void store_segment(const GemmArgs& a, uint8_t* stg, int row0, int col, int part_row, int lane) {
  constexpr int ES = OUT == OUT_BF16 ? 2 : 4, PER = 16 / ES, COLS = 64 / ES;
  __syncwarp();
  if (a.vec && col + COLS <= a.N) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + 8 * i, row = row0 + r;
      if (row >= a.M) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(stg + stg_off(r, lane & 3));
      uint8_t* d = reinterpret_cast<uint8_t*>(a.D) + ((long)(part_row + row) * a.ldd + col + (lane & 3) * PER) * ES;
      if constexpr (OUT == OUT_ACC_F32)
        // each element is added to once, by one thread: the reduction happens in L2 and nothing waits for the
        // old value
        asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(d), "f"(__uint_as_float(v.x)),
                     "f"(__uint_as_float(v.y)), "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w))
                     : "memory");
      else
        *reinterpret_cast<uint4*>(d) = v;
    }
  } else {
    constexpr int ROWS = 32 / COLS;  // rows per access: 1 (bf16) or 2 (fp32)
    const int c = lane % COLS;
#pragma unroll 4
    for (int i = 0; i < 32; i += ROWS) {
      const int r = i + lane / COLS, row = row0 + r;
      if (row >= a.M || col + c >= a.N) continue;
      const uint8_t* e = stg + stg_off(r, c / PER) + (c % PER) * ES;
      const long at = (long)(part_row + row) * a.ldd + col + c;
      if constexpr (OUT == OUT_BF16) {
        reinterpret_cast<__nv_bfloat16*>(a.D)[at] = *reinterpret_cast<const __nv_bfloat16*>(e);
      } else {
        float* d = reinterpret_cast<float*>(a.D) + at;
        *d = (OUT == OUT_ACC_F32 ? *d : 0.f) + *reinterpret_cast<const float*>(e);
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

template <int BN, bool PAIR, int OUT>
__global__ void __launch_bounds__(320, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                    const GemmArgs args) {
  static_assert(PAIR == (BN == 256), "CTA pairs compute 256-column tiles");
  using L = Smem<BN, PAIR>;
  constexpr int ACCS = BN == 256 ? 1 : 2;  // accumulators of BN columns in 256
  constexpr int TILE_M = PAIR ? 2 * BM : BM, CTAS = PAIR ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = PAIR ? (int)cluster_ctarank() : 0;
  const bool leader = cta == 0;
  const int unit = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 8 * CTAS);
    }
    if constexpr (PAIR) fence_mbar_init_cluster();
    else fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_holder, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_holder, TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the peer's barriers exist before any remote arrive
  tc_fence_after();
  let_successor_start();
  wait_for_predecessor();
  // all 512 columns are allocated, so the allocation starts at column 0: a constant base keeps the
  // addresses below warp-uniform
  if (*tmem_holder != 0 && threadIdx.x == 0) atomicExch(args.err, ERR_BAD_ARG);
  constexpr uint32_t tmem = 0;

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0, issued = 0, issued_phase = 0;  // a bit per stage
    bool ok = true;
    for (int u = unit; u < args.num_tiles * args.splits && ok; u += units) {
      const int tile = u / args.splits, k0 = (u - tile * args.splits) * args.k_per;
      const int k1 = min(args.k_iters, k0 + args.k_per);
      int mb, nb;
      tile_coords(tile, args.m_blocks, args.n_blocks, mb, nb);
      // row blocks of this CTA; a pair's CTAs both take all of B's scales, for their own tensor memory
      const int arow = mb * CTAS + cta, brow = nb * (BN / 128);
      int sa_tile = arow * args.k_quads + k0 / SF_STEP, sb_tile = brow * args.k_quads + k0 / SF_STEP;
      for (int k = k0; k < k1; ++k) {
        if (!warp_wait(smem_u32(&empty[stage]), phase ^ 1, args.err)) {
          ok = false;
          break;
        }
        uint8_t* sa = smem + stage * L::STAGE;
        uint8_t* sf = smem + L::SF_OFF + stage * L::SF_STAGE;
        const bool with_sf = k % SF_STEP == 0;
        // a pair's bytes complete on the leader's barrier
        const uint32_t fb = PAIR ? mapa_shared(smem_u32(&full[stage]), 0) : 0;
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(&full[stage], CTAS * (args.a_bytes + L::B_BYTES + (with_sf ? L::SF_STAGE : 0)));
          if constexpr (PAIR) {
            tma_load_2d_pair(sa, &tmA, fb, k * BK, arow * BM);
            tma_load_2d_pair(sa + L::A_BYTES, &tmB, fb, k * BK, (brow + cta) * 128);
            if (with_sf) {
              tma_load_2d_pair(sf, &tmSA, fb, 0, sa_tile);
#pragma unroll
              for (int j = 0; j < BN / 128; ++j)
                tma_load_2d_pair(sf + 512 * (1 + j), &tmSB, fb, 0, sb_tile + j * args.k_quads);
            }
          } else {
            tma_load_2d(sa, &tmA, &full[stage], k * BK, arow * BM);
            tma_load_2d(sa + L::A_BYTES, &tmB, &full[stage], k * BK, brow * 128);
            if (with_sf) {
              tma_load_2d(sf, &tmSA, &full[stage], 0, sa_tile);
              tma_load_2d(sf + 512, &tmSB, &full[stage], 0, sb_tile);
            }
          }
        }
        __syncwarp();
        if (with_sf) ++sa_tile, ++sb_tile;
        issued |= 1u << stage;
        issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
    }
    // copies in flight land before the shared memory goes away (a pair's follower has no barrier of its own
    // for them: its bounded waits outlast its last copy by far)
    if (!ok && leader)
      for (int s = 0; s < STAGES; ++s)
        if (issued >> s & 1) warp_wait(smem_u32(&full[s]), issued_phase >> s & 1, args.err);
  } else if (warp == 1) {
    if (leader) {
      int stage = 0, t = 0, slot = SF_SLOTS - 1;
      uint32_t phase = 0;
      bool ok = true;
      // descriptors of the ring's first stage; a stage or a 32-byte step only adds to the address field
      const uint64_t ad0 = sdesc_sw128(smem_u32(smem), 16, 1024), bd0 = sdesc_sw128(smem_u32(smem) + L::A_BYTES, 16, 1024);
      const uint32_t sf0 = smem_u32(smem + L::SF_OFF);
      for (int u = unit; u < args.num_tiles * args.splits && ok; u += units, ++t) {
        const int k0 = u % args.splits * args.k_per, k1 = min(args.k_iters, k0 + args.k_per);
        const int acc = t % ACCS;
        const uint32_t acc_phase = (t / ACCS) & 1;
        if (!warp_wait(smem_u32(&acc_empty[acc]), acc_phase ^ 1, args.err)) break;
        tc_fence_after();
        for (int k = k0; k < k1; ++k) {
          if (!warp_wait(smem_u32(&full[stage]), phase, args.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sub = k % SF_STEP;
          if (sub == 0) slot = (slot + 1) % SF_SLOTS;
          const uint32_t sfa = tmem + SF_COL + slot * 16, sfb = sfa + 4;
          const uint64_t ad = ad0 + stage * (L::STAGE >> 4), bd = bd0 + stage * (L::STAGE >> 4);
          const uint32_t idesc = idesc_mxf8(TILE_M, BN, 0) | (sub << 4) | (sub << 29);
          if (elect_one()) {
            if (sub == 0) {
              const uint32_t sf = sf0 + stage * L::SF_STAGE;
              tmem_copy_scales<PAIR>(sfa, sf);
#pragma unroll
              for (int j = 0; j < BN / 128; ++j) tmem_copy_scales<PAIR>(sfb + 4 * j, sf + 512 * (1 + j));
            }
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk) {
              if constexpr (PAIR) umma_mxf8_pair(tmem + acc * BN, ad + 2 * kk, bd + 2 * kk, idesc, sfa, sfb, k != k0 || kk != 0);
              else umma_mxf8(tmem + acc * BN, ad + 2 * kk, bd + 2 * kk, idesc, sfa, sfb, k != k0 || kk != 0);
            }
            if constexpr (PAIR) umma_commit_pair(&empty[stage]);
            else umma_commit(&empty[stage]);
          }
          __syncwarp();
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
        if (elect_one()) {
          if constexpr (PAIR) umma_commit_pair(&acc_full[acc]);
          else umma_commit(&acc_full[acc]);
        }
        __syncwarp();
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;  // TMEM lanes 32 quad .., columns half * BN / 2 ..
    uint8_t* stg = smem + L::STG_OFF + (warp - 2) * 2048;
    constexpr int COLS = BN / 2;
    int t = 0;
    for (int u = unit; u < args.num_tiles * args.splits; u += units, ++t) {
      const int tile = u / args.splits;
      const int part_row = (u - tile * args.splits) * args.M;  // the part's first row in D
      const int acc = t % ACCS;
      const uint32_t acc_phase = (t / ACCS) & 1;
      int mb, nb;
      tile_coords(tile, args.m_blocks, args.n_blocks, mb, nb);
      if (!warp_wait(smem_u32(&acc_full[acc]), acc_phase, args.err)) break;
      tc_fence_after();
      const uint32_t tb = tmem + ((uint32_t)(quad * 32) << 16) + acc * BN + half * COLS;
      const int row0 = mb * TILE_M + cta * BM + quad * 32, col0 = nb * BN + half * COLS;
      // the whole share into registers (COLS fp32), so that the accumulator is free before the stores begin
      uint32_t v[COLS / 32][32];
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) tmem_ld32_async(tb + c * 32, v[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) tmem_regs(v[c]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[acc]), 0));
        else mbar_arrive(&acc_empty[acc]);
      }
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) {
        const int col = col0 + c * 32;
        if (col >= args.N) break;
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[c][i]);
        if constexpr (OUT == OUT_BF16) {
          if (args.R != nullptr) add_residual(args, row0 + lane, col, f);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stg + stg_off(lane, i)) =
                make_uint4(pack_bf16x2(f[8 * i], f[8 * i + 1]), pack_bf16x2(f[8 * i + 2], f[8 * i + 3]),
                           pack_bf16x2(f[8 * i + 4], f[8 * i + 5]), pack_bf16x2(f[8 * i + 6], f[8 * i + 7]));
          store_segment<OUT>(args, stg, row0, col, part_row, lane);
        } else {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<float4*>(stg + stg_off(lane, i)) =
                  make_float4(f[16 * g + 4 * i], f[16 * g + 4 * i + 1], f[16 * g + 4 * i + 2], f[16 * g + 4 * i + 3]);
            store_segment<OUT>(args, stg, row0, col + 16 * g, part_row, lane);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // no remote arrive or operand read targets a CTA that has left
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) tmem_dealloc_pair(tmem, TMEM_COLS);
    else tmem_dealloc(tmem, TMEM_COLS);
  }
}

__global__ void __launch_bounds__(128) scale_tiles_kernel(const TileJob t) {
  let_successor_start();
  make_tile_word(t, blockIdx.x, threadIdx.x);
}

// D = sum over the parts of K, in part order (+ R): parts [splits, M, N] fp32.
__global__ void __launch_bounds__(256) join_parts_kernel(const float* __restrict__ parts, int splits, int M, int N, void* D,
                                                         long ldd, const __nv_bfloat16* R, long ldr, int out) {
  wait_for_predecessor();
  const long i = (long)blockIdx.x * 256 + threadIdx.x, mn = (long)M * N;
  if (i >= mn) return;
  const long row = i / N, col = i - row * N;
  float s = 0.f;
#pragma unroll 8
  for (int p = 0; p < splits; ++p) s += parts[p * mn + i];
  if (out == OUT_BF16) {
    if (R != nullptr) s += __bfloat162float(R[row * ldr + col]);
    reinterpret_cast<__nv_bfloat16*>(D)[row * ldd + col] = __float2bfloat16_rn(s);
  } else {
    float* d = reinterpret_cast<float*>(D) + row * ldd + col;
    *d = out == OUT_ACC_F32 ? *d + s : s;
  }
}

// Codes whose rows do not start on 16 bytes -> rows padded to 16 bytes (zeros behind the codes).  A thread
// makes 16 bytes from the five 4-byte words that hold them; no word that begins past the row's end is read.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint8_t* __restrict__ q, long ld, int rows, int K,
                                                       uint4* __restrict__ out) {
  const int per = (K + 15) >> 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)rows * per) return;
  const long row = i / per;
  const int k = (int)(i - row * per) * 16;
  const uintptr_t p = reinterpret_cast<uintptr_t>(q + row * ld + k), end = reinterpret_cast<uintptr_t>(q + row * ld + K);
  const uint32_t sel = 0x3210u + 0x1111u * (uint32_t)(p & 3);
  uint32_t u[5], w[4];
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const uintptr_t a = (p & ~uintptr_t(3)) + 4 * j;
    u[j] = a < end && (j < 4 || (p & 3)) ? __ldg(reinterpret_cast<const uint32_t*>(a)) : 0u;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int left = K - (k + 4 * j);
    w[j] = __byte_perm(u[j], u[j + 1], sel);
    w[j] = left >= 4 ? w[j] : left <= 0 ? 0u : w[j] & (0xffffffffu >> (32 - 8 * left));
  }
  out[i] = make_uint4(w[0], w[1], w[2], w[3]);
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

static CUtensorMap make_map(CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base, long inner, long rows,
                            long pitch, int box_inner, int box_rows) {
  static thread_local bool bound = false;
  if (!bound) {  // the driver call needs a current context on this thread (autograd's workers)
    DTB_CUDA(cudaFree(nullptr));
    bound = true;
  }
  CUtensorMap m;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_fn()(&m, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  DTB_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d): inner=%ld rows=%ld pitch=%ld base=%p", (int)r, inner, rows, pitch, base);
  return m;
}
// codes: boxes of `box_rows` rows x 128 bytes; bytes past the matrix read as zero
static CUtensorMap code_map(const torch::Tensor& t, int box_rows) {
  const long rows = t.size(0), k = t.size(1);
  return make_map(CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, t.data_ptr(), k, rows,
                  rows > 1 ? t.stride(0) : (k + 15) / 16 * 16, 128, box_rows);
}
// scale tiles [row blocks, k blocks / 4, 512 bytes]: one tile per box
static CUtensorMap tile_map(const torch::Tensor& t) {
  return make_map(CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE, t.data_ptr(), 128, t.size(0) * t.size(1),
                  512, 128, 1);
}

template <int BN, bool PAIR, int OUT>
static void launch(const CUtensorMap* t, GemmArgs& g, cudaStream_t st) {
  using L = Smem<BN, PAIR>;
  constexpr int CTAS = PAIR ? 2 : 1;
  auto kern = fp8_gemm_kernel<BN, PAIR, OUT>;
  static bool configured[64] = {false};
  int dev = 0;
  DTB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    DTB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
    if (dev < 64) configured[dev] = true;
  }
  g.m_blocks = (g.M + CTAS * BM - 1) / (CTAS * BM);
  g.n_blocks = (g.N + BN - 1) / BN;
  g.num_tiles = g.m_blocks * g.n_blocks;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(CTAS * std::min(g.num_tiles * g.splits, device_sm_count() / CTAS), 1, 1);
  cfg.blockDim = dim3(320, 1, 1);
  cfg.dynamicSmemBytes = L::TOTAL;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  DTB_CUDA(cudaLaunchKernelEx(&cfg, kern, t[0], t[1], t[2], t[3], g));
}

}  // namespace fp8
}  // namespace dtb

using namespace dtb;

// D [M, N] = A [M, K] B [N, K]^T (+ R): D bf16 (R bf16, optional) or fp32 (accumulate: D += the product).
// tA, tB: the operands' scale tiles, uint8 [ceil(rows / 128), ceil(K / 512), 512].
void fp8_gemm(torch::Tensor A, torch::Tensor tA, torch::Tensor B, torch::Tensor tB, torch::Tensor D,
              c10::optional<torch::Tensor> R, bool accumulate) {
  for (const torch::Tensor* t : {&A, &B})
    DTB_CHECK(t->is_cuda() && t->device() == A.device() && t->scalar_type() == at::kFloat8_e4m3fn && t->dim() == 2 && (t->numel() == 0 || ((t->size(1) == 1 || t->stride(1) == 1) && (t->size(0) == 1 || t->stride(0) % 16 == 0) && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0)), "fp8_gemm: operands must be 2-D e4m3 on one GPU, rows contiguous and starting on 16-byte boundaries");
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
  const torch::Tensor* q[2] = {&A, &B};
  const torch::Tensor* t[2] = {&tA, &tB};
  for (int i = 0; i < 2; ++i)
    DTB_CHECK(t[i]->device() == A.device() && t[i]->scalar_type() == at::kByte && t[i]->is_contiguous() && t[i]->dim() == 3 && t[i]->size(0) == (q[i]->size(0) + 127) / 128 && t[i]->size(1) == (K + 511) / 512 && t[i]->size(2) == 512 && t[i]->size(0) * t[i]->size(1) < (1L << 31) && (reinterpret_cast<uintptr_t>(t[i]->data_ptr()) & 15) == 0, "fp8_gemm: scale tiles must be contiguous uint8 [ceil(rows / 128), ceil(K / 512), 512]");
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
  g.k_quads = (g.K + 511) / 512;
  g.k_iters = (g.K + fp8::BK - 1) / fp8::BK;
  auto st = at::cuda::getCurrentCUDAStream();
  // Few tokens: A's box holds only as many rows (a stage's 256 rows of 128 bytes would take the copy engine
  // longer than the weights' bytes take to arrive).  The tile's other rows keep whatever the shared memory
  // holds; a row of A reaches only its own row of the result, and those are not stored.
  const int a_rows = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  g.a_bytes = a_rows * fp8::BK;
  const CUtensorMap maps[4] = {fp8::code_map(A, a_rows), fp8::code_map(B, 128), fp8::tile_map(tA), fp8::tile_map(tB)};
  // Which kernel, and K in how many parts: the least modelled time.  A 128-deep stage takes about 500 cycles on a
  // single CTA (128 x 128 tile) and 700 on a pair (256 x 256) when nothing else holds it up; a unit of work
  // costs two stages more for its start and end, and parts of K, whose fp32 sums a second kernel adds in
  // order, about 11 stages more and their bytes (100 cycles for 275 kB).  Parts fill the SMs where tiles are few (a few tokens against the weights).
  // 48 x 4096 x 11008: one part 28 us, several and their join 16; 1 x 22016 x 4096: pairs 30 us, single CTAs
  // in four parts 20 and the join 3.
  const int sms = device_sm_count();
  const long tiles = ((M + 127) / 128) * ((N + 127) / 128), tiles2 = ((M + 255) / 256) * ((N + 255) / 256);
  auto cost = [&](long splits, long k_per) { return (tiles * splits + sms - 1) / sms * (k_per + 2) * 5 + (splits > 1 ? 55 + splits * M * N * 8 / 275000 : 0); };
  const long pair_cost = (tiles2 + sms / 2 - 1) / (sms / 2) * (g.k_iters + 2) * 7;
  long best = cost(1, g.k_iters);
  g.splits = 1;
  g.k_per = g.k_iters;
  for (int k_per = fp8::SF_STEP; k_per < g.k_iters; k_per += fp8::SF_STEP) {
    const long splits = (g.k_iters + k_per - 1) / k_per;
    if (splits * M * N * 4 <= (64L << 20) && cost(splits, k_per) < best) {
      best = cost(splits, k_per);
      g.splits = (int)splits;
      g.k_per = k_per;
    }
  }
  const bool pair = pair_cost < best;
  if (pair) {
    g.splits = 1;
    g.k_per = g.k_iters;
  }
  const int out = D.scalar_type() == at::kBFloat16 ? fp8::OUT_BF16 : accumulate ? fp8::OUT_ACC_F32 : fp8::OUT_F32;
  if (g.splits > 1) {
    auto parts = torch::empty({g.splits, M, N}, D.options().dtype(at::kFloat));
    fp8::GemmArgs p = g;
    p.D = parts.data_ptr();
    p.ldd = N;
    p.R = nullptr;
    p.vec = N % 4 == 0;
    fp8::launch<128, false, fp8::OUT_F32>(maps, p, st);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((M * N + 255) / 256), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    DTB_CUDA(cudaLaunchKernelEx(&cfg, fp8::join_parts_kernel, (const float*)parts.data_ptr<float>(), g.splits, g.M, g.N, g.D, g.ldd, g.R, g.ldr, out));
    return;
  }
  if (out == fp8::OUT_BF16) pair ? fp8::launch<256, true, fp8::OUT_BF16>(maps, g, st) : fp8::launch<128, false, fp8::OUT_BF16>(maps, g, st);
  else if (out == fp8::OUT_F32) pair ? fp8::launch<256, true, fp8::OUT_F32>(maps, g, st) : fp8::launch<128, false, fp8::OUT_F32>(maps, g, st);
  else pair ? fp8::launch<256, true, fp8::OUT_ACC_F32>(maps, g, st) : fp8::launch<128, false, fp8::OUT_ACC_F32>(maps, g, st);
}

// The scale tiles of plain scales: e8m0 [ceil(rows / gran), k blocks], gran 1 or 128.
torch::Tensor fp8_scale_tiles(torch::Tensor s, int64_t gran, int64_t rows) {
  DTB_CHECK(s.is_cuda() && s.scalar_type() == at::kFloat8_e8m0fnu && s.dim() == 2 && (gran == 1 || gran == 128) && rows >= 0 && rows < (1L << 30) && s.size(0) == (rows + gran - 1) / gran, "fp8_scale_tiles: e8m0 scales of 1 x 128 or 128 x 128 blocks");
  const c10::cuda::CUDAGuard guard(s.device());
  const long mt = (rows + 127) / 128, kb = s.size(1), kq = (kb + fp8::SF_STEP - 1) / fp8::SF_STEP;
  DTB_CHECK(mt * kq < (1L << 31), "fp8_scale_tiles: too large");
  auto t = torch::empty({mt, kq, 512}, s.options().dtype(at::kByte));
  if (mt * kq == 0) return t;
  const fp8::TileJob job{reinterpret_cast<const uint8_t*>(s.data_ptr()), s.stride(0), s.stride(1), (int)gran, (int)rows,
                         (int)kb, (int)kq, reinterpret_cast<uint32_t*>(t.data_ptr()), (int)(mt * kq)};
  fp8::scale_tiles_kernel<<<(unsigned)job.count, 128, 0, at::cuda::getCurrentCUDAStream()>>>(job);
  DTB_LAUNCH_CHECK();
  return t;
}

// The codes with rows on 16-byte boundaries: a padded copy where they are not.
static torch::Tensor fp8_aligned(torch::Tensor q) {
  if (q.numel() == 0 || ((reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0 && (q.size(1) == 1 || q.stride(1) == 1) &&
                         (q.size(0) == 1 || q.stride(0) % 16 == 0)))
    return q;
  if (q.size(1) > 1 && q.stride(1) != 1) q = q.contiguous();
  const long rows = q.size(0), K = q.size(1), per = (K + 15) / 16;
  DTB_CHECK(rows < (1L << 30) && K < (1L << 30) && (rows * per + 255) / 256 < (1L << 31), "fp8_product: too large");
  auto pad = torch::empty({rows, per * 16}, q.options());
  fp8::pad_rows_kernel<<<(unsigned)((rows * per + 255) / 256), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      reinterpret_cast<const uint8_t*>(q.data_ptr()), rows > 1 ? q.stride(0) : K, (int)rows, (int)K,
      reinterpret_cast<uint4*>(pad.data_ptr()));
  DTB_LAUNCH_CHECK();
  return pad.narrow(1, 0, K);
}

void fp8_check_blocks(const torch::Tensor& q, const torch::Tensor& s);

// fp8_gemm for operands as a user holds them: codes in rows of any alignment, plain scales, scale tiles or none.
void fp8_product(torch::Tensor A, torch::Tensor sA, c10::optional<torch::Tensor> tA, torch::Tensor B, torch::Tensor sB,
                 c10::optional<torch::Tensor> tB, torch::Tensor D, c10::optional<torch::Tensor> R, bool accumulate) {
  for (const torch::Tensor* t : {&A, &B})
    DTB_CHECK(t->is_cuda() && t->scalar_type() == at::kFloat8_e4m3fn && t->dim() == 2, "fp8_product: operands must be 2-D e4m3 on the GPU");
  fp8_check_blocks(A, sA);
  fp8_check_blocks(B, sB);
  const c10::cuda::CUDAGuard guard(A.device());
  auto tiles = [](const torch::Tensor& q, const torch::Tensor& s, const c10::optional<torch::Tensor>& t) {
    return t.has_value() ? *t : fp8_scale_tiles(s, s.size(0) == (q.size(0) + 127) / 128 ? 128 : 1, q.size(0));
  };
  fp8_gemm(fp8_aligned(A), tiles(A, sA, tA), fp8_aligned(B), tiles(B, sB, tB), D, R, accumulate);
}
