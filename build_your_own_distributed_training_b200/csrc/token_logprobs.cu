// Log probabilities of given tokens with the distribution's entropy and its top alternatives, and
// the gradient with respect to the logits (sm_100a).
//
// Per row x of V logits, temperature T, m = max x, z = (x - m) / T, S = sum exp z:
//
//   logprob = z_tok - ln S,   entropy = ln S - (sum exp(z) z) / S,
//   top k:   the k largest x, ties to the lowest index, with their log probabilities;
//   dx_i = (g_lp ([i = tok] - p_i) - g_H p_i (ln p_i + entropy)) / T,   p = exp(z) / S.
//
// Forward: one read of the logits.  Every thread keeps a running (m, S, A = sum exp(z) z) of its
// 16-byte vectors, rescaled when its maximum grows; the triples are merged over the block and, when
// rows are few, over a cluster of up to 8 blocks that share a row through distributed shared memory.
// The backward reads the logits once more and writes the gradient; it needs only (m, log2 S, entropy)
// of the row.  Exponentials are taken in base 2 with (x - m) formed first, so that masks of the
// type's lowest value cannot overflow, and exponents are held at -256 or above, where 2^t is zero:
// an excluded logit (-inf) then adds exactly nothing to S and A.
//
// 4096 x 32000 fp32 without alternatives: forward 86 us (6.1 TB/s, memory), backward 144 us.  777 x 32003 bf16
// with 5 alternatives: 35 and 21 us.  A thread of the 512 sees 8 vectors of such a row, so the forward's merges
// weigh as much as the elements (53% of the issue slots, warps wait at barriers most); the backward uses 67%
// of the slots, one element at a time.  One row of 128256 fp32 with 20 alternatives: 11 us in a cluster of 8, all latency.
//
// Top k (k <= 32) without sorting the row: the k largest thread maxima name the k threads that can
// own one of the k largest elements, and the k-th of these maxima is a lower bound for all of them;
// the warps read those threads' vectors again (a few per owner, from L2) and keep sorted lists of 32
// in registers.  Elements are compared as 64-bit keys (value, then lower index first), so there are
// no ties and the work is bounded for any row.
//
// Rows: an ignored token gives 0, 0 and no gradient; a row with no logit above -inf gives -inf and
// entropy 0 and no gradient; NaN or +inf in a row gives NaN; a token outside [0, V) gives NaN and
// sets the device error word.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "vecio.cuh"

namespace dtb {
namespace lp {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMinExp = -256.f;  // 2^-256 is zero in fp32
constexpr int MAX_TOP = 32;

// row state for the backward: (m, log2 S, entropy, kind)
enum : int { ROW_OK = 0, ROW_ZERO = 1, ROW_NAN = 2 };

struct Acc {
  float m, s, a;  // a: sum of 2^t t, t in base-2 units
};

__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

__device__ __forceinline__ Acc merge(const Acc& p, const Acc& q, float c) {
  Acc r;
  r.m = max_nan(p.m, q.m);
  const float dp = fmaxf((p.m - r.m) * c, kMinExp), dq = fmaxf((q.m - r.m) * c, kMinExp);
  const float fp = ex2_approx(dp), fq = ex2_approx(dq);
  r.s = p.s * fp + q.s * fq;
  r.a = fp * fmaf(dp, p.s, p.a) + fq * fmaf(dq, q.s, q.a);
  return r;
}

// unsigned order of floats; larger key = larger value, then lower index
__device__ __forceinline__ unsigned long long make_key(float v, uint32_t idx) {
  uint32_t u = __float_as_uint(v);
  if (u == 0x80000000u) u = 0;  // -0 ties with +0
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) { return ~(uint32_t)k; }

__device__ __forceinline__ unsigned long long exchange(unsigned long long k, int j, bool keep_max) {
  const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, j);
  return (o > k) == keep_max ? o : k;
}
// the warp's 32 keys, largest in lane 0
__device__ __forceinline__ unsigned long long warp_sort(unsigned long long k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int j = size >> 1; j > 0; j >>= 1) k = exchange(k, j, ((lane & j) == 0) == ((lane & size) == 0));
  return k;
}
// largest 32 of two sorted lists; `rev` is the second one from its end (lane l holds element 31 - l)
__device__ __forceinline__ unsigned long long warp_merge(unsigned long long k, unsigned long long rev, int lane) {
  k = rev > k ? rev : k;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) k = exchange(k, j, (lane & j) == 0);
  return k;
}

// (x0 - m) c and (x1 - m) c, at least kMinExp
__device__ __forceinline__ f2 exponents(float x0, float x1, f2 neg_m, f2 c) {
  float a, b;
  unpair(mul2(add2(pair(x0, x1), neg_m), c), a, b);
  return pair(fmaxf(a, kMinExp), fmaxf(b, kMinExp));
}

// largest element of a vector, NaN if one is
template <typename T>
__device__ __forceinline__ float vec_max(const Pack<T, 16 / sizeof(T)>& p) {
  if constexpr (sizeof(T) == 4) {
    return max_nan(max_nan(p.at(0), p.at(1)), max_nan(p.at(2), p.at(3)));
  } else {
    const uint4& w = p.w[0];
    uint32_t a, b;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
      asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    } else {
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(w.x), "r"(w.y));
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(b) : "r"(w.z), "r"(w.w));
      asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    }
    Pack<T, 2> q;
    q.e[0] = reinterpret_cast<const T*>(&a)[0];
    q.e[1] = reinterpret_cast<const T*>(&a)[1];
    return max_nan(q.at(0), q.at(1));
  }
}

struct FwdArgs {
  const void* x;
  long ld;
  const int64_t* tokens;
  long ignore;
  int V;
  float invT;
  int top_k;
  float* logprob;
  float* entropy;
  float* top_v;      // [M, k]
  int64_t* top_i;    // [M, k]
  float4* state;     // [M], or null when nothing will ask for the gradient
  int* err;
};

template <int NW>
struct Shared {
  unsigned long long list[NW][32];
  unsigned long long owner[32];
  Acc acc[NW];
  Acc block;
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long ld_cluster_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// vector j of a row whose first element is element `shift` of its first 16-byte word
template <typename T>
__device__ __forceinline__ void load_vec(Pack<T, 16 / sizeof(T)>& p, const T* row, int j, int shift, int V) {
  constexpr int VEC = 16 / sizeof(T);
  const int e0 = j * VEC - shift;
  if (e0 >= 0 && e0 + VEC <= V) {
    p.load(row + e0);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.e[e] = (e0 + e >= 0 && e0 + e < V) ? row[e0 + e] : from_float<T>(-INFINITY);
  }
}

template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT) logprob_fwd_kernel(const FwdArgs a, int csize) {
  constexpr int VEC = 16 / sizeof(T), NW = NT / 32, U = 4;
  __shared__ Shared<NW> sh;
  const int rank = csize > 1 ? (int)cluster_ctarank() : 0;
  const long row = blockIdx.x / csize;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long tok = a.tokens[row];
  if (tok == a.ignore) {  // the same for the whole cluster
    if (rank == 0) {
      if (tid == 0) {
        a.logprob[row] = 0.f;
        a.entropy[row] = 0.f;
        if (a.state) a.state[row] = make_float4(0.f, 0.f, 0.f, __int_as_float(ROW_ZERO));
      }
      if (TOP && tid < a.top_k) {
        a.top_v[row * a.top_k + tid] = -INFINITY;
        a.top_i[row * a.top_k + tid] = -1;
      }
    }
    return;
  }
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int nvec = (shift + a.V + VEC - 1) / VEC;
  const int G = csize * NT, g = rank * NT + tid;
  const float c = a.invT * kLog2e;

  float m = -INFINITY;
  f2 s2 = pair(0.f, 0.f), a2 = s2;
  const f2 c2 = pair(c, c);
  float best = -INFINITY;
  int best_i = -1;
  for (int j = g; j < nvec; j += U * G) {
    Pack<T, VEC> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u * G < nvec) {
        load_vec<T>(p[u], x, j + u * G, shift, a.V);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[u].set(e, -INFINITY);
      }
    }
    float cm = vec_max<T>(p[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) cm = max_nan(cm, vec_max<T>(p[u]));
    if (TOP && (cm > best || best_i < 0)) {
      best = cm;
#pragma unroll
      for (int u = U - 1; u >= 0; --u)
#pragma unroll
        for (int e = VEC - 1; e >= 0; --e) {
          const int idx = (j + u * G) * VEC + e - shift;
          if (p[u].at(e) == cm && idx >= 0 && idx < a.V) best_i = idx;
        }
    }
    const float mn = max_nan(m, cm);
    if (mn != m) {
      const float d = fmaxf((m - mn) * c, kMinExp), f = ex2_approx(d);
      const f2 f2v = pair(f, f);
      a2 = mul2(f2v, fma2(pair(d, d), s2, a2));
      s2 = mul2(f2v, s2);
      m = mn;
    }
    const f2 neg_m = pair(-mn, -mn);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const f2 t = exponents(p[u].at(e), p[u].at(e + 1), neg_m, c2);
        float t0, t1;
        unpair(t, t0, t1);
        const f2 w = pair(ex2_approx(t0), ex2_approx(t1));
        s2 = add2(s2, w);
        a2 = fma2(w, t, a2);
      }
  }
  Acc acc;
  acc.m = m;
  {
    float x0, x1;
    unpair(s2, x0, x1);
    acc.s = x0 + x1;
    unpair(a2, x0, x1);
    acc.a = x0 + x1;
  }
  // threads -> warp -> block -> cluster, in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Acc q{__shfl_xor_sync(0xffffffffu, acc.m, o), __shfl_xor_sync(0xffffffffu, acc.s, o),
          __shfl_xor_sync(0xffffffffu, acc.a, o)};
    acc = merge(acc, q, c);
  }
  if (lane == 0) sh.acc[warp] = acc;

  unsigned long long list = 0;
  if constexpr (TOP) {
    // the block's 32 largest thread maxima
    list = warp_sort(best_i >= 0 ? make_key(best, (uint32_t)best_i) : 0ull, lane);
    sh.list[warp][lane] = list;
#pragma unroll
    for (int s = 1; s < NW; s <<= 1) {
      __syncthreads();
      if (warp % (2 * s) == 0) {
        list = warp_merge(list, sh.list[warp + s][31 - lane], lane);
        sh.list[warp][lane] = list;
      }
    }
    if (warp == 0) sh.owner[lane] = list;
    __syncthreads();
    // every element that can be among the k largest: vectors of the k owners, keys from the k-th on
    const unsigned long long least = sh.owner[a.top_k - 1];
    list = 0;
    for (int o = warp; o < a.top_k; o += NW) {
      const unsigned long long ok = sh.owner[o];
      if (ok == 0) break;  // sorted: no more owners
      const int first = ((int)key_index(ok) + shift) / VEC % G;
      for (int i0 = 0; first + (long)i0 * G < nvec; i0 += 32) {
        const long j = first + (long)(i0 + lane) * G;
        Pack<T, VEC> p;
        const bool in = j < nvec;
        if (in) load_vec<T>(p, x, (int)j, shift, a.V);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int idx = in ? (int)j * VEC + e - shift : -1;
          unsigned long long k = idx >= 0 && idx < a.V ? make_key(p.at(e), (uint32_t)idx) : 0ull;
          if (k < least) k = 0;
          if (__ballot_sync(0xffffffffu, k != 0)) {
            k = warp_sort(k, lane);
            list = warp_merge(list, __shfl_sync(0xffffffffu, k, 31 - lane), lane);
          }
        }
      }
    }
    sh.list[warp][lane] = list;
#pragma unroll
    for (int s = 1; s < NW; s <<= 1) {
      __syncthreads();
      if (warp % (2 * s) == 0) {
        list = warp_merge(list, sh.list[warp + s][31 - lane], lane);
        sh.list[warp][lane] = list;
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    Acc q = lane < NW ? sh.acc[lane] : Acc{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = NW >> 1; o > 0; o >>= 1) {
      Acc r{__shfl_xor_sync(0xffffffffu, q.m, o), __shfl_xor_sync(0xffffffffu, q.s, o),
            __shfl_xor_sync(0xffffffffu, q.a, o)};
      q = merge(q, r, c);
    }
    acc = q;
    if (lane == 0) sh.block = q;
  }
  if (csize > 1) cluster_sync();
  if (rank == 0 && warp == 0) {
    acc.m = __shfl_sync(0xffffffffu, acc.m, 0);
    acc.s = __shfl_sync(0xffffffffu, acc.s, 0);
    acc.a = __shfl_sync(0xffffffffu, acc.a, 0);
    for (int r = 1; r < csize; ++r) {
      const uint32_t b = mapa_shared(smem_u32(&sh.block), r);
      Acc q{__uint_as_float(ld_cluster_u32(b)), __uint_as_float(ld_cluster_u32(b + 4)),
            __uint_as_float(ld_cluster_u32(b + 8))};
      acc = merge(acc, q, c);
      if constexpr (TOP) list = warp_merge(list, ld_cluster_u64(mapa_shared(smem_u32(&sh.list[0][31 - lane]), r)), lane);
    }
    const bool in_range = tok >= 0 && tok < a.V;
    if (!in_range && lane == 0) atomicExch(a.err, ERR_BAD_ARG);
    const bool empty = acc.m == -INFINITY;
    const bool bad = !in_range || acc.m != acc.m || acc.m == INFINITY;
    const float nan = __int_as_float(0x7fc00000);
    const float ln_s = logf(acc.s);
    if (lane == 0) {
      const float xt = in_range ? as_float<T>(x[tok]) : 0.f;
      const float ent = ln_s - acc.a / acc.s / kLog2e;
      a.logprob[row] = bad ? nan : empty ? -INFINITY : (xt - acc.m) * a.invT - ln_s;
      a.entropy[row] = bad ? nan : empty ? 0.f : ent;
      if (a.state) a.state[row] = make_float4(acc.m, log2f(acc.s), ent, __int_as_float(bad ? ROW_NAN : empty ? ROW_ZERO : ROW_OK));
    }
    if (TOP && lane < a.top_k) {
      a.top_v[row * a.top_k + lane] = bad ? nan : empty ? -INFINITY : (key_value(list) - acc.m) * a.invT - ln_s;
      a.top_i[row * a.top_k + lane] = bad ? -1 : (int64_t)key_index(list);
    }
  }
  if (csize > 1) cluster_sync();  // the other blocks' shared memory stays until rank 0 has read it
}

struct BwdArgs {
  const void* x;
  long ld;
  void* dx;
  long ldd;
  const int64_t* tokens;
  const float4* state;
  const float* g_lp;   // [M] or null
  const float* g_ent;  // [M] or null
  int V;
  int split;           // blocks per row
  float invT;
};

// WIDE: the row of x and the row of dx sit alike within their vectors
template <typename T, typename TO, bool WIDE>
__global__ void __launch_bounds__(256) logprob_bwd_kernel(const BwdArgs a) {
  constexpr int VEC = WIDE ? 16 / sizeof(T) : 1, U = 4;
  const long row = blockIdx.x / a.split;
  const int part = (int)(blockIdx.x % a.split);
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ld;
  TO* dx = reinterpret_cast<TO*>(a.dx) + row * a.ldd;
  const float4 st = a.state[row];
  const int kind = __float_as_int(st.w);
  const int shift = WIDE ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
  const int nvec = (shift + a.V + VEC - 1) / VEC;
  const float gl = a.g_lp ? a.g_lp[row] * a.invT : 0.f, ge = a.g_ent ? a.g_ent[row] * a.invT : 0.f;
  const float c = a.invT * kLog2e, m = st.x, l2s = st.y, ent = st.z;
  const long tok = a.tokens[row];
  // d = p (g0 + g1 log2 p) + [i = tok] gl
  const float g0 = -fmaf(ge, ent, gl), g1 = -ge / kLog2e;
  const int first = part * 256 + threadIdx.x, step = a.split * 256;
  for (int j0 = first; j0 < nvec; j0 += U * step) {
    Pack<T, VEC> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * step;
      if (kind == ROW_OK && j < nvec) {
        if constexpr (WIDE) load_vec<T>(p[u], x, j, shift, a.V);
        else p[u].load(x + j);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * step, e0 = j * VEC - shift;
      if (j >= nvec) break;
      Pack<TO, VEC> o;
      if (kind == ROW_OK) {
        float d[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float t = fmaxf((p[u].at(e) - m) * c, kMinExp) - l2s;  // log2 p
          d[e] = ex2_approx(t) * fmaf(g1, t, g0);
        }
        if (tok >= e0 && tok < e0 + VEC) {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (e0 + e == tok) d[e] += gl;
        }
        o.set_all(d);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.set(e, kind == ROW_ZERO ? 0.f : __int_as_float(0x7fc00000));
      }
      if (e0 >= 0 && e0 + VEC <= a.V) {
        o.store(dx + e0);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (e0 + e >= 0 && e0 + e < a.V) dx[e0 + e] = o.e[e];
      }
    }
  }
}

template <typename T, int NT>
void launch_fwd(const FwdArgs& a, long M, int csize, bool top, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(M * csize), 1, 1);
  cfg.blockDim = dim3(NT, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = csize > 1 ? 1 : 0;
  if (top) DTB_CUDA(cudaLaunchKernelEx(&cfg, logprob_fwd_kernel<T, NT, true>, a, csize));
  else DTB_CUDA(cudaLaunchKernelEx(&cfg, logprob_fwd_kernel<T, NT, false>, a, csize));
}

}  // namespace lp
}  // namespace dtb

using namespace dtb;

static void lp_check_logits(const char* op, const torch::Tensor& x, const torch::Tensor& tokens, double temperature) {
  DTB_CHECK(x.is_cuda() && x.dim() == 2 && is_float_type(x.scalar_type()) && x.size(1) > 0 && x.size(1) < (1L << 30) && (x.numel() == 0 || x.size(1) == 1 || x.stride(1) == 1), "%s: logits must be a 2-D CUDA tensor of fp32, bf16 or fp16 with contiguous columns", op);
  DTB_CHECK(tokens.device() == x.device() && tokens.scalar_type() == at::kLong && tokens.is_contiguous() && tokens.numel() == x.size(0), "%s: tokens must be contiguous int64, one per row, on the logits' device", op);
  DTB_CHECK(temperature >= 0x1p-126 && temperature <= 0x1p126, "%s: temperature must lie in [2^-126, 2^126]", op);
}

// x [M, V], tokens of any shape with M entries -> {logprob, entropy} of the tokens' shape, then {top log
// probabilities, top tokens} of that shape and k when top_k > 0, then the backward's state [M, 4] if asked for.
std::vector<torch::Tensor> token_logprobs_fwd(torch::Tensor x, torch::Tensor tokens, double temperature, int64_t top_k,
                                              int64_t ignore, bool want_state) {
  lp_check_logits("token_log_probs", x, tokens, temperature);
  DTB_CHECK(top_k >= 0 && top_k <= lp::MAX_TOP && top_k <= x.size(1), "token_log_probs: top_k must lie in [0, %d] and not exceed the vocabulary", lp::MAX_TOP);
  const c10::cuda::CUDAGuard guard(x.device());
  const long M = x.size(0);
  auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
  std::vector<torch::Tensor> r;
  r.push_back(torch::empty(tokens.sizes(), f32));
  r.push_back(torch::empty(tokens.sizes(), f32));
  if (top_k > 0) {
    auto shape = tokens.sizes().vec();
    shape.push_back(top_k);
    r.push_back(torch::empty(shape, f32));
    r.push_back(torch::empty(shape, tokens.options()));
  }
  if (want_state) r.push_back(torch::empty({M, 4}, f32));
  if (M == 0) return r;
  lp::FwdArgs a{};
  a.x = x.data_ptr();
  a.ld = x.stride(0);
  a.tokens = tokens.data_ptr<int64_t>();
  a.ignore = ignore;
  a.V = (int)x.size(1);
  a.invT = (float)(1.0 / temperature);
  a.top_k = (int)top_k;
  a.logprob = r[0].data_ptr<float>();
  a.entropy = r[1].data_ptr<float>();
  if (top_k > 0) {
    a.top_v = r[2].data_ptr<float>();
    a.top_i = r[3].data_ptr<int64_t>();
  }
  if (want_state) a.state = reinterpret_cast<float4*>(r.back().data_ptr<float>());
  a.err = dtb_error_word();
  // One block of 512 threads per row; short rows take 128.  When the rows do not fill the machine a
  // cluster of blocks shares each row, as long as every block keeps a few vectors per thread.
  const long vecs = (long)a.V * (long)x.element_size() / 16 + 1;
  const bool small = vecs <= 1024;
  int csize = 1;
  if (!small)
    while (csize < 8 && M * csize * 2 <= 2L * device_sm_count() && vecs / (csize * 2) >= 1024) csize *= 2;
  DTB_CHECK(M * csize < (1L << 31), "token_log_probs: too many rows");
  auto st = at::cuda::getCurrentCUDAStream();
  DTB_FLOAT_TYPES(x.scalar_type(), {
    if (small) lp::launch_fwd<T, 128>(a, M, 1, top_k > 0, st);
    else lp::launch_fwd<T, 512>(a, M, csize, top_k > 0, st);
  });
  DTB_LAUNCH_CHECK();
  return r;
}

// Gradient of the logits into dx ([M, V], the logits' type or bf16, contiguous columns).
void token_logprobs_bwd(torch::Tensor x, torch::Tensor tokens, torch::Tensor state, c10::optional<torch::Tensor> g_lp,
                        c10::optional<torch::Tensor> g_ent, double temperature, torch::Tensor dx) {
  lp_check_logits("token_log_probs backward", x, tokens, temperature);
  const c10::cuda::CUDAGuard guard(x.device());
  const long M = x.size(0);
  DTB_CHECK(state.device() == x.device() && state.scalar_type() == at::kFloat && state.is_contiguous() && state.numel() == 4 * M, "token_log_probs backward: state must be the forward's");
  for (const auto* g : {&g_lp, &g_ent})
    if (g->has_value())
      DTB_CHECK((*g)->device() == x.device() && (*g)->scalar_type() == at::kFloat && (*g)->is_contiguous() && (*g)->numel() == M, "token_log_probs backward: gradients must be contiguous fp32, one per row");
  DTB_CHECK(dx.device() == x.device() && dx.sizes() == x.sizes() && (dx.numel() == 0 || dx.size(1) == 1 || dx.stride(1) == 1) && (dx.scalar_type() == x.scalar_type() || (x.scalar_type() == at::kFloat && dx.scalar_type() == at::kBFloat16)), "token_log_probs backward: dlogits must have the logits' shape and type (or bf16) and contiguous columns");
  if (M == 0) return;
  lp::BwdArgs a{};
  a.x = x.data_ptr();
  a.ld = x.stride(0);
  a.dx = dx.data_ptr();
  a.ldd = dx.stride(0);
  a.tokens = tokens.data_ptr<int64_t>();
  a.state = reinterpret_cast<const float4*>(state.data_ptr<float>());
  a.g_lp = g_lp.has_value() ? g_lp->data_ptr<float>() : nullptr;
  a.g_ent = g_ent.has_value() ? g_ent->data_ptr<float>() : nullptr;
  a.V = (int)x.size(1);
  a.invT = (float)(1.0 / temperature);
  const long es = (long)x.element_size(), eo = (long)dx.element_size(), vec = 16 / es;
  // rows start alike within their vectors when base and row step do
  const long xs = (long)(reinterpret_cast<uintptr_t>(a.x) / es) % vec, ds = (long)(reinterpret_cast<uintptr_t>(a.dx) / eo) % vec;
  const bool wide = xs == ds && a.ld % vec == a.ldd % vec;
  // about 2048 vectors per block when rows are many, more blocks per row when they are few
  const long vecs = ((long)a.V + vec - 1) / vec;
  long split = std::max(1L, vecs / 2048);
  split = std::max(split, std::min((vecs + 255) / 256, (long)device_sm_count() * 8 / M));
  a.split = (int)std::max(1L, split);
  DTB_CHECK(M * a.split < (1L << 31), "token_log_probs backward: too many rows");
  auto st = at::cuda::getCurrentCUDAStream();
  const unsigned grid = (unsigned)(M * a.split);
  const bool to_bf16 = dx.scalar_type() != x.scalar_type();
  if (to_bf16) {
    if (wide) lp::logprob_bwd_kernel<float, __nv_bfloat16, true><<<grid, 256, 0, st>>>(a);
    else lp::logprob_bwd_kernel<float, __nv_bfloat16, false><<<grid, 256, 0, st>>>(a);
  } else DTB_FLOAT_TYPES(x.scalar_type(), {
    if (wide) lp::logprob_bwd_kernel<T, T, true><<<grid, 256, 0, st>>>(a);
    else lp::logprob_bwd_kernel<T, T, false><<<grid, 256, 0, st>>>(a);
  });
  DTB_LAUNCH_CHECK();
}
