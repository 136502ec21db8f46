// Per-head RMSNorm of queries and keys with the rotary rotation in the same pass (sm_100a).
//
// On the packed projection [q | k | v] of a token, for every query and key head x of hd elements:
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  u = n w          (w: one [hd] weight for q, one for k)
//   y_j = u_j c_j - u_{j+hd/2} s_j,  y_{j+hd/2} = u_{j+hd/2} c_j + u_j s_j      (j < hd/2)
//
// and v is carried over.  Backward, from g = dL/dy:  gu = R^T g,  dw = sum over tokens and heads of
// gu n,  dx = r (gu w - n mean(gu w n)),  dv = g.  r is recomputed from x, which the backward reads
// anyway, so nothing but the input is saved.
//
// Both directions are bound by memory.  A group of L lanes holds one head, each lane 4 elements of the
// first half and their partners of the second, so the rotation needs no exchange and the only cross-lane
// step is the L-lane sum.  (8 + 8 elements a lane filled the register file in the backward: 121 us for 8192
// tokens of 48 heads of 128.)  A warp stays on one token: its cos/sin row is read once and lives in
// registers while the token's heads stream through, several heads per lane group in flight; arithmetic goes
// two fp32 at a time.  8192 tokens of 32 + 8 + 8 heads of 128, bf16: forward 39 us (5.1 TB/s), backward
// 75 us (3.8 TB/s).  Both wait on latency: half the issue slots are used, and the registers of the heads in
// flight allow four blocks an SM forward (three took 44 us) and two backward (three with half the heads in
// flight spilled and took 105 us).  Statistics, rotation and
// weight gradients are fp32; y and dx are rounded once, to the storage type.
//
// dw: every warp adds up the heads of its tokens in registers, the block's warps are added in order
// and written as one partial per block, and qk_dw_reduce_kernel adds the partials in order: the same
// bits on every run.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "common.cuh"
#include "vecio.cuh"

namespace dtb {
namespace qk {

constexpr int NT = 256;  // threads per block

struct Args {
  const void* x;       // [tokens, ld]
  long ld;
  const void* g;       // backward: dL/dy [tokens, ldg]
  long ldg;
  void* out;           // y or dx, [tokens, ldo]
  long ldo;
  const void* wq;
  const void* wk;
  int wdt;             // storage type of the weights
  const float* cos_t;  // [table_rows, hd]; the first hd/2 columns are read
  const float* sin_t;
  const void* pos;     // [tokens] int64 / int32, or null: token % seqlen
  int pos64;
  long tokens, table_rows, seqlen;
  int nq, nkv, hd;
  int lanes;           // lanes per head, a power of two
  int split;           // warps that share a token's heads
  float eps;
  float* part;         // backward: [blocks, 2 hd]
  int* err;
};

__device__ __forceinline__ long position(const Args& a, long token) {
  if (a.pos == nullptr) return token % a.seqlen;
  return a.pos64 ? (long)reinterpret_cast<const int64_t*>(a.pos)[token]
                 : (long)reinterpret_cast<const int32_t*>(a.pos)[token];
}

// The lane's NP chunks of VEC pairs: chunk i starts at element (i * lanes + l) * VEC of either half.
template <int VEC, int NP>
struct Lane {
  int off[NP];
  bool on[NP];
  __device__ __forceinline__ Lane(int l, int lanes, int half) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      off[i] = (i * lanes + l) * VEC;
      on[i] = off[i] < half;
    }
  }
};

template <int VEC, int NP>
__device__ __forceinline__ void load_table(const Args& a, const Lane<VEC, NP>& ln, long token, float (&c)[NP][VEC],
                                           float (&s)[NP][VEC], int lane) {
  const long pos = position(a, token);
  const bool ok = pos >= 0 && pos < a.table_rows;
  if (!ok && lane == 0) atomicExch(a.err, ERR_BAD_ARG);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    Pack<float, VEC> pc, ps;
    if (ok && ln.on[i]) {
      pc.load(a.cos_t + pos * a.hd + ln.off[i]);
      ps.load(a.sin_t + pos * a.hd + ln.off[i]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      // a position outside the table gives NaN heads and sets the device error word
      c[i][v] = ok ? (ln.on[i] ? pc.at(v) : 0.f) : __int_as_float(0x7fc00000);
      s[i][v] = ok ? (ln.on[i] ? ps.at(v) : 0.f) : __int_as_float(0x7fc00000);
    }
  }
}

template <int VEC, int NP>
__device__ __forceinline__ void load_weight(const void* w, int wdt, const Lane<VEC, NP>& ln, int half,
                                            float (&lo)[NP][VEC], float (&hi)[NP][VEC]) {
  // a weight of the model's type is a few hundred bytes that stay in L1
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (wdt == DT_F32) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        lo[i][v] = ln.on[i] ? __ldg(reinterpret_cast<const float*>(w) + ln.off[i] + v) : 0.f;
        hi[i][v] = ln.on[i] ? __ldg(reinterpret_cast<const float*>(w) + ln.off[i] + half + v) : 0.f;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        lo[i][v] = ln.on[i] ? load_as(w, ln.off[i] + v, wdt) : 0.f;
        hi[i][v] = ln.on[i] ? load_as(w, ln.off[i] + half + v, wdt) : 0.f;
      }
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A token's heads come in three runs, [0, nq) queries, [nq, nq + nkv) keys and as many values; each run is
// walked by itself, so the weight of a run is one set of registers and nothing is selected per element.  A
// warp takes `per` heads of the run at a time, one per lane group, and every `split`-th such step; U steps
// are in flight.
enum : int { Q = 0, K = 1, V = 2 };

template <typename T, int VEC, int NP>
__device__ __forceinline__ void load_head(Pack<T, VEC> (&lo)[NP], Pack<T, VEC> (&hi)[NP], const T* p, int half,
                                          const Lane<VEC, NP>& ln, bool live) {
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (live && ln.on[i]) {
      lo[i].load(p + ln.off[i]);
      hi[i].load(p + half + ln.off[i]);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) lo[i].set(v, 0.f), hi[i].set(v, 0.f);
    }
}
template <typename T, int VEC, int NP>
__device__ __forceinline__ void store_head(const Pack<T, VEC> (&lo)[NP], const Pack<T, VEC> (&hi)[NP], T* p, int half,
                                           const Lane<VEC, NP>& ln, bool live) {
#pragma unroll
  for (int i = 0; i < NP; ++i)
    if (live && ln.on[i]) {
      lo[i].store(p + ln.off[i]);
      hi[i].store(p + half + ln.off[i]);
    }
}

// elements i and i + 1 of a lane's row as a pair (0 past its end)
template <int VEC>
__device__ __forceinline__ f2 two(const float (&v)[VEC], int i) { return pair(v[i], i + 1 < VEC ? v[i + 1] : 0.f); }
template <int VEC>
__device__ __forceinline__ void put(float (&v)[VEC], int i, f2 p) {
  float a, b;
  unpair(p, a, b);
  v[i] = a;
  if (i + 1 < VEC) v[i + 1] = b;
}
__device__ __forceinline__ float sum2(f2 p) {
  float a, b;
  unpair(p, a, b);
  return a + b;
}

// With the weight taken into the rotation's factors, y_lo = r (x_lo wl c - x_hi wh s) and
// y_hi = r (x_hi wh c + x_lo wl s).
template <int KIND, typename T, int VEC, int NP, int U>
__device__ __forceinline__ void fwd_run(const Args& a, const T* x, T* y, const Lane<VEC, NP>& ln, int grp, int part,
                                        const float (&c)[NP][VEC], const float (&s)[NP][VEC]) {
  const int half = a.hd >> 1, per = 32 / a.lanes, stride = per * a.split;
  const int first = KIND == Q ? 0 : KIND == K ? a.nq : a.nq + a.nkv, end = first + (KIND == Q ? a.nq : a.nkv);
  const float inv_hd = 1.f / (float)a.hd;
  constexpr int PAIRS = (VEC + 1) / 2;
  f2 lc[NP][PAIRS], ls[NP][PAIRS], hc[NP][PAIRS], hs[NP][PAIRS];  // wl c, wl s, wh c, -wh s
  if constexpr (KIND != V) {
    float wl[NP][VEC], wh[NP][VEC];
    load_weight(KIND == Q ? a.wq : a.wk, a.wdt, ln, half, wl, wh);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int v = 0; v < VEC; v += 2) {
        const f2 cc = two(c[i], v), ss = two(s[i], v), l = two(wl[i], v), h = two(wh[i], v);
        lc[i][v / 2] = mul2(l, cc);
        ls[i][v / 2] = mul2(l, ss);
        hc[i][v / 2] = mul2(h, cc);
        hs[i][v / 2] = mul2(mul2(h, ss), pair(-1.f, -1.f));
      }
  }
  for (int h0 = first + part * per; h0 < end; h0 += U * stride) {
    Pack<T, VEC> lo[U][NP], hi[U][NP];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride + grp;
      load_head(lo[u], hi[u], x + (long)h * a.hd, half, ln, h < end);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride + grp;
      if constexpr (KIND != V) {
        f2 ss = pair(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int v = 0; v < VEC; v += 2) {
            const f2 p = lo[u][i].at2(v), q = hi[u][i].at2(v);
            ss = fma2(p, p, fma2(q, q, ss));
          }
        const float r = rsqrtf(group_sum(sum2(ss), a.lanes) * inv_hd + a.eps);
        const f2 rr = pair(r, r);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float yl[VEC], yh[VEC];
#pragma unroll
          for (int v = 0; v < VEC; v += 2) {
            const f2 p = mul2(lo[u][i].at2(v), rr), q = mul2(hi[u][i].at2(v), rr);
            put(yl, v, fma2(q, hs[i][v / 2], mul2(p, lc[i][v / 2])));
            put(yh, v, fma2(p, ls[i][v / 2], mul2(q, hc[i][v / 2])));
          }
          lo[u][i].set_all(yl);
          hi[u][i].set_all(yh);
        }
      }
      store_head(lo[u], hi[u], y + (long)h * a.hd, half, ln, h < end);
    }
  }
}

template <typename T, int VEC, int NP, int U>
__global__ void __launch_bounds__(NT, VEC > 1 ? 4 : 1) qk_fwd_kernel(const Args a) {
  const int lane = threadIdx.x & 31;
  const long item = (long)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
  if (item >= a.tokens * a.split) return;
  const long token = item / a.split;
  const int part = (int)(item % a.split), grp = lane / a.lanes;
  const Lane<VEC, NP> ln(lane & (a.lanes - 1), a.lanes, a.hd >> 1);
  const T* x = reinterpret_cast<const T*>(a.x) + token * a.ld;
  T* y = reinterpret_cast<T*>(a.out) + token * a.ldo;
  float c[NP][VEC], s[NP][VEC];
  load_table(a, ln, token, c, s, lane);
  fwd_run<Q, T, VEC, NP, U>(a, x, y, ln, grp, part, c, s);
  fwd_run<K, T, VEC, NP, U>(a, x, y, ln, grp, part, c, s);
  fwd_run<V, T, VEC, NP, U>(a, x, y, ln, grp, part, c, s);
}

template <int KIND, typename T, int VEC, int NP, int U>
__device__ __forceinline__ void bwd_run(const Args& a, const T* x, const T* g, T* dx, const Lane<VEC, NP>& ln, int grp,
                                        int part, const float (&c)[NP][VEC], const float (&s)[NP][VEC],
                                        float (&dl)[NP][VEC], float (&dh)[NP][VEC]) {
  const int half = a.hd >> 1, per = 32 / a.lanes, stride = per * a.split;
  const int first = KIND == Q ? 0 : KIND == K ? a.nq : a.nq + a.nkv, end = first + (KIND == Q ? a.nq : a.nkv);
  const float inv_hd = 1.f / (float)a.hd;
  float wl[NP][VEC], wh[NP][VEC];
  if constexpr (KIND != V) load_weight(KIND == Q ? a.wq : a.wk, a.wdt, ln, half, wl, wh);
  for (int h0 = first + part * per; h0 < end; h0 += U * stride) {
    Pack<T, VEC> gl[U][NP], gh[U][NP], xl[U][NP], xh[U][NP];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride + grp;
      load_head(gl[u], gh[u], g + (long)h * a.hd, half, ln, h < end);
      if constexpr (KIND != V) load_head(xl[u], xh[u], x + (long)h * a.hd, half, ln, h < end);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * stride + grp;
      if constexpr (KIND != V) {
        // gu = R^T g; with n = x r, mean(gu w n) = r mean(gu w x), so both sums go over the lanes together
        constexpr int PAIRS = (VEC + 1) / 2;
        f2 ul[NP][PAIRS], uh[NP][PAIRS], ss = pair(0.f, 0.f), dot = ss;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int v = 0; v < VEC; v += 2) {
            const f2 p = xl[u][i].at2(v), q = xh[u][i].at2(v), e = gl[u][i].at2(v), f = gh[u][i].at2(v);
            const f2 cc = two(c[i], v), sn = two(s[i], v);
            ul[i][v / 2] = fma2(f, sn, mul2(e, cc));
            uh[i][v / 2] = fma2(mul2(e, sn), pair(-1.f, -1.f), mul2(f, cc));
            ss = fma2(p, p, fma2(q, q, ss));
            dot = fma2(mul2(ul[i][v / 2], two(wl[i], v)), p, fma2(mul2(uh[i][v / 2], two(wh[i], v)), q, dot));
          }
        const float sq = group_sum(sum2(ss), a.lanes), dt = group_sum(sum2(dot), a.lanes);
        // heads past the run were loaded as zeros: with r = 0 they add nothing, at eps = 0 neither
        const float r = h < end ? rsqrtf(sq * inv_hd + a.eps) : 0.f, m = r * dt * inv_hd;  // m = mean(gu w n)
        const f2 rr = pair(r, r), mm = pair(-m, -m);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          float al[VEC], ah[VEC];
#pragma unroll
          for (int v = 0; v < VEC; v += 2) {
            const f2 nl = mul2(xl[u][i].at2(v), rr), nh = mul2(xh[u][i].at2(v), rr);
            put(al, v, mul2(rr, fma2(nl, mm, mul2(ul[i][v / 2], two(wl[i], v)))));
            put(ah, v, mul2(rr, fma2(nh, mm, mul2(uh[i][v / 2], two(wh[i], v)))));
            put(dl[i], v, fma2(ul[i][v / 2], nl, two(dl[i], v)));
            put(dh[i], v, fma2(uh[i][v / 2], nh, two(dh[i], v)));
          }
          gl[u][i].set_all(al);
          gh[u][i].set_all(ah);
        }
      }
      store_head(gl[u], gh[u], dx + (long)h * a.hd, half, ln, h < end);
    }
  }
}

template <typename T, int VEC, int NP, int U>
__global__ void __launch_bounds__(NT, VEC > 1 ? 2 : 1) qk_bwd_kernel(const Args a) {
  extern __shared__ float sh[];  // [NT / 32][2 hd]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = a.hd >> 1;
  const Lane<VEC, NP> ln(lane & (a.lanes - 1), a.lanes, half);
  const int grp = lane / a.lanes;
  float dl[2][NP][VEC], dh[2][NP][VEC];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int v = 0; v < VEC; ++v) dl[t][i][v] = 0.f, dh[t][i][v] = 0.f;
  for (long item = (long)blockIdx.x * (NT / 32) + warp; item < a.tokens * a.split;
       item += (long)gridDim.x * (NT / 32)) {
    const long token = item / a.split;
    const int part = (int)(item % a.split);
    const T* x = reinterpret_cast<const T*>(a.x) + token * a.ld;
    const T* g = reinterpret_cast<const T*>(a.g) + token * a.ldg;
    T* dx = reinterpret_cast<T*>(a.out) + token * a.ldo;
    float c[NP][VEC], s[NP][VEC];
    load_table(a, ln, token, c, s, lane);
    bwd_run<Q, T, VEC, NP, U>(a, x, g, dx, ln, grp, part, c, s, dl[0], dh[0]);
    bwd_run<K, T, VEC, NP, U>(a, x, g, dx, ln, grp, part, c, s, dl[1], dh[1]);
    bwd_run<V, T, VEC, NP, U>(a, x, g, dx, ln, grp, part, c, s, dl[0], dh[0]);
  }
  // the groups of a warp, then the warps of the block, in a fixed order
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float l = dl[t][i][v], h = dh[t][i][v];
        for (int o = a.lanes; o < 32; o <<= 1) {
          l += __shfl_xor_sync(0xffffffffu, l, o);
          h += __shfl_xor_sync(0xffffffffu, h, o);
        }
        if (grp == 0 && ln.on[i]) {
          float* row = sh + (long)warp * 2 * a.hd + t * a.hd;
          row[ln.off[i] + v] = l;
          row[ln.off[i] + half + v] = h;
        }
      }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * a.hd; j += NT) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) t += sh[w * 2 * a.hd + j];
    a.part[(long)blockIdx.x * 2 * a.hd + j] = t;
  }
}

// Column sums of part[nparts, 2 hd] in a fixed order (32 warps, each every 32nd row, added in warp
// order): columns [0, hd) to dq, [hd, 2 hd) to dk, stored in their own type or added to fp32.
__global__ void __launch_bounds__(1024) qk_dw_reduce_kernel(const float* __restrict__ part, int nparts, int hd,
                                                            void* dq, void* dk, int dt, int accumulate) {
  __shared__ float red[32][33];
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  const int col = blockIdx.x * 32 + l;
  float s = 0.f;
  if (col < 2 * hd)
    for (int b = w; b < nparts; b += 32) s += part[(long)b * 2 * hd + col];
  red[w][l] = s;
  __syncthreads();
  if (w == 0 && col < 2 * hd) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][l];
    void* d = col < hd ? dq : dk;
    const int j = col < hd ? col : col - hd;
    if (accumulate) t += reinterpret_cast<float*>(d)[j];
    store_as(d, j, dt, t);
  }
}

}  // namespace qk
}  // namespace dtb

using namespace dtb;

namespace {

// Fills what both directions share; whether the vector kernels apply (single elements otherwise).
bool qk_common(qk::Args& a, const char* op, const torch::Tensor& x, const torch::Tensor& wq, const torch::Tensor& wk,
               const torch::Tensor& cos_t, const torch::Tensor& sin_t, const c10::optional<torch::Tensor>& pos,
               int64_t nq, int64_t nkv, int64_t hd, int64_t seqlen, double eps) {
  DTB_CHECK(x.is_cuda() && x.dim() == 2 && is_float_type(x.scalar_type()), "%s: qkv must be a 2-D CUDA tensor of fp32, bf16 or fp16", op);
  DTB_CHECK(nq > 0 && nkv > 0 && hd > 0 && hd % 2 == 0 && hd <= 512, "%s: needs heads > 0 and an even head size up to 512 (nq=%ld nkv=%ld hd=%ld)", op, (long)nq, (long)nkv, (long)hd);
  DTB_CHECK(x.size(1) == (nq + 2 * nkv) * hd, "%s: qkv has %ld columns, (nq + 2 nkv) * head_dim = %ld", op, (long)x.size(1), (long)((nq + 2 * nkv) * hd));
  DTB_CHECK(x.numel() == 0 || x.stride(1) == 1, "%s: qkv columns must be contiguous", op);
  for (const torch::Tensor* w : {&wq, &wk})
    DTB_CHECK(w->is_cuda() && w->is_contiguous() && w->numel() == hd && is_float_type(w->scalar_type()) && w->scalar_type() == wq.scalar_type(), "%s: the norm weights must be contiguous [%ld] tensors of one float type on the GPU", op, (long)hd);
  for (const torch::Tensor* t : {&cos_t, &sin_t})
    DTB_CHECK(t->is_cuda() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 && t->size(1) == hd && t->size(0) == cos_t.size(0), "%s: cos and sin must be contiguous fp32 [positions, %ld]", op, (long)hd);
  for (const torch::Tensor* t : {&wq, &wk, &cos_t, &sin_t})
    DTB_CHECK(t->device() == x.device(), "%s: all tensors must be on one device", op);
  a.x = x.data_ptr();
  a.ld = x.stride(0);
  a.wq = wq.data_ptr();
  a.wk = wk.data_ptr();
  a.wdt = dt_code(wq.scalar_type());
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.tokens = x.size(0);
  a.table_rows = cos_t.size(0);
  a.seqlen = seqlen;
  if (pos.has_value()) {
    DTB_CHECK(pos->device() == x.device() && pos->is_contiguous() && pos->numel() == x.size(0) && (pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt), "%s: positions must be a contiguous int64 or int32 tensor with one entry per token, on the tokens' device", op);
    a.pos = pos->data_ptr();
    a.pos64 = pos->scalar_type() == at::kLong;
  } else {
    DTB_CHECK(seqlen > 0 && (seqlen <= cos_t.size(0) || x.size(0) <= cos_t.size(0)), "%s: seqlen=%ld needs as many table rows (have %ld)", op, (long)seqlen, (long)cos_t.size(0));
  }
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.hd = (int)hd;
  a.eps = (float)eps;
  a.err = dtb_error_word();
  // 4 elements at a time: a head of 8 n elements, every row on a boundary of 4 elements
  const long es = (long)x.element_size(), bound = 4 * es;
  return hd % 8 == 0 && hd <= 256 && reinterpret_cast<uintptr_t>(a.x) % bound == 0 && (a.ld * es) % bound == 0 &&
         (reinterpret_cast<uintptr_t>(a.cos_t) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.sin_t) & 15) == 0;
}

void qk_lanes(qk::Args& a, bool vec) {
  int lanes = 32;
  if (vec) {
    lanes = 1;
    while (lanes * 8 < a.hd) lanes *= 2;
  }
  a.lanes = lanes;
  // few tokens: their heads are spread over more warps, down to one round of heads per warp
  const int per = 32 / lanes, rounds = (a.nq + 2 * a.nkv + per - 1) / per;
  const long want = (long)device_sm_count() * 32;
  long split = a.tokens > 0 ? want / a.tokens : 1;
  a.split = (int)std::max(1L, std::min<long>(split, rounds));
}

}  // namespace

torch::Tensor qk_norm_rope_fwd(torch::Tensor x, torch::Tensor wq, torch::Tensor wk, torch::Tensor cos_t,
                               torch::Tensor sin_t, c10::optional<torch::Tensor> pos, int64_t nq, int64_t nkv,
                               int64_t hd, int64_t seqlen, double eps) {
  const c10::cuda::CUDAGuard guard(x.device());
  qk::Args a{};
  const bool vec = qk_common(a, "qk_norm_rope", x, wq, wk, cos_t, sin_t, pos, nq, nkv, hd, seqlen, eps);
  auto y = torch::empty({x.size(0), x.size(1)}, x.options());
  if (x.size(0) == 0) return y;
  a.out = y.data_ptr();
  a.ldo = y.stride(0);
  qk_lanes(a, vec);
  const long blocks = (a.tokens * a.split + qk::NT / 32 - 1) / (qk::NT / 32);
  DTB_CHECK(blocks < (1L << 31), "qk_norm_rope: too many tokens");
  auto st = at::cuda::getCurrentCUDAStream();
  DTB_FLOAT_TYPES(x.scalar_type(), {
    if (vec) qk::qk_fwd_kernel<T, 4, 1, sizeof(T) == 4 ? 2 : 4><<<(unsigned)blocks, qk::NT, 0, st>>>(a);
    else qk::qk_fwd_kernel<T, 1, 8, 1><<<(unsigned)blocks, qk::NT, 0, st>>>(a);
  });
  DTB_LAUNCH_CHECK();
  return y;
}

// dx; the weight gradients go to dwq / dwk: stored in their type, or added to fp32 when `accumulate`.
torch::Tensor qk_norm_rope_bwd(torch::Tensor g, torch::Tensor x, torch::Tensor wq, torch::Tensor wk,
                               torch::Tensor cos_t, torch::Tensor sin_t, c10::optional<torch::Tensor> pos, int64_t nq,
                               int64_t nkv, int64_t hd, int64_t seqlen, double eps, torch::Tensor dwq,
                               torch::Tensor dwk, bool accumulate) {
  const c10::cuda::CUDAGuard guard(x.device());
  qk::Args a{};
  bool vec = qk_common(a, "qk_norm_rope backward", x, wq, wk, cos_t, sin_t, pos, nq, nkv, hd, seqlen, eps);
  DTB_CHECK(g.device() == x.device() && g.sizes() == x.sizes() && g.scalar_type() == x.scalar_type() && (g.numel() == 0 || g.stride(1) == 1), "qk_norm_rope backward: the gradient must have the input's shape and type and contiguous columns");
  for (const torch::Tensor* d : {&dwq, &dwk})
    DTB_CHECK(d->device() == x.device() && d->is_contiguous() && d->numel() == hd && is_float_type(d->scalar_type()) && d->scalar_type() == dwq.scalar_type() && (!accumulate || d->scalar_type() == at::kFloat), "qk_norm_rope backward: weight gradients must be contiguous [%ld] tensors of one float type (fp32 to accumulate)", (long)hd);
  auto dx = torch::empty({x.size(0), x.size(1)}, x.options());
  if (x.size(0) == 0) {
    if (!accumulate) {
      dwq.zero_();
      dwk.zero_();
    }
    return dx;
  }
  a.g = g.data_ptr();
  a.ldg = g.stride(0);
  a.out = dx.data_ptr();
  a.ldo = dx.stride(0);
  const long bound = 4 * (long)x.element_size();
  vec = vec && reinterpret_cast<uintptr_t>(a.g) % bound == 0 && (a.ldg * (long)x.element_size()) % bound == 0;
  qk_lanes(a, vec);
  const int warps = qk::NT / 32;
  const int blocks = (int)std::min<long>((a.tokens * a.split + warps - 1) / warps, (long)device_sm_count() * 2);  // one wave: two blocks an SM
  auto part = torch::empty({blocks, 2 * hd}, x.options().dtype(at::kFloat));
  a.part = part.data_ptr<float>();
  auto st = at::cuda::getCurrentCUDAStream();
  const size_t smem = sizeof(float) * warps * 2 * hd;
  DTB_FLOAT_TYPES(x.scalar_type(), {
    if (vec) qk::qk_bwd_kernel<T, 4, 1, sizeof(T) == 4 ? 2 : 4><<<blocks, qk::NT, smem, st>>>(a);
    else qk::qk_bwd_kernel<T, 1, 8, 1><<<blocks, qk::NT, smem, st>>>(a);
  });
  DTB_LAUNCH_CHECK();
  qk::qk_dw_reduce_kernel<<<(unsigned)((2 * hd + 31) / 32), 1024, 0, st>>>(
      a.part, blocks, (int)hd, dwq.data_ptr(), dwk.data_ptr(), dt_code(dwq.scalar_type()), accumulate ? 1 : 0);
  DTB_LAUNCH_CHECK();
  return dx;
}
