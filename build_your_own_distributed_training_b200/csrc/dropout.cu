// Residual add with dropout whose mask comes from a counter-based generator and is never stored.
//
//   y_e = r_e + keep(e) x_e / (1 - p'),   dx_e = keep(e) g_e / (1 - p'),   dr = g
//
// keep(e) compares 16 random bits with cut = round(p 2^16), p' = cut / 2^16, so the expectation is
// exact for the probability really used.  The bits are Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): key = the 64-bit seed, counter = element / 8,
// and element e takes the (e % 8)-th 16-bit field of the 128-bit result.  The mask is therefore a
// function of (seed, element number) alone: a recomputed forward, the backward, another launch shape
// or a rank that holds only rows [a, b) of the activation (start = a * columns) all see the same one.
//
// One thread makes one counter's 8 elements (two counters' when there is work enough, so that more loads are
// in flight).  16 bits per element instead of 32 halve the generator's work: ten rounds of two 32 x 32 ->
// 64-bit products per 8 elements.  The forward is bound by memory, 8192 x 4096 bf16 in 32 us (6.4 TB/s of
// x, r and y); the backward moves a third less and comes near the generator's own time, 27 us (4.9 TB/s).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "common.cuh"
#include "vecio.cuh"

namespace dtb {
namespace drop {

constexpr int NT = 256;

__device__ __forceinline__ uint4 philox(uint64_t ctr, uint32_t k0, uint32_t k1) {
  uint32_t a = (uint32_t)ctr, b = (uint32_t)(ctr >> 32), c = 0, d = 0;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = (uint64_t)0xD2511F53u * a, q = (uint64_t)0xCD9E8D57u * c;
    a = (uint32_t)(q >> 32) ^ b ^ k0;
    b = (uint32_t)q;
    c = (uint32_t)(p >> 32) ^ d ^ k1;
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(a, b, c, d);
}

__device__ __forceinline__ uint32_t field(const uint4& r, int i) {
  const uint32_t w = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
  return (i & 1) ? w >> 16 : w & 0xffffu;
}

// Groups of 8 consecutive element numbers, U per thread (their loads go out together); an element's number
// minus `start` indexes the tensors.  WIDE: start % 8 == 0 and 16-byte aligned bases, so whole groups move as
// vectors.
template <typename T, bool RES, bool WIDE, int U>
__global__ void __launch_bounds__(NT) dropout_kernel(const T* __restrict__ x, const T* __restrict__ r,
                                                     T* __restrict__ y, uint64_t n, uint64_t start, uint64_t groups,
                                                     uint32_t k0, uint32_t k1, uint32_t cut, float scale) {
  const uint64_t first = (uint64_t)blockIdx.x * (NT * U) + threadIdx.x;
  Pack<T, 8> px[U], pr[U];
  bool whole[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t t = first + u * NT, grp = (start >> 3) + t;
    const int64_t base = (int64_t)(grp * 8 - start);  // may be negative in the first group
    whole[u] = WIDE && t < groups && base >= 0 && (uint64_t)base + 8 <= n;
    if (whole[u]) {
      px[u].load(x + base);
      if (RES) pr[u].load(r + base);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t t = first + u * NT, grp = (start >> 3) + t;
    if (t >= groups) return;
    const int64_t base = (int64_t)(grp * 8 - start);
    const uint4 bits = philox(grp, k0, k1);
    if (whole[u]) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = field(bits, i) >= cut ? px[u].at(i) * scale : 0.f;
        f[i] = RES ? pr[u].at(i) + v : v;
      }
      px[u].set_all(f);
      px[u].store(y + base);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t e = base + i;
        if (e < 0 || (uint64_t)e >= n) continue;
        const float v = field(bits, i) >= cut ? as_float<T>(x[e]) * scale : 0.f;
        y[e] = from_float<T>(RES ? as_float<T>(r[e]) + v : v);
      }
    }
  }
}

}  // namespace drop
}  // namespace dtb

using namespace dtb;

// x: contiguous; residual: same shape and type, or none; elements are numbered from `start`.
torch::Tensor dropout_add(torch::Tensor x, c10::optional<torch::Tensor> residual, int64_t cut, int64_t seed,
                          int64_t start) {
  DTB_CHECK(x.is_cuda() && x.is_contiguous() && is_float_type(x.scalar_type()), "dropout_add: x must be a contiguous CUDA tensor of fp32, bf16 or fp16");
  DTB_CHECK(cut >= 0 && cut <= 65536 && start >= 0, "dropout_add: probability outside [0, 1] or negative start");
  const c10::cuda::CUDAGuard guard(x.device());
  if (residual.has_value())
    DTB_CHECK(residual->device() == x.device() && residual->is_contiguous() && residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), "dropout_add: the residual must be contiguous with x's shape, type and device");
  auto y = torch::empty_like(x);
  const uint64_t n = (uint64_t)x.numel(), s = (uint64_t)start;
  if (n == 0) return y;
  const uint64_t groups = (s + n + 7) / 8 - s / 8;
  const float scale = cut < 65536 ? (float)(65536.0 / (double)(65536 - cut)) : 0.f;
  const uint32_t k0 = (uint32_t)(uint64_t)seed, k1 = (uint32_t)((uint64_t)seed >> 32);
  uintptr_t bases = reinterpret_cast<uintptr_t>(x.data_ptr()) | reinterpret_cast<uintptr_t>(y.data_ptr());
  if (residual.has_value()) bases |= reinterpret_cast<uintptr_t>(residual->data_ptr());
  const bool wide = (s % 8) == 0 && (bases & 15) == 0;
  auto st = at::cuda::getCurrentCUDAStream();
  DTB_FLOAT_TYPES(x.scalar_type(), {
    const T* xp = reinterpret_cast<const T*>(x.data_ptr());
    const T* rp = residual.has_value() ? reinterpret_cast<const T*>(residual->data_ptr()) : nullptr;
    T* yp = reinterpret_cast<T*>(y.data_ptr());
    const uint32_t c = (uint32_t)cut;
    auto go = [&](auto kernel, int per) {
      const uint64_t blocks = (groups + drop::NT * per - 1) / (drop::NT * per);
      DTB_CHECK(blocks < (1ull << 31), "dropout_add: too many elements");
      kernel<<<(unsigned)blocks, drop::NT, 0, st>>>(xp, rp, yp, n, s, groups, k0, k1, c, scale);
    };
    // two groups a thread once that still gives every SM its blocks
    const bool deep = groups >= (uint64_t)device_sm_count() * drop::NT * 16;
    if (rp && wide) deep ? go(drop::dropout_kernel<T, true, true, 2>, 2) : go(drop::dropout_kernel<T, true, true, 1>, 1);
    else if (rp) go(drop::dropout_kernel<T, true, false, 1>, 1);
    else if (wide) deep ? go(drop::dropout_kernel<T, false, true, 2>, 2) : go(drop::dropout_kernel<T, false, true, 1>, 1);
    else go(drop::dropout_kernel<T, false, false, 1>, 1);
  });
  DTB_LAUNCH_CHECK();
  return y;
}
