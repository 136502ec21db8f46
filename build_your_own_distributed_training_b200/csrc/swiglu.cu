// silu(g) * u of a packed [tokens, g | u] bf16 tensor, for projections whose GEMM has no SwiGLU epilogue
// (8-bit weights).  Bound by memory: 6 bytes an output element; one thread moves 16-byte vectors of g, u
// and the product.  fp32 math, one rounding.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "vecio.cuh"

namespace dtb {
namespace {

template <int VEC>
__global__ void __launch_bounds__(256) swiglu_fwd_kernel(const __nv_bfloat16* __restrict__ gu,
                                                         __nv_bfloat16* __restrict__ act, long total, long F) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const long per = F / VEC, row = i / per, c = (i % per) * VEC;
  Pack<__nv_bfloat16, VEC> g, u;
  g.load(gu + row * 2 * F + c);
  u.load(gu + row * 2 * F + F + c);
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const float x = g.at(k);
    g.set(k, x / (1.f + expf(-x)) * u.at(k));
  }
  g.store(act + row * F + c);
}

}  // namespace
}  // namespace dtb

using namespace dtb;

void swiglu_fwd(torch::Tensor gu, torch::Tensor act) {
  DTB_CHECK(gu.is_cuda() && act.device() == gu.device() && gu.scalar_type() == at::kBFloat16 && act.scalar_type() == at::kBFloat16 && gu.dim() == 2 && act.dim() == 2 && gu.is_contiguous() && act.is_contiguous() && gu.size(0) == act.size(0) && gu.size(1) == 2 * act.size(1), "swiglu_fwd: contiguous bf16 [M, 2F] -> [M, F]");
  const c10::cuda::CUDAGuard guard(gu.device());
  const long M = act.size(0), F = act.size(1);
  if (M * F == 0) return;
  const bool wide = F % 8 == 0 && ((reinterpret_cast<uintptr_t>(gu.data_ptr()) | reinterpret_cast<uintptr_t>(act.data_ptr())) & 15) == 0;
  const long total = wide ? M * F / 8 : M * F, blocks = (total + 255) / 256;
  DTB_CHECK(blocks < (1L << 31), "swiglu_fwd: too large");
  auto st = at::cuda::getCurrentCUDAStream();
  const auto* g = reinterpret_cast<const __nv_bfloat16*>(gu.data_ptr());
  auto* a = reinterpret_cast<__nv_bfloat16*>(act.data_ptr());
  if (wide) swiglu_fwd_kernel<8><<<(unsigned)blocks, 256, 0, st>>>(g, a, total, F);
  else swiglu_fwd_kernel<1><<<(unsigned)blocks, 256, 0, st>>>(g, a, total, F);
  DTB_LAUNCH_CHECK();
}
