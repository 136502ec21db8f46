// Element types and 16-byte vector access shared by the elementwise and row kernels:
// fp32, bf16 and fp16 storage, arithmetic in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace dtb {

template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two fp32 at a time: add / mul / fma on register pairs, half the instructions of kernels that stream 16-bit
// elements.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// VEC consecutive elements as they lie in memory: moved as 16-byte words (8-byte ones where the elements fill
// just that; the address must be aligned alike) or else one by one.
template <typename T, int VEC>
struct Pack {
  static constexpr int BYTES = VEC * (int)sizeof(T);
  static constexpr bool WIDE = BYTES % 16 == 0, HALF = BYTES == 8;
  static constexpr int WORDS = WIDE ? BYTES / 16 : 1;
  union {
    uint4 w[WORDS];
    uint2 h;
    T e[VEC];
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else if constexpr (HALF) {
      h = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
    } else if constexpr (HALF) {
      *reinterpret_cast<uint2*>(p) = h;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = e[i];
    }
  }
  __device__ __forceinline__ float at(int i) const { return as_float<T>(e[i]); }
  __device__ __forceinline__ void set(int i, float v) { e[i] = from_float<T>(v); }
  // elements i and i + 1 as a pair; 0 stands for an element past the end
  __device__ __forceinline__ unsigned long long at2(int i) const { return pair(at(i), i + 1 < VEC ? at(i + 1) : 0.f); }
  // elements i and i + 1 (i even): one conversion instruction for a pair of 16-bit elements
  __device__ __forceinline__ void set2(int i, float a, float b) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
      e[i] = v.x;
      e[i + 1] = v.y;
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 v = __floats2half2_rn(a, b);
      e[i] = v.x;
      e[i + 1] = v.y;
    } else {
      e[i] = a;
      e[i + 1] = b;
    }
  }
  // all elements of f
  __device__ __forceinline__ void set_all(const float (&f)[VEC]) {
    if constexpr (VEC % 2 == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) set2(i, f[i], f[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) set(i, f[i]);
    }
  }
};

// storage type of an operand whose type is chosen at run time
enum : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

__device__ __forceinline__ float load_as(const void* p, long i, int dt) {
  if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (dt == DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_as(void* p, long i, int dt, float v) {
  if (dt == DT_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == DT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

}  // namespace dtb

#ifdef TORCH_EXTENSION_NAME
#include <torch/extension.h>
namespace dtb {
inline bool is_float_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
inline int dt_code(at::ScalarType t) { return t == at::kFloat ? DT_F32 : t == at::kBFloat16 ? DT_BF16 : DT_F16; }
}  // namespace dtb
// runs `...` with T the storage type of scalar type `st`
#define DTB_FLOAT_TYPES(st, ...)                                   \
  do {                                                             \
    if ((st) == at::kFloat) { using T = float; __VA_ARGS__; }      \
    else if ((st) == at::kBFloat16) { using T = __nv_bfloat16; __VA_ARGS__; } \
    else { using T = __half; __VA_ARGS__; }                        \
  } while (0)
#endif
