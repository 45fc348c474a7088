// Device helpers shared by the token operators (linear.hip, layer_norm.hip, attention.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "yk_internal.h"

namespace yk {
namespace tok {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// 16 / 8 bytes at an element's alignment: gfx950 loads and stores them in one instruction at any
// address, so rows of an odd width need no path of their own
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

// Storage types.  V8 is 8 elements, the operand of one 16x16x32 MFMA step: lane l holds row (or
// column) l % 16 and the K elements 8 * (l / 16) .. + 7.  float32 keeps the same layout and issues
// eight v_mfma_f32_16x16x4_f32, element e of every lane each time (exact f32 products, f32 sums).
struct B16 {
  using T = unsigned short;
  using V8 = s16x8;
  static constexpr int kBytes = 2;
};
struct H16 {
  using T = _Float16;
  using V8 = s16x8;
  static constexpr int kBytes = 2;
};
struct F32 {
  using T = float;
  using V8 = f32x8;
  static constexpr int kBytes = 4;
};

template <class Tr>
__device__ __forceinline__ f32x4 mma(typename Tr::V8 a, typename Tr::V8 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma<B16>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma<H16>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma<F32>(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <class Tr>
__device__ __forceinline__ float to_f32(typename Tr::T v);
template <>
__device__ __forceinline__ float to_f32<B16>(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
template <>
__device__ __forceinline__ float to_f32<H16>(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f32<F32>(float v) { return v; }

// Round to nearest, ties to even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32).
template <class Tr>
__device__ __forceinline__ typename Tr::T from_f32(float v);
template <>
__device__ __forceinline__ unsigned short from_f32<B16>(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
template <>
__device__ __forceinline__ _Float16 from_f32<H16>(float v) { return (_Float16)v; }
template <>
__device__ __forceinline__ float from_f32<F32>(float v) { return v; }

// 4 elements from registers to any address / to LDS order
template <class Tr>
__device__ __forceinline__ void store4(typename Tr::T* p, f32x4 v) {
  if constexpr (Tr::kBytes == 4) {
    *(u32x4_any*)p = __builtin_bit_cast(u32x4, v);
  } else {
    typename Tr::T t[4] = {from_f32<Tr>(v[0]), from_f32<Tr>(v[1]), from_f32<Tr>(v[2]), from_f32<Tr>(v[3])};
    u32x2 u;
    __builtin_memcpy(&u, t, 8);
    *(u32x2_any*)p = u;
  }
}
template <class Tr>
__device__ __forceinline__ f32x4 load4(const typename Tr::T* p) {
  if constexpr (Tr::kBytes == 4) {
    return __builtin_bit_cast(f32x4, (u32x4) * (const u32x4_any*)p);
  } else {
    const u32x2 u = *(const u32x2_any*)p;
    typename Tr::T t[4];
    __builtin_memcpy(t, &u, 8);
    return f32x4{to_f32<Tr>(t[0]), to_f32<Tr>(t[1]), to_f32<Tr>(t[2]), to_f32<Tr>(t[3])};
  }
}

// 8 elements between registers and any address
template <class Tr>
__device__ __forceinline__ void store8(typename Tr::T* p, const float* v) {
  if constexpr (Tr::kBytes == 4) {
    *(u32x4_any*)p = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
    *(u32x4_any*)(p + 4) = __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]});
  } else {
    typename Tr::T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = from_f32<Tr>(v[e]);
    u32x4 u;
    __builtin_memcpy(&u, t, 16);
    *(u32x4_any*)p = u;
  }
}
template <class Tr>
__device__ __forceinline__ void add8(const typename Tr::T* p, float* v) {
  const f32x4 lo = load4<Tr>(p), hi = load4<Tr>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] += lo[e];
    v[4 + e] += hi[e];
  }
}

// 16 bytes (kEpc elements) of a row, elements at or past n0 zero: one load where they are all
// there, element loads at the row's end
template <class Tr>
__device__ __forceinline__ u32x4 load16(const typename Tr::T* p, int n) {
  constexpr int kEpc = 16 / Tr::kBytes;
  u32x4 u{0, 0, 0, 0};
  if (n >= kEpc) {
    u = *(const u32x4_any*)p;
  } else if (n > 0) {
    typename Tr::T t[kEpc];
#pragma unroll
    for (int e = 0; e < kEpc; ++e) t[e] = e < n ? p[e] : (typename Tr::T)0;
    __builtin_memcpy(&u, t, 16);
  }
  return u;
}
// The same of a row that may not be there (`ok`), without branches: what is not to be read is
// loaded from `safe` (an element, or with `whole` 16 bytes, that exist) and replaced by zero.
// whole: n is a multiple of the chunk, so a chunk is there or not.
template <class Tr>
__device__ __forceinline__ u32x4 load16_if(const typename Tr::T* p, const typename Tr::T* safe, int n, bool ok, bool whole) {
  constexpr int kEpc = 16 / Tr::kBytes;
  u32x4 u;
  if (whole) {
    ok = ok && n > 0;
    u = *(const u32x4_any*)(ok ? p : safe);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = ok ? u[i] : 0u;
  } else {
    typename Tr::T t[kEpc];
#pragma unroll
    for (int e = 0; e < kEpc; ++e) {
      const bool k = ok && e < n;
      const typename Tr::T v = *(k ? p + e : safe);
      t[e] = k ? v : (typename Tr::T)0;
    }
    __builtin_memcpy(&u, t, 16);
  }
  return u;
}

__device__ __forceinline__ float load_param(const void* p, int64_t i, int is_f32, int dtype) {
  if (is_f32) return ((const float*)p)[i];
  return dtype == YK_ACT_BF16 ? to_f32<B16>(((const unsigned short*)p)[i]) : (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void store_param(void* p, int64_t i, float v, int is_f32, int dtype) {
  if (is_f32) ((float*)p)[i] = v;
  else if (dtype == YK_ACT_BF16) ((unsigned short*)p)[i] = from_f32<B16>(v);
  else ((_Float16*)p)[i] = (_Float16)v;
}

// 2^x and 1 / x: one instruction each, off by about one unit in the last place
__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_f(float x) { return __builtin_amdgcn_rcpf(x); }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// Phi(-|z|) and e^(-z^2 / 2): Phi's tail as in Abramowitz and Stegun 7.1.26 (Hastings), a polynomial
// in t = 1 / (1 + p |z| / sqrt 2) times that exponential, off by less than 7.5e-8 of 1.  14
// instructions against some 40 of erff, whose two ranges a wave walks both; the product z Phi(z)
// is then off by less than 2 float32 roundings of z.
__device__ __forceinline__ float normal_tail(float z, float& e) {
  const float t = rcp_f(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
  e = exp2_f(z * z * (-0.5f * kLog2e));
  float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
  p = fmaf(p, t, 0.5f * 1.421413741f);
  p = fmaf(p, t, 0.5f * -0.284496736f);
  p = fmaf(p, t, 0.5f * 0.254829592f);
  return p * t * e;
}

// act(z) and act'(z) in float32.  GELU is z Phi(z).
__device__ __forceinline__ float act_f32(float z, int act) {
  if (act == YK_TOK_GELU) {
    float e;
    const float q = normal_tail(z, e);
    return z * (z < 0.f ? q : 1.f - q);
  }
  if (act == YK_TOK_SILU) return z * rcp_f(1.f + exp2_f(z * -kLog2e));
  if (act == YK_TOK_RELU) return z > 0.f ? z : z != z ? z : 0.f;
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == YK_TOK_GELU) {
    float e;
    const float q = normal_tail(z, e);
    return fmaf(z * 0.39894228040143268f, e, z < 0.f ? q : 1.f - q);
  }
  if (act == YK_TOK_SILU) {
    const float s = rcp_f(1.f + exp2_f(z * -kLog2e));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (act == YK_TOK_RELU) return z > 0.f ? 1.f : 0.f;
  return 1.f;
}

__device__ __forceinline__ int rfl(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Work item of this workgroup among n: the dispatcher deals workgroups round-robin to the 8 XCDs,
// each with an L2 of its own, so XCD i % 8 gets one contiguous range of items and neighbours
// (which read the same operand rows) meet in one L2.  A bijection for any n.
__device__ __forceinline__ int xcd_item(int i, int n) {
  const int x = i & 7, q = n >> 3, r = n & 7;
  return x * q + (x < r ? x : r) + (i >> 3);
}

// Bytes of one 16-bit / 32-bit element; 0 for a type the token operators do not take
inline int tok_bytes(int dtype) {
  return dtype == YK_ACT_F32 ? 4 : dtype == YK_ACT_BF16 || dtype == YK_ACT_F16 ? 2 : 0;
}
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Workgroups of `threads` that one launch holds along x: HIP takes fewer than 2^32 threads there.
inline int64_t most_groups(int threads) { return 0xffffffffll / threads; }

// Every launch of the token operators; a call's first error is kept for launched().  (The runtime's last
// error may be another call's, of the caller's own, and is neither reported nor cleared here.)
inline thread_local hipError_t t_launch_error = hipSuccess;
template <class... P>
inline void launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, std::common_type_t<P>... args) {
  if (KernelNames* names = KernelNames::current()) return names->add((const void*)kernel);
  if (t_launch_error != hipSuccess) return;
  void* ptrs[] = {(void*)&args...};
  t_launch_error = hipLaunchKernel((const void*)kernel, grid, block, ptrs, lds, st);
}
inline int launched(const char* what) {
  const hipError_t e = t_launch_error;
  if (e == hipSuccess) return YK_OK;
  t_launch_error = hipSuccess;
  (void)hipGetLastError();  // reported here
  set_error(std::string(what) + ": launch failed: " + hipGetErrorString(e));
  return YK_ERR_HIP;
}

}  // namespace tok
}  // namespace yk
