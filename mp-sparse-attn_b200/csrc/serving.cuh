// What the kernels that serve a model token by token share: 8 elements of a row in fp32, MX element codes and page look-up.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/mpsa.h"

namespace mpsa {

enum Elem : int { E4M3 = 0, E5M2 = 1, E2M1 = 2 };

// 4 neighbouring elements, 8 or 16 bytes at once: as they are in memory, and in fp32
template <typename T> struct Raw4 { uint2 u; };
template <> struct Raw4<float> { float4 u; };
template <typename T>
__device__ __forceinline__ Raw4<T> raw4(const T* p) { return {*reinterpret_cast<const decltype(Raw4<T>::u)*>(p)}; }
__device__ __forceinline__ void wide4(const Raw4<__nv_bfloat16>& r, float (&x)[4]) {
  x[0] = __uint_as_float(r.u.x << 16); x[1] = __uint_as_float(r.u.x & 0xffff0000u);
  x[2] = __uint_as_float(r.u.y << 16); x[3] = __uint_as_float(r.u.y & 0xffff0000u);
}
__device__ __forceinline__ void wide4(const Raw4<__half>& r, float (&x)[4]) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&r.u.y));
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
__device__ __forceinline__ void wide4(const Raw4<float>& r, float (&x)[4]) { x[0] = r.u.x; x[1] = r.u.y; x[2] = r.u.z; x[3] = r.u.w; }
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]) { wide4(raw4(p), x); }

__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2(T(), x[0], x[1]), pack2(T(), x[2], x[3]));
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }

// The page of a table entry, or -1 where there is none.
__device__ __forceinline__ int page_of(const int* table, int entry, int max_pages, int num_pages) {
  if ((unsigned)entry >= (unsigned)max_pages) return -1;
  const int p = table[entry];
  return (unsigned)p < (unsigned)num_pages ? p : -1;
}

constexpr __host__ __device__ int code_bytes(int elem, int D) { return elem == E2M1 ? D / 2 : D; }

// What a word of codes stands for in units of the block's scale, as fp16 pairs (exact): four 8-bit codes, or eight 4-bit ones.
template <int ELEM>
__device__ __forceinline__ void elem_two(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (ELEM == E4M3) asm("{\n.reg .b16 x, y;\nmov.b32 {x, y}, %2;\ncvt.rn.f16x2.e4m3x2 %0, x;\ncvt.rn.f16x2.e4m3x2 %1, y;\n}" : "=r"(a), "=r"(b) : "r"(w));
  else asm("{\n.reg .b16 x, y;\nmov.b32 {x, y}, %2;\ncvt.rn.f16x2.e5m2x2 %0, x;\ncvt.rn.f16x2.e5m2x2 %1, y;\n}" : "=r"(a), "=r"(b) : "r"(w));
}
__device__ __forceinline__ void elem_quads(uint32_t w, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm("{\n.reg .b8 x, y, z, u;\nmov.b32 {x, y, z, u}, %4;\ncvt.rn.f16x2.e2m1x2 %0, x;\ncvt.rn.f16x2.e2m1x2 %1, y;\ncvt.rn.f16x2.e2m1x2 %2, z;\n"
      "cvt.rn.f16x2.e2m1x2 %3, u;\n}"
      : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(w));
}

// 2^(code - 127); 255 is NaN, and 0 (which mpsa_kv_append never writes) counts as zero
__device__ __forceinline__ float scale_value(uint32_t code) { return __uint_as_float(code == 255u ? 0x7fffffffu : code << 23); }

// Host side: whether a cache can be used (an error is set otherwise).
int check_cache(const mpsa_kv_cache& c, const char* what);

}  // namespace mpsa
