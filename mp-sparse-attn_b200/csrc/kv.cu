// The paged MX cache of keys and values: quantised as it is written (mpsa_kv_append) and read back (mpsa_kv_read).  See include/mpsa.h for
// the layout.  Both are memory traffic: every element is read once and written once.  4 prefixes of 8192 tokens of 8 heads read back in 32 us
// (5.9 TB/s); 2 x 4099 tokens appended in 12 us (4.2 TB/s: 16 loads and 60 ALU operations, 2.3 waves of CTAs at 36 registers).
#include "api_internal.h"
#include "common.cuh"
#include "serving.cuh"

namespace mpsa {

int check_cache(const mpsa_kv_cache& c, const char* what) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return set_error(MPSA_ERR_BAD_ARG, "%s: null cache pointer", what);
  if (((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.k_scale | (uintptr_t)c.v_scale) % 16)
    return set_error(MPSA_ERR_BAD_ARG, "%s: the cache must be 16-byte aligned", what);
  if (c.elem < 0 || c.elem > 2) return set_error(MPSA_ERR_BAD_ARG, "%s: elem must be 0 (E4M3), 1 (E5M2) or 2 (E2M1)", what);
  if (c.D != 64 && c.D != 128) return set_error(MPSA_ERR_UNSUPPORTED, "%s: D must be 64 or 128", what);
  if (c.num_pages <= 0 || c.Hkv <= 0 || c.Hkv > 65535) return set_error(MPSA_ERR_BAD_ARG, "%s: the cache needs pages and 1 to 65535 heads", what);
  if (c.page_size < 16 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)))
    return set_error(MPSA_ERR_UNSUPPORTED, "%s: page_size must be a power of two from 16 to 1024", what);
  if ((double)c.num_pages * c.Hkv * c.page_size >= 4294967295.0) return set_error(MPSA_ERR_UNSUPPORTED, "%s: the cache may have 2^32 - 2 rows at most", what);
  return MPSA_OK;
}

namespace {

constexpr int kThreads = 128;

template <int ELEM> struct Largest;
template <> struct Largest<E4M3> { static constexpr int exponent = 8; static constexpr uint32_t mantissa = 0x600000; };     // 448
template <> struct Largest<E5M2> { static constexpr int exponent = 15; static constexpr uint32_t mantissa = 0x600000; };    // 57344
template <> struct Largest<E2M1> { static constexpr int exponent = 2; static constexpr uint32_t mantissa = 0x400000; };     // 6

// The smallest power of two at which amax (bits) does not exceed the type's largest value, as its exponent.
template <int ELEM>
__device__ __forceinline__ int block_exponent(uint32_t amax) {
  const int e = (int)(amax >> 23) - 127 - Largest<ELEM>::exponent + ((amax & 0x7fffffu) > Largest<ELEM>::mantissa);
  return max(e, -126);                     // (and with it every subnormal amax, and zero)
}

template <int ELEM>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[8], bool fine) {       // zeros where not fine
  if constexpr (ELEM == E2M1) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t two;
      asm("{\n.reg .b8 h;\ncvt.rn.satfinite.e2m1x2.f32 h, %2, %1;\ncvt.u32.u8 %0, h;\n}" : "=r"(two) : "f"(x[2 * i]), "f"(x[2 * i + 1]));
      r |= two << (8 * i);
    }
    *reinterpret_cast<uint32_t*>(p) = fine ? r : 0u;
  } else {
    uint32_t r[2] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned short two;
      if constexpr (ELEM == E4M3) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(two) : "f"(x[2 * i]), "f"(x[2 * i + 1]));
      else asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(two) : "f"(x[2 * i]), "f"(x[2 * i + 1]));
      r[i / 2] |= (uint32_t)two << (16 * (i % 2));
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(fine ? r[0] : 0u, fine ? r[1] : 0u);
  }
}

// The largest magnitude of 8 elements, as the bits of an fp32 number: a NaN is the largest.  16-bit elements two at a time.
__device__ __forceinline__ uint32_t magnitude(const Raw4<__nv_bfloat16> (&r)[2]) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t a = __vmaxu2(__vmaxu2(r[0].u.x & m, r[0].u.y & m), __vmaxu2(r[1].u.x & m, r[1].u.y & m));
  return max(a << 16, a & 0xffff0000u);
}
__device__ __forceinline__ uint32_t magnitude(const Raw4<__half> (&r)[2]) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t a = __vmaxu2(__vmaxu2(r[0].u.x & m, r[0].u.y & m), __vmaxu2(r[1].u.x & m, r[1].u.y & m));
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(a & 0xffffu, a >> 16))));
}
__device__ __forceinline__ uint32_t magnitude(const Raw4<float> (&r)[2]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    a = max(max(a, max(__float_as_uint(r[i].u.x) & 0x7fffffffu, __float_as_uint(r[i].u.y) & 0x7fffffffu)),
            max(__float_as_uint(r[i].u.z) & 0x7fffffffu, __float_as_uint(r[i].u.w) & 0x7fffffffu));
  return a;
}

// D/8 lanes take a row of K and the same row of V, 8 elements each; 4 lanes share a block of 32.  U tokens a group, all requested before the
// first is worked on, and before the page table has answered.
template <typename T, int ELEM, int LANES, int U>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ mpsa_kv_append_args a) {
  constexpr int D = 8 * LANES, NB = D / 32, kRows = kThreads / LANES;
  const int j = threadIdx.x % LANES, h = blockIdx.y, b = blockIdx.z;
  const int t0 = blockIdx.x * (kRows * U) + threadIdx.x / LANES;
  const mpsa_kv_cache& c = a.cache;
  grid_dependency_wait();
  grid_dependents_go();
  const T* const k = static_cast<const T*>(a.k) + b * a.k_sb + h * a.k_sh + 8 * j;
  const T* const v = static_cast<const T*>(a.v) + b * a.v_sb + h * a.v_sh + 8 * j;
  Raw4<T> raw[U][2][2] = {};
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * kRows;
    if (t < a.T) {
      raw[i][0][0] = raw4(k + t * a.k_sl);
      raw[i][0][1] = raw4(k + t * a.k_sl + 4);
      raw[i][1][0] = raw4(v + t * a.v_sl);
      raw[i][1][1] = raw4(v + t * a.v_sl + 4);
    }
  }
  const int n = a.counts ? min(a.counts[b], a.T) : a.T;
  const long long start = a.start[b];
  const int shift = __popc(c.page_size - 1);
  int page[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const long long pos = start + t0 + i * kRows;
    page[i] = t0 + i * kRows < n && pos >= 0 && pos < (1ll << 31) ? page_of(a.page_table + b * a.table_sb, (int)pos >> shift, a.max_pages, c.num_pages) : -1;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const long long row = (((long long)max(page[i], 0) * c.Hkv + h) << shift) + ((start + t0 + i * kRows) & (c.page_size - 1));
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      uint32_t amax = page[i] >= 0 ? magnitude(raw[i][o]) : 0u;
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const bool fine = amax < 0x7f800000u;
      const int s = fine ? block_exponent<ELEM>(amax) : 128;
      const float r = __uint_as_float((uint32_t)(127 - s) << 23);  // exact: s is -126 .. 126
      float lo[4], hi[4], x[8];
      wide4(raw[i][o][0], lo);
      wide4(raw[i][o][1], hi);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = lo[e] * r, x[4 + e] = hi[e] * r;
      if (page[i] >= 0) {
        store_codes<ELEM>(static_cast<uint8_t*>(o ? c.v : c.k) + row * code_bytes(ELEM, D) + code_bytes(ELEM, 8 * j), x, fine);
        if (j % 4 == 0) static_cast<uint8_t*>(o ? c.v_scale : c.k_scale)[row * NB + j / 4] = (uint8_t)(s + 127);
      }
    }
  }
}

// Eight codes
template <int ELEM> struct alignas(ELEM == E2M1 ? 4 : 8) Codes { uint32_t w[ELEM == E2M1 ? 1 : 2]; };
template <int ELEM>
__device__ __forceinline__ void read_codes(const Codes<ELEM>& c, float (&lo)[4], float (&hi)[4]) {
  uint32_t r[4];
  if constexpr (ELEM == E2M1) {
    elem_quads(c.w[0], r[0], r[1], r[2], r[3]);
  } else {
    elem_two<ELEM>(c.w[0], r[0], r[1]);
    elem_two<ELEM>(c.w[1], r[2], r[3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
    (i < 2 ? lo : hi)[2 * (i % 2)] = f.x;
    (i < 2 ? lo : hi)[2 * (i % 2) + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&lo)[4], const float (&hi)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(T(), lo[0], lo[1]), pack2(T(), lo[2], lo[3]), pack2(T(), hi[0], hi[1]), pack2(T(), hi[2], hi[3]));
}
__device__ __forceinline__ void store8(float* p, const float (&lo)[4], const float (&hi)[4]) {
  store4(p, lo);
  store4(p + 4, hi);
}

template <typename T, int ELEM, int LANES, int U>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ mpsa_kv_read_args a) {
  constexpr int D = 8 * LANES, NB = D / 32, kRows = kThreads / LANES;
  const int j = threadIdx.x % LANES, h = blockIdx.y, b = blockIdx.z;
  const int t0 = blockIdx.x * (kRows * U) + threadIdx.x / LANES;
  const mpsa_kv_cache& c = a.cache;
  grid_dependency_wait();
  grid_dependents_go();
  const int n = min(a.lengths[b], a.max_len), shift = __popc(c.page_size - 1);
  Codes<ELEM> code[U][2];
  uint32_t scale[U][2];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * kRows;
    const int page = t < n ? page_of(a.page_table + b * a.table_sb, t >> shift, a.max_pages, c.num_pages) : -1;
    const long long row = (((long long)max(page, 0) * c.Hkv + h) << shift) + (t & (c.page_size - 1));
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      code[i][o] = {};
      scale[i][o] = 0;
      if (page >= 0) {
        code[i][o] = *reinterpret_cast<const Codes<ELEM>*>(static_cast<const uint8_t*>(o ? c.v : c.k) + row * code_bytes(ELEM, D) + code_bytes(ELEM, 8 * j));
        scale[i][o] = static_cast<const uint8_t*>(o ? c.v_scale : c.k_scale)[row * NB + j / 4];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * kRows;
    if (t >= a.max_len) return;
    const long long to = (((long long)b * c.Hkv + h) * a.max_len + t) * D + 8 * j;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      float lo[4], hi[4];
      read_codes<ELEM>(code[i][o], lo, hi);
      const float s = scale_value(scale[i][o]);
#pragma unroll
      for (int e = 0; e < 4; ++e) lo[e] *= s, hi[e] *= s;
      T* y = static_cast<T*>(o ? a.v_out : a.k_out) + to;
      store8(y, lo, hi);
    }
  }
}

// Tokens of a lane group, where there are enough of them for eight CTAs an SM.  2 x 4099 tokens of 8 heads appended, calls back to back: 12.7 us
// with two, 13.4 with four; prefixes of 4 x 8192 read 35.2 us with one, two or four.
constexpr int kAppendRows = 2, kReadRows = 2;

template <typename T, int ELEM, int LANES>
void append_lanes(const mpsa_kv_append_args& a, cudaStream_t st) {
  constexpr int rows = kThreads / LANES;
  const bool many = (long long)a.T * a.cache.Hkv * a.B > 8ll * kAppendRows * rows * sm_count();
  const int per = many ? kAppendRows * rows : rows;
  const dim3 grid((a.T + per - 1) / per, a.cache.Hkv, a.B);
  const auto kernel = many ? kv_append_kernel<T, ELEM, LANES, kAppendRows> : kv_append_kernel<T, ELEM, LANES, 1>;
  launch_dependent(kernel, grid, kThreads, 0, st, overlaps_previous(st), a);
}
template <typename T, int ELEM>
int append_as(const mpsa_kv_append_args& a, cudaStream_t st) {
  if (a.cache.D == 64) append_lanes<T, ELEM, 8>(a, st);
  else append_lanes<T, ELEM, 16>(a, st);
  return check_launch("kv_append");
}
template <typename T>
int append_elem(const mpsa_kv_append_args& a, cudaStream_t st) {
  return a.cache.elem == E4M3 ? append_as<T, E4M3>(a, st) : a.cache.elem == E5M2 ? append_as<T, E5M2>(a, st) : append_as<T, E2M1>(a, st);
}

template <typename T, int ELEM>
int read_as(const mpsa_kv_read_args& a, cudaStream_t st) {
  const int rows = kThreads / (a.cache.D / 8) * kReadRows;
  const dim3 grid((a.max_len + rows - 1) / rows, a.cache.Hkv, a.B);
  const auto kernel = a.cache.D == 64 ? kv_read_kernel<T, ELEM, 8, kReadRows> : kv_read_kernel<T, ELEM, 16, kReadRows>;
  launch_dependent(kernel, grid, kThreads, 0, st, overlaps_previous(st), a);
  return check_launch("kv_read");
}
template <typename T>
int read_elem(const mpsa_kv_read_args& a, cudaStream_t st) {
  return a.cache.elem == E4M3 ? read_as<T, E4M3>(a, st) : a.cache.elem == E5M2 ? read_as<T, E5M2>(a, st) : read_as<T, E2M1>(a, st);
}

}  // namespace
}  // namespace mpsa

using namespace mpsa;

extern "C" int mpsa_kv_append(const mpsa_kv_append_args* a, void* stream) {
  if (!a || !a->k || !a->v || !a->page_table || !a->start) return set_error(MPSA_ERR_BAD_ARG, "kv_append: null pointer");
  if (int rc = check_cache(a->cache, "kv_append")) return rc;
  if (a->in_dtype < 0 || a->in_dtype > 2) return set_error(MPSA_ERR_UNSUPPORTED, "kv_append: inputs must be bf16, fp16 or fp32");
  if (a->B <= 0 || a->T <= 0 || a->max_pages <= 0) return set_error(MPSA_ERR_BAD_ARG, "kv_append: non-positive shape");
  if (a->B > 65535) return set_error(MPSA_ERR_UNSUPPORTED, "kv_append: at most 65535 sequences");
  if ((a->k_sb | a->k_sh | a->k_sl | a->v_sb | a->v_sh | a->v_sl) % 8 || ((uintptr_t)a->k | (uintptr_t)a->v) % 16)
    return set_error(MPSA_ERR_UNSUPPORTED, "kv_append: k and v need 16-byte aligned bases and strides that are multiples of 8 elements");
  const cudaStream_t st = (cudaStream_t)stream;
  return a->in_dtype == 0 ? append_elem<__nv_bfloat16>(*a, st) : a->in_dtype == 1 ? append_elem<__half>(*a, st) : append_elem<float>(*a, st);
}

extern "C" int mpsa_kv_read(const mpsa_kv_read_args* a, void* stream) {
  if (!a || !a->k_out || !a->v_out || !a->page_table || !a->lengths) return set_error(MPSA_ERR_BAD_ARG, "kv_read: null pointer");
  if (int rc = check_cache(a->cache, "kv_read")) return rc;
  if (a->out_dtype < 0 || a->out_dtype > 2) return set_error(MPSA_ERR_UNSUPPORTED, "kv_read: outputs are fp32, fp16 or bf16");
  if (a->B <= 0 || a->max_len <= 0 || a->max_pages <= 0) return set_error(MPSA_ERR_BAD_ARG, "kv_read: non-positive shape");
  if (a->B > 65535) return set_error(MPSA_ERR_UNSUPPORTED, "kv_read: at most 65535 sequences");
  if (((uintptr_t)a->k_out | (uintptr_t)a->v_out) % 16) return set_error(MPSA_ERR_BAD_ARG, "kv_read: outputs must be 16-byte aligned");
  const cudaStream_t st = (cudaStream_t)stream;
  return a->out_dtype == 0 ? read_elem<float>(*a, st) : a->out_dtype == 1 ? read_elem<__half>(*a, st) : read_elem<__nv_bfloat16>(*a, st);
}
