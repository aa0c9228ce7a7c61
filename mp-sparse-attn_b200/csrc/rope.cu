// RMS norm of queries and keys and their rotation by position in one pass (mpsa_norm_rope): every element is read once and written once.
#include "api_internal.h"
#include "common.cuh"
#include "serving.cuh"

namespace mpsa {
namespace {

constexpr int kThreads = 256, kMaxAxes = 4;

struct NormRope : mpsa_norm_rope_args {
  int heads_per_cta;            // norm 0 / 1: heads of one CTA, of the H[0] + H[1] in a row
};

__device__ __forceinline__ float weight_at(const void* w, int type, int i) {
  return type == 2 ? static_cast<const float*>(w)[i]
                   : type == 1 ? __half2float(static_cast<const __half*>(w)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// A lane holds 8 elements of a row as two runs of 4: where rotated pairs lie half the rotated width apart, 4 of each half, so that both
// elements of a pair are in one lane; otherwise 8 neighbours.  In both forms the lane's pairs are 4j .. 4j+3.
struct Place {
  int at[2];
  bool turned;
};
__device__ __forceinline__ Place place(int j, int rot, bool interleaved) {
  if (8 * j >= rot) return {{8 * j, 8 * j + 4}, false};
  if (interleaved) return {{8 * j, 8 * j + 4}, true};
  return {{4 * j, rot / 2 + 4 * j}, true};
}

// Cosines and sines of the lane's four pairs for token (b, l).
__device__ __forceinline__ void angles(const NormRope& a, int b, int l, int j, float (&c)[4], float (&s)[4]) {
  const float *cos = static_cast<const float*>(a.cos), *sin = static_cast<const float*>(a.sin);
  const int half = a.rot / 2;
  bool there = true;
  long long row[4];
  if (!a.positions) {
    row[0] = row[1] = row[2] = row[3] = l;
    there = l < a.table_rows;
  } else {
    long long pos[kMaxAxes] = {};
    const long long at = b * a.pos_sb + (long long)l * a.axes;
#pragma unroll
    for (int i = 0; i < kMaxAxes; ++i)
      if (i < a.axes) {
        pos[i] = a.pos64 ? static_cast<const long long*>(a.positions)[at + i] : static_cast<const int*>(a.positions)[at + i];
        there = there && pos[i] >= 0 && pos[i] < a.table_rows;
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row[i] = pos[0];
#pragma unroll
      for (int x = 1; x < kMaxAxes; ++x)
        if (x < a.axes && 4 * j + i >= a.section_end[x - 1]) row[i] = pos[x];
    }
  }
  if (!there) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
  } else if (a.axes == 1) {
    load4(cos + row[0] * half + 4 * j, c);
    load4(sin + row[0] * half + 4 * j, s);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = cos[row[i] * half + 4 * j + i];
      s[i] = sin[row[i] * half + 4 * j + i];
    }
  }
}

__device__ __forceinline__ void turn(float (&u)[4], float (&v)[4], const float (&c)[4], const float (&s)[4], bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float a = u[2 * i], b = u[2 * i + 1], d = v[2 * i], e = v[2 * i + 1];
      u[2 * i] = a * c[i] - b * s[i];
      u[2 * i + 1] = b * c[i] + a * s[i];
      v[2 * i] = d * c[i + 2] - e * s[i + 2];
      v[2 * i + 1] = e * c[i + 2] + d * s[i + 2];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = u[i], b = v[i];
      u[i] = a * c[i] - b * s[i];
      v[i] = b * c[i] + a * s[i];
    }
  }
}

__device__ __forceinline__ float squares(const float (&u)[4], const float (&v)[4]) {
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q += u[i] * u[i] + v[i] * v[i];
  return q;
}

// Norm of each head, or none: D/8 lanes hold a row; they keep the token's angles for all of the CTA's heads.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) norm_rope_heads_kernel(const __grid_constant__ NormRope a) {
  const int j = threadIdx.x % LANES;
  const long long n = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = n < (long long)a.B * a.L;
  const int b = live ? (int)(n / a.L) : 0, l = live ? (int)(n % a.L) : 0;
  const Place p = place(j, a.cos ? a.rot : 0, a.interleaved);
  float c[4], s[4], w[2][8];
  if (p.turned) angles(a, b, l, j, c, s);
#pragma unroll
  for (int o = 0; o < 2; ++o)
#pragma unroll
    for (int i = 0; i < 8; ++i) w[o][i] = a.weight[o] ? weight_at(a.weight[o], a.w_dtype[o], p.at[i / 4] + i % 4) : 1.0f;
  const int first = blockIdx.y * a.heads_per_cta, last = min(first + a.heads_per_cta, a.H[0] + a.H[1]);
#pragma unroll 2
  for (int h = first; h < last; ++h) {
    const int o = h >= a.H[0], head = o ? h - a.H[0] : h;
    const T* x = static_cast<const T*>(o ? a.x[1] : a.x[0]) + (b * (o ? a.x_sb[1] : a.x_sb[0]) + head * (o ? a.x_sh[1] : a.x_sh[0]) + l * (o ? a.x_sl[1] : a.x_sl[0]));
    T* y = static_cast<T*>(o ? a.y[1] : a.y[0]) + (b * (o ? a.y_sb[1] : a.y_sb[0]) + head * (o ? a.y_sh[1] : a.y_sh[0]) + l * (o ? a.y_sl[1] : a.y_sl[0]));
    float u[4], v[4];
    load4(x + p.at[0], u);
    load4(x + p.at[1], v);
    if (a.norm) {
      float q = squares(u, v);
#pragma unroll
      for (int d = LANES / 2; d; d /= 2) q += __shfl_xor_sync(0xffffffffu, q, d);
      const float r = 1.0f / sqrtf(q * (1.0f / (8 * LANES)) + a.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u[i] = u[i] * r * (o ? w[1][i] : w[0][i]);
        v[i] = v[i] * r * (o ? w[1][4 + i] : w[0][4 + i]);
      }
    }
    if (p.turned) turn(u, v, c, s, a.interleaved);
    if (live) {
      store4(y + p.at[0], u);
      store4(y + p.at[1], v);
    }
  }
}

// Norm across the heads of a token: a CTA holds one token of one operand in registers, CHUNKS x 8 elements a thread.
template <typename T, int LANES, int CHUNKS>
__global__ void norm_rope_across_kernel(const __grid_constant__ NormRope a) {
  __shared__ float part[32];
  const int o = blockIdx.y, H = a.H[o];
  const int b = blockIdx.x / a.L, l = blockIdx.x % a.L;
  const T* x = static_cast<const T*>(a.x[o]) + (b * a.x_sb[o] + l * a.x_sl[o]);
  T* y = static_cast<T*>(a.y[o]) + (b * a.y_sb[o] + l * a.y_sl[o]);
  const int j = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = blockDim.x / LANES;
  const Place p = place(j, a.cos ? a.rot : 0, a.interleaved);
  float u[CHUNKS][4], v[CHUNKS][4], q = 0.0f;
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    const int h = k * groups + group;
    if (h < H) {
      load4(x + h * a.x_sh[o] + p.at[0], u[k]);
      load4(x + h * a.x_sh[o] + p.at[1], v[k]);
      q += squares(u[k], v[k]);
    }
  }
  float c[4], s[4];
  if (p.turned) angles(a, b, l, j, c, s);
#pragma unroll
  for (int d = 16; d; d /= 2) q += __shfl_xor_sync(0xffffffffu, q, d);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = q;
  __syncthreads();
  q = 0.0f;
  for (int i = 0; i < (int)(blockDim.x / 32); ++i) q += part[i];
  const float r = 1.0f / sqrtf(q / (float)(H * 8 * LANES) + a.eps);
#pragma unroll
  for (int k = 0; k < CHUNKS; ++k) {
    const int h = k * groups + group;
    if (h >= H) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[k][i] *= r;
      v[k][i] *= r;
      if (a.weight[o]) {
        u[k][i] *= weight_at(a.weight[o], a.w_dtype[o], h * 8 * LANES + p.at[0] + i);
        v[k][i] *= weight_at(a.weight[o], a.w_dtype[o], h * 8 * LANES + p.at[1] + i);
      }
    }
    if (p.turned) turn(u[k], v[k], c, s, a.interleaved);
    store4(y + h * a.y_sh[o] + p.at[0], u[k]);
    store4(y + h * a.y_sh[o] + p.at[1], v[k]);
  }
}

template <typename T, int LANES>
int launch(NormRope& a, cudaStream_t st) {
  const long long tokens = (long long)a.B * a.L;
  const int heads = a.H[0] + a.H[1];
  if (a.norm == 2) {
    const int most = a.H[0] > a.H[1] ? a.H[0] : a.H[1];
    const dim3 grid((unsigned)tokens, a.x[1] ? 2 : 1);
    const int chunks = (most * LANES + 511) / 512;                   // of a thread, with 512 threads at most
    const int per = (most + chunks - 1) / chunks;
    const int threads = (per * LANES + 31) / 32 * 32;
    if (chunks == 1) norm_rope_across_kernel<T, LANES, 1><<<grid, threads, 0, st>>>(a);
    else if (chunks == 2) norm_rope_across_kernel<T, LANES, 2><<<grid, threads, 0, st>>>(a);
    else norm_rope_across_kernel<T, LANES, 4><<<grid, threads, 0, st>>>(a);
    return check_launch("norm_rope");
  }
  const long long groups = (tokens + kThreads / LANES - 1) / (kThreads / LANES);
  a.heads_per_cta = heads;                                           // split over CTAs where there are few tokens
  while (a.heads_per_cta > 1 && groups * ((heads + a.heads_per_cta - 1) / a.heads_per_cta) < 8ll * sm_count()) a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const dim3 grid((unsigned)groups, (heads + a.heads_per_cta - 1) / a.heads_per_cta);
  norm_rope_heads_kernel<T, LANES><<<grid, kThreads, 0, st>>>(a);
  return check_launch("norm_rope");
}

}  // namespace
}  // namespace mpsa

using namespace mpsa;

extern "C" int mpsa_norm_rope(const mpsa_norm_rope_args* args, void* stream) {
  if (!args || !args->x[0] || !args->y[0] || (args->x[1] && !args->y[1])) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: null pointer");
  NormRope a = {};
  static_cast<mpsa_norm_rope_args&>(a) = *args;
  if (!a.x[1]) a.H[1] = 0;
  if (a.in_dtype < 0 || a.in_dtype > 2) return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: inputs must be bf16, fp16 or fp32");
  if (a.D != 64 && a.D != 128) return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: D must be 64 or 128");
  if (a.B <= 0 || a.L <= 0 || a.H[0] <= 0 || a.H[1] < 0 || (a.x[1] && a.H[1] == 0)) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: non-positive shape");
  if ((long long)a.B * a.L > 0x7fffffffll || a.H[0] > 32768 || a.H[1] > 32768) return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: too many tokens or heads");
  if (a.norm < 0 || a.norm > 2) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: norm must be 0, 1 or 2");
  if (a.norm && !(a.eps >= 0.0f)) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: eps must not be negative");
  if (a.norm == 2 && (a.H[0] * a.D > 16384 || a.H[1] * a.D > 16384))
    return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: a norm across the heads takes at most 16384 elements a token");
  const int size = a.in_dtype == 2 ? 4 : 2;
  for (int o = 0; o < (a.x[1] ? 2 : 1); ++o) {
    if ((a.x_sb[o] | a.x_sh[o] | a.x_sl[o] | a.y_sb[o] | a.y_sh[o] | a.y_sl[o]) % 4 || (uintptr_t)a.x[o] % (4 * size) || (uintptr_t)a.y[o] % (4 * size))
      return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: bases and strides must be multiples of 4 elements");
    if (a.w_dtype[o] < 0 || a.w_dtype[o] > 2) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: weights must be bf16, fp16 or fp32");
  }
  if ((a.cos != nullptr) != (a.sin != nullptr)) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: cos and sin go together");
  if (a.cos) {
    if (a.rot <= 0 || a.rot % 8 || a.rot > a.D) return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: rot must be a multiple of 8, at most D");
    if (a.table_rows <= 0 || (uintptr_t)a.cos % 16 || (uintptr_t)a.sin % 16) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: cos and sin must be 16-byte aligned and have rows");
    if (a.axes < 1 || a.axes > kMaxAxes || (a.axes > 1 && !a.positions)) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: 1 to 4 axes, with positions where there are several");
    for (int i = 0, before = 0; a.axes > 1 && i < a.axes; before = a.section_end[i++])
      if (a.section_end[i] < before || (i == a.axes - 1 && a.section_end[i] != a.rot / 2))
        return set_error(MPSA_ERR_BAD_ARG, "norm_rope: sections must ascend and end at rot / 2");
  }
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.D == 64)
    return a.in_dtype == 0 ? launch<__nv_bfloat16, 8>(a, st) : a.in_dtype == 1 ? launch<__half, 8>(a, st) : launch<float, 8>(a, st);
  return a.in_dtype == 0 ? launch<__nv_bfloat16, 16>(a, st) : a.in_dtype == 1 ? launch<__half, 16>(a, st) : launch<float, 16>(a, st);
}
