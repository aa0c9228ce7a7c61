// RMS norm of queries and keys and their rotation by position in one pass (mpsa_norm_rope): every element is read once and written once.
// Bound by HBM: 40 heads of 32768 tokens, each head's norm, 120 us (5.7 TB/s); 80 heads of 32760 tokens, norm across 40 heads, three axes,
// 276 - 289 us by box (4.6 - 4.9 TB/s, issue 71 %).  A decoding step of 32 sequences takes the host's 7.8 us.
#include "api_internal.h"
#include "common.cuh"
#include "serving.cuh"

namespace mpsa {
namespace {

constexpr int kThreads = 256, kMaxAxes = 4;

struct NormRope : mpsa_norm_rope_args {
  int heads_per_cta;            // norm 0 / 1: heads of one CTA, of the H[0] + H[1] in a row
};

// 4 weights at i, a multiple of 4
template <typename W>
__device__ __forceinline__ void weights4(const void* w, int i, float (&x)[4]) {
  if (w) load4(static_cast<const W*>(w) + i, x);
  else x[0] = x[1] = x[2] = x[3] = 1.0f;
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

// The table's rows for the axes of token (b, l); false: a position outside it.
__device__ __forceinline__ bool positions_of(const NormRope& a, int b, int l, long long (&pos)[kMaxAxes]) {
  if (!a.positions) {
    pos[0] = l;
    return l < a.table_rows;
  }
  bool there = true;
  const long long at = b * a.pos_sb + (long long)l * a.axes;
#pragma unroll
  for (int i = 0; i < kMaxAxes; ++i)
    if (i < a.axes) {
      pos[i] = a.pos64 ? static_cast<const long long*>(a.positions)[at + i] : static_cast<const int*>(a.positions)[at + i];
      there = there && pos[i] >= 0 && pos[i] < a.table_rows;
    }
  return there;
}
__device__ __forceinline__ long long row_of_pair(const NormRope& a, const long long (&pos)[kMaxAxes], int pair) {
  long long row = pos[0];
#pragma unroll
  for (int x = 1; x < kMaxAxes; ++x)
    if (x < a.axes && pair >= a.section_end[x - 1]) row = pos[x];
  return row;
}

// Cosines and sines of a lane's four pairs for token (b, l).
__device__ __forceinline__ void angles(const NormRope& a, int b, int l, int j, float (&c)[4], float (&s)[4]) {
  const float *cos = static_cast<const float*>(a.cos), *sin = static_cast<const float*>(a.sin);
  const int half = a.rot / 2;
  long long pos[kMaxAxes] = {};
  if (!positions_of(a, b, l, pos)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
  } else if (a.axes == 1) {
    load4(cos + pos[0] * half + 4 * j, c);
    load4(sin + pos[0] * half + 4 * j, s);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long at = row_of_pair(a, pos, 4 * j + i) * half + 4 * j + i;
      c[i] = cos[at];
      s[i] = sin[at];
    }
  }
}

template <bool INTERLEAVED>
__device__ __forceinline__ void turn(float (&u)[4], float (&v)[4], const float (&c)[4], const float (&s)[4]) {
  if constexpr (INTERLEAVED) {
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

// Norm of each head, or none: D/8 lanes hold a row; they keep the token's angles for all of the CTA's heads, and the operand's weights.
// kAhead rows are requested before the first is worked on.  Few heads a CTA where there are few tokens, all of them otherwise: four CTAs for a
// token's 40 heads instead of one read its angles four times and took 154 us instead of 120.
constexpr int kAhead = 4;
template <typename T, typename W, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 4) norm_rope_heads_kernel(const __grid_constant__ NormRope a) {
  const int j = threadIdx.x % LANES;
  const long long n = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = n < (long long)a.B * a.L;
  const int b = live ? (int)(n / a.L) : 0, l = live ? (int)(n % a.L) : 0;
  const Place p = place(j, a.cos ? a.rot : 0, INTERLEAVED);
  grid_dependency_wait();
  grid_dependents_go();
  float c[4] = {1, 1, 1, 1}, s[4] = {};
  if (p.turned) angles(a, b, l, j, c, s);
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int before = o ? a.H[0] : 0;
    const int first = max((int)blockIdx.y * a.heads_per_cta - before, 0), last = min(((int)blockIdx.y + 1) * a.heads_per_cta - before, a.H[o]);
    if (first >= last) continue;
    float w0[4], w1[4];
    weights4<W>(a.weight[o], p.at[0], w0);
    weights4<W>(a.weight[o], p.at[1], w1);
    const long long xh = a.x_sh[o], yh = a.y_sh[o];
    const T* x = static_cast<const T*>(a.x[o]) + (b * a.x_sb[o] + l * a.x_sl[o] + first * xh);
    T* y = static_cast<T*>(a.y[o]) + (b * a.y_sb[o] + l * a.y_sl[o] + first * yh);
    for (int h = first; h < last; h += kAhead) {
      Raw4<T> r[kAhead][2];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        r[k][0] = raw4(x + p.at[0]);
        r[k][1] = raw4(x + p.at[1]);
        if (h + k + 1 < last) x += xh;                               // (the last row again, behind the last)
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        float u[4], v[4];
        wide4(r[k][0], u);
        wide4(r[k][1], v);
        if (a.norm) {
          float q = squares(u, v);
#pragma unroll
          for (int d = LANES / 2; d; d /= 2) q += __shfl_xor_sync(0xffffffffu, q, d);
          const float n = rsqrtf(q * (1.0f / (8 * LANES)) + a.eps);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u[i] *= n * w0[i];
            v[i] *= n * w1[i];
          }
        }
        if (p.turned) turn<INTERLEAVED>(u, v, c, s);
        if (live && h + k < last) {
          store4(y + p.at[0], u);
          store4(y + p.at[1], v);
          y += yh;
        }
      }
    }
  }
}

// Norm across the heads of a token: a CTA takes one token of one operand, up to kChunks x 8 elements a thread, all in registers between the
// sum and the rest.  Few threads a token and many CTAs an SM: the others' loads run under one's barrier.
constexpr int kChunks = 8;
template <typename T, typename W, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 3) norm_rope_across_kernel(const __grid_constant__ NormRope a) {
  __shared__ float part[16];
  __shared__ __align__(16) float angle[2][4 * LANES];
  const int o = blockIdx.y, H = a.H[o];
  const int b = blockIdx.x / a.L, l = blockIdx.x % a.L;
  const int j = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = blockDim.x / LANES, warps = blockDim.x / 32;
  const Place p = place(j, a.cos ? a.rot : 0, INTERLEAVED);
  const T* x = static_cast<const T*>(a.x[o]) + (b * a.x_sb[o] + l * a.x_sl[o] + group * a.x_sh[o]);
  T* y = static_cast<T*>(a.y[o]) + (b * a.y_sb[o] + l * a.y_sl[o] + group * a.y_sh[o]);
  const long long xh = groups * a.x_sh[o], yh = groups * a.y_sh[o];
  grid_dependency_wait();
  grid_dependents_go();
  Raw4<T> r0[kChunks], r1[kChunks];
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    r0[k] = {}, r1[k] = {};
    if (k * groups + group < H) {
      r0[k] = raw4(x + p.at[0]);
      r1[k] = raw4(x + p.at[1]);
    }
    x += xh;
  }
  if (a.cos) {
    const int half = a.rot / 2;
    long long pos[kMaxAxes] = {};
    const bool there = positions_of(a, b, l, pos);
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
      const long long at = there ? row_of_pair(a, pos, i) * half + i : 0;
      angle[0][i] = there ? static_cast<const float*>(a.cos)[at] : __int_as_float(0x7fffffff);
      angle[1][i] = there ? static_cast<const float*>(a.sin)[at] : __int_as_float(0x7fffffff);
    }
  }
  float q = 0.0f;
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    float u[4], v[4];
    wide4(r0[k], u);
    wide4(r1[k], v);
    q += squares(u, v);
  }
#pragma unroll
  for (int d = 16; d; d /= 2) q += __shfl_xor_sync(0xffffffffu, q, d);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = q;
  __syncthreads();
  q = (int)(threadIdx.x % 16) < warps ? part[threadIdx.x % 16] : 0.0f;
#pragma unroll
  for (int d = 8; d; d /= 2) q += __shfl_xor_sync(0xffffffffu, q, d);
  const float r = rsqrtf(q / (float)(H * 8 * LANES) + a.eps);
  float c[4] = {1, 1, 1, 1}, s[4] = {};
  if (p.turned) {
    load4(&angle[0][4 * j], c);
    load4(&angle[1][4 * j], s);
  }
  const W* wp = static_cast<const W*>(a.weight[o]) + group * 8 * LANES;
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    if (k * groups + group >= H) return;
    float u[4], v[4], w0[4] = {1, 1, 1, 1}, w1[4] = {1, 1, 1, 1};
    if (a.weight[o]) {
      load4(wp + p.at[0], w0);
      load4(wp + p.at[1], w1);
      wp += groups * 8 * LANES;
    }
    wide4(r0[k], u);
    wide4(r1[k], v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] *= r * w0[i];
      v[i] *= r * w1[i];
    }
    if (p.turned) turn<INTERLEAVED>(u, v, c, s);
    store4(y + p.at[0], u);
    store4(y + p.at[1], v);
    y += yh;
  }
}

template <typename T, typename W, int LANES, bool INTERLEAVED>
int launch(NormRope& a, cudaStream_t st) {
  const long long tokens = (long long)a.B * a.L;
  const int heads = a.H[0] + a.H[1];
  if (a.norm == 2) {
    const int most = a.H[0] > a.H[1] ? a.H[0] : a.H[1];
    const int threads = (most * LANES + 32 * kChunks - 1) / (32 * kChunks) * 32;
    const auto kernel = norm_rope_across_kernel<T, W, LANES, INTERLEAVED>;
    launch_dependent(kernel, dim3((unsigned)tokens, a.x[1] ? 2 : 1), threads, 0, st, overlaps_previous(st), a);
    return check_launch("norm_rope");
  }
  const long long groups = (tokens + kThreads / LANES - 1) / (kThreads / LANES);
  a.heads_per_cta = heads;                                           // split over CTAs where there are few tokens
  while (a.heads_per_cta > kAhead && groups * ((heads + a.heads_per_cta - 1) / a.heads_per_cta) < 8ll * sm_count()) a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const dim3 grid((unsigned)groups, (heads + a.heads_per_cta - 1) / a.heads_per_cta);
  const auto kernel = norm_rope_heads_kernel<T, W, LANES, INTERLEAVED>;
  launch_dependent(kernel, grid, kThreads, 0, st, overlaps_previous(st), a);
  return check_launch("norm_rope");
}
template <typename T, typename W>
int launch_depth(NormRope& a, cudaStream_t st) {
  if (a.D == 64) return a.interleaved ? launch<T, W, 8, true>(a, st) : launch<T, W, 8, false>(a, st);
  return a.interleaved ? launch<T, W, 16, true>(a, st) : launch<T, W, 16, false>(a, st);
}
template <typename T>
int launch_weights(NormRope& a, cudaStream_t st) {
  for (int o = 0; o < 2; ++o)
    if (a.weight[o] && a.w_dtype[o] == 2) return launch_depth<T, float>(a, st);
  return launch_depth<T, T>(a, st);
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
    if (a.weight[o] && a.w_dtype[o] != 2 && a.w_dtype[o] != a.in_dtype) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: weights must be fp32 or of the inputs' type");
    if ((uintptr_t)a.weight[o] % 16) return set_error(MPSA_ERR_UNSUPPORTED, "norm_rope: weights must be 16-byte aligned");
  }
  if (a.weight[0] && a.weight[1] && a.x[1] && a.w_dtype[0] != a.w_dtype[1]) return set_error(MPSA_ERR_BAD_ARG, "norm_rope: the weights must have one type");
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
  return a.in_dtype == 0 ? launch_weights<__nv_bfloat16>(a, st) : a.in_dtype == 1 ? launch_weights<__half>(a, st) : launch_weights<float>(a, st);
}
