// Attention of a sequence's last tokens over its paged MX cache (mpsa_kv_attention).
#include "api_internal.h"
#include "common.cuh"
#include "serving.cuh"

namespace mpsa {
namespace {

constexpr int kWarps = 4;

// One row of one query head a CTA; its warps take keys in turn, a lane D/32 elements of each, and every warp keeps a running maximum and sum.
template <typename T, int ELEM, int D>
__global__ void __launch_bounds__(32 * kWarps) kv_attention_kernel(const __grid_constant__ mpsa_kv_attention_args a) {
  constexpr int N = D / 32;
  const mpsa_kv_cache& c = a.cache;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int i = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, h = hq / (a.Hq / c.Hkv);
  const int len = min(max(a.lengths[b], 0), (int)min(0x7fffffffll, (long long)a.max_pages * c.page_size));
  const int ql = min(a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T, len), first = len - ql;
  const T* q = static_cast<const T*>(a.q) + b * a.q_sb + hq * a.q_sh + i * a.q_sl + lane * N;
  float x[N], o[N] = {}, m = -INFINITY, l = 0.0f;
  for (int e = 0; e < N; ++e) x[e] = (float)q[e] * a.sm_scale * 1.44269504f;
  for (int pos = warp; pos < len && i < ql; pos += kWarps) {
    const int j = pos - first;
    if (j >= 0 && !(a.mask ? a.mask[b * a.mask_sb + (long long)i * a.T + j] != 0 : j <= i)) continue;
    const int page = page_of(a.page_table + b * a.table_sb, pos / c.page_size, a.max_pages, c.num_pages);
    if (page < 0) continue;
    const long long row = ((long long)page * c.Hkv + h) * c.page_size + (pos & (c.page_size - 1));
    float kv[2][N];
    for (int s = 0; s < 2; ++s) {
      const uint8_t* p = static_cast<const uint8_t*>(s ? c.v : c.k) + row * code_bytes(ELEM, D);
      const float sc = scale_value(static_cast<const uint8_t*>(s ? c.v_scale : c.k_scale)[row * (D / 32) + lane * N / 32]);
      for (int e = 0; e < N; e += 2) {
        const uint32_t two = ELEM == E2M1 ? p[(lane * N + e) / 2] : *reinterpret_cast<const unsigned short*>(p + lane * N + e);
        const float2 f = __half22float2(elem_pair<ELEM>(two));
        kv[s][e] = f.x * sc;
        kv[s][e + 1] = f.y * sc;
      }
    }
    float s = 0.0f;
    for (int e = 0; e < N; ++e) s += x[e] * kv[0][e];
    for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float up = fmaxf(m, s), w = up == -INFINITY ? 1.0f : exp2f(m - up), p = exp2f(s - (up == -INFINITY ? 0.0f : up));
    m = up;
    l = l * w + p;
    for (int e = 0; e < N; ++e) o[e] = o[e] * w + p * kv[1][e];
  }
  __shared__ float part[kWarps][D], stat[kWarps][2];
  for (int e = 0; e < N; ++e) part[warp][lane * N + e] = o[e];
  if (lane == 0) stat[warp][0] = m, stat[warp][1] = l;
  __syncthreads();
  if (warp) return;
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stat[w][0]);
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int w = 0; w < kWarps; ++w) sum += stat[w][1] * exp2f(stat[w][0] - ref);
  T* y = static_cast<T*>(a.out) + b * a.o_sb + hq * a.o_sh + i * a.o_sl;
  for (int e = lane; e < D; e += 32) {
    float v = 0.0f;
    for (int w = 0; w < kWarps; ++w) v += part[w][e] * exp2f(stat[w][0] - ref);
    y[e] = (T)(sum == 0.0f ? 0.0f : v / sum);
  }
  if (a.lse && lane == 0) static_cast<float*>(a.lse)[((long long)b * a.Hq + hq) * a.T + i] = sum == 0.0f ? -INFINITY : top + log2f(sum);
}

template <typename T, int ELEM>
int launch(const mpsa_kv_attention_args& a, cudaStream_t st) {
  const dim3 grid(a.T, a.Hq, a.B);
  if (a.cache.D == 64) kv_attention_kernel<T, ELEM, 64><<<grid, 32 * kWarps, 0, st>>>(a);
  else kv_attention_kernel<T, ELEM, 128><<<grid, 32 * kWarps, 0, st>>>(a);
  return check_launch("kv_attention");
}
template <typename T>
int launch_elem(const mpsa_kv_attention_args& a, cudaStream_t st) {
  return a.cache.elem == E4M3 ? launch<T, E4M3>(a, st) : a.cache.elem == E5M2 ? launch<T, E5M2>(a, st) : launch<T, E2M1>(a, st);
}

int check(const mpsa_kv_attention_args* a) {
  if (!a || !a->page_table || !a->lengths) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: null pointer");
  if (int rc = check_cache(a->cache, "kv_attention")) return rc;
  if (a->dtype != 0 && a->dtype != 1) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: queries must be bf16 or fp16");
  if (a->B <= 0 || a->T <= 0 || a->Hq <= 0 || a->max_pages <= 0) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: non-positive shape");
  if (a->Hq % a->cache.Hkv) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: Hq must be a multiple of Hkv");
  if (a->B > 65535 || a->Hq > 65535 || a->T > 1024) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: at most 65535 sequences and 1024 query tokens");
  if (!(a->sm_scale > 0.0f) || a->sm_scale > 1e30f) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: sm_scale must be positive and finite");
  return MPSA_OK;
}

}  // namespace
}  // namespace mpsa

using namespace mpsa;

extern "C" long long mpsa_kv_attention_workspace(const mpsa_kv_attention_args* a) {
  if (int rc = check(a)) return rc;
  return 0;
}

extern "C" int mpsa_kv_attention(const mpsa_kv_attention_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (!a->q || !a->out) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: null pointer");
  if ((a->q_sb | a->q_sh | a->q_sl | a->o_sb | a->o_sh | a->o_sl) % 8 || ((uintptr_t)a->q | (uintptr_t)a->out) % 16)
    return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: q and out need 16-byte aligned bases and strides that are multiples of 8 elements");
  const cudaStream_t st = (cudaStream_t)stream;
  return a->dtype == 0 ? launch_elem<__nv_bfloat16>(*a, st) : launch_elem<__half>(*a, st);
}
