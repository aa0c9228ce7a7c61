// Attention of a sequence's last tokens over its paged MX cache (mpsa_kv_attention).
//
// A unit of work is one sequence, one KV head and up to 16 of its query rows (row r = token r / G, query head r % G of the KV head's G).
// A step is 32 keys.  The steps of all units, laid end to end, are cut into equal runs, one per CTA, whatever the lengths are: CTAs compute
// the cut from the lengths in device memory.  A unit that falls to several CTAs leaves parts (fp32 sums with their row maxima and
// denominators), which the combining kernel adds up in the order of the keys.
//
// Within a CTA the warps take steps in turn and have nothing to do with each other until the run's part of a unit is done: each copies its own
// keys to its own shared memory with cp.async, and keeps its own maxima, sums and output in registers.
//
//   scores    S = Q K^T by m16n8k16 on fp16 operands.  Element codes convert exactly; a block's 32 depth elements are two instructions of
//             their own, whose fp32 result is multiplied by the key's scale of that block.  Queries are brought to a largest magnitude of
//             1 .. 2 by a power of two of their row, so that their 8 or 11 significant bits survive in fp16.
//   output    O = P V: the block scales of V differ from key to key, so they go to P: for each block of the depth P times the scales is
//             rounded to fp16 and multiplied by the codes.  The scales enter relative to the largest one so far, 2^15 above it at most: fp16
//             then keeps 11 bits down to 2^-29 of the largest product.  That rounding of P is the only one below fp32.
//
// It is bound by the cache's bytes (HBM) as long as the conversions keep up: two ALU-pipe instructions for two elements.
#include "api_internal.h"
#include "common.cuh"
#include "serving.cuh"

#include <type_traits>

namespace mpsa {
namespace {

constexpr int kWarps = 4, kStep = 32, kRows = 16;
constexpr int kMinShare = 4;                   // steps of a run at least: one for each warp

struct Call : mpsa_kv_attention_args {
  int groups;                                  // row groups of a (sequence, KV head)
  float* part;                                 // [2 x CTAs][kRows][D], a CTA's run has at most two units that it shares with others
  float2* stat;                                // [2 x CTAs][kRows]: row maximum (log2), denominator relative to it
};

__device__ __forceinline__ int length_of(const Call& a, int b) {
  return min(max(a.lengths[b], 0), (int)min(0x7fffffc0ll, (long long)a.max_pages * a.cache.page_size));
}
__device__ __forceinline__ int queries_of(const Call& a, int b, int len) { return min(a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T, len); }
__device__ __forceinline__ int steps_of(int len) { return max(1, (len + kStep - 1) / kStep); }    // (an empty sequence: one, which writes its zeros)

// The steps of all units, and how many a CTA of `ctas` takes.  By a whole warp.
__device__ long long share_of(const Call& a, int ctas, int lane) {
  long long sum = 0;
  for (int b = lane; b < a.B; b += 32) sum += steps_of(length_of(a, b));
#pragma unroll
  for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  sum *= a.cache.Hkv * a.groups;
  return max((sum + ctas - 1) / ctas, (long long)kMinShare);
}

// The sequence that step `at` of all steps belongs to (a.B: beyond the last), and where that sequence's steps begin.
__device__ int sequence_at(const Call& a, long long at, long long& begin, int lane) {
  const int units = a.cache.Hkv * a.groups;
  begin = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const long long n = b0 + lane < a.B ? (long long)steps_of(length_of(a, b0 + lane)) * units : 0;
    long long up = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const long long v = __shfl_up_sync(0xffffffffu, up, d);
      if (lane >= d) up += v;
    }
    const unsigned beyond = __ballot_sync(0xffffffffu, b0 + lane < a.B && begin + up > at);
    if (beyond) {
      const int l = __ffs(beyond) - 1;
      begin += __shfl_sync(0xffffffffu, up - n, l);
      return b0 + l;
    }
    begin += __shfl_sync(0xffffffffu, up, 31);
  }
  return a.B;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {       // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Shared memory of a warp: kStages steps of [K codes][V codes][K scales][V scales], then the step's scales as floats.
template <int ELEM, int D>
struct Layout {
  static constexpr int row = code_bytes(ELEM, D), nb = D / 32;
  static constexpr int codes = kStep * row, stage = 2 * codes + 2 * kStep * nb;
  static constexpr int stages = 2;
  static constexpr int scales = stages * stage, warp = scales + 2 * kStep * nb * 4;
  static constexpr int pitch = D + 4;                                  // floats of a row in the merge buffer
  static constexpr int merge = kWarps * kRows * pitch * 4;
  static constexpr int bytes = kWarps * warp > merge ? kWarps * warp : merge;
  // Where a row's block of 32 elements lies: blocks change places so that the lanes of a fragment load meet different banks.  K: 8 rows
  // at a time, V: rows 2t of the quarter.
  static constexpr int block = row / nb;                               // bytes
  static __device__ __forceinline__ int k_swap(int r) { return D == 64 ? (ELEM == E2M1 ? r >> 2 : r >> 1) & 1 : (ELEM == E2M1 ? r >> 1 : r) & 3; }
  static __device__ __forceinline__ int v_swap(int r) { return D == 64 ? (ELEM == E2M1 ? r >> 2 : r >> 1) & 1 : (r >> 1) & 3; }
};

// Eight codes of K (depth 8t .. 8t + 7 of a block), as the fp16 pairs of two instructions' B operands
template <int ELEM>
__device__ __forceinline__ void k_fragments(uint32_t p, uint32_t (&f)[4]) {
  if constexpr (ELEM == E2M1) {
    uint32_t w;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = bits(elem_pair<ELEM>(w >> (8 * i)));
  } else {
    uint32_t w[2];
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = bits(elem_pair<ELEM>(w[i / 2] >> (16 * (i % 2))));
  }
}

// Codes of V for depth 4g .. 4g + 3 of a block at two keys, as four fp16 pairs (one key in each half)
template <int ELEM>
__device__ __forceinline__ void v_fragments(uint32_t p0, uint32_t p1, int g, uint32_t (&f)[4]) {
  uint32_t x, y;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(p0));
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(y) : "r"(p1));
  if constexpr (ELEM == E2M1) {                      // the word holds eight depth elements: g odd takes its upper half
    const uint32_t w = __byte_perm(x, y, g & 1 ? 0x7632 : 0x5410);                 // x's four codes, y's four
    const uint32_t a = bits(elem_pair<ELEM>(w)), b = bits(elem_pair<ELEM>(w >> 8)), c = bits(elem_pair<ELEM>(w >> 16)), d = bits(elem_pair<ELEM>(w >> 24));
    f[0] = __byte_perm(a, c, 0x5410); f[1] = __byte_perm(a, c, 0x7632);
    f[2] = __byte_perm(b, d, 0x5410); f[3] = __byte_perm(b, d, 0x7632);
  } else {
    const uint32_t lo = __byte_perm(x, y, 0x5140), hi = __byte_perm(x, y, 0x7362);  // x0 y0 x1 y1, x2 y2 x3 y3
    f[0] = bits(elem_pair<ELEM>(lo)); f[1] = bits(elem_pair<ELEM>(lo >> 16));
    f[2] = bits(elem_pair<ELEM>(hi)); f[3] = bits(elem_pair<ELEM>(hi >> 16));
  }
}

// RH: halves of the 16 rows that are in use (1: at most 8 rows).
template <typename T, int ELEM, int D, int RH>
__global__ void __launch_bounds__(32 * kWarps, 3) kv_attention_kernel(const __grid_constant__ Call a) {
  using Y = Layout<ELEM, D>;
  constexpr int NB = D / 32, NT = kStep / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 row_stat[kWarps][kRows];
  const mpsa_kv_cache& c = a.cache;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring = smem_u32(smem) + warp * Y::warp;
  float* const ksc = reinterpret_cast<float*>(smem + warp * Y::warp + Y::scales);
  float* const vsc = ksc + kStep * NB;
  const int G = a.Hq / c.Hkv, R = a.T * G, units = c.Hkv * a.groups;

  grid_dependents_go();
  const long long share = share_of(a, gridDim.x, lane);
  long long at = blockIdx.x * share;
  const long long stop = at + share;
  long long begin;
  int b = sequence_at(a, at, begin, lane);
  bool first_run = true;
  for (; b < a.B && at < stop;) {
    const int len = length_of(a, b), steps = steps_of(len);
    const long long off = at - begin;
    const int u = (int)(off / steps), s0 = (int)(off % steps), s1 = (int)min((long long)steps, s0 + (stop - at));
    const int h = u / a.groups, row0 = u % a.groups * kRows;
    const int ql = queries_of(a, b, len), first = len - ql;
    const int* const table = a.page_table + b * a.table_sb;
    if (!first_run) __syncthreads();                  // (the merge buffer has been read)
    first_run = false;

    // queries: this lane's rows g and g + 8, depth 8t .. 8t + 7 of every block
    uint32_t qf[NB][RH][4];
    float rs[RH];
    int token[RH];
#pragma unroll
    for (int x = 0; x < RH; ++x) {
      const int r = row0 + g + 8 * x;
      token[x] = r < R ? r / G : -1;
      float q[NB][8];
      uint32_t amax = 0;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        if (r < R) {
          const T* p = static_cast<const T*>(a.q) + (b * a.q_sb + (h * G + r % G) * a.q_sh + token[x] * a.q_sl + 32 * k + 8 * t);
          float lo[4], hi[4];
          load4(p, lo);
          load4(p + 4, hi);
#pragma unroll
          for (int e = 0; e < 4; ++e) q[k][e] = lo[e], q[k][4 + e] = hi[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[k][e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(q[k][e]) & 0x7fffffffu);
      }
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = min(max((int)(amax >> 23), 1), 253);              // biased exponent of the row
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      rs[x] = amax >= 0x7f800000u ? __int_as_float(0x7fffffff) : a.sm_scale * 1.44269504f * __uint_as_float((uint32_t)e << 23);
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[k][x][i] = pack2(__half(), q[k][2 * i] * down, q[k][2 * i + 1] * down);
    }

    float o[NB][4][4] = {}, m[RH], l[RH];
#pragma unroll
    for (int x = 0; x < RH; ++x) m[x] = -INFINITY, l[x] = 0.0f;
    int vref = 0;                                     // largest scale code of V so far

    // pages: a lane holds one of the warp's next 16 steps' two (16 keys each)
    const int mine = (s1 - s0 - warp + kWarps - 1) / kWarps;          // steps of this warp (may be negative)
    auto look_up = [&](int k0) {
      const int s = s0 + warp + (k0 + lane / 2) * kWarps;
      return k0 + lane / 2 < mine ? page_of(table, (kStep * s + 16 * (lane & 1)) / c.page_size, a.max_pages, c.num_pages) : -1;
    };
    int pages = look_up(0), pages_next = -1;

    auto request = [&](int k, int p0, int p1) {
      const int s = s0 + warp + k * kWarps, pos = kStep * s;
      const uint32_t to = ring + k % Y::stages * Y::stage;
      const int pg[2] = {p0, p1};
      constexpr int CPR = Y::row / 16, RPI = 32 / CPR;                // 16-byte pieces of a row, rows of one instruction
      const int rl = lane / CPR, ch = lane % CPR;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const long long row = ((long long)max(pg[half], 0) * c.Hkv + h) * c.page_size + ((pos + 16 * half) & (c.page_size - 1));
        const uint8_t* kp = static_cast<const uint8_t*>(c.k) + row * Y::row + lane * 16;
        const uint8_t* vp = static_cast<const uint8_t*>(c.v) + row * Y::row + lane * 16;
#pragma unroll
        for (int i = 0; i < CPR / 2; ++i) {
          const int r = 16 * half + i * RPI + rl;
          const bool there = pg[half] >= 0 && pos + r < len;
          constexpr int per = Y::block / 16;                          // pieces of a block: 2 (8 bits) or 1
          const int kd = ((ch / per) ^ Y::k_swap(r)) * Y::block + ch % per * 16, vd = ((ch / per) ^ Y::v_swap(r)) * Y::block + ch % per * 16;
          copy16(to + r * Y::row + kd, kp + i * 512, there);
          copy16(to + Y::codes + r * Y::row + vd, vp + i * 512, there);
        }
      }
      constexpr int SP = 16 * NB / 16;                                // 16-byte pieces of 16 keys' scales
      if (lane < 4 * SP) {
        const int half = lane / SP % 2, v = lane / (2 * SP);
        const int p = half ? p1 : p0;
        const long long row = ((long long)max(p, 0) * c.Hkv + h) * c.page_size + ((pos + 16 * half) & (c.page_size - 1));
        copy16(to + 2 * Y::codes + lane * 16, static_cast<const uint8_t*>(v ? c.v_scale : c.k_scale) + row * NB + lane % SP * 16, p >= 0);
      }
    };
    auto page = [&](int k, int half) { return __shfl_sync(0xffffffffu, pages, 2 * (k % 16) + half); };

    int cur0 = page(0, 0), cur1 = page(0, 1);         // pages of step k
    if (mine > 0) request(0, cur0, cur1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int k = 0; k < mine; ++k) {
      int nx0 = -1, nx1 = -1;
      if (k + 1 < mine) {
        if ((k + 1) % 16 == 0) pages = pages_next;
        if ((k + 1) % 16 == 8) pages_next = look_up(k + 1 + 8);
        nx0 = page(k + 1, 0);
        nx1 = page(k + 1, 1);
        request(k + 1, nx0, nx1);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      const int pos = kStep * (s0 + warp + k * kWarps);
      const uint32_t buf = ring + k % Y::stages * Y::stage;
      const bool special = pos + kStep > (R > 1 && a.T > 1 || a.mask ? first : len) || cur0 < 0 || cur1 < 0;

      // scales of key `lane`, as floats for everybody
      {
        const bool there = pos + lane < len && (lane < 16 ? cur0 : cur1) >= 0;
        uint32_t kb, vb;
        if constexpr (NB == 4) {
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(kb) : "r"(buf + 2 * Y::codes + 4 * lane));
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(vb) : "r"(buf + 2 * Y::codes + kStep * NB + 4 * lane));
        } else {
          unsigned short x, y;
          asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x) : "r"(buf + 2 * Y::codes + 2 * lane));
          asm volatile("ld.shared.b16 %0, [%1];" : "=h"(y) : "r"(buf + 2 * Y::codes + kStep * NB + 2 * lane));
          kb = x;
          vb = y;
        }
        if (!there) kb = vb = 0;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const uint32_t e = vb >> (8 * i) & 255u;
          top = max(top, e == 255u ? 0u : e);
        }
        const int up = max((int)__reduce_max_sync(0xffffffffu, top), vref);
        if (up > vref) {                              // (for the whole warp)
          const int d = up - vref;
          const float f = d > 126 ? 0.0f : __uint_as_float((uint32_t)(127 - d) << 23);
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[i][j][e] *= f;
          vref = up;
        }
        float kf[NB], vf[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          kf[i] = scale_value(kb >> (8 * i) & 255u);
          const uint32_t e = vb >> (8 * i) & 255u;
          vf[i] = e == 255u ? __int_as_float(0x7fffffff) : e == 0u ? 0.0f : __uint_as_float((uint32_t)max((int)e - vref + 142, 0) << 23);
        }
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
          *reinterpret_cast<float2*>(ksc + lane * NB + i) = make_float2(kf[i], kf[i + 1]);
          *reinterpret_cast<float2*>(vsc + lane * NB + i) = make_float2(vf[i], vf[i + 1]);
        }
        __syncwarp();
      }

      // scores in log2 units: s[n][..] is row g, keys 8n + 2t and + 1, then row g + 8
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float k0[NB], k1[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          k0[i] = ksc[(8 * n + 2 * t) * NB + i];
          k1[i] = ksc[(8 * n + 2 * t + 1) * NB + i];
        }
        const int r = 8 * n + g;
        const uint32_t kp = buf + r * Y::row;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          uint32_t f[4];
          k_fragments<ELEM>(kp + (i ^ Y::k_swap(r)) * Y::block + t * (Y::block / 4), f);
          float d[4] = {};
          mma(d, qf[i][0][0], RH > 1 ? qf[i][RH - 1][0] : 0u, qf[i][0][1], RH > 1 ? qf[i][RH - 1][1] : 0u, f[0], f[1]);
          mma(d, qf[i][0][2], RH > 1 ? qf[i][RH - 1][2] : 0u, qf[i][0][3], RH > 1 ? qf[i][RH - 1][3] : 0u, f[2], f[3]);
#pragma unroll
          for (int x = 0; x < RH; ++x) {
            s[n][2 * x] = fmaf(d[2 * x], k0[i], s[n][2 * x]);
            s[n][2 * x + 1] = fmaf(d[2 * x + 1], k1[i], s[n][2 * x + 1]);
          }
        }
#pragma unroll
        for (int x = 0; x < RH; ++x) {
          s[n][2 * x] *= rs[x];
          s[n][2 * x + 1] *= rs[x];
        }
      }
      if (special) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int p = pos + 8 * n + 2 * t + e, j = p - first;
            const bool there = p < len && (n < 2 ? cur0 : cur1) >= 0;
#pragma unroll
            for (int x = 0; x < RH; ++x) {
              const bool seen = there && (j < 0 || (token[x] >= 0 && token[x] < ql && (a.mask ? a.mask[b * a.mask_sb + (long long)token[x] * a.T + j] != 0 : j <= token[x])));
              if (!seen) s[n][2 * x + e] = -INFINITY;
            }
          }
      }

      // running maxima, probabilities, sums
#pragma unroll
      for (int x = 0; x < RH; ++x) {
        float up = m[x];
#pragma unroll
        for (int n = 0; n < NT; ++n) up = fmaxf(up, fmaxf(s[n][2 * x], s[n][2 * x + 1]));
        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 1));
        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 2));
        const float ref = up == -INFINITY ? 0.0f : up;
        if (__any_sync(0xffffffffu, up > m[x])) {
          const float f = exp2_fast(m[x] - ref);
          l[x] *= f;
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[i][j][2 * x] *= f;
              o[i][j][2 * x + 1] *= f;
            }
          m[x] = up;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[n][2 * x] = exp2_fast(s[n][2 * x] - ref);
          s[n][2 * x + 1] = exp2_fast(s[n][2 * x + 1] - ref);
          l[x] += s[n][2 * x] + s[n][2 * x + 1];
        }
      }

      // O += P V, 16 keys at a time: keys 16w + 2t, + 1, + 8, + 9
#pragma unroll
      for (int w = 0; w < kStep / 16; ++w) {
        const int k0 = 16 * w + 2 * t;
        const uint32_t vp = buf + Y::codes;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const float v[4] = {vsc[k0 * NB + i], vsc[(k0 + 1) * NB + i], vsc[(k0 + 8) * NB + i], vsc[(k0 + 9) * NB + i]};
          float p[2][RH][2];
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < RH; ++x)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float q = s[2 * w + y][2 * x + e];
                p[y][x][e] = q * v[2 * y + e];
                if (special && q == 0.0f) p[y][x][e] = 0.0f;          // (a scale that is NaN, of a key that the row does not see)
              }
          const uint32_t a0 = pack2(__half(), p[0][0][0], p[0][0][1]), a2 = pack2(__half(), p[1][0][0], p[1][0][1]);
          const uint32_t a1 = RH > 1 ? pack2(__half(), p[0][RH - 1][0], p[0][RH - 1][1]) : 0u, a3 = RH > 1 ? pack2(__half(), p[1][RH - 1][0], p[1][RH - 1][1]) : 0u;
          uint32_t f[2][4];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int r = k0 + 8 * y;                                 // (rows r and r + 1 have their blocks in the same places)
            const uint32_t pl = vp + r * Y::row + (i ^ Y::v_swap(r)) * Y::block + (ELEM == E2M1 ? 4 * (g / 2) : 4 * g);
            v_fragments<ELEM>(pl, pl + Y::row, g, f[y]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) mma(o[i][j], a0, a1, a2, a3, f[0][j], f[1][j]);
        }
      }
      __syncwarp();                                   // the step's buffers are free
      cur0 = nx0;
      cur1 = nx1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // the warps' parts together: o[i][j] holds depth 32i + 8t + j and + 4 of rows g and g + 8
    float* const merge = reinterpret_cast<float*>(smem);
    const float back = scale_value(vref) * 0x1p-15f;
#pragma unroll
    for (int x = 0; x < RH; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (t == 0) row_stat[warp][g + 8 * x] = make_float2(m[x], l[x]);
      float* const to = merge + (warp * kRows + g + 8 * x) * Y::pitch + 8 * t;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float4*>(to + 32 * i + 4 * e) =
              make_float4(o[i][0][2 * x + e] * back, o[i][1][2 * x + e] * back, o[i][2][2 * x + e] * back, o[i][3][2 * x + e] * back);
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const long long slot = 2ll * blockIdx.x + (s0 == 0);
    for (int i = threadIdx.x; i < 8 * RH * (D / 4); i += 32 * kWarps) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      if (row0 + r >= R) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, row_stat[w][r].x);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_fast(row_stat[w][r].x - ref);
        const float4 y = *reinterpret_cast<const float4*>(merge + (w * kRows + r) * Y::pitch + d);
        sum += f * row_stat[w][r].y;
        v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
      }
      if (whole) {
        const int tok = (row0 + r) / G, hq = h * G + (row0 + r) % G;
        const bool none = sum == 0.0f || tok >= ql;
        const float f = none ? 0.0f : 1.0f / sum;
        const float y[4] = {none ? 0.0f : v.x * f, none ? 0.0f : v.y * f, none ? 0.0f : v.z * f, none ? 0.0f : v.w * f};
        store4(static_cast<T*>(a.out) + (b * a.o_sb + hq * a.o_sh + tok * a.o_sl + d), y);
        if (a.lse && d == 0) static_cast<float*>(a.lse)[((long long)b * a.Hq + hq) * a.T + tok] = none ? -INFINITY : top + log2f(sum);
      } else {
        *reinterpret_cast<float4*>(a.part + (slot * kRows + r) * D + d) = v;
        if (d == 0) a.stat[slot * kRows + r] = make_float2(top, sum);
      }
    }
    at += s1 - s0;
    if (at >= begin + (long long)steps * units) {
      begin += (long long)steps * units;
      ++b;
    }
  }
}

// Units that several CTAs had a part of: a warp adds up one row's parts, in the order of the keys.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kWarps) kv_combine_kernel(const __grid_constant__ Call a, int ctas) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, units = a.cache.Hkv * a.groups;
  const int b = blockIdx.x / units, u = blockIdx.x % units;
  const int r = blockIdx.y * kWarps + warp, G = a.Hq / a.cache.Hkv, row = u % a.groups * kRows + r;
  const long long share = share_of(a, ctas, lane);
  long long begin = 0;
  for (int i = lane; i < b; i += 32) begin += (long long)steps_of(length_of(a, i)) * units;
#pragma unroll
  for (int d = 16; d; d /= 2) begin += __shfl_xor_sync(0xffffffffu, begin, d);
  const int len = length_of(a, b), steps = steps_of(len), ql = queries_of(a, b, len);
  begin += (long long)u * steps;
  const long long c0 = begin / share, c1 = (begin + steps - 1) / share;
  grid_dependency_wait();                             // (by everybody: what follows on the stream counts on it)
  if (c0 == c1 || row >= a.T * G) return;
  float top = -INFINITY, sum = 0.0f;
  for (long long i = c0; i <= c1; ++i) top = fmaxf(top, a.stat[(2 * i + (i == c0)) * kRows + r].x);
  const float ref = top == -INFINITY ? 0.0f : top;
  constexpr int N = D / 32;
  float v[N] = {};
#pragma unroll 4
  for (long long i = c0; i <= c1; ++i) {
    const long long at = (2 * i + (i == c0)) * kRows + r;
    const float2 st = a.stat[at];
    const float f = exp2_fast(st.x - ref);
    sum += f * st.y;
    if constexpr (N == 4) {
      const float4 x = *reinterpret_cast<const float4*>(a.part + at * D + 4 * lane);
      v[0] += f * x.x; v[1] += f * x.y; v[2] += f * x.z; v[3] += f * x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(a.part + at * D + 2 * lane);
      v[0] += f * x.x; v[1] += f * x.y;
    }
  }
  const int tok = row / G, hq = u / a.groups * G + row % G;
  const bool none = sum == 0.0f || tok >= ql;
  const float f = none ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = none ? 0.0f : v[i] * f;
  T* const y = static_cast<T*>(a.out) + (b * a.o_sb + hq * a.o_sh + tok * a.o_sl + N * lane);
  if constexpr (N == 4) {
    const float x[4] = {v[0], v[1], v[2], v[3]};
    store4(y, x);
  } else {
    *reinterpret_cast<uint32_t*>(y) = pack2(T(), v[0], v[1]);
  }
  if (a.lse && lane == 0) static_cast<float*>(a.lse)[((long long)b * a.Hq + hq) * a.T + tok] = none ? -INFINITY : top + log2f(sum);
}

constexpr int kPerSm = 3;

int ctas_of(const Call& a) {
  const long long most = (long long)a.B * a.cache.Hkv * a.groups * (((long long)a.max_pages * a.cache.page_size + kStep - 1) / kStep + 1);
  const long long all = (long long)kPerSm * sm_count();
  return (int)(most < all ? most : all);
}

template <typename T, int ELEM, int D>
int launch(const Call& a, cudaStream_t st) {
  constexpr int bytes = Layout<ELEM, D>::bytes;
  const int ctas = ctas_of(a), rows = a.T * (a.Hq / a.cache.Hkv);
  constexpr int id = (std::is_same_v<T, __half> ? 100 : 0) + ELEM * 10 + D;
  if (rows <= 8) {
    if (!allow_smem<1000 + id>(kv_attention_kernel<T, ELEM, D, 1>, bytes)) return set_error(MPSA_ERR_LAUNCH, "kv_attention: shared memory not granted");
    kv_attention_kernel<T, ELEM, D, 1><<<ctas, 32 * kWarps, bytes, st>>>(a);
  } else {
    if (!allow_smem<2000 + id>(kv_attention_kernel<T, ELEM, D, 2>, bytes)) return set_error(MPSA_ERR_LAUNCH, "kv_attention: shared memory not granted");
    kv_attention_kernel<T, ELEM, D, 2><<<ctas, 32 * kWarps, bytes, st>>>(a);
  }
  if (int rc = check_launch("kv_attention")) return rc;
  const dim3 grid(a.B * a.cache.Hkv * a.groups, (min(rows, kRows) + kWarps - 1) / kWarps);
  launch_dependent(kv_combine_kernel<T, D>, grid, 32 * kWarps, 0, st, true, a, ctas);
  return check_launch("kv_attention");
}
template <typename T, int ELEM>
int launch_depth(const Call& a, cudaStream_t st) {
  return a.cache.D == 64 ? launch<T, ELEM, 64>(a, st) : launch<T, ELEM, 128>(a, st);
}
template <typename T>
int launch_elem(const Call& a, cudaStream_t st) {
  return a.cache.elem == E4M3 ? launch_depth<T, E4M3>(a, st) : a.cache.elem == E5M2 ? launch_depth<T, E5M2>(a, st) : launch_depth<T, E2M1>(a, st);
}

// The call with its plan and its workspace's parts; the workspace's bytes, or an error.
long long plan(const mpsa_kv_attention_args* args, Call& a) {
  if (!args || !args->page_table || !args->lengths) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: null pointer");
  a = {};
  static_cast<mpsa_kv_attention_args&>(a) = *args;
  if (int rc = check_cache(a.cache, "kv_attention")) return rc;
  if (a.dtype != 0 && a.dtype != 1) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: queries must be bf16 or fp16");
  if (a.B <= 0 || a.T <= 0 || a.Hq <= 0 || a.max_pages <= 0) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: non-positive shape");
  if (a.Hq % a.cache.Hkv) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: Hq must be a multiple of Hkv");
  if (a.B > 65535 || a.Hq > 65535 || a.T > 1024) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: at most 65535 sequences and 1024 query tokens");
  if (!(a.sm_scale > 0.0f) || a.sm_scale > 1e30f) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: sm_scale must be positive and finite");
  a.groups = (a.T * (a.Hq / a.cache.Hkv) + kRows - 1) / kRows;
  if ((long long)a.B * a.cache.Hkv * a.groups > 0x7fffffffll) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: too many sequences and heads");
  const long long slots = 2ll * ctas_of(a) * kRows;
  a.part = static_cast<float*>(a.workspace);
  a.stat = reinterpret_cast<float2*>(a.part + slots * a.cache.D);
  return slots * (a.cache.D * 4 + 8);
}

}  // namespace
}  // namespace mpsa

using namespace mpsa;

extern "C" long long mpsa_kv_attention_workspace(const mpsa_kv_attention_args* args) {
  Call a;
  return plan(args, a);
}

extern "C" int mpsa_kv_attention(const mpsa_kv_attention_args* args, void* stream) {
  Call a;
  const long long need = plan(args, a);
  if (need < 0) return (int)need;
  if (!a.q || !a.out) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: null pointer");
  if ((a.q_sb | a.q_sh | a.q_sl | a.o_sb | a.o_sh | a.o_sl) % 8 || ((uintptr_t)a.q | (uintptr_t)a.out) % 16)
    return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: q and out need 16-byte aligned bases and strides that are multiples of 8 elements");
  if (!a.workspace || a.workspace_bytes < need || (uintptr_t)a.workspace % 256)
    return set_error(MPSA_ERR_BAD_ARG, "kv_attention: the workspace must hold %lld bytes and be 256-byte aligned", need);
  const cudaStream_t st = (cudaStream_t)stream;
  return a.dtype == 0 ? launch_elem<__nv_bfloat16>(a, st) : launch_elem<__half>(a, st);
}
