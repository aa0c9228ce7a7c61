// Attention of a sequence's last tokens over its paged MX cache (mpsa_kv_attention).
//
// This kernel: up to 32 query rows of a KV head, steps of 32 keys (decode.cuh says what a unit, a step and a run are; decode_wide.cu has the
// kernel for more rows).  Within a CTA the warps take steps in turn and have nothing to do with each other until the run's part of a unit is done: each copies its own
// keys to its own shared memory with cp.async, and keeps its own references, sums and output in registers.
//
//   scores    S^T = K Q^T by m16n8k16 on fp16 operands, keys in the M dimension: a few query rows fill the N of 8.  Element codes convert
//             exactly; a block's 32 depth elements are two instructions of their own, whose fp32 result is multiplied by the key's scale of
//             that block.  Queries are brought to a largest magnitude of 1 .. 2 by a power of two of their row, so that their 8 or 11
//             significant bits survive in fp16.
//   output    O^T = V^T P^T, depth in the M dimension.  The block scales of V differ from key to key, so they go to P: for each block of the
//             depth P times the scales is rounded to fp16 and multiplied by the codes.  This rounding of P, and that of query elements below
//             2^-14 of their row's largest (2^-17 where they come in bf16), are the only ones below fp32.
//   softmax   against a reference U of the row that keeps those products, not P, within fp16: U is set so that the largest (score plus log2
//             of the key's largest scale) gives 2^7, and raised when one would give more than 2^15.  Products keep 11 bits down to 2^-21 of
//             the row's largest, whatever the sizes of other keys' values are.  P and the row's sum of P are fp32; U is at least the largest
//             score - 100, so that they stay finite (values below 2^-90 have fewer bits, then).  Weights below 2^-126 in units of U are dropped: beside
//             values of 2^110 or more, where U is that much above the scores, they would matter.
// Fragments of K and V come from ldmatrix on the codes as they are (.trans for V: two keys of neighbouring depth elements in a register).
//
// It is bound by the cache's bytes (HBM) as long as the conversions keep up: ALU-pipe instructions, two elements each; in E2M1, with twice the
// elements a byte, by latency before any one pipe (issue and ALU 62 %, DRAM 50 %, 16 warps an SM).  8 KV heads of depth 128,
// 4 query heads each: 32 sequences of up to 16384 tokens in E4M3 111 us (5.1 - 5.8 TB/s; 705 instructions a step and warp), 4 of 131072 in E2M1
// 147 us (3.9 TB/s).  With queries in the M dimension the first took 140 us: half of each instruction's 16 rows were padding.
#include "api_internal.h"
#include "decode.cuh"

#include <algorithm>
#include <type_traits>

namespace mpsa {
namespace {

constexpr int kWarps = 4, kStep = 32;
constexpr int kMostCluster = 8, kClusterSteps = 40;
constexpr float kMost = 15.0f, kSet = 7.0f;    // log2 of the largest product that raises no reference, and of the largest one after a raise
constexpr int kLeast = -85;                    // log2 of a scale that counts as that at least: references are the largest score - 100 at least

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {       // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {          // an 8 x 8 matrix of 16-bit values, two of a row in a lane
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Shared memory: for each warp kStages steps of [K codes][V codes][K scales][V scales] and the step's scales as floats, then the unit's
// queries in the order of the fragments and the factors of its rows.  The warps' parts of the output go where the steps were.
template <int ELEM, int D, int NR>
struct Layout {
  static constexpr int row = code_bytes(ELEM, D), nb = D / 32, rows = 8 * NR;
  static constexpr int codes = kStep * row, stage = 2 * codes + 2 * kStep * nb;
  static constexpr int stages = 2;
  static constexpr int scales = stages * stage, warp = scales + 2 * kStep * nb * 4;
  static constexpr int pitch = D + 8;                                  // floats of a row of a warp's part
  static constexpr int merge = kWarps * rows * pitch * 4;
  static constexpr int queries = kWarps * warp > merge ? kWarps * warp : merge;
  static constexpr int bytes = queries + rows * D * 2 + rows * 4;
  static constexpr int pairs = row / 32;                               // pieces of 32 bytes of a row: what one ldmatrix takes of 16 keys
  static_assert(stage % 128 == 0 && warp % 128 == 0 && queries % 128 == 0, "the blocks' places are found by exclusive or");
  // Where a row's 16-byte pieces lie: the eight rows of a matrix meet different banks.
  static __device__ __forceinline__ int swap(int r) { return row == 128 ? r & 7 : row == 64 ? (r >> 1) & 3 : (r >> 2) & 1; }
  // A lane's first depth element in instruction s of a block: four in the order of a fragment of K and Q; two of V^T and O^T
  static __device__ __forceinline__ int k_depth(int s, int t) { return ELEM == E2M1 ? 8 * t + 4 * s : 16 * s + 4 * t; }
  static __device__ __forceinline__ int v_depth(int s, int g) { return ELEM == E2M1 ? 4 * g + 2 * s : 16 * s + 2 * g; }
};

// One piece of 32 bytes of 16 keys (K): the A operands of its instructions; 8 bits: one block, 4 bits: two.
template <int ELEM>
__device__ __forceinline__ void k_fragments(uint32_t p, uint32_t (&f)[ELEM == E2M1 ? 4 : 2][4]) {
  uint32_t w[4];
  ldmatrix(w, p);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint32_t v = w[2 * i + x];                 // keys g + 8x
      if constexpr (ELEM == E2M1) elem_quads(v, f[2 * i][x], f[2 * i][2 + x], f[2 * i + 1][x], f[2 * i + 1][2 + x]);
      else elem_two<ELEM>(v, f[i][x], f[i][2 + x]);
    }
}

// The same of V, transposed: rows of A are depth elements, its columns the keys.
template <int ELEM>
__device__ __forceinline__ void v_fragments(uint32_t p, uint32_t (&f)[ELEM == E2M1 ? 4 : 2][4]) {
  uint32_t w[4];
  ldmatrix_trans(w, p);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint32_t v = w[2 * i + x];                 // keys 8x + 2t (lower half) and 8x + 2t + 1
      if constexpr (ELEM == E2M1) {
        uint32_t a, b, c, d;
        elem_quads(v, a, b, c, d);
        f[2 * i][2 * x] = __byte_perm(a, c, 0x5410);
        f[2 * i][2 * x + 1] = __byte_perm(a, c, 0x7632);
        f[2 * i + 1][2 * x] = __byte_perm(b, d, 0x5410);
        f[2 * i + 1][2 * x + 1] = __byte_perm(b, d, 0x7632);
      } else {
        elem_two<ELEM>(__byte_perm(v, 0, 0x3120), f[i][2 * x], f[i][2 * x + 1]);
      }
    }
}

// CTAs of an SM: what shared memory (four-bit codes need half) and registers let in.  16 rows of depth 128 spill with three: 8 sequences of 8192
// with 4 x 4 rows 60.8 us, with two 41.7.
constexpr __host__ __device__ int per_sm(int tiles, int elem, int D) { return tiles == 4 || (tiles == 2 && D == 128) ? 2 : tiles == 2 || elem != E2M1 ? 3 : 4; }

// Cluster barrier: what its CTAs wrote to shared memory before it can be read by all of them after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t p) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ float2 load_cluster2(uint32_t p) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p) : "memory");
  return v;
}

// Four elements of a row's output.
template <typename T>
__device__ __forceinline__ void write_out(const Call& a, int b, int h, int G, int row, int ql, int d, float4 v, float top, float sum) {
  const int tok = row / G, hq = h * G + row % G;
  const bool none = sum == 0.0f || tok >= ql;
  const float f = none ? 0.0f : 1.0f / sum;
  const float y[4] = {none ? 0.0f : v.x * f, none ? 0.0f : v.y * f, none ? 0.0f : v.z * f, none ? 0.0f : v.w * f};
  store4(static_cast<T*>(a.out) + (b * a.o_sb + hq * a.o_sh + (long long)tok * a.o_sl + d), y);
  if (a.lse && d == 0) static_cast<float*>(a.lse)[((long long)b * a.Hq + hq) * a.T + tok] = none ? -INFINITY : top + log2f(sum);
}

// CLUSTER: a.cluster CTAs share a unit, each has an equal run of its steps, and they add up their parts through shared memory.
template <typename T, int ELEM, int D, int NR, bool CLUSTER>
__global__ void __launch_bounds__(32 * kWarps, per_sm(NR, ELEM, D)) kv_attention_kernel(const __grid_constant__ Call a) {
  using Y = Layout<ELEM, D, NR>;
  constexpr int NB = D / 32, NM = kStep / 16;          // blocks of the depth, key tiles of a step
  constexpr int BP = ELEM == E2M1 ? 2 : 1;             // blocks of a 32-byte piece
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 row_stat[kWarps][8 * NR], unit_stat[CLUSTER ? 8 * NR : 1];
  const mpsa_kv_cache& c = a.cache;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring = smem_u32(smem) + warp * Y::warp;
  float* const ksc = reinterpret_cast<float*>(smem + warp * Y::warp + Y::scales);
  float* const vsc = ksc + kStep * NB;
  uint2* const queries = reinterpret_cast<uint2*>(smem + Y::queries);                  // [block][instruction][row tile][lane]
  float* const factors = reinterpret_cast<float*>(smem + Y::queries + Y::rows * D * 2);
  const int G = a.Hq / c.Hkv, R = a.T * G, units = c.Hkv * a.groups;
  const uint32_t mat = (lane & 15) * Y::row + ((lane >> 4) ^ Y::swap(lane & 15)) * 16;  // this lane's row address for ldmatrix

  grid_dependency_wait();
  grid_dependents_go();
  uint32_t share, begin = 0, at = 0, stop = 1;
  int b = CLUSTER ? blockIdx.x / a.cluster / units : locate(a, gridDim.x, blockIdx.x, share, begin, lane);
  if constexpr (!CLUSTER) {
    at = blockIdx.x * share;
    stop = at + min(share, ~at);
  }
  for (bool again = false; b < a.B && at < stop; again = true) {
    const int len = length_of(a, b), steps = steps_of(a, len);
    int u, s0, s1;
    if constexpr (CLUSTER) {
      const int rank = blockIdx.x % a.cluster, per = (steps + a.cluster - 1) / a.cluster;
      u = blockIdx.x / a.cluster % units;
      s0 = min(rank * per, steps);
      s1 = min(s0 + per, steps);
    } else {
      const uint32_t off = at - begin;
      u = off / (uint32_t)steps;
      s0 = off - u * (uint32_t)steps;
      s1 = min((uint32_t)steps, s0 + (stop - at));
    }
    const int h = u / a.groups, row0 = u % a.groups * Y::rows;
    const int ql = queries_of(a, b, len), first = len - ql;
    const int* const table = a.page_table + b * a.table_sb;
    if (again) __syncthreads();                       // (the merge buffer has been read)

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
          const uint32_t d = to + r * Y::row + (ch ^ Y::swap(i * RPI + rl)) * 16;
          copy16(d, kp + i * 512, there);
          copy16(d + Y::codes, vp + i * 512, there);
        }
      }
      if (lane < 4 * NB) {                                            // 16-byte pieces: NB for 16 keys of K or V
        const int half = lane / NB % 2, p = half ? p1 : p0;
        const long long row = ((long long)max(p, 0) * c.Hkv + h) * c.page_size + ((pos + 16 * half) & (c.page_size - 1));
        copy16(to + 2 * Y::codes + lane * 16, static_cast<const uint8_t*>(lane >= 2 * NB ? c.v_scale : c.k_scale) + row * NB + lane % NB * 16, p >= 0);
      }
    };
    auto page = [&](int k, int half) { return __shfl_sync(0xffffffffu, pages, 2 * (k % 16) + half); };

    int cur0 = page(0, 0), cur1 = page(0, 1);         // pages of step k
    if (mine > 0) request(0, cur0, cur1);
    asm volatile("cp.async.commit_group;" ::: "memory");

    // queries of the unit in the order of the B fragments: a warp takes row tiles in turn, a lane row g of it
    for (int n = warp; n < NR; n += kWarps) {
      const int r = row0 + 8 * n + g;
      float q[NB][2][4];
      uint32_t amax = 0;
      const T* p = static_cast<const T*>(a.q) + (b * a.q_sb + (h * G + r % G) * a.q_sh + (long long)(r / G) * a.q_sl);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (r < R) load4(p + 32 * i + Y::k_depth(s, t), q[i][s]);
          else q[i][s][0] = q[i][s][1] = q[i][s][2] = q[i][s][3] = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) amax = max(amax, __float_as_uint(q[i][s][e]) & 0x7fffffffu);
        }
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = min(max((int)(amax >> 23), 1), 253);              // biased exponent of the row
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      if (t == 0) factors[8 * n + g] = amax >= 0x7f800000u ? __int_as_float(0x7fffffff) : a.sm_scale * 1.44269504f * __uint_as_float((uint32_t)e << 23);
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          queries[((2 * i + s) * NR + n) * 32 + lane] = make_uint2(pack2(__half(), q[i][s][0] * down, q[i][s][1] * down), pack2(__half(), q[i][s][2] * down, q[i][s][3] * down));
    }
    __syncthreads();
    float rs[NR][2], m[NR][2], l[NR][2];              // rows 8n + 2t and + 1
    uint2 qf[NR <= 2 ? 2 * NB : 1][NR <= 2 ? NR : 1];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        rs[n][x] = factors[8 * n + 2 * t + x];
        m[n][x] = -INFINITY;
        l[n][x] = 0.0f;
      }
      if constexpr (NR <= 2)
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) qf[i][n] = queries[(i * NR + n) * 32 + lane];
    }
    float o[NB][2][NR][4] = {};                       // depth v_depth(s, g) (elements 0, 1: rows 2t, 2t + 1) and the next one (2, 3)

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
      const bool special = pos + kStep > (a.T > 1 || a.mask ? first : len) || cur0 < 0 || cur1 < 0;     // some key not seen by some row

      // scales of key `lane`, as floats for everybody
      bool strange;                                   // a scale of V is NaN
      float size;                                     // log2 of key `lane`'s largest scale of V
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
        uint32_t e[NB], top = 0;
        float kf[NB], vf[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          e[i] = vb >> (8 * i) & 255u;
          top = max(top, e[i]);
          kf[i] = scale_value(kb >> (8 * i) & 255u);
          vf[i] = __uint_as_float(e[i] << 23);
        }
        strange = __any_sync(0xffffffffu, top == 255u);
        if (strange) {
          top = 0;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            if (e[i] == 255u) vf[i] = __int_as_float(0x7fffffff);
            else top = max(top, e[i]);
          }
        }
        size = (float)max((int)top - 127, kLeast);
        if constexpr (NB == 4) {
          reinterpret_cast<float4*>(ksc)[lane] = make_float4(kf[0], kf[1], kf[2], kf[3]);
          reinterpret_cast<float4*>(vsc)[lane] = make_float4(vf[0], vf[1], vf[2], vf[3]);
        } else {
          reinterpret_cast<float2*>(ksc)[lane] = make_float2(kf[0], kf[1]);
          reinterpret_cast<float2*>(vsc)[lane] = make_float2(vf[0], vf[1]);
        }
        __syncwarp();
      }

      // s[w][n][..]: key 16w + g of rows 2t, 2t + 1 of tile n, then key 16w + g + 8
      float s[NM][NR][4] = {};
      auto scale_of = [&](const float* p, int key, float (&f)[NB]) {
        if constexpr (NB == 4) {
          const float4 v = reinterpret_cast<const float4*>(p)[key];
          f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        } else {
          const float2 v = reinterpret_cast<const float2*>(p)[key];
          f[0] = v.x; f[1] = v.y;
        }
      };
#pragma unroll
      for (int w = 0; w < NM; ++w) {
        float k0[NB], k1[NB];
        scale_of(ksc, 16 * w + g, k0);
        scale_of(ksc, 16 * w + g + 8, k1);
#pragma unroll
        for (int j = 0; j < Y::pairs; ++j) {
          uint32_t f[2 * BP][4];
          k_fragments<ELEM>((buf + 16 * w * Y::row + mat) ^ (32 * j), f);
#pragma unroll
          for (int i = 0; i < BP; ++i) {
            const int blk = BP * j + i;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              float d[4] = {};
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint2 q = NR <= 2 ? qf[NR <= 2 ? 2 * blk + x : 0][NR <= 2 ? n : 0] : queries[((2 * blk + x) * NR + n) * 32 + lane];
                mma(d, f[2 * i + x][0], f[2 * i + x][1], f[2 * i + x][2], f[2 * i + x][3], q.x, q.y);
              }
              s[w][n][0] = fmaf(d[0], k0[blk], s[w][n][0]);
              s[w][n][1] = fmaf(d[1], k0[blk], s[w][n][1]);
              s[w][n][2] = fmaf(d[2], k1[blk], s[w][n][2]);
              s[w][n][3] = fmaf(d[3], k1[blk], s[w][n][3]);
            }
          }
        }
      }

      // scores in log2 units, and whether a reference has to be raised
      bool above = false;
      float sz[NM][2];
#pragma unroll
      for (int w = 0; w < NM; ++w) {
        sz[w][0] = __shfl_sync(0xffffffffu, size, 16 * w + g);
        sz[w][1] = __shfl_sync(0xffffffffu, size, 16 * w + g + 8);
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int w = 0; w < NM; ++w)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[w][n][x] *= rs[n][x & 1];
      if (special) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = row0 + 8 * n + 2 * t + x, tok = r / G;
            const bool real = r < R && tok < ql;
            const unsigned char* const mk = a.mask + b * a.mask_sb + (long long)tok * a.T;
#pragma unroll
            for (int w = 0; w < NM; ++w)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const int p = pos + 16 * w + g + 8 * y, j = p - first;
                const bool seen = p < len && (w ? cur1 : cur0) >= 0 && (j < 0 || (real && (a.mask ? mk[j] != 0 : j <= tok)));
                if (!seen) s[w][n][2 * y + x] = -INFINITY;
              }
          }
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float top = fmaxf(fmaxf(s[0][n][x] + sz[0][0], s[0][n][2 + x] + sz[0][1]), fmaxf(s[1][n][x] + sz[1][0], s[1][n][2 + x] + sz[1][1]));
          above |= top > m[n][x] + kMost;
        }
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = fmaxf(fmaxf(s[0][n][x] + sz[0][0], s[0][n][2 + x] + sz[0][1]), fmaxf(s[1][n][x] + sz[1][0], s[1][n][2 + x] + sz[1][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) - kSet;
            if (top > m[n][x]) {
              const float f = exp2_fast(m[n][x] - top);
              l[n][x] = lowered(l[n][x], m[n][x] - top);
#pragma unroll
              for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                  o[i][y][n][x] *= f;
                  o[i][y][n][2 + x] *= f;
                }
              m[n][x] = top;
            }
          }
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float ref = m[n][x] == -INFINITY ? 0.0f : m[n][x];
#pragma unroll
          for (int w = 0; w < NM; ++w) {
            s[w][n][x] = exp2_fast(s[w][n][x] - ref);
            s[w][n][2 + x] = exp2_fast(s[w][n][2 + x] - ref);
            l[n][x] += s[w][n][x] + s[w][n][2 + x];
          }
        }

      // O^T += V^T P^T, 16 keys at a time
#pragma unroll
      for (int w = 0; w < NM; ++w) {
        float v0[NB], v1[NB];
        scale_of(vsc, 16 * w + g, v0);
        scale_of(vsc, 16 * w + g + 8, v1);
#pragma unroll
        for (int j = 0; j < Y::pairs; ++j) {
          uint32_t f[2 * BP][4];
          v_fragments<ELEM>((buf + Y::codes + 16 * w * Y::row + mat) ^ (32 * j), f);
#pragma unroll
          for (int i = 0; i < BP; ++i) {
            const int blk = BP * j + i;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              float p[4] = {s[w][n][0] * v0[blk], s[w][n][1] * v0[blk], s[w][n][2] * v1[blk], s[w][n][3] * v1[blk]};
              if (special && strange)                 // NaN of a key that the row does not see
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (s[w][n][x] == 0.0f) p[x] = 0.0f;
              const uint32_t b0 = transposed(pack2(__half(), p[0], p[1])), b1 = transposed(pack2(__half(), p[2], p[3]));
#pragma unroll
              for (int x = 0; x < 2; ++x) mma(o[blk][x][n], f[2 * i + x][0], f[2 * i + x][1], f[2 * i + x][2], f[2 * i + x][3], b0, b1);
            }
          }
        }
      }
      __syncwarp();                                   // the step's buffers are free
      cur0 = nx0;
      cur1 = nx1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // the warps' parts together
    float* const merge = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 4);
        l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 8);
        l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 16);
        const int r = 8 * n + 2 * t + x;
        if (g == 0) row_stat[warp][r] = make_float2(m[n][x], l[n][x]);
        float* const to = merge + (warp * Y::rows + r) * Y::pitch;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int s = 0; s < 2; ++s)
            *reinterpret_cast<float2*>(to + 32 * i + Y::v_depth(s, g)) = make_float2(o[i][s][n][x], o[i][s][n][2 + x]);
      }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const long long slot = 2ll * blockIdx.x + (s0 == 0);
    for (int i = threadIdx.x; i < Y::rows * (D / 4); i += 32 * kWarps) {
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
        const float4 y = *reinterpret_cast<const float4*>(merge + (w * Y::rows + r) * Y::pitch + d);
        sum += lowered(row_stat[w][r].y, row_stat[w][r].x - ref);
        v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
      }
      if constexpr (CLUSTER) {                        // (the place of warp 0's part: nobody else reads it)
        *reinterpret_cast<float4*>(merge + r * Y::pitch + d) = v;
        if (d == 0) unit_stat[r] = make_float2(top, sum);
      } else if (whole) {
        write_out<T>(a, b, h, G, row0 + r, ql, d, v, top, sum);
      } else {
        *reinterpret_cast<float4*>(a.part + (slot * Y::rows + r) * D + d) = v;
        if (d == 0) a.stat[slot * Y::rows + r] = make_float2(top, sum);
      }
    }
    if constexpr (CLUSTER) {
      cluster_sync();
      const uint32_t parts = smem_u32(merge), stats = smem_u32(unit_stat);
      for (int i = blockIdx.x % a.cluster * (32 * kWarps) + threadIdx.x; i < Y::rows * (D / 4); i += a.cluster * (32 * kWarps)) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (row0 + r >= R) continue;
        float top = -INFINITY, sum = 0.0f;
        for (int c = 0; c < a.cluster; ++c) top = fmaxf(top, load_cluster2(at_rank(stats + r * 8, c)).x);
        const float ref = top == -INFINITY ? 0.0f : top;
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (int c = 0; c < a.cluster; ++c) {
          const float2 st = load_cluster2(at_rank(stats + r * 8, c));
          const float4 y = load_cluster4(at_rank(parts + (r * Y::pitch + d) * 4, c));
          const float f = exp2_fast(st.x - ref);
          sum += lowered(st.y, st.x - ref);
          v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
        }
        write_out<T>(a, b, h, G, row0 + r, ql, d, v, top, sum);
      }
      cluster_sync();                                 // (nobody's shared memory goes before all have read it)
      return;
    }
    at += s1 - s0;
    if (!CLUSTER && at - begin >= (uint32_t)steps * units) {
      begin += (uint32_t)steps * units;
      ++b;
    }
  }
}

// Units that several CTAs had a part of: a warp adds up one row's parts, in the order of the keys.  (Four rows a warp where units have 128, for a
// quarter of the CTAs: trees of 32 tokens 181 us instead of 174.)
template <typename T, int D>
__global__ void __launch_bounds__(32 * kWarps) kv_combine_kernel(const __grid_constant__ Call a, int ctas) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, units = a.cache.Hkv * a.groups;
  const int b = blockIdx.x / units, u = blockIdx.x % units;
  const int rows = a.rows, r = blockIdx.y * kWarps + warp, G = a.Hq / a.cache.Hkv, row = u % a.groups * rows + r;
  uint32_t share, begin;
  locate(a, ctas, 0, share, begin, lane);
  begin = 0;
  for (int i = lane; i < b; i += 32) begin += steps_of(a, length_of(a, i)) * units;
  begin = __reduce_add_sync(0xffffffffu, begin);
  const int len = length_of(a, b), steps = steps_of(a, len), ql = queries_of(a, b, len);
  begin += u * steps;
  const int c0 = begin / share, parts = (begin + steps - 1) / share - c0 + 1;
  grid_dependency_wait();                             // (by everybody: what follows on the stream counts on it)
  if (parts == 1 || row >= a.T * G) return;
  // part i lies in slot 2 (c0 + i), the first one in 2 c0 + 1: a lane takes one of 32 parts' statistics, and then all add up the rows
  auto slot = [&](int i) { return (long long)(2 * (c0 + i) + (i == 0)) * rows + r; };
  const float2 nothing = make_float2(-INFINITY, 0.0f), first = lane < parts ? a.stat[slot(lane)] : nothing;
  float top = first.x, sum = 0.0f;
  for (int i = lane + 32; i < parts; i += 32) top = fmaxf(top, a.stat[slot(i)].x);
#pragma unroll
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float ref = top == -INFINITY ? 0.0f : top;
  constexpr int N = D / 32;
  float v[N] = {};
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const float2 st = i0 == 0 ? first : i0 + lane < parts ? a.stat[slot(i0 + lane)] : nothing;
    const float f = exp2_fast(st.x - ref);
    sum += lowered(st.y, st.x - ref);
    const int n = min(parts - i0, 32);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, f, i);
      const float* const p = a.part + slot(i0 + i) * D + N * lane;
      if constexpr (N == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] += w * x.x; v[1] += w * x.y; v[2] += w * x.z; v[3] += w * x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] += w * x.x; v[1] += w * x.y;
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
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

bool wide(const Call& a) { return a.rows == kWideRows; }

int ctas_of(const Call& a) {
  const double most = (double)a.B * a.cache.Hkv * a.groups * ((double)a.max_pages * a.cache.page_size / a.step + 1);
  const double all = (double)(wide(a) ? kWideCtas : per_sm(a.rows / 8, a.cache.elem, a.cache.D)) * sm_count();
  return (int)(most < all ? most : all);
}

template <typename T, int ELEM, int D, int NR>
int launch(const Call& a, int ctas, cudaStream_t st) {
  constexpr int bytes = Layout<ELEM, D, NR>::bytes;
  constexpr int id = (std::is_same_v<T, __half> ? 10000 : 0) + ELEM * 1000 + D * 8 + NR;
  if constexpr (NR <= 2) {
    if (a.cluster) {
      const auto kernel = kv_attention_kernel<T, ELEM, D, NR, true>;
      if (!allow_smem<20000 + id>(kernel, bytes)) return set_error(MPSA_ERR_LAUNCH, "kv_attention: shared memory not granted");
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(a.B * a.cache.Hkv * a.groups * a.cluster);
      cfg.blockDim = dim3(32 * kWarps);
      cfg.dynamicSmemBytes = bytes;
      cfg.stream = st;
      cudaLaunchAttribute at[2];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = a.cluster;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[1].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at;
      cfg.numAttrs = overlaps_previous(st) ? 2 : 1;
      cudaLaunchKernelEx(&cfg, kernel, a);
      return check_launch("kv_attention");
    }
  }
  const auto kernel = kv_attention_kernel<T, ELEM, D, NR, false>;
  if (!allow_smem<id>(kernel, bytes)) return set_error(MPSA_ERR_LAUNCH, "kv_attention: shared memory not granted");
  launch_dependent(kernel, dim3(ctas), 32 * kWarps, bytes, st, overlaps_previous(st), a);
  return check_launch("kv_attention");
}
template <typename T, int ELEM, int D>
int launch_rows(const Call& a, int ctas, cudaStream_t st) {
  return a.rows == 8 ? launch<T, ELEM, D, 1>(a, ctas, st) : a.rows == 16 ? launch<T, ELEM, D, 2>(a, ctas, st) : launch<T, ELEM, D, 4>(a, ctas, st);
}
template <typename T, int ELEM>
int launch_depth(const Call& a, int ctas, cudaStream_t st) {
  return a.cache.D == 64 ? launch_rows<T, ELEM, 64>(a, ctas, st) : launch_rows<T, ELEM, 128>(a, ctas, st);
}
template <typename T>
int launch_all(const Call& a, cudaStream_t st) {
  const int ctas = ctas_of(a), elem = a.cache.elem;
  if (int rc = wide(a) ? launch_wide(a, ctas, st)
                       : elem == E4M3 ? launch_depth<T, E4M3>(a, ctas, st) : elem == E5M2 ? launch_depth<T, E5M2>(a, ctas, st) : launch_depth<T, E2M1>(a, ctas, st))
    return rc;
  if (a.cluster) return MPSA_OK;
  const int rows = a.T * (a.Hq / a.cache.Hkv);
  const dim3 grid(a.B * a.cache.Hkv * a.groups, (std::min(rows, a.rows) + kWarps - 1) / kWarps);
  if (a.cache.D == 64) launch_dependent(kv_combine_kernel<T, 64>, grid, 32 * kWarps, 0, st, true, a, ctas);
  else launch_dependent(kv_combine_kernel<T, 128>, grid, 32 * kWarps, 0, st, true, a, ctas);
  return check_launch("kv_attention");
}

// CTAs of a cluster for each unit, or 0 for runs and the combining launch.  Clusters where the table holds so little that the combining launch
// costs more than what equal runs gain.  8 KV heads of depth 128 in E4M3, tables as long as the sequences, us with clusters / with runs: one
// sequence of 2048 7.6 / 9.6, 8192 13.9 / 19.0, 16384 22.2 / 21.2; 8 of 4096 20.3 / 20.7 (uneven lengths 14.8 / 16.5); 32 of 1024 19.6 / 20.5
// (14.5 / 17.8), 32 of 2048 35.2 / 32.0 (24.6 / 20.8).
int cluster_of(const Call& a) {
  if (a.rows > 16) return 0;
  const double units = (double)a.B * a.cache.Hkv * a.groups, room = 3.0 * sm_count(), steps = (double)a.max_pages * a.cache.page_size / a.step;
  int c = 1;
  while (c < kMostCluster && units * 2 * c <= room && steps > 4 * c) c *= 2;
  return steps <= (double)kClusterSteps * c && units * c <= 65535.0 * 16 ? c : 0;
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
  const int rows = a.T * (a.Hq / a.cache.Hkv);
  // (8 sequences of 8192, 4 query heads a KV head, 128 keys a step / 32 keys, us: 32 rows 70.7 / 64.7, 40 rows 74.3 / 109.8, 96 rows 83.6 / 155.7)
  a.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : kWideRows;
  a.step = wide(a) ? kWideStep : kStep;
  a.least = wide(a) ? 2 : 4;                          // (four: a step for each warp)
  a.groups = (rows + a.rows - 1) / a.rows;
  a.cluster = cluster_of(a);
  const double most = (double)a.B * a.cache.Hkv * a.groups * ((double)a.max_pages * a.cache.page_size / a.step + 1);
  if ((double)a.B * a.cache.Hkv * a.groups > 2147483647.0) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: too many sequences and heads");
  if (most > 4e9) return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: sequences x heads x page table too large (%.1e steps of %d keys, at most 4e9)", most, a.step);
  const long long slots = 2ll * ctas_of(a) * a.rows;
  a.part = static_cast<float*>(a.workspace);
  a.stat = reinterpret_cast<float2*>(a.part + slots * a.cache.D);
  return a.cluster ? 0 : slots * (a.cache.D * 4 + 8);
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
  if (!a.q || !a.out || !a.status) return set_error(MPSA_ERR_BAD_ARG, "kv_attention: null pointer");
  if ((a.q_sb | a.q_sh | a.q_sl | a.o_sb | a.o_sh | a.o_sl) % 8 || ((uintptr_t)a.q | (uintptr_t)a.out) % 16)
    return set_error(MPSA_ERR_UNSUPPORTED, "kv_attention: q and out need 16-byte aligned bases and strides that are multiples of 8 elements");
  if (need && (!a.workspace || a.workspace_bytes < need || (uintptr_t)a.workspace % 256))
    return set_error(MPSA_ERR_BAD_ARG, "kv_attention: the workspace must hold %lld bytes and be 256-byte aligned", need);
  const cudaStream_t st = (cudaStream_t)stream;
  return a.dtype == 0 ? launch_all<__nv_bfloat16>(a, st) : launch_all<__half>(a, st);
}
