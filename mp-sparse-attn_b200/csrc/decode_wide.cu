// Attention of many query rows over a paged MX cache (mpsa_kv_attention with more than 32 rows of a KV head: trees of drafted tokens, short
// chunks) on the 5th-generation tensor cores.
//
// A unit is up to 128 query rows, a step 128 keys.  Eight warps: 4 convert, 4 are the softmax, the first of which also issues the
// tensor operations: what they wait for is what it has just done.
//   convert   the codes of a step's keys and values, kept on their way in registers one step ahead, become fp16 in shared memory: V relative to
//             the largest scale of its key (a factor of P), K to the largest of 32 keys (a factor of the scores) where their scales are so near
//             that all codes are exact, and otherwise to its key's too.  What fp16 cannot hold is 2^-31 of the key's largest element.
//             Both lie as rows of 128 bytes, 128-byte swizzle: K is a K-major operand, V, untransposed, an MN-major one.
//   Q K^T     128 x 128 x D, fp16 in, fp32 in TMEM.  Queries are scaled by a power of two of their row, as in decode.cu.
//   softmax   a thread a row: P times V's factor, rounded to fp16, goes over S; the reference U keeps that within fp16 as decode.cu says
//             (there it is each block's own scale).  One factor for 32 keys was 4 % faster, and took bits from all others where a key without
//             weight had large values.  The denominator adds up P itself: a key whose values are nothing, and whose product is, has its weight
//             in it.  Steps in which every row sees every key (and K is alike) are tried against the references as they are, in one pass;
//             where a product gets too large, and in the other steps, a pass over the scores finds the largest one first.
//   P V       128 x D x 128, P from TMEM, added up in TMEM.
// One step is a chain (Q K^T, softmax, P V) but for the conversion of the next one; the two CTAs of an SM fill each other's gaps.
// 8 sequences of up to 32768 tokens, 8 KV heads, trees of 32 tokens x 4 query heads: 177 - 186 us by box in E4M3, 179 in E5M2, 165 in E2M1.  7500 cycles a
// step with two in flight on an SM: softmax 2650, P V 1500 and Q K^T 2300 with the wait for their operands.  The converting warps are never idle:
// 950 and 800 cycles for the conversion of K and V, 2150 and 2000 until the loads of the next ones are issued, 900 for the look-ups.
// (128 registers a thread, 56 - 96 bytes of which spill.)
#include "api_internal.h"
#include "decode.cuh"

#include <type_traits>

namespace mpsa {
namespace {

constexpr int kThreads = 256, kColumns = 256;          // TMEM: S, over it P, then O from column 128
constexpr float kMost = 15.0f, kSet = 7.0f;            // as in decode.cu
constexpr float kLeast = -85.0f;

template <int D>
struct Layout {
  static constexpr int half = 128 * 128;               // 64 depth elements of 128 rows
  static constexpr int tile = half * (D / 64);
  static constexpr int q = 0, k = tile, v = 2 * tile;
  static constexpr int factors = 3 * tile;             // a converting warp's factors of its keys' blocks
  static constexpr int bytes = factors + 4 * 32 * 16 + 1024;           // (and what aligning the base may take)
};

struct Shared {
  uint64_t k_full, v_full, s_full, p_full, pv_done, q_full, drained;
  uint32_t tmem;
  alignas(16) float v_size[2][128], v_log[2][128];     // each key's largest scale of V, and log2 of it (two steps' worth, as below)
  float k_size[2][4];                                  // largest scale of K of 32 keys, in units of K's operand
  float k_part[2][128];                                // where these keys differ by more than kSpread: each key's largest scale as part of it
  uint32_t uneven[2][4];
  alignas(4) uint8_t odd[2][4];                        // uneven, or not all there
  uint32_t there[2][4];                                // keys with a page and within the length
  uint32_t strange[2][4][4];                           // [32 keys][block of the depth]: scales of V that are NaN
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
               "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
               "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void store_shared16(uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// What an element of the largest size becomes in an operand is 2^13 to 2^16: fp16 then goes as far down from it as it can.
template <int ELEM> constexpr int kUp = ELEM == E4M3 ? 7 : ELEM == E5M2 ? 0 : 13;
// Octaves that scales of K of 32 keys may differ by: all element codes are exact in the operand then.
template <int ELEM> constexpr int kSpread = ELEM == E4M3 ? 22 : ELEM == E5M2 ? 8 : 36;
constexpr __host__ __device__ float down_by(int up) { return 1.0f / (float)(1 << up); }
// 2^d in both halves (0 below 2^-24), d at most 15
__device__ __forceinline__ uint32_t power2(int d) { return pack2(__half(), __uint_as_float((uint32_t)(max(d, -40) + 127) << 23), __uint_as_float((uint32_t)(max(d, -40) + 127) << 23)); }

// The parts of a unit that a CTA's run covers, one after the other, for each role alike.
struct Run {
  uint32_t at, stop, begin;
  int b;
  int len, steps, u, s0, s1, h, row0, ql, first;
  __device__ __forceinline__ Run(const Call& a, int lane) {
    uint32_t share;
    b = locate(a, gridDim.x, blockIdx.x, share, begin, lane);
    at = blockIdx.x * share;
    stop = at + min(share, ~at);
  }
  __device__ __forceinline__ bool next(const Call& a) {
    if (b >= a.B || at >= stop) return false;
    len = length_of(a, b);
    steps = steps_of(a, len);
    const uint32_t off = at - begin, units = a.cache.Hkv * a.groups;
    u = off / (uint32_t)steps;
    s0 = off - u * (uint32_t)steps;
    s1 = min((uint32_t)steps, s0 + (stop - at));
    h = u / a.groups;
    row0 = u % a.groups * kWideRows;
    ql = queries_of(a, b, len);
    first = len - ql;
    at += s1 - s0;
    now = b;
    if (at - begin >= (uint32_t)steps * units) {
      begin += (uint32_t)steps * units;
      ++b;
    }
    return true;
  }
  int now;                                             // the sequence
};

// Keys on their way: a warp's 32 rows of K or V, and the scale codes of key `lane`.  A load takes rpi rows; which row and which 16 bytes a lane
// has is chosen so that the lanes that store together meet different banks.
template <int ELEM, int D>
struct Rows {
  static constexpr int row = code_bytes(ELEM, D), cpr = row / 16, rpi = 32 / cpr;
  uint4 code[cpr];
  uint32_t scale;
  static __device__ __forceinline__ int piece(int lane) {
    return cpr == 8 ? (lane & 3) | (lane >> 1 & 4) : cpr == 4 && ELEM == E2M1 ? (lane & 1) | (lane >> 2 & 2) : lane % cpr;
  }
  static __device__ __forceinline__ int key(int lane) {
    return cpr == 8 ? (lane >> 2 & 1) | (lane >> 3 & 2) : cpr == 4 && ELEM == E2M1 ? (lane >> 1 & 3) | (lane >> 2 & 4) : lane / cpr;
  }
};

// 16 bytes, or zeros: one predicated load.  (Written in C++ it becomes a choice between the loaded value and zero, which waits for the load.)
__device__ __forceinline__ void load16(uint4& r, const void* p, bool there) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
               "@p ld.global.v4.b32 {%0,%1,%2,%3}, [%4];\n\t}" : "=&r"(r.x), "=&r"(r.y), "=&r"(r.z), "=&r"(r.w) : "l"(p), "r"((uint32_t)there) : "memory");
}

// Rows at the warp's 32 keys; at: row of key `lane` in the cache (fewer than 2^32 fit the memory), kNone where there is none (16 keys lie side
// by side in a page)
constexpr uint32_t kNone = ~0u;
template <int ELEM, int D>
__device__ __forceinline__ void request(Rows<ELEM, D>& r, const void* codes, const void* scales, uint32_t at, int keys, int lane) {
  using R = Rows<ELEM, D>;
  const uint32_t there = at != kNone && lane < keys;
  if constexpr (D == 128)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "=&r"(r.scale)
                 : "l"(static_cast<const uint32_t*>(scales) + at), "r"(there) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.u16 %0, [%1];\n\t}" : "=&r"(r.scale)
                 : "l"(static_cast<const unsigned short*>(scales) + at), "r"(there) : "memory");
  const int key = R::key(lane);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t base = __shfl_sync(0xffffffffu, at, 16 * half);
    const uint8_t* const p = static_cast<const uint8_t*>(codes) + ((unsigned long long)base + key) * R::row + R::piece(lane) * 16;
#pragma unroll
    for (int i = 0; i < R::cpr / 2; ++i) {
      load16(r.code[half * (R::cpr / 2) + i], p + i * R::rpi * R::row, base != kNone && 16 * half + i * R::rpi + key < keys);
    }
  }
}

// fp16 rows into shared memory.  factors (shared memory of the warp): what the blocks of each key are multiplied by; base: the scale code of key
// `lane` that stands for 2^kUp; nan: what a NaN scale becomes.
template <int ELEM, int D>
__device__ __forceinline__ void convert(const Rows<ELEM, D>& r, uint32_t tile, int row0, uint32_t factors, int base, uint32_t nan, int lane) {
  using R = Rows<ELEM, D>;
  constexpr int NB = D / 32;
  uint32_t f[4] = {};
  // E5M2: codes reach 2^16, and a factor below 2^-24 would be nothing where the product is not yet.  Such blocks are multiplied twice.
  bool again = false;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const uint32_t e = r.scale >> (8 * i) & 255u;
    const int d = (int)e - base + kUp<ELEM>;
    f[i] = e == 255u ? nan : power2(ELEM == E5M2 && e >= 2u ? max(d, -24) : d);
    if (ELEM == E5M2) again |= d < -24 && e >= 2u;
  }
  __syncwarp();
  store_shared16(factors + 16 * lane, f[0], f[1], f[2], f[3]);
  __syncwarp();
  // A row's 16-byte pieces lie exclusive-ored with the row's last three bits: for one lane the places of all its pieces differ from the first
  // one's by bits that are known here (rows of one lane are rpi apart) and by whole rows.
  const int ch = R::piece(lane), key = R::key(lane);
  constexpr int out = ELEM == E2M1 ? 4 : 2;            // pieces that 16 bytes of codes become
  constexpr int halves = 8 / out;                      // code pieces of 64 depth elements
  const uint32_t first = tile + ch / halves * (128 * 128) + (row0 + key) * 128 + ((ch % halves * out) ^ (key & 7)) * 16;
  const uint32_t mul = factors + 16 * key + 4 * (ELEM == E2M1 ? ch : ch / 2);
#pragma unroll
  for (int i = 0; i < R::cpr; ++i) {
    uint32_t m;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(m) : "r"(mul + i * R::rpi * 16) : "memory");
    const uint32_t w[4] = {r.code[i].x, r.code[i].y, r.code[i].z, r.code[i].w};
#pragma unroll
    for (int j = 0; j < out; ++j) {
      uint32_t x[4];
      if constexpr (ELEM == E2M1) {
        elem_quads(w[j], x[0], x[1], x[2], x[3]);
      } else {
        elem_two<ELEM>(w[2 * j], x[0], x[1]);
        elem_two<ELEM>(w[2 * j + 1], x[2], x[3]);
      }
      store_shared16((first ^ (16 * j + (R::rpi == 4 ? i % 2 * 64 : 0))) + i * R::rpi * 128, times(x[0], m), times(x[1], m), times(x[2], m), times(x[3], m));
    }
  }
  if (ELEM == E5M2 && __any_sync(0xffffffffu, again)) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t e = r.scale >> (8 * i) & 255u;
      f[i] = power2(e >= 2u && e < 255u ? min((int)e - base + kUp<ELEM> + 24, 0) : 0);
    }
    __syncwarp();
    store_shared16(factors + 16 * lane, f[0], f[1], f[2], f[3]);
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < R::cpr * out; ++i) {           // (each lane what it has written itself)
      const int n = i / out;
      const uint32_t at = (first ^ (16 * (i % out) + (R::rpi == 4 ? n % 2 * 64 : 0))) + n * R::rpi * 128;
      uint32_t m, x[4];
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(m) : "r"(mul + n * R::rpi * 16) : "memory");
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
      store_shared16(at, times(x[0], m), times(x[1], m), times(x[2], m), times(x[3], m));
    }
  }
}

// Which of the 32 keys from j0 on (counted among the query tokens) token `tok` sees.
__device__ uint32_t seen_keys(const unsigned char* mask, int j0, int tok, int ql) {
  const uint32_t before = j0 >= 0 ? 0u : j0 <= -32 ? ~0u : ~0u >> (32 + j0);           // bits below -j0: cached before the query tokens
  if (tok >= ql || j0 <= -32) return before;
  const int n = min((mask ? ql : tok + 1) - j0, 32);                                   // bits below n can be set
  if (n <= 0) return before;
  const uint32_t range = (~0u >> (32 - n)) & ~before;
  if (!mask) return before | range;
  uint32_t v = 0;
#pragma unroll 8
  for (int i = 0; i < 32; ++i)
    if (range >> i & 1) v |= (uint32_t)(mask[j0 + i] != 0) << i;
  return before | v;
}

template <typename T, int ELEM, int D>
__global__ void __launch_bounds__(kThreads, kWideCtas) kv_attention_wide_kernel(const __grid_constant__ Call a) {
  using Y = Layout<D>;
  constexpr int NB = D / 32;
  extern __shared__ uint8_t raw[];
  __shared__ Shared sh;
  uint8_t* const smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = a.Hq / a.cache.Hkv, R = a.T * G;

  grid_dependency_wait();                              // (before TMEM is taken: whoever is before may still need it)
  if (warp == 7) {
    tmem_alloc(&sh.tmem, kColumns);
    if (lane == 0) {
      mbar_init(&sh.k_full, 128);
      mbar_init(&sh.v_full, 128);
      mbar_init(&sh.s_full, 1);
      mbar_init(&sh.p_full, 128);
      mbar_init(&sh.pv_done, 1);
      mbar_init(&sh.q_full, 128);
      mbar_init(&sh.drained, 1);
      fence_mbar_init();
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  grid_dependents_go();

  Run run(a, lane);
  uint32_t n = 0;                                      // steps so far: every barrier but q_full completes once a step
  uint32_t units = 0;
  bool ok = true;

  const uint32_t qt = smem_u32(smem + Y::q), kt = smem_u32(smem + Y::k), vt = smem_u32(smem + Y::v);
  if (warp < 4) {
    // ---- softmax: row warp * 32 + lane of the unit; warp 0 issues the tensor operations too
    constexpr uint32_t kQk = idesc_f16(0, 0, 128, 128), kPv = idesc_f16(0, 0, 128, D) | 1u << 16;     // (bit 16: B is MN-major)
    // Q K^T of step n.  (S, where P was, is free: P V of the step before has been waited for.)
    auto qk = [&]() {
      if (!mbar_wait(&sh.k_full, n & 1, a.status, KS_TIMEOUT_PIPE)) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          mma_f16_ss(tmem, sdesc_kmajor_sw128(qt + i / 4 * Y::half + i % 4 * 32), sdesc_kmajor_sw128(kt + i / 4 * Y::half + i % 4 * 32), kQk, i > 0);
        tc_commit(&sh.s_full);
      }
      __syncwarp();
      return true;
    };
    auto pv = [&]() {
      if (!mbar_wait(&sh.p_full, n & 1, a.status, KS_TIMEOUT_PIPE) || !mbar_wait(&sh.v_full, n & 1, a.status, KS_TIMEOUT_PIPE)) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < 8; ++i) mma_f16_ts(tmem + 128, tmem + 8 * i, make_sdesc(vt + i * 2048, Y::half, 1024, kLayoutSw128), kPv, 1);
        tc_commit(&sh.pv_done);
      }
      __syncwarp();
      return true;
    };
    const uint32_t mine = tmem + (uint32_t)(warp * 32) * 65536u;
    for (; ok && run.next(a); ++units) {
      const int r = run.row0 + warp * 32 + lane, tok = r / G, hq = run.h * G + r % G;
      const bool live = r < R, busy = run.row0 + warp * 32 < R;        // busy: the warp has rows
      // queries (every Q K^T of the unit before is over: this thread has seen its scores)
      float rs = 0.0f;
      {
        const T* q = static_cast<const T*>(a.q) + (run.now * a.q_sb + hq * a.q_sh + (long long)tok * a.q_sl);
        uint32_t amax = 0;
        if (live)
          for (int i = 0; i < D / 4; ++i) {
            float x[4];
            load4(q + 4 * i, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) amax = max(amax, __float_as_uint(x[e]) & 0x7fffffffu);
          }
        const int e = min(max((int)(amax >> 23), 1), 253);
        const float down = __uint_as_float((uint32_t)(254 - e) << 23);
        rs = amax >= 0x7f800000u ? __int_as_float(0x7fffffff) : a.sm_scale * 1.44269504f * __uint_as_float((uint32_t)e << 23);
        const int row = warp * 32 + lane;
        const uint32_t to = smem_u32(smem + Y::q) + row * 128;
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          float x[4] = {}, y[4] = {};
          if (live) {
            load4(q + 8 * i, x);
            load4(q + 8 * i + 4, y);
          }
          store_shared16(to + i / 8 * Y::half + ((i % 8) ^ (row & 7)) * 16, pack2(__half(), x[0] * down, x[1] * down), pack2(__half(), x[2] * down, x[3] * down),
                         pack2(__half(), y[0] * down, y[1] * down), pack2(__half(), y[2] * down, y[3] * down));
        }
        fence_proxy_async_smem();
        const uint32_t zero[16] = {};
#pragma unroll
        for (int i = 0; i < D / 16; ++i) tmem_st16(mine + 128 + 16 * i, zero);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sh.q_full);
        if (warp == 0) ok = mbar_wait(&sh.q_full, units & 1, a.status, KS_TIMEOUT_PIPE) && qk();
      }
      float U = -INFINITY, l = 0.0f;
      for (int s = run.s0; ok && s < run.s1; ++s) {
        if (!(ok = mbar_wait(&sh.s_full, n & 1, a.status, KS_TIMEOUT_MMA))) break;
        tc_fence_after();
        const int par = n & 1, pos = s * kWideStep;
        if (busy) {
          const bool special = pos + kWideStep > (a.T > 1 || a.mask ? run.first : run.len) ||
                               *reinterpret_cast<const uint32_t*>(sh.odd[par]) != 0u;
          auto scores = [&](int c, uint32_t (&x)[32]) { // of 32 keys, in units of the largest
            tmem_ld32(mine + 32 * c, x);
            tmem_ld_wait();
            if (sh.uneven[par][c])
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * sh.k_part[par][32 * c + i]);
          };
          bool done = false;
          if (!special && __all_sync(0xffffffffu, U != -INFINITY)) {
            // as it is: products in registers, and over S if none has become too large
            uint32_t p[64], top = 0;
            float sum = 0.0f, sum2 = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t x[32];
              tmem_ld32(mine + 32 * c, x);
              const float f = rs * sh.k_size[par][c];
              const float* const vs = &sh.v_size[par][32 * c];
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = exp2_fast(fmaf(__uint_as_float(x[i + e]), f, -U));
                sum += y[0] + y[1];
                sum2 += y[2] + y[3];
                const float4 v = *reinterpret_cast<const float4*>(vs + i);
                uint32_t* const q = p + 16 * c + i / 2;
                q[0] = pack2(__half(), y[0] * v.x, y[1] * v.y);
                q[1] = pack2(__half(), y[2] * v.z, y[3] * v.w);
                top = __vmaxu2(top, __vmaxu2(q[0], q[1]));
              }
            }
            const float now = l + (sum + sum2);
            // (a product of more than 2^15 is 0x7801 or more, an infinity or a NaN among them; none is negative)
            done = !__any_sync(0xffffffffu, __vcmpgtu2(top, 0x78007800u) != 0 || !(now < 0x1p115f));
            if (done) {
              l = now;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = p[16 * c + i];
                tmem_st16(mine + 16 * c, w);
              }
            }
          }
          uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};      // keys that this row sees
          if (!__all_sync(0xffffffffu, done)) {
            if (special) {
              const unsigned char* const mk = a.mask ? a.mask + run.now * a.mask_sb + (long long)min(tok, a.T - 1) * a.T : nullptr;
#pragma unroll
              for (int c = 0; c < 4; ++c) vis[c] = seen_keys(mk, pos + 32 * c - run.first, live ? tok : a.T, run.ql) & sh.there[par][c];
            }
            // The largest product.  Scores are rounded before anything is added to them, here and below: the largest one must come out as the same
            // number, as where U is large, what a fused product keeps in its last bits is more than all a weight can be.
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t x[32];
              scores(c, x);
              const float f = rs * sh.k_size[par][c];
              const uint32_t seen = c == 0 ? vis[0] : c == 1 ? vis[1] : c == 2 ? vis[2] : vis[3];
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float y = __fmul_rn(__uint_as_float(x[i]), f) + sh.v_log[par][32 * c + i];
                top = fmaxf(top, seen >> i & 1 ? y : -INFINITY);
              }
            }
            const bool raise = top > U + kMost;
            if (__any_sync(0xffffffffu, raise)) {
              const float up = raise ? top - kSet : U, w = raise ? exp2_fast(U - up) : 1.0f;
              if (__any_sync(0xffffffffu, raise && U != -INFINITY)) { // (P V of the step before is over: Q K^T was issued behind it)
#pragma unroll 1
                for (int i = 0; i < D / 16; ++i) {
                  uint32_t x[16];
                  tmem_ld16(mine + 128 + 16 * i, x);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * w);
                  tmem_st16(mine + 128 + 16 * i, x);
                }
              }
              if (raise) l = lowered(l, U - up);
              U = up;
            }
            const float ref = U == -INFINITY ? 0.0f : U;
            // P times V's factors over S: columns 16c .. of the 32c .. that have been read
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t x[32], p[16];
              scores(c, x);
              const float f = rs * sh.k_size[par][c];
              const float* const vs = &sh.v_size[par][32 * c];
              const uint32_t seen = c == 0 ? vis[0] : c == 1 ? vis[1] : c == 2 ? vis[2] : vis[3];
              float sum = 0.0f;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float y[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  y[e] = exp2_fast(__fmul_rn(__uint_as_float(x[i + e]), f) - ref);
                  if (!(seen >> (i + e) & 1)) y[e] = 0.0f;
                }
                sum += y[0] + y[1];
                p[i / 2] = pack2(__half(), y[0] * vs[i], y[1] * vs[i + 1]);
              }
              l += sum;
              tmem_st16(mine + 16 * c, p);
            }
          }
          // a value that is NaN: its block of the depth is, in the rows that see it
          uint32_t any = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NB; ++i) any |= sh.strange[par][c][i];
          if (any) {
            tmem_st_wait();
#pragma unroll 1
            for (int i = 0; i < NB; ++i) {
              uint32_t hit = 0;
#pragma unroll
              for (int c = 0; c < 4; ++c) hit |= sh.strange[par][c][i] & vis[c];
#pragma unroll 1
              for (int y = 0; y < 2; ++y) {
                uint32_t x[16];
                tmem_ld16(mine + 128 + 32 * i + 16 * y, x);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = hit ? 0x7fffffffu : x[e];
                tmem_st16(mine + 128 + 32 * i + 16 * y, x);
              }
            }
          }
          tmem_st_wait();
        }
        tc_fence_before();
        mbar_arrive(&sh.p_full);
        if (warp == 0 && !(ok = pv())) break;
        ++n;
        if (warp == 0 && s + 1 < run.s1) ok = mbar_wait(&sh.pv_done, (n - 1) & 1, a.status, KS_TIMEOUT_MMA) && qk();
      }
      if (!ok || !(ok = mbar_wait(&sh.pv_done, (n - 1) & 1, a.status, KS_TIMEOUT_MMA))) break;
      tc_fence_after();
      if (!busy) continue;
      const bool whole = run.s0 == 0 && run.s1 == run.steps;
      const long long slot = (2ll * blockIdx.x + (run.s0 == 0)) * kWideRows + warp * 32 + lane;
      const bool none = l == 0.0f || tok >= run.ql;
      const float w = !whole ? down_by(kUp<ELEM>) : none ? 0.0f : down_by(kUp<ELEM>) / l;
      T* const y = static_cast<T*>(a.out) + (run.now * a.o_sb + hq * a.o_sh + (long long)tok * a.o_sl);
#pragma unroll 1
      for (int i = 0; i < D / 16; ++i) {
        uint32_t x[16];
        tmem_ld16(mine + 128 + 16 * i, x);
        tmem_ld_wait();
        if (live)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float z[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) z[d] = whole && none ? 0.0f : __uint_as_float(x[e + d]) * w;
            if (whole) store4(y + 16 * i + e, z);
            else store4(a.part + slot * D + 16 * i + e, z);
          }
      }
      tc_fence_before();
      if (live) {
        if (!whole) a.stat[slot] = make_float2(U, l);
        else if (a.lse) static_cast<float*>(a.lse)[((long long)run.now * a.Hq + hq) * a.T + tok] = none ? -INFINITY : U + log2f(l);
      }
    }
    if (warp == 0 && !ok) {                            // what has been issued ends before its memory goes
      if (elect_one()) {
        tc_commit(&sh.drained);
        mbar_drain(&sh.drained, 0);
      }
      __syncwarp();
    }
  } else {
    // ---- conversion: keys 32 (warp - 4) .. of every step
    const int w = warp - 4, shift = __popc(a.cache.page_size - 1);
    const uint32_t factors = smem_u32(smem + Y::factors) + w * (32 * 16);
    const mpsa_kv_cache& c = a.cache;
    Rows<ELEM, D> k, v;
    bool more = run.next(a);                           // `run` is one step ahead, at what is requested
    int as = more ? run.s0 : 0, keys = 0;
    uint32_t at = kNone;
    // the table's entries for this lane's key of step `as` and the two behind it: asked for two steps early, and the rows brought to L2 one step early
    auto entry_of = [&](int step) {
      const int e = (kWideStep * step + 32 * w + lane) >> shift;
      int r;
      asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, -1;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "=&r"(r)
                   : "l"(a.page_table + run.now * a.table_sb + e), "r"((uint32_t)(more && step < run.s1 && e < a.max_pages)) : "memory");
      return r;
    };
    int entry = -1, after = entry_of(as), later = entry_of(as + 1);
    auto row_of = [&](int e, int pos) {
      return (unsigned)e < (unsigned)c.num_pages ? (((uint32_t)e * c.Hkv + run.h) << shift) + ((pos + lane) & (c.page_size - 1)) : kNone;
    };
    auto look_up = [&]() {
      const int pos = kWideStep * as + 32 * w;
      at = row_of(entry, pos);
      keys = run.len - pos;
      const uint32_t row = row_of(after, pos + kWideStep);
      if (row != kNone && lane < keys - kWideStep) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(c.k) + (unsigned long long)row * code_bytes(ELEM, D)));
        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(c.v) + (unsigned long long)row * code_bytes(ELEM, D)));
      }
    };
    // A turn converts a step (the first one none) and requests the one behind it.  Each operand is requested in one place: where two places
    // meet, the loaded registers are copied, and a copy waits for the load.
    for (bool have = false;;) {
      const int par = n & 1;
      const bool now = have, here = at != kNone && lane < keys;
      if (now && ++as == run.s1) {
        more = run.next(a);
        as = more ? run.s0 : 0;
        after = entry_of(as);
        later = entry_of(as + 1);
      }
      uint32_t vtop = 0;
      have = more;
      entry = after;
      after = later;
      later = entry_of(as + 2);
      look_up();
      if (now) {
        // One reference for the warp's keys of K where they are alike, one for each key of V, and for each of K otherwise: a key that a row
        // does not see, or gives no weight, may be larger than the rest by far.  (Codes 0 and 1 are blocks of nothing: no element reaches 2^-110.)
        uint32_t own = 0, low = 255;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const uint32_t e = k.scale >> (8 * i) & 255u;
          own = max(own, e == 255u ? 0u : e);
          low = min(low, e < 2u ? 255u : e);
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, own);
        const bool uneven = __any_sync(0xffffffffu, low + kSpread<ELEM> < top);
        if (uneven) sh.k_part[par][32 * w + lane] = __uint_as_float((uint32_t)max(127 - (int)(top - own), 0) << 23);
        if (n > 0 && !(ok = mbar_wait(&sh.s_full, (n - 1) & 1, a.status, KS_TIMEOUT_MMA))) break;      // K is free
        convert<ELEM, D>(k, kt, 32 * w, factors, (int)(uneven ? own : top), 0x7fff7fffu, lane);
        // (the scales of V were requested last: they have had K's conversion to come in)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const uint32_t e = v.scale >> (8 * i) & 255u;
          vtop = max(vtop, e == 255u ? 0u : e);
          const uint32_t strange = __ballot_sync(0xffffffffu, e == 255u);
          if (lane == 0) sh.strange[par][w][i] = strange;
        }
        sh.v_size[par][32 * w + lane] = scale_value(vtop);
        sh.v_log[par][32 * w + lane] = fmaxf((float)((int)vtop - 127), kLeast);
        const uint32_t has = __ballot_sync(0xffffffffu, here);
        if (lane == 0) {
          sh.there[par][w] = has;
          sh.uneven[par][w] = uneven;
          sh.odd[par][w] = uneven || has != 0xffffffffu;
          sh.k_size[par][w] = scale_value(top) * down_by(kUp<ELEM>);
        }
        fence_proxy_async_smem();
        mbar_arrive(&sh.k_full);
      }
      request<ELEM, D>(k, c.k, c.k_scale, at, keys, lane);
      if (now) {
        if (n > 0 && !(ok = mbar_wait(&sh.pv_done, (n - 1) & 1, a.status, KS_TIMEOUT_MMA))) break;     // V is free
        convert<ELEM, D>(v, vt, 32 * w, factors, (int)vtop, 0u, lane);
        fence_proxy_async_smem();
        mbar_arrive(&sh.v_full);
        ++n;
      }
      if (!have) break;
      request<ELEM, D>(v, c.v, c.v_scale, at, keys, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 7) tmem_dealloc(tmem, kColumns);
}

template <typename T, int ELEM, int D>
int launch(const Call& a, int ctas, cudaStream_t st) {
  constexpr int id = 100000 + (std::is_same_v<T, __half> ? 1 : 0) + ELEM * 10 + D * 100;
  const auto kernel = kv_attention_wide_kernel<T, ELEM, D>;
  if (!allow_smem<id>(kernel, Layout<D>::bytes)) return set_error(MPSA_ERR_LAUNCH, "kv_attention: shared memory not granted");
  launch_dependent(kernel, dim3(ctas), kThreads, Layout<D>::bytes, st, overlaps_previous(st), a);
  return check_launch("kv_attention");
}
template <typename T, int ELEM>
int launch_depth(const Call& a, int ctas, cudaStream_t st) {
  return a.cache.D == 64 ? launch<T, ELEM, 64>(a, ctas, st) : launch<T, ELEM, 128>(a, ctas, st);
}
template <typename T>
int launch_elem(const Call& a, int ctas, cudaStream_t st) {
  return a.cache.elem == E4M3 ? launch_depth<T, E4M3>(a, ctas, st) : a.cache.elem == E5M2 ? launch_depth<T, E5M2>(a, ctas, st) : launch_depth<T, E2M1>(a, ctas, st);
}

}  // namespace

int launch_wide(const Call& a, int ctas, cudaStream_t st) { return a.dtype == 0 ? launch_elem<__nv_bfloat16>(a, ctas, st) : launch_elem<__half>(a, ctas, st); }

}  // namespace mpsa
