// What the two kernels of mpsa_kv_attention share: the call, how its work is cut into runs, and its parts.
//
// A unit of work is one sequence, one KV head and up to `rows` of its query rows (row r = token r / G, query head r % G of the KV head's G).
// A step is `step` keys.  The steps of all units, laid end to end, are cut into equal runs, one per CTA, whatever the lengths are: CTAs compute
// the cut from the lengths in device memory.  A unit that falls to several CTAs leaves parts (fp32 sums with their row references and
// denominators), which the combining kernel adds up in the order of the keys.
#pragma once
#include "common.cuh"
#include "serving.cuh"

namespace mpsa {

struct Call : mpsa_kv_attention_args {
  int rows;                                    // query rows of a unit, at most
  int step;                                    // keys of a step
  int least;                                   // steps of a run at least
  int groups;                                  // units of a (sequence, KV head)
  int cluster;                                 // CTAs of a unit: nobody else has part of it, and there are no runs (0: runs)
  float* part;                                 // [2 x CTAs][rows][D], a CTA's run has at most two units that it shares with others
  float2* stat;                                // [2 x CTAs][rows]: row reference (log2), denominator relative to it
};

__device__ __forceinline__ int length_of(const Call& a, int b) {
  return min(max(a.lengths[b], 0), (int)min(0x7ffffe00ll, (long long)a.max_pages * a.cache.page_size));
}
__device__ __forceinline__ int queries_of(const Call& a, int b, int len) { return min(a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T, len); }
__device__ __forceinline__ int steps_of(const Call& a, int len) { return max(1, (len + a.step - 1) / a.step); }    // (an empty sequence: one, which writes its zeros)

// How many steps of all units a CTA takes (`share`), the sequence that step cta * share belongs to (returned; a.B: beyond the last) and where
// that sequence's steps begin.  By a whole warp; plan() has seen to it that the steps of all units fit 32 bits.
__device__ __forceinline__ int locate(const Call& a, uint32_t ctas, uint32_t cta, uint32_t& share, uint32_t& begin, int lane) {
  const uint32_t units = a.cache.Hkv * a.groups;
  const uint32_t mine = lane < a.B ? steps_of(a, length_of(a, lane)) * units : 0;       // the first 32 sequences: read once
  uint32_t sum = mine;
  for (int b = lane + 32; b < a.B; b += 32) sum += steps_of(a, length_of(a, b)) * units;
  sum = __reduce_add_sync(0xffffffffu, sum);
  share = max((sum + ctas - 1) / ctas, (uint32_t)a.least);
  const unsigned long long want = (unsigned long long)cta * share;
  begin = 0;
  if (want >= sum) return a.B;
  const uint32_t at = (uint32_t)want;
  for (int b0 = 0;; b0 += 32) {
    const uint32_t n = b0 == 0 ? mine : b0 + lane < a.B ? steps_of(a, length_of(a, b0 + lane)) * units : 0;
    uint32_t up = n;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, up, d);
      if (lane >= d) up += v;
    }
    const unsigned beyond = __ballot_sync(0xffffffffu, begin + up > at);
    if (beyond) {
      const int l = __ffs(beyond) - 1;
      begin += __shfl_sync(0xffffffffu, up - n, l);
      return b0 + l;
    }
    begin += __shfl_sync(0xffffffffu, up, 31);
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A denominator relative to a reference 2^-d as large, d at most 0 (-infinity with l = 0).  In two steps where 2^d is no number: keys without values
// set a reference that may be 2^-200 of another's, and their denominators are as much larger.
__device__ __forceinline__ float lowered(float l, float d) {
  const float a = fmaxf(d, -100.0f);
  return l * exp2_fast(a) * exp2_fast(d - a);
}

// Many query rows (csrc/decode_wide.cu): launches the kernel that leaves whole units in a.out and parts in a.part, a.stat.
constexpr int kWideRows = 128, kWideStep = 128, kWideCtas = 2;       // CTAs of an SM
int launch_wide(const Call& a, int ctas, cudaStream_t st);

}  // namespace mpsa
