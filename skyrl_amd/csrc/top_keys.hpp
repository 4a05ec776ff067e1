// What the kernels that look for the best logits of a row have in common: keys that sort as (logit, lower column first) do, a wave's list of
// candidates, and the bound that few logits reach.
#pragma once
#include "logits_rows.hpp"

namespace logits {

typedef unsigned long long topkey_t;

constexpr int kGroups = 128;  // of four lanes, whose maxima bound the k-th largest logit from below
constexpr int kWaveList = 256;  // candidates a wave holds before it drops all but its k best

// Bits of a float that compare as the floats do; 0 for NaN, -0 as +0.
__device__ __forceinline__ uint32_t ordered_bits(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return z != z ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of_bits(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
// A larger key sorts earlier.
__device__ __forceinline__ topkey_t make_key(float z, int column) { return ((topkey_t)ordered_bits(z) << 32) | (topkey_t)(uint32_t)(~column); }
__device__ __forceinline__ int key_column(topkey_t k) { return (int)(~(uint32_t)k); }
__device__ __forceinline__ uint32_t key_bits(topkey_t k) { return (uint32_t)(k >> 32); }

// LDS operations of a wave execute in order; this keeps the compiler from holding entries that another lane has rewritten.
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// The k largest of the n keys (k < n <= kWaveList) of a wave's list to its front, in any order; returns the smallest of them.  A bisection over
// the key bits on keys held in registers.
static __device__ __noinline__ topkey_t keep_best(topkey_t* list, int n, int k) {
  const int lane = threadIdx.x & 63;
  constexpr int B = kWaveList / 64;
  topkey_t x[B];
#pragma unroll
  for (int u = 0; u < B; ++u) x[u] = u * 64 + lane < n ? list[u * 64 + lane] : 0;  // 0 reaches no trial
  topkey_t reach = 0;
  for (int b = 63; b >= 0; --b) {
    const topkey_t trial = reach | ((topkey_t)1 << b);
    int c = 0;
#pragma unroll
    for (int u = 0; u < B; ++u) c += (int)__popcll(__ballot(x[u] >= trial));
    if (c >= k) reach = trial;  // all 64 bits: `reach` ends as the k-th largest key
  }
  wave_fence();
  int w = 0;
#pragma unroll
  for (int u = 0; u < B; ++u) {
    const bool keep = u * 64 + lane < n && x[u] >= reach;
    const unsigned long long mask = __ballot(keep);
    if (keep) list[w + __popcll(mask & ((1ull << lane) - 1))] = x[u];
    w += (int)__popcll(mask);
  }
  wave_fence();
  return reach;
}

// A value that at least k of the 128 groups reach, from the first 16 bits of their maxima (exact for bf16); by one wave.
__device__ __forceinline__ float group_bound(const float* group_max, int k) {
  const int lane = threadIdx.x & 63;
  const uint32_t a = ordered_bits(group_max[lane]) >> 16, b = ordered_bits(group_max[64 + lane]) >> 16;
  uint32_t reach = 0;
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t trial = reach | (1u << bit);
    if ((int)(__popcll(__ballot(a >= trial)) + __popcll(__ballot(b >= trial))) >= k) reach = trial;
  }
  const uint32_t bits = reach << 16;
  return bits < 0x00800000u ? -INFINITY : value_of_bits(bits);  // NaN, or -inf: no bound yet
}

// Where `mine` stands among n keys of LDS.
__device__ __forceinline__ int place_among(const topkey_t* keys, int n, topkey_t mine) {
  int place = 0;
#pragma unroll 8
  for (int i = 0; i < n; ++i) place += keys[i] > mine ? 1 : 0;
  return place;
}

}  // namespace logits
