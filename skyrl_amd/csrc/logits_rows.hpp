// What the kernels that walk rows of materialised logits have in common: the 16-byte pieces of a row, and the running statistics of a softmax.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "../../include/skyrl_lmhead.h"

namespace logits {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.0e38f;  // start of a running maximum: finite, so that (-inf) - max is -inf and never NaN
// A logit of -inf (a masked vocabulary entry) has probability exactly 0; in the products z * p it is taken as this finite
// value so that 0 * inf does not turn the row into NaN (the reference's entropy does return NaN there, torch_utils.py:99-100).
constexpr float kMostNegativeFactor = -1.0e30f;

// Eight bf16 or four fp32 logits of one 16-byte piece, widened to fp32.
template <bool F32>
struct Piece {
  static constexpr int kElems = F32 ? 4 : 8;
  float v[kElems];
  __device__ __forceinline__ void load(const void* p) { widen(*(const u32x4*)p); }
  __device__ __forceinline__ void widen(const u32x4& w) {
    if (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

// Where the 16-byte pieces of a row lie: logits [head, head + pieces * E); the other `single` logits are numbered head first.
struct RowPieces {
  int head, pieces, single;
};
template <bool F32>
__device__ __forceinline__ RowPieces row_pieces(const char* row, int V, bool vector_ok) {
  constexpr int E = Piece<F32>::kElems, ES = F32 ? 4 : 2;
  int head = (int)((16u - (uint32_t)((uintptr_t)row & 15u)) & 15u) / ES;
  head = head < V ? head : V;
  const int pieces = vector_ok ? (V - head) / E : 0;
  return RowPieces{head, pieces, V - pieces * E};
}
__device__ __forceinline__ int single_column(const RowPieces& r, int elems, int i) { return i < r.head ? i : i + r.pieces * elems; }

__device__ __forceinline__ float load_one(const void* base, size_t i, bool f32) {
  return f32 ? ((const float*)base)[i] : __uint_as_float((uint32_t)((const uint16_t*)base)[i] << 16);
}

__device__ __forceinline__ uint16_t bf16_bits(float x) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  const f32x2 pair = {x, 0.f};
  const bf16x2 b = __builtin_convertvector(pair, bf16x2);
  return (uint16_t)(*(const uint32_t*)&b & 0xffffu);
}

// Running statistics of a row in base 2, with y2 = z * log2e / temperature:  m = max y2,  s = sum 2^(y2 - m),
// e = sum (y2 - m) * 2^(y2 - m).  The third sum is kept relative to the maximum, like the other two, so that a large common
// offset of a row's logits costs no accuracy:  entropy = ln s - ln 2 * e / s,  logprob = ln 2 * (y2[label] - m) - ln s.
struct Stats {
  float m, s, e;
};

template <bool ENT>
__device__ __forceinline__ void absorb(Stats& st, float z, float scale2) {
  const float t = fmaf(z, scale2, -st.m);
  const float p = __builtin_amdgcn_exp2f(t);
  st.s += p;
  if (ENT) st.e = fmaf(fmaxf(t, kMostNegativeFactor), p, st.e);
}

// Sums taken relative to maximum `from`, re-expressed relative to `to` >= from.
__device__ __forceinline__ void rebase(float& s, float& e, float from, float to) {
  const float d = fmaxf(from - to, kMostNegativeFactor);  // <= 0; finite, so that d * 0 is 0 for an empty sum
  const float c = __builtin_amdgcn_exp2f(d);
  e = c * fmaf(d, s, e);
  s *= c;
}

// A running maximum for sums over logits up to z: z * scale2.  That product's rounding is what absorb() will see of z itself: +440 for a mask of -1e10, whose
// sum would be infinite, and NaN beside a larger maximum.  There it is a little above z, and the sum 0.
__device__ __forceinline__ float max_from(float z, float scale2) {
  const float y2 = z * scale2;
  return fmaf(z, scale2, -y2) > 64.f ? fmaf(fabsf(y2), 0x1p-22f, y2) : y2;
}
// Raise the running maximum to at least `to`, of max_from().
__device__ __forceinline__ void raise_max(Stats& st, float to) {
  if (to > st.m) {
    rebase(st.s, st.e, st.m, to);
    st.m = to;
  }
}

__device__ __forceinline__ void merge(Stats& a, const Stats& b) {
  const float m = fmaxf(a.m, b.m);
  float bs = b.s, be = b.e;
  rebase(a.s, a.e, a.m, m);
  rebase(bs, be, b.m, m);
  a.s += bs;
  a.e += be;
  a.m = m;
}

// The row's statistics in every thread of WAVES waves.
template <int WAVES>
__device__ __forceinline__ Stats block_merge(Stats st, Stats* sm) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    Stats other;
    other.m = __shfl_xor(st.m, o, 64);
    other.s = __shfl_xor(st.s, o, 64);
    other.e = __shfl_xor(st.e, o, 64);
    merge(st, other);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) sm[wave] = st;
  __syncthreads();
  Stats all = sm[0];
  for (int w = 1; w < WAVES; ++w) merge(all, sm[w]);
  return all;
}

// Statistics keep y2 = z * log2e / temperature in fp32, whose step at m is up to |m| * 2^-24: from |m| = 2^24 on the largest logit's own
// 2^(y2 - m) is anything, from about 2^31 on 0 or infinite, and y2 itself overflows for logits beyond 2.3e38 * temperature.  The row's logits
// may be ordinary but for a mask of -1e10 that one wave has seen nothing else of: an infinite sum shows that.
constexpr float kFar = 0x1p24f;
__device__ __forceinline__ bool is_far(const Stats& st) { return !(fabsf(st.m) < kFar && st.s < INFINITY); }

// Such a row's statistics from differences of logits, which do not overflow where it matters: m is the largest LOGIT, t = (z - m) * scale2, s = sum 2^t,
// e = sum t 2^t.  By a whole workgroup in two passes; sm: 2 * WAVES floats of LDS that nothing else is in.  -inf, 0, 0 where no logit is above -inf.
__device__ __forceinline__ float far_origin(float top) { return top > -INFINITY ? top : 0.f; }  // (-inf) minus it is -inf

template <bool F32, int WAVES>
__device__ __noinline__ Stats far_row(const char* base, int V, float scale2, float* sm) {
  constexpr int E = Piece<F32>::kElems;
  const RowPieces rp = row_pieces<F32>(base, V, true);
  const char* vec = base + (size_t)rp.head * (F32 ? 4 : 2);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto each = [&](auto f) {
    for (int p = tid; p < rp.pieces; p += WAVES * 64) {
      Piece<F32> pc;
      pc.load(vec + (size_t)p * 16);
#pragma unroll
      for (int i = 0; i < E; ++i) f(pc.v[i]);
    }
    for (int i = tid; i < rp.single; i += WAVES * 64) f(load_one(base, (size_t)single_column(rp, E, i), F32));
  };
  float top = -INFINITY, s = 0.f, e = 0.f;
  each([&](float z) { top = fmaxf(top, z); });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  __syncthreads();
  if (lane == 0) sm[wave] = top;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sm[w]);
  const float from = far_origin(top);
  each([&](float z) {
    const float t = (z - from) * scale2, p = __builtin_amdgcn_exp2f(t);
    s += p;
    e = fmaf(fmaxf(t, kMostNegativeFactor), p, e);
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64), e += __shfl_xor(e, o, 64);
  __syncthreads();
  if (lane == 0) sm[wave] = s, sm[WAVES + wave] = e;
  __syncthreads();
  s = e = 0.f;
  for (int w = 0; w < WAVES; ++w) s += sm[w], e += sm[WAVES + w];
  return Stats{top, s, e};
}

// The nearest finite value of a log-sum-exp or mean that may have left fp32.
__device__ __forceinline__ float finite(float x) { return x == INFINITY ? 3.402823466e38f : x == -INFINITY ? -3.402823466e38f : x; }

constexpr int64_t kCacheBytes = (int64_t)256 << 20;
constexpr int64_t kMaxRows = (int64_t)1 << 31;  // the grid's x extent

// Whether every row of b starts as far from a 16-byte boundary as the same row of a.
inline bool same_row_offsets(const void* a, int64_t lda, const void* b, int64_t ldb, bool f32) {
  return (((uintptr_t)a - (uintptr_t)b) & 15u) == 0 && (lda - ldb) * (f32 ? 4 : 2) % 16 == 0;
}

// A gradient is written in place, or apart: a buffer that overlaps the logits in any other way would be read after it was written.
inline bool overlaps_otherwise(const void* logits, int64_t ld_logits, const void* dlogits, int64_t ld_dlogits, int64_t T, int64_t V, bool f32) {
  if (dlogits == logits && ld_dlogits == ld_logits) return false;
  const char *a0 = (const char*)logits, *b0 = (const char*)dlogits;
  const size_t es = f32 ? 4 : 2;
  const char *a1 = a0 + ((size_t)(T - 1) * (size_t)ld_logits + (size_t)V) * es, *b1 = b0 + ((size_t)(T - 1) * (size_t)ld_dlogits + (size_t)V) * es;
  return a0 < b1 && b0 < a1;
}

inline int check_logits(const void* logits, int dtype, int64_t ld, int64_t T, int64_t V, float rcp_temperature) {
  if (!logits) return SKYRL_LMHEAD_ERR_NULL;
  if (dtype != SKYRL_LOGITS_BF16 && dtype != SKYRL_LOGITS_F32) return SKYRL_LMHEAD_ERR_ARG;
  if (T < 1 || V < 1 || ld < V || T >= kMaxRows || V >= ((int64_t)1 << 31) || ld >= ((int64_t)1 << 40)) return SKYRL_LMHEAD_ERR_SHAPE;
  if ((uintptr_t)logits & (dtype == SKYRL_LOGITS_F32 ? 3u : 1u)) return SKYRL_LMHEAD_ERR_ALIGN;
  if (!(rcp_temperature > 0.f) || !std::isfinite(rcp_temperature)) return SKYRL_LMHEAD_ERR_ARG;
  return SKYRL_LMHEAD_OK;
}

}  // namespace logits
