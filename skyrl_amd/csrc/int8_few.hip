// Few tokens and the head in 8-bit integers: the weight streams through registers.
//
// What bounds such a call is the weight coming from HBM, and a tile that stages it in LDS stops that stream at its start and its end
// (half_tile.hpp).  Here the hidden values of all tokens lie in LDS, in the order of the matrix instruction's operands, for the whole launch.  A wave
// takes 16 vocabulary rows at a time over the whole contraction, CH steps of them in registers, and loads each register anew as soon as its products are
// done: 56 KiB a CU are always on their way.  Per 16 rows and step NB LDS reads of 1 KiB and NB matrix instructions, which is what more tokens cost.
// Weights from HBM: 28 us at T=1, H=896, V=151936 (4.9 TB/s; half tiles 31), 94 to 99 us of statistics and 101 of logits at T=16, H=3584, V=152064 (5.4 to
// 5.8 TB/s; half tiles 118), 60 at T=64, H=2048.  At 96 tokens of H=896 it takes as long as half tiles (33 and 34 us), at 137 as long as square ones.
//   int8_logits_stream   writes the logits
//   int8_fwd_stream      keeps the running statistics of a lane, of each token block, in registers over all of its rows, so that a workgroup leaves
//                        one partial a token behind instead of one for every 128 rows
#include <type_traits>

#include "int8.hpp"

#include "logits_tile.hpp"

namespace lmhead {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int kStep = 64;    // k of a matrix instruction
constexpr int kRows = 16;    // vocabulary rows of one
constexpr int kStreamWaves = 8;
constexpr int64_t kStreamTokens = 64;
constexpr size_t kStreamLds = 150 * 1024;
constexpr size_t kJoinBytes = (size_t)3 * kStreamWaves * kStreamTokens * 4;  // the waves' statistics, in the hidden values' place

// consume(unit, v0, c, acc): the sums of 16 vocabulary rows, of which the lane has rows v0 .. v0 + 3 with scales c, and column lane & 15 of each token block.
template <int CH, int NB, class Args, class Consume>
__device__ __forceinline__ void stream_rows(const Args& a, char* hidden, Consume consume) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kq = lane >> 4;
  const int steps = a.K / kStep, chunks = (steps + CH - 1) / CH;
  const int units = (a.V + kRows - 1) / kRows;
  const int first = (int)((int64_t)units * blockIdx.x / gridDim.x), last = (int)((int64_t)units * (blockIdx.x + 1) / gridDim.x);
  auto row_of = [&](int unit) {
    int v = (unit < last ? unit : last - 1) * kRows + n;
    v = v < a.V ? v : a.V - 1;
    return a.W.values + (size_t)v * (size_t)a.W.ld + kq * 16;
  };
  i32x4 w[CH];
  const int8_t* row = row_of(first + wave);
#pragma unroll
  for (int s = 0; s < CH; ++s) w[s] = *(const i32x4*)(row + (s < steps ? s : steps - 1) * kStep);
  // Steps behind the contraction's end multiply whatever weight by zeros.
  for (int f = wave; f < chunks * CH * NB; f += kStreamWaves) {
    const int step = f / NB, t = (f - step * NB) * 16 + n;
    i32x4 h = {0, 0, 0, 0};
    if (step < steps) h = *(const i32x4*)(a.Hd.values + (size_t)(t < a.T ? t : a.T - 1) * (size_t)a.Hd.ld + step * kStep + kq * 16);
    *(i32x4*)(hidden + (f * 64 + lane) * 16) = h;
  }
  __syncthreads();
  for (int unit = first + wave; unit < last; unit += kStreamWaves) {
    // In front of the weights that are in flight when they are needed: loads return in order.
    const int v0 = unit * kRows + kq * 4;
    float c[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) c[r] = a.W.scale[v0 + r < a.V ? v0 + r : a.V - 1];
    i32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = i32x4{0, 0, 0, 0};
    const int8_t* const next_row = row_of(unit + kStreamWaves);
    for (int chunk = 0; chunk < chunks; ++chunk) {
      const bool more = chunk + 1 < chunks;
      const int8_t* const next = more ? row : next_row;
      const int step0 = more ? (chunk + 1) * CH : 0;
      const char* h = hidden + (chunk * CH * NB * 64 + lane) * 16;
#pragma unroll
      for (int s = 0; s < CH; ++s) {
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s], *(const i32x4*)(h + (s * NB + j) * 1024), acc[j], 0, 0, 0);
        w[s] = *(const i32x4*)(next + (step0 + s < steps ? step0 + s : steps - 1) * kStep);
      }
    }
    row = next_row;
    consume(unit, v0, c, acc);
  }
}

template <int CH, int NB, bool F32>
__global__ __launch_bounds__(kStreamWaves * 64) void int8_logits_stream(const Int8LogitsArgs a) {
  extern __shared__ __attribute__((aligned(16))) char hidden[];
  typedef float f32x4u __attribute__((ext_vector_type(4)));
  struct __attribute__((packed, aligned(4))) Four32 {
    f32x4u v;
  };
  struct __attribute__((packed, aligned(2))) Four16 {
    bf16x4 v;
  };
  const int n = threadIdx.x & 15;
  float s_t[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) s_t[j] = a.Hd.scale[j * 16 + n < a.T ? j * 16 + n : a.T - 1];
  stream_rows<CH, NB>(a, hidden, [&](int unit, int v0, const float (&c)[4], const i32x4 (&acc)[NB]) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int t = j * 16 + n;
      if (t >= a.T) continue;
      f32x4u z;
#pragma unroll
      for (int r = 0; r < 4; ++r) z[r] = (float)acc[j][r] * c[r] * s_t[j];
      char* const to = (char*)a.out + ((size_t)t * (size_t)a.ldo + (size_t)v0) * (F32 ? 4 : 2);
      if ((unit + 1) * kRows <= a.V) {
        if constexpr (F32) ((Four32*)to)->v = z;
        else ((Four16*)to)->v = __builtin_convertvector(z, bf16x4);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (v0 + r >= a.V) break;
          if constexpr (F32) ((float*)to)[r] = z[r];
          else ((__bf16*)to)[r] = (__bf16)z[r];
        }
      }
    }
  });
}

template <int CH, int NB, bool ENTROPY>
__global__ __launch_bounds__(kStreamWaves * 64) void int8_fwd_stream(const Int8FwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) char hidden[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & 15, kq = lane >> 4;
  float scale2[NB], m[NB], sum[NB], e[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int t = j * 16 + n;
    scale2[j] = a.Hd.scale[t < a.T ? t : a.T - 1] * a.rcp_temp * kLog2e;
    m[j] = kLowestMax, sum[j] = 0.f, e[j] = 0.f;
  }
  stream_rows<CH, NB>(a, hidden, [&](int unit, int v0, const float (&c)[4], const i32x4 (&acc)[NB]) {
    auto add = [&](auto masked) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float x[4], top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = (float)acc[j][r] * c[r];
          if (!masked || v0 + r < a.V) top = fmaxf(top, x[r]);
        }
        const float m2 = top * scale2[j];
        if (__any(m2 > m[j])) {  // by far the most often not: a few times for each token
          const float to = fmaxf(m[j], m2), d = m[j] - to, f = __builtin_amdgcn_exp2f(d);
          if (ENTROPY) e[j] = f * fmaf(fmaxf(d, -1.0e30f), sum[j], e[j]);
          sum[j] *= f;
          m[j] = to;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float t2 = fmaf(x[r], scale2[j], -m[j]);
          float p = __builtin_amdgcn_exp2f(t2);
          if (masked && v0 + r >= a.V) p = 0.f;
          sum[j] += p;
          if (ENTROPY) e[j] = fmaf(t2, p, e[j]);
        }
      }
    };
    if ((unit + 1) * kRows <= a.V) add(std::false_type{});
    else add(std::true_type{});
  });
  // One partial a token: the four lanes of a token, then the waves through LDS.
  auto join = [&](float& m0, float& s0, float& e0, float m1, float s1, float e1) {
    const float to = fmaxf(m0, m1), d0 = fmaxf(m0 - to, -1.0e30f), d1 = fmaxf(m1 - to, -1.0e30f);
    const float f0 = __builtin_amdgcn_exp2f(d0), f1 = __builtin_amdgcn_exp2f(d1);
    e0 = fmaf(f0, fmaf(d0, s0, e0), f1 * fmaf(d1, s1, e1));
    s0 = fmaf(f0, s0, f1 * s1);
    m0 = to;
  };
  __syncthreads();  // every wave has left the hidden values
  float* const all = (float*)hidden;  // [3][waves][NB * 16]
#pragma unroll
  for (int j = 0; j < NB; ++j) {
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1) {
      const float m1 = __shfl_xor(m[j], o, 64), s1 = __shfl_xor(sum[j], o, 64), e1 = __shfl_xor(e[j], o, 64);
      join(m[j], sum[j], e[j], m1, s1, e1);
    }
    if (kq == 0) {
      all[(0 * kStreamWaves + wave) * (NB * 16) + j * 16 + n] = m[j];
      all[(1 * kStreamWaves + wave) * (NB * 16) + j * 16 + n] = sum[j];
      all[(2 * kStreamWaves + wave) * (NB * 16) + j * 16 + n] = e[j];
    }
  }
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= a.T) return;
  float m0 = all[t], s0 = all[kStreamWaves * NB * 16 + t], e0 = all[2 * kStreamWaves * NB * 16 + t];
  for (int x = 1; x < kStreamWaves; ++x)
    join(m0, s0, e0, all[x * NB * 16 + t], all[(kStreamWaves + x) * NB * 16 + t], all[(2 * kStreamWaves + x) * NB * 16 + t]);
  const size_t at = part_index(blockIdx.x, t, gridDim.x);
  a.part_max[at] = m0 * kLn2;
  a.part_sum[at] = s0;
  if (ENTROPY) a.part_pz[at] = e0 * kLn2;
}

// Token blocks of the kernel that takes T tokens.
int stream_blocks(int64_t T) { return T <= 16 ? 1 : T <= 32 ? 2 : 4; }
// Steps in registers: the fewer steps behind the contraction's end the better.
int stream_chunk(int64_t K) {
  const int64_t steps = K / kStep;
  return (steps + 6) / 7 * 7 < (steps + 7) / 8 * 8 ? 7 : 8;
}
size_t stream_lds(int64_t T, int64_t K) {
  const int64_t ch = stream_chunk(K);
  return (size_t)((K / kStep + ch - 1) / ch * ch * stream_blocks(T)) * 1024;
}
// One workgroup a CU.  (Two: 99 -> 105 us at T=32, H=3584, 60 -> 66 at T=64, H=2048; at H=896 the same.)
int stream_grid(int64_t V, int64_t most) {
  const int64_t units = (V + kRows - 1) / kRows;
  return (int)(most < units ? most : units);
}

// pick(chunk, blocks, flag) for those of a call as compile-time constants, launched.
template <class Pick, class Args>
hipError_t launch_stream(hipStream_t s, const Args& a, bool flag, int grid, Pick pick) {
  const size_t lds = stream_lds(a.T, a.K);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kStreamWaves * 64), lds > kJoinBytes ? lds : kJoinBytes, s, a); };
  auto with = [&](auto ch, auto f) {
    const int blocks = stream_blocks(a.T);
    if (blocks == 1) go(pick(ch, std::integral_constant<int, 1>{}, f));
    else if (blocks == 2) go(pick(ch, std::integral_constant<int, 2>{}, f));
    else go(pick(ch, std::integral_constant<int, 4>{}, f));
  };
  const std::integral_constant<int, 7> seven;
  const std::integral_constant<int, 8> eight;
  if (stream_chunk(a.K) == 7) flag ? with(seven, std::true_type{}) : with(seven, std::false_type{});
  else flag ? with(eight, std::true_type{}) : with(eight, std::false_type{});
  return hipGetLastError();
}

}  // namespace

bool int8_streams(int64_t T, int64_t K) { return T <= kStreamTokens && stream_lds(T, K) <= kStreamLds; }

int int8_stream_parts(int64_t V, int ncu) {
  const int64_t room = 2 * ((V + BM - 1) / BM);  // of the partials
  return stream_grid(V, room < ncu ? room : ncu);
}

hipError_t launch_int8_fwd_stream(hipStream_t s, const Int8FwdArgs& a, int parts) {
  return launch_stream(s, a, a.part_pz != nullptr, parts, [](auto ch, auto nb, auto f) { return &int8_fwd_stream<ch.value, nb.value, f.value>; });
}

hipError_t launch_int8_logits_stream(hipStream_t s, const Int8LogitsArgs& a, int ncu) {
  return launch_stream(s, a, a.out_f32 != 0, stream_grid(a.V, ncu),
                       [](auto ch, auto nb, auto f) { return &int8_logits_stream<ch.value, nb.value, f.value>; });
}

}  // namespace lmhead
