// Logits of few tokens from the head in 8-bit integers: the weight streams through registers.
//
// What bounds such a call is the weight coming from HBM, and a tile that stages it in LDS stops that stream at its start and its end
// (half_tile.hpp).  Here a workgroup's waves share the contraction: wave w holds its k steps of all tokens' hidden values in registers for
// the whole launch, and of each 16 vocabulary rows it loads its part straight into the operand registers of the matrix instruction, the next 16 rows'
// while it multiplies these.  Nothing but the waves' partial sums goes through LDS, four times 16 rows at a time, two buffers, one barrier each.  They are
// integers: the sums are those of any other order.
#include "int8.hpp"

#include "../../include/skyrl_lmhead.h"

namespace lmhead {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int kStep = 64;    // k of a matrix instruction
constexpr int kRows = 16;    // vocabulary rows of one
constexpr int kUnits = 4;    // times 16 rows between barriers

// A wave's partial sums of 16 rows x 16 tokens, in LDS: lane (kq, n) holds rows kq * 4 .. + 3 of token n.  Lanes that read 64 rows of one token
// find them in different banks.
__device__ __forceinline__ int part_at(int unit, int kq, int n) { return unit * 1024 + kq * 256 + ((n + kq * 4 + unit) & 15) * 16; }

template <int WAVES, int S, int NB, bool F32>
__global__ __launch_bounds__(WAVES * 64) void int8_logits_stream(const Int8LogitsArgs a) {
  constexpr int kPart = kUnits * 1024;  // bytes of a wave's partial sums of one token block
  __shared__ __attribute__((aligned(16))) char parts[2][WAVES][NB][kPart];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, kq = lane >> 4;
  const int steps = a.K / kStep;
  // The wave's hidden values; zeros where the contraction has fewer steps, whose weight is any.
  i32x4 b[S][NB];
  int k_at[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int step = wave * S + s;
    k_at[s] = (step < steps ? step : steps - 1) * kStep + kq * 16;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int t = j * 16 + n;
      b[s][j] = *(const i32x4*)(a.Hd.values + (size_t)(t < a.T ? t : a.T - 1) * (size_t)a.Hd.ld + k_at[s]);
      if (step >= steps) b[s][j] = i32x4{0, 0, 0, 0};
    }
  }
  const int units = (a.V + kRows - 1) / kRows;
  const int first = (int)((int64_t)units * blockIdx.x / gridDim.x), last = (int)((int64_t)units * (blockIdx.x + 1) / gridDim.x);
  auto load = [&](int unit, i32x4 (&w)[S]) {
    int v = unit * kRows + n;
    v = v < a.V ? v : a.V - 1;
    const int8_t* row = a.W.values + (size_t)v * (size_t)a.W.ld;
#pragma unroll
    for (int s = 0; s < S; ++s) w[s] = *(const i32x4*)(row + k_at[s]);
  };
  // The tokens of this wave's results, and their scales.
  constexpr int kTokens = (NB * 16 + WAVES - 1) / WAVES;
  float s_t[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) s_t[i] = a.Hd.scale[wave + i * WAVES < a.T ? wave + i * WAVES : a.T - 1];
  auto multiply = [&](const i32x4 (&w)[S], char* to) {
    i32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s], b[s][j], acc[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < NB; ++j) *(i32x4*)(to + j * kPart) = acc[j];
  };
  i32x4 w0[S], w1[S];
  load(first, w0);
  int buffer = 0, held = 0;  // held: times 16 rows whose partial sums wait in the buffer
  for (int u = first; u < last; u += 2) {
    // In front of the weights that are in flight when it is needed: loads return in order.
    const int v = (u - held) * kRows + lane;
    const float c = a.W.scale[v < a.V ? v : a.V - 1];
    load(u + 1 < last ? u + 1 : last - 1, w1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(w0, parts[buffer][wave][0] + part_at(held, kq, n));
    load(u + 2 < last ? u + 2 : last - 1, w0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(w1, parts[buffer][wave][0] + part_at(held + 1, kq, n));
    held += 2;
    if (held < kUnits && u + 2 < last) continue;
    // Waits for the LDS writes alone: a barrier of the language would wait for the loads in flight too.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // 64 rows of a token per wave and turn.
    const int unit = lane >> 4, rq = (lane >> 2) & 3, r = lane & 3;
    if (unit < held && u + 2 - held + unit < last && v < a.V) {
#pragma unroll
      for (int i = 0; i < kTokens; ++i) {
        const int t = wave + i * WAVES;
        if (t >= a.T) break;
        const int at = part_at(unit, rq, t & 15) + r * 4;
        int sum = 0;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) sum += *(const int*)(parts[buffer][x][NB == 1 ? 0 : t >> 4] + at);
        const float z = (float)sum * c * s_t[i];
        const size_t to = (size_t)t * (size_t)a.ldo + (size_t)v;
        if constexpr (F32) ((float*)a.out)[to] = z;
        else ((__bf16*)a.out)[to] = (__bf16)z;
      }
    }
    held = 0, buffer ^= 1;
  }
}

template <int WAVES, int S, int NB>
void launch(hipStream_t s, const Int8LogitsArgs& a, int ncu) {
  const int units = (a.V + kRows - 1) / kRows;
  int grid = ncu * (16 / WAVES);
  if (grid > units) grid = units;
  hipLaunchKernelGGL((a.out_f32 ? int8_logits_stream<WAVES, S, NB, true> : int8_logits_stream<WAVES, S, NB, false>), dim3((unsigned)grid), dim3(WAVES * 64), 0, s, a);
}

template <int WAVES, int NB>
void launch_steps(hipStream_t s, const Int8LogitsArgs& a, int ncu) {
  const int each = (a.K / kStep + WAVES - 1) / WAVES;
  if (each <= 2) launch<WAVES, 2, NB>(s, a, ncu);
  else if (each <= 4) launch<WAVES, 4, NB>(s, a, ncu);
  else if (each <= 5) launch<WAVES, 5, NB>(s, a, ncu);
  else if (each <= 6) launch<WAVES, 6, NB>(s, a, ncu);
  else if (each <= 7) launch<WAVES, 7, NB>(s, a, ncu);
  else launch<WAVES, 8, NB>(s, a, ncu);
}

}  // namespace

bool int8_streams(int64_t T, int64_t K) { return T <= 16 && K <= 16 * 8 * kStep; }

hipError_t launch_int8_logits_stream(hipStream_t s, const Int8LogitsArgs& a, int ncu) {
  const int steps = a.K / kStep;
  if (steps <= 32) launch_steps<4, 1>(s, a, ncu);
  else if (steps <= 64) launch_steps<8, 1>(s, a, ncu);
  else launch_steps<16, 1>(s, a, ncu);
  return hipGetLastError();
}

}  // namespace lmhead
