// What the head with adapters needs besides its tiles (adapters.hpp): u of every token, the label's logit, and in the backward, from the dz panel
//     du_t = s_a B_a^T dz_t        dB_a = sum_t dz_t u_t^T        dA_a = sum_t du_t h_t^T        d_hidden_t += A_a^T du_t
// over rows that are grouped by adapter.  All of it is bound by the panel, which two kernels read once each, or by latency.
//
// Operand layouts of v_mfma_f32_16x16x32_bf16 are in gemm_core.hpp.  Operands whose contraction is not their contiguous axis go through LDS
// and the transposing read: lane (kq, s) supplies row kq * 8 + half * 4 + (s >> 2), columns (s & 3) * 4 .. + 3 of the 16, and receives column s
// of the eight rows kq * 8 .. + 7.
#include "adapters.hpp"
#include "dh_reduce.hpp"

namespace lmhead {
namespace {

// x as two bf16 terms (exact to 2^-17 of it).
struct Terms {
  uint2 hi, lo;
};
__device__ __forceinline__ Terms two_terms(const f32x4& x) {
  const bf16x4 hi = __builtin_convertvector(x, bf16x4);
  const uint2 h = *(const uint2*)&hi;
  const float w[4] = {__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16), __uint_as_float(h.y & 0xffff0000u)};
  f32x4 rest;
#pragma unroll
  for (int i = 0; i < 4; ++i) rest[i] = __builtin_isfinite(w[i]) ? x[i] - w[i] : 0.f;  // an inf stays one
  const bf16x4 lo = __builtin_convertvector(rest, bf16x4);
  return Terms{h, *(const uint2*)&lo};
}

__device__ __forceinline__ int tokens_in_force(int T, const int* T_dev) { return T_dev ? __builtin_amdgcn_readfirstlane(*T_dev) : T; }

// ------------------------------------------------------------------------------------------------------------
// u = s A h.  One workgroup per 16 tokens, 32 ranks and every so many of the tokens' adapters (grid.z, so that a batch of unlike tokens does not
// read its adapters one behind the other); its waves share the hidden size and their sums meet in LDS.  M: rank, N: token.  Bound by the
// latency of its loads: with all adapters of 16 tokens in one workgroup of eight waves 97 us at T=16, H=3584, ten adapters.
// ------------------------------------------------------------------------------------------------------------
constexpr int kShrinkWaves = 16;
__global__ __launch_bounds__(kShrinkWaves * 64) void adapter_shrink(const Adapters ad, const uint16_t* __restrict__ hidden, int64_t ldh,
                                                                    const int64_t* __restrict__ ids, int T_, const int* T_dev, int H,
                                                                    uint16_t* __restrict__ U, int* __restrict__ ids32) {
  __shared__ f32x4 part[kShrinkWaves][2][64];
  const int tid = threadIdx.x, lane = tid & 63, lrow = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pitch = 2 * padded_rank(ad.rank), r0 = blockIdx.y * 32;
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && tid * 8 < pitch) *(uint4*)(U + tid * 8) = make_uint4(0, 0, 0, 0);
  const int T = tokens_in_force(T_, T_dev), t0 = blockIdx.x * 16;
  if (t0 >= T) return;
  const int t = t0 + lrow;
  int id = -1;
  if (t < T) {
    const int64_t x = ids[t];
    id = x >= 0 && x < (int64_t)ad.N ? (int)x : -1;
    if (blockIdx.y == 0 && blockIdx.z == 0 && tid < 16) ids32[t] = id;
  }
  const uint16_t* x_row = hidden + (size_t)(t < T ? t : T - 1) * (size_t)ldh + kq * 8;
  f32x4 u[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  bool mine = blockIdx.z == 0 && id < 0;  // whether this workgroup writes the token's row
  bool any = __any(mine);
  unsigned left = (unsigned)__ballot(id >= 0) & 0xffffu;
  for (unsigned n = 0; left; ++n) {
    const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    left &= ~(unsigned)__ballot(id == a);
    if (n % gridDim.z != blockIdx.z) continue;
    any = true;
    const uint16_t* rows[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int r = r0 + m * 16 + lrow;
      rows[m] = ad.A + (size_t)a * (size_t)ad.a_adapter + (size_t)(r < ad.rank ? r : ad.rank - 1) * (size_t)ad.a_row + kq * 8;
    }
    f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    constexpr int kAhead = 8, kStep = kShrinkWaves * 32;  // loads in flight; the compiler does not unroll a loop of MFMAs by itself
    for (int k0 = wave * 32; k0 < H; k0 += kAhead * kStep) {
      bf16x8 x[kAhead], w[kAhead][2];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * kStep < H ? k0 + i * kStep : k0;
        x[i] = *(const bf16x8*)(x_row + k);
#pragma unroll
        for (int m = 0; m < 2; ++m) w[i][m] = *(const bf16x8*)(rows[m] + k);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k0 + i * kStep >= H) break;
#pragma unroll
        for (int m = 0; m < 2; ++m) acc[m] = mfma(w[i][m], x[i], acc[m]);
      }
    }
    const float s = ad.scaling[a];
    if (id == a) u[0] = acc[0] * s, u[1] = acc[1] * s, mine = true;
  }
  if (!any) return;  // alike in all waves
#pragma unroll
  for (int m = 0; m < 2; ++m) part[wave][m][lane] = u[m];
  __syncthreads();
  if (tid >= 128 || t >= T || !mine) return;
  const int m = tid >> 6;
  f32x4 sum = part[0][m][lane];
#pragma unroll
  for (int w = 1; w < kShrinkWaves; ++w) sum += part[w][m][lane];
  const int r = r0 + m * 16 + kq * 4;
  if (r >= ad.rank) sum = f32x4{0.f, 0.f, 0.f, 0.f};  // the rank is a multiple of 8
  const Terms terms = two_terms(sum);
  uint16_t* to = U + (size_t)(1 + t) * (size_t)pitch + r;
  *(uint2*)to = terms.hi;
  *(uint2*)(to + pitch / 2) = terms.lo;
}

// The adapter's part of the label's logit, 16 lanes a token, and the way of grouped rows' results to their tokens.
__global__ __launch_bounds__(256) void adapter_label(const Adapters ad, const uint16_t* __restrict__ U, const int* __restrict__ ids,
                                                     const int64_t* __restrict__ labels, int T, int64_t V, float rcp_temp, const RowResults from,
                                                     const int* __restrict__ row_map, const RowResults to) {
  const int t = blockIdx.x * 16 + (threadIdx.x >> 4), part = threadIdx.x & 15;
  if (t >= T) return;
  const int a = ids[t];
  const int64_t y = labels[t];
  float sum = 0.f;
  if (a >= 0 && y >= 0 && y < V) {  // the 16 lanes alike
    const int pitch = 2 * padded_rank(ad.rank);
    const uint16_t* b = ad.B + (size_t)a * (size_t)ad.b_adapter + (size_t)y * (size_t)ad.b_row;
    const uint16_t* u = U + (size_t)(1 + t) * (size_t)pitch;
    for (int r = part; r < ad.rank; r += 16) {
      const float x = __uint_as_float((uint32_t)u[r] << 16) + __uint_as_float((uint32_t)u[pitch / 2 + r] << 16);
      sum = fmaf(x, __uint_as_float((uint32_t)b[r] << 16), sum);
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 16);
  }
  const int row = row_map ? row_map[t] : t;
  if (part == 0) to.logprobs[row] = a >= 0 ? fmaf(sum, rcp_temp, from.logprobs[t]) : from.logprobs[t];
  if (!row_map) return;
  if (part == 1 && to.entropy) to.entropy[row] = from.entropy[t];
  if (part == 2 && to.row_lse) to.row_lse[row] = from.row_lse[t];
  if (part == 3 && to.row_pz) to.row_pz[row] = from.row_pz[t];
}

// A token's dz is of order g in its label's column and of order g p elsewhere, so what the rounding to bf16 takes from that one value is most of the
// error of its gradients: 2.3e-3 to 2.5e-3 of dB's norm, where rounding the result alone takes 1.7e-3, which is what this leaves.  dz is linear in
// (g, q): both are multiplied by the factor, within 2^-8 of 1, that makes the label's value a bf16 number, and what is formed from the row is divided by
// it: du and d_hidden in fp32 (`back`), dB through the two terms of U_back.  Rows without an adapter stay as they are, as in the head
// without adapters.  The label's value is formed anew, one wave a token, from a row of the weight and one of B: latency, 3 us of 446 at 96 tokens.
__global__ __launch_bounds__(256) void adapter_fit_rows(const Adapters ad, const uint16_t* __restrict__ hidden, const uint16_t* __restrict__ weight, int64_t ldw,
                                                        const int64_t* __restrict__ labels, const int* __restrict__ ids, const float* __restrict__ lse,
                                                        const float* __restrict__ pz, int T_, const int* __restrict__ T_dev, int H, int V, float rcp_temp,
                                                        const uint16_t* __restrict__ U, float* __restrict__ g, float* __restrict__ q,
                                                        float* __restrict__ back, uint16_t* __restrict__ U_back) {
  const int T = tokens_in_force(T_, T_dev), lane = threadIdx.x & 63;
  const int t = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (t >= T) return;
  const int Rp = padded_rank(ad.rank), a = ids[t];
  const int64_t y = labels[t];
  const uint16_t* u = U + (size_t)(1 + t) * (size_t)(2 * Rp);
  auto wide = [](uint16_t x) { return __uint_as_float((uint32_t)x << 16); };
  float inverse = 1.f;
  if (a >= 0 && y >= 0 && y < V) {
    const uint16_t *w = weight + (size_t)y * (size_t)ldw, *h = hidden + (size_t)t * (size_t)H;
    float z = 0.f;
    for (int c = lane * 8; c < H; c += 64 * 8) {
      const u32x4 x = *(const u32x4*)(w + c), v = *(const u32x4*)(h + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(v[i] << 16), z);
        z = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(v[i] & 0xffff0000u), z);
      }
    }
    const uint16_t* b = ad.B + (size_t)a * (size_t)ad.b_adapter + (size_t)y * (size_t)ad.b_row;
    for (int r = lane; r < ad.rank; r += 64) z = fmaf(wide(u[r]) + wide(u[Rp + r]), wide(b[r]), z);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) z += __shfl_xor(z, o, 64);
    const float gt = g[t], qt = q ? q[t] : 0.f;
    const float p = __builtin_amdgcn_exp2f((z * rcp_temp - lse[t]) * kLog2e);
    const float c0 = -(gt - (q ? qt * pz[t] : 0.f)) * rcp_temp, c1 = -qt * rcp_temp * rcp_temp;
    const float d = fmaf(p, fmaf(c1, z, c0), gt * rcp_temp);
    if (fabsf(d) > 0x1p-100f && fabsf(d) < 0x1p100f) {  // neither NaN nor infinite, and so is what follows
      const float fit = (float)(__bf16)d;
      inverse = d / fit;
      if (lane == 0) {
        g[t] = gt * (fit / d);
        if (q) q[t] = qt * (fit / d);
      }
    }
  }
  if (lane == 0) back[t] = inverse;
  uint16_t* to = U_back + (size_t)(1 + t) * (size_t)(2 * Rp);
  for (int r = lane * 4; r < Rp; r += 64 * 4) {
    const uint2 hi = *(const uint2*)(u + r), lo = *(const uint2*)(u + Rp + r);
    const f32x4 x = {__uint_as_float(hi.x << 16) + __uint_as_float(lo.x << 16), __uint_as_float(hi.x & 0xffff0000u) + __uint_as_float(lo.x & 0xffff0000u),
                     __uint_as_float(hi.y << 16) + __uint_as_float(lo.y << 16), __uint_as_float(hi.y & 0xffff0000u) + __uint_as_float(lo.y & 0xffff0000u)};
    const Terms terms = two_terms(x * inverse);
    *(uint2*)(to + r) = terms.hi;
    *(uint2*)(to + Rp + r) = terms.lo;
  }
}

// Rows of the hidden states (and labels) in the order of idx.
__global__ __launch_bounds__(256) void adapter_gather_rows(const int* __restrict__ idx, const uint16_t* __restrict__ hidden, int64_t ldh, int H,
                                                           const int64_t* __restrict__ labels, uint16_t* __restrict__ hidden_c, int64_t* __restrict__ labels_c) {
  const int r = blockIdx.x, t = idx[r];
  const uint16_t* src = hidden + (size_t)t * (size_t)ldh;
  uint16_t* dst = hidden_c + (size_t)r * (size_t)H;
  for (int c = threadIdx.x * 8; c < H; c += 256 * 8) *(uint4*)(dst + c) = *(const uint4*)(src + c);
  if (labels && threadIdx.x == 0) labels_c[r] = labels[t];
}

// ------------------------------------------------------------------------------------------------------------
// Rows with a gradient (without GRADS all of them), grouped by adapter (those without one last), ascending inside a group: idx, their adapters, and seg[a], the place of
// adapter a's first row; seg[N] that of the rows without an adapter, seg[N + 1] the number of rows.  One workgroup per group: it counts the rows of
// the groups before its own, then lists its own.  The order is a function of the inputs alone, so the sums over rows are the same bits on each call.
// ------------------------------------------------------------------------------------------------------------
constexpr int kGroupThreads = 1024, kGroupTokens = 4;  // tokens per thread and step
template <bool GRADS>
__global__ __launch_bounds__(kGroupThreads) void adapter_group_rows(const float* __restrict__ g, const float* __restrict__ q,
                                                                    const int64_t* __restrict__ labels, int64_t V, const int64_t* __restrict__ ids, int T, int N, int* __restrict__ idx,
                                                                    int64_t* __restrict__ ids_c, int* __restrict__ seg) {
  constexpr int kCounts = kGroupTokens * kGroupThreads / 64;
  static_assert(kCounts == 64, "one lane per count");
  __shared__ int count[2][kCounts];
  __shared__ int before[kGroupThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, mine = blockIdx.x;
  auto group_of = [&](int t) -> int {  // -1: no gradient
    if (t >= T) return -1;
    const int64_t x = ids[t];
    if constexpr (GRADS) {
      const float gv = target_grad<true>(g, labels, V, t), qv = q ? q[t] : 0.f;
      if (gv == 0.f && qv == 0.f) return -1;
    }
    return x >= 0 && x < (int64_t)N ? (int)x : N;
  };
  int less = 0;
  for (int t0 = 0; t0 < T; t0 += kGroupTokens * kGroupThreads) {
    int k[kGroupTokens];
#pragma unroll
    for (int j = 0; j < kGroupTokens; ++j) k[j] = group_of(t0 + j * kGroupThreads + tid);
#pragma unroll
    for (int j = 0; j < kGroupTokens; ++j) less += (int)__popcll(__ballot(k[j] >= 0 && k[j] < mine));
  }
  if (lane == 0) before[wave] = less;
  __syncthreads();
  int n = 0;
  for (int w = 0; w < kGroupThreads / 64; ++w) n += before[w];
  if (tid == 0) seg[mine] = n;
  for (int t0 = 0, turn = 0; t0 < T; t0 += kGroupTokens * kGroupThreads, turn ^= 1) {
    unsigned long long ballot[kGroupTokens];
#pragma unroll
    for (int j = 0; j < kGroupTokens; ++j) ballot[j] = __ballot(group_of(t0 + j * kGroupThreads + tid) == mine);
#pragma unroll
    for (int j = 0; j < kGroupTokens; ++j)
      if (lane == 0) count[turn][j * (kGroupThreads / 64) + wave] = (int)__popcll(ballot[j]);
    __syncthreads();
    const int here = count[turn][lane];
    int upto = here;
#pragma unroll
    for (int o = 1; o < kCounts; o <<= 1) {
      const int below = __shfl_up(upto, o, 64);
      upto += lane >= o ? below : 0;
    }
#pragma unroll
    for (int j = 0; j < kGroupTokens; ++j) {
      const int base = n + __shfl(upto - here, j * (kGroupThreads / 64) + wave, 64);
      if (ballot[j] >> lane & 1) {
        const int at = base + (int)__popcll(ballot[j] & ((1ull << lane) - 1ull));
        idx[at] = t0 + j * kGroupThreads + tid;
        ids_c[at] = mine < N ? mine : -1;
      }
    }
    n += __shfl(upto, kCounts - 1, 64);
  }
  if (tid == 0 && mine == N) seg[N + 1] = n;
}

// The rows of every adapter cut in pieces of at most SIZE, laid end to end: piece p's adapter and rows, or a < 0 behind the last one.  Of the rows
// row0 .. row0 + T - 1 that seg counts, numbered from 0.
struct RowPiece {
  int a, begin, end;
};
template <int SIZE>
__device__ __forceinline__ RowPiece row_piece(const int* seg, int N, int row0, int T, int p) {
  const int lane = threadIdx.x & 63;
  auto inside = [&](int at) { return at < row0 ? 0 : at - row0 < T ? at - row0 : T; };
  int before = 0;  // pieces of adapters in front of this step's 64
  for (int a0 = 0; a0 < N; a0 += 64) {
    const int a = a0 + lane;
    const int from = a < N ? inside(seg[a]) : 0, to = a < N ? inside(seg[a + 1]) : 0, n = (to - from + SIZE - 1) / SIZE;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(upto, o, 64);
      upto += lane >= o ? below : 0;
    }
    const unsigned long long past = __ballot(before + upto > p);
    if (past) {
      const int l = (int)__builtin_ctzll(past);
      const int k = p - before - __shfl(upto - n, l, 64);
      const int begin = __shfl(from, l, 64) + k * SIZE, last = __shfl(to, l, 64);
      return RowPiece{__builtin_amdgcn_readfirstlane(a0 + l), __builtin_amdgcn_readfirstlane(begin),
                      __builtin_amdgcn_readfirstlane(begin + SIZE < last ? begin + SIZE : last)};
    }
    before += __shfl(upto, 63, 64);
  }
  return RowPiece{-1, 0, 0};
}

// The vocabulary row that panel column c of a chunk stands for; columns that stand for none hold zeros (VocabTail in gemm_core.hpp).
__device__ __forceinline__ int panel_row(int vc0, int c, const VocabTail& tail) {
  const int column = vc0 + c;
  return tail.back > 0 && column >= tail.from ? column - tail.back : column;
}

// ------------------------------------------------------------------------------------------------------------
// Partial sums of B_a^T dz over a range of panel columns.  One workgroup per piece of at most 128 rows of one adapter, range and 64 ranks; 32 rows a
// wave.  M: rank (B's rows through LDS), N: row (panel rows as they lie).  B's next rows and the panel's next pieces are loaded while the
// present ones are multiplied.  HBM: the panel once and B once per piece, which is why pieces are not smaller (64 rows that adapters share:
// 202 us for 1024 rows x 151936 columns of six adapters, rank 32).
// ------------------------------------------------------------------------------------------------------------
constexpr int kDuColumns = 128, kDuRanks = 64;
constexpr int kDuPitch = kDuRanks * 2 + 16;
__global__ __launch_bounds__(256) void adapter_du_partial(const AdapterPanel p, const int* __restrict__ seg, int row0, int columns, int per_range,
                                                          float* __restrict__ out, int Rp) {
  __shared__ __attribute__((aligned(16))) char lds[2][kDuColumns * kDuPitch];
  const RowPiece piece = row_piece<kDuPiece>(seg, p.ad.N, row0, tokens_in_force(p.T, p.T_dev), blockIdx.x);
  if (piece.a < 0) return;
  const int tid = threadIdx.x, lane = tid & 63, lrow = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r0 = blockIdx.z * kDuRanks, R = p.ad.rank;
  const int tiles = __builtin_amdgcn_readfirstlane(((R - r0 < kDuRanks ? R - r0 : kDuRanks) + 15) / 16);
  const int c0 = blockIdx.y * per_range, c1 = c0 + per_range < columns ? c0 + per_range : columns;
  const int t0 = piece.begin + wave * 32;
  const int blocks = piece.end - t0 > 16 ? 2 : piece.end > t0 ? 1 : 0;  // of 16 rows that this wave has
  const uint16_t* d_row[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = t0 + n * 16 + lrow;
    d_row[n] = p.D + (size_t)(t < piece.end ? t : piece.end - 1) * (size_t)p.ldd + kq * 8;
  }
  const uint16_t* Ba = p.ad.B + (size_t)piece.a * (size_t)p.ad.b_adapter;
  // 128 rows of 64 ranks: four 16-byte pieces a thread
  constexpr int kPieces = kDuColumns * kDuRanks / 8 / 256, kSteps = kDuColumns / 32;
  u32x4 b[kPieces];
  bf16x8 d[2][kSteps];
  auto load = [&](int c) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int at = j * 256 + tid, row = at >> 3, r = r0 + (at & 7) * 8;
      int v = panel_row(p.vc0, c + row, p.tail);
      v = v < p.V ? v : p.V - 1;  // a column behind the vocabulary: zeros in the panel
      b[j] = r < R ? *(const u32x4*)(Ba + (size_t)v * (size_t)p.ad.b_row + r) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        if (n < blocks) d[n][j] = *(const bf16x8*)(d_row[n] + c + j * 32);
  };
  f32x4 acc[2][4];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int m = 0; m < 4; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (c0 < c1) load(c0);
  int turn = 0;
  for (int c = c0; c < c1; c += kDuColumns, turn ^= 1) {
    char* const at = lds[turn];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int e = j * 256 + tid;
      *(u32x4*)(at + (e >> 3) * kDuPitch + (e & 7) * 16) = b[j];
    }
    bf16x8 now[2][kSteps];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < kSteps; ++j) now[n][j] = d[n][j];
    if (c + kDuColumns < c1) load(c + kDuColumns);
    __syncthreads();  // the rows stand; the other buffer is written behind the next barrier's reads only
    if (blocks > 0) {
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m < tiles) {
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            const bf16x8 f = transposed(at + j * 32 * kDuPitch + m * 32, kDuPitch);
            acc[0][m] = mfma(f, now[0][j], acc[0][m]);
            if (blocks > 1) acc[1][m] = mfma(f, now[1][j], acc[1][m]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int t = t0 + n * 16 + lrow;
    if (t >= piece.end) continue;
    float* to = out + ((size_t)blockIdx.y * (size_t)p.T + (size_t)t) * (size_t)Rp + r0 + kq * 4;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (r0 + m * 16 < Rp) *(f32x4*)(to + m * 16) = acc[n][m];
  }
}

// du = s * back * (the sum of `slots` partial sums) as two bf16 terms, rows of U's form.  Sixteen threads share the slots of four ranks of a token, in an
// order that the number of slots alone determines.
__global__ __launch_bounds__(256) void adapter_du_sum(const Adapters ad, const float* __restrict__ part, int slots, int T_, const int* T_dev,
                                                      const int* __restrict__ ids, const float* __restrict__ back, int Rp, uint16_t* __restrict__ dU) {
  __shared__ f32x4 sums[16][16];
  const int T = tokens_in_force(T_, T_dev);
  const int q = threadIdx.x & 15, share = threadIdx.x >> 4;
  const int e = (blockIdx.x * 16 + q) * 4;  // Rp is a multiple of 32: the 16 quads of a workgroup lie in one or two tokens
  const int t = e / Rp, r = e - t * Rp;
  const size_t step = (size_t)T_ * (size_t)Rp;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  const int a = t < T ? ids[t] : -1;
  if (a >= 0) {  // rows without an adapter have no partial sums
    const float* from = part + (size_t)t * (size_t)Rp + r;
#pragma unroll 4
    for (int s = share; s < slots; s += 16) sum += *(const f32x4*)(from + (size_t)s * step);
  }
  sums[share][q] = sum;
  __syncthreads();
  if (share != 0 || t >= T) return;
#pragma unroll
  for (int s = 1; s < 16; ++s) sum += sums[s][q];
  const Terms terms = two_terms(sum * (a >= 0 ? ad.scaling[a] * back[t] : 0.f));
  uint16_t* to = dU + (size_t)(1 + t) * (size_t)(2 * Rp) + r;
  *(uint2*)to = terms.hi;
  *(uint2*)(to + Rp) = terms.lo;
}

// ------------------------------------------------------------------------------------------------------------
// dB_a[v, r] = sum over adapter a's rows of dz[t, v] u[t, r].  One workgroup per 256 panel columns, adapter and 64 ranks, 64 columns a wave; M: rank,
// N: column, both through LDS in steps of 32 rows.  HBM: the panel once, 5.3 TB/s at 8192 rows x 76032 columns (235 us).
// ------------------------------------------------------------------------------------------------------------
constexpr int kDbColumns = 256, kDbRows = 32, kDbRanks = 64;
constexpr int kDbPitchD = kDbColumns * 2 + 16, kDbPitchU = kDbRanks * 2 + 16;
__global__ __launch_bounds__(256) void adapter_db(const AdapterPanel p, const uint16_t* __restrict__ U, const int* __restrict__ seg, int row0,
                                                  const float* sum_in, float* sum_out, uint16_t* __restrict__ dB) {
  __shared__ __attribute__((aligned(16))) char lds_d[2][kDbRows * kDbPitchD];
  __shared__ __attribute__((aligned(16))) char lds_u[2][2 * kDbRows * kDbPitchU];  // the upper terms' rows, then the lower ones'
  const int T = tokens_in_force(p.T, p.T_dev);
  const int tid = threadIdx.x, lane = tid & 63, lrow = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int a = blockIdx.y, r0 = blockIdx.z * kDbRanks, R = p.ad.rank, Rp = padded_rank(R);
  const int c0 = blockIdx.x * kDbColumns;
  auto in_block = [&](int at) { return at < row0 ? 0 : at - row0 < T ? at - row0 : T; };
  const int begin = in_block(__builtin_amdgcn_readfirstlane(seg[a])), end = in_block(__builtin_amdgcn_readfirstlane(seg[a + 1]));
  f32x4 acc[4][4];  // [rank tile][column tile]
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 d[4], u[2];
  const int u_row = tid >> 3, u_rank = r0 + (tid & 7) * 8;
  auto load = [&](int t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // 32 rows of 512 bytes; rows behind the last one repeat it, against zeros of u
      const int piece = j * 256 + tid, row = t + (piece >> 5);
      d[j] = *(const u32x4*)(p.D + (size_t)(row < end ? row : end - 1) * (size_t)p.ldd + c0 + (piece & 31) * 8);
    }
#pragma unroll
    for (int term = 0; term < 2; ++term)
      u[term] = t + u_row < end && u_rank < Rp ? *(const u32x4*)(U + (size_t)(1 + t + u_row) * (size_t)(2 * Rp) + term * Rp + u_rank)
                                               : u32x4{0u, 0u, 0u, 0u};
  };
  if (begin < end) load(begin);
  int turn = 0;
  for (int t = begin; t < end; t += kDbRows, turn ^= 1) {
    char *const at_d = lds_d[turn], *const at_u = lds_u[turn];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int piece = j * 256 + tid;
      *(u32x4*)(at_d + (piece >> 5) * kDbPitchD + (piece & 31) * 16) = d[j];
    }
#pragma unroll
    for (int term = 0; term < 2; ++term) *(u32x4*)(at_u + (term * kDbRows + u_row) * kDbPitchU + (tid & 7) * 16) = u[term];
    if (t + kDbRows < end) load(t + kDbRows);
    __syncthreads();
    bf16x8 df[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) df[n] = transposed(at_d + (wave * 64 + n * 16) * 2, kDbPitchD);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (r0 + m * 16 >= R) continue;
#pragma unroll
      for (int term = 0; term < 2; ++term) {
        const bf16x8 uf = transposed(at_u + term * kDbRows * kDbPitchU + m * 32, kDbPitchU);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = mfma(uf, df[n], acc[m][n]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int column = p.vc0 + c0 + wave * 64 + n * 16 + lrow;
    int v = column;
    if (p.tail.back > 0 && column >= p.tail.from) {  // the moved group: its first columns repeat the group before it
      if (column - p.tail.from < p.tail.back || column - p.tail.from >= 2 * BK) continue;
      v = column - p.tail.back;
    }
    if (v >= p.V) continue;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int r = r0 + m * 16 + kq * 4;
      if (r >= R) continue;
      const size_t at = ((size_t)a * (size_t)p.V + (size_t)v) * (size_t)R + r;
      f32x4 x = acc[m][n];
      if (sum_in) x += *(const f32x4*)(sum_in + at);
      if (sum_out) *(f32x4*)(sum_out + at) = x;
      if (dB) {
        const bf16x4 b = __builtin_convertvector(x, bf16x4);
        *(uint2*)(dB + at) = *(const uint2*)&b;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// d_hidden[row_map[t], :] = back_t d_hidden[row_map[t], :] + A_a^T du_t.  One workgroup per 64 tokens and 64 hidden columns, 16 tokens a wave.  M: hidden column (A's rows through
// LDS), N: token.  d_hidden holds the product with the weight, rounded to bf16; the sum is rounded once more.  Only for the small vocabularies whose
// weight is transposed (reads_weight_in_place); elsewhere lmhead_dh_reduce adds the adapters' part in fp32.
// ------------------------------------------------------------------------------------------------------------
constexpr int kDhPitch = 64 * 2 + 16;
__global__ __launch_bounds__(256) void adapter_dh_add(const Adapters ad, const uint16_t* __restrict__ dU, const int* __restrict__ ids, int T_,
                                                      const int* T_dev, const int* __restrict__ row_map, const float* __restrict__ back, int H,
                                                      uint16_t* __restrict__ d_hidden) {
  __shared__ __attribute__((aligned(16))) char lds[32 * kDhPitch];
  const int T = tokens_in_force(T_, T_dev), t0 = blockIdx.x * 64, h0 = blockIdx.y * 64;
  if (t0 >= T) return;
  const int tid = threadIdx.x, lane = tid & 63, lrow = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int Rp = padded_rank(ad.rank);
  const int id64 = t0 + lane < T ? ids[t0 + lane] : -1;
  const int t = t0 + wave * 16 + lrow;
  const int id = t < T ? ids[t] : -1;
  const uint16_t* du = dU + (size_t)(1 + (t < T ? t : T - 1)) * (size_t)(2 * Rp) + kq * 8;
  f32x4 sum[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  unsigned long long left = __ballot(id64 >= 0);
  while (left) {
    const int a = __builtin_amdgcn_readlane(id64, (int)__builtin_ctzll(left));
    left &= ~__ballot(id64 == a);
    const uint16_t* Aa = ad.A + (size_t)a * (size_t)ad.a_adapter + h0;
    f32x4 acc[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < Rp; k += 32) {
      const int row = tid >> 3;  // 32 rows of 128 bytes
      const uint4 x = k + row < ad.rank ? *(const uint4*)(Aa + (size_t)(k + row) * (size_t)ad.a_row + (tid & 7) * 8) : make_uint4(0, 0, 0, 0);
      __syncthreads();
      *(uint4*)(lds + row * kDhPitch + (tid & 7) * 16) = x;
      __syncthreads();
      const bf16x8 hi = *(const bf16x8*)(du + k), lo = *(const bf16x8*)(du + Rp + k);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const bf16x8 f = transposed(lds + m * 32, kDhPitch);
        acc[m] = mfma(f, hi, acc[m]);
        acc[m] = mfma(f, lo, acc[m]);
      }
    }
    if (id == a) {
#pragma unroll
      for (int m = 0; m < 4; ++m) sum[m] = acc[m];
    }
  }
  if (t >= T) return;
  const float by = back[t];
  uint16_t* to = d_hidden + (size_t)row_map[t] * (size_t)H + h0 + kq * 4;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const uint2 w = *(const uint2*)(to + m * 16);
    const f32x4 x = {fmaf(by, __uint_as_float(w.x << 16), sum[m][0]), fmaf(by, __uint_as_float(w.x & 0xffff0000u), sum[m][1]),
                     fmaf(by, __uint_as_float(w.y << 16), sum[m][2]), fmaf(by, __uint_as_float(w.y & 0xffff0000u), sum[m][3])};
    const bf16x4 b = __builtin_convertvector(x, bf16x4);
    *(uint2*)(to + m * 16) = *(const uint2*)&b;
  }
}

// ------------------------------------------------------------------------------------------------------------
// dA_a[r, h] = sum over adapter a's rows of du[t, r] h[t, h], in pieces of at most kDaPiece rows whose sums are added in order.
// ------------------------------------------------------------------------------------------------------------
// One workgroup per piece, 256 hidden columns (64 a wave) and 32 ranks.  M: hidden column, N: rank, steps of 32 rows.
constexpr int kDaPitchH = 256 * 2 + 16, kDaPitchU = 2 * 32 * 2 + 16;
__global__ __launch_bounds__(256) void adapter_da_partial(const Adapters ad, const uint16_t* __restrict__ hidden, int64_t ldh, const uint16_t* __restrict__ dU,
                                                          const int* __restrict__ seg, int H, float* __restrict__ part) {
  __shared__ __attribute__((aligned(16))) char lds_h[2][32 * kDaPitchH];
  __shared__ __attribute__((aligned(16))) char lds_u[2][32 * kDaPitchU];
  const RowPiece piece = row_piece<kDaPiece>(seg, ad.N, 0, seg[ad.N], blockIdx.x);
  if (piece.a < 0) return;
  const int begin = piece.begin, end = piece.end;
  const int tid = threadIdx.x, lane = tid & 63, lrow = lane & 15, kq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h0 = blockIdx.y * 256, r0 = blockIdx.z * 32, Rp = padded_rank(ad.rank);
  f32x4 acc[4][2];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 x[4], u;
  const int u_row = tid >> 3, u_term = (tid >> 2) & 1, u_rank = (tid & 3) * 8;  // 32 rows of 32 upper, then 32 lower terms
  auto load = [&](int t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = j * 256 + tid, row = t + (p >> 5), h = h0 + (p & 31) * 8;
      x[j] = *(const u32x4*)(hidden + (size_t)(row < end ? row : end - 1) * (size_t)ldh + (h < H ? h : H - 8));
    }
    u = t + u_row < end ? *(const u32x4*)(dU + (size_t)(1 + t + u_row) * (size_t)(2 * Rp) + u_term * Rp + r0 + u_rank) : u32x4{0u, 0u, 0u, 0u};
  };
  load(begin);
  int turn = 0;
  for (int t = begin; t < end; t += 32, turn ^= 1) {
    char *const at_h = lds_h[turn], *const at_u = lds_u[turn];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = j * 256 + tid;
      *(u32x4*)(at_h + (p >> 5) * kDaPitchH + (p & 31) * 16) = x[j];
    }
    *(u32x4*)(at_u + u_row * kDaPitchU + u_term * 64 + u_rank * 2) = u;
    if (t + 32 < end) load(t + 32);
    __syncthreads();
    bf16x8 hi[2], lo[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) hi[n] = transposed(at_u + n * 32, kDaPitchU), lo[n] = transposed(at_u + 64 + n * 32, kDaPitchU);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const bf16x8 f = transposed(at_h + (wave * 64 + m * 16) * 2, kDaPitchH);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        acc[m][n] = mfma(f, hi[n], acc[m][n]);
        acc[m][n] = mfma(f, lo[n], acc[m][n]);
      }
    }
  }
  // A lane holds four consecutive hidden columns of one rank.
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int r = r0 + n * 16 + lrow;
    float* to = part + ((size_t)blockIdx.x * (size_t)Rp + (size_t)r) * (size_t)H;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int h = h0 + wave * 64 + m * 16 + kq * 4;
      if (h < H) *(f32x4*)(to + h) = acc[m][n];
    }
  }
}

// dA of an adapter: the sum of its pieces, rounded.  One workgroup per adapter and rank.
__global__ __launch_bounds__(256) void adapter_da_sum(const float* __restrict__ part, const int* __restrict__ seg, int H, int R, uint16_t* __restrict__ dA) {
  const int a = blockIdx.x, r = blockIdx.y, Rp = padded_rank(R);
  __shared__ int first_piece;
  if (threadIdx.x < 64) {
    int before = 0;
    for (int b = threadIdx.x; b < a; b += 64) before += (seg[b + 1] - seg[b] + kDaPiece - 1) / kDaPiece;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) before += __shfl_xor(before, o, 64);
    if (threadIdx.x == 0) first_piece = before;
  }
  __syncthreads();
  const int n = (seg[a + 1] - seg[a] + kDaPiece - 1) / kDaPiece;
  const float* from = part + ((size_t)first_piece * (size_t)Rp + (size_t)r) * (size_t)H;
  uint16_t* to = dA + ((size_t)a * (size_t)R + (size_t)r) * (size_t)H;
  for (int h = threadIdx.x * 4; h < H; h += 256 * 4) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < n; ++p) sum += *(const f32x4*)(from + (size_t)p * (size_t)Rp * (size_t)H + h);
    const bf16x4 b = __builtin_convertvector(sum, bf16x4);
    *(uint2*)(to + h) = *(const uint2*)&b;
  }
}

}  // namespace

hipError_t launch_adapter_shrink(hipStream_t s, const Adapters& ad, const uint16_t* hidden, int64_t ldh, const int64_t* ids, int64_t T, const int* T_dev,
                                 int64_t H, uint16_t* U, int* ids32) {
  // Up to 16 workgroups share the adapters of 16 tokens; with many tokens their tiles fill the chip by themselves, and workgroups without an adapter
  // only cost.  us with 16 / 4 / 2 / 1 of them, rank 32, mixed: T=16, H=3584, 48 adapters 12.9 / 38.4 / 65.6 / 147; T=256 12.4 / 20.9 / 30.1 / 56.6; T=1024 12.4 / 12.4
  // / 12.4 / 21.6; T=2048, H=896 12.2 / 6.7 / 6.4 / 10.6, H=3584 16.8 / 13.0 / 13.2 / 21.6; T=4096, H=896 19.6 / 9.7 / 9.5 / 11.0, eight adapters 13.0 / 8.0 / 8.9 / 9.0;
  // T=8192, H=896 20.2 / 14.6 / 13.4 / 12.9, H=3584 32.6 / 32.3 / 31.8 / 31.2.
  const int64_t tiles = (T + 15) / 16, most = tiles <= 64 ? 16 : tiles <= 256 ? 4 : 2;
  hipLaunchKernelGGL(adapter_shrink, dim3((unsigned)tiles, (unsigned)(padded_rank(ad.rank) / 32), (unsigned)(ad.N < most ? ad.N : most)),
                     dim3(kShrinkWaves * 64), 0, s, ad, hidden, ldh, ids, (int)T, T_dev, (int)H, U, ids32);
  return hipGetLastError();
}

hipError_t launch_adapter_label(hipStream_t s, const Adapters& ad, const uint16_t* U, const int* ids32, const int64_t* labels, int64_t T, int64_t V,
                                float rcp_temp, const RowResults& from, const int* row_map, const RowResults& to) {
  hipLaunchKernelGGL(adapter_label, dim3((unsigned)((T + 15) / 16)), dim3(256), 0, s, ad, U, ids32, labels, (int)T, V, rcp_temp, from, row_map, to);
  return hipGetLastError();
}

hipError_t launch_adapter_fit_rows(hipStream_t s, const Adapters& ad, const uint16_t* hidden, const uint16_t* weight, int64_t ldw, const int64_t* labels,
                                   const int* ids32, const float* lse, const float* pz, int64_t T, const int* T_dev, int64_t H, int64_t V, float rcp_temp,
                                   const uint16_t* U, float* g, float* q, float* back, uint16_t* U_back) {
  hipLaunchKernelGGL(adapter_fit_rows, dim3((unsigned)((T + 3) / 4)), dim3(256), 0, s, ad, hidden, weight, ldw, labels, ids32, lse, pz, (int)T, T_dev, (int)H,
                     (int)V, rcp_temp, U, g, q, back, U_back);
  return hipGetLastError();
}

hipError_t launch_adapter_gather_rows(hipStream_t s, const int* idx, const uint16_t* hidden, int64_t ldh, int64_t T, int64_t H, const int64_t* labels,
                                      uint16_t* hidden_c, int64_t* labels_c) {
  hipLaunchKernelGGL(adapter_gather_rows, dim3((unsigned)T), dim3(256), 0, s, idx, hidden, ldh, (int)H, labels, hidden_c, labels_c);
  return hipGetLastError();
}

hipError_t launch_adapter_group_rows(hipStream_t s, const float* g, const float* q, const int64_t* labels, int64_t V, const int64_t* ids, int64_t T, int N,
                                     int* idx, int64_t* ids_c, int* seg) {
  hipLaunchKernelGGL((g ? adapter_group_rows<true> : adapter_group_rows<false>), dim3((unsigned)(N + 1)), dim3(kGroupThreads), 0, s, g, q, labels, V, ids, (int)T, N, idx, ids_c, seg);
  return hipGetLastError();
}

int adapter_du_ranges(int64_t T, int64_t columns, int ncu) {
  const int64_t tiles = (T + kDuPiece - 1) / kDuPiece, wanted = (8 * (int64_t)ncu + tiles - 1) / tiles, most = (columns + 511) / 512;
  return (int)(wanted < most ? wanted : most);
}

hipError_t launch_adapter_panel(hipStream_t s, const AdapterPanel& p, int ranges, float* du_part, const uint16_t* U, const int* seg, int row0,
                                const float* sum_in, float* sum_out, uint16_t* dB) {
  const int Rp = padded_rank(p.ad.rank), ranks = (Rp + 63) / 64;
  const int per_range = ((p.columns + ranges - 1) / ranges + kDuColumns - 1) / kDuColumns * kDuColumns;
  hipLaunchKernelGGL(adapter_du_partial, dim3((unsigned)row_pieces(p.T, p.ad.N, kDuPiece), (unsigned)ranges, (unsigned)ranks), dim3(256), 0, s, p, seg, row0,
                     p.columns, per_range, du_part, Rp);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(adapter_db, dim3((unsigned)(p.columns / kDbColumns), (unsigned)p.ad.N, (unsigned)ranks), dim3(256), 0, s, p, U, seg, row0, sum_in,
                     sum_out, dB);
  return hipGetLastError();
}

hipError_t launch_adapter_du_sum(hipStream_t s, const Adapters& ad, const float* part, int slots, int64_t T, const int* T_dev, const int* ids32,
                                 const float* back, uint16_t* dU) {
  const int Rp = padded_rank(ad.rank);
  hipLaunchKernelGGL(adapter_du_sum, dim3((unsigned)((T * (Rp / 4) + 15) / 16)), dim3(256), 0, s, ad, part, slots, (int)T, T_dev, ids32, back, Rp, dU);
  return hipGetLastError();
}

hipError_t launch_adapter_dh_reduce(hipStream_t s, const DhReduceArgs& a, bool shares, int tiles) {
  hipLaunchKernelGGL((shares ? lmhead_dh_reduce<true, true> : lmhead_dh_reduce<false, true>), dim3((unsigned)(tiles * kReduceGroups)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_adapter_finish(hipStream_t s, const Adapters& ad, const uint16_t* hidden, int64_t ldh, const uint16_t* dU, const int* ids32, const int* seg,
                                 int64_t T, const int* T_dev, const int* row_map, const float* back, int64_t H, uint16_t* d_hidden, float* da_part, uint16_t* dA) {
  const unsigned ranks = (unsigned)(padded_rank(ad.rank) / 32);
  if (d_hidden) hipLaunchKernelGGL(adapter_dh_add, dim3((unsigned)((T + 63) / 64), (unsigned)(H / 64)), dim3(256), 0, s, ad, dU, ids32, (int)T, T_dev, row_map,
                     back, (int)H, d_hidden);
  hipLaunchKernelGGL(adapter_da_partial, dim3((unsigned)adapter_da_pieces(T, ad.N), (unsigned)((H + 255) / 256), ranks), dim3(256), 0, s, ad, hidden, ldh, dU,
                     seg, (int)H, da_part);
  hipLaunchKernelGGL(adapter_da_sum, dim3((unsigned)ad.N, (unsigned)ad.rank), dim3(256), 0, s, (const float*)da_part, seg, (int)H, ad.rank, dA);
  return hipGetLastError();
}

}  // namespace lmhead
