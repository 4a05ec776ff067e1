// dHidden rows from slabs of partial sums, with the adapters' part where there is one.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "adapters.hpp"
#include "dh_split.hpp"
#include "gemm_core.hpp"

namespace lmhead {

constexpr int kSlabWaveFloats = TM * TN * 64 * 4;            // one wave's accumulators
constexpr int64_t kSlabTileFloats = NWAVES * kSlabWaveFloats;  // one tile's: 256 KiB

// dHidden rows from the slabs of a split contraction: C[m, n] = bf16(sum of the slabs), added in split order.  One workgroup per
// 16 tokens x 128 columns (an MFMA row block of a wave): 16-byte loads of contiguous slab pieces, 16-byte row pieces out
// through LDS.  HBM-bound, splits x tokens x H x 4 bytes: 8 us at 240 slab tiles (60 MB).  SHARES: of a launch that may have been cut in shares; the
// code for these costs calls of few tokens, which bring it from memory each time: 6.9 -> 8.4 us at 20 tokens, H=1536, 10.0 -> 12.1 at 300, H=512,
// 8.6 -> 11.4 in the draft loss of 20 tokens, H=896, V=246016.
struct DhReduceArgs {
  const float* P;
  int M, H, splits;
  const int *T_dev, *splits_dev, *row_map;  // as in GemmArgs
  uint16_t* C;
  int ldc;
  // The adapters' part (adapters.hpp): every sum, of one slab too, is multiplied by back[token], and A^T du is added to it, before it is rounded.
  Adapters ad;
  const uint16_t* dU;
  const int* ids;
  const float* back;
};
constexpr int kReduceGroups = NWAVES * TM;  // workgroups per tile

template <bool SHARES, bool ADAPTERS = false>
__global__ __launch_bounds__(256) void lmhead_dh_reduce(const DhReduceArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t rows[MT][WN + 8];
  const int splits = a.splits_dev ? *a.splits_dev : a.splits;
  const int M = a.T_dev ? *a.T_dev : a.M;
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (a.H + BN - 1) / BN, tiles = tiles_m * tiles_n;
  const int tile = blockIdx.x / kReduceGroups, wave = blockIdx.x / TM % NWAVES, i = blockIdx.x % TM;
  if ((!ADAPTERS && splits < 2) || tile >= tiles) return;  // without splits the GEMM epilogue has written C
  // Splits: the slabs of a tile stand `tiles` apart, in row order; shares: `groups` apart, in the launch's order.
  int tm = tile / tiles_n, tn = tile % tiles_n, count = splits, step = tiles, slot = tile;
  if (SHARES && splits >= 256) {
    const Shares sh = shares_of(splits, tiles);
    const int in_group = tile / sh.groups, g = tile - in_group * sh.groups, bg = sh.tiles_of(g, tiles), first = sh.first_workgroup(in_group, bg);
    count = __builtin_amdgcn_readfirstlane(sh.last_workgroup(in_group, bg) - first + 1), step = __builtin_amdgcn_readfirstlane(sh.groups);
    slot = __builtin_amdgcn_readfirstlane(sh.slot(g, in_group, first));
    if (!ADAPTERS && count < 2) return;  // one workgroup made the tile, and its epilogue has written C
    banded_tile(tile, tiles_m, tiles_n, kGroupM, tm, tn);
  }
  const int m0 = tm * BM + wave / WAVES_N * WM + i * MT;
  const int n0 = tn * BN + wave % WAVES_N * WN;
  if (m0 >= M || n0 >= a.H) return;
  const int tid = threadIdx.x;
  const float* part = a.P + ((size_t)slot * NWAVES + wave) * kSlabWaveFloats + (size_t)(i * TN) * (64 * 4) + (size_t)tid * 4;
  const size_t slab = (size_t)step * kSlabTileFloats;
  f32x4 sum[2] = {*(const f32x4*)part, *(const f32x4*)(part + 1024)};
#pragma unroll 4
  for (int s = 1; s < count; ++s) {
    sum[0] += *(const f32x4*)(part + (size_t)s * slab);
    sum[1] += *(const f32x4*)(part + (size_t)s * slab + 1024);
  }
  const int lane = tid & 63, lrow = lane & 15, kq = lane >> 4;
  if constexpr (ADAPTERS) {
    // M: the 16 tokens, N: hidden column (A's rows through LDS); the accumulator layout is that of the slabs.
    constexpr int kPitch = WN * 2 + 16;
    __shared__ __attribute__((aligned(16))) char lds[32 * kPitch];
    const int Rp = padded_rank(a.ad.rank), t = m0 + lrow;
    const int id = t < M ? a.ids[t] : -1;
    const uint16_t* du = a.dU + (size_t)(1 + (t < M ? t : M - 1)) * (size_t)(2 * Rp) + kq * 8;
    const float by = a.back[t < M ? t : M - 1];
    int id_of[4];  // of the tokens whose sums this lane holds
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      id_of[r] = __shfl(id, kq * 4 + r, 64);
      const float by_r = __shfl(by, kq * 4 + r, 64);
#pragma unroll
      for (int u = 0; u < 2; ++u) sum[u][r] *= by_r;
    }
    unsigned left = (unsigned)__ballot(id >= 0) & 0xffffu;  // alike in all waves
    while (left) {
      const int one = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
      left &= ~(unsigned)__ballot(id == one);
      const uint16_t* Aa = a.ad.A + (size_t)one * (size_t)a.ad.a_adapter;
      f32x4 more[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      for (int k = 0; k < Rp; k += 32) {
        u32x4 x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // 32 rows of 256 bytes
          const int e = j * 256 + tid, row = k + (e >> 4), h = n0 + (e & 15) * 8;
          x[j] = row < a.ad.rank && h < a.H ? *(const u32x4*)(Aa + (size_t)row * (size_t)a.ad.a_row + h) : u32x4{0u, 0u, 0u, 0u};
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) *(u32x4*)(lds + ((j * 256 + tid) >> 4) * kPitch + (tid & 15) * 16) = x[j];
        __syncthreads();
        const bf16x8 hi = *(const bf16x8*)(du + k), lo = *(const bf16x8*)(du + Rp + k);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 f = transposed(lds + (u * 4 + (tid >> 6)) * MT * 2, kPitch);
          more[u] = mfma(hi, f, more[u]);
          more[u] = mfma(lo, f, more[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[u][r] = id_of[r] == one ? sum[u][r] + more[u][r] : sum[u][r];
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const bf16x4 b4 = __builtin_convertvector(sum[u], bf16x4);
    const uint16_t* h4 = (const uint16_t*)&b4;
#pragma unroll
    for (int r = 0; r < 4; ++r) rows[kq * 4 + r][(u * 4 + (tid >> 6)) * MT + lrow] = h4[r];
  }
  __syncthreads();
  const int r = tid >> 4, c = (tid & 15) * 8, m = m0 + r;
  if (m < M && n0 + c < a.H)
    *(uint4*)(a.C + (size_t)(a.row_map ? a.row_map[m] : m) * (size_t)a.ldc + n0 + c) = *(const uint4*)&rows[r][c];
}

// The reduction with the adapters' part (adapter_kernels.hip), over `tiles` dHidden tiles.
hipError_t launch_adapter_dh_reduce(hipStream_t s, const DhReduceArgs& a, bool shares, int tiles);

}  // namespace lmhead
