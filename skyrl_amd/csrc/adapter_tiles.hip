// Tiles of the head with adapters: the statistics of the forward, the logits themselves, and dz.  Each is a tile of the head without adapters
// (lmhead_kernels.hip, few_tokens.hip) whose epilogue reads the accumulators through AdapterTerms.
#include "adapters.hpp"
#include "head_tiles.hpp"

namespace lmhead {
namespace {

// tile_product() with the loads of the first adapter's rows and of the first block's u between its first copies and the mainloop, which hides
// them: behind the mainloop they cost every tile a trip to memory.
template <int SHAPE, bool EVEN, class Terms>
__device__ __forceinline__ void tile_product_and_start(const Operand& a, const Operand& b, int nk, char* lds, f32x4 (&acc)[TM][wave_cols(SHAPE)],
                                                       Terms& terms) {
  prefetch_first_tiles<false, SHAPE>(a, b, 0, nk, lds);
  terms.start();
  zero_acc(acc);
  if constexpr (SHAPE == kSquare) mainloop<false, EVEN>(a, b, 0, nk, lds, acc);
  else mainloop_ksteps<false, SHAPE>(a, b, 0, nk, lds, acc);
}

// Statistics of a wave's sums, as fwd_epilogue() (logits_tile.hpp) makes them of its accumulators.
template <int NB>
__device__ __forceinline__ void fwd_stats(f32x4 (&acc)[TM][NB], AdapterTerms<NB>& terms, const AdapterFwdArgs& a, int part, int nparts) {
  const int lane = threadIdx.x & 63, lrow = lane & 15, kq = lane >> 4;
  const int vbase = part * WM;
  const float scale2 = a.rcp_temp * kLog2e;
  const int rows_kind = __builtin_amdgcn_readfirstlane(vbase + WM <= a.V ? 0 : (vbase < a.V ? 1 : 2));
  for_each_int(std::make_integer_sequence<int, NB>{}, [&](auto block) {
    constexpr int j = decltype(block)::value;
    const int t = terms.t0 + j * MT + lrow;
    float m = -INFINITY, s = 0.f, e = 0.f;
    f32x4 z[TM][1];
    {
      f32x4 x[TM];
      terms.block(j, acc, x);
#pragma unroll
      for (int i = 0; i < TM; ++i) z[i][0] = x[i];
    }
    if (rows_kind == 0) fwd_tile_stats<true, false, false>(z, 0, vbase, a.V, scale2, kq, m, s, e);
    else if (rows_kind == 1) fwd_tile_stats<true, true, false>(z, 0, vbase, a.V, scale2, kq, m, s, e);
    if (kq == 0 && t < a.T) {
      const size_t idx = part_index(part, t, nparts);
      a.part_max[idx] = m;
      a.part_sum[idx] = s;
      a.part_pz[idx] = e;
    }
  });
}

// epilogue(acc, terms) of a tile of whatever shape; v0: its first vocabulary row.
template <int SHAPE, bool EVEN, class Args, class Epilogue>
__device__ __forceinline__ void head_tile(const Args& a, int v0, int tn, char* lds, Epilogue epilogue) {
  const int wave = threadIdx.x >> 6;
  AdapterTerms<wave_cols(SHAPE)> terms(a.adapters, v0 + wave / waves_n(SHAPE) * WM, a.V, tn * BN + wave % waves_n(SHAPE) * (wave_cols(SHAPE) * MT), a.T);
  // A part behind the vocabulary (the upper half of the last tile) is made of any row and dropped behind this.
  const Operand oa{a.W, a.ldw, SHAPE == kShort && v0 >= a.V ? a.V - 1 : v0, a.V}, ob{a.Hd, a.ldh, tn * BN, a.T};
  f32x4 acc[TM][wave_cols(SHAPE)];
  tile_product_and_start<SHAPE, EVEN>(oa, ob, a.H / BK, lds, acc, terms);
  epilogue(acc, terms);
}

template <class Args, class Epilogue>
__device__ __forceinline__ void head_half_tile(const Args& a, char* lds, Epilogue epilogue) {
  const int tiles_m = (a.V + BM - 1) / BM, tiles_n = (a.T + kHalfBN - 1) / kHalfBN;
  int tm, tn;
  tile_coords(blockIdx.x, tiles_m, tiles_n, kGroupM, tm, tn);
  const int wave = threadIdx.x >> 6, wm = wave / WAVES_N, wn = wave % WAVES_N;
  AdapterTerms<kHalfTN> terms(a.adapters, tm * BM + wm * WM, a.V, tn * kHalfBN + wn * kHalfWN, a.T);
  half_acc_t acc;
  half_tile_product(Operand{a.W, a.ldw, tm * BM, a.V}, Operand{a.Hd, a.ldh, tn * kHalfBN, a.T}, a.H / kHalfBK, lds, acc);
  terms.start();
  epilogue(acc, terms);
}

template <bool EVEN, bool SHAPES>
__global__ __launch_bounds__(NTHREADS) void adapter_fwd_tiles(const AdapterFwdArgs a, int split) {
  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
  const int tiles_m = (a.V + BM - 1) / BM, tiles_n = (a.T + BN - 1) / BN;
  const Tile t = tile_of<false, SHAPES>(blockIdx.x, tiles_m, tiles_n, kGroupM, split);
  tile_of_shape<SHAPES>(t, a.T, [&](auto shape, int v0) {
    constexpr int SHAPE = decltype(shape)::value;
    head_tile<SHAPE, EVEN>(a, v0, t.tn, lds, [&](auto& acc, auto& terms) { fwd_stats(acc, terms, a, terms.v0 / WM, tiles_m * WAVES_M); });
  });
}

__global__ __launch_bounds__(NTHREADS, 2) void adapter_fwd_half_tiles(const AdapterFwdArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[kHalfLdsBytes];
  head_half_tile(a, lds, [&](auto& acc, auto& terms) { fwd_stats(acc, terms, a, terms.v0 / WM, (a.V + BM - 1) / BM * WAVES_M); });
}

template <bool F32, int NB>
__device__ __forceinline__ void store_logits(f32x4 (&acc)[TM][NB], AdapterTerms<NB>& terms, const AdapterLogitsArgs& a, char* lds) {
  store_logits_tile<F32, NB>(a.out, a.ldo, a.row_map, a.T, a.V, terms.v0, terms.t0, lds, [&](int j, f32x4 (&z)[TM]) { terms.block(j, acc, z); });
}

template <bool F32, bool EVEN, bool SHAPES>
__global__ __launch_bounds__(NTHREADS) void adapter_logits_tiles(const AdapterLogitsArgs a, int split) {
  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
  const int tiles_m = (a.V + BM - 1) / BM, tiles_n = (a.T + BN - 1) / BN;
  const Tile t = tile_of<false, SHAPES>(blockIdx.x, tiles_m, tiles_n, kGroupM, split);
  tile_of_shape<SHAPES>(t, a.T, [&](auto shape, int v0) {
    constexpr int SHAPE = decltype(shape)::value;
    head_tile<SHAPE, EVEN>(a, v0, t.tn, lds, [&](auto& acc, auto& terms) { store_logits<F32>(acc, terms, a, lds); });
  });
}

template <bool F32>
__global__ __launch_bounds__(NTHREADS, 2) void adapter_logits_half_tiles(const AdapterLogitsArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[kHalfLdsBytes];
  head_half_tile(a, lds, [&](auto& acc, auto& terms) { store_logits<F32>(acc, terms, a, lds); });
}

// ------------------------------------------------------------------------------------------------------------
// dz (logits_tile.hpp), the adapters' part in the recomputed logits.
// ------------------------------------------------------------------------------------------------------------
template <bool ENTGRAD, bool EVEN, bool SHAPES>
__global__ __launch_bounds__(NTHREADS) void adapter_bwd_dz(const DzArgs z, const AdapterTile ad) {
  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
  static_assert(NWAVES * WN * (kDzTokRow + kDzTokBytes) <= LDS_BYTES, "dz staging and per-token values do not fit LDS");
  int T;
  Tile t;
  if (!dz_tile_of<SHAPES>(z, blockIdx.x, BN, T, t)) return;
  tile_of_shape<SHAPES>(t, T, [&](auto shape, int col0) {
    constexpr int SHAPE = decltype(shape)::value;
    constexpr int NB = wave_cols(SHAPE);
    const int wave = threadIdx.x >> 6;
    const WaveRows rows = wave_vocab_rows(z.vc0 + col0 + wave / waves_n(SHAPE) * WM, z.V, z.tail);
    AdapterTerms<NB> terms(ad, rows.v0, z.V, t.tn * BN + wave % waves_n(SHAPE) * (NB * MT), T);
    dz_tile<ENTGRAD, NB, SHAPE == kShort>(
        z, T, col0, t.tn * BN, lds,
        [&](Operand a, Operand b, f32x4 (&acc)[TM][NB]) {
          tile_product_and_start<SHAPE, EVEN>(a, b, z.H / BK, lds, acc, terms);
          return true;
        },
        [](u32x4 v, u32x4* p) { __builtin_nontemporal_store(v, p); },
        [&](int j, f32x4 (&acc)[TM][NB], f32x4 (&x)[TM]) { terms.block(j, acc, x); });
  });
}

constexpr int kHalfDzLdsBytes = NWAVES * kHalfWN * (kDzTokRow + kDzTokBytes);
static_assert(kHalfDzLdsBytes >= kHalfLdsBytes && 2 * kHalfDzLdsBytes <= LDS_BYTES, "two workgroups per CU");
template <bool ENTGRAD>
__global__ __launch_bounds__(NTHREADS, 2) void adapter_bwd_half_dz(const DzArgs z, const AdapterTile ad) {
  __shared__ __attribute__((aligned(1024))) char lds[kHalfDzLdsBytes];
  int T;
  Tile tile;
  if (!dz_tile_of<false>(z, blockIdx.x, kHalfBN, T, tile)) return;
  const int wave = threadIdx.x >> 6, wm = wave / WAVES_N, wn = wave % WAVES_N;
  const WaveRows rows = wave_vocab_rows(z.vc0 + tile.tm * BM + wm * WM, z.V, z.tail);
  AdapterTerms<kHalfTN> terms(ad, rows.v0, z.V, tile.tn * kHalfBN + wn * kHalfWN, T);
  dz_tile<ENTGRAD, kHalfTN, false>(
      z, T, tile.tm * BM, tile.tn * kHalfBN, lds,
      [&](const Operand& a, const Operand& b, half_acc_t& acc) {
        half_tile_product(a, b, z.H / kHalfBK, lds, acc);
        terms.start();
        return true;
      },
      [](u32x4 v, u32x4* p) { __builtin_nontemporal_store(v, p); },
      [&](int j, half_acc_t& acc, f32x4 (&x)[TM]) { terms.block(j, acc, x); });
}

}  // namespace

hipError_t launch_adapter_fwd_tiles(hipStream_t s, const AdapterFwdArgs& a, bool half, bool even, bool shapes, int split, int workgroups) {
  const dim3 grid((unsigned)workgroups), block(NTHREADS);
  if (half) hipLaunchKernelGGL(adapter_fwd_half_tiles, grid, block, 0, s, a);
  else if (shapes) hipLaunchKernelGGL((even ? adapter_fwd_tiles<true, true> : adapter_fwd_tiles<false, true>), grid, block, 0, s, a, split);
  else hipLaunchKernelGGL((even ? adapter_fwd_tiles<true, false> : adapter_fwd_tiles<false, false>), grid, block, 0, s, a, split);
  return hipGetLastError();
}

hipError_t launch_adapter_logits(hipStream_t s, const AdapterLogitsArgs& a, bool half, bool even, bool shapes, int split, int workgroups) {
  const dim3 grid((unsigned)workgroups), block(NTHREADS);
  if (half) {
    hipLaunchKernelGGL(a.out_f32 ? adapter_logits_half_tiles<true> : adapter_logits_half_tiles<false>, grid, block, 0, s, a);
    return hipGetLastError();
  }
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a, split); };
  if (a.out_f32) {
    if (shapes) launch(even ? adapter_logits_tiles<true, true, true> : adapter_logits_tiles<true, false, true>);
    else launch(even ? adapter_logits_tiles<true, true, false> : adapter_logits_tiles<true, false, false>);
  } else {
    if (shapes) launch(even ? adapter_logits_tiles<false, true, true> : adapter_logits_tiles<false, false, true>);
    else launch(even ? adapter_logits_tiles<false, true, false> : adapter_logits_tiles<false, false, false>);
  }
  return hipGetLastError();
}

hipError_t launch_adapter_dz(hipStream_t s, const DzArgs& z, const AdapterTile& a, bool entgrad, bool half, bool even, bool shapes, int workgroups) {
  const dim3 grid((unsigned)workgroups), block(NTHREADS);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, z, a); };
  if (half) launch(entgrad ? adapter_bwd_half_dz<true> : adapter_bwd_half_dz<false>);
  else if (shapes && even) launch(entgrad ? adapter_bwd_dz<true, true, true> : adapter_bwd_dz<false, true, true>);
  else if (shapes) launch(entgrad ? adapter_bwd_dz<true, false, true> : adapter_bwd_dz<false, false, true>);
  else if (even) launch(entgrad ? adapter_bwd_dz<true, true, false> : adapter_bwd_dz<false, true, false>);
  else launch(entgrad ? adapter_bwd_dz<true, false, false> : adapter_bwd_dz<false, false, false>);
  return hipGetLastError();
}

}  // namespace lmhead
