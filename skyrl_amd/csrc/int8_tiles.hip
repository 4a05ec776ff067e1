// The head in 8-bit integers: hidden rows and weight rows as int8 values with one fp32 scale each,
//
//   z[t, v] = s_t c_v sum_i q[t, i] w[v, i]
//
// The sum is exact (32-bit integers); it is rounded to fp32, as the bf16 head's sums are, and multiplied by the two scales there.  The tiles are
// those of the bf16 head (gemm_core.hpp, half_tile.hpp): a 16-byte chunk holds sixteen values instead of eight, the matrix instruction takes twice the k
// in the same time, so that slots, copies and schedules stay as they are and a k-tile is 128 k long.
// Statistics: 3.05 ms at T=8192, H=3584, V=152064 (2.9 POP/s; matrix pipe 73 % busy at the 1.85 GHz that power leaves), 326 to 372 us at T=2047, H=1536,
// V=128261 (pipe 55 % busy: 6 of a tile's 21 us are the epilogue, which does not shrink with H), 41 to 45 us at T=137, H=896, V=151936.  Half tiles take 413 us
// where square ones take 359 (T=2047), as for the bf16 head, whose rules choose here too.
#include "int8.hpp"

#include "head_tiles.hpp"

namespace lmhead {
namespace {

constexpr int kRowThreads = 256;

// A workgroup per row: the largest magnitude m, then the values, the second time from the caches.
// Quotients 127 x / m are rounded as if they were exact.  With significands X and M of p bits, 127 x / m is 127 X / (M 2^d), d >= 0: what is not
// exactly between two integers is at least 1 / (M 2^(d + 1)) away from it, 2^-(p + 8) of the quotient or more.  In fp32 (p = 24) a 64-bit division, off
// by 2^-53, stays on its side, and is exact where the quotient lies exactly between.  In bf16 (p = 8) x times the 64-bit 127 / m, rounded to fp32, is off
// by 2^-24, and where the quotient is exactly between, a number of 9 bits, the rounding to fp32 leads back to it.
// Bound by latency (2 us for a row of 896) and then by HBM: 8192 rows of 3584 in bf16 23 us (3.8 TB/s read and written), 2047 of 1536 in fp32 7.3.
template <bool F32>
__global__ __launch_bounds__(kRowThreads) void int8_rows(const char* __restrict__ src, int64_t ld_src, int H, int8_t* __restrict__ values, int64_t ld,
                                                         int K, float* __restrict__ scale) {
  constexpr int ES = F32 ? 4 : 2, E = 8;
  struct __attribute__((packed, aligned(ES))) Piece {
    u32x4 v;
  };
  __shared__ uint32_t most[kRowThreads / 64];
  const int64_t row = blockIdx.x;
  const char* from = src + (size_t)row * (size_t)ld_src * ES;
  auto load = [&](int e0, float (&x)[E]) {  // elements e0 .. e0 + 7, zeros behind the row
    if (e0 + E <= H) {
      const u32x4 a = ((const Piece*)(from + (size_t)e0 * ES))[0].v;
      if constexpr (F32) {
        const u32x4 b = ((const Piece*)(from + (size_t)e0 * ES))[1].v;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(a[i]), x[4 + i] = __uint_as_float(b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(a[i] << 16), x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[i] = 0.f;
        if (e0 + i < H) {
          if constexpr (F32) x[i] = ((const float*)from)[e0 + i];
          else x[i] = __uint_as_float((uint32_t)((const uint16_t*)from)[e0 + i] << 16);
        }
      }
    }
  };
  // Magnitudes as integers compare as they do as floats, and NaN is the largest.
  uint32_t m = 0;
  for (int e0 = threadIdx.x * E; e0 < H; e0 += kRowThreads * E) {
    float x[E];
    load(e0, x);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
      m = m > b ? m : b;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint32_t b = (uint32_t)__shfl_xor((int)m, o, 64);
    m = m > b ? m : b;
  }
  if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
  __syncthreads();
  m = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) m = m > most[w] ? m : most[w];
  const bool odd = m >= 0x7f800000u;  // NaN or an infinity
  const float top = __uint_as_float(m);
  if (threadIdx.x == 0) scale[row] = odd ? NAN : top / 127.f;
  const double per = odd || m == 0 ? 0.0 : 127.0 / (double)top;
  int8_t* const to = values + (size_t)row * (size_t)ld;
  for (int e0 = threadIdx.x * E; e0 < K; e0 += kRowThreads * E) {
    float x[E];
    load(e0, x);
    uint32_t packed[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float q;
      if constexpr (F32) q = per == 0.0 ? 0.f : (float)rint((double)x[i] * 127.0 / (double)top);
      else q = per == 0.0 ? 0.f : rintf((float)((double)x[i] * per));
      packed[i / 4] |= ((uint32_t)(int)q & 0xffu) << (8 * (i % 4));
    }
    *(uint2*)(to + e0) = make_uint2(packed[0], packed[1]);
  }
}

__device__ __forceinline__ Operand bytes_of(const Int8Rows& r, int row0, int rows) { return Operand{(const uint16_t*)r.values, (int)(r.ld / 2), row0, rows}; }

// The scales of a wave's vocabulary rows and tokens, loaded behind the mainloop.  (In front of it they save nothing, because the branch for the vocabulary's last
// rows makes the compiler wait there: 326 -> 400 us at T=2047, H=1536, V=128261; without that branch 322 -> 322.)
template <int NB>
struct Scales {
  f32x4 c[TM];  // of rows v0 + i * 16 + (lane >> 4) * 4 .. + 3
  float s[NB];  // of tokens t0 + j * 16 + (lane & 15)
  int v0, t0;
  __device__ __forceinline__ Scales(const Int8Rows& W, int v0_, int V, const Int8Rows& Hd, int t0_, int T) : v0(v0_), t0(t0_) {
    struct __attribute__((packed, aligned(4))) Four {
      f32x4 v;
    };
    const int lane = threadIdx.x & 63, first = v0 + (lane >> 4) * 4;
    if (v0 + WM <= V) {
#pragma unroll
      for (int i = 0; i < TM; ++i) c[i] = ((const Four*)(W.scale + first + i * MT))->v;
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) c[i][r] = W.scale[first + i * MT + r < V ? first + i * MT + r : V - 1];
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int t = t0 + j * MT + (lane & 15);
      s[j] = Hd.scale[t < T ? t : T - 1];
    }
  }
  // The sums of token block j times the scales of the rows.
  __device__ __forceinline__ void rows(const f32x4 (&acc)[TM][NB], int j, f32x4 (&z)[TM]) const {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) z[i][r] = (float)__float_as_int(acc[i][j][r]) * c[i][r];
  }
};

// Statistics of a wave's logits, as fwd_epilogue() (logits_tile.hpp) makes them; the token's scale enters with the temperature.  Whether all of the wave's rows
// exist is decided in front of the loop over token blocks: inside it, 330 us instead of 326 there, 284 instead of 274 at T=2048, H=896, V=151936.
template <bool ENTROPY, int NB>
__device__ __forceinline__ void int8_stats(const f32x4 (&acc)[TM][NB], const Scales<NB>& scales, const Int8FwdArgs& a, int nparts) {
  const int lane = threadIdx.x & 63, lrow = lane & 15, kq = lane >> 4;
  const int vbase = scales.v0, part = vbase / WM;
  const float per = a.rcp_temp * kLog2e;
  const int rows_kind = __builtin_amdgcn_readfirstlane(vbase + WM <= a.V ? 0 : (vbase < a.V ? 1 : 2));
  auto token_blocks = [&](auto kind) {
    constexpr int KIND = decltype(kind)::value;
    for_each_int(std::make_integer_sequence<int, NB>{}, [&](auto index) {
      constexpr int j = decltype(index)::value;
      const int t = scales.t0 + j * MT + lrow;
      float m = -INFINITY, s = 0.f, e = 0.f;
      if (KIND < 2) {
        f32x4 x[TM], z[TM][1];
        scales.rows(acc, j, x);
#pragma unroll
        for (int i = 0; i < TM; ++i) z[i][0] = x[i];
        fwd_tile_stats<ENTROPY, KIND == 1, false>(z, 0, vbase, a.V, scales.s[j] * per, kq, m, s, e);
      }
      if (kq == 0 && t < a.T) {
        const size_t idx = part_index(part, t, nparts);
        a.part_max[idx] = m;
        a.part_sum[idx] = s;
        if (ENTROPY) a.part_pz[idx] = e;
      }
    });
  };
  if (rows_kind == 0) token_blocks(std::integral_constant<int, 0>{});
  else if (rows_kind == 1) token_blocks(std::integral_constant<int, 1>{});
  else token_blocks(std::integral_constant<int, 2>{});
}

// epilogue(acc, scales) of a tile of whatever shape; v0: its first vocabulary row.
template <int SHAPE, bool EVEN, class Args, class Epilogue>
__device__ __forceinline__ void int8_tile(const Args& a, int v0, int tn, char* lds, Epilogue epilogue) {
  constexpr int NB = wave_cols(SHAPE);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // A part behind the vocabulary (the upper half of the last tile) is made of any row and dropped behind this.
  const Operand oa = bytes_of(a.W, SHAPE == kShort && v0 >= a.V ? a.V - 1 : v0, a.V), ob = bytes_of(a.Hd, tn * BN, a.T);
  f32x4 acc[TM][NB];
  tile_product<SHAPE, EVEN, true>(oa, ob, a.K / kInt8K, lds, acc);
  epilogue(acc, Scales<NB>(a.W, v0 + wave / waves_n(SHAPE) * WM, a.V, a.Hd, tn * BN + wave % waves_n(SHAPE) * (NB * MT), a.T));
}

template <class Args, class Epilogue>
__device__ __forceinline__ void int8_half_tile(const Args& a, char* lds, Epilogue epilogue) {
  const int tiles_m = (a.V + BM - 1) / BM, tiles_n = (a.T + kHalfBN - 1) / kHalfBN;
  int tm, tn;
  tile_coords(blockIdx.x, tiles_m, tiles_n, kGroupM, tm, tn);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  half_acc_t acc;
  half_tile_product<true>(bytes_of(a.W, tm * BM, a.V), bytes_of(a.Hd, tn * kHalfBN, a.T), a.K / kHalfRowBytes, lds, acc);
  epilogue(acc, Scales<kHalfTN>(a.W, tm * BM + wave / WAVES_N * WM, a.V, a.Hd, tn * kHalfBN + wave % WAVES_N * kHalfWN, a.T));
}

template <bool ENTROPY, bool EVEN, bool SHAPES>
__global__ __launch_bounds__(NTHREADS) void int8_fwd_tiles(const Int8FwdArgs a, int split) {
  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
  const int tiles_m = (a.V + BM - 1) / BM, tiles_n = (a.T + BN - 1) / BN;
  const Tile t = tile_of<false, SHAPES>(blockIdx.x, tiles_m, tiles_n, kGroupM, split);
  tile_of_shape<SHAPES>(t, a.T, [&](auto shape, int v0) {
    constexpr int SHAPE = decltype(shape)::value;
    int8_tile<SHAPE, EVEN>(a, v0, t.tn, lds, [&](auto& acc, const auto& scales) { int8_stats<ENTROPY>(acc, scales, a, tiles_m * WAVES_M); });
  });
}

template <bool ENTROPY>
__global__ __launch_bounds__(NTHREADS, 2) void int8_fwd_half_tiles(const Int8FwdArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[kHalfLdsBytes];
  int8_half_tile(a, lds, [&](auto& acc, const auto& scales) { int8_stats<ENTROPY>(acc, scales, a, (a.V + BM - 1) / BM * WAVES_M); });
}

template <bool F32, int NB>
__device__ __forceinline__ void int8_store(const f32x4 (&acc)[TM][NB], const Scales<NB>& scales, const Int8LogitsArgs& a, char* lds) {
  store_logits_tile<F32, NB>(a.out, a.ldo, nullptr, a.T, a.V, scales.v0, scales.t0, lds, [&](int j, f32x4 (&z)[TM]) {
    scales.rows(acc, j, z);
#pragma unroll
    for (int i = 0; i < TM; ++i) z[i] *= scales.s[j];
  });
}

template <bool F32, bool EVEN, bool SHAPES>
__global__ __launch_bounds__(NTHREADS) void int8_logits_tiles(const Int8LogitsArgs a, int split) {
  __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
  const int tiles_m = (a.V + BM - 1) / BM, tiles_n = (a.T + BN - 1) / BN;
  const Tile t = tile_of<false, SHAPES>(blockIdx.x, tiles_m, tiles_n, kGroupM, split);
  tile_of_shape<SHAPES>(t, a.T, [&](auto shape, int v0) {
    constexpr int SHAPE = decltype(shape)::value;
    int8_tile<SHAPE, EVEN>(a, v0, t.tn, lds, [&](auto& acc, const auto& scales) { int8_store<F32>(acc, scales, a, lds); });
  });
}

template <bool F32>
__global__ __launch_bounds__(NTHREADS, 2) void int8_logits_half_tiles(const Int8LogitsArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[kHalfLdsBytes];
  int8_half_tile(a, lds, [&](auto& acc, const auto& scales) { int8_store<F32>(acc, scales, a, lds); });
}

// pick(x, y, z) for the three flags as compile-time constants.
template <class Pick>
auto flagged(Pick pick, bool x, bool y, bool z) {
  const std::true_type t;
  const std::false_type f;
  if (x) return y ? (z ? pick(t, t, t) : pick(t, t, f)) : (z ? pick(t, f, t) : pick(t, f, f));
  return y ? (z ? pick(f, t, t) : pick(f, t, f)) : (z ? pick(f, f, t) : pick(f, f, f));
}

bool even_ktiles(int K) { return K / kInt8K % 2 == 0; }

}  // namespace

hipError_t launch_int8_rows(hipStream_t s, const void* src, bool f32, int64_t ld_src, int64_t rows, int64_t H, int8_t* values, int64_t ld, float* scale) {
  hipLaunchKernelGGL(f32 ? int8_rows<true> : int8_rows<false>, dim3((unsigned)rows), dim3(kRowThreads), 0, s, (const char*)src, ld_src, (int)H, values, ld,
                     (int)((H + kInt8K - 1) / kInt8K * kInt8K), scale);
  return hipGetLastError();
}

hipError_t launch_int8_fwd_tiles(hipStream_t s, const Int8FwdArgs& a, bool half, bool shapes, int split, int workgroups) {
  const dim3 grid((unsigned)workgroups), block(NTHREADS);
  if (half) {
    hipLaunchKernelGGL(a.part_pz ? int8_fwd_half_tiles<true> : int8_fwd_half_tiles<false>, grid, block, 0, s, a);
  } else {
    auto kernel = flagged([](auto pz, auto even, auto others) { return &int8_fwd_tiles<pz.value, even.value, others.value>; }, a.part_pz != nullptr,
                          even_ktiles(a.K), shapes);
    hipLaunchKernelGGL(kernel, grid, block, 0, s, a, split);
  }
  return hipGetLastError();
}

hipError_t launch_int8_logits(hipStream_t s, const Int8LogitsArgs& a, bool half, bool shapes, int split, int workgroups) {
  const dim3 grid((unsigned)workgroups), block(NTHREADS);
  if (half) {
    hipLaunchKernelGGL(a.out_f32 ? int8_logits_half_tiles<true> : int8_logits_half_tiles<false>, grid, block, 0, s, a);
  } else {
    auto kernel = flagged([](auto f32, auto even, auto others) { return &int8_logits_tiles<f32.value, even.value, others.value>; }, a.out_f32 != 0,
                          even_ktiles(a.K), shapes);
    hipLaunchKernelGGL(kernel, grid, block, 0, s, a, split);
  }
  return hipGetLastError();
}

}  // namespace lmhead
