// What the tile kernels of heads other than the plain bf16 one (adapter_tiles.hip, int8_tiles.hip) have in common: the shapes of a launch's tiles, and
// the way of a tile's logits into memory.
#pragma once
#include "half_tile.hpp"
#include "logits_tile.hpp"

namespace lmhead {

// f(shape, v0): the tile of that shape from vocabulary row v0 on, for the workgroup's tile t.
template <bool SHAPES, class F>
__device__ __forceinline__ void tile_of_shape(const Tile& t, int T, F f) {
  if constexpr (SHAPES) {
    const int shape = shape_of_tile(t.tn, T);
    if (shape == kNarrow) {  // of the two workgroups of a split tile the first makes it
      if (t.half < 1) f(std::integral_constant<int, kNarrow>{}, t.tm * BM);
      return;
    }
    if (t.half >= 0) return f(std::integral_constant<int, kShort>{}, t.tm * BM + t.half * WM);
    if (shape == kMedium) return f(std::integral_constant<int, kMedium>{}, t.tm * BM);
  }
  f(std::integral_constant<int, kSquare>{}, t.tm * BM);
}

// ------------------------------------------------------------------------------------------------------------
// The logits themselves, [T, V] bf16 or fp32.  A lane holds four consecutive vocabulary rows of a token; a wave's 16 tokens x 128 rows go through
// its own part of LDS and leave as 16-byte pieces of whole row segments (256 or 512 bytes).  The rows of an odd vocabulary start anywhere:
// stores of unaligned 16 bytes.
// ------------------------------------------------------------------------------------------------------------
struct __attribute__((packed, aligned(2))) Piece16 {
  u32x4 v;
};

// row_map: where a row of the tile goes, or NULL.  block(j, z): the logits of the wave's token block j.
template <bool F32, int NB, class Block>
__device__ __forceinline__ void store_logits_tile(void* out, int64_t ldo, const int* row_map, int T, int V, int v0, int t0, char* lds, Block block) {
  constexpr int ES = F32 ? 4 : 2, E = 16 / ES;   // elements of a piece
  constexpr int kRow = WM * ES + 16;             // of the stage: 16 bytes further into the banks per token
  constexpr int kPieces = WM / E;                // per token
  static_assert(NWAVES * MT * kRow <= kHalfLdsBytes, "the stage takes the ring's place");
  char* const stage = lds + (threadIdx.x >> 6) * (MT * kRow);  // every wave has left the ring
  const int lane = threadIdx.x & 63, lrow = lane & 15, kq = lane >> 4;
  const int rows = V - v0 < WM ? V - v0 : WM;  // of the wave that exist
  if (rows <= 0) return;
  for_each_int(std::make_integer_sequence<int, NB>{}, [&](auto index) {
    constexpr int j = decltype(index)::value;
    const int here = t0 + j * MT + lrow;
    const int out_row = row_map ? row_map[here < T ? here : T - 1] : here;
    f32x4 z[TM];
    block(j, z);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      char* at = stage + lrow * kRow + (i * MT + kq * 4) * ES;
      if constexpr (F32) {
        *(f32x4*)at = z[i];
      } else {
        const bf16x4 b = __builtin_convertvector(z[i], bf16x4);
        *(uint2*)at = *(const uint2*)&b;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int at = lane % kPieces * E;
    int t = t0 + j * MT + lane / kPieces;
    const char* from = stage + lane / kPieces * kRow + at * ES;
#pragma unroll 2
    for (int it = 0; it < MT * kPieces / 64; ++it) {
      const int row = __shfl(out_row, it * (64 / kPieces) + lane / kPieces, 64);
      if (t < T) {
        char* to = (char*)out + ((size_t)row * (size_t)ldo + (size_t)(v0 + at)) * ES;
        if (at + E <= rows) {
          ((Piece16*)to)->v = *(const u32x4*)from;
        } else {
          for (int e = 0; e < rows - at; ++e) {
            if constexpr (F32) ((float*)to)[e] = ((const float*)from)[e];
            else ((uint16_t*)to)[e] = ((const uint16_t*)from)[e];
          }
        }
      }
      t += 64 / kPieces, from += 64 / kPieces * kRow;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  });
}

}  // namespace lmhead
