// The LM head with low-rank adapters of many requests: z_t = W h_t + s_a B_a (A_a h_t), a = the adapter of token t.
//
// The products with W are the tiles of the head without adapters (gemm_core.hpp, half_tile.hpp).  What a token's adapter adds is a contraction
// over its rank, a few dozen terms next to the hidden size's thousands, and joins the accumulators in a tile's epilogue, straight from
// global memory: u = s A h, in fp32, is made once per token (adapter_kernels.hip) and kept as two bf16 terms, u = hi +
// lo (exact to 2^-17: bf16 alone would cost a logit 2^-9 of what the adapter adds), and B_a's rows are the A operand of the MFMAs as they
// lie.  A wave walks the distinct adapters of its tokens, whatever their order is; a batch of sequences one behind the other has one or two.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/skyrl_lmhead.h"
#include "gemm_core.hpp"
#include "logits_tile.hpp"

namespace lmhead {

constexpr int64_t kMaxAdapterRank = SKYRL_LMHEAD_MAX_ADAPTER_RANK;

// Rows of u: [T + 1][2][rank padded to 32], hi then lo; row 0 is zeros, row 1 + t token t's (zeros where it has no adapter).
inline __host__ __device__ int padded_rank(int R) { return (R + 31) / 32 * 32; }

struct AdapterTile {
  const uint16_t* B;   // adapters of rows [V, ldb] with `rank` values each; NULL: no adapters
  int64_t b_adapter;   // elements between adapters
  int ldb, rank;
  const uint16_t* U;   // the rows above, from the first token of the tiles' tokens on (row 0 there is not read)
  const uint16_t* zero_row;
  const int* ids;      // adapter of a token, -1 for none
};

// What the adapters of a wave's tokens t0 .. t0 + 16 NB - 1 (of T) add to its accumulators of the vocabulary rows v0 .. v0 + 127 (of V), 16
// tokens at a time: the epilogues, which go through the accumulators block by block, read them through block().  The accumulators
// themselves are left alone: the mainloop holds them in fixed registers, and any loop over adapters that wrote them would have the compiler
// move them about, past MFMAs that it does not know.  A block's sums are one assembly statement of MFMAs into vector registers, and every
// lane, which holds one token, takes the sums of its own adapter only: an adapter's inf or NaN does not reach the tokens of others.
// HOLD: the rows of B are kept from block to block while the adapter stays the same (ranks up to 32); the half tiles, with half of the
// registers, take four row blocks at a time and load them again.
template <int NB, bool HOLD>
struct AdapterTerms {
  static constexpr int kRows = 4;  // row blocks per statement
  const AdapterTile& a;
  int v0, V, t0, id[(NB + 3) / 4];
  int held = -1;
  bf16x8 rows[HOLD ? TM : kRows];

  // In front of the mainloop: the loads of the tokens' adapters.
  __device__ __forceinline__ AdapterTerms(const AdapterTile& a_, int v0_, int V_, int t0_, int T) : a(a_), v0(v0_), V(V_), t0(t0_) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < (NB + 3) / 4; ++u) {
      const int t = t0 + u * 64 + lane;
      id[u] = u * 64 + lane < NB * MT && t < T ? a.ids[t] : -1;
    }
  }

  __device__ __forceinline__ bf16x8 row(const uint16_t* B, int i) const {
    const int v = v0 + i * MT + (threadIdx.x & 15);
    return *(const bf16x8*)(B + (size_t)(v < V ? v : V - 1) * (size_t)a.ldb);
  }
  // Wait states in front for the writes of the operands, behind for the reads of the sums.
  static __device__ __forceinline__ void products(f32x4& s0, f32x4& s1, f32x4& s2, f32x4& s3, const bf16x8* r, const bf16x8& hi, const bf16x8& lo) {
    asm volatile(
        "s_nop 7\n\t"
        "v_mfma_f32_16x16x32_bf16 %0, %4, %8, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %5, %8, %1\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %6, %8, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %7, %8, %3\n\t"
        "v_mfma_f32_16x16x32_bf16 %0, %4, %9, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %5, %9, %1\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %6, %9, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %7, %9, %3\n\t"
        "s_nop 15\n\ts_nop 3"
        : "+v"(s0), "+v"(s1), "+v"(s2), "+v"(s3)
        : "v"(r[0]), "v"(r[1]), "v"(r[2]), "v"(r[3]), "v"(hi), "v"(lo));
  }

  // z = acc[.][j] + the adapters' part.  PIN: the block's accumulators come to vector registers here; left to itself the compiler brings all of
  // them there at the mainloop's end, in front of the stores of logits (which it then spills), not in front of the other epilogues.
  template <bool PIN = false>
  __device__ __forceinline__ void block(int j, f32x4 (&acc)[TM][NB], f32x4 (&z)[TM]) {
    const int lane = threadIdx.x & 63, lrow = lane & 15, kq = lane >> 4;
    __builtin_amdgcn_sched_barrier(0);  // one block's accumulators at a time: there are no registers for the next one's
    const int mine = __shfl(id[j / 4], (j & 3) * 16 + lrow, 64);  // the adapter of this lane's token
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if constexpr (PIN) asm volatile("" : "+a"(acc[i][j]));
      z[i] = acc[i][j];
    }
    unsigned left = (unsigned)__ballot(mine >= 0) & 0xffffu;
    if (left == 0) return;
    const int pitch = 2 * padded_rank(a.rank);
    const uint16_t* u = mine >= 0 ? a.U + (size_t)(1 + t0 + j * MT + lrow) * (size_t)pitch : a.zero_row;
    while (left) {
      const int first = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
      left &= ~(unsigned)__ballot(mine == first);
      const uint16_t* B = a.B + (size_t)first * (size_t)a.b_adapter;
      if constexpr (HOLD) {
        f32x4 sum[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < a.rank; k0 += 32) {
          const int k = k0 + kq * 8;
          const bf16x8 hi = *(const bf16x8*)(u + k), lo = *(const bf16x8*)(u + pitch / 2 + k);
          if (held != first || a.rank > 32) {
#pragma unroll
            for (int i = 0; i < TM; ++i) rows[i] = row(B + (k < a.rank ? k : 0), i);  // behind the rank any value does: u is zero there
            held = first;
          }
          products(sum[0], sum[1], sum[2], sum[3], rows, hi, lo);
          products(sum[4], sum[5], sum[6], sum[7], rows + kRows, hi, lo);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) z[i][r] = mine == first ? z[i][r] + sum[i][r] : z[i][r];
      } else {
#pragma unroll
        for (int i0 = 0; i0 < TM; i0 += kRows) {
          f32x4 sum[kRows];
#pragma unroll
          for (int i = 0; i < kRows; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
          for (int k0 = 0; k0 < a.rank; k0 += 32) {
            const int k = k0 + kq * 8;
            const bf16x8 hi = *(const bf16x8*)(u + k), lo = *(const bf16x8*)(u + pitch / 2 + k);
#pragma unroll
            for (int i = 0; i < kRows; ++i) rows[i] = row(B + (k < a.rank ? k : 0), i0 + i);
            products(sum[0], sum[1], sum[2], sum[3], rows, hi, lo);
          }
#pragma unroll
          for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[i0 + i][r] = mine == first ? z[i0 + i][r] + sum[i][r] : z[i0 + i][r];
        }
      }
    }
  }
};

// ---- launches (adapter_tiles.hip) ----

struct AdapterFwdArgs {
  const uint16_t *W, *Hd;
  int ldw, ldh, T, H, V;
  float rcp_temp;
  float *part_max, *part_sum, *part_pz;
  AdapterTile adapters;
};
// The forward's statistics; shapes / split: which of the kernels, and short tiles, as for lmhead_fwd_tiles.
hipError_t launch_adapter_fwd_tiles(hipStream_t s, const AdapterFwdArgs& a, bool half, bool even, bool shapes, int split, int workgroups);

struct AdapterLogitsArgs {
  const uint16_t *W, *Hd;
  int ldw, ldh, T, H, V;
  void* out;
  int64_t ldo;
  int out_f32;
  AdapterTile adapters;
};
hipError_t launch_adapter_logits(hipStream_t s, const AdapterLogitsArgs& a, bool half, bool even, bool shapes, int split, int workgroups);

hipError_t launch_adapter_dz(hipStream_t s, const DzArgs& z, const AdapterTile& a, bool entgrad, bool half, bool even, bool shapes, int workgroups);

// ---- launches (adapter_kernels.hip) ----

// The adapters of a call.  A [N, rank, H] and B [N, V, rank] bf16, scaling fp32 [N].
struct Adapters {
  const uint16_t* A;
  int64_t a_adapter, a_row;
  const uint16_t* B;
  int64_t b_adapter, b_row;
  const float* scaling;
  int N, rank;
};

// Rows 1 .. T of U (and the zero row 0), and the tokens' adapters as the tiles take them, from ids [T] (int64; outside [0, N): none).  With T_dev
// only that many tokens.
hipError_t launch_adapter_shrink(hipStream_t s, const Adapters& ad, const uint16_t* hidden, int64_t ldh, const int64_t* ids, int64_t T, const int* T_dev,
                                 int64_t H, uint16_t* U, int* ids32);
// logprobs[t] += u_t . B_a[label_t] * rcp_temp: the adapter's part of the label's logit.
hipError_t launch_adapter_label(hipStream_t s, const Adapters& ad, const uint16_t* U, const int* ids32, const int64_t* labels, int64_t T, int64_t V,
                                float rcp_temp, float* logprobs);
// The T rows whose g or q is not zero, grouped by adapter: idx, their ids and the groups' places, seg [N + 2].
hipError_t launch_adapter_group_rows(hipStream_t s, const float* g, const float* q, const int64_t* ids, int64_t T, int N, int* idx, int64_t* ids_c, int* seg);

// A chunk's dz panel, of rows grouped by adapter.
struct AdapterPanel {
  Adapters ad;
  const uint16_t* D;
  int ldd, T;
  const int* T_dev;
  const int* ids;      // of the panel's rows
  int vc0, columns;    // the chunk's first column; panel columns that hold values, a multiple of 256
  int V;
  VocabTail tail;
};
// Ranges of columns that the contraction over a chunk is cut in, whose sums are kept apart: du_part holds [chunks * ranges][T][padded rank] fp32.
int adapter_du_ranges(int64_t T, int64_t columns, int ncu);
// Partial sums of B^T dz, and dB of the chunk's vocabulary rows, (sum_in) + sum -> sum_out fp32 and / or dB bf16, each [N, V, rank] or NULL.  U: of the
// panel's rows; row0: the place of the panel's first row among all rows that seg counts.
hipError_t launch_adapter_panel(hipStream_t s, const AdapterPanel& p, int ranges, float* du_part, const uint16_t* U, const int* seg, int row0,
                                const float* sum_in, float* sum_out, uint16_t* dB);
hipError_t launch_adapter_du_sum(hipStream_t s, const Adapters& ad, const float* part, int slots, int64_t T, const int* T_dev, const int* ids32, uint16_t* dU);

constexpr int kDaPiece = 256;  // rows whose dA is one sum
inline int64_t adapter_da_pieces(int64_t T, int64_t N) { return T / kDaPiece + (N < T ? N : T); }
// d_hidden += A^T du through row_map, and dA [N, rank, H]; da_part: [adapter_da_pieces][padded rank][H] fp32.
hipError_t launch_adapter_finish(hipStream_t s, const Adapters& ad, const uint16_t* hidden, int64_t ldh, const uint16_t* dU, const int* ids32, const int* seg,
                                 int64_t T, const int* T_dev, const int* row_map, int64_t H, uint16_t* d_hidden, float* da_part, uint16_t* dA);

}  // namespace lmhead
