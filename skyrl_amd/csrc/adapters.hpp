// The LM head with low-rank adapters of many requests: z_t = W h_t + s_a B_a (A_a h_t), a = the adapter of token t.
//
// The products with W are the tiles of the head without adapters (gemm_core.hpp, half_tile.hpp).  What a token's adapter adds is a contraction
// over its rank, a few dozen terms next to the hidden size's thousands, and joins the accumulators in a tile's epilogue, straight from
// global memory: u = s A h, in fp32, is made once per token (adapter_kernels.hip) and kept as two bf16 terms, u = hi +
// lo (exact to 2^-17: bf16 alone would cost a logit 2^-9 of what the adapter adds), and B_a's rows are the A operand of the MFMAs as they
// lie.  A wave walks the distinct adapters of its tokens, whatever their order is; a batch of sequences one behind the other has one or two.
//
// What that costs a tile is a trip to memory per 16 tokens' adapter, hidden for the first one behind the mainloop, and its products, 2 of H / 32 per 32 ranks.
// Forwards without / with adapters, all kernels: T=2048, H=896, V=151936, six adapters of rank 32, 446 / 580 us; T=8192, H=3584, V=152064, four, 5.63 / 6.08 ms
// (power). Logits of 16 tokens, H=3584, eight of rank 16: 250 us, 4.5 TB/s of weight, B and logits; rank 64 275 us, 128 314 us.
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
// move them about, past MFMAs that it does not know.  A block's products are one assembly statement of MFMAs into vector registers, once per
// adapter that its tokens have, against zeros for the tokens of others.  The rows of B are kept from block to block while the adapter
// stays the same (ranks up to 32).
//
// A token must not depend on the values of another's adapter, and 0 * inf would be NaN.  So in a block that adapters share the rows' top
// exponent bits are looked at (set from 2.0 on, and in every inf and NaN); where one is set the values that are not finite are replaced by zero, and
// the adapter's own tokens get the NaN.
template <int NB>
struct AdapterTerms {
  static constexpr int kNoToken = -2;
  const AdapterTile& a;
  int v0, V, t0, id[NB];
  int held = -1;
  bf16x8 rows[TM], hi_, lo_;  // hi_, lo_: u of the next block's tokens, the first 32 ranks

  // The loads of the tokens' adapters.
  __device__ __forceinline__ AdapterTerms(const AdapterTile& a_, int v0_, int V_, int t0_, int T) : a(a_), v0(v0_), V(V_), t0(t0_) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int t = t0 + j * MT + (threadIdx.x & 15);
      id[j] = t < T ? a.ids[t] : kNoToken;
    }
  }

  __device__ __forceinline__ const uint16_t* u_row(int j) const {
    return id[j] >= 0 ? a.U + (size_t)((1 + t0 + j * MT + (threadIdx.x & 15)) * (2 * padded_rank(a.rank))) : a.zero_row;
  }
  __device__ __forceinline__ void load_u(int j, int k, bf16x8& hi, bf16x8& lo) const {
    const uint16_t* u = u_row(j) + k;
    hi = *(const bf16x8*)u, lo = *(const bf16x8*)(u + padded_rank(a.rank));
  }
  __device__ __forceinline__ void load_rows(int adapter, int k) {
    const uint16_t* B = a.B + (size_t)adapter * (size_t)a.b_adapter + (k < a.rank ? k : 0);  // behind the rank any value does: u is zero there
    int first = v0 + (threadIdx.x & 15);
    asm volatile("" : "+v"(first));  // the addresses are formed here, where they are needed once in many blocks, and not in front of every block's loop
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int v = first + i * MT;
      rows[i] = *(const bf16x8*)(B + (size_t)(v < V ? v : V - 1) * (size_t)a.ldb);
    }
    held = adapter;
  }
  // The loads of the first block's u and of the first adapter's rows.
  __device__ __forceinline__ void start() {
    const int k = ((threadIdx.x & 63) >> 4) * 8;
    load_u(0, k, hi_, lo_);
    const unsigned long long any = __ballot(id[0] >= 0);
    if (any) load_rows(__builtin_amdgcn_readlane(id[0], (int)__builtin_ctzll(any)), k);
  }

  // z += rows . (hi + lo).  Wait states in front for the writes of the operands, behind for the reads of the sums.
  static __device__ __forceinline__ void products(f32x4 (&z)[TM], const bf16x8 (&r)[TM], const bf16x8& hi, const bf16x8& lo) {
    asm volatile(
        "s_nop 1\n\t"
        "v_mfma_f32_16x16x32_bf16 %0, %8, %16, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %9, %16, %1\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %10, %16, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %11, %16, %3\n\t"
        "v_mfma_f32_16x16x32_bf16 %4, %12, %16, %4\n\tv_mfma_f32_16x16x32_bf16 %5, %13, %16, %5\n\t"
        "v_mfma_f32_16x16x32_bf16 %6, %14, %16, %6\n\tv_mfma_f32_16x16x32_bf16 %7, %15, %16, %7\n\t"
        "v_mfma_f32_16x16x32_bf16 %0, %8, %17, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %9, %17, %1\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %10, %17, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %11, %17, %3\n\t"
        "v_mfma_f32_16x16x32_bf16 %4, %12, %17, %4\n\tv_mfma_f32_16x16x32_bf16 %5, %13, %17, %5\n\t"
        "v_mfma_f32_16x16x32_bf16 %6, %14, %17, %6\n\tv_mfma_f32_16x16x32_bf16 %7, %15, %17, %7\n\t"
        "s_nop 12"
        : "+v"(z[0]), "+v"(z[1]), "+v"(z[2]), "+v"(z[3]), "+v"(z[4]), "+v"(z[5]), "+v"(z[6]), "+v"(z[7])
        : "v"(r[0]), "v"(r[1]), "v"(r[2]), "v"(r[3]), "v"(r[4]), "v"(r[5]), "v"(r[6]), "v"(r[7]), "v"(hi), "v"(lo));
  }

  // Rows of a shared block: values that are not finite become zero, and z NaN there for the adapter's own tokens.
  __device__ __forceinline__ void make_finite(f32x4 (&z)[TM], bool own) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const u32x4 w = __builtin_bit_cast(u32x4, rows[i]);
      bits |= w[0] | w[1] | w[2] | w[3];
    }
    if (!__any((bits & 0x40004000u) != 0u)) return;
    const int kq = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      u32x4 w = __builtin_bit_cast(u32x4, rows[i]);
      bool bad = false;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const bool low = (w[d] & 0x7f80u) == 0x7f80u, high = (w[d] & 0x7f800000u) == 0x7f800000u;
        bad |= low || high;
        w[d] = (low ? 0u : w[d] & 0xffffu) | (high ? 0u : w[d] & 0xffff0000u);
      }
      rows[i] = __builtin_bit_cast(bf16x8, w);
      const unsigned long long lanes = __ballot(bad);
      const unsigned in_row = (unsigned)(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) >> (kq * 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) z[i][r] = own && (in_row >> r & 1u) ? NAN : z[i][r];
    }
    held = -1;  // they are not the adapter's rows any more
  }

  // z = acc[.][j] + the adapters' part.  The accumulators are read by name: left to itself the compiler either brings all of them to vector
  // registers at the mainloop's end and spills them, or works on them where they are and moves them there and back around the products.
  __device__ __forceinline__ void block(int j, f32x4 (&acc)[TM][NB], f32x4 (&z)[TM]) {
    __builtin_amdgcn_sched_barrier(0);  // one block's accumulators at a time: there are no registers for the next one's
    const int mine = id[j], kq8 = ((threadIdx.x & 63) >> 4) * 8;
    bf16x8 hi = hi_, lo = lo_;
    if (j + 1 < NB) load_u(j + 1, kq8, hi_, lo_);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(z[i][r]) : "a"(acc[i][j][r]));
    }
    unsigned left = (unsigned)__ballot(mine >= 0) & 0xffffu;
    while (left) {
      const int first = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
      const unsigned own = (unsigned)__ballot(mine == first) & 0xffffu;
      const bool shared = ((unsigned)__ballot(mine == first || mine == kNoToken) & 0xffffu) != 0xffffu;
      left &= ~own;
      for (int k0 = 0; k0 < a.rank; k0 += 32) {
        if (k0 > 0) {
          int k = k0 + kq8;
          asm volatile("" : "+v"(k));  // as in load_rows()
          load_u(j, k, hi, lo);
        }
        if (held != first || a.rank > 32) load_rows(first, k0 + kq8);
        bf16x8 h = hi, l = lo;
        if (shared) {
          const u32x4 none = {0u, 0u, 0u, 0u};
          h = __builtin_bit_cast(bf16x8, mine == first ? __builtin_bit_cast(u32x4, hi) : none);
          l = __builtin_bit_cast(bf16x8, mine == first ? __builtin_bit_cast(u32x4, lo) : none);
          make_finite(z, mine == first);
        }
        products(z, rows, h, l);
      }
      if (left && a.rank > 32) load_u(j, kq8, hi, lo);
    }
  }
};

typedef __attribute__((ext_vector_type(8))) short i16x8;
typedef __attribute__((address_space(3))) i16x4* lds_half_ptr;

__device__ __forceinline__ f32x4 mfma(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The transposed fragment whose 32 rows of `pitch` bytes begin at `at` (LDS), at the columns that `at` points to.
__device__ __forceinline__ bf16x8 transposed(const char* at, int pitch) {
  const int lane = threadIdx.x & 63, kq = lane >> 4, s = lane & 15;
  const uint32_t addr = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)at + (uint32_t)((kq * 8 + (s >> 2)) * pitch + (s & 3) * 8);
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half_ptr)(uintptr_t)addr);
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half_ptr)(uintptr_t)(addr + 4u * (uint32_t)pitch));
  const i16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8, v);
}

// The gradient on token t's log-probability.  TARGETS: 0 for a label outside [0, V), whose log-probability is the constant 0.
template <bool TARGETS>
__device__ __forceinline__ float target_grad(const float* g, const int64_t* labels, int64_t V, int t) {
  const float gv = g[t];
  if constexpr (!TARGETS) return gv;
  const int64_t y = labels[t];
  return y >= 0 && y < V ? gv : 0.f;
}

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
  const int* row_map;  // NULL, or the row of `out` that a token's logits go to
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
// The results of rows; entropy, row_lse and row_pz may be NULL.
struct RowResults {
  float *logprobs, *entropy, *row_lse, *row_pz;
};
// to.logprobs = from.logprobs + u_t . B_a[label_t] * rcp_temp, the adapter's part of the label's logit.  With row_map all results of row t go to row
// row_map[t] of `to`.
hipError_t launch_adapter_label(hipStream_t s, const Adapters& ad, const uint16_t* U, const int* ids32, const int64_t* labels, int64_t T, int64_t V,
                                float rcp_temp, const RowResults& from, const int* row_map, const RowResults& to);
// The T rows whose g (of a label in [0, V)) or q is not zero (without g all, and no labels), grouped by adapter: idx, their ids and the groups'
// places, seg [N + 2].
hipError_t launch_adapter_group_rows(hipStream_t s, const float* g, const float* q, const int64_t* labels, int64_t V, const int64_t* ids, int64_t T, int N,
                                     int* idx, int64_t* ids_c, int* seg);
// hidden_c [T, H] and labels_c (both or neither of the labels' pointers): the rows that idx names.
hipError_t launch_adapter_gather_rows(hipStream_t s, const int* idx, const uint16_t* hidden, int64_t ldh, int64_t T, int64_t H, const int64_t* labels,
                                      uint16_t* hidden_c, int64_t* labels_c);

// g and q (or NULL) of rows in place, times what makes the label's dz value a bf16 number; its inverse, and U times that in U's form.
hipError_t launch_adapter_fit_rows(hipStream_t s, const Adapters& ad, const uint16_t* hidden, const uint16_t* weight, int64_t ldw, const int64_t* labels,
                                   const int* ids32, const float* lse, const float* pz, int64_t T, const int* T_dev, int64_t H, int64_t V, float rcp_temp,
                                   const uint16_t* U, float* g, float* q, float* back, uint16_t* U_back);

// A chunk's dz panel, of rows grouped by adapter.
struct AdapterPanel {
  Adapters ad;
  const uint16_t* D;
  int ldd, T;
  const int* T_dev;
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
hipError_t launch_adapter_du_sum(hipStream_t s, const Adapters& ad, const float* part, int slots, int64_t T, const int* T_dev, const int* ids32,
                                 const float* back, uint16_t* dU);

constexpr int kDaPiece = 256;  // rows whose dA is one sum
constexpr int kDuPiece = 128;  // rows of one adapter whose du a workgroup forms
// Pieces of at most `size` rows that T rows of N adapters are cut in, at most.
inline int64_t row_pieces(int64_t T, int64_t N, int64_t size) { return T / size + (N < T ? N : T); }
inline int64_t adapter_da_pieces(int64_t T, int64_t N) { return row_pieces(T, N, kDaPiece); }
// d_hidden (when not NULL) = back * d_hidden + A^T du through row_map, and dA [N, rank, H]; da_part: [adapter_da_pieces][padded rank][H] fp32.
hipError_t launch_adapter_finish(hipStream_t s, const Adapters& ad, const uint16_t* hidden, int64_t ldh, const uint16_t* dU, const int* ids32, const int* seg,
                                 int64_t T, const int* T_dev, const int* row_map, const float* back, int64_t H, uint16_t* d_hidden, float* da_part, uint16_t* dA);

}  // namespace lmhead
