// One step of beam search from materialised logits: of each item's beams x vocabulary the k candidates with the largest total, and the beams'
// states brought to the candidates' order.
//
//   y[b, v] = z[b, v] / temperature;   total[b, v] = score_b + y[b, v] - log sum_v exp y[b, v]
//
// Order: the larger total first, the lower beam and then the lower column first among equal ones.  A beam offers its k largest logits (the lower
// column first among equal ones), and they come in that order.  Which of two candidates of different beams comes first hangs on
// the last bits of their totals: those, the row's sum of exponentials and its logarithm are formed in 64 bits, from exponentials in 32 bits that are relative
// to the row's largest logit and off by no more than a unit of their last place: a logarithm is off by 2^-23 (1.2e-7) where all terms are alike, by less
// elsewhere, so that candidates come in the order of their exact totals but where those differ by less than 2.4e-7.
// A beam whose score is -inf, or that has no logit above -inf, offers columns 0 .. k - 1 with a total of -inf; one with NaN among its logits, a
// logit of +inf, or a score that is NaN or +inf offers the same columns with NaN, which sorts behind -inf.
//
// beam_rows   a workgroup per beam and part of its row: one pass for the largest logit, the sum and the k best (as logits_top_rows,
//             top_logits_kernels.hip).  Bound by instructions where there are many beams (the sums, below), for few beams by the way through a workgroup:
//             votes and candidates between the loads of its two steps.  Times of a call: 4 x 151936 in bf16 20 us, the host's; 16 x 8 x 128261 in fp32 30;
//             64 x 8 x 151936 in bf16 58.
// beam_join   a workgroup per item: joins the parts' sums; finds the k best of all parts' sorted lists.  Entry j of a list whose head r heads
//             precede can only be among the k best if j + r < k, and must reach the best of eight bounds, each from the m-th entries of the ceil(k / m) lists
//             with the best heads.  Some 2 k to 8 k entries are left; where that is many, the rank of 64 of them cuts them again.  Each then counts those before
//             it.  8 to 9 us where k is 8 or 16, nearly all of it the latency of what it does one after the other.  Calls of 4 x 151936 in bf16 with k = 8, 64,
//             128: 20, 29, 72 us (elementary torch operations 300), of 16 x 8 x 128261 with k = 16, 64, 128: 30, 39, 107; of that with k = 128 the keys of the
//             rows are the most, whose bound is the least of 128 groups' maxima.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "top_keys.hpp"

namespace {

using namespace logits;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
// 16-byte loads a thread has in flight; with eight the registers of four waves a SIMD have to do.  Four: 54 us for 64 x 8 x 151936 in bf16, 25.4 for
// 16 x 8 x 128261 in fp32; eight: 46 and 24.5.
constexpr int kInFlight = 8;
constexpr int kMaxTop = SKYRL_LOGITS_TOP_MAX;
constexpr int kMaxBeams = SKYRL_LOGITS_BEAMS_MAX;
constexpr int kMaxLists = 512;  // of an item: beams * parts
constexpr int kMaxParts = 64;
constexpr int kGroupsPerWave = kGroups / kWaves;
constexpr int kJoinThreads = 512;
static_assert(kMaxTop <= kGroups && kMaxTop + 64 <= kWaveList && kMaxBeams <= kMaxLists && kMaxParts <= 64, "as in top_logits_kernels.hip; a part a lane");
static_assert((kMaxBeams & (kMaxBeams - 1)) == 0, "a beam in the last bits of a total");
static_assert(1 << (kJoinThreads / 64 - 1) >= kMaxTop, "a wave for each power of two up to k");

// Of one part of a row: its largest logit, sum 2^((z - top) * scale2), how many keys it has found.
struct PartSum {
  double sum;
  float top;
  int keys;
};

struct BeamArgs {
  const void* logits;
  int64_t ld_item, ld_beam;  // elements between items and between an item's beams
  const float* scores;       // [items, beams]
  int beams, V, k, each;     // each: keys of a list, min(k, V)
  double rcp_temp;
  float scale_hi, scale_lo;  // log2(e) / temperature
  PartSum* part;             // [rows, parts]
  topkey_t* keys;            // [rows, parts, each], best first
  float* out_scores;         // [items, k]
  int64_t *parents, *tokens;
};

struct Shared {
  double sum[kWaves];
  float top[kWaves];
  int count[kWaves];
  float bound;  // every wave's candidates reach it
  float group_max[kGroups];
  topkey_t list[kWaves][kWaveList];
  topkey_t all[kWaves * kMaxTop];
};

template <bool F32>
__global__ __launch_bounds__(kThreads, 4) void beam_rows(const BeamArgs a) {
  constexpr int E = Piece<F32>::kElems, ES = F32 ? 4 : 2;
  __shared__ Shared sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x, item = row / a.beams;
  const int V = a.V, k = a.each, part = blockIdx.y, parts = gridDim.y;
  const char* base = (const char*)a.logits + ((size_t)item * (size_t)a.ld_item + (size_t)(row - item * a.beams) * (size_t)a.ld_beam) * ES;
  // Pieces begin at column 0 wherever the row does: beams of the same logits have the same sum, bit for bit, and their totals are equal.
  struct __attribute__((packed, aligned(ES))) Unaligned {
    u32x4 v;
  };
  const int all_pieces = V / E;
  const int first = (int)((int64_t)all_pieces * part / parts), pieces = (int)((int64_t)all_pieces * (part + 1) / parts);
  const int single = part == parts - 1 ? V - all_pieces * E : 0;

  float wave_top = -INFINITY;  // the largest logit of the wave so far
  double sum = 0.0;            // of this lane, relative to it
  float rest = 0.f;            // sum 2^t r of the parts r of the exponents that t leaves
  float lane_max = -INFINITY;
  int count = 0;               // candidates in the wave's list
  topkey_t least = 0;          // candidates have larger keys
  float bound = -INFINITY;
  topkey_t* const list = sm.list[wave];

  // 2^((z - top) scale) into the sums.  An exponent of 10 rounded to 32 bits is off by up to 5e-7, alike for equal logits: what the roundings of the
  // difference and of its product leave, r, comes in with the derivative, ln 2 sum 2^t r.  Of the exponential's own error, a unit of its last place, equal
  // logits have the same share.  Terms are added in 64 bits: beside one of 1 the small ones of a piece would all be rounded the same way.  With neither of the
  // two 39 us instead of 56 for 64 x 8 x 151936 in bf16, bound by instructions, and 26 instead of 29 for 16 x 8 x 128261 in fp32, but sums off by up to 5e-7
  // (with 32-bit sums that keep what each addition loses 59 and 29.5).
  auto add = [&](float z) {
#pragma clang fp contract(off)
    const float top = wave_top > -INFINITY ? wave_top : 0.f;  // -inf - top is -inf and never NaN
    const float d = z - top, back = d - z, lost = (z - (d - back)) + (-top - back);
    const float t = d * a.scale_hi, p = __builtin_amdgcn_exp2f(t);
    const float r = fmaf(lost, a.scale_hi, fmaf(d, a.scale_lo, fmaf(d, a.scale_hi, -t)));
    sum += (double)p;
    rest = fmaf(p, __builtin_amdgcn_fmed3f(r, -1e-3f, 1e-3f), rest);  // NaN or large only where p is 0, or NaN itself
  };
  auto raise = [&](float z) {  // the wave's largest logit, to the largest z of its lanes
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) z = fmaxf(z, __shfl_xor(z, o, 64));
    if (z > wave_top) {
      if (wave_top > -INFINITY) {
        const double f = exp2(((double)wave_top - (double)z) * ((double)a.scale_hi + (double)a.scale_lo));
        sum *= f, rest *= (float)f;
      }
      wave_top = z;
    }
  };
  auto append = [&](float z, int column, bool there) {
    const bool reaches = there && z >= bound;
    if (!__any(reaches)) return;
    const topkey_t key = make_key(z, column);
    const bool hit = reaches && key > least;
    const unsigned long long mask = __ballot(hit);
    if (mask == 0) return;
    if (hit) list[count + __popcll(mask & ((1ull << lane) - 1))] = key;
    count += (int)__popcll(mask);
    wave_fence();
    if (count > kWaveList - 64) {
      least = keep_best(list, count, k);
      count = k;
      bound = fmaxf(bound, value_of_bits(key_bits(least)));
    }
  };

  int step = 0;
  for (int p0 = first + tid; p0 - tid < pieces; p0 += kThreads * kInFlight, ++step) {
    Piece<F32> pc[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int p = p0 + u * kThreads;
      pc[u].widen(((const Unaligned*)(base + (size_t)(p < pieces ? p : pieces - 1) * 16))->v);
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (p0 + u * kThreads < pieces) {
#pragma unroll
        for (int i = 0; i < E; ++i) top = fmaxf(top, pc[u].v[i]);
      }
    }
    lane_max = fmaxf(lane_max, top);
    if (__any(top > wave_top)) raise(top);
    if ((step & (step + 1)) == 0) {  // steps 0, 1, 3, 7: what has been seen doubles
      float m = fmaxf(lane_max, __shfl_xor(lane_max, 1, 64));
      m = fmaxf(m, __shfl_xor(m, 2, 64));
      if ((lane & 3) == 0) sm.group_max[wave * kGroupsPerWave + (lane >> 2)] = m;
      if (step == 0) {
        __syncthreads();
        if (wave == 0) {
          const float b = group_bound(sm.group_max, k);
          if (lane == 0) sm.bound = b;
        }
        __syncthreads();
      } else if (wave == (step & (kWaves - 1))) {  // whatever the other waves have published: a bound all the same
        wave_fence();
        const float b = group_bound(sm.group_max, k);
        if (lane == 0) *(volatile float*)&sm.bound = fmaxf(*(volatile float*)&sm.bound, b);
      }
    }
    bound = fmaxf(bound, *(volatile float*)&sm.bound);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (p0 + u * kThreads < pieces) {
#pragma unroll
        for (int i = 0; i < E; ++i) add(pc[u].v[i]);
      }
    }
    if (__any(top >= bound)) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int p = p0 + u * kThreads;
        float mx = pc[u].v[0];  // again: held since then, the pieces' maxima would not fit the registers
#pragma unroll
        for (int i = 1; i < E; ++i) mx = fmaxf(mx, pc[u].v[i]);
        if (!__any(p < pieces && mx >= bound)) continue;
#pragma unroll
        for (int i = 0; i < E; ++i) append(pc[u].v[i], p * E + i, p < pieces);
      }
    }
  }
  if (single > 0) {  // fewer than a piece
    const bool there = tid < single;
    const int c = all_pieces * E + (there ? tid : 0);
    const float z = load_one(base, (size_t)c, F32);
    raise(there ? z : -INFINITY);
    if (there) add(z);
    append(z, c, there);
  }
  if (count > k && __builtin_amdgcn_readfirstlane(count) > kThreads / kWaves) {  // so that all fit behind each other
    (void)keep_best(list, count, k);
    count = k;
  }
  sum += 0.6931471805599453094 * (double)rest;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) sm.count[wave] = count, sm.sum[wave] = sum, sm.top[wave] = wave_top;
  __syncthreads();
  int total = 0, mine_at = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) mine_at = total;
    total += sm.count[w];
  }
  if (tid == 0) {
    float top = -INFINITY;
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, sm.top[w]);
    double s = 0.0;
    for (int w = 0; w < kWaves; ++w) {
      const double d = ((double)sm.top[w] - (double)top) * ((double)a.scale_hi + (double)a.scale_lo);
      s += sm.top[w] == top ? sm.sum[w] : sm.top[w] > -INFINITY ? sm.sum[w] * exp2(d) : sm.sum[w];  // without a logit: 0, or NaN
    }
    a.part[row * parts + part] = PartSum{s, top, total < k ? total : k};
  }
  for (int e = lane; e < count; e += 64) sm.all[mine_at + e] = list[e];
  __syncthreads();
  for (int e = tid; e < total; e += kThreads) {
    const topkey_t mine = sm.all[e];
    const int place = place_among(sm.all, total, mine);
    if (place < k) a.keys[(row * parts + part) * (int64_t)k + place] = mine;
  }
}

// A candidate: larger ones sort earlier, by `first` and then by the key.  first: the total's bits, so that they compare as the 64-bit floats do and all but the
// last seven, and in their place the beam, lower ones larger.  So candidates of one beam come in the order of their keys even where its score is so large
// that their totals are the same, which the lists of the parts rely on.  NaN is next to 0, none 0.
struct Candidate {
  unsigned long long first, key;
};
__device__ __forceinline__ bool precedes(const Candidate& a, const Candidate& b) { return a.first > b.first || (a.first == b.first && a.key > b.key); }
__device__ __forceinline__ unsigned long long ordered_total(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return x != x ? (unsigned long long)kMaxBeams : b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ Candidate candidate_of(double total, int beam, topkey_t key) {
  return Candidate{(ordered_total(total) & ~(unsigned long long)(kMaxBeams - 1)) | (unsigned)(kMaxBeams - 1 - beam), key};
}
__device__ __forceinline__ int beam_of(const Candidate& c) { return kMaxBeams - 1 - (int)(c.first & (kMaxBeams - 1)); }

__global__ __launch_bounds__(kJoinThreads) void beam_join(const BeamArgs a, int parts) {
  extern __shared__ __attribute__((aligned(16))) char dynamic[];
  __shared__ Candidate heads[kMaxLists];
  __shared__ double offset[kMaxBeams];  // score - log-sum-exp; not finite: the beam's total whatever the column
  __shared__ int have[kMaxLists], rank[kMaxLists];
  __shared__ Candidate bounds[kJoinThreads / 64];
  __shared__ int precede[64];
  __shared__ int kept, fewer;
  Candidate* const left = (Candidate*)dynamic;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t item = blockIdx.x, row0 = item * a.beams;
  const int lists = a.beams * parts, each = a.each, k = a.k;
  // The first keys that a thread will look at, loaded beside the sums: what a list does not have is not looked at later.
  const topkey_t* const keys = a.keys + row0 * parts * (int64_t)each;
  const topkey_t head0 = keys[(int64_t)(tid < lists ? tid : 0) * each], key0 = keys[tid < lists * each ? tid : 0];
  for (int b = wave; b < a.beams; b += kJoinThreads / 64) {
    PartSum p{0.0, -INFINITY, 0};
    if (lane < parts) p = a.part[(row0 + b) * parts + lane];
    float top = p.top;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    double s = p.sum;
    if (p.top > -INFINITY && p.top != top) s *= exp2(((double)p.top - (double)top) * ((double)a.scale_hi + (double)a.scale_lo));
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    const float score = a.scores[row0 + b];
    // No logit above -inf: s is 0, and its logarithm -inf; NaN comes in with s.
    double off = (double)score - ((double)(top > -INFINITY ? top : 0.f) * a.rcp_temp + log(s));
    if (!(score < INFINITY) || s != s || top == INFINITY) off = (double)NAN;
    else if (s == 0.0 || score == -INFINITY) off = -(double)INFINITY;
    if (lane < parts) have[b * parts + lane] = off - off == 0.0 ? p.keys : lane == 0 ? each : 0;
    if (lane == 0) offset[b] = off;
  }
  if (tid < 64) precede[tid] = 0;
  if (tid == 0) kept = 0, fewer = 0;
  __syncthreads();
  auto total_of = [&](int beam, topkey_t key) {
    const double off = offset[beam];
    return off - off == 0.0 ? off + (double)value_of_bits(key_bits(key)) * a.rcp_temp : off;
  };
  auto candidate = [&](int list, int j, topkey_t key) {
    const int b = list / parts;
    const topkey_t mine = offset[b] - offset[b] == 0.0 ? key : make_key(0.f, j);  // of a beam that has no order of its own: columns 0, 1, ...
    return candidate_of(total_of(b, mine), b, mine);
  };
  for (int l = tid; l < lists; l += kJoinThreads) heads[l] = have[l] > 0 ? candidate(l, 0, l == tid ? head0 : keys[(int64_t)l * each]) : Candidate{0, 0};
  __syncthreads();
  for (int l = tid; l < lists; l += kJoinThreads) {
    const Candidate mine = heads[l];
    int r = 0;
#pragma unroll 8
    for (int i = 0; i < lists; ++i) r += precedes(heads[i], mine) ? 1 : 0;
    rank[l] = have[l] > 0 ? r : kMaxLists;
  }
  __syncthreads();
  // Wave w: the m-th entries of the s lists of the best heads, s m >= k.  k candidates reach the last of them.  (The heads of k lists alone, m = 1: 31 us
  // instead of 30 for 16 x 8 x 128261 and k = 16, and no bound where there are fewer lists.)
  {
    const int s = 1 << wave < k ? 1 << wave : k, m = (k + s - 1) / s;
    Candidate last{~0ull, ~0ull};
    int deep = 0;  // lists that have an m-th entry
    for (int l = lane; l < lists; l += 64) {
      if (rank[l] >= s || have[l] < m) continue;
      const Candidate c = candidate(l, m - 1, keys[(int64_t)l * each + m - 1]);
      if (precedes(last, c)) last = c;
      ++deep;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const Candidate c{__shfl_xor(last.first, o, 64), __shfl_xor(last.key, o, 64)};
      if (precedes(last, c)) last = c;
      deep += __shfl_xor(deep, o, 64);
    }
    if (lane == 0) bounds[wave] = deep == s ? last : Candidate{0, 0};
  }
  __syncthreads();
  Candidate least = bounds[0];
#pragma unroll
  for (int w = 1; w < kJoinThreads / 64; ++w)
    if (precedes(bounds[w], least)) least = bounds[w];
  for (int e = tid; e < lists * each; e += kJoinThreads) {
    const int l = e / each, j = e - l * each;
    if (j + rank[l] >= k || j >= have[l]) continue;
    const Candidate c = candidate(l, j, e == tid ? key0 : keys[e]);
    if (!precedes(least, c)) left[atomicAdd(&kept, 1)] = c;  // in any order: places depend on the candidates alone
  }
  __syncthreads();
  int n = kept;
  const Candidate* some = left;
  // Many: of 64 of them the first that k - 1 precede is another bound, behind which about k + n / 64 are left.  They go where the heads were.
  if (n > 2 * kMaxTop) {
    const Candidate sample = left[(int)((int64_t)n * lane / 64)];
    int before = 0;
#pragma unroll 8
    for (int i = wave; i < n; i += kJoinThreads / 64) before += precedes(left[i], sample) ? 1 : 0;
    atomicAdd(&precede[lane], before);
    __syncthreads();
    int b = precede[lane] >= k - 1 ? precede[lane] : 0x7fffffff, at = lane;  // of the sample with the fewest before it, k - 1 or more
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const int b1 = __shfl_xor(b, o, 64), at1 = __shfl_xor(at, o, 64);
      if (b1 < b || (b1 == b && at1 < at)) b = b1, at = at1;
    }
    if (b < kMaxLists) {  // b + 1 are left
      const Candidate last = left[(int)((int64_t)n * at / 64)];
      for (int e = tid; e < n; e += kJoinThreads) {
        const Candidate c = left[e];
        if (!precedes(last, c)) heads[atomicAdd(&fewer, 1)] = c;
      }
      __syncthreads();
      some = heads, n = b + 1;
    }
  }
  for (int e = tid; e < n; e += kJoinThreads) {
    const Candidate mine = some[e];
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) place += precedes(some[i], mine) ? 1 : 0;
    if (place < k) {
      const int64_t at = item * k + place;
      const int b = beam_of(mine);
      a.out_scores[at] = (float)total_of(b, mine.key);
      a.parents[at] = b;
      a.tokens[at] = key_column(mine.key);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// The states of the beams, rows [items * beams] of `segments` segments of `bytes` contiguous bytes each: row j of an item becomes its row
// parents[j].  One launch for all tensors of a layout.  Bound by HBM; rows that several beams take are read from the caches.
// 16 x 8 rows of 4 MiB: 153 us (read and written 1.07 GB: 7.0 TB/s), in place, where rows that stay are left, 164.  16 tensors of 16 x 8 rows, 1.05 GB, as
// segments of 128000 bytes 271 us, of 256 (a transposed cache) 315 (3020 with a workgroup a segment), of 81162 in bf16 at any place 203 us for half as much
// (1040 a byte a lane).
// ------------------------------------------------------------------------------------------------------------
constexpr int kStates = SKYRL_LOGITS_STATES_MAX;
// Pieces that a thread has in flight.  A copy of 64 rows of 4 MiB: 78 us with one or two, 80 with four, 130 with eight.
constexpr int kCopyThreads = 256, kCopyPieces = 2;
// In place.  Eight, four and two: 203, 220 and 240 us for 128 beams of 2 MiB, 427, 409 and 333 for 16 x 16 of 4 MiB, whose pieces of one column, a power of
// two apart, meet in the same channels of the memory; 157, 154 and 153 where they are 4000256 bytes apart, 16 x 8.
constexpr int kHeldPieces = 2;

struct ReorderArgs {
  const char* from[kStates];
  char* to[kStates];
  int64_t from_row, from_segment, to_row, to_segment;  // bytes
  const int64_t* parents;  // [items, beams_out]
  int beams_in, beams_out;
  uint32_t all, pieces;    // pieces of a row, below 2^31, and of a segment
  uint32_t last;           // bytes of a segment's last piece
  uint32_t magic, shift;   // p / pieces is p * magic >> shift
  uint32_t blocks;         // workgroups of a row
};

// Sixteen bytes of a segment, whose begin, end and neighbours are multiples of G bytes; or the fewer that it ends with.
template <int G>
struct Piece16 {
  struct __attribute__((packed, aligned(G))) Whole {
    u32x4 v;
  };
  static __device__ __forceinline__ u32x4 load(const char* from, uint32_t bytes) {
    if (G == 16 || bytes == 16) return ((const Whole*)from)->v;
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / G; ++i) {
      if (i * G >= (int)bytes) break;
      if constexpr (G == 4) w[i] = ((const uint32_t*)from)[i];
      if constexpr (G == 2) w[i / 2] |= (uint32_t)((const uint16_t*)from)[i] << (16 * (i % 2));
      if constexpr (G == 1) w[i / 4] |= (uint32_t)((const uint8_t*)from)[i] << (8 * (i % 4));
    }
    return w;
  }
  static __device__ __forceinline__ void store(char* to, uint32_t bytes, const u32x4& w) {
    if (G == 16 || bytes == 16) {
      ((Whole*)to)->v = w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 16 / G; ++i) {
      if (i * G >= (int)bytes) break;
      if constexpr (G == 4) ((uint32_t*)to)[i] = w[i];
      if constexpr (G == 2) ((uint16_t*)to)[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
      if constexpr (G == 1) ((uint8_t*)to)[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    }
  }
};

// Where piece p of a row lies: its segment, its place in that in bytes and how many it has.  Pieces are numbered through the segments, so that a workgroup has
// as much to do where they are short.
struct Place {
  int64_t segment, at;
  uint32_t bytes;
  __device__ __forceinline__ Place(const ReorderArgs& a, uint32_t p) {
    const uint32_t q = (uint32_t)(((uint64_t)p * a.magic) >> a.shift), r = p - q * a.pieces;
    segment = q, at = (int64_t)r * 16, bytes = r + 1 == a.pieces ? a.last : 16u;
  }
};

template <int G>
__global__ __launch_bounds__(kCopyThreads) void beam_copy(const ReorderArgs a) {
  const uint32_t row = blockIdx.x / a.blocks, block = blockIdx.x - row * a.blocks;
  const uint32_t item = row / (uint32_t)a.beams_out;
  const int64_t parent = a.parents[row];
  const bool has = parent >= 0 && parent < a.beams_in;
  const char* const from = a.from[blockIdx.y] + ((int64_t)item * a.beams_in + (has ? parent : 0)) * a.from_row;
  char* const to = a.to[blockIdx.y] + (int64_t)row * a.to_row;
  const uint32_t p0 = block * (kCopyThreads * kCopyPieces) + threadIdx.x;
  u32x4 w[kCopyPieces];
#pragma unroll
  for (int u = 0; u < kCopyPieces; ++u) {
    const uint32_t p = p0 + u * kCopyThreads;
    w[u] = u32x4{0, 0, 0, 0};
    if (has && p < a.all) {
      const Place x(a, p);
      w[u] = Piece16<G>::load(from + x.segment * a.from_segment + x.at, x.bytes);
    }
  }
#pragma unroll
  for (int u = 0; u < kCopyPieces; ++u) {
    const uint32_t p = p0 + u * kCopyThreads;
    if (p < a.all) {
      const Place x(a, p);
      Piece16<G>::store(to + x.segment * a.to_segment + x.at, x.bytes, w[u]);
    }
  }
}

// In place: a thread reads one piece of all beams of an item into LDS before it writes any.  Rows that stay are not written, and those that no
// other beam takes not read.
template <int G>
__global__ __launch_bounds__(kCopyThreads) void beam_permute(const ReorderArgs a) {
  extern __shared__ __attribute__((aligned(16))) char dynamic[];
  __shared__ int parent[kMaxBeams];
  __shared__ int wanted[kMaxBeams];
  __shared__ int source[kMaxBeams];  // the beams that are wanted, one behind the other
  __shared__ int sources;
  const uint32_t item = blockIdx.x / a.blocks, block = blockIdx.x - item * a.blocks;
  const int beams = a.beams_in;
  for (int b = threadIdx.x; b < beams; b += blockDim.x) wanted[b] = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < beams; b += blockDim.x) {
    const int64_t p = a.parents[(int64_t)item * beams + b];
    parent[b] = p >= 0 && p < beams ? (int)p : -1;
    if (p >= 0 && p < beams && p != b) wanted[p] = 1;  // the same value from whichever beam
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    int n = 0;
    for (int b0 = 0; b0 < beams; b0 += 64) {
      const int b = b0 + (int)threadIdx.x;
      const bool take = b < beams && wanted[b];
      const unsigned long long mask = __ballot(take);
      if (take) source[n + __popcll(mask & ((1ull << threadIdx.x) - 1))] = b;
      n += (int)__popcll(mask);
    }
    if (threadIdx.x == 0) sources = n;
  }
  __syncthreads();
  const uint32_t p = block * blockDim.x + threadIdx.x;
  if (p >= a.all) return;
  const Place x(a, p);
  char* const base = a.to[blockIdx.y] + (int64_t)item * beams * a.to_row + x.segment * a.to_segment + x.at;
  u32x4* const mine = (u32x4*)dynamic + threadIdx.x;
  const int n = __builtin_amdgcn_readfirstlane(sources);
  for (int i = 0; i < n; i += kHeldPieces) {
    u32x4 w[kHeldPieces];
#pragma unroll
    for (int u = 0; u < kHeldPieces; ++u)
      if (i + u < n) w[u] = Piece16<G>::load(base + (int64_t)source[i + u] * a.to_row, x.bytes);
#pragma unroll
    for (int u = 0; u < kHeldPieces; ++u)
      if (i + u < n) mine[source[i + u] * blockDim.x] = w[u];
  }
#pragma unroll 4
  for (int b = 0; b < beams; ++b) {
    const int from = parent[b];
    if (from == b) continue;
    Piece16<G>::store(base + (int64_t)b * a.to_row, x.bytes, from < 0 ? u32x4{0, 0, 0, 0} : mine[from * blockDim.x]);
  }
}

// Entries that can be left of `lists` lists of `each`: sum over the heads' ranks r of what j + r < k allows.
size_t most_left(int lists, int each, int k) {
  size_t n = 0;
  for (int r = 0; r < lists && r < k; ++r) n += (size_t)(each < k - r ? each : k - r);
  return n;
}

// Parts of a row: so many that 512 workgroups share the logits (two a CU, all at once), of at least 8192 logits each.  16 x 8 x 128261 in bf16 and fp32: 23
// and 25 us with 512 workgroups, 26 and 25 with 768, 27 and 29 with 1024.
int beam_parts(int64_t rows, int64_t beams, int64_t V) {
  int64_t n = 512 / rows;
  if (n > V / 8192) n = V / 8192;
  if (n > kMaxParts) n = kMaxParts;
  if (n > kMaxLists / beams) n = kMaxLists / beams;
  return n < 1 ? 1 : (int)n;
}

bool beam_extents(int64_t items, int64_t beams, int64_t V, int64_t k) {
  return items >= 1 && beams >= 1 && beams <= kMaxBeams && items <= ((int64_t)1 << 22) / beams && V >= 1 && V < ((int64_t)1 << 31) && k >= 1 && k <= kMaxTop &&
         k <= beams * V;
}

// A launch for as many rows as one grid holds (2^32 threads), or as many segments of one row.
template <int G>
int launch_reorder(hipStream_t s, const ReorderArgs& whole, int64_t items, int64_t segments, int64_t bytes, int count, bool in_place) {
  const int64_t pieces = (bytes + 15) / 16;
  if (pieces >= ((int64_t)1 << 31)) return SKYRL_LMHEAD_ERR_SHAPE;
  int threads = kCopyThreads;
  if (in_place)  // two workgroups a CU, but for 128 beams.  (One: within 4 % for 32 and 64 beams.)
    while (threads > 64 && (size_t)whole.beams_in * threads * 16 > 65536) threads /= 2;
  const int64_t each = in_place ? threads : kCopyThreads * kCopyPieces;
  const int64_t most = (((int64_t)1 << 32) - 1) / threads;  // workgroups
  int log = 0;
  while (((int64_t)1 << log) < pieces) ++log;
  const int64_t most_segments = (((int64_t)1 << 31) - 1) / pieces, step_segments = segments < most_segments ? segments : most_segments;
  const int64_t blocks = (step_segments * pieces + each - 1) / each, rows = most / blocks;  // of a launch; 2^31 pieces are 2^23 or 2^25 workgroups
  const int64_t step_items = in_place ? rows : (rows >= whole.beams_out ? rows / whole.beams_out : 1);
  const int64_t step_beams = in_place || rows >= whole.beams_out ? whole.beams_out : rows;  // of an item, where a launch has part of one
  for (int64_t item = 0; item < items; item += step_items)
    for (int64_t beam = 0; beam < whole.beams_out; beam += step_beams)
      for (int64_t segment = 0; segment < segments; segment += step_segments) {
        ReorderArgs a = whole;
        const int64_t n_items = items - item < step_items ? items - item : step_items;
        const int64_t n_beams = whole.beams_out - beam < step_beams ? whole.beams_out - beam : step_beams;
        const int64_t n_segments = segments - segment < step_segments ? segments - segment : step_segments;
        for (int t = 0; t < count; ++t) {
          a.from[t] += item * whole.beams_in * whole.from_row + segment * whole.from_segment;
          a.to[t] += (item * whole.beams_out + beam) * whole.to_row + segment * whole.to_segment;
        }
        a.parents += item * whole.beams_out + beam;
        a.beams_out = (int)n_beams;
        a.all = (uint32_t)(n_segments * pieces), a.pieces = (uint32_t)pieces, a.last = (uint32_t)(bytes - (pieces - 1) * 16);
        // magic = 2^(31 + log) / pieces, rounded up, is too large by less than one part in 2^31, which no p < 2^31 sees.
        a.magic = (uint32_t)((((uint64_t)1 << (31 + log)) + (uint64_t)pieces - 1) / (uint64_t)pieces), a.shift = (uint32_t)(31 + log);
        a.blocks = (uint32_t)((n_segments * pieces + each - 1) / each);
        const dim3 grid((unsigned)(a.blocks * (in_place ? n_items : n_items * n_beams)), (unsigned)count);
        if (in_place) hipLaunchKernelGGL(beam_permute<G>, grid, dim3((unsigned)threads), (size_t)a.beams_in * threads * 16, s, a);
        else hipLaunchKernelGGL(beam_copy<G>, grid, dim3(kCopyThreads), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
      }
  return SKYRL_LMHEAD_OK;
}

}  // namespace

extern "C" {

size_t skyrl_logits_beam_select_workspace_bytes(int64_t items, int64_t beams, int64_t V, int64_t k) {
  if (!beam_extents(items, beams, V, k)) return 0;
  const int64_t rows = items * beams;
  return (size_t)rows * (size_t)beam_parts(rows, beams, V) * (sizeof(PartSum) + (size_t)(k < V ? k : V) * sizeof(topkey_t));
}

int skyrl_logits_beam_select(const void* logits, int logits_dtype, int64_t ld_item, int64_t ld_beam, const float* scores, int64_t items, int64_t beams,
                             int64_t V, int64_t k, double rcp_temperature, float* out_scores, int64_t* parents, int64_t* tokens, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (!logits || !scores || !out_scores || !parents || !tokens) return SKYRL_LMHEAD_ERR_NULL;
  if (logits_dtype != SKYRL_LOGITS_BF16 && logits_dtype != SKYRL_LOGITS_F32) return SKYRL_LMHEAD_ERR_ARG;
  if (!beam_extents(items, beams, V, k) || ld_item < 0 || ld_beam < 0 || ld_item >= ((int64_t)1 << 40) || ld_beam >= ((int64_t)1 << 40))
    return SKYRL_LMHEAD_ERR_SHAPE;
  const bool f32 = logits_dtype == SKYRL_LOGITS_F32;
  if (((uintptr_t)logits & (f32 ? 3u : 1u)) || (((uintptr_t)scores | (uintptr_t)out_scores) & 3u) ||
      (((uintptr_t)parents | (uintptr_t)tokens | (uintptr_t)workspace) & 7u))
    return SKYRL_LMHEAD_ERR_ALIGN;
  const double scale2 = rcp_temperature * 1.4426950408889634074;
  const float scale_hi = (float)scale2;
  if (!(rcp_temperature > 0.0) || !std::isfinite(scale_hi) || !(scale_hi >= 0x1p-100f)) return SKYRL_LMHEAD_ERR_ARG;
  if (!workspace || workspace_bytes < skyrl_logits_beam_select_workspace_bytes(items, beams, V, k)) return SKYRL_LMHEAD_ERR_WORKSPACE;
  const int64_t rows = items * beams;
  const int parts = beam_parts(rows, beams, V), each = (int)(k < V ? k : V);
  topkey_t* const keys = (topkey_t*)workspace;
  const BeamArgs a{logits, ld_item, ld_beam, scores, (int)beams, (int)V, (int)k, each, rcp_temperature, scale_hi, (float)(scale2 - (double)scale_hi),
                   (PartSum*)(keys + (size_t)rows * (size_t)parts * (size_t)each), keys, out_scores, parents, tokens};
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(f32 ? beam_rows<true> : beam_rows<false>, dim3((unsigned)rows, (unsigned)parts), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(beam_join, dim3((unsigned)items), dim3(kJoinThreads), most_left((int)beams * parts, each, (int)k) * sizeof(Candidate), s, a, parts);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SKYRL_LMHEAD_OK : (int)e;
}

int skyrl_logits_beam_reorder(const void* const* from, void* const* to, int64_t count, int64_t from_row, int64_t from_segment, int64_t to_row,
                              int64_t to_segment, int64_t segments, int64_t bytes, const int64_t* parents, int64_t items, int64_t beams_in, int64_t beams_out,
                              void* stream) {
  if (!from || !to || !parents) return SKYRL_LMHEAD_ERR_NULL;
  const int64_t most = (int64_t)1 << 40;
  if (count < 1 || count > kStates || segments < 1 || segments >= ((int64_t)1 << 31) || bytes < 1 || bytes >= most || items < 1 || beams_in < 1 || beams_out < 1 ||
      items >= ((int64_t)1 << 31) || beams_in >= ((int64_t)1 << 31) || beams_out >= ((int64_t)1 << 31) || items * beams_out >= ((int64_t)1 << 31) ||
      items * beams_in >= ((int64_t)1 << 31) || from_row < 0 || from_segment < 0 || to_row < 0 || to_segment < 0 || from_row >= most || from_segment >= most ||
      to_row >= most || to_segment >= most)
    return SKYRL_LMHEAD_ERR_SHAPE;
  const double far = (double)((int64_t)1 << 62);  // no memory has such places, whose products might not be held in 64 bits
  if ((double)items * (double)beams_in * (double)from_row + (double)segments * (double)from_segment >= far ||
      (double)items * (double)beams_out * (double)to_row + (double)segments * (double)to_segment >= far)
    return SKYRL_LMHEAD_ERR_SHAPE;
  if ((uintptr_t)parents & 7u) return SKYRL_LMHEAD_ERR_ALIGN;
  const bool in_place = from[0] == to[0];
  if (in_place && (beams_in != beams_out || beams_in > kMaxBeams || from_row != to_row || from_segment != to_segment)) return SKYRL_LMHEAD_ERR_ARG;
  ReorderArgs a{};
  uintptr_t all = (uintptr_t)bytes | (uintptr_t)from_row | (uintptr_t)from_segment | (uintptr_t)to_row | (uintptr_t)to_segment;
  for (int64_t i = 0; i < count; ++i) {
    if (!from[i] || !to[i]) return SKYRL_LMHEAD_ERR_NULL;
    if ((from[i] == to[i]) != in_place) return SKYRL_LMHEAD_ERR_ARG;
    a.from[i] = (const char*)from[i], a.to[i] = (char*)to[i];
    all |= (uintptr_t)from[i] | (uintptr_t)to[i];
  }
  a.from_row = from_row, a.from_segment = from_segment, a.to_row = to_row, a.to_segment = to_segment;
  a.parents = parents, a.beams_in = (int)beams_in, a.beams_out = (int)beams_out;
  hipStream_t s = (hipStream_t)stream;
  if (all % 16 == 0) return launch_reorder<16>(s, a, items, segments, bytes, (int)count, in_place);
  if (all % 4 == 0) return launch_reorder<4>(s, a, items, segments, bytes, (int)count, in_place);
  if (all % 2 == 0) return launch_reorder<2>(s, a, items, segments, bytes, (int)count, in_place);
  return launch_reorder<1>(s, a, items, segments, bytes, (int)count, in_place);
}

}  // extern "C"
