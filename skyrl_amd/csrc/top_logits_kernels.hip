// Log-probability, rank and entropy of given tokens and the k best alternatives with their log-probabilities, from materialised logits
// [T, V] in ONE pass over them; and the gradient of the logits from gradients on all of those, in one read and write pass.
//
//   y = z / temperature;  lse = log sum exp y;  logprob = y[label] - lse;  entropy = lse - sum softmax(y) y
//   rank = 1 + number of columns that sort before the label;  top = the first k columns of that order, with y[column] - lse
//   dz = ( g (1[label] - p) - q p (y - pz) + sum_j h_j (1[top_j] - p) ) / temperature,      p = exp(y - lse)
//
// Order of columns: the larger logit first, the lower column first among equal ones (-0 equals +0); NaN behind everything.  It is total, so that
// the k best are one set whatever order candidates are found in.
// A row without any logit above -inf has lse = -inf: log-probabilities -inf, entropy 0, zero gradient, columns 0 .. k - 1.
//
// Selection.  A candidate must reach the k-th largest of the maxima of 128 groups of lanes: those are 128 different logits, so at least k
// logits reach it, and hardly more do (-128 ln(1 - k / 128): 22 for k = 20, 37 for k = 32).  The bound is formed from a workgroup's first 32 KiB (n =
// 16384 bf16 or 8192 fp32 logits) before any of them is looked at, and again whenever what has been seen doubles, so that a workgroup that walks v
// logits has about k (1 + ln(v / n)) candidates.
// The running maximum of the softmax is one value per wave, so that it, the bound and the label's logit (the rank) cost one comparison and
// vote each per four pieces of a lane; only where a vote says so are the pieces gone through again.
//
// Few rows are cut in parts, a workgroup each, whose statistics and k best are joined by a second launch.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "top_keys.hpp"

namespace {

using namespace logits;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBwdThreads = 1024;
constexpr int kInFlight = 4;  // 16-byte loads a thread has in flight
constexpr int kMaxTop = SKYRL_LOGITS_TOP_MAX;
constexpr int kGroupsPerWave = kGroups / kWaves;
static_assert(kMaxTop <= kGroups && kMaxTop + 64 <= kWaveList, "a bound of k groups; room for the candidates of one step behind the k best");

constexpr int kMaxJoin = 2048;  // candidates that the parts of a row bring to the join
constexpr int kMaxParts = 64;

// What the waves of a workgroup share.
struct Shared {
  Stats stats[kWaves];
  topkey_t list[kWaves][kWaveList];
  topkey_t all[kWaves * kMaxTop];  // the candidates of all waves, side by side
  float group_max[kGroups];
  float bound;  // every wave's candidates reach it
  int count[kWaves], better[kWaves];
};
static_assert(kWaves * kMaxTop >= kThreads, "up to a candidate per thread without dropping any");

// The maximum of a part whose logits all lie below kLowest: only where there is no logit above -inf it stays kLowest itself.
constexpr float kFarPart = -2.9e38f;

// A part's result: its statistics, the columns that sort before the label, and how many of its k keys there are, best first.
struct Part {
  Stats st;
  int better, keys;
};

// The smallest float above z (z is not NaN; +inf gives NaN, which nothing reaches).
__device__ __forceinline__ float next_above(float z) {
  const int b = __float_as_int(z + 0.f);
  return __int_as_float(b >= 0 ? b + 1 : b - 1);
}

struct TopArgs {
  const void* logits;
  int64_t ld;
  const int64_t* labels;  // NULL: no log-probability and no rank wanted
  int V, k;
  float rcp_temp;
  float *logprobs, *entropy, *row_lse, *row_pz;
  int64_t* ranks;
  float* top_logprobs;
  int64_t* top_ids;
  Part* part;   // [T, parts], and the keys [T, parts, k], where rows are cut
  topkey_t* keys;
};

// The results of a row from its statistics (far: those of far_row) and the number of columns before the label, by one thread; logprob_of for
// the alternatives.
struct RowResult {
  bool empty, far;
  float log_s, m, scale2, rcp_temp;
  __device__ __forceinline__ RowResult(const Stats& st, float rcp_temp_, bool far_)
      : empty(!far_ && st.s == 0.f), far(far_), m(st.m), scale2(rcp_temp_ * kLog2e), rcp_temp(rcp_temp_) {
    log_s = empty ? -INFINITY : logf(st.s);
  }
  __device__ __forceinline__ float logprob_of(float z) const {
    if (empty) return -INFINITY;
    const bool finite_z = fabsf(z) < INFINITY;
    if (far) {
      const float d = z - m;
      return (finite_z && fabsf(d) == INFINITY ? z * rcp_temp - m * rcp_temp : d * rcp_temp) - log_s;
    }
    const float t = fmaf(z, scale2, -m);
    if (finite_z && fabsf(t) == INFINITY) return z * rcp_temp - fmaf(m, kLn2, log_s);  // y in base 2 overflows before y does
    return t * kLn2 - log_s;
  }
  __device__ __forceinline__ void write(const TopArgs& a, int64_t row, const Stats& st, bool has_label, float z_label, int before) const {
    if (a.ranks) a.ranks[row] = has_label && z_label == z_label ? 1 + before : 0;
    if (a.logprobs) a.logprobs[row] = has_label ? logprob_of(z_label) : 0.f;
    if (a.entropy) a.entropy[row] = empty ? 0.f : log_s - st.e / st.s * kLn2;
    const float mean = st.e / st.s;
    if (a.row_lse) a.row_lse[row] = empty ? -INFINITY : far ? finite(fmaf(m, rcp_temp, log_s)) : fmaf(m, kLn2, log_s);
    if (a.row_pz) a.row_pz[row] = empty ? 0.f : far ? finite(fmaf(m, rcp_temp, mean * kLn2)) : (mean + m) * kLn2;
  }
};

// Fewer logits than k that are numbers (`place` of them): the first NaN columns, in order, by one wave.
template <bool F32>
__device__ __noinline__ void fill_with_nan(int V, int k, int64_t* ids, float* logprobs, const char* base, int place) {
  const int lane = threadIdx.x & 63;
  for (int c0 = 0; c0 < V && place < k; c0 += 64) {
    const int c = c0 + lane;
    const float z = c < V ? load_one(base, (size_t)c, F32) : 0.f;
    const unsigned long long mask = __ballot(z != z);
    const int at = place + (int)__popcll(mask & ((1ull << lane) - 1));
    if (z != z && at < k) ids[at] = c, logprobs[at] = NAN;
    place += (int)__popcll(mask);
  }
}

// One workgroup per row and part (PARTS: grid.y of them).
// Bound by HBM on fp32 logits, by the vector instructions (an exponential, the comparisons, widening) on bf16: 2048 x 152064 fp32, k = 5, 217 us (5.7
// TB/s); 4096 x 151936 bf16, k = 32, 316 us (3.9 TB/s; in a graph of two calls 277), of which 36 are the ranks and candidates.  What brought it there from 510: one running maximum
// a wave and votes per four pieces instead of one (437), keys formed only where a logit reaches the bound (394), no memory for
// arguments of a call (322).  Loading a step ahead changed nothing (328 to 358): two or three workgroups a CU overlap enough.
template <bool F32, bool PARTS>
__global__ __launch_bounds__(kThreads, 6) void logits_top_rows(const TopArgs a) {
  constexpr int E = Piece<F32>::kElems, ES = F32 ? 4 : 2;
  __shared__ Shared sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x;
  const int V = a.V, k = a.k;
  const char* base = (const char*)a.logits + (size_t)row * (size_t)a.ld * ES;
  const float scale2 = a.rcp_temp * kLog2e;
  const RowPieces rp = row_pieces<F32>(base, V, true);
  const char* vec = base + (size_t)rp.head * ES;
  const int part = PARTS ? blockIdx.y : 0, parts = PARTS ? gridDim.y : 1;
  const int first = PARTS ? (int)((int64_t)rp.pieces * part / parts) : 0;
  const int pieces = PARTS ? (int)((int64_t)rp.pieces * (part + 1) / parts) : rp.pieces;  // where the part ends
  const int single = part == 0 ? rp.single : 0;

  int64_t label = a.labels ? a.labels[row] : (int64_t)-1;
  const bool has_label = label >= 0 && label < (int64_t)V;
  const float z_label = has_label ? load_one(base, (size_t)label, F32) : NAN;
  const int y = has_label ? (int)label : -1;
  const float above_label = next_above(z_label);  // NaN (no label, or its logit is NaN): nothing reaches it

  Stats st{kLowest, 0.f, 0.f};  // the maximum is the wave's
  float lane_max = -INFINITY;
  int better = 0;       // columns of this lane that sort before the label
  int count = 0;        // candidates in the wave's list
  topkey_t least = 0;      // candidates have larger keys: the worst of k that the wave has seen
  float bound = -INFINITY;
  topkey_t* const list = sm.list[wave];

  auto append = [&](float z, int column, bool there) {
    const bool reaches = there && z >= bound;
    if (!__any(reaches)) return;  // by far the most often: the key is formed behind this
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
  auto publish = [&]() {  // the maxima of groups of four lanes
    float m = fmaxf(lane_max, __shfl_xor(lane_max, 1, 64));
    m = fmaxf(m, __shfl_xor(m, 2, 64));
    if ((lane & 3) == 0) sm.group_max[wave * kGroupsPerWave + (lane >> 2)] = m;
  };
  auto raise_wave_max = [&](float z) {  // to the largest z of the wave
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) z = fmaxf(z, __shfl_xor(z, o, 64));
    raise_max(st, max_from(z, scale2));
  };

  int step = 0;
  for (int p0 = first + tid; p0 - tid < pieces; p0 += kThreads * kInFlight, ++step) {
    Piece<F32> pc[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int p = p0 + u * kThreads;
      pc[u].load(vec + (size_t)(p < pieces ? p : pieces - 1) * 16);
    }
    float mx[kInFlight], top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      mx[u] = -INFINITY;
      if (p0 + u * kThreads < pieces) {
#pragma unroll
        for (int i = 0; i < E; ++i) mx[u] = fmaxf(mx[u], pc[u].v[i]);
      }
      top = fmaxf(top, mx[u]);
    }
    lane_max = fmaxf(lane_max, top);
    if (__any(top * scale2 > st.m)) raise_wave_max(top);
    if (k > 0) {
      if ((step & (step + 1)) == 0) {  // steps 0, 1, 3, 7: what has been seen doubles
        publish();
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
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (p0 + u * kThreads < pieces) {
#pragma unroll
        for (int i = 0; i < E; ++i) absorb<true>(st, pc[u].v[i], scale2);
      }
    }
    if (__any(top >= z_label)) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int p = p0 + u * kThreads, c0 = rp.head + p * E;
        if (p < pieces) {
          // columns in front of the label's precede it with an equal logit already
          const float reach = c0 + E <= y ? z_label : above_label;
#pragma unroll
          for (int i = 0; i < E; ++i) better += pc[u].v[i] >= reach ? 1 : 0;
          if (c0 < y && y < c0 + E) {
#pragma unroll
            for (int i = 0; i < E; ++i) better += c0 + i < y && pc[u].v[i] == z_label ? 1 : 0;
          }
        }
      }
    }
    if (k > 0 && __any(top >= bound)) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int p = p0 + u * kThreads;
        if (!__any(mx[u] >= bound)) continue;
#pragma unroll
        for (int i = 0; i < E; ++i) append(pc[u].v[i], rp.head + p * E + i, p < pieces);
      }
    }
  }
  for (int i0 = 0; i0 < single; i0 += kThreads) {
    const int i = i0 + tid;
    const bool there = i < single;
    const int c = single_column(rp, E, there ? i : 0);
    const float z = load_one(base, (size_t)c, F32);
    raise_wave_max(there ? z : -INFINITY);
    if (there) {
      lane_max = fmaxf(lane_max, z);
      absorb<true>(st, z, scale2);
      better += z >= above_label || (z == z_label && c < y) ? 1 : 0;
    }
    if (k > 0) append(z, c, there);
  }

#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) better += __shfl_xor(better, o, 64);
  if (count > k && k > 0 && __builtin_amdgcn_readfirstlane(count) > kThreads / kWaves) {  // so that all fit behind each other
    (void)keep_best(list, count, k);
    count = k;
  }
  if (lane == 0) sm.count[wave] = count, sm.better[wave] = better;
  st = block_merge<kWaves>(st, sm.stats);  // a barrier: the lists and counts of all waves stand
  const bool far = is_far(st) && __syncthreads_or(lane_max > -INFINITY ? 1 : 0) != 0;  // else it is empty, or its logits are NaN and -inf
  if (far) {
    if (!PARTS) st = far_row<F32, kWaves>(base, V, scale2, (float*)sm.stats);
    else if (st.m == kLowest) st.m = kFarPart;
  }
  const RowResult result(st, a.rcp_temp, far);
  int total = 0, before = 0, mine_at = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) mine_at = total;
    total += sm.count[w], before += sm.better[w];
  }
  if (tid == 0) {
    if (PARTS) a.part[row * parts + part] = Part{st, before, total < k ? total : k};
    else result.write(a, row, st, has_label, z_label, before);
  }
  if (k == 0) return;
  for (int e = lane; e < count; e += 64) sm.all[mine_at + e] = list[e];
  __syncthreads();
  // The place of a candidate is the number of better ones.
  for (int e = tid; e < total; e += kThreads) {
    const topkey_t mine = sm.all[e];
    const int place = place_among(sm.all, total, mine);
    if (place < k) {
      if (PARTS) {
        a.keys[(row * parts + part) * (int64_t)k + place] = mine;
      } else {
        a.top_ids[row * (int64_t)k + place] = key_column(mine);
        a.top_logprobs[row * (int64_t)k + place] = result.logprob_of(value_of_bits(key_bits(mine)));
      }
    }
  }
  if (!PARTS && total < k && wave == 0) fill_with_nan<F32>(V, k, a.top_ids + row * (int64_t)k, a.top_logprobs + row * (int64_t)k, base, total);
}

// Joins the parts of a row.  The k best of the parts' first ceil(k / parts) keys give a bound that few keys of a row reach; those find their
// places.
constexpr int kJoinThreads = 256;
template <bool F32>
__global__ __launch_bounds__(kJoinThreads) void logits_top_join(const TopArgs a, int parts) {
  __shared__ topkey_t keys[kMaxJoin];
  __shared__ topkey_t firsts[kMaxTop + kMaxParts];
  __shared__ topkey_t bound;
  __shared__ int have[kMaxParts], kept;
  __shared__ float far_sums[2 * kJoinThreads / 64];
  const int tid = threadIdx.x, k = a.k;
  const int64_t row = blockIdx.x;
  const char* base = (const char*)a.logits + (size_t)row * (size_t)a.ld * (F32 ? 4 : 2);
  const int each = k > 0 ? (k + parts - 1) / parts : 0;
  // Every wave joins the statistics for itself, a part a lane.
  const int lane = tid & 63;
  Part q{{kLowest, 0.f, 0.f}, 0, 0};
  if (lane < parts) q = a.part[row * parts + lane];
  Stats st = q.st;
  int before = q.better, found = q.keys;
  if (tid < kMaxParts) have[tid] = q.keys;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    Stats other;
    other.m = __shfl_xor(st.m, o, 64), other.s = __shfl_xor(st.s, o, 64), other.e = __shfl_xor(st.e, o, 64);
    merge(st, other);
    before += __shfl_xor(before, o, 64), found += __shfl_xor(found, o, 64);
  }
  // Lane 0's for all: the lanes' sums differ in their last bits, and which lane writes an alternative below is not fixed.
  auto of_lane_0 = [](float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); };
  st = Stats{of_lane_0(st.m), of_lane_0(st.s), of_lane_0(st.e)};
  if (tid == 0) bound = 0, kept = 0;
  __syncthreads();
  for (int e = tid; e < parts * each; e += kJoinThreads) {
    const int p = e / each, i = e - p * each;
    firsts[e] = i < have[p] ? a.keys[(row * parts + p) * (int64_t)k + i] : 0;
  }
  const bool far = is_far(st) && !(st.m == kLowest && st.s == 0.f);
  if (far) st = far_row<F32, kJoinThreads / 64>(base, a.V, a.rcp_temp * kLog2e, far_sums);
  const RowResult result(st, a.rcp_temp, far);
  if (tid == 0) {
    const int64_t label = a.labels ? a.labels[row] : (int64_t)-1;
    const bool has_label = label >= 0 && label < (int64_t)a.V;
    result.write(a, row, st, has_label, has_label ? load_one(base, (size_t)label, F32) : NAN, before);
  }
  if (k == 0) return;
  __syncthreads();
  for (int e = tid; e < parts * each; e += kJoinThreads) {
    const topkey_t mine = firsts[e];
    if (mine != 0 && place_among(firsts, parts * each, mine) == k - 1) bound = mine;  // at most one: keys differ
  }
  __syncthreads();
  const topkey_t least = bound;  // 0 where the firsts have fewer than k keys: everything is kept
  for (int e = tid; e < parts * k; e += kJoinThreads) {
    const int p = e / k, i = e - p * k;
    const topkey_t key = i < have[p] ? a.keys[(row * parts + p) * (int64_t)k + i] : 0;
    if (key != 0 && key >= least) keys[atomicAdd(&kept, 1)] = key;  // in any order: places depend on the keys alone
  }
  __syncthreads();
  const int n = kept;
  for (int e = tid; e < n; e += kJoinThreads) {
    const topkey_t mine = keys[e];
    const int place = place_among(keys, n, mine);
    if (place < k) {
      a.top_ids[row * (int64_t)k + place] = key_column(mine);
      a.top_logprobs[row * (int64_t)k + place] = result.logprob_of(value_of_bits(key_bits(mine)));
    }
  }
  if (found < k && tid < 64) fill_with_nan<F32>(a.V, k, a.top_ids + row * (int64_t)k, a.top_logprobs + row * (int64_t)k, base, found);
}

// The gradient.  As logits_bwd_rows (logits_kernels.hip), with sum_j h_j in the coefficient of p, and the k + 1 columns that have a term of their
// own written once more behind a barrier, from logits read in front of the pass (dlogits may be the logits themselves).
struct TopBwdArgs {
  const void* logits;
  int64_t ld;
  const int64_t* labels;
  int V, k;
  float rcp_temp;
  int vector_ok;
  const float *row_lse, *row_pz, *dlogprobs, *dentropy;
  const int64_t* top_ids;
  const float* dtop;
  void* dlogits;
  int64_t ldd;
};

// From this size on the fp32 log-sum-exp costs p more than 2^-12 of its value (the rounding of lse, and of lse in base 2): such a row's statistics are
// formed anew, and its gradient from differences of logits.  No model's row, but a row that a mask of finite values has all of.
constexpr float kFarLse = 4096.f;

template <bool F32, bool ENTGRAD, bool NONTEMPORAL>
__global__ __launch_bounds__(kBwdThreads) void logits_top_bwd_rows(const TopBwdArgs a) {
  constexpr int E = Piece<F32>::kElems, ES = F32 ? 4 : 2;
  __shared__ float h_sum[kBwdThreads / 64], far_sums[2 * kBwdThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = (int64_t)(gridDim.x - 1 - blockIdx.x);  // the rows that the forward read last first
  const int V = a.V, k = a.dtop ? a.k : 0;
  const char* src = (const char*)a.logits + (size_t)row * (size_t)a.ld * ES;
  char* dst = (char*)a.dlogits + (size_t)row * (size_t)a.ldd * ES;
  int64_t y = a.labels ? a.labels[row] : (int64_t)-1;
  if (y < 0 || y >= (int64_t)V) y = -1;
  const float g = a.dlogprobs && y >= 0 ? a.dlogprobs[row] : 0.f;
  const float q = ENTGRAD ? a.dentropy[row] : 0.f;
  const float lse = a.row_lse[row], lse2 = lse * kLog2e;
  const float pz = ENTGRAD ? a.row_pz[row] : 0.f;
  const float scale2 = a.rcp_temp * kLog2e;
  // Thread j < k has the gradient of alternative j, thread k that of the label.  Ids that lie outside the row, which the forward does not
  // give, have no term.
  int64_t own = -1;
  float own_grad = 0.f;
  if (tid < k) {
    own = a.top_ids[row * (int64_t)k + tid];
    if (own < 0 || own >= (int64_t)V) own = -1;
    own_grad = own >= 0 ? a.dtop[row * (int64_t)k + tid] : 0.f;
  } else if (tid == k && y >= 0) {
    own = y, own_grad = g;
  }
  float s = tid <= k ? own_grad : 0.f;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) h_sum[wave] = s;
  __syncthreads();
  float all = 0.f;
  for (int w = 0; w * 64 <= k; ++w) all += h_sum[w];  // waves behind the k + 1 threads hold nothing
  // A column may be both an alternative and the label, or be listed twice: the first thread that has it takes all of its terms.
  float own_z = 0.f;
  bool writes = own >= 0;
  if (own >= 0) {
    own_z = load_one(src, (size_t)own, F32);
    for (int j = 0; j < k; ++j) {
      const int64_t id = a.top_ids[row * (int64_t)k + j];
      if (id != own || j == tid) continue;
      if (j < tid) writes = false;
      else own_grad += a.dtop[row * (int64_t)k + j];
    }
    if (tid < k && own == y) own_grad += g;
  }
  // dz = p * (c0 + c1 * z) [+ the column's own gradient / temperature],  c0 = -(g + sum h - q pz) / temperature,  c1 = -q / temperature^2
  const float c0 = -(all - q * pz) * a.rcp_temp, c1 = -q * a.rcp_temp * a.rcp_temp;
  const bool empty = lse == -INFINITY;  // no logit above -inf: no gradient
  bool any = tid <= k && own_grad != 0.f;
  const bool zero_row = empty || (__syncthreads_or((any || all != 0.f || q != 0.f) ? 1 : 0) == 0);
  if (!zero_row && fabsf(lse) >= kFarLse) {
    const Stats st = far_row<F32, kBwdThreads / 64>(src, V, scale2, far_sums);
    const float from = far_origin(st.m), rcp_s = st.s == 0.f ? 0.f : 1.f / st.s, mean = st.s == 0.f ? 0.f : st.e / st.s;
    auto dz = [&](float z) {
      const float t = (z - from) * scale2, p = __builtin_amdgcn_exp2f(t) * rcp_s;
      return p * (-all - q * ((fmaxf(t, kMostNegativeFactor) - mean) * kLn2)) * a.rcp_temp;
    };
    auto write = [&](int64_t c, float d) {
      if (F32) ((float*)dst)[c] = d;
      else ((uint16_t*)dst)[c] = bf16_bits(d);
    };
    for (int c = tid; c < V; c += kBwdThreads) write(c, dz(load_one(src, (size_t)c, F32)));
    __syncthreads();
    if (writes && st.s != 0.f) write(own, fmaf(own_grad, a.rcp_temp, dz(own_z)));
    return;
  }
  auto dz = [&](float z) {
    const float p = __builtin_amdgcn_exp2f(fmaf(z, scale2, -lse2));
    return ENTGRAD ? p * fmaf(c1, fmaxf(z, kMostNegativeFactor), c0) : p * c0;
  };
  const RowPieces rp = row_pieces<F32>(src, V, a.vector_ok != 0);
  const char* vsrc = src + (size_t)rp.head * ES;
  char* vdst = dst + (size_t)rp.head * ES;
  for (int p0 = tid; p0 < rp.pieces; p0 += kBwdThreads * kInFlight) {
    Piece<F32> pc[kInFlight];
    if (!zero_row) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int p = p0 + u * kBwdThreads;
        pc[u].load(vsrc + (size_t)(p < rp.pieces ? p : p0) * 16);
      }
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int p = p0 + u * kBwdThreads;
      if (p >= rp.pieces) continue;
      float d[E];
#pragma unroll
      for (int i = 0; i < E; ++i) d[i] = zero_row ? 0.f : dz(pc[u].v[i]);
      uint4 out;
      if (F32) {
        out = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3]));
      } else {
        typedef __attribute__((ext_vector_type(4))) float f32x4;
        typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
        const f32x4 lo4 = {d[0], d[1], d[2], d[3]}, hi4 = {d[4 % E], d[5 % E], d[6 % E], d[7 % E]};
        const bf16x4 lo = __builtin_convertvector(lo4, bf16x4), hi = __builtin_convertvector(hi4, bf16x4);
        const uint2 x = *(const uint2*)&lo, z = *(const uint2*)&hi;
        out = make_uint4(x.x, x.y, z.x, z.y);
      }
      if constexpr (NONTEMPORAL) __builtin_nontemporal_store(*(const u32x4*)&out, (u32x4*)(vdst + (size_t)p * 16));
      else *(uint4*)(vdst + (size_t)p * 16) = out;
    }
  }
  for (int i = tid; i < rp.single; i += kBwdThreads) {
    const int c = single_column(rp, E, i);
    const float d = zero_row ? 0.f : dz(load_one(src, (size_t)c, F32));
    if (F32) ((float*)dst)[c] = d;
    else ((uint16_t*)dst)[c] = bf16_bits(d);
  }
  if (zero_row) return;
  __syncthreads();  // the pass over the row is done: what is written here comes behind it
  if (writes) {
    const float d = fmaf(own_grad, a.rcp_temp, dz(own_z));
    if (F32) ((float*)dst)[own] = d;
    else ((uint16_t*)dst)[own] = bf16_bits(d);
  }
}

int check_top(int64_t V, int64_t k) {
  return k < 0 || k > V || k > kMaxTop ? SKYRL_LMHEAD_ERR_SHAPE : SKYRL_LMHEAD_OK;
}

// Parts of a row: so many that 512 workgroups share the logits, of at least 8192 logits each, and none for rows so short that the second launch costs
// what the parts save.  us in a graph, both launches, k = 20, one workgroup a row / parts for 256, 512 and 1024 workgroups:
//             8 rows                  64 rows                      128 rows                     255 rows
//   bf16 32001  13.2 / 14.4           13.6 / 15.0                  14.4 / 16.3, 17.3, 17.2      15.4 / -, 19.3, 20.0
//        40000  14.3 / 13.7           15.1 / 14.6, 14.4, 14.3      16.0 / 18.0, 16.9, 16.9      17.0 / -, 21.3, 23.3
//        49152  15.7 / 13.5           16.5 / 14.6, 15.6, 15.6      17.8 / 19.1, 17.8, 18.5      18.3 / -, 22.2, 24.3
//        80000  19.9 / 13.9           22.1 / 17.9, 17.0, 18.6      22.3 / 22.1, 21.0, 23.1      23.4 / -, 26.1, 29.6
//       151936  29.9 / 14.5           32.3 / 21.8, 21.2, 23.6      33.1 / 27.9, 25.5, 29.1      36.6 / -, 35.1, 38.2
//   fp32 32001  15.7 / 16.3           17.0 / 17.7                  17.9 / 19.3, 19.8, 20.0      19.0 / -, 21.6, 22.9
//        49152  18.6 / 13.9           20.4 / 18.2, 17.3, 17.2      21.0 / 21.3, 20.2, 19.7      22.2 / -, 24.6, 28.2
//       151936  36.2 / 15.7           41.5 / 25.2, 23.3, 27.9      45.2 / 36.3, 30.2, 33.9      49.3 / -, 45.6, 50.1
// What one limit for all costs: two parts a row (171 to 256 rows) lose 2 to 4 us below some 100000 bf16 or 70000 fp32 columns.
int top_parts(int64_t T, int64_t V, int64_t k) {
  int64_t n = V < 6 * 8192 ? 1 : 512 / T;
  if (n > V / 8192) n = V / 8192;
  if (n > kMaxParts) n = kMaxParts;
  if (k > 0 && n > kMaxJoin / k) n = kMaxJoin / k;
  return n < 1 ? 1 : (int)n;
}

}  // namespace

extern "C" {

size_t skyrl_logits_top_workspace_bytes(int64_t T, int64_t V, int64_t k) {
  if (T < 1 || V < 1 || T >= kMaxRows || V >= ((int64_t)1 << 31) || check_top(V, k)) return 0;
  const size_t parts = (size_t)top_parts(T, V, k);
  return parts == 1 ? 0 : (size_t)T * parts * (sizeof(Part) + (size_t)k * sizeof(topkey_t)) + 8;
}

int skyrl_logits_top_fwd(const void* logits, int logits_dtype, int64_t ld_logits, const int64_t* labels, int64_t T, int64_t V, int64_t k,
                         float rcp_temperature, float* logprobs, float* entropy, float* row_lse, float* row_pz, int64_t* ranks,
                         float* top_logprobs, int64_t* top_ids, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_logits(logits, logits_dtype, ld_logits, T, V, rcp_temperature);
  if (st) return st;
  if ((st = check_top(V, k))) return st;
  if ((logprobs || ranks) && !labels) return SKYRL_LMHEAD_ERR_NULL;
  if (k > 0 && (!top_logprobs || !top_ids)) return SKYRL_LMHEAD_ERR_NULL;
  if (k == 0 && !logprobs && !entropy && !row_lse && !row_pz && !ranks) return SKYRL_LMHEAD_ERR_NULL;
  if (((uintptr_t)labels | (uintptr_t)ranks | (uintptr_t)top_ids | (uintptr_t)workspace) & 7u) return SKYRL_LMHEAD_ERR_ALIGN;
  const size_t need = skyrl_logits_top_workspace_bytes(T, V, k);
  if (need > 0 && (!workspace || workspace_bytes < need)) return SKYRL_LMHEAD_ERR_WORKSPACE;
  const int parts = top_parts(T, V, k);
  const bool f32 = logits_dtype == SKYRL_LOGITS_F32;
  topkey_t* const keys = (topkey_t*)workspace;
  const TopArgs a{logits, ld_logits, labels, (int)V, (int)k, rcp_temperature, logprobs, entropy, row_lse, row_pz, ranks, top_logprobs, top_ids,
                  (Part*)(keys + (size_t)T * (size_t)parts * (size_t)k), keys};
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)T, (unsigned)parts), block(kThreads);
  if (parts == 1) {
    hipLaunchKernelGGL((f32 ? logits_top_rows<true, false> : logits_top_rows<false, false>), grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL((f32 ? logits_top_rows<true, true> : logits_top_rows<false, true>), grid, block, 0, s, a);
    hipLaunchKernelGGL(f32 ? logits_top_join<true> : logits_top_join<false>, dim3((unsigned)T), dim3(kJoinThreads), 0, s, a, parts);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SKYRL_LMHEAD_OK : (int)e;
}

int skyrl_logits_top_bwd(const void* logits, int logits_dtype, int64_t ld_logits, const int64_t* labels, const float* row_lse,
                         const float* row_pz, const float* dlogprobs, const float* dentropy, const int64_t* top_ids, const float* dtop,
                         int64_t T, int64_t V, int64_t k, float rcp_temperature, void* dlogits, int64_t ld_dlogits, void* stream) {
  int st = check_logits(logits, logits_dtype, ld_logits, T, V, rcp_temperature);
  if (st) return st;
  if ((st = check_top(V, k))) return st;
  if (!row_lse || !dlogits || (!dlogprobs && !dentropy && !dtop) || (dlogprobs && !labels) || (dentropy && !row_pz) || (dtop && !top_ids))
    return SKYRL_LMHEAD_ERR_NULL;
  if (ld_dlogits < V || ld_dlogits >= ((int64_t)1 << 40)) return SKYRL_LMHEAD_ERR_SHAPE;
  const bool f32 = logits_dtype == SKYRL_LOGITS_F32;
  if (((uintptr_t)dlogits & (f32 ? 3u : 1u)) || (((uintptr_t)labels | (uintptr_t)top_ids) & 7u)) return SKYRL_LMHEAD_ERR_ALIGN;
  if (overlaps_otherwise(logits, ld_logits, dlogits, ld_dlogits, T, V, f32)) return SKYRL_LMHEAD_ERR_ARG;
  const int vec = same_row_offsets(logits, ld_logits, dlogits, ld_dlogits, f32) ? 1 : 0;
  const TopBwdArgs a{logits, ld_logits, labels, (int)V, (int)k, rcp_temperature, vec, row_lse, row_pz, dlogprobs, dentropy, top_ids, dtop, dlogits,
                     ld_dlogits};
  const bool entgrad = dentropy != nullptr, beyond = T * V * (f32 ? 4 : 2) > kCacheBytes;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)T), dim3(kBwdThreads), 0, (hipStream_t)stream, a); };
  if (f32 && entgrad) launch(beyond ? logits_top_bwd_rows<true, true, true> : logits_top_bwd_rows<true, true, false>);
  else if (f32) launch(beyond ? logits_top_bwd_rows<true, false, true> : logits_top_bwd_rows<true, false, false>);
  else if (entgrad) launch(beyond ? logits_top_bwd_rows<false, true, true> : logits_top_bwd_rows<false, true, false>);
  else launch(beyond ? logits_top_bwd_rows<false, false, true> : logits_top_bwd_rows<false, false, false>);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SKYRL_LMHEAD_OK : (int)e;
}

}  // extern "C"
