// Rows of an embedding table by token id, scaled, and the gradient of the table.
//
//   out[t] = scale E[id_t]          zeros where id_t lies outside [0, V)
//   dE[v]  = scale sum_{t: id_t = v} dout[t]      added up in fp32 in an order that the ids fix, rounded once; no row where v is the padding id
//
// Gradient.  Tokens are sorted by id, ties by position, so that the tokens of a row lie side by side.
//   embedding_rank   sorts blocks of kSortBlock tokens by counting: a token's place is the number of keys that sort before its own, two
//                    instructions a pair.  No passes, no atomics, one launch.
//   embedding_merge  (more than one block) makes one block of kWay: a token's place in it is its place in its own block plus, by bisection, the keys
//                    of each other that sort before its own.
//   embedding_rows   the sorted tokens in windows of kWindow: a wave loads its window's rows of dout, 1 KiB of each, all at once and adds
//                    up those of one id.  A sum that no other window adds to is a result; the others are kept as fp32 partial sums.  So every row
//                    of dout is read once, by as many waves whatever the ids are: one id for all tokens or another one for each.  For a dense
//                    result other workgroups of the same launch write the rows that no token names as zeros.
//   embedding_join   adds the partial sums of an id whose tokens lie in several windows.
// Bound by HBM: the table's gradient is written (almost all of it zeros), dout read.  16384 tokens, H=3584, V=152064, bf16: lookup 46 us (5.1 TB/s),
// rank 12, merge 7, rows 210 (5.8 TB/s), join 11; added into an fp32 buffer 88 us for all launches.  Few tokens are bound by the zeros: 512 of H=896,
// V=151936 46 us (5.9 TB/s); added, by latency: 16 of H=896 12 us.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <cmath>

#include "../../include/skyrl_lmhead.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kSortBlock = 4096;  // 2048 and 4096 the same (250 us for the whole gradient there), 8192 260
constexpr int kRankTokens = 64, kRankWaves = 8;  // a lane per token, a wave per eighth of the block's keys
// Rows of dout that a wave has in flight.  Ids as in text, one id, all ids alike: 255, 347, 247 us with 8, 250, 297, 267 with 16, 268, 280, 279 with 32.
constexpr int kWindow = 16;
// Sorted blocks that become one.  2^20 tokens of H=896: 1071 us with 8, 1141 with 16, 2375 with all blocks in one launch.
constexpr int kWay = 8;
constexpr int kRowThreads = 256, kRowWaves = kRowThreads / 64;
constexpr int kJoinWaves = 8;
// Of the result that a workgroup looks after where it writes zeros.  512 tokens of H=896 and 2047 of 1023 fp32 columns: 59 and 34 us with 16 KiB, 46 and
// 34 with 64, 52 and 48 with 256.
constexpr int kZeroBytes = 65536;

// Sixteen bytes of a row from element e0 on.  Rows of odd sizes begin anywhere: loads and stores of unaligned 16 bytes.  The last piece of a row
// ends with it and so may repeat elements of the one before; a row shorter than a piece goes element by element.
template <bool F32>
struct Row16 {
  static constexpr int E = F32 ? 4 : 8, ES = F32 ? 4 : 2;
  struct __attribute__((packed, aligned(ES))) Piece {
    u32x4 v;
  };
  static __host__ __device__ int pieces(int H) { return (H + E - 1) / E; }
  static __device__ __forceinline__ int first(int piece, int H) { return H < E ? 0 : (piece * E < H - E ? piece * E : H - E); }
  static __device__ __forceinline__ u32x4 load(const char* row, int e0, int H) {
    if (H >= E) return ((const Piece*)(row + (size_t)e0 * ES))->v;
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (i >= H) break;
      if constexpr (F32) w[i] = ((const uint32_t*)row)[i];
      else w[i / 2] |= (uint32_t)((const uint16_t*)row)[i] << (16 * (i % 2));
    }
    return w;
  }
  static __device__ __forceinline__ void store(char* row, int e0, int H, const u32x4& w) {
    if (H >= E) {
      ((Piece*)(row + (size_t)e0 * ES))->v = w;
      return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (i >= H) break;
      if constexpr (F32) ((uint32_t*)row)[i] = w[i];
      else ((uint16_t*)row)[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
    }
  }
  static __device__ __forceinline__ float at(const u32x4& w, int i) {
    if constexpr (F32) return __uint_as_float(w[i]);
    else return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  // x * scale, rounded to nearest, ties to even
  static __device__ __forceinline__ u32x4 scaled(const float (&x)[E], float scale) {
    u32x4 w;
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i] * scale);
    } else {
      typedef __attribute__((ext_vector_type(2))) float f32x2;
      typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 pair = {x[2 * i] * scale, x[2 * i + 1] * scale};
        const bf16x2 b = __builtin_convertvector(pair, bf16x2);
        w[i] = *(const uint32_t*)&b;
      }
    }
    return w;
  }
};

// A wave per token and 256 pieces of its row.
template <bool F32>
__global__ __launch_bounds__(kRowThreads) void embedding_fwd(const char* __restrict__ table, int64_t ld, const int64_t* __restrict__ ids, int64_t T, int H,
                                                             int64_t V, float scale, char* __restrict__ out) {
  typedef Row16<F32> R;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = (int64_t)blockIdx.x * kRowWaves + wave;
  if (t >= T) return;
  const int64_t id = ids[t];
  const bool has = id >= 0 && id < V;
  const char* row = table + (size_t)(has ? id : 0) * (size_t)ld * R::ES;
  char* to = out + (size_t)t * (size_t)H * R::ES;
  const int pieces = R::pieces(H), p0 = blockIdx.y * 256 + lane;
  u32x4 w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    w[u] = u32x4{0, 0, 0, 0};
    if (has && p0 + u * 64 < pieces) w[u] = R::load(row, R::first(p0 + u * 64, H), H);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (p0 + u * 64 >= pieces) continue;
    float x[R::E];
#pragma unroll
    for (int i = 0; i < R::E; ++i) x[i] = R::at(w[u], i);
    R::store(to, R::first(p0 + u * 64, H), H, has ? R::scaled(x, scale) : w[u]);
  }
}

// The key of a token: its id, or V, which sorts behind all, where it takes no part.
__device__ __forceinline__ int key_of(int64_t id, int64_t V, int64_t padding) { return id >= 0 && id < V && id != padding ? (int)id : (int)V; }

__global__ __launch_bounds__(64 * kRankWaves) void embedding_rank(const int64_t* __restrict__ ids, int64_t T, int64_t V, int64_t padding,
                                                                  int* __restrict__ keys, int* __restrict__ tokens) {
  __shared__ __attribute__((aligned(16))) int key[kSortBlock];
  __shared__ int part[kRankWaves][kRankTokens];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kGroups = kSortBlock / kRankTokens;  // workgroups of a block
  const int64_t first = (int64_t)(blockIdx.x / kGroups) * kSortBlock;
  const int n = (int)(T - first < kSortBlock ? T - first : kSortBlock);
  const int t0 = (int)(blockIdx.x % kGroups) * kRankTokens;
  if (t0 >= n) return;
  const int filled = (n + 4 * kRankWaves - 1) / (4 * kRankWaves) * (4 * kRankWaves);
  for (int i = threadIdx.x; i < filled; i += 64 * kRankWaves) key[i] = i < n ? key_of(ids[first + i], V, padding) : 0x7fffffff;
  __syncthreads();
  const int mine = key[t0 + lane < n ? t0 + lane : n - 1];
  // Keys in front of the workgroup's tokens precede one of theirs that is equal, keys behind them do not; among them the position decides.
  const int each = filled / kRankWaves;
  const int from = wave * each, to = from + each;
  int before = 0;
  auto count = [&](int a, int b, auto sorts_before) {
#pragma unroll 8
    for (int i = a; i < b; i += 4) {
      const int4 k = *(const int4*)(key + i);
      before += sorts_before(k.x, i) + sorts_before(k.y, i + 1) + sorts_before(k.z, i + 2) + sorts_before(k.w, i + 3);
    }
  };
  auto clamp = [&](int x) { return x < from ? from : (x > to ? to : x); };
  const int a = clamp(t0), b = clamp(t0 + kRankTokens);
  count(from, a, [&](int k, int) { return k <= mine ? 1 : 0; });
  count(a, b, [&](int k, int i) { return k < mine || (k == mine && i < t0 + lane) ? 1 : 0; });
  count(b, to, [&](int k, int) { return k < mine ? 1 : 0; });
  part[wave][lane] = before;
  __syncthreads();
  if (wave != 0 || t0 + lane >= n) return;
  int place = 0;
#pragma unroll
  for (int w = 0; w < kRankWaves; ++w) place += part[w][lane];
  keys[first + place] = mine;
  tokens[first + place] = (int)(first + t0 + lane);
}

// How many of the first n sorted keys are below k (or, with `equal`, not above it).
__device__ __forceinline__ int keys_before(const int* __restrict__ keys, int n, int k, bool equal) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1, x = keys[mid];
    const bool before = equal ? x <= k : x < k;
    lo = before ? mid + 1 : lo;
    hi = before ? hi : mid;
  }
  return lo;
}

// Blocks of `block` tokens, the last one shorter.  All blocks in one launch would be as many bisections a token as there are blocks.
__global__ __launch_bounds__(256) void embedding_merge(const int* __restrict__ block_keys, const int* __restrict__ block_tokens, int T, int block,
                                                       int* __restrict__ keys, int* __restrict__ tokens) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (i >= T) return;
  const int own = i / block, first = own / kWay * kWay, all = (T + block - 1) / block, blocks = all < first + kWay ? all : first + kWay;
  const int k = block_keys[i];
  int place = first * block + (i - own * block);
  // Four blocks at a time, whose bisections do not wait for each other.
  for (int b0 = first; b0 < blocks; b0 += 4) {
    const int* base[4];
    int lo[4], hi[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int b = b0 + u < blocks ? b0 + u : own, left = T - b * block;
      base[u] = block_keys + b * block;
      lo[u] = 0;
      hi[u] = b == own ? 0 : (left < block ? left : block);
    }
    for (int step = 0; (block >> step) > 0; ++step) {  // a block halves to nothing in as many steps
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool open = lo[u] < hi[u];
        const int mid = open ? (lo[u] + hi[u]) >> 1 : 0;
        const int x = base[u][mid];
        const bool before = b0 + u < own ? x <= k : x < k;
        if (open && before) lo[u] = mid + 1;
        if (open && !before) hi[u] = mid;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) place += lo[u];
  }
  keys[place] = k;
  tokens[place] = block_tokens[i];
}

struct RowArgs {
  const char* dout;
  int64_t ld;
  int64_t T, V;
  int H;
  float scale;
  const int* keys;
  const int* tokens;
  float* partial;  // [windows, 2, pieces of a row * E]: of the id that the window begins with and one before has, of the one that it ends with
  char* dtable;    // [V, H]
  int slices;      // of 64 pieces, of a row
  int64_t units;   // windows * slices
  int zero_rows;   // rows of the result a workgroup that writes zeros looks after
};

// ADD: into an fp32 result.  Elements e0 .. e0 + E - 1 of its row, which a piece ends up with.
template <int E>
__device__ __forceinline__ void load_base(const RowArgs& a, int id, int e0, float (&base)[E]) {
  struct __attribute__((packed, aligned(4))) Four {
    f32x4 v;
  };
  const float* const row = (const float*)a.dtable + (size_t)id * (size_t)a.H;
  if (a.H >= E) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const f32x4 x = ((const Four*)(row + e0 + i))->v;
      base[i] = x[0], base[i + 1] = x[1], base[i + 2] = x[2], base[i + 3] = x[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) base[i] = i < a.H ? row[i] : 0.f;
  }
}

// Each element is written by the one piece that begins at or before it and is the last to do so (pieces may overlap at a row's end).  base: what ADD adds to.
template <bool F32, bool ADD>
__device__ __forceinline__ void finish(const RowArgs& a, int id, int piece, const float (&sum)[Row16<F32>::E], const float (&base)[Row16<F32>::E]) {
  typedef Row16<F32> R;
  const int e0 = R::first(piece, a.H);
  if constexpr (ADD) {
    struct __attribute__((packed, aligned(4))) Four {
      f32x4 v;
    };
    float* const row = (float*)a.dtable + (size_t)id * (size_t)a.H;
    float x[R::E];
#pragma unroll
    for (int i = 0; i < R::E; ++i) x[i] = fmaf(sum[i], a.scale, base[i]);
    if (a.H >= R::E && e0 == piece * R::E) {
#pragma unroll
      for (int i = 0; i < R::E; i += 4) ((Four*)(row + e0 + i))->v = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < R::E; ++i)
        if (e0 + i >= piece * R::E && e0 + i < a.H) row[e0 + i] = x[i];
    }
  } else {
    R::store(a.dtable + (size_t)id * (size_t)a.H * R::ES, e0, a.H, R::scaled(sum, a.scale));
  }
}

template <bool F32, bool ADD>
__global__ __launch_bounds__(kRowThreads) void embedding_rows(const RowArgs a) {
  typedef Row16<F32> R;
  constexpr int E = R::E;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t sum_groups = (a.units + kRowWaves - 1) / kRowWaves;
  const int pieces = R::pieces(a.H);
  if (!ADD && (int64_t)blockIdx.x >= sum_groups) {
    __shared__ uint8_t named[256];
    const int64_t v0 = ((int64_t)blockIdx.x - sum_groups) * a.zero_rows;
    const int rows = (int)(a.V - v0 < a.zero_rows ? a.V - v0 : a.zero_rows);
    if ((int)threadIdx.x < rows) {
      const int v = (int)v0 + threadIdx.x, at = keys_before(a.keys, (int)a.T, v, false);
      named[threadIdx.x] = at < (int)a.T && a.keys[at] == v ? 1 : 0;
    }
    __syncthreads();
    // The rows as one run of memory in whole 16-byte pieces from the first row on (groups of rows begin on one, if the table does), so that rows of any
    // size keep all lanes at work.
    char* base = a.dtable + (size_t)v0 * (size_t)a.H * R::ES;
    const uint32_t H = (uint32_t)a.H, all = (uint32_t)rows * H;
    for (uint32_t e0 = threadIdx.x * E; e0 < all; e0 += kRowThreads * E) {
      const uint32_t row = e0 / H, left = (row + 1) * H - e0;  // elements to the row's end
      char* to = base + (size_t)e0 * R::ES;
      if (left >= E ? !named[row] : left + H >= E && e0 + E <= all && !named[row] && !named[row + 1]) {
        ((typename R::Piece*)to)->v = u32x4{0, 0, 0, 0};
        continue;
      }
      if (left >= E) continue;
#pragma unroll
      for (uint32_t i = 0; i < E; ++i) {
        if (e0 + i >= all || named[(e0 + i) / H]) continue;
        if constexpr (F32) ((uint32_t*)to)[i] = 0;
        else ((uint16_t*)to)[i] = 0;
      }
    }
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * kRowWaves + wave;
  if (unit >= a.units) return;
  const int64_t window = unit / a.slices;
  const int piece = (int)(unit - window * a.slices) * 64 + lane;
  const int64_t at = window * kWindow;
  const int n = (int)(a.T - at < kWindow ? a.T - at : kWindow);
  // Lane j + 1 has the key of the window's token j; lanes 0 and kWindow + 1 those of the tokens beside it.
  const int64_t near = at - 1 + lane;
  const int key = near >= 0 && near < a.T && lane < kWindow + 2 ? a.keys[near] : -1;
  const int token = lane < n ? a.tokens[at + lane] : 0;
  const int V = (int)a.V;
  if (__builtin_amdgcn_readlane(key, 1) == V) return;  // this and all that follow take no part
  const bool there = piece < pieces;
  const int e0 = R::first(there ? piece : 0, a.H);
  u32x4 w[kWindow];
#pragma unroll
  for (int j = 0; j < kWindow; ++j) w[j] = R::load(a.dout + (size_t)__builtin_amdgcn_readlane(token, j) * (size_t)a.ld * R::ES, e0, a.H);
  // What results are added to comes in with the rows: read one behind the other, the sixteen ids of one window took 28 us instead of 9, and 16384 tokens of H=3584
  // 141 instead of 88 for all launches.
  float base[ADD ? kWindow : 1][E];
  if constexpr (ADD) {
#pragma unroll
    for (int j = 1; j <= kWindow; ++j) {
      const int id = __builtin_amdgcn_readlane(key, j);
      if (j <= n && id != V && (j == n || __builtin_amdgcn_readlane(key, j + 1) != id)) load_base<E>(a, id, e0, base[j - 1]);
    }
  }
  float sum[E];
#pragma unroll
  for (int i = 0; i < E; ++i) sum[i] = R::at(w[0], i);
  int start = 0;
#pragma unroll
  for (int j = 1; j <= kWindow; ++j) {
    const int id = __builtin_amdgcn_readlane(key, j);  // of token j - 1
    const bool last = j >= n;
    if (!last && __builtin_amdgcn_readlane(key, j + 1) == id) {
      if (j < kWindow) {
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] += R::at(w[j % kWindow], i);
      }
      continue;
    }
    if (id == V) return;
    const bool from_before = start == 0 && __builtin_amdgcn_readlane(key, 0) == id;
    const bool goes_on = j == kWindow && __builtin_amdgcn_readlane(key, kWindow + 1) == id;
    if (there) {
      if (from_before || goes_on) {
        float* to = a.partial + ((size_t)window * 2 + (from_before ? 0 : 1)) * (size_t)(pieces * E) + (size_t)piece * E;
#pragma unroll
        for (int i = 0; i < E; i += 4) *(f32x4*)(to + i) = f32x4{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
      } else {
        finish<F32, ADD>(a, id, piece, sum, base[ADD ? j - 1 : 0]);
      }
    }
    if (last) return;
    start = j;
    if (j < kWindow) {
#pragma unroll
      for (int i = 0; i < E; ++i) sum[i] = R::at(w[j % kWindow], i);
    }
  }
}

// The partial sums p0 .. p1 - 1 of an id whose tokens begin in window `window`, of one slice.
template <int E>
__device__ __forceinline__ void add_parts(const float* base, size_t row, int64_t p0, int64_t p1, float (&sum)[E]) {
  for (int64_t p = p0; p < p1; p += 4) {
    f32x4 x[4][E / 4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t q = p + u < p1 ? p + u : p;
      const float* from = base + (size_t)q * 2 * row + (q == 0 ? row : 0);  // the first part is what its window ends with
#pragma unroll
      for (int i = 0; i < E / 4; ++i) x[u][i] = *(const f32x4*)(from + 4 * i);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (p + u < p1) {
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] += x[u][i / 4][i % 4];
      }
    }
  }
}

// A workgroup per kJoinWaves windows and slice.  A window has something to add where an id's tokens begin in it and go on behind it: its wave adds a
// few partial sums alone, all waves many (a limit of 4, 16 or 64: within 1 %).  A workgroup a window, nearly all of which had nothing to do, took 15 us
// for 16384 tokens.
constexpr int kAlone = 16;
template <bool F32, bool ADD>
__global__ __launch_bounds__(64 * kJoinWaves) void embedding_join(const RowArgs a) {
  typedef Row16<F32> R;
  constexpr int E = R::E;
  __shared__ float sums[kJoinWaves][64][E];
  __shared__ int many[kJoinWaves];  // partial sums of the windows that all waves add
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t group = blockIdx.x / a.slices, first = group * kJoinWaves;
  const int pieces = R::pieces(a.H), piece = (int)(blockIdx.x - group * a.slices) * 64 + lane;
  const bool there = piece < pieces;
  const size_t row = (size_t)(pieces * E);
  const float* const partial = a.partial + (size_t)(there ? piece : 0) * E;
  const int64_t window = first + wave, at = window * kWindow, end = at + kWindow;
  int parts = 0;
  if (end < a.T) {
    const int id = a.keys[end], before = at > 0 ? a.keys[at - 1] : -1;
    if (a.keys[end - 1] == id && id != (int)a.V && !(a.keys[at] == id && before == id)) {
      const int64_t stop = end + keys_before(a.keys + end, (int)(a.T - end), id, true);  // behind the id's last token
      parts = (int)((stop - 1) / kWindow - window + 1);
      if (parts <= kAlone) {
        float sum[E];
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] = 0.f;
        add_parts<E>(partial + (size_t)window * 2 * row, row, 0, parts, sum);
        if (there) {
          float base[E];
          if constexpr (ADD) load_base<E>(a, id, R::first(piece, a.H), base);
          finish<F32, ADD>(a, id, piece, sum, base);
        }
      }
    }
  }
  if (lane == 0) many[wave] = parts > kAlone ? parts : 0;
  __syncthreads();
  for (int x = 0; x < kJoinWaves; ++x) {
    const int all = many[x];
    if (all == 0) continue;
    const int each = (all + kJoinWaves - 1) / kJoinWaves, p0 = wave * each;
    float sum[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sum[i] = 0.f;
    add_parts<E>(partial + (size_t)(first + x) * 2 * row, row, p0, p0 + each < all ? p0 + each : all, sum);
#pragma unroll
    for (int i = 0; i < E; ++i) sums[wave][lane][i] = sum[i];
    __syncthreads();
    if (wave == 0 && there) {
#pragma unroll
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] += sums[w][lane][i];
      const int id = a.keys[(first + x + 1) * kWindow];
      float base[E];
      if constexpr (ADD) load_base<E>(a, id, R::first(piece, a.H), base);
      finish<F32, ADD>(a, id, piece, sum, base);
    }
    __syncthreads();
  }
}

constexpr int64_t kMostTokens = (int64_t)1 << 24, kMostHidden = (int64_t)1 << 22;

int check_extents(int dtype, int64_t T, int64_t H, int64_t V) {
  if (dtype != SKYRL_LOGITS_BF16 && dtype != SKYRL_LOGITS_F32) return SKYRL_LMHEAD_ERR_ARG;
  if (T < 1 || H < 1 || V < 1 || T > kMostTokens || H > kMostHidden || V >= ((int64_t)1 << 31) - 1) return SKYRL_LMHEAD_ERR_SHAPE;
  return SKYRL_LMHEAD_OK;
}

// Windows of a backward and slices of their rows, workgroups that write zeros: as many as one grid holds.
int zero_rows(int pieces) {  // a multiple of 8, whose rows are whole 16-byte pieces
  const int rows = kZeroBytes / 16 / pieces / 8 * 8;
  return rows < 8 ? 8 : (rows > 256 ? 256 : rows);
}
bool fits_grid(int64_t T, int64_t V, int pieces) {
  const int64_t units = (T + kWindow - 1) / kWindow * ((pieces + 63) / 64), zeros = (V + zero_rows(pieces) - 1) / zero_rows(pieces);
  return (units + zeros + kRowWaves) * kRowThreads < ((int64_t)1 << 32);
}

size_t round_256(size_t x) { return (x + 255) / 256 * 256; }

struct Scratch {
  size_t lists[2];  // of keys, each followed by its tokens; the second one where blocks are merged
  size_t list, partial, bytes;
};
Scratch scratch(int64_t T, int64_t H) {
  const size_t windows = (size_t)((T + kWindow - 1) / kWindow);
  Scratch s;
  s.list = round_256((size_t)T * 4);
  s.lists[0] = 0, s.lists[1] = 2 * s.list;
  s.partial = (T > kSortBlock ? 4 : 2) * s.list;
  s.bytes = s.partial + (windows > 1 ? windows * 2 * (size_t)((H + 7) / 8 * 8) * 4 : 0);
  return s;
}

template <bool F32, bool ADD>
hipError_t launch_rows(hipStream_t s, RowArgs a) {
  const int pieces = Row16<F32>::pieces(a.H);
  a.slices = (pieces + 63) / 64;
  a.units = (a.T + kWindow - 1) / kWindow * a.slices;
  a.zero_rows = zero_rows(pieces);
  const int64_t groups = (a.units + kRowWaves - 1) / kRowWaves + (ADD ? 0 : (a.V + a.zero_rows - 1) / a.zero_rows);
  hipLaunchKernelGGL((embedding_rows<F32, ADD>), dim3((unsigned)groups), dim3(kRowThreads), 0, s, a);
  const int64_t windows = (a.T + kWindow - 1) / kWindow, joins = (windows + kJoinWaves - 1) / kJoinWaves * a.slices;
  if (windows > 1) hipLaunchKernelGGL((embedding_join<F32, ADD>), dim3((unsigned)joins), dim3(64 * kJoinWaves), 0, s, a);
  return hipGetLastError();
}

}  // namespace

extern "C" {

int skyrl_lmhead_embedding_fwd(const void* table, int dtype, int64_t ld_table, const int64_t* ids, int64_t T, int64_t H, int64_t V, float scale, void* out,
                               void* stream) {
  if (!table || !ids || !out) return SKYRL_LMHEAD_ERR_NULL;
  const int st = check_extents(dtype, T, H, V);
  if (st) return st;
  if (ld_table < H || ld_table >= ((int64_t)1 << 40)) return SKYRL_LMHEAD_ERR_SHAPE;
  const bool f32 = dtype == SKYRL_LOGITS_F32;
  if ((((uintptr_t)table | (uintptr_t)out) & (f32 ? 3u : 1u)) || ((uintptr_t)ids & 7u)) return SKYRL_LMHEAD_ERR_ALIGN;
  if (!std::isfinite(scale)) return SKYRL_LMHEAD_ERR_ARG;
  const int pieces = f32 ? Row16<true>::pieces((int)H) : Row16<false>::pieces((int)H);
  const dim3 grid((unsigned)((T + kRowWaves - 1) / kRowWaves), (unsigned)((pieces + 255) / 256)), block(kRowThreads);
  hipLaunchKernelGGL(f32 ? embedding_fwd<true> : embedding_fwd<false>, grid, block, 0, (hipStream_t)stream, (const char*)table, ld_table, ids, T, (int)H, V,
                     scale, (char*)out);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? SKYRL_LMHEAD_OK : (int)e;
}

size_t skyrl_lmhead_embedding_bwd_workspace_bytes(int64_t T, int64_t H, int64_t V) {
  return check_extents(SKYRL_LOGITS_F32, T, H, V) || !fits_grid(T, V, Row16<true>::pieces((int)H)) ? 0 : scratch(T, H).bytes;
}

int skyrl_lmhead_embedding_bwd(const void* dout, int dtype, int64_t ld_dout, const int64_t* ids, int64_t padding, int64_t T, int64_t H, int64_t V,
                               float scale, int accumulate, void* dtable, void* workspace, size_t workspace_bytes, void* stream) {
  if (!dout || !ids || !dtable) return SKYRL_LMHEAD_ERR_NULL;
  const int st = check_extents(dtype, T, H, V);
  if (st) return st;
  // One row for all tokens (a pitch of zero) is a gradient like others.
  if ((ld_dout != 0 && ld_dout < H) || ld_dout >= ((int64_t)1 << 40)) return SKYRL_LMHEAD_ERR_SHAPE;
  const bool f32 = dtype == SKYRL_LOGITS_F32, add = accumulate != 0;
  if (((uintptr_t)dout & (f32 ? 3u : 1u)) || ((uintptr_t)dtable & (f32 || add ? 3u : 1u)) || ((uintptr_t)ids & 7u)) return SKYRL_LMHEAD_ERR_ALIGN;
  if (!std::isfinite(scale) || accumulate < 0 || accumulate > 1) return SKYRL_LMHEAD_ERR_ARG;
  if (!fits_grid(T, V, Row16<true>::pieces((int)H))) return SKYRL_LMHEAD_ERR_SHAPE;
  const Scratch w = scratch(T, H);
  if (!workspace || workspace_bytes < w.bytes) return SKYRL_LMHEAD_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 255u) return SKYRL_LMHEAD_ERR_ALIGN;
  hipStream_t s = (hipStream_t)stream;
  char* const base = (char*)workspace;
  auto keys = [&](int x) { return (int*)(base + w.lists[x & 1]); };
  auto tokens = [&](int x) { return (int*)(base + w.lists[x & 1] + w.list); };
  const int64_t blocks = (T + kSortBlock - 1) / kSortBlock;
  const int64_t groups = blocks > 1 ? blocks * (kSortBlock / kRankTokens) : (T + kRankTokens - 1) / kRankTokens;
  hipLaunchKernelGGL(embedding_rank, dim3((unsigned)groups), dim3(64 * kRankWaves), 0, s, ids, T, V, padding, keys(0), tokens(0));
  int in = 0;  // where the sorted tokens are
  for (int64_t block = kSortBlock; block < T; block *= kWay, ++in)
    hipLaunchKernelGGL(embedding_merge, dim3((unsigned)((T + 255) / 256)), dim3(256), 0, s, (const int*)keys(in), (const int*)tokens(in), (int)T, (int)block,
                       keys(in + 1), tokens(in + 1));
  RowArgs a{(const char*)dout, ld_dout, T, V, (int)H, scale, keys(in), tokens(in), (float*)(base + w.partial), (char*)dtable, 0, 0, 0};
  hipError_t e;
  if (f32) e = add ? launch_rows<true, true>(s, a) : launch_rows<true, false>(s, a);
  else e = add ? launch_rows<false, true>(s, a) : launch_rows<false, false>(s, a);
  return e == hipSuccess ? SKYRL_LMHEAD_OK : (int)e;
}

}  // extern "C"
