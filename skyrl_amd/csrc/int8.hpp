// The head in 8-bit integers (int8_tiles.hip): what lmhead_kernels.hip launches.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lmhead {

constexpr int kInt8K = 128;  // k of a k-tile: rows of values are whole k-tiles long, zeros behind the hidden size
// |sum of products| <= 127 * 128 * H stays below 2^31: hidden values are 127 at most, weights from elsewhere may be -128
constexpr int64_t kInt8MostHidden = (((int64_t)1 << 31) - 1) / (127 * 128) / kInt8K * kInt8K;

struct Int8Rows {
  const int8_t* values;  // [rows, ld], ld a multiple of kInt8K bytes
  int64_t ld;
  const float* scale;    // [rows]
};

// values[r, :H] = round(127 x / max |x|) of row r of src (bf16 or fp32), zeros up to the next multiple of kInt8K; scale[r] = max |x| / 127.  A row with
// NaN or an infinity has values of zero and a scale of NaN.
hipError_t launch_int8_rows(hipStream_t s, const void* src, bool f32, int64_t ld_src, int64_t rows, int64_t H, int8_t* values, int64_t ld, float* scale);

struct Int8FwdArgs {
  Int8Rows W, Hd;
  int T, K, V;  // K: bytes of a row that are contracted, a multiple of kInt8K
  float rcp_temp;
  float *part_max, *part_sum, *part_pz;  // part_pz NULL: no entropy
};
// Few tokens: the weight streams through registers (int8_few.hip).
bool int8_streams(int64_t T, int64_t K);
int int8_stream_parts(int64_t V, int ncu);  // partials a token of the statistics
hipError_t launch_int8_fwd_stream(hipStream_t s, const Int8FwdArgs& a, int parts);
hipError_t launch_int8_fwd_tiles(hipStream_t s, const Int8FwdArgs& a, bool half, bool shapes, int split, int workgroups);

struct Int8LogitsArgs {
  Int8Rows W, Hd;
  int T, K, V;
  void* out;
  int64_t ldo;
  int out_f32;
};
hipError_t launch_int8_logits_stream(hipStream_t s, const Int8LogitsArgs& a, int ncu);
hipError_t launch_int8_logits(hipStream_t s, const Int8LogitsArgs& a, bool half, bool shapes, int split, int workgroups);

}  // namespace lmhead
