// What the two kernels of attention over the 8-bit paged cache share: one row at a time
// (attention_q8.cu) and tiles of rows on the tensor cores (attention_q8_tile.cu).
#pragma once

#include "cache_q8.cuh"

namespace nml_sm100 {

constexpr float kLog2e = 1.4426950408889634f;
// Sum of weights up to which the maximum so far still serves: F16 holds each of them.
constexpr float kLargestSum = 16384.0f;

struct AttentionParams {
  CacheQ8 cache;
  const void* query;
  const int32_t* offsets;  // [batch + 1] or null
  const float* sinks;
  float* partial;          // [rows, query_heads, splits, D + 4]: out, maximum, sum, exponent, -
  void* output;
  int64_t query_token_stride, query_head_stride;
  int tokens, query_heads, group, head_tiles, splits, window, first;
  float scale_log2;
  int* status;
};

// Value exponents, relative to the largest one met so far, that weights narrowed to F16 carry:
// within these, weights of 2^-8 and more of the row's largest keep all their bits and the smallest
// step is 2^-18 of it.  Pages of smaller values are multiplied by plain weights and their products
// scaled in f32; larger ones raise the largest and scale what was summed.
constexpr float kAboveExponent = 2.0f, kBelowExponent = -4.0f;
// (for the tile kernel, which keeps one exponent throughout: of all pages of a walk)
constexpr int kExponentRange = 6;

// Floats of a partial result: a multiple of 16 bytes.
template <int D>
constexpr int kPartial = D + 4;

// 2^x to 2 units in the last place (CUDA's documented bound of ex2.approx); results below 2^-126
// are zero.  exp2f() itself would spend two more instructions on those.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A factor of scores among which are masked ones, -infinity: what rounds to zero (a query row below
// 2^-85 or a tiny scale, times the factor of a block of zero keys, 2^-48) would make NaN of them.
// Scores are below 2^32, so that a factor of 2^-126 changes no weight.
__device__ __forceinline__ float masked_factor(float factor) {
  return factor < 1.1754944e-38f ? 1.1754944e-38f : factor;
}

// Power of two that puts the largest magnitude of a BF16 row (given as f32 bits) into
// [2^14, 2^15), so that the row's narrowing to F16 is exact down to 2^-29 of it; none for rows of
// zeros or with an infinity or a NaN.
__device__ __forceinline__ int query_shift(uint32_t largest_bits) {
  const int shift = 14 - (static_cast<int>(largest_bits >> 23) - 127);
  return largest_bits == 0 || largest_bits >= 0x7f800000u ? 0 : min(shift, 100);
}

// Which logical pages queries see: [0, front) and [back, end), of `pages` entries in this order.
struct Visible {
  int length;  // tokens in front of (and with) the last query's own, those of the table
  int start;   // first token of the first query's window
  int front, back, pages;
};

// `most`: tokens that the sequence's table can address; positions may lie past them.
__device__ __forceinline__ Visible visible_pages(int length, int start, int first, int most) {
  Visible v;
  v.length = min(max(length, 0), most);
  v.start = min(max(start, 0), v.length);
  const int end = (v.length + kCachePage - 1) / kCachePage;
  v.back = min(v.start / kCachePage, end);
  v.front = v.start > 0 ? min((first + kCachePage - 1) / kCachePage, v.back) : 0;
  v.pages = v.front + end - v.back;
  return v;
}

// Rows of a query tile of the tile kernel and the number of its work items: the most tiles that
// the sequences' rows can need, which no device data is asked for.
constexpr int kTileRows = 128;
inline int64_t query_tiles(int64_t tokens, int64_t batch, int64_t group) {
  const int64_t per_tile = kTileRows / group;
  return (tokens + (per_tile - 1) * (batch < tokens ? batch : tokens)) / per_tile;
}

template <typename T, int D>
int32_t launch_tiles(const AttentionParams& p, cudaStream_t stream, char* message,
                     size_t capacity);

}  // namespace nml_sm100
