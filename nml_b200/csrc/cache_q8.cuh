// Shared by the kernels over the 8-bit paged K/V cache: the cache as kernels see it, the search
// for a row's sequence, E4M3 conversions and the block exponent rule.
#pragma once

#include "common.cuh"

namespace nml_sm100 {

constexpr int kCachePage = 16;      // tokens of a page, the tokens of a scale block
constexpr int kLowestExponent = -48;
constexpr int kHighestExponent = 48;

struct CacheQ8 {
  uint8_t* codes[2];   // keys, values: [pages, kv_heads, 16, head_dim]
  uint8_t* scales[2];  // [pages, kv_heads]
  const int32_t* page_table;
  const int32_t* lengths;
  int batch, kv_heads, physical_pages, table_width;
};

// Checks what every entry point asks of the cache; `lengths` says whether it is read.
inline bool valid_cache_q8(const NmlSm100CacheQ8& c, bool lengths) {
  return c.key != nullptr && c.key_scales != nullptr && c.value != nullptr &&
         c.value_scales != nullptr && c.page_table != nullptr &&
         (!lengths || c.sequence_lengths != nullptr) && fits_i32(c.batch) &&
         fits_i32(c.kv_heads) && fits_i32(c.physical_pages) && fits_i32(c.table_width) &&
         (c.head_dim == 64 || c.head_dim == 128) && c.page_size == kCachePage &&
         // (some tokens short of the largest position, so that sums with a page's never pass it)
         c.table_width <= (std::numeric_limits<int32_t>::max() - 1024) / kCachePage &&
         reinterpret_cast<uintptr_t>(c.key) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(c.value) % 16 == 0;
}

inline CacheQ8 cache_params(const NmlSm100CacheQ8& c) {
  CacheQ8 p = {};
  p.codes[0] = c.key;
  p.codes[1] = c.value;
  p.scales[0] = c.key_scales;
  p.scales[1] = c.value_scales;
  p.page_table = c.page_table;
  p.lengths = c.sequence_lengths;
  p.batch = static_cast<int>(c.batch);
  p.kv_heads = static_cast<int>(c.kv_heads);
  p.physical_pages = static_cast<int>(c.physical_pages);
  p.table_width = static_cast<int>(c.table_width);
  return p;
}

// The sequence whose rows [offsets[b], offsets[b + 1]) hold `row`, or -1: the last b with
// offsets[b] <= row (empty sequences share their offset with the next one), checked against its
// end.  offsets has batch + 1 entries.
__device__ __forceinline__ int sequence_of_row(const int32_t* __restrict__ offsets, int batch,
                                               int row) {
  int low = 0, high = batch;  // offsets[low] <= row (if any), the answer is in [low, high)
  while (high - low > 1) {
    const int middle = (low + high) >> 1;
    if (offsets[middle] <= row) {
      low = middle;
    } else {
      high = middle;
    }
  }
  return offsets[low] <= row && row < offsets[low + 1] ? low : -1;
}

// Physical page of a logical one, -1 (and the status bit) for an entry outside the cache.
__device__ __forceinline__ int physical_page(const CacheQ8& cache, int sequence, int logical,
                                             int* status) {
  const int32_t page =
      cache.page_table[static_cast<int64_t>(sequence) * cache.table_width + logical];
  if (page < 0 || page >= cache.physical_pages) {
    atomicOr(status, NML_SM100_STATUS_INDEX_RANGE);
    return -1;
  }
  return page;
}

// Tokens of a sequence as given, which its rows' positions follow from; more than its table can
// address raise the status bit, fewer than none are none.
__device__ __forceinline__ int sequence_length(const CacheQ8& cache, int sequence, int* status) {
  const int length = max(cache.lengths[sequence], 0);
  if (length > cache.table_width * kCachePage) atomicOr(status, NML_SM100_STATUS_INDEX_RANGE);
  return length;
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float exp2_int(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Scale exponent of an E8M0 byte as the append writes it; bytes it cannot write are clamped.
__device__ __forceinline__ int scale_exponent(uint32_t byte) {
  return min(max(static_cast<int>(byte) - 127, kLowestExponent), kHighestExponent);
}

// Smallest exponent e in [-48, 48] with |x| <= 448 * 2^e for the largest |x|, given as the bits of
// a finite f32.  448 = 1.75 * 2^8, so 2^k * 1.f asks for k - 8 up to 1.f = 1.75 and k - 7 above.
__device__ __forceinline__ int block_exponent(uint32_t largest_bits) {
  const int k = static_cast<int>(largest_bits >> 23) - 127;
  const int e = k - 8 + ((largest_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kLowestExponent), kHighestExponent);
}

// Two E4M3 codes (low byte first) as two f16: exact, every code is an f16 number.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes16) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes16)));
  return r;
}

// Two f32 as E4M3 codes, `lo` in the low byte: nearest even, saturating, NaN stays NaN.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace nml_sm100
