// Writing the 8-bit paged K/V cache (with the rotary positions of keys and queries) and reading it
// back.  One 16-token page of one kv head is a scale block: 16 * head_dim contiguous E4M3 codes and
// one E8M0 byte, so a block is quantised by one warp that holds all its new rows in registers: no
// second pass over the data, no atomics.
//
// Both are bound by memory (6.46 TB/s measured).  Appending 16384 tokens with 64 query and 8 kv heads
// of 64, 323 MB: 74 us, 4.3 TB/s (106 with queries and cache writes in one CTA, 173 with every
// element's partner and angles loaded again); 4600 tokens with 32 and 8 heads of 128, 77 MB: 37 us, 2.1
// TB/s, where registers allow two CTAs an SM; a decode batch of 64: 4.1 us, one of 1: 3.8 us, which is
// the launch and four dependent loads (length, page, old scale, codes).  Reading back 64 sequences
// of about 4050 tokens, 792 MB: 141 us, 5.6 TB/s.
#include "cache_q8.cuh"

namespace nml_sm100 {
namespace {

struct AppendParams {
  CacheQ8 cache;
  const void* source[2];  // key, value
  const void* query;
  void* query_output;
  const int32_t* offsets;
  const float* rotary;
  int64_t token_stride[2], head_stride[2];
  int64_t query_token_stride, query_head_stride, output_token_stride, output_head_stride;
  int tokens, query_heads, rotary_rows, rotary_dim;
  int* status;
};

// Eight consecutive elements as f32.
template <typename T>
__device__ __forceinline__ void load8(const T* address, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(address);
  const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Elem<T>::from_bits(words[i] & 0xffffu);
    x[2 * i + 1] = Elem<T>::from_bits(words[i] >> 16);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* address, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(address) =
      make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]),
                 Elem<T>::pack2(x[4], x[5]), Elem<T>::pack2(x[6], x[7]));
}

// A head's row is cut into units of 16 elements that rotate among themselves: elements
// [8u, 8u + 8) and their partners half the rotary width behind, or 16 neighbours (interleaved
// pairs, and everything past the rotary width).  `a` and `b` are where its two halves lie.
template <bool kInterleaved>
__device__ __forceinline__ void unit_places(int unit, int rotary_dim, int& a, int& b) {
  const bool apart = !kInterleaved && 16 * unit < rotary_dim;
  a = apart ? 8 * unit : 16 * unit;
  b = apart ? 8 * unit + (rotary_dim >> 1) : 16 * unit + 8;
}

// Angles of a unit at one position (`row` of the table: cosines, then sines); identity outside the
// rotary width or without a table.
struct Angles {
  float cos[8], sin[8];
  bool turn;
};

__device__ __forceinline__ Angles unit_angles(const float* row, int unit, int rotary_dim) {
  Angles angles;
  angles.turn = row != nullptr && 16 * unit < rotary_dim;
  if (!angles.turn) return angles;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float4 c = *reinterpret_cast<const float4*>(row + 8 * unit + 4 * j);
    const float4 s = *reinterpret_cast<const float4*>(row + (rotary_dim >> 1) + 8 * unit + 4 * j);
    angles.cos[4 * j] = c.x; angles.cos[4 * j + 1] = c.y;
    angles.cos[4 * j + 2] = c.z; angles.cos[4 * j + 3] = c.w;
    angles.sin[4 * j] = s.x; angles.sin[4 * j + 1] = s.y;
    angles.sin[4 * j + 2] = s.z; angles.sin[4 * j + 3] = s.w;
  }
  return angles;
}

// Products and their sum are rounded one by one, so that the result does not depend on how the
// compiler contracts them.
__device__ __forceinline__ void turn_pair(float& a, float& b, float cos, float sin) {
  const float x = a, y = b;
  a = __fsub_rn(__fmul_rn(x, cos), __fmul_rn(y, sin));
  b = __fadd_rn(__fmul_rn(y, cos), __fmul_rn(x, sin));
}

template <bool kInterleaved>
__device__ __forceinline__ void turn_unit(float (&a)[8], float (&b)[8], const Angles& angles) {
  if (!angles.turn) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (kInterleaved) {
      float (&half)[8] = i < 4 ? a : b;
      turn_pair(half[2 * (i & 3)], half[2 * (i & 3) + 1], angles.cos[i], angles.sin[i]);
    } else {
      turn_pair(a[i], b[i], angles.cos[i], angles.sin[i]);
    }
  }
}

__device__ __forceinline__ uint2 to_codes(const float (&x)[8], float inverse) {
  uint32_t words[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    words[w] = f32x2_to_e4m3x2(x[4 * w] * inverse, x[4 * w + 1] * inverse) |
               f32x2_to_e4m3x2(x[4 * w + 2] * inverse, x[4 * w + 3] * inverse) << 16;
  }
  return make_uint2(words[0], words[1]);
}

// Codes at an exponent smaller by log2(shrink).
__device__ __forceinline__ uint2 shrink_codes(uint2 old, float shrink) {
  const uint32_t words[2] = {old.x, old.y};
  float x[8];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t lo = e4m3x2_to_f16x2(words[w] & 0xffffu);
    const uint32_t hi = e4m3x2_to_f16x2(words[w] >> 16);
    x[4 * w] = Elem<__half>::from_bits(lo & 0xffffu);
    x[4 * w + 1] = Elem<__half>::from_bits(lo >> 16);
    x[4 * w + 2] = Elem<__half>::from_bits(hi & 0xffffu);
    x[4 * w + 3] = Elem<__half>::from_bits(hi >> 16);
  }
  return to_codes(x, shrink);
}

// A CTA takes kChunk consecutive rows: first the sequence and position of each, then every block
// whose first new row is among them (one warp for a block of one kv head's keys or values, all its
// new rows at once, up to 15 of which may lie behind the chunk) and the chunk's query rows.  A lane
// holds 16 elements of a row that rotate among themselves, so every element is read once, and the
// angles of a query row's unit serve all its heads.
template <typename T, int D, bool kInterleaved, int kChunk, int kThreads>
__global__ void __launch_bounds__(kThreads, kChunk == 1 ? 1 : D == 64 ? 4 : 2)
append_kernel(const AppendParams p) {
  constexpr int kWarps = kThreads / 32;
  constexpr int kLanes = D / 16;           // lanes of a row
  constexpr int kRows = 32 / kLanes;       // rows of one pass of a warp
  constexpr int kPasses = kCachePage / kRows;
  __shared__ int s_position[kChunk];       // -1: no row here, or nothing to write for it
  __shared__ int s_sequence[kChunk];
  __shared__ int s_count[kChunk];          // new rows of the block that starts at this row, else 0
  // of two CTAs for a chunk of many rows one writes the cache, one rotates the queries
  constexpr bool kApart = kChunk > 1;
  const bool both = !kApart || p.query == nullptr;
  const bool write_cache = both || (blockIdx.x & 1) != 0;
  const bool rotate_query = p.query != nullptr && (both || (blockIdx.x & 1) == 0);
  const int first_row = (both ? blockIdx.x : blockIdx.x >> 1) * kChunk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kChunk) {
    const int row = first_row + threadIdx.x;
    int position = -1, count = 0, sequence = -1;
    if (row < p.tokens) {
      sequence = p.offsets == nullptr ? row : sequence_of_row(p.offsets, p.cache.batch, row);
      if (sequence >= 0) {
        const int begin = p.offsets == nullptr ? row : p.offsets[sequence];
        const int given_end = p.offsets == nullptr ? row + 1 : p.offsets[sequence + 1];
        const int end = min(given_end, p.tokens);
        position = max(p.cache.lengths[sequence], 0) - given_end + row;
        const int limit = p.cache.table_width * kCachePage;
        const int usable = p.rotary == nullptr ? limit : min(limit, p.rotary_rows);
        if (position >= usable) {
          atomicOr(p.status, NML_SM100_STATUS_INDEX_RANGE);
          position = -1;
        }
        if (position >= 0 && (row == begin || position == 0 || position % kCachePage == 0)) {
          count = min(min(end - row, kCachePage - position % kCachePage), usable - position);
        }
        if (position < 0) position = -1;
      }
    }
    s_position[threadIdx.x] = position;
    s_sequence[threadIdx.x] = sequence;
    s_count[threadIdx.x] = count;
  }
  __syncthreads();
  const int unit = lane % kLanes;
  int place_a, place_b;
  unit_places<kInterleaved>(unit, p.rotary_dim, place_a, place_b);

  // ---- keys and values ----
  const int tasks = write_cache ? kChunk * p.cache.kv_heads * 2 : 0;
  for (int task = warp; task < tasks; task += kWarps) {
    const int leader = task / (p.cache.kv_heads * 2);
    const int count = s_count[leader];
    if (count == 0) continue;
    const int head = (task >> 1) % p.cache.kv_heads;
    const bool is_key = (task & 1) == 0;
    const int position = s_position[leader];
    const int lead = position % kCachePage;
    // one lane reads the block's old exponent and, at the end, writes its new one: lanes that run
    // apart could otherwise meet the new one as the old
    int page = 0;
    uint32_t old_scale = 0;  // (below every exponent: no older tokens)
    if (lane == 0) {
      page = physical_page(p.cache, s_sequence[leader], position / kCachePage, p.status);
      if (lead > 0 && page >= 0) {
        old_scale = (is_key ? p.cache.scales[0] : p.cache.scales[1])
            [static_cast<int64_t>(page) * p.cache.kv_heads + head];
      }
    }
    const int64_t token_stride = is_key ? p.token_stride[0] : p.token_stride[1];
    const T* source = static_cast<const T*>(is_key ? p.source[0] : p.source[1]) +
                      static_cast<int64_t>(first_row + leader) * token_stride +
                      head * (is_key ? p.head_stride[0] : p.head_stride[1]);
    float a[kPasses][8], b[kPasses][8];
    uint32_t largest = 0;
    uint32_t bad = 0;  // bit i: the row of pass i holds an infinity or a NaN
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + lane / kLanes;  // slot in the block
      if (r >= lead && r < lead + count) {
        const T* row = source + static_cast<int64_t>(r - lead) * token_stride;
        load8(row + place_a, a[i]);
        load8(row + place_b, b[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[i][j] = b[i][j] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + lane / kLanes;
      if (is_key && p.rotary != nullptr && r >= lead && r < lead + count) {
        turn_unit<kInterleaved>(
            a[i], b[i],
            unit_angles(p.rotary + static_cast<int64_t>(position - lead + r) * p.rotary_dim, unit,
                        p.rotary_dim));
      }
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m = max(m, max(__float_as_uint(a[i][j]) & 0x7fffffffu,
                       __float_as_uint(b[i][j]) & 0x7fffffffu));
      }
#pragma unroll
      for (int offset = 1; offset < kLanes; offset <<= 1) {
        m = max(m, __shfl_xor_sync(0xffffffffu, m, offset));
      }
      if (m >= 0x7f800000u) {
        bad |= 1u << i;
      } else {
        largest = max(largest, m);
      }
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    page = __shfl_sync(0xffffffffu, page, 0);
    if (page < 0) continue;
    const int64_t block = static_cast<int64_t>(page) * p.cache.kv_heads + head;
    uint8_t* codes = (is_key ? p.cache.codes[0] : p.cache.codes[1]) + block * (kCachePage * D);
    uint8_t* scale = (is_key ? p.cache.scales[0] : p.cache.scales[1]) + block;
    // tokens in front of the first new row are older ones of this sequence
    const int before = scale_exponent(__shfl_sync(0xffffffffu, old_scale, 0));
    const int exponent = max(block_exponent(largest), before);
    if (lead > 0 && exponent > before) {
      // older codes move to the grown exponent
      const float shrink = exp2_int(before - exponent);
      for (int r = lane / kLanes; r < lead; r += kRows) {
        uint4* place = reinterpret_cast<uint4*>(codes + r * D + 16 * unit);
        const uint4 old = *place;
        const uint2 lo = shrink_codes(make_uint2(old.x, old.y), shrink);
        const uint2 hi = shrink_codes(make_uint2(old.z, old.w), shrink);
        *place = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
    }
    const float inverse = exp2_int(-exponent);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + lane / kLanes;
      if (r < lead || r >= lead + count) continue;
      const uint2 nan = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
      const bool is_bad = (bad >> i & 1u) != 0;
      *reinterpret_cast<uint2*>(codes + r * D + place_a) = is_bad ? nan : to_codes(a[i], inverse);
      *reinterpret_cast<uint2*>(codes + r * D + place_b) = is_bad ? nan : to_codes(b[i], inverse);
    }
    if (lane == 0) *scale = static_cast<uint8_t>(exponent + 127);
  }

  // ---- query rows ----
  if (!rotate_query) return;
  auto rotate_heads = [&](int local, int first_head, int head_step) {
    const int row = first_row + local;
    if (row >= p.tokens || s_sequence[local] < 0) return;  // outside every sequence: untouched
    const int position = s_position[local];
    const Angles angles = unit_angles(
        p.rotary == nullptr || position < 0
            ? nullptr
            : p.rotary + static_cast<int64_t>(position) * p.rotary_dim,
        unit, p.rotary_dim);
    const T* source =
        static_cast<const T*>(p.query) + static_cast<int64_t>(row) * p.query_token_stride;
    T* out = static_cast<T*>(p.query_output) + static_cast<int64_t>(row) * p.output_token_stride;
#pragma unroll 4
    for (int head = first_head + lane / kLanes; head < p.query_heads; head += head_step) {
      float a[8], b[8];
      if (position >= 0) {
        load8(source + head * p.query_head_stride + place_a, a);
        load8(source + head * p.query_head_stride + place_b, b);
        turn_unit<kInterleaved>(a, b, angles);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.0f;
      }
      store8(out + head * p.output_head_stride + place_a, a);
      store8(out + head * p.output_head_stride + place_b, b);
    }
  };
  if constexpr (kChunk == 1) {  // the warps share one row's heads
    rotate_heads(0, (kWarps - 1 - warp) * kRows, kWarps * kRows);
  } else {
    for (int local = warp; local < kChunk; local += kWarps) rotate_heads(local, 0, kRows);
  }
}

struct ReadParams {
  CacheQ8 cache;
  const int32_t* offsets;
  void* output[2];
  int tokens;
  int* status;
};

constexpr int kReadThreads = 256;
constexpr int kReadRows = 16;

// A CTA takes 16 output rows: where each comes from once, then pieces of 16 codes (16 bytes in,
// 32 bytes out) of keys and values.
template <typename T, int D>
__global__ void __launch_bounds__(kReadThreads)
read_kernel(const ReadParams p) {
  __shared__ int64_t s_source[kReadRows];  // slot of the row: page * 16 + slot, -1: zeros, -2: none
  const int first_row = blockIdx.x * kReadRows;
  if (threadIdx.x < kReadRows) {
    const int row = first_row + threadIdx.x;
    int64_t source = -2;
    if (row < p.tokens) {
      const int sequence = sequence_of_row(p.offsets, p.cache.batch, row);
      if (sequence >= 0) {
        const int position = row - p.offsets[sequence];
        source = -1;
        if (position < 0 || position >= p.cache.table_width * kCachePage) {
          atomicOr(p.status, NML_SM100_STATUS_INDEX_RANGE);
        } else {
          const int page = physical_page(p.cache, sequence, position / kCachePage, p.status);
          if (page >= 0) source = static_cast<int64_t>(page) * kCachePage + position % kCachePage;
        }
      }
    }
    s_source[threadIdx.x] = source;
  }
  __syncthreads();
  constexpr int kPieces = D / 16;
  const int per_row = p.cache.kv_heads * kPieces;
  for (int item = threadIdx.x; item < 2 * kReadRows * per_row; item += kReadThreads) {
    const int local = item / (2 * per_row);
    int rest = item - local * 2 * per_row;
    const int which = rest >= per_row ? 1 : 0;
    rest -= which * per_row;
    const int head = rest / kPieces, piece = rest % kPieces;
    const int64_t source = s_source[local];
    if (source == -2) continue;
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (source >= 0) {
      const int64_t block = (source >> 4) * p.cache.kv_heads + head;
      const uint8_t* base = which == 0 ? p.cache.codes[0] : p.cache.codes[1];
      const uint8_t* scales = which == 0 ? p.cache.scales[0] : p.cache.scales[1];
      const uint4 codes = *reinterpret_cast<const uint4*>(
          base + (block * kCachePage + (source & 15)) * D + 16 * piece);
      const float scale = exp2_int(scale_exponent(scales[block]));
      const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
      uint32_t values[8];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a = e4m3x2_to_f16x2(words[w] & 0xffffu);
        const uint32_t b = e4m3x2_to_f16x2(words[w] >> 16);
        values[2 * w] = Elem<T>::pack2(Elem<__half>::from_bits(a & 0xffffu) * scale,
                                       Elem<__half>::from_bits(a >> 16) * scale);
        values[2 * w + 1] = Elem<T>::pack2(Elem<__half>::from_bits(b & 0xffffu) * scale,
                                           Elem<__half>::from_bits(b >> 16) * scale);
      }
      lo = make_uint4(values[0], values[1], values[2], values[3]);
      hi = make_uint4(values[4], values[5], values[6], values[7]);
    }
    T* out = static_cast<T*>(which == 0 ? p.output[0] : p.output[1]) +
             (static_cast<int64_t>(first_row + local) * p.cache.kv_heads + head) * D + 16 * piece;
    *reinterpret_cast<uint4*>(out) = lo;
    *reinterpret_cast<uint4*>(out + 8) = hi;
  }
}

template <typename T, int D, bool kInterleaved>
void launch_append(const AppendParams& p, cudaStream_t stream) {
  // Few rows: one row and many warps for a CTA, so that a decode batch spreads over the SMs.  Many:
  // 16 rows, so that most CTAs own about one block of every head.
  if (p.offsets == nullptr || p.tokens < 1024) {
    append_kernel<T, D, kInterleaved, 1, 512>
        <<<static_cast<unsigned>(p.tokens), 512, 0, stream>>>(p);
  } else {
    const int64_t chunks = (static_cast<int64_t>(p.tokens) + kCachePage - 1) / kCachePage;
    append_kernel<T, D, kInterleaved, kCachePage, 256>
        <<<static_cast<unsigned>(p.query == nullptr ? chunks : 2 * chunks), 256, 0, stream>>>(p);
  }
}

template <typename T>
void launch_append(const AppendParams& p, int dim, bool interleaved, cudaStream_t stream) {
  if (dim == 64) {
    interleaved ? launch_append<T, 64, true>(p, stream) : launch_append<T, 64, false>(p, stream);
  } else {
    interleaved ? launch_append<T, 128, true>(p, stream) : launch_append<T, 128, false>(p, stream);
  }
}

bool valid_rows(const void* data, int64_t token_stride, int64_t head_stride) {
  return data != nullptr && reinterpret_cast<uintptr_t>(data) % 16 == 0 && token_stride >= 0 &&
         head_stride >= 0 && token_stride % 8 == 0 && head_stride % 8 == 0;
}

bool valid_dtype(int32_t dtype) { return dtype == NML_SM100_F16 || dtype == NML_SM100_BF16; }

}  // namespace
}  // namespace nml_sm100

using namespace nml_sm100;

extern "C" int32_t nml_sm100_paged_append_q8(const NmlSm100PagedAppendQ8* request,
                                             char* error_message, size_t error_message_capacity) {
  if (request == nullptr || request->struct_size < sizeof(NmlSm100PagedAppendQ8)) {
    return fail(NML_SM100_INVALID_ARGUMENT, "truncated paged append request", error_message,
                error_message_capacity);
  }
  const NmlSm100PagedAppendQ8& r = *request;
  const bool query = r.query != nullptr;
  if (!valid_cache_q8(r.cache, true) || r.stream == nullptr || !fits_i32(r.tokens) ||
      !valid_rows(r.key, r.key_token_stride, r.key_head_stride) ||
      !valid_rows(r.value, r.value_token_stride, r.value_head_stride) ||
      (r.token_offsets == nullptr && r.tokens != r.cache.batch) ||
      (query && (!valid_rows(r.query, r.query_token_stride, r.query_head_stride) ||
                 !valid_rows(r.query_output, r.output_token_stride, r.output_head_stride) ||
                 r.query_output == r.query || r.query_heads <= 0 || r.query_heads > 65536)) ||
      r.cache.kv_heads > 65536) {
    return fail(NML_SM100_INVALID_ARGUMENT,
                "invalid paged append request (head_dim 64 or 128, page size 16, rows of 16-byte "
                "aligned heads)",
                error_message, error_message_capacity);
  }
  if (r.rotary != nullptr &&
      (!fits_i32(r.rotary_rows) || r.rotary_dim <= 0 || r.rotary_dim % 16 != 0 ||
       r.rotary_dim > r.cache.head_dim || reinterpret_cast<uintptr_t>(r.rotary) % 16 != 0)) {
    return fail(NML_SM100_INVALID_ARGUMENT,
                "the rotary width must be a multiple of 16 up to head_dim, its table 16-byte "
                "aligned",
                error_message, error_message_capacity);
  }
  if (!valid_dtype(r.dtype)) {
    return fail(NML_SM100_INVALID_ARGUMENT, "paged append supports F16 and BF16 only",
                error_message, error_message_capacity);
  }
  const DeviceInfo* device = current_device(error_message, error_message_capacity);
  if (device == nullptr) return NML_SM100_LAUNCH_FAILURE;
  AppendParams p = {};
  p.cache = cache_params(r.cache);
  p.source[0] = r.key;
  p.source[1] = r.value;
  p.token_stride[0] = r.key_token_stride;
  p.token_stride[1] = r.value_token_stride;
  p.head_stride[0] = r.key_head_stride;
  p.head_stride[1] = r.value_head_stride;
  p.query = r.query;
  p.query_output = r.query_output;
  p.query_token_stride = r.query_token_stride;
  p.query_head_stride = r.query_head_stride;
  p.output_token_stride = r.output_token_stride;
  p.output_head_stride = r.output_head_stride;
  p.query_heads = query ? static_cast<int>(r.query_heads) : 0;
  p.offsets = r.token_offsets;
  p.rotary = r.rotary;
  p.rotary_rows = r.rotary != nullptr ? static_cast<int>(r.rotary_rows) : 0;
  p.rotary_dim = r.rotary != nullptr ? static_cast<int>(r.rotary_dim) : 0;
  p.tokens = static_cast<int>(r.tokens);
  p.status = device->status_word;
  cudaStream_t stream = static_cast<cudaStream_t>(r.stream);
  const int dim = static_cast<int>(r.cache.head_dim);
  if (r.dtype == NML_SM100_F16) {
    launch_append<__half>(p, dim, r.rotary_interleaved != 0, stream);
  } else {
    launch_append<__nv_bfloat16>(p, dim, r.rotary_interleaved != 0, stream);
  }
  return launch_result(error_message, error_message_capacity);
}

extern "C" int32_t nml_sm100_paged_read_q8(const NmlSm100PagedReadQ8* request, char* error_message,
                                           size_t error_message_capacity) {
  if (request == nullptr || request->struct_size < sizeof(NmlSm100PagedReadQ8)) {
    return fail(NML_SM100_INVALID_ARGUMENT, "truncated paged read request", error_message,
                error_message_capacity);
  }
  const NmlSm100PagedReadQ8& r = *request;
  if (!valid_cache_q8(r.cache, false) || r.token_offsets == nullptr || r.key_output == nullptr ||
      r.value_output == nullptr || r.stream == nullptr || !fits_i32(r.tokens) ||
      r.cache.kv_heads > 65536 || reinterpret_cast<uintptr_t>(r.key_output) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(r.value_output) % 16 != 0) {
    return fail(NML_SM100_INVALID_ARGUMENT,
                "invalid paged read request (head_dim 64 or 128, page size 16)", error_message,
                error_message_capacity);
  }
  if (!valid_dtype(r.dtype)) {
    return fail(NML_SM100_INVALID_ARGUMENT, "paged read supports F16 and BF16 only", error_message,
                error_message_capacity);
  }
  const DeviceInfo* device = current_device(error_message, error_message_capacity);
  if (device == nullptr) return NML_SM100_LAUNCH_FAILURE;
  ReadParams p = {};
  p.cache = cache_params(r.cache);
  p.offsets = r.token_offsets;
  p.output[0] = r.key_output;
  p.output[1] = r.value_output;
  p.tokens = static_cast<int>(r.tokens);
  p.status = device->status_word;
  const unsigned grid =
      static_cast<unsigned>((static_cast<int64_t>(r.tokens) + kReadRows - 1) / kReadRows);
  cudaStream_t stream = static_cast<cudaStream_t>(r.stream);
  const bool half = r.dtype == NML_SM100_F16;
  if (r.cache.head_dim == 64) {
    half ? read_kernel<__half, 64><<<grid, kReadThreads, 0, stream>>>(p)
         : read_kernel<__nv_bfloat16, 64><<<grid, kReadThreads, 0, stream>>>(p);
  } else {
    half ? read_kernel<__half, 128><<<grid, kReadThreads, 0, stream>>>(p)
         : read_kernel<__nv_bfloat16, 128><<<grid, kReadThreads, 0, stream>>>(p);
  }
  return launch_result(error_message, error_message_capacity);
}
