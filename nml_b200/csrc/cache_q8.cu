// Writing the 8-bit paged K/V cache (with the rotary positions of keys and queries) and reading it
// back.  One 16-token page of one kv head is a scale block: 16 * head_dim contiguous E4M3 codes and
// one E8M0 byte, so a block is quantised by one warp that holds all its new rows in registers: no
// second pass over the data, no atomics.
#include "cache_q8.cuh"

namespace nml_sm100 {
namespace {

constexpr int kAppendThreads = 256;

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

// Elements [d0, d0 + 8) of a head's row after rotation by the angles of one position (`angles`:
// cosines then sines, null for none).  Products and their sum are rounded one by one, so the
// result does not depend on how the compiler contracts them.
template <typename T, bool kInterleaved>
__device__ __forceinline__ void rotated8(const T* row, int d0, const float* angles, int rotary_dim,
                                         float (&x)[8]) {
  load8(row + d0, x);
  if (angles == nullptr || d0 >= rotary_dim) return;
  const int half = rotary_dim >> 1;
  if constexpr (kInterleaved) {
    const float4 cos = *reinterpret_cast<const float4*>(angles + (d0 >> 1));
    const float4 sin = *reinterpret_cast<const float4*>(angles + half + (d0 >> 1));
    const float c[4] = {cos.x, cos.y, cos.z, cos.w}, s[4] = {sin.x, sin.y, sin.z, sin.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
    }
  } else {
    const bool upper = d0 >= half;
    const int index = upper ? d0 - half : d0;
    float other[8];
    load8(row + (upper ? d0 - half : d0 + half), other);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float4 cos = *reinterpret_cast<const float4*>(angles + index + 4 * j);
      const float4 sin = *reinterpret_cast<const float4*>(angles + half + index + 4 * j);
      const float c[4] = {cos.x, cos.y, cos.z, cos.w}, s[4] = {sin.x, sin.y, sin.z, sin.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float own = __fmul_rn(x[4 * j + i], c[i]);
        const float turn = __fmul_rn(other[4 * j + i], s[i]);
        x[4 * j + i] = upper ? __fadd_rn(own, turn) : __fsub_rn(own, turn);
      }
    }
  }
}

// A CTA takes kChunk consecutive rows: first the sequence and position of each, then every block
// whose first new row is among them (one warp for a block of one kv head's keys or values, all its
// new rows at once, up to 16 of which may lie behind the chunk), then the chunk's query rows.
template <typename T, int D, bool kInterleaved, int kChunk>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8;            // lanes of a row, eight elements each
  constexpr int kRows = 32 / kLanes;       // rows of one pass of a warp
  constexpr int kPasses = kCachePage / kRows;
  __shared__ int s_position[kChunk];       // -1: no row here, or nothing to write for it
  __shared__ int s_sequence[kChunk];
  __shared__ int s_count[kChunk];          // new rows of the block that starts at this row, else 0
  const int first_row = blockIdx.x * kChunk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kChunk) {
    const int row = first_row + threadIdx.x;
    int position = -1, count = 0, sequence = -1;
    if (row < p.tokens) {
      sequence = p.offsets == nullptr ? row : sequence_of_row(p.offsets, p.cache.batch, row);
      if (sequence >= 0) {
        const int begin = p.offsets == nullptr ? row : p.offsets[sequence];
        const int end = p.offsets == nullptr ? row + 1 : min(p.offsets[sequence + 1], p.tokens);
        const int given_end = p.offsets == nullptr ? end : p.offsets[sequence + 1];
        const int length = p.cache.lengths[sequence];
        position = length - given_end + row;
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

  // ---- keys and values ----
  const int units = kChunk * p.cache.kv_heads * 2;
  for (int unit = warp; unit < units; unit += kAppendThreads / 32) {
    const int leader = unit / (p.cache.kv_heads * 2);
    const int count = s_count[leader];
    if (count == 0) continue;
    const int head = (unit >> 1) % p.cache.kv_heads;
    const int which = unit & 1;  // 0: keys, 1: values
    const int position = s_position[leader];
    const int lead = position % kCachePage;
    int page = 0;
    if (lane == 0) {
      page = physical_page(p.cache, s_sequence[leader], position / kCachePage, p.status);
    }
    page = __shfl_sync(0xffffffffu, page, 0);
    if (page < 0) continue;
    const int64_t block = static_cast<int64_t>(page) * p.cache.kv_heads + head;
    const bool is_key = which == 0;
    uint8_t* codes = (is_key ? p.cache.codes[0] : p.cache.codes[1]) + block * (kCachePage * D);
    uint8_t* scale = (is_key ? p.cache.scales[0] : p.cache.scales[1]) + block;
    // tokens in front of the first new row are older ones of this sequence
    const int before = lead > 0 ? scale_exponent(*scale) : kLowestExponent;
    const int64_t token_stride = is_key ? p.token_stride[0] : p.token_stride[1];
    const T* source = static_cast<const T*>(is_key ? p.source[0] : p.source[1]) +
                      static_cast<int64_t>(first_row + leader) * token_stride +
                      head * (is_key ? p.head_stride[0] : p.head_stride[1]);
    const int d0 = 8 * (lane % kLanes);
    float x[kPasses][8];
    uint32_t largest = 0;
    uint32_t bad = 0;  // bit i: the row of pass i holds an infinity or a NaN
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + lane / kLanes;  // slot in the block
      const bool live = r >= lead && r < lead + count;
      if (live) {
        const T* row = source + static_cast<int64_t>(r - lead) * token_stride;
        const float* angles =
            is_key && p.rotary != nullptr
                ? p.rotary + static_cast<int64_t>(position - lead + r) * p.rotary_dim
                : nullptr;
        rotated8<T, kInterleaved>(row, d0, angles, p.rotary_dim, x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = 0.0f;
      }
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7fffffffu);
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
    const int exponent = max(block_exponent(largest), before);
    if (lead > 0 && exponent > before) {
      // older codes move to the grown exponent
      const float shrink = exp2_int(before - exponent);
      for (int r = lane / kLanes; r < lead; r += kRows) {
        uint2* place = reinterpret_cast<uint2*>(codes + r * D + d0);
        const uint2 old = *place;
        const uint32_t words[2] = {old.x, old.y};
        uint32_t again[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t lo = e4m3x2_to_f16x2(words[w] & 0xffffu);
          const uint32_t hi = e4m3x2_to_f16x2(words[w] >> 16);
          again[w] = f32x2_to_e4m3x2(Elem<__half>::from_bits(lo & 0xffffu) * shrink,
                                     Elem<__half>::from_bits(lo >> 16) * shrink) |
                     f32x2_to_e4m3x2(Elem<__half>::from_bits(hi & 0xffffu) * shrink,
                                     Elem<__half>::from_bits(hi >> 16) * shrink)
                         << 16;
        }
        *place = make_uint2(again[0], again[1]);
      }
    }
    const float inverse = exp2_int(-exponent);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + lane / kLanes;
      if (r < lead || r >= lead + count) continue;
      uint32_t words[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        words[w] = f32x2_to_e4m3x2(x[i][4 * w] * inverse, x[i][4 * w + 1] * inverse) |
                   f32x2_to_e4m3x2(x[i][4 * w + 2] * inverse, x[i][4 * w + 3] * inverse) << 16;
      }
      if (bad >> i & 1u) words[0] = words[1] = 0x7f7f7f7fu;
      *reinterpret_cast<uint2*>(codes + r * D + d0) = make_uint2(words[0], words[1]);
    }
    if (lane == 0) *scale = static_cast<uint8_t>(exponent + 127);
  }

  // ---- query rows ----
  if (p.query == nullptr) return;
  const int per_row = p.query_heads * kLanes;
  for (int item = threadIdx.x; item < kChunk * per_row; item += kAppendThreads) {
    const int local = item / per_row;
    const int rest = item - local * per_row;
    const int head = rest / kLanes;
    const int d0 = 8 * (rest % kLanes);
    const int row = first_row + local;
    if (row >= p.tokens || s_sequence[local] < 0) continue;  // outside every sequence: untouched
    const int position = s_position[local];
    float x[8];
    if (position >= 0) {
      const T* source = static_cast<const T*>(p.query) +
                        static_cast<int64_t>(row) * p.query_token_stride +
                        head * p.query_head_stride;
      const float* angles = p.rotary == nullptr
                                ? nullptr
                                : p.rotary + static_cast<int64_t>(position) * p.rotary_dim;
      rotated8<T, kInterleaved>(source, d0, angles, p.rotary_dim, x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.0f;
    }
    T* out = static_cast<T*>(p.query_output) + static_cast<int64_t>(row) * p.output_token_stride +
             head * p.output_head_stride + d0;
    *reinterpret_cast<uint4*>(out) =
        make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]),
                   Elem<T>::pack2(x[4], x[5]), Elem<T>::pack2(x[6], x[7]));
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
        if (position >= p.cache.table_width * kCachePage) {
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
  // Few rows: one row for a CTA, so that a decode batch spreads over the SMs.  Many: 16 rows, so
  // that most CTAs own about one block of every head.
  if (p.offsets == nullptr || p.tokens < 1024) {
    append_kernel<T, D, kInterleaved, 1>
        <<<static_cast<unsigned>(p.tokens), kAppendThreads, 0, stream>>>(p);
  } else {
    append_kernel<T, D, kInterleaved, kCachePage>
        <<<static_cast<unsigned>((static_cast<int64_t>(p.tokens) + kCachePage - 1) / kCachePage),
           kAppendThreads, 0, stream>>>(p);
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
