// Attention over the 8-bit paged K/V cache for runs of tokens (prompts, chunks of them, drafted
// tokens) on the tcgen05 tensor cores; the mathematics is that of attention_q8.cu.
//
// A CTA takes 128 query rows of one kv head: 128 / group consecutive tokens of a sequence times
// the group's query heads, so that every key and value is widened once for all of them, and walks
// the visible pages in steps of 64 tokens.  Two CTAs share an SM (half of tensor memory each): one
// computes exponentials while the other's matrix products, prologue or epilogue run.  Roles:
//   warps 0-3  softmax, one thread for each row: q into tensor memory (F16, a power of two for the
//              row), then for every step the scores out of tensor memory, maximum, weights back
//              into tensor memory over the scores; rescales the accumulator when needed
//   warp 4     issues the products: S = Q K^T (A: q in tensor memory, B: keys, K-major) and
//              O += W V (A: weights in tensor memory, B: values, MN-major: tokens are rows)
//   warps 5-7  widen the codes: 16-byte loads, E4M3 to F16 (exact, the block scales stay out),
//              128-byte swizzled stores; the next step's loads are in flight meanwhile
//
// The running maximum M only stabilises: weights reach up to 2^8 before it is raised (F16 holds
// them, sums are f32), so the accumulator in tensor memory is rescaled a few times for a row and
// not at every step.  A value row of NaN codes (stored whole by the append) becomes zeros in the
// product and NaN scores for the rows that see it, so that it does not reach the rows that do not.
//
// What bounds it: one exponential for each score.  A step of 128 x 64 takes 512 clocks of the SM's
// 16 exponentials per clock and 256 (head_dim 64) of the tensor cores.
#include <type_traits>

#include "attention_q8.cuh"
#include "sm100_primitives.cuh"

namespace nml_sm100 {
namespace {

constexpr int kStepTokens = 64;
constexpr int kStepPages = kStepTokens / kCachePage;
constexpr int kSoftmaxThreads = 128;
constexpr int kMmaWarp = 4;
constexpr int kWidenWarps = 3;
constexpr int kThreads = 256;
constexpr float kSlack = 8.0f;  // log2 of the largest weight before the maximum is raised
constexpr int kTmemColumns = 256;

// Bits 8 + site of the status word say which wait ran out.
constexpr int kSiteScores = 16, kSiteWeights = 17, kSiteTiles = 18, kSiteProduct = 19,
              kSiteFree = 20;

// What the softmax needs to know of a page: score factor, exponent of the values, its inverse
// power for the denominator, first token.
struct alignas(16) PageInfo {
  float key_scale, value_exponent, unscale;
  int token;
};

template <int D>
struct Shape {
  static constexpr int kTileBytes = kStepTokens * D * 2;
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kBuffers = D == 64 ? 2 : 1;  // score buffers in tensor memory
  static constexpr int kOut = 0, kQuery = D, kScores = D + D / 2;
  static constexpr int kSharedBytes = kStages * 2 * kTileBytes + 1024;
  static_assert(kScores + kBuffers * kStepTokens <= kTmemColumns, "tensor memory");
};

template <int D>
struct Control {
  uint64_t tiles_full[Shape<D>::kStages], tiles_free[Shape<D>::kStages];
  uint64_t scores_full[Shape<D>::kBuffers];
  uint64_t query_full, weights_full, product_done, drained;
  uint32_t tmem;
  int abort_flag;
  int sequence, tile;
  PageInfo pages[Shape<D>::kStages][kStepPages];
  alignas(16) uint32_t any_nan[Shape<D>::kStages][4];  // read 16 bytes at a time
  uint8_t row_nan[Shape<D>::kStages][kStepTokens];
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
tile_kernel(const AttentionParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t raw_shared[];
  uint8_t* const shared = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(raw_shared) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ __align__(16) Control<D> control;
  volatile int* const abort_flag = &control.abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_head = blockIdx.x % p.cache.kv_heads;
  const int item = blockIdx.x / p.cache.kv_heads / p.splits;
  const int split = blockIdx.x / p.cache.kv_heads % p.splits;
  const int per_tile = kTileRows / p.group;

  // ---- which sequence, which of its tiles: the last tile (the longest walk) comes first ----
  if (warp == 0) {
    int sequence = -1, tile = 0, passed = 0;
    for (int base = 0; base < p.cache.batch && sequence < 0; base += 32) {
      const int b = base + lane;
      int tiles = 0;
      if (b < p.cache.batch) {
        const int rows = min(p.offsets[b + 1], p.tokens) - max(p.offsets[b], 0);
        tiles = rows > 0 ? (rows + per_tile - 1) / per_tile : 0;
      }
      int upto = tiles;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if (lane >= offset) upto += other;
      }
      const uint32_t holds = __ballot_sync(0xffffffffu, item - passed < upto);
      if (holds != 0) {
        const int at = __ffs(holds) - 1;
        sequence = base + at;
        tile = __shfl_sync(0xffffffffu, upto, at) - 1 - (item - passed);
      }
      passed += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      control.sequence = sequence;
      control.tile = tile;
    }
  }
  if (threadIdx.x == kMmaWarp * 32) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&control.tiles_full[i], kWidenWarps * 32);
      mbar_init(&control.tiles_free[i], 1);
    }
    for (int i = 0; i < S::kBuffers; ++i) mbar_init(&control.scores_full[i], 1);
    mbar_init(&control.query_full, kSoftmaxThreads);
    mbar_init(&control.weights_full, kSoftmaxThreads);
    mbar_init(&control.product_done, 1);
    mbar_init(&control.drained, 1);
    control.abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  const int sequence = control.sequence;
  if (sequence < 0) return;  // more work items than tiles

  const int begin = max(p.offsets[sequence], 0);
  const int end = min(p.offsets[sequence + 1], p.tokens);
  const int first_row = begin + control.tile * per_tile;
  const int rows = min(per_tile, end - first_row);
  const int first_position =
      sequence_length(p.cache, sequence, p.status) - p.offsets[sequence + 1] + first_row;
  const Visible v = visible_pages(first_position + rows,
                                  p.window > 0 ? first_position + 1 - p.window : 0, p.first);
  const int all_steps = (v.pages + kStepPages - 1) / kStepPages;
  const int per_split = (all_steps + p.splits - 1) / p.splits;
  const int step_begin = min(all_steps, split * per_split);
  const int steps = min(all_steps - step_begin, per_split);

  if (warp == kMmaWarp) {
    tmem_alloc(&control.tmem, kTmemColumns);
    tmem_relinquish_alloc_permit();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = control.tmem;

  auto wait = [&](uint64_t* bar, int phase, int site) {
    mbar_wait_or_abort(bar, static_cast<uint32_t>(phase) & 1u, abort_flag, p.status, site);
    __syncwarp();
  };

  if (warp < kMmaWarp) {
    // ------------------------------------------------------------------ softmax
    const int row = threadIdx.x;
    const int token = row / p.group;
    const int head = kv_head * p.group + row - token * p.group;
    const bool live = token < rows;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // rows of nobody walk like the last row, so that they do not ask for masks
    const int length = first_position + 1 + (live ? token : rows - 1);
    const int start = p.window > 0 ? max(0, length - p.window) : 0;

    // q: largest magnitude, then F16 into tensor memory, column c holding elements 2c and 2c + 1
    float factor = p.scale_log2;
    {
      const T* source = static_cast<const T*>(p.query) +
                        static_cast<int64_t>(first_row + token) * p.query_token_stride +
                        head * p.query_head_stride;
      uint32_t largest = 0;
      if constexpr (!std::is_same<T, __half>::value) {
        if (live) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const uint4 x = reinterpret_cast<const uint4*>(source)[i];
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              largest = max(largest, max((words[w] & 0x7fffu) << 16, words[w] & 0x7fff0000u));
            }
          }
        }
      }
      const int shift = std::is_same<T, __half>::value ? 0 : query_shift(largest);
      const float up = exp2_int(shift);
      factor *= exp2_int(-shift);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        uint32_t packed[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (live) x = reinterpret_cast<const uint4*>(source)[2 * i + h];
          const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if constexpr (std::is_same<T, __half>::value) {
              packed[4 * h + w] = words[w];
            } else {
              packed[4 * h + w] = Elem<__half>::pack2(Elem<T>::from_bits(words[w] & 0xffffu) * up,
                                                      Elem<T>::from_bits(words[w] >> 16) * up);
            }
          }
        }
        __syncwarp();
        tmem_store_32x8(lanes + S::kQuery + 8 * i, packed);
      }
      tmem_store_wait();
      tcgen05_fence_before_sync();
      mbar_arrive(&control.query_full);
    }

    float running_max = -INFINITY, running_sum = 0.0f;
    for (int j = 0; j < steps; ++j) {
      const int buffer = j % S::kBuffers, stage = j % S::kStages;
      const uint32_t columns = lanes + S::kScores + buffer * kStepTokens;
      wait(&control.scores_full[buffer], j / S::kBuffers, kSiteScores);
      tcgen05_fence_after_sync();
      // long complete; orders the reads of the stage's page data behind their writes
      wait(&control.tiles_full[stage], j / S::kStages, kSiteTiles);
      float s[kStepTokens];
      {
        uint32_t x[32];
        tmem_load_32x32(columns, x);
        tmem_load_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(x[i]);
        tmem_load_32x32(columns + 32, x);
        tmem_load_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) s[32 + i] = __uint_as_float(x[i]);
      }
      const uint4 nan_words = *reinterpret_cast<const uint4*>(control.any_nan[stage]);
      bool whole = (nan_words.x | nan_words.y | nan_words.z) == 0;
#pragma unroll
      for (int q = 0; q < kStepPages; ++q) {
        const int t = control.pages[stage][q].token;
        whole = whole && t + kCachePage <= length && (t >= start || t + kCachePage <= p.first);
      }
      if (!__all_sync(0xffffffffu, whole)) {
#pragma unroll
        for (int q = 0; q < kStepPages; ++q) {
          const int t = control.pages[stage][q].token;
#pragma unroll
          for (int i = 0; i < kCachePage; ++i) {
            const bool seen = t + i < length && (t + i >= start || t + i < p.first);
            const bool nan = control.row_nan[stage][q * kCachePage + i] != 0;
            s[q * kCachePage + i] =
                seen ? (nan ? __uint_as_float(0x7fc00000u) : s[q * kCachePage + i]) : -INFINITY;
          }
        }
      }
      float page_factor[kStepPages];
      float top = -INFINITY;
#pragma unroll
      for (int q = 0; q < kStepPages; ++q) {
        float m = s[q * kCachePage];
#pragma unroll
        for (int i = 1; i < kCachePage; ++i) m = fmaxf(m, s[q * kCachePage + i]);
        page_factor[q] = factor * control.pages[stage][q].key_scale;
        top = fmaxf(top, fmaf(m, page_factor[q], control.pages[stage][q].value_exponent));
      }
      // raise the maximum only when the weights would leave F16's comfortable range
      const bool raise = top > running_max + kSlack;  // also from -infinity
      if (__any_sync(0xffffffffu, raise)) {
        const float next = raise ? top : running_max;
        const float rescale = raise ? exp2_fast(running_max - next) : 1.0f;
        if (j > 0) {
          wait(&control.product_done, j - 1, kSiteProduct);
          tcgen05_fence_after_sync();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t x[16], y[8], z[8];
            tmem_load_32x16(lanes + S::kOut + c, x);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y[i] = __float_as_uint(__uint_as_float(x[i]) * rescale);
              z[i] = __float_as_uint(__uint_as_float(x[i + 8]) * rescale);
            }
            tmem_store_32x8(lanes + S::kOut + c, y);
            tmem_store_32x8(lanes + S::kOut + c + 8, z);
          }
        }
        running_sum *= rescale;
        running_max = next;
      }
      const float base = running_max == -INFINITY ? 0.0f : running_max;
#pragma unroll
      for (int q = 0; q < kStepPages; ++q) {
        const float offset = control.pages[stage][q].value_exponent - base;
        uint32_t packed[8];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = exp2_fast(fmaf(s[q * kCachePage + 2 * i], page_factor[q], offset));
          const float b = exp2_fast(fmaf(s[q * kCachePage + 2 * i + 1], page_factor[q], offset));
          sum += a + b;
          packed[i] = Elem<__half>::pack2(a, b);
        }
        running_sum = fmaf(sum, control.pages[stage][q].unscale, running_sum);
        tmem_store_32x8(columns + 8 * q, packed);
      }
      tmem_store_wait();
      tcgen05_fence_before_sync();
      mbar_arrive(&control.weights_full);
    }

    // ---- the rows' results ----
    if (steps > 0) {
      wait(&control.product_done, steps - 1, kSiteProduct);
      tcgen05_fence_after_sync();
    }
    const int64_t query_head = static_cast<int64_t>(first_row + token) * p.query_heads + head;
    float denominator = running_sum;
    if (p.sinks != nullptr && live) {
      denominator += exp2f(p.sinks[head] * kLog2e - running_max);
    }
    // only a row that sees nothing has a sum of exactly zero; its output is zero
    const float inverse = running_sum == 0.0f ? 0.0f : 1.0f / denominator;
    float* partial = p.partial + (query_head * p.splits + split) * (D + 2);
    T* out = static_cast<T*>(p.output) + query_head * D;
#pragma unroll
    for (int c = 0; c < D; c += 16) {
      uint32_t x[16];
      if (steps > 0) {
        tmem_load_32x16(lanes + S::kOut + c, x);
        tmem_load_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0;
      }
      if (live && p.splits > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          *reinterpret_cast<uint2*>(partial + c + i) = make_uint2(x[i], x[i + 1]);
        }
      } else if (live) {
        uint32_t packed[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          packed[i] = Elem<T>::pack2(__uint_as_float(x[2 * i]) * inverse,
                                     __uint_as_float(x[2 * i + 1]) * inverse);
        }
        reinterpret_cast<uint4*>(out + c)[0] =
            make_uint4(packed[0], packed[1], packed[2], packed[3]);
        reinterpret_cast<uint4*>(out + c)[1] =
            make_uint4(packed[4], packed[5], packed[6], packed[7]);
      }
      __syncwarp();
    }
    if (live && p.splits > 1) {
      *reinterpret_cast<float2*>(partial + D) = make_float2(running_max, running_sum);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------------ matrix products
    constexpr uint64_t desc_hi = static_cast<uint64_t>(kUmmaDescHiSw128) << 32;
    constexpr uint32_t score_idesc = umma_idesc_f16(kUmmaF16, kUmmaF16, kTileRows, kStepTokens);
    constexpr uint32_t product_idesc =
        umma_idesc_f16(kUmmaF16, kUmmaF16, kTileRows, D) | (1u << 16);  // B is MN-major
    auto scores = [&](int j) {
      const int stage = j % S::kStages, buffer = j % S::kBuffers;
      wait(&control.tiles_full[stage], j / S::kStages, kSiteTiles);
      tcgen05_fence_after_sync();
      const uint32_t keys = smem_u32(shared + stage * 2 * S::kTileBytes);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        // 64-element halves of the head are tiles of their own, 16 elements are 32 bytes of a row
        const uint32_t address = keys + (k / 4) * (kStepTokens * 128) + (k % 4) * 32;
        umma_f16_tmem_a_elect(tmem + S::kScores + buffer * kStepTokens, tmem + S::kQuery + 8 * k,
                              desc_hi | umma_desc_lo(address), score_idesc, k > 0 ? 1u : 0u);
      }
      umma_commit_elect(&control.scores_full[buffer]);
    };
    if (steps > 0) {
      wait(&control.query_full, 0, kSiteWeights);
      tcgen05_fence_after_sync();
      for (int j = 0; j < min(steps, S::kBuffers); ++j) scores(j);
    }
    for (int j = 0; j < steps; ++j) {
      const int stage = j % S::kStages, buffer = j % S::kBuffers;
      wait(&control.weights_full, j, kSiteWeights);
      tcgen05_fence_after_sync();
      const uint32_t values = smem_u32(shared + stage * 2 * S::kTileBytes + S::kTileBytes);
#pragma unroll
      for (int k = 0; k < kStepTokens / 16; ++k) {
        // 16 tokens are 2 KB of 128-byte rows; the leading offset is the next 64 dimensions' tile
        const uint32_t address = values + k * 2048;
        const uint32_t low = ((address & 0x3ffffu) >> 4) | ((kStepTokens * 128 >> 4) << 16);
        umma_f16_tmem_a_elect(tmem + S::kOut, tmem + S::kScores + buffer * kStepTokens + 8 * k,
                              desc_hi | low, product_idesc, j > 0 || k > 0 ? 1u : 0u);
      }
      umma_commit_elect(&control.tiles_free[stage]);
      umma_commit_elect(&control.product_done);
      if (j + S::kBuffers < steps) {
        // the scores go over the weights that this product reads
        wait(&control.product_done, j, kSiteProduct);
        scores(j + S::kBuffers);
      }
    }
    umma_commit_elect(&control.drained);
    if (!mbar_wait(&control.drained, 0)) {
      *abort_flag = 1;
      atomicOr(p.status, NML_SM100_STATUS_BARRIER_TIMEOUT | (0x100 << kSiteProduct));
    }
  } else {
    // ------------------------------------------------------------------ codes to F16 tiles
    constexpr int kWidenThreads = kWidenWarps * 32;
    constexpr int kRowPieces = D / 16;                  // pieces of 16 codes of a token's row
    constexpr int kHalf = kStepTokens * kRowPieces;     // pieces of the keys (then of the values)
    constexpr int kRounds = (2 * kHalf + kWidenThreads - 1) / kWidenThreads;
    const int thread = threadIdx.x - (kMmaWarp + 1) * 32;
    const int widen_warp = warp - kMmaWarp - 1;

    // lane q < 4 holds what page q of a step is: its block (-1: nothing there) and scale bytes
    int64_t block = -1;
    PageInfo info;
    auto look_up = [&](int j) {
      block = -1;
      info = PageInfo{0.0f, -INFINITY, 0.0f, -kStepTokens};  // a page of nobody: weights of zero
      const int i = (step_begin + j) * kStepPages + lane;
      if (lane < kStepPages && j < steps && i < v.pages) {
        const int logical = i < v.front ? i : i - v.front + v.back;
        const int page = physical_page(p.cache, sequence, logical, p.status);
        if (page >= 0) {
          block = static_cast<int64_t>(page) * p.cache.kv_heads + kv_head;
          const int e = scale_exponent(p.cache.scales[1][block]);
          info = PageInfo{exp2_int(scale_exponent(p.cache.scales[0][block])),
                          static_cast<float>(e), exp2_int(-e), logical * kCachePage};
        }
      }
    };
    uint4 codes[kRounds];
    auto load = [&](uint4 (&to)[kRounds]) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int piece = r * kWidenThreads + thread;
        const int within = piece % kHalf;
        const int token = within / kRowPieces;
        const int64_t b = __shfl_sync(0xffffffffu, block, token / kCachePage);
        to[r] = make_uint4(0, 0, 0, 0);
        if (piece < 2 * kHalf && b >= 0) {
          const uint8_t* base = piece < kHalf ? p.cache.codes[0] : p.cache.codes[1];
          to[r] = *reinterpret_cast<const uint4*>(base + b * (kCachePage * D) +
                                                  (token % kCachePage) * D +
                                                  (within % kRowPieces) * 16);
        }
      }
    };
    look_up(0);
    load(codes);
    for (int j = 0; j < steps; ++j) {
      const int stage = j % S::kStages;
      const PageInfo current = info;
      look_up(j + 1);
      uint4 next[kRounds];
      load(next);
      if (j >= S::kStages) wait(&control.tiles_free[stage], j / S::kStages - 1, kSiteFree);
      uint8_t* const tiles = shared + stage * 2 * S::kTileBytes;
      bool any_nan = false;
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const int piece = r * kWidenThreads + thread;
        const int within = piece % kHalf;
        const int token = within / kRowPieces, part = within % kRowPieces;
        uint4 x = codes[r];
        const int page_token =
            __shfl_sync(0xffffffffu, current.token, token / kCachePage) + token % kCachePage;
        const uint32_t first_code = __shfl_sync(0xffffffffu, x.x, lane & ~(kRowPieces - 1));
        if (piece < 2 * kHalf) {
          if (piece >= kHalf) {
            // values that no row sees, or that are NaN, must not meet the product
            const bool nan = (first_code & 0x7fu) == 0x7fu && page_token < v.length;
            if (nan || page_token >= v.length) x = make_uint4(0, 0, 0, 0);
            if (part == 0) control.row_nan[stage][token] = nan ? 1 : 0;
            any_nan = any_nan || nan;
          }
          uint8_t* const tile = tiles + (piece < kHalf ? 0 : S::kTileBytes) +
                                (part / 4) * (kStepTokens * 128) + token * 128;
          const int chunk = 2 * (part % 4);
          *reinterpret_cast<uint4*>(tile + ((chunk ^ (token & 7)) * 16)) =
              make_uint4(e4m3x2_to_f16x2(x.x & 0xffffu), e4m3x2_to_f16x2(x.x >> 16),
                         e4m3x2_to_f16x2(x.y & 0xffffu), e4m3x2_to_f16x2(x.y >> 16));
          *reinterpret_cast<uint4*>(tile + (((chunk + 1) ^ (token & 7)) * 16)) =
              make_uint4(e4m3x2_to_f16x2(x.z & 0xffffu), e4m3x2_to_f16x2(x.z >> 16),
                         e4m3x2_to_f16x2(x.w & 0xffffu), e4m3x2_to_f16x2(x.w >> 16));
        }
      }
      any_nan = __any_sync(0xffffffffu, any_nan);
      if (lane == 0) control.any_nan[stage][widen_warp] = any_nan ? 1u : 0u;
      if (widen_warp == 0 && lane < kStepPages) control.pages[stage][lane] = current;
      fence_proxy_async_smem();
      mbar_arrive(&control.tiles_full[stage]);
#pragma unroll
      for (int r = 0; r < kRounds; ++r) codes[r] = next[r];
    }
  }

  tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

}  // namespace

template <typename T, int D>
int32_t launch_tiles(const AttentionParams& p, cudaStream_t stream, char* message,
                     size_t capacity) {
  if (cudaFuncSetAttribute(tile_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           Shape<D>::kSharedBytes) != cudaSuccess ||
      cudaFuncSetAttribute(tile_kernel<T, D>, cudaFuncAttributePreferredSharedMemoryCarveout,
                           cudaSharedmemCarveoutMaxShared) != cudaSuccess) {
    return fail(NML_SM100_LAUNCH_FAILURE, "cannot configure shared memory", message, capacity);
  }
  const int64_t items = query_tiles(p.tokens, p.cache.batch, p.group);
  tile_kernel<T, D><<<static_cast<unsigned>(items * p.splits * p.cache.kv_heads), kThreads,
                      Shape<D>::kSharedBytes, stream>>>(p);
  return NML_SM100_OK;
}

template int32_t launch_tiles<__half, 64>(const AttentionParams&, cudaStream_t, char*, size_t);
template int32_t launch_tiles<__half, 128>(const AttentionParams&, cudaStream_t, char*, size_t);
template int32_t launch_tiles<__nv_bfloat16, 64>(const AttentionParams&, cudaStream_t, char*,
                                                 size_t);
template int32_t launch_tiles<__nv_bfloat16, 128>(const AttentionParams&, cudaStream_t, char*,
                                                  size_t);

}  // namespace nml_sm100
